// attention_rope.cu -- new tokens' queries, keys and values into attention
// over a cache of shares, for both parties on one GPU: the rotary positions,
// the truncation after them and the masked opens in one pass.
//
// Per token and head, with the public cosine c and sine s of its position (f
// fractional bits), each party rotates its own shares,
//   y1 = x1 c - x2 s,  y2 = x2 c + x1 s   (mod 2^64, 2f fractional bits);
// y^ = sum_p (y_p + r_p) is opened and every party takes its GapARS share of
// floor(y / 2^f) (the truncation bundle's postproc, with the carry's
// predicate shares read from the bundle's full-domain tables).  Words past
// the rotated part keep their share.  What leaves is opened again:
//   queries: D = sum_p (q'_p - A_p)              (the scores' left operand)
//   keys:    E[slot] = sum_p (k'_p - B_p[slot])  (into the cache's pages)
//   values:  E[slot] = sum_p (v_p - B_p[slot]).
#include "attention.hpp"
#include "prefix.cuh"

namespace sufb200 {

namespace {

constexpr int kThreads = 256;
int fail(int code, const std::string& msg) { return record_error(code, msg); }

// A party's GapARS share of floor(y / 2^f) from the opened y^ and its carry
// share (GapArsPostProc::run_batch, include/gates/postproc_hooks.hpp:324-375).
__device__ __forceinline__ uint64_t gapars_share(const sufb200_trunc_desc& d, uint64_t yhat, uint64_t carry) {
  const int f = d.frac_bits;
  const uint64_t hb = yhat + (1ull << 62);
  uint64_t y = d.haty - d.r_hi - carry;
  if (d.party == 0) y += (hb >> f) - (1ull << (62 - f));
  if ((hb >> 63) == 0) y += d.m;
  return y;
}

// A party's share of the carry out of the low f bits (the AddU64 plan of
// composite_eval_batch_backend, include/gates/composite_fss.hpp:1539-1605).
__device__ __forceinline__ uint64_t carry_share(const sufb200_trunc_desc& d, const void* tables, uint64_t yhat) {
  if (d.carry_a < 0) return 0;  // the mask's low bits are zero: no carry
  const uint64_t x = yhat & ((1ull << d.frac_bits) - 1);
  const auto* entry = reinterpret_cast<const FrontierEntry*>(static_cast<const uint8_t*>(tables) + kTruncTablesHead);
  const uint64_t qa = __ldg(&entry[(static_cast<uint64_t>(d.carry_a) << d.frac_bits) + x].v);
  const uint64_t qb = __ldg(&entry[(static_cast<uint64_t>(d.carry_b) << d.frac_bits) + x].v);
  return (d.party == 0 ? 1ull : 0ull) - ((qb - qa) + d.carry_w);
}

// sum_p of the parties' truncated shares.
__device__ __forceinline__ uint64_t trunc_open(const sufb200_rope_append& a, uint64_t y0, uint64_t y1) {
  const uint64_t yhat = (y0 + a.r[0]) + (y1 + a.r[1]);
  return gapars_share(a.trunc[0], yhat, carry_share(a.trunc[0], a.d_tables[0], yhat)) +
         gapars_share(a.trunc[1], yhat, carry_share(a.trunc[1], a.d_tables[1], yhat));
}

__global__ void __launch_bounds__(kThreads) rope_append_kernel(const __grid_constant__ sufb200_rope_append a,
                                                               uint32_t* status) {
  const int P = a.head_dim / 2, half = a.rot_dim / 2, heads = a.q_heads + 2 * a.kv_heads;
  const int64_t total = static_cast<int64_t>(a.tokens) * heads * P;
  for (int64_t w = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; w < total;
       w += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int p = static_cast<int>(w % P);
    const int hh = static_cast<int>((w / P) % heads), t = static_cast<int>(w / P / heads);
    const int64_t slot = a.d_slots[t];
    if (slot == -1) continue;  // a padding token
    const bool is_q = hh < a.q_heads, is_v = hh >= a.q_heads + a.kv_heads, turn = !is_v && p < half;
    const int pos = turn ? a.d_positions[t] : 0;
    if (slot < 0 || slot >= static_cast<int64_t>(a.pages) * a.page_size || (turn && (pos < 0 || pos >= a.max_pos))) {
      atomicOr(status, kStatusBadArgument);
      continue;
    }
    const int d1 = turn && !a.interleaved ? p : 2 * p, d2 = turn && !a.interleaved ? p + half : 2 * p + 1;
    const int h = is_q ? hh : (is_v ? hh - a.q_heads - a.kv_heads : hh - a.q_heads);
    const int64_t at = is_q ? t * a.q_ts + h * a.q_hs : (is_v ? t * a.v_ts + h * a.v_hs : t * a.k_ts + h * a.k_hs);
    const uint64_t* x0 = (is_q ? a.d_q[0] : (is_v ? a.d_v[0] : a.d_k[0])) + at;
    const uint64_t* x1 = (is_q ? a.d_q[1] : (is_v ? a.d_v[1] : a.d_k[1])) + at;
    const uint64_t u0 = x0[d1], w0 = x0[d2], u1 = x1[d1], w1 = x1[d2];
    uint64_t z1, z2;
    if (turn) {
      const int64_t ci = static_cast<int64_t>(pos) * half + p;
      const uint64_t c = static_cast<uint64_t>(static_cast<int64_t>(a.d_cos[ci]));
      const uint64_t s = static_cast<uint64_t>(static_cast<int64_t>(a.d_sin[ci]));
      z1 = trunc_open(a, u0 * c - w0 * s, u1 * c - w1 * s);
      z2 = trunc_open(a, w0 * c + u0 * s, w1 * c + u1 * s);
    } else {
      z1 = u0 + u1;
      z2 = w0 + w1;
    }
    if (is_q) {
      const int64_t o = (static_cast<int64_t>(t) * a.q_heads + h) * a.head_dim;
      a.d_dq[o + d1] = z1 - a.d_a[0][o + d1] - a.d_a[1][o + d1];
      a.d_dq[o + d2] = z2 - a.d_a[0][o + d2] - a.d_a[1][o + d2];
    } else {
      const int64_t pg = slot / a.page_size;
      const int64_t o = ((pg * a.kv_heads + h) * a.page_size + slot % a.page_size) * a.head_dim;
      uint64_t* e = is_v ? a.d_ev : a.d_ek;
      const uint64_t* b0 = is_v ? a.d_bv[0] : a.d_bk[0];
      const uint64_t* b1 = is_v ? a.d_bv[1] : a.d_bk[1];
      e[o + d1] = z1 - b0[o + d1] - b1[o + d1];
      e[o + d2] = z2 - b0[o + d2] - b1[o + d2];
    }
  }
}

int check_rope(const sufb200_rope_append* a) {
  if (!a) return fail(SUFB200_ERR_INVALID, "rope_append_pair: null arguments");
  if (a->tokens < 0 || a->q_heads < 0 || a->kv_heads < 1 || a->pages < 1 || a->page_size < 1)
    return fail(SUFB200_ERR_INVALID, "rope_append_pair: bad token, head or page count");
  if (a->head_dim < 2 || a->head_dim > 256 || a->head_dim % 2)
    return fail(SUFB200_ERR_UNSUPPORTED, "rope_append_pair: head size must be even, 2..256");
  if (a->rot_dim < 0 || a->rot_dim > a->head_dim || a->rot_dim % 2)
    return fail(SUFB200_ERR_INVALID, "rope_append_pair: the rotated part must be even and within the head");
  if (a->tokens == 0) return SUFB200_OK;
  if (!a->d_slots) return fail(SUFB200_ERR_INVALID, "rope_append_pair: null slots");
  for (int p = 0; p < 2; p++) {
    if (!a->d_k[p] || !a->d_v[p] || !a->d_bk[p] || !a->d_bv[p] || (a->q_heads > 0 && (!a->d_q[p] || !a->d_a[p])))
      return fail(SUFB200_ERR_INVALID, "rope_append_pair: null share or mask pointer");
    for (const void* v : {static_cast<const void*>(a->d_k[p]), static_cast<const void*>(a->d_v[p]),
                          static_cast<const void*>(a->d_bk[p]), static_cast<const void*>(a->d_bv[p]),
                          static_cast<const void*>(a->q_heads ? a->d_q[p] : nullptr),
                          static_cast<const void*>(a->q_heads ? a->d_a[p] : nullptr)})
      if (!aligned_to(v, 8)) return fail(SUFB200_ERR_INVALID, "rope_append_pair: misaligned share or mask pointer");
  }
  if (!a->d_ek || !a->d_ev || (a->q_heads > 0 && !a->d_dq) || !aligned_to(a->d_ek, 8) || !aligned_to(a->d_ev, 8) ||
      (a->q_heads > 0 && !aligned_to(a->d_dq, 8)))
    return fail(SUFB200_ERR_INVALID, "rope_append_pair: null or misaligned output");
  if (a->rot_dim > 0) {
    if (!a->d_positions || !a->d_cos || !a->d_sin || a->max_pos < 1)
      return fail(SUFB200_ERR_INVALID, "rope_append_pair: positions or cosine and sine tables missing");
    for (int p = 0; p < 2; p++) {
      const sufb200_trunc_desc& d = a->trunc[p];
      if (d.kind != SUFB200_TRUNC_GAPARS || d.party != p || d.frac_bits < 1 || d.frac_bits > 16 ||
          d.frac_bits != a->trunc[0].frac_bits)
        return fail(SUFB200_ERR_INVALID, "rope_append_pair: needs both parties' GapARS bundle of 1..16 fractional bits");
      if (d.carry_a < 0) continue;
      if (d.nq < 1 || d.nq > 4 || d.carry_a >= d.nq || d.carry_b < 0 || d.carry_b >= d.nq)
        return fail(SUFB200_ERR_INVALID, "rope_append_pair: bad truncation plan");
      for (int q = 0; q < d.nq; q++)
        if (d.q_bits[q] != d.frac_bits) return fail(SUFB200_ERR_INVALID, "rope_append_pair: bad truncation plan");
      if (!a->d_tables[p] || !aligned_to(a->d_tables[p], 256))
        return fail(SUFB200_ERR_INVALID, "rope_append_pair: the bundle's tables are missing or misaligned");
    }
  }
  return SUFB200_OK;
}

}  // namespace

}  // namespace sufb200

using namespace sufb200;

extern "C" int sufb200_rope_append_pair(sufb200_ctx ctx, const sufb200_rope_append* args, void* stream) {
  if (int rc = check_rope(args)) return rc;
  if (args->tokens == 0) return SUFB200_OK;
  if (int rc = attn_check_ctx(ctx)) return rc;
  const int64_t total = static_cast<int64_t>(args->tokens) * (args->q_heads + 2 * args->kv_heads) * (args->head_dim / 2);
  const int64_t want = (total + kThreads - 1) / kThreads, cap = static_cast<int64_t>(ctx->sm_count) * 8;
  rope_append_kernel<<<static_cast<unsigned>(want < cap ? want : cap), kThreads, 0,
                       reinterpret_cast<cudaStream_t>(stream)>>>(*args, ctx->d_status);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SUFB200_OK : fail(SUFB200_ERR_CUDA, std::string("rope_append_pair: ") + cudaGetErrorString(e));
}

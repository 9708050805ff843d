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
// Bound by memory: 4,133 tokens, 32 / 8 heads of 128, all words turned, move
// 1.02 GB in 167 us (6.1 TB/s of 6.5); with the words of a token dealt out one
// by one and four gathers from the bundle's tables each it took 437 us.
#include "attention.hpp"
#include "prefix.cuh"

namespace sufb200 {

namespace {

constexpr int kThreads = 256;
int fail(int code, const std::string& msg) { return record_error(code, msg); }

// Everything of the two parties' GapARS postproc that does not depend on the
// element (GapArsPostProc::run_batch, include/gates/postproc_hooks.hpp:
// 324-375): with h = y^ + 2^62,
//   sum_p share_p = base + (h >> f) - sum_p carry_p [+ m when h < 2^63].
struct GapArs {
  uint64_t base;  // sum_p (haty_p - r_hi_p) - 2^(62 - f)
  uint64_t m;     // sum_p m_p
  uint64_t r;     // sum_p r_p
  int f;
};

// A party's share of the carry out of the low f bits of y^ (the AddU64 plan of
// composite_eval_batch_backend, include/gates/composite_fss.hpp:1539-1605),
// its two predicate shares read from the bundle's full-domain tables.
__device__ __forceinline__ uint64_t carry_share(const sufb200_trunc_desc& d, const void* tables, uint32_t x) {
  if (d.carry_a < 0) return 0;  // the mask's low bits are zero: no carry
  const auto* entry = reinterpret_cast<const FrontierEntry*>(static_cast<const uint8_t*>(tables) + kTruncTablesHead);
  const uint64_t qa = __ldg(&entry[(static_cast<uint64_t>(d.carry_a) << d.frac_bits) + x].v);
  const uint64_t qb = __ldg(&entry[(static_cast<uint64_t>(d.carry_b) << d.frac_bits) + x].v);
  return (d.party == 0 ? 1ull : 0ull) - ((qb - qa) + d.carry_w);
}

__device__ __forceinline__ uint64_t carry_both(const sufb200_rope_append& a, uint32_t x) {
  return carry_share(a.trunc[0], a.d_tables[0], x) + carry_share(a.trunc[1], a.d_tables[1], x);
}

// The carry shares of every low part, both parties', as one packed table.
__global__ void carry_table_kernel(const __grid_constant__ sufb200_rope_append a, uint64_t* __restrict__ table) {
  pdl_trigger();
  const uint32_t n = 1u << a.trunc[0].frac_bits;
  for (uint32_t x = blockIdx.x * blockDim.x + threadIdx.x; x < n; x += gridDim.x * blockDim.x)
    table[x] = carry_both(a, x);
}

// A warp per (token, head): its lanes hold the head's pairs, two neighbouring
// pairs a lane with 16-byte accesses when VEC (every row 16-byte aligned and
// the pairs' halves at even words), one pair with 8-byte accesses otherwise.
// PACKED: the carries come from carry_table_kernel's table (32 KB at 12 bits:
// L1 holds it), else from the bundle's own tables.
template <bool PACKED, bool VEC>
__global__ void __launch_bounds__(kThreads) rope_append_kernel(const __grid_constant__ sufb200_rope_append a,
                                                               const GapArs g, const uint64_t* __restrict__ table,
                                                               uint32_t* status) {
  if (PACKED) pdl_wait();
  const auto open = [&](uint64_t y0, uint64_t y1) {  // sum_p of the truncated shares of y
    const uint64_t yhat = y0 + y1 + g.r, h = yhat + (1ull << 62);
    const uint32_t x = static_cast<uint32_t>(yhat) & ((1u << g.f) - 1);
    const uint64_t carry = PACKED ? __ldg(table + x) : carry_both(a, x);
    return g.base + (h >> g.f) - carry + ((h >> 63) == 0 ? g.m : 0);
  };
  const int half = a.rot_dim / 2, heads = a.q_heads + 2 * a.kv_heads, lane = threadIdx.x & 31;
  const int64_t rows = static_cast<int64_t>(a.tokens) * heads, step = static_cast<int64_t>(gridDim.x) * (kThreads / 32);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5); row < rows; row += step) {
    const int t = static_cast<int>(row / heads), hh = static_cast<int>(row - static_cast<int64_t>(t) * heads);
    const int64_t slot = a.d_slots[t];
    if (slot == -1) continue;  // a padding token
    const bool is_q = hh < a.q_heads, is_v = hh >= a.q_heads + a.kv_heads;
    const int turned = is_v ? 0 : half;  // pairs of this head that turn
    const int pos = turned ? a.d_positions[t] : 0;
    if (slot < 0 || slot >= static_cast<int64_t>(a.pages) * a.page_size || (turned && (pos < 0 || pos >= a.max_pos))) {
      if (lane == 0) atomicOr(status, kStatusBadArgument);
      continue;
    }
    // the head's shares, the masks it is opened against and where it goes
    const uint64_t *x0, *x1, *m0, *m1;
    uint64_t* out;
    if (is_q) {
      const int64_t at = t * a.q_ts + hh * a.q_hs, o = row - static_cast<int64_t>(t) * 2 * a.kv_heads;
      x0 = a.d_q[0] + at;
      x1 = a.d_q[1] + at;
      m0 = a.d_a[0] + o * a.head_dim;
      m1 = a.d_a[1] + o * a.head_dim;
      out = a.d_dq + o * a.head_dim;
    } else {
      const int h = is_v ? hh - a.q_heads - a.kv_heads : hh - a.q_heads;
      const int64_t at = is_v ? t * a.v_ts + h * a.v_hs : t * a.k_ts + h * a.k_hs;
      const int64_t pg = slot / a.page_size;
      const int64_t o = ((pg * a.kv_heads + h) * a.page_size + (slot - pg * a.page_size)) * a.head_dim;
      x0 = (is_v ? a.d_v[0] : a.d_k[0]) + at;
      x1 = (is_v ? a.d_v[1] : a.d_k[1]) + at;
      m0 = (is_v ? a.d_bv[0] : a.d_bk[0]) + o;
      m1 = (is_v ? a.d_bv[1] : a.d_bk[1]) + o;
      out = (is_v ? a.d_ev : a.d_ek) + o;
    }
    const int32_t* cs = a.d_cos + static_cast<int64_t>(pos) * half;
    const int32_t* sn = a.d_sin + static_cast<int64_t>(pos) * half;
    if (VEC) {
      // a lane's four words: interleaved and unturned, four neighbours; else
      // two of the first half of the turned part and their partners
      for (int p = 2 * lane; p < a.head_dim / 2; p += 64) {
        const bool turn = p < turned;
        const int d1 = turn && !a.interleaved ? p : 2 * p, d2 = turn && !a.interleaved ? p + half : 2 * p + 2;
        const ulonglong2 u0 = *reinterpret_cast<const ulonglong2*>(x0 + d1), w0 = *reinterpret_cast<const ulonglong2*>(x0 + d2);
        const ulonglong2 u1 = *reinterpret_cast<const ulonglong2*>(x1 + d1), w1 = *reinterpret_cast<const ulonglong2*>(x1 + d2);
        const ulonglong2 ma = *reinterpret_cast<const ulonglong2*>(m0 + d1), mb = *reinterpret_cast<const ulonglong2*>(m0 + d2);
        const ulonglong2 na = *reinterpret_cast<const ulonglong2*>(m1 + d1), nb = *reinterpret_cast<const ulonglong2*>(m1 + d2);
        ulonglong2 z1, z2;
        if (turn) {
          const int2 ci = *reinterpret_cast<const int2*>(cs + p), si = *reinterpret_cast<const int2*>(sn + p);
          const uint64_t ca = static_cast<uint64_t>(static_cast<int64_t>(ci.x)), sa = static_cast<uint64_t>(static_cast<int64_t>(si.x));
          const uint64_t cb = static_cast<uint64_t>(static_cast<int64_t>(ci.y)), sb = static_cast<uint64_t>(static_cast<int64_t>(si.y));
          if (a.interleaved) {  // pairs (u.x, u.y) and (w.x, w.y)
            z1.x = open(u0.x * ca - u0.y * sa, u1.x * ca - u1.y * sa);
            z1.y = open(u0.y * ca + u0.x * sa, u1.y * ca + u1.x * sa);
            z2.x = open(w0.x * cb - w0.y * sb, w1.x * cb - w1.y * sb);
            z2.y = open(w0.y * cb + w0.x * sb, w1.y * cb + w1.x * sb);
          } else {  // pairs (u.x, w.x) and (u.y, w.y)
            z1.x = open(u0.x * ca - w0.x * sa, u1.x * ca - w1.x * sa);
            z2.x = open(w0.x * ca + u0.x * sa, w1.x * ca + u1.x * sa);
            z1.y = open(u0.y * cb - w0.y * sb, u1.y * cb - w1.y * sb);
            z2.y = open(w0.y * cb + u0.y * sb, w1.y * cb + u1.y * sb);
          }
        } else {
          z1 = make_ulonglong2(u0.x + u1.x, u0.y + u1.y);
          z2 = make_ulonglong2(w0.x + w1.x, w0.y + w1.y);
        }
        *reinterpret_cast<ulonglong2*>(out + d1) = make_ulonglong2(z1.x - ma.x - na.x, z1.y - ma.y - na.y);
        *reinterpret_cast<ulonglong2*>(out + d2) = make_ulonglong2(z2.x - mb.x - nb.x, z2.y - mb.y - nb.y);
      }
    } else {
      for (int p = lane; p < a.head_dim / 2; p += 32) {
        const bool turn = p < turned;
        const int d1 = turn && !a.interleaved ? p : 2 * p, d2 = turn && !a.interleaved ? p + half : 2 * p + 1;
        const uint64_t u0 = x0[d1], w0 = x0[d2], u1 = x1[d1], w1 = x1[d2];
        uint64_t z1 = u0 + u1, z2 = w0 + w1;
        if (turn) {
          const uint64_t c = static_cast<uint64_t>(static_cast<int64_t>(cs[p]));
          const uint64_t s = static_cast<uint64_t>(static_cast<int64_t>(sn[p]));
          z1 = open(u0 * c - w0 * s, u1 * c - w1 * s);
          z2 = open(w0 * c + u0 * s, w1 * c + u1 * s);
        }
        out[d1] = z1 - m0[d1] - m1[d1];
        out[d2] = z2 - m0[d2] - m1[d2];
      }
    }
  }
}

int check_rope(const sufb200_rope_append* a) {
  if (!a) return fail(SUFB200_ERR_INVALID, "rope_append_pair: null arguments");
  if (a->tokens < 0 || a->q_heads < 0 || a->kv_heads < 1 || a->pages < 1 || a->page_size < 1)
    return fail(SUFB200_ERR_INVALID, "rope_append_pair: bad token, head or page count");
  if (a->head_dim < 2 || a->head_dim > 256 || a->head_dim % 2)
    return fail(SUFB200_ERR_UNSUPPORTED, "rope_append_pair: head size must be even, 2..256");
  if (a->q_heads + 2 * static_cast<int64_t>(a->kv_heads) > INT32_MAX)
    return fail(SUFB200_ERR_UNSUPPORTED, "rope_append_pair: more than 2^31 heads of a token");
  if (a->rot_dim < 0 || a->rot_dim > a->head_dim || a->rot_dim % 2)
    return fail(SUFB200_ERR_INVALID, "rope_append_pair: the rotated part must be even and within the head");
  if (a->tokens == 0) return SUFB200_OK;
  if (!a->d_slots || !aligned_to(a->d_slots, 8))
    return fail(SUFB200_ERR_INVALID, "rope_append_pair: null or misaligned slots");
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
    if (!aligned_to(a->d_positions, 4) || !aligned_to(a->d_cos, 4) || !aligned_to(a->d_sin, 4))
      return fail(SUFB200_ERR_INVALID, "rope_append_pair: misaligned positions or tables");
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

// Every 16-byte access of the paired form aligned, its four words of one kind:
// pairs p, p + 1 with p even turn together and (half layout) start at even words.
bool paired(const sufb200_rope_append& a) {
  const int half = a.rot_dim / 2;
  bool ok = a.head_dim % 4 == 0 && half % 2 == 0 && a.q_ts % 2 == 0 && a.q_hs % 2 == 0 && a.k_ts % 2 == 0 &&
            a.k_hs % 2 == 0 && a.v_ts % 2 == 0 && a.v_hs % 2 == 0 && aligned_to(a.d_cos, 8) && aligned_to(a.d_sin, 8) &&
            aligned_to(a.d_ek, 16) && aligned_to(a.d_ev, 16) && (a.q_heads == 0 || aligned_to(a.d_dq, 16));
  for (int p = 0; p < 2; p++) {
    ok = ok && aligned_to(a.d_k[p], 16) && aligned_to(a.d_v[p], 16) && aligned_to(a.d_bk[p], 16) && aligned_to(a.d_bv[p], 16);
    if (a.q_heads > 0) ok = ok && aligned_to(a.d_q[p], 16) && aligned_to(a.d_a[p], 16);
  }
  return ok;
}

// Fewest turned words for which the carries are packed into a table first: a
// launch of its own, then 8 bytes of a 32 KB table per word instead of four
// 32-byte entries of 512 KB.  40 turned heads of 128 words: 64 tokens 20 us
// unpacked, 29 us packed; 128 tokens 29 and 28 us; 4,133 tokens 321 and 165 us.
// (The packed table in shared memory took the same 165 us.)
constexpr int64_t kPackWords = 1 << 19;

template <bool PACKED>
cudaError_t launch_rope(const sufb200_ctx_s* ctx, const sufb200_rope_append& a, const GapArs& g, const uint64_t* table,
                        cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(a.tokens) * (a.q_heads + 2 * a.kv_heads);
  const auto kernel = paired(a) ? rope_append_kernel<PACKED, true> : rope_append_kernel<PACKED, false>;
  const int64_t want = (rows + kThreads / 32 - 1) / (kThreads / 32);
  const dim3 grid(static_cast<unsigned>(want > 1 << 20 ? 1 << 20 : want));
  if (PACKED) return launch_pdl(kernel, grid, dim3(kThreads), 0, st, a, g, table, ctx->d_status);
  kernel<<<grid, kThreads, 0, st>>>(a, g, table, ctx->d_status);
  return cudaGetLastError();
}

}  // namespace

}  // namespace sufb200

using namespace sufb200;

extern "C" int sufb200_rope_append_pair(sufb200_ctx ctx, const sufb200_rope_append* args, void* stream) {
  if (int rc = check_rope(args)) return rc;
  if (args->tokens == 0) return SUFB200_OK;
  if (int rc = attn_check_ctx(ctx)) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  GapArs g{};
  g.f = 1;
  if (args->rot_dim > 0) {
    g.f = args->trunc[0].frac_bits;
    for (int p = 0; p < 2; p++) {
      g.base += args->trunc[p].haty - args->trunc[p].r_hi;
      g.m += args->trunc[p].m;
      g.r += args->r[p];
    }
    g.base -= 1ull << (62 - g.f);
  }
  const int64_t turned = static_cast<int64_t>(args->tokens) * (args->q_heads + args->kv_heads) * args->rot_dim;
  cudaError_t e;
  if (turned < kPackWords) {
    e = launch_rope<false>(ctx, *args, g, nullptr, st);
  } else {
    uint64_t* table = nullptr;
    e = cudaMallocFromPoolAsync(reinterpret_cast<void**>(&table), sizeof(uint64_t) << g.f, ctx->pool, st);
    if (e == cudaSuccess) {
      carry_table_kernel<<<((1 << g.f) + 127) / 128, 128, 0, st>>>(*args, table);
      e = cudaGetLastError();
      if (e == cudaSuccess) e = launch_rope<true>(ctx, *args, g, table, st);
      const cudaError_t f = cudaFreeAsync(table, st);
      if (e == cudaSuccess) e = f;
    }
  }
  return attn_result("rope_append_pair", e);
}

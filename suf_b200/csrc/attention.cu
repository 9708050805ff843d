// attention.cu -- the two products of attention over a paged cache of
// secret-shared keys and values, for both parties on one GPU.
//
// A cached entry X (a key or value row) is held as the public E = X - B and
// the dealer's shares B_0, B_1 of its mask B, which stays fixed for the
// entry's life; a call's other operand Y has the fresh mask A (shares A_p),
// D = Y - A is public, and C_p are the shares of the triple's product.  Then
//   Z_p = C_p + D B_p + A_p E (+ D E for party 0),  Z_0 + Z_1 = Y X,
// and what a call writes is the open of the masked result for its truncation,
//   x^ = sum_p (Z_p + r_p)
//      = (C_0 + C_1) + D (B_0 + B_1) + (D + A_0 + A_1) E + (r_0 + r_1).
// The second line is what the kernels compute: sums mod 2^64 may be
// regrouped, so a pair call spends two products per entry where the parties
// by themselves spend two each.
//   scores: Y = the rotated queries (D opened by the append), X = keys,
//           contraction over the head, packed ragged rows out;
//   values: Y = the probabilities (D = P - A opened while loading), X =
//           values, contraction over the row's valid keys, [token][head] out.
// Queries share key heads in groups of q_heads / kv_heads; row rho of a
// (sequence, key head) is query rho / group of head kh * group + rho % group,
// so rows of one tile have nearly equal causal lengths.
#include "attention.hpp"

namespace sufb200 {

namespace {

constexpr int kThreads = 256;

// Rows of a (sequence, key head) up to which the row kernels are used; above,
// the tensor cores (whose pre-pass reads the cache once and writes its planes).
// Four sequences of 8,192 tokens, 32 / 8 heads of 128, row kernels (16 rows in two
// passes over the cache) against tensor cores: scores of 8 rows 238 and 407 us, 16
// rows 455 and 419 us; values of 8 rows 291 and 346 us, 16 rows 568 and 354 us.
constexpr int kFewRows = SUFB200_ATTN_FEW_ROWS;

int fail(int code, const std::string& msg) { return record_error(code, msg); }

// ---- few rows (single tokens): bound by the cache's three words per entry --
// scores_rows: eight lanes per key, 16 bytes of the head each; the rows' U =
// D + A_0 + A_1 and D sit in shared memory and are read once for two keys.  Up
// to four rows the multiplies (two per word and row, three integer
// instructions each) stay below the memory's time.  One decode step over
// 73,279 cached tokens, 32 / 8 heads of 128: 350 us cold, 5.3 TB/s of 6.5; what
// is left is waiting on memory with 32 warps an SM (long_scoreboard 11 per
// issue, DRAM 83 %).
constexpr int kKeyChunk = 256;  // most keys per CTA

// The run of `per` cached tokens that this block has, of which sequence and key
// head; false: none, or the sequence has more rows than the row kernels take.
// Runs are listed sequence after sequence, so that short caches beside a long
// one leave no idle blocks (200 caches of 50 - 400 tokens beside one of 40,000,
// 32 / 8 heads of 128: scores 438 us, 883 by a grid of every sequence's longest
// possible cache), and by key heads within a run, whose rows of a page lie one
// behind the other (eight rows, 73,279 tokens: 467 us, 541 with the heads outside).
// Where one run holds any cache (ONE, or by the lengths) a block is a sequence.
template <bool ONE>
__device__ __forceinline__ bool run_of(const AttnSeqs& s, int per, uint32_t* status, int& b, int& kh, int& beg,
                                       SeqInfo& q) {
  const unsigned g = blockIdx.x / static_cast<unsigned>(s.kv_heads);
  kh = static_cast<int>(blockIdx.x - g * s.kv_heads);
  beg = 0;
  if (ONE || s.max_ctx <= per) {
    b = static_cast<int>(g);
    if (!seq_info(s, b, status, q)) return false;
  } else {
    // every sequence is looked at, also where wrong lengths hide it from the search
    if (g < static_cast<unsigned>(s.batch) && kh == 0) seq_info(s, static_cast<int>(g), status, q);
    b = block_seq(s.d_cu_ctx, s.batch, 1, per, g);
    if (!seq_info(s, b, status, q)) return false;
    const int64_t first = g - first_block(q.l0, b, per);
    if (first < 0 || first * per >= q.L) return false;
    beg = static_cast<int>(first) * per;
  }
  return q.n > 0 && s.q_heads / s.kv_heads * q.n <= kFewRows;
}

dim3 runs_grid(const AttnSeqs& s, int per) {
  const int64_t runs = s.max_ctx <= per ? s.batch : blocks_of(s.cached, s.batch, per);
  return dim3(static_cast<unsigned>(runs * s.kv_heads));
}

template <int RT>
__global__ void __launch_bounds__(kThreads, RT == 4 ? 4 : 3) scores_rows_kernel(const __grid_constant__ AttnSeqs s,
                                                                                const __grid_constant__ AttnOperands o,
                                                                                int chunk) {
  extern __shared__ __align__(16) uint64_t sm[];
  const int t = threadIdx.x, dh = s.head_dim, group = s.q_heads / s.kv_heads;
  int b, kh, k0;
  SeqInfo q;
  if (!run_of<false>(s, chunk, o.status, b, kh, k0, q)) return;
  const int R = group * q.n, len = q.L;  // the last row has every key
  uint64_t* sU = sm;                    // [RT][dh]
  uint64_t* sD = sU + RT * dh;          // [RT][dh]
  uint64_t* s_out = sD + RT * dh;       // [RT][chunk + 1]
  int64_t* s_key = reinterpret_cast<int64_t*>(s_out + RT * (chunk + 1));  // [chunk]
  for (int e = t; e < RT * dh; e += kThreads) {
    const int rho = e / dh, c = e % dh;
    uint64_t d = 0, u = 0;
    if (rho < R) {
      const int64_t at = (static_cast<int64_t>(q.t0 + rho / group) * s.q_heads + kh * group + rho % group) * dh + c;
      d = o.x[0][at];
      u = d + o.a[0][at] + o.a[1][at];
    }
    sU[e] = u;
    sD[e] = d;
  }
  for (int e = t; e < chunk; e += kThreads) s_key[e] = k0 + e < len ? key_off(s, b, kh, k0 + e, o.status) : -1;
  __syncthreads();
  const int l8 = t & 7, grp = t >> 3;
  for (int kk = grp; kk < chunk; kk += 64) {
    const int64_t o0 = s_key[kk], o1 = s_key[kk + 32];
    uint64_t acc[2][RT] = {};
    for (int c = l8; c < dh / 2; c += 8) {
      ulonglong2 e0 = make_ulonglong2(0, 0), w0 = e0, e1 = e0, w1 = e0;
      if (o0 >= 0) {
        e0 = ld_stream(o.e + o0 + 2 * c);
        const ulonglong2 p = ld_stream(o.b[0] + o0 + 2 * c), r = ld_stream(o.b[1] + o0 + 2 * c);
        w0 = make_ulonglong2(p.x + r.x, p.y + r.y);
      }
      if (o1 >= 0) {
        e1 = ld_stream(o.e + o1 + 2 * c);
        const ulonglong2 p = ld_stream(o.b[0] + o1 + 2 * c), r = ld_stream(o.b[1] + o1 + 2 * c);
        w1 = make_ulonglong2(p.x + r.x, p.y + r.y);
      }
#pragma unroll
      for (int rr = 0; rr < RT; rr++) {
        const ulonglong2 u = *reinterpret_cast<const ulonglong2*>(sU + rr * dh + 2 * c);
        const ulonglong2 d = *reinterpret_cast<const ulonglong2*>(sD + rr * dh + 2 * c);
        acc[0][rr] += u.x * e0.x + u.y * e0.y + d.x * w0.x + d.y * w0.y;
        acc[1][rr] += u.x * e1.x + u.y * e1.y + d.x * w1.x + d.y * w1.y;
      }
    }
    // sums over the key's eight lanes, halving the rows a lane holds in every
    // exchange: RT - 1 exchanges (and log2(8 / RT) more) instead of 3 RT
#pragma unroll
    for (int v = 0; v < 2; v++) {
      int row = 0;
#pragma unroll
      for (int m = 1; m < RT; m *= 2) {
        const bool up = l8 & m;
#pragma unroll
        for (int rr = 0; rr < RT / (2 * m); rr++) {
          const uint64_t keep = up ? acc[v][2 * rr + 1] : acc[v][2 * rr];
          const uint64_t give = up ? acc[v][2 * rr] : acc[v][2 * rr + 1];
          acc[v][rr] = keep + __shfl_xor_sync(0xffffffffu, give, m);
        }
        row += up ? m : 0;
      }
#pragma unroll
      for (int m = RT; m < 8; m *= 2) acc[v][0] += __shfl_xor_sync(0xffffffffu, acc[v][0], m);
      if (l8 < RT) s_out[row * (chunk + 1) + kk + 32 * v] = acc[v][0];
    }
  }
  __syncthreads();
  for (int e = t; e < RT * chunk; e += kThreads) {
    const int rho = e / chunk, kk = e % chunk, i = rho / group;
    if (rho >= R || k0 + kk >= row_len(q.n, q.L, s.causal, i)) continue;
    const int64_t at = q.base + (kh * group + rho % group) * q.blk + row_off(q.n, q.L, s.causal, i) + k0 + kk;
    o.out[at] = s_out[rho * (chunk + 1) + kk] + o.c[0][at] + o.c[1][at] + o.r;
  }
}

// out = C_0 + C_1 + r, what the values kernels add to: of all tokens, or (FEW, a
// sequence per blockIdx.y) of the sequences the row kernels take, where the
// others are stored whole (2,748 prompt tokens beside a single one: 25 us less).
template <bool FEW>
__global__ void values_init_kernel(const __grid_constant__ AttnSeqs s, const __grid_constant__ AttnOperands o) {
  int64_t first = 0, tokens;
  if (FEW) {
    SeqInfo q;
    if (!seq_info(s, blockIdx.y, o.status, q) || s.q_heads / s.kv_heads * q.n > kFewRows) return;
    first = q.t0;
    tokens = q.n;
  } else {
    tokens = s.d_cu_q[s.batch];
    if (tokens < 0 || tokens > s.tokens) {
      if (blockIdx.x == 0 && threadIdx.x == 0) atomicOr(o.status, kStatusBadArgument);
      return;
    }
  }
  const int64_t width = static_cast<int64_t>(s.q_heads) * s.head_dim, end = (first + tokens) * width;
  for (int64_t i = first * width + blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < end;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x)
    o.out[i] = o.c[0][i] + o.c[1][i] + o.r;
}

// values_rows: a thread holds two words of the head for RT rows; the CTA's
// key lanes walk its range of keys, whose probabilities sit in shared memory.
// Ranges of one row meet by 64-bit atomic adds: sums mod 2^64 do not depend
// on their order.  The same decode step: 351 us cold, 5.3 TB/s.  (Two and four
// keys a thread at a time, for more loads in flight: 387 us, for fewer warps.)
constexpr int kValStage = 64;

// SOLO: one CTA has every key of its rows and stores whole results.
template <int RT, bool SOLO>
__global__ void __launch_bounds__(kThreads, RT == 4 ? 4 : 3) values_rows_kernel(const __grid_constant__ AttnSeqs s,
                                                                                const __grid_constant__ AttnOperands o,
                                                                                int range) {
  __shared__ __align__(16) uint64_t sU[kValStage][RT], sD[kValStage][RT];
  __shared__ ulonglong2 s_sum[SOLO ? kThreads : 1];
  __shared__ int64_t s_key[kValStage];
  const int t = threadIdx.x, dh = s.head_dim, group = s.q_heads / s.kv_heads, P = dh / 2;
  int b, kh, beg;
  SeqInfo q;
  if (!run_of<SOLO>(s, range, o.status, b, kh, beg, q)) return;
  const int R = group * q.n, len = q.L, end = range < len - beg ? beg + range : len;
  const int lanes = kThreads / P, kl = t / P, c = t % P;
  uint64_t ax[RT] = {}, ay[RT] = {};
  for (int j0 = beg; j0 < end; j0 += kValStage) {
    __syncthreads();
    for (int e = t; e < kValStage * RT; e += kThreads) {
      const int kk = e % kValStage, rho = e / kValStage, i = rho / group, j = j0 + kk;
      uint64_t d = 0, u = 0;
      if (rho < R && j < end && j < row_len(q.n, q.L, s.causal, i)) {
        const int64_t at = q.base + (kh * group + rho % group) * q.blk + row_off(q.n, q.L, s.causal, i) + j;
        const uint64_t a0 = o.a[0][at], a1 = o.a[1][at];
        d = (o.x[0][at] - a0) + (o.x[1][at] - a1);
        u = d + a0 + a1;
      }
      sU[kk][rho] = u;
      sD[kk][rho] = d;
    }
    for (int e = t; e < kValStage; e += kThreads) s_key[e] = j0 + e < end ? key_off(s, b, kh, j0 + e, o.status) : -1;
    __syncthreads();
    if (kl < lanes)
      for (int kk = kl; kk < kValStage; kk += lanes) {
        const int64_t at = s_key[kk];
        if (at < 0) continue;
        const ulonglong2 e = ld_stream(o.e + at + 2 * c), b0 = ld_stream(o.b[0] + at + 2 * c),
                         b1 = ld_stream(o.b[1] + at + 2 * c);
        const uint64_t wx = b0.x + b1.x, wy = b0.y + b1.y;
#pragma unroll
        for (int rr = 0; rr < RT; rr++) {
          const uint64_t u = sU[kk][rr], d = sD[kk][rr];
          ax[rr] += u * e.x + d * wx;
          ay[rr] += u * e.y + d * wy;
        }
      }
  }
#pragma unroll
  for (int rho = 0; rho < RT; rho++) {
    if (rho >= R) break;
    const int64_t at = (static_cast<int64_t>(q.t0 + rho / group) * s.q_heads + kh * group + rho % group) * dh + 2 * c;
    if (SOLO) {
      __syncthreads();
      s_sum[t] = make_ulonglong2(ax[rho], ay[rho]);
      __syncthreads();
      if (kl > 0) continue;
      uint64_t x = o.c[0][at] + o.c[1][at] + o.r, y = o.c[0][at + 1] + o.c[1][at + 1] + o.r;
      for (int l = 0; l < lanes; l++) {
        x += s_sum[l * P + c].x;
        y += s_sum[l * P + c].y;
      }
      o.out[at] = x;
      o.out[at + 1] = y;
    } else if (kl < lanes) {
      unsigned long long* to = reinterpret_cast<unsigned long long*>(o.out + at);
      atomicAdd(to, static_cast<unsigned long long>(ax[rho]));
      atomicAdd(to + 1, static_cast<unsigned long long>(ay[rho]));
    }
  }
}

// The most rows of a (sequence, key head), and the most the row kernels take
// (0: every sequence has more): a batch of prompts and single tokens runs both
// kinds of kernel, each on its own sequences.
struct Rows {
  int most, few;
};

Rows rows_of(const AttnSeqs& s) {
  const int group = s.q_heads / s.kv_heads;
  Rows r{group * s.max_q, 0};
  if (group * s.min_q <= kFewRows) r.few = s.short_rows > 0 ? s.short_rows : (r.most <= kFewRows ? r.most : kFewRows);
  return r;
}

int check_seqs(const sufb200_attn_seqs* s, const char* who) {
  const std::string at = std::string(who) + ": ";
  if (!s) return fail(SUFB200_ERR_INVALID, at + "null sequences");
  if (s->batch < 0 || s->max_pages < 0 || s->pages < 0 || s->min_q < 0 || s->max_q < s->min_q || s->max_ctx < 0 ||
      s->tokens < 0 || s->cached < 0 || s->packed < 0)
    return fail(SUFB200_ERR_INVALID, at + "negative size");
  if (s->page_size < 1 || s->kv_heads < 1 || s->q_heads < s->kv_heads || s->q_heads % s->kv_heads)
    return fail(SUFB200_ERR_INVALID, at + "page size, or query heads not a multiple of key heads");
  if (s->head_dim < 2 || s->head_dim > 256 || s->head_dim % 2)
    return fail(SUFB200_ERR_UNSUPPORTED, at + "head size must be even, 2..256");
  if (static_cast<int64_t>(s->batch) * s->kv_heads > 65535)
    return fail(SUFB200_ERR_UNSUPPORTED, at + "more than 65535 (sequence, key head) pairs");
  if (static_cast<int64_t>(s->q_heads / s->kv_heads) * s->max_q > 1 << 20)
    return fail(SUFB200_ERR_UNSUPPORTED, at + "more than 2^20 rows per (sequence, key head)");
  // grids count row tiles x key heads x 128-word tiles of the head
  const int64_t tiles = s->q_heads / s->kv_heads * s->tokens / SUFB200_ATTN_ROW_TILE + s->n_tiles + s->batch;
  const int64_t runs = blocks_of(s->cached, s->batch, kValStage);  // the row kernels' shortest runs
  if (s->tokens > INT32_MAX || s->cached > INT32_MAX || tiles > INT32_MAX / 2 / s->kv_heads || runs > INT32_MAX / s->kv_heads)
    return fail(SUFB200_ERR_UNSUPPORTED, at + "too many tokens for one call");
  if (s->max_ctx > 1 << 26) return fail(SUFB200_ERR_UNSUPPORTED, at + "more than 2^26 cached tokens in a sequence");
  if (static_cast<int64_t>(s->max_ctx) > static_cast<int64_t>(s->max_pages) * s->page_size)
    return fail(SUFB200_ERR_INVALID, at + "max_ctx is more than the block table's pages hold");
  if (static_cast<__int128>(s->q_heads) * s->max_q * s->max_ctx >= (static_cast<__int128>(1) << 60))
    return fail(SUFB200_ERR_UNSUPPORTED, at + "more than 2^60 packed words");
  if (s->long_ctx < 0 || s->long_ctx > s->max_ctx || s->short_rows < 0 || s->short_rows > kFewRows)
    return fail(SUFB200_ERR_INVALID, at + "bounds of the long or short sequences");
  if (s->n_tiles < 0 || (s->n_tiles > 0) != (s->d_tiles != nullptr))
    return fail(SUFB200_ERR_INVALID, at + "null or empty tile list");
  if ((s->plane_keys > 0) != (s->d_plane_keys != nullptr) || s->plane_keys < 0 || s->plane_keys > INT32_MAX ||
      s->plane_keys % SUFB200_ATTN_KEY_TILE)
    return fail(SUFB200_ERR_INVALID, at + "null or empty list of places, or not in whole key tiles");
  if (s->batch > 0 && (!s->d_cu_q || !s->d_cu_ctx || !s->d_row_base || (s->max_ctx > 0 && !s->d_block_table)))
    return fail(SUFB200_ERR_INVALID, at + "null sequence array");
  for (const void* p : {s->d_cu_q, s->d_cu_ctx, s->d_block_table, s->d_tiles, s->d_plane_keys})
    if (!aligned_to(p, 4)) return fail(SUFB200_ERR_INVALID, at + "misaligned sequence array");
  if (!aligned_to(s->d_row_base, 8)) return fail(SUFB200_ERR_INVALID, at + "misaligned sequence array");
  return SUFB200_OK;
}

int check_operands(const AttnOperands& o, const char* who) {
  const std::string at = std::string(who) + ": ";
  const void* words[] = {o.x[0], o.x[1], o.a[0], o.a[1], o.c[0], o.c[1], o.out};
  for (const void* p : words)
    if (!p || !aligned_to(p, 8)) return fail(SUFB200_ERR_INVALID, at + "null or misaligned operand");
  for (const void* p : {static_cast<const void*>(o.e), static_cast<const void*>(o.b[0]), static_cast<const void*>(o.b[1])})
    if (!p || !aligned_to(p, 16)) return fail(SUFB200_ERR_INVALID, at + "the cache's pools must be 16-byte aligned");
  return SUFB200_OK;
}

// Longest context whose values one CTA per (row tile, key head) takes whole,
// in one launch instead of an init pass and adds.
constexpr int kSoloKeys = 256;

// Keys a CTA of the row kernels walks: the longest run (least, doubled up to
// most) that still leaves `per_sm` CTAs per SM.  A long run pays its set-up
// once, a short cache wants every SM, and many short runs end more evenly.  One
// step over 73,279 cached tokens of 8 x 128 words: scores 328 us in runs of 256
// (eight CTAs per SM asked for), 333 of 128, with eight rows 467 and 483 us;
// values 321 us in runs of 512 (three asked for), 322 of 1,024, 325 of 256, with
// eight rows 544, 667 (two uneven waves) and 531 us.  200 caches of 50 - 400
// tokens beside one of 40,000: scores 438 us of 256, 409 of 128, 539 of 512;
// values 402 of 512, 396 of 256, 528 of 2,048.
int keys_per_cta(const sufb200_ctx_s* ctx, const AttnSeqs& s, int least, int most, int per_sm) {
  const int64_t keys = s.cached * s.kv_heads, ctas = static_cast<int64_t>(ctx->sm_count) * per_sm;
  int run = least;
  while (run < most && keys / (2 * run) >= ctas) run *= 2;
  return run;
}

}  // namespace

int attn_result(const char* who, cudaError_t e) {
  if (e == cudaSuccess) return SUFB200_OK;
  cudaGetLastError();
  return fail(SUFB200_ERR_CUDA, std::string(who) + ": " + cudaGetErrorString(e));
}

int attn_check_ctx(sufb200_ctx ctx) {
  if (!ctx) return fail(SUFB200_ERR_INVALID, "null context");
  if (ctx->device < 0) return fail(SUFB200_ERR_UNSUPPORTED, "host-only context: no device to evaluate on");
  const cudaError_t e = cudaSetDevice(ctx->device);
  return attn_result("cudaSetDevice", e);
}

}  // namespace sufb200

using namespace sufb200;

extern "C" {

int sufb200_attn_scores_pair(sufb200_ctx ctx, const sufb200_attn_seqs* seqs, const uint64_t* d_dq,
                             const uint64_t* const* d_a, const uint64_t* const* d_c, const uint64_t* r,
                             const uint64_t* d_ek, const uint64_t* const* d_bk, uint64_t* d_xhat, void* stream) {
  if (int rc = check_seqs(seqs, "attn_scores_pair")) return rc;
  if (seqs->batch == 0 || seqs->packed == 0 || seqs->max_q == 0 || seqs->max_ctx == 0) return SUFB200_OK;
  if (!d_a || !d_c || !r || !d_bk) return fail(SUFB200_ERR_INVALID, "attn_scores_pair: null pointer array");
  AttnOperands o{{d_dq, d_dq}, {d_a[0], d_a[1]}, {d_c[0], d_c[1]}, d_ek, {d_bk[0], d_bk[1]}, r[0] + r[1], 0, d_xhat,
                 nullptr};
  if (int rc = check_operands(o, "attn_scores_pair")) return rc;
  if (int rc = attn_check_ctx(ctx)) return rc;
  o.status = ctx->d_status;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const Rows rows = rows_of(*seqs);
  if (rows.few > 0) {
    const int rt = rows.few <= 4 ? 4 : 8;
    // rows of 8 x 256 words and 256 keys would pass 48 KB of shared memory
    const int chunk = keys_per_cta(ctx, *seqs, 64, rt * seqs->head_dim > 1024 ? kKeyChunk / 2 : kKeyChunk, 8);
    const size_t smem = sizeof(uint64_t) * (2 * rt * seqs->head_dim + rt * (chunk + 1) + chunk);
    const dim3 grid = runs_grid(*seqs, chunk);
    if (rt == 4)
      scores_rows_kernel<4><<<grid, kThreads, smem, st>>>(*seqs, o, chunk);
    else
      scores_rows_kernel<8><<<grid, kThreads, smem, st>>>(*seqs, o, chunk);
  }
  o.few = rows.few > 0 ? kFewRows : 0;
  if (rows.most > kFewRows) {
    const cudaError_t e = launch_scores_tc(ctx, *seqs, o, st);
    if (e != cudaSuccess) return attn_result("attn_scores_pair", e);
  }
  return attn_result("attn_scores_pair", cudaGetLastError());
}

int sufb200_attn_values_pair(sufb200_ctx ctx, const sufb200_attn_seqs* seqs, const uint64_t* const* d_p,
                             const uint64_t* const* d_a, const uint64_t* const* d_c, const uint64_t* r,
                             const uint64_t* d_ev, const uint64_t* const* d_bv, uint64_t* d_xhat, void* stream) {
  if (int rc = check_seqs(seqs, "attn_values_pair")) return rc;
  if (seqs->batch == 0 || seqs->max_q == 0 || seqs->tokens == 0) return SUFB200_OK;
  if (!d_p || !d_a || !d_c || !r || !d_bv) return fail(SUFB200_ERR_INVALID, "attn_values_pair: null pointer array");
  AttnOperands o{{d_p[0], d_p[1]}, {d_a[0], d_a[1]}, {d_c[0], d_c[1]}, d_ev, {d_bv[0], d_bv[1]}, r[0] + r[1], 0, d_xhat,
                 nullptr};
  if (seqs->packed == 0) {  // every row is empty: no probability is read
    o.x[0] = o.x[1] = o.a[0] = o.a[1] = o.c[0];
  }
  if (int rc = check_operands(o, "attn_values_pair")) return rc;
  if (int rc = attn_check_ctx(ctx)) return rc;
  o.status = ctx->d_status;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const Rows rows = rows_of(*seqs);
  const bool any = seqs->packed > 0 && seqs->max_ctx > 0;
  const bool few_solo = seqs->max_ctx <= kSoloKeys, many_solo = rows.most > kFewRows && values_tc_solo(ctx, *seqs);
  if (!any || (rows.most > kFewRows && !many_solo) || (rows.few > 0 && !few_solo)) {
    const bool few_only = any && rows.most > kFewRows && many_solo;
    const int64_t words = few_only ? static_cast<int64_t>(rows.few) * seqs->kv_heads * seqs->head_dim
                                   : seqs->tokens * seqs->q_heads * seqs->head_dim;
    const int64_t want = (words + kThreads - 1) / kThreads, cap = static_cast<int64_t>(ctx->sm_count) * 8;
    const unsigned x = static_cast<unsigned>(want < cap ? want : cap);
    if (few_only)
      values_init_kernel<true><<<dim3(x, seqs->batch), kThreads, 0, st>>>(*seqs, o);
    else
      values_init_kernel<false><<<x, kThreads, 0, st>>>(*seqs, o);
  }
  if (any && rows.few > 0) {
    const int range = few_solo ? kSoloKeys : keys_per_cta(ctx, *seqs, kValStage, rows.few <= 4 ? 512 : 256, 3);
    const dim3 grid = runs_grid(*seqs, range);
    const auto kernel = rows.few <= 4 ? (few_solo ? values_rows_kernel<4, true> : values_rows_kernel<4, false>)
                                      : (few_solo ? values_rows_kernel<8, true> : values_rows_kernel<8, false>);
    kernel<<<grid, kThreads, 0, st>>>(*seqs, o, range);
  }
  o.few = rows.few > 0 ? kFewRows : 0;
  if (any && rows.most > kFewRows) {
    const cudaError_t e = launch_values_tc(ctx, *seqs, o, st);
    if (e != cudaSuccess) return attn_result("attn_values_pair", e);
  }
  return attn_result("attn_values_pair", cudaGetLastError());
}

}  // extern "C"

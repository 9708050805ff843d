// rowmax.cu -- the row-max tournament of nn::RowMaxDiffTask
// (include/nn/row_maxdiff_task.hpp) over packed rows of any lengths, for both
// parties on one GPU: max(a, b) = b + ReLU(a - b), the ReLU a coefficient gate
// on the opened difference between two rounds' launches.
//
// A round halves every row, w -> ceil(w / 2): pair j of a row is its values
// 2j, 2j + 1, and the last value of an odd row moves on as it is.  With off_k
// the packed row offsets of round k, row r has off_k[r+1] - off_k[r] values,
// and its pairs start at word off_k[r] - off_{k+1}[r] of the packed pairs
// (values minus survivors of the rows before it).  Rows may start at any word,
// so accesses are 8 bytes wide and a warp's are adjacent; a round of 14.7 M
// values in 21,712 rows runs at 5.5 - 6 TB/s (91 us for the first merge), below
// some 10,000 values a round is one launch's latency (5.5 us).
#include "attention.hpp"

namespace sufb200 {

namespace {

constexpr int kThreads = 256;

int fail(int code, const std::string& msg) { return record_error(code, msg); }

// Value j of the next round: the pair's winner, or the odd row's last value.
__device__ __forceinline__ uint64_t survivor(const uint64_t* c, const uint64_t* relu, int w, int at, int pair, int j) {
  return 2 * j + 1 < w ? c[at + 2 * j + 1] + relu[pair + j] : c[at + 2 * j];
}

// A row is dealt to `tpr` threads.  MERGE: the round's winners into next_p,
// then (xhat set) the open of the next round's differences; else the open of
// the first round's differences of c.
template <bool MERGE>
__global__ void __launch_bounds__(kThreads)
    rowmax_round_kernel(const uint64_t* __restrict__ c0, const uint64_t* __restrict__ c1,
                        const uint64_t* __restrict__ q0, const uint64_t* __restrict__ q1, int rows,
                        const int32_t* __restrict__ off, const int32_t* __restrict__ off1,
                        const int32_t* __restrict__ off2, uint64_t rsum, uint64_t* __restrict__ n0,
                        uint64_t* __restrict__ n1, uint64_t* __restrict__ xhat, int tpr) {
  const int per = kThreads / tpr;
  const int lane = threadIdx.x % tpr;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * per + threadIdx.x / tpr; r < rows;
       r += static_cast<int64_t>(gridDim.x) * per) {
    const int at = off[r], w = off[r + 1] - at;
    const int pos = blockIdx.y * tpr + lane, step = gridDim.y * tpr;
    if (MERGE) {
      const int at1 = off1[r], w1 = off1[r + 1] - at1, pair = at - at1;
      const int pair1 = xhat ? at1 - off2[r] : 0;
      for (int j = pos; 2 * j < w1; j += step) {
        const uint64_t a0 = survivor(c0, q0, w, at, pair, 2 * j), a1 = survivor(c1, q1, w, at, pair, 2 * j);
        n0[at1 + 2 * j] = a0;
        n1[at1 + 2 * j] = a1;
        if (2 * j + 1 >= w1) continue;
        const uint64_t b0 = survivor(c0, q0, w, at, pair, 2 * j + 1), b1 = survivor(c1, q1, w, at, pair, 2 * j + 1);
        n0[at1 + 2 * j + 1] = b0;
        n1[at1 + 2 * j + 1] = b1;
        if (xhat) xhat[pair1 + j] = (a0 - b0) + (a1 - b1) + rsum;
      }
    } else {
      const int pair = at - off1[r];
      for (int j = pos; 2 * j + 1 < w; j += step)
        xhat[pair + j] = (c0[at + 2 * j] - c0[at + 2 * j + 1]) + (c1[at + 2 * j] - c1[at + 2 * j + 1]) + rsum;
    }
  }
}

__global__ void __launch_bounds__(kThreads)
    maxdiff_ragged_kernel(const uint64_t* __restrict__ m0, const uint64_t* __restrict__ m1,
                          const uint64_t* __restrict__ s0, const uint64_t* __restrict__ s1, int rows,
                          const int32_t* __restrict__ off, const int32_t* __restrict__ moff,
                          uint64_t* __restrict__ t0, uint64_t* __restrict__ t1, int tpr) {
  const int per = kThreads / tpr;
  const int lane = threadIdx.x % tpr;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * per + threadIdx.x / tpr; r < rows;
       r += static_cast<int64_t>(gridDim.x) * per) {
    const int at = off[r], w = off[r + 1] - at;
    if (w <= 0) continue;
    const uint64_t a = m0[moff[r]], b = m1[moff[r]];
    const int step = gridDim.y * tpr;
    for (int j = blockIdx.y * tpr + lane; j < w; j += 4 * step) {  // four words' loads before their first use
      uint64_t v0[4], v1[4];
#pragma unroll
      for (int x = 0; x < 4; x++) {
        v0[x] = ld_if(s0 + at + j + x * step, j + x * step < w);
        v1[x] = ld_if(s1 + at + j + x * step, j + x * step < w);
      }
#pragma unroll
      for (int x = 0; x < 4; x++)
        if (j + x * step < w) {
          t0[at + j + x * step] = a - v0[x];
          t1[at + j + x * step] = b - v1[x];
        }
    }
  }
}

// Threads of a row and the grid: about 16 values a thread (with four, the
// chain of offset, maximum and first load weighs more: maxdiff of 14.7 M values
// 96 us, 85 with 16; the rounds are alike), blocks over the rows first and
// along long rows where the rows alone do not fill the GPU.
struct Shape {
  int tpr;
  dim3 grid;
};

Shape shape_for(const sufb200_ctx_s* ctx, int rows, int width) {
  Shape s;
  s.tpr = 8;
  while (s.tpr < kThreads && s.tpr * 16 < width) s.tpr *= 2;
  const int64_t per = kThreads / s.tpr;
  const int64_t blocks = (rows + per - 1) / per, cap = static_cast<int64_t>(ctx->sm_count) * 16;
  const int64_t along = (width + 16 * s.tpr - 1) / (16 * s.tpr);
  const int64_t x = blocks < cap ? blocks : cap;
  const int64_t fit = cap / x;
  const int64_t y = along < fit ? along : fit;
  s.grid = dim3(static_cast<unsigned>(x), static_cast<unsigned>(y < 1 ? 1 : (y > 65535 ? 65535 : y)));
  return s;
}

// Rows stop at 2^30 words: places are 32 bits wide and a row's threads step past
// its end by up to four strides of the grid (at most 16 blocks of kThreads an SM: below 2^20).
int check_rows(int rows, int max_width, const char* who) {
  if (rows < 0 || max_width < 0) return fail(SUFB200_ERR_INVALID, std::string(who) + ": negative size");
  if (max_width > 1 << 30) return fail(SUFB200_ERR_UNSUPPORTED, std::string(who) + ": rows of more than 2^30 words");
  return SUFB200_OK;
}

int check_offsets(std::initializer_list<const void*> ps, const char* who) {
  for (const void* p : ps)
    if (!aligned_to(p, 4)) return fail(SUFB200_ERR_INVALID, std::string(who) + ": misaligned offsets");
  return SUFB200_OK;
}

int check_words(std::initializer_list<const void*> ps, const char* who) {
  for (const void* p : ps)
    if (!p || !aligned_to(p, 8)) return fail(SUFB200_ERR_INVALID, std::string(who) + ": null or misaligned device pointer");
  return SUFB200_OK;
}

}  // namespace

}  // namespace sufb200

using namespace sufb200;

extern "C" {

int sufb200_rowmax_open_pair(sufb200_ctx ctx, const uint64_t* const* d_c, int rows, int max_width,
                             const int32_t* d_off, const int32_t* d_off1, const uint64_t* r, uint64_t* d_xhat,
                             void* stream) {
  if (int rc = check_rows(rows, max_width, "rowmax_open_pair")) return rc;
  if (rows == 0 || max_width < 2) return SUFB200_OK;
  if (!d_c || !r || !d_off || !d_off1) return fail(SUFB200_ERR_INVALID, "rowmax_open_pair: null argument");
  if (int rc = check_offsets({d_off, d_off1}, "rowmax_open_pair")) return rc;
  if (int rc = check_words({d_c[0], d_c[1], d_xhat}, "rowmax_open_pair")) return rc;
  if (int rc = attn_check_ctx(ctx)) return rc;
  const Shape s = shape_for(ctx, rows, max_width);
  rowmax_round_kernel<false><<<s.grid, kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      d_c[0], d_c[1], nullptr, nullptr, rows, d_off, d_off1, nullptr, r[0] + r[1], nullptr, nullptr, d_xhat, s.tpr);
  return attn_result("rowmax_open_pair", cudaGetLastError());
}

int sufb200_rowmax_round_pair(sufb200_ctx ctx, const uint64_t* const* d_c, const uint64_t* const* d_relu, int rows,
                              int max_width, const int32_t* d_off, const int32_t* d_off1, const int32_t* d_off2,
                              const uint64_t* r, uint64_t* const* d_next, uint64_t* d_xhat, void* stream) {
  if (int rc = check_rows(rows, max_width, "rowmax_round_pair")) return rc;
  if (rows == 0 || max_width == 0) return SUFB200_OK;
  if (!d_c || !d_relu || !d_off || !d_off1 || !d_next) return fail(SUFB200_ERR_INVALID, "rowmax_round_pair: null argument");
  if (int rc = check_offsets({d_off, d_off1, d_off2}, "rowmax_round_pair")) return rc;
  if (int rc = check_words({d_c[0], d_c[1], d_next[0], d_next[1]}, "rowmax_round_pair")) return rc;
  if (max_width > 1)
    if (int rc = check_words({d_relu[0], d_relu[1]}, "rowmax_round_pair")) return rc;
  if (d_xhat && (!d_off2 || !r || !aligned_to(d_xhat, 8)))
    return fail(SUFB200_ERR_INVALID, "rowmax_round_pair: the next open needs its offsets and masks");
  if (int rc = attn_check_ctx(ctx)) return rc;
  const Shape s = shape_for(ctx, rows, max_width);
  rowmax_round_kernel<true><<<s.grid, kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      d_c[0], d_c[1], d_relu[0], d_relu[1], rows, d_off, d_off1, d_off2, d_xhat ? r[0] + r[1] : 0, d_next[0], d_next[1],
      d_xhat, s.tpr);
  return attn_result("rowmax_round_pair", cudaGetLastError());
}

int sufb200_maxdiff_ragged_pair(sufb200_ctx ctx, const uint64_t* const* d_max, const uint64_t* const* d_s, int rows,
                                int max_width, const int32_t* d_off, const int32_t* d_max_off, uint64_t* const* d_t,
                                void* stream) {
  if (int rc = check_rows(rows, max_width, "maxdiff_ragged_pair")) return rc;
  if (rows == 0 || max_width == 0) return SUFB200_OK;
  if (!d_max || !d_s || !d_t || !d_off || !d_max_off) return fail(SUFB200_ERR_INVALID, "maxdiff_ragged_pair: null argument");
  if (int rc = check_offsets({d_off, d_max_off}, "maxdiff_ragged_pair")) return rc;
  if (int rc = check_words({d_max[0], d_max[1], d_s[0], d_s[1], d_t[0], d_t[1]}, "maxdiff_ragged_pair")) return rc;
  if (int rc = attn_check_ctx(ctx)) return rc;
  const Shape s = shape_for(ctx, rows, max_width);
  maxdiff_ragged_kernel<<<s.grid, kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      d_max[0], d_max[1], d_s[0], d_s[1], rows, d_off, d_max_off, d_t[0], d_t[1], s.tpr);
  return attn_result("maxdiff_ragged_pair", cudaGetLastError());
}

}  // extern "C"

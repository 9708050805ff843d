// attention.hpp -- what the kernels of attention over a paged cache of shares
// have in common (attention.cu, attention_rope.cu, rowmax.cu).  Internal.
#pragma once

#include <string>

#include "kernels.hpp"
#include "sufb200_internal.cuh"

namespace sufb200 {

// The packed sequences as the kernels see them (a copy of the public struct:
// plain device pointers and sizes).
using AttnSeqs = sufb200_attn_seqs;

// One sequence: n new tokens (packed tokens t0 .. t0 + n), L cached tokens
// (the new ones included), its packed rows at word `base`, `blk` words a head.
struct SeqInfo {
  int n, L, t0, l0;  // l0: cached tokens of the sequences before it
  int64_t base, blk;
};

// Valid keys of query i.  Causal: query i is token L - n + i of the sequence
// and sees itself and what is before it; with L < n the first n - L queries
// see nothing (empty rows).
SUFB200_HD int row_len(int n, int L, int causal, int i) {
  if (!causal) return L;
  const int m = L - n + i + 1;
  return m < 0 ? 0 : m;
}

// Words in front of row i of one (sequence, head): the sum of the lengths of
// the rows before it.
SUFB200_HD int64_t row_off(int n, int L, int causal, int i) {
  if (!causal) return static_cast<int64_t>(i) * L;
  const int64_t first = L - n + 1;  // length of row 0 where it is positive
  const int64_t skip = first < 0 ? -first : 0;  // rows 0 .. skip - 1 have lengths below 0: empty
  const int64_t k = i - skip;
  if (k <= 0) return 0;
  const int64_t f = first < 0 ? 0 : first;
  return k * f + k * (k - 1) / 2;
}

// Blocks of `per` items over packed sequences, as one list: the sequence with
// c items before it starts at block c / per + b, which leaves room for every
// sequence's last, partly filled block; blocks_of bounds them all.
SUFB200_HD int64_t first_block(int64_t c, int b, int per) { return c / per + b; }
inline int64_t blocks_of(int64_t items, int batch, int per) { return items / per + batch; }

// The long sequences' places in the planes' workspace: from the list where the
// call has one, else every sequence's cached tokens have room (a prompt of 2,048
// beside 32 caches of 16,384, 16 / 8 heads of 128: 32 MB and 8,320 MB).
inline int64_t plane_blocks(const AttnSeqs& s, int per) {
  return s.d_plane_keys ? s.plane_keys / per : blocks_of(s.cached, s.batch, per);
}

// Whether the list's entries p0, p1 of a sequence of L cached tokens give it
// room inside the workspace, from a whole key tile on.
SUFB200_HD bool plane_fits(const AttnSeqs& s, int p0, int p1, int L) {
  return p0 >= 0 && p0 % SUFB200_ATTN_KEY_TILE == 0 && p1 <= s.plane_keys && p1 >= p0 && p1 - p0 >= L;
}

// Whether a sequence's lengths and rows lie inside what the host arguments
// say (so every address formed from them does too); fills q.
SUFB200_HD bool seq_fits(const AttnSeqs& s, int c0, int c1, int l0, int l1, int64_t base, SeqInfo& q) {
  q = SeqInfo{0, 0, c0, l0, base, 0};
  if (l0 < 0 || l1 < l0 || l1 > s.cached) return false;
  const int L = q.L = l1 - l0;
  if (c0 < 0 || c1 < c0 || c1 > s.tokens || c1 - c0 > s.max_q || L > s.max_ctx ||
      L > static_cast<int64_t>(s.max_pages) * s.page_size || base < 0 || base > s.packed)
    return false;
  q.n = c1 - c0;
  if (s.long_ctx > 0 || s.short_rows > 0) {
    const int rows = s.q_heads / s.kv_heads * q.n;  // of a key head
    if (rows > SUFB200_ATTN_FEW_ROWS ? s.long_ctx > 0 && L > s.long_ctx : s.short_rows > 0 && rows > s.short_rows) return false;
  }
  q.blk = row_off(q.n, L, s.causal, q.n);
  return q.blk * s.q_heads <= s.packed - base;
}

// Word offset of place j % page_size of page pg, key head kh, in a pool
// [pages][kv_heads][page_size][head_dim]; -1 when the pool has no such page.
SUFB200_HD int64_t page_word(const AttnSeqs& s, int pg, int kh, int j) {
  if (pg < 0 || pg >= s.pages) return -1;
  return ((static_cast<int64_t>(pg) * s.kv_heads + kh) * s.page_size + j % s.page_size) * s.head_dim;
}

#if defined(__CUDACC__)
// The sequence block g of the list belongs to (m items per entry of cu, [batch
// + 1]; room = 0: sequences fill whole blocks and none is left between them): the
// last one that starts at or before g.  A whole warp searches, 32 sequences a round.
__device__ __forceinline__ int block_seq(const int32_t* cu, int batch, int m, int per, int64_t g, int room = 1) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, i = lo + (lane + 1) * step;
    const bool before = i < hi && first_block(static_cast<int64_t>(m) * cu[i], i * room, per) <= g;
    lo += __popc(__ballot_sync(0xffffffffu, before)) * step;
    hi = lo + step < hi ? lo + step : hi;
  }
  return lo;
}

// Sequence b; false (and the status word flagged) when the device arrays do
// not fit what the host was told.
__device__ __forceinline__ bool seq_info(const AttnSeqs& s, int b, uint32_t* status, SeqInfo& q) {
  const bool ok = seq_fits(s, s.d_cu_q[b], s.d_cu_q[b + 1], s.d_cu_ctx[b], s.d_cu_ctx[b + 1], s.d_row_base[b], q);
  if (!ok) atomicOr(status, kStatusBadArgument);
  return ok;
}

// First block of `per` keys of sequence b in the planes; -1 (and the status word
// flagged) when the list of places does not hold it.
__device__ __forceinline__ int64_t plane_first(const AttnSeqs& s, int b, const SeqInfo& q, int per, uint32_t* status) {
  if (!s.d_plane_keys) return first_block(q.l0, b, per);
  const int p0 = s.d_plane_keys[b], p1 = s.d_plane_keys[b + 1];
  if (plane_fits(s, p0, p1, q.L)) return p0 / per;
  atomicOr(status, kStatusBadArgument);
  return -1;
}

// Word offset of cached token j of sequence b, key head kh; -1 (and the
// status word flagged) when the block table names no page of the pool.
__device__ __forceinline__ int64_t key_off(const AttnSeqs& s, int b, int kh, int j, uint32_t* status) {
  const int64_t at = page_word(s, s.d_block_table[static_cast<int64_t>(b) * s.max_pages + j / s.page_size], kh, j);
  if (at < 0) atomicOr(status, kStatusBadArgument);
  return at;
}

// A 16-byte load of cached words, which one CTA reads once: past L1.
__device__ __forceinline__ ulonglong2 ld_stream(const uint64_t* p) {
  ulonglong2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u64 {%0, %1}, [%2];" : "=l"(v.x), "=l"(v.y) : "l"(p));
  return v;
}

// *p where `in`, else 0, as one predicated load: a batch of them stays a
// batch, where a conditional load may become a branch that waits.
__device__ __forceinline__ uint64_t ld_if(const uint64_t* p, bool in) {
  uint64_t v;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %2, 0;\n\t"
      "mov.u64 %0, 0;\n\t"
      "@p ld.global.nc.u64 %0, [%1];\n\t}"
      : "=l"(v)
      : "l"(p), "r"(static_cast<int>(in)));
  return v;
}
#endif

// Context check of the entry points (null, host-only, device made current).
int attn_check_ctx(sufb200_ctx ctx);

// An entry point's result: OK, or the CUDA error reported (and taken out of the
// runtime's own last error: a workspace that could not be had is not an error
// of the calls after it).
int attn_result(const char* who, cudaError_t e);

// The longest context of the sequences on the tensor cores.
inline int long_ctx(const AttnSeqs& s) { return s.long_ctx > 0 ? s.long_ctx : s.max_ctx; }

inline bool aligned_to(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// The operands of one attention product, both parties.
struct AttnOperands {
  const uint64_t* x[2];  // scores: x[0] = opened D [tokens][q_heads][head_dim]; values: the parties' shares of P (packed)
  const uint64_t* a[2];  // the triple's A: [tokens][q_heads][head_dim], or packed
  const uint64_t* c[2];  // the triple's C: packed, or [tokens][q_heads][head_dim]
  const uint64_t* e;     // opened pool [pages][kv_heads][page_size][head_dim]
  const uint64_t* b[2];  // its masks' shares
  uint64_t r;            // r_0 + r_1
  int few;               // sequences of at most this many rows per key head are another kernel's
  uint64_t* out;
  uint32_t* status;
};

// The products on the tensor cores (attention_tc.cu), for sequences with many
// rows per key head.  The values form adds to o.out unless values_tc_solo: then
// it stores whole results.
cudaError_t launch_scores_tc(const sufb200_ctx_s* ctx, const AttnSeqs& s, const AttnOperands& o, cudaStream_t st);
bool values_tc_solo(const sufb200_ctx_s* ctx, const AttnSeqs& s);
cudaError_t launch_values_tc(const sufb200_ctx_s* ctx, const AttnSeqs& s, const AttnOperands& o, cudaStream_t st);

}  // namespace sufb200

// attention_tc.cu -- the two products of attention over a cache of shares
// (attention.cu has the formula) on the tensor cores, for sequences with many
// rows per key head (prompts).
//
// A product mod 2^64 is 36 limb products of bytes, twelve tcgen05 kind::i8
// MMAs a 32-deep step into eight diagonals of int32 in tensor memory
// (umma_i8.cuh; exact up to depth 8192).  The cached operand is the M = 128
// side, the query rows the N = 64 side:
//   scores: out[key][row] = sum_k E[key][k] U[row][k] + W[key][k] D[row][k]
//   values: out[d][row]   = sum_j E[j][d]   U[row][j] + W[j][d]   D[row][j]
// with W = B_0 + B_1, U = D + A_0 + A_1: two steps per 32 of depth, one
// accumulator.  A thread of the epilogue holds one key (or word of the head)
// for 16 rows, so a warp's stores and its loads of C are 256 adjacent bytes
// whatever the packed rows' offsets are.
//
// The cached operand is read by every row tile of its group of heads, so a
// pre-pass writes its byte planes once, one contiguous 32 KB block per step
// (bulk copies, no multicast); a list of places keeps room for the long
// sequences alone.  The rows' planes are made inside: for the
// scores once per CTA (they stay in shared memory while the keys stream past),
// for the values chunk by chunk from the packed shares, which are read
// nowhere else.
//
// What bounds them (packed prompts of 2,048, 700 behind 1,024 and one token, 16
// / 4 heads of 128; 49 M scores): a step's MMAs alone take 1,170 - 1,210 cycles,
// 211 us in all, with the clock near 1.65 - 1.8 GHz under them.  On one set of
// inputs (548 and 487 us with inputs that change from pass to pass) the scores take
// 490 us: without their 24 bytes of C and output a score 411 us, without the
// keys' copies too 410 us; the MMAs alone, one tile in tensor memory at a time, take
// 1,530 cycles a step, a CTA's set-up and rows' planes 11 of its 90 us.  The values
// take 415 us: 1,580 cycles a step, the tensor core's reads of shared memory (123
// KB), the copies into it and the splitting of the shares filling its 128 bytes a
// cycle.  On the integer pipes the two took 5,030 and 5,293 us.
#include <atomic>

#include "attention.hpp"
#include "umma_i8.cuh"

namespace sufb200 {

namespace {

static_assert(kTN == SUFB200_ATTN_ROW_TILE && kTM == SUFB200_ATTN_KEY_TILE && kTM % kTK == 0, "tiles");
constexpr int kThreads = 640;  // warp 0 copies A, warp 1 issues MMAs, warps 4-19 make B planes and store
constexpr int kWorkers = 512;
constexpr uint32_t kAStage = 8 * kPlaneX;  // 32 KB: A planes of one step
constexpr uint32_t kBStage = 8 * kPlaneY;  // 16 KB: B planes of one step
constexpr int kAStages = 3;
constexpr uint32_t kBOff = kAStages * kAStage;
constexpr int kBStages = 4;  // values: two chunks of 32 keys, U and D each
constexpr uint32_t kCtrlBytes = 2048;
constexpr int kMaxDepthKeys = 4096;  // values: two products deep, 8192 in all

struct AttnTc {
  AttnSeqs s;
  AttnOperands o;
  uint8_t* planes;
  int64_t tiles;  // blocks (scores: 128 keys; values: 32 keys) per key head in `planes`
  int chunks;     // scores: 32-word chunks of the head; values: 128-word tiles of the head
  int chunk0, part;  // scores: the chunks of this launch
  int span;       // scores: key tiles per CTA; values: keys per CTA
};

// Byte i of four K-consecutive words into plane i at `at`, for all planes.
__device__ __forceinline__ void put4(uint8_t* at, uint32_t plane, const uint64_t (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const uint32_t a0 = static_cast<uint32_t>(v[0] >> (i < 4 ? 0 : 32)), a1 = static_cast<uint32_t>(v[1] >> (i < 4 ? 0 : 32));
    const uint32_t a2 = static_cast<uint32_t>(v[2] >> (i < 4 ? 0 : 32)), a3 = static_cast<uint32_t>(v[3] >> (i < 4 ? 0 : 32));
    const uint32_t sel = static_cast<uint32_t>(i & 3) | (static_cast<uint32_t>(4 + (i & 3)) << 4);
    *reinterpret_cast<uint32_t*>(at + i * plane) = __byte_perm(__byte_perm(a0, a1, sel), __byte_perm(a2, a3, sel), 0x5410);
  }
}

// A warp's unit of the rows' planes is eight rows x 16 depths.  It is loaded
// with lane = (row parity, depth), register j = row 2 j + parity (128 adjacent
// bytes of two rows a load), and turned by a 4 x 4 transpose in every group of
// four lanes: then a lane holds row 2 (lane % 4) + parity of the four depths
// 4 (lane % 16 / 4) ..., and a warp's four-byte stores of one plane cover all 32
// banks.
__device__ __forceinline__ void turn4(uint64_t (&v)[4], int lane) {
  const bool odd = lane & 1, high = lane & 2;
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const uint64_t got = __shfl_xor_sync(0xffffffffu, odd ? v[i] : v[i + 1], 1);
    v[i] = odd ? got : v[i];
    v[i + 1] = odd ? v[i + 1] : got;
  }
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const uint64_t got = __shfl_xor_sync(0xffffffffu, high ? v[i] : v[i + 2], 2);
    v[i] = high ? got : v[i];
    v[i + 2] = high ? v[i + 2] : got;
  }
}

// Where a lane of a turned unit (rows r0 ..., half h of the step) puts its bytes.
__device__ __forceinline__ uint32_t turned_off(int r0, int h, int lane) {
  return core_off(r0 + 2 * (lane & 3) + (lane >> 4), h) + 4 * ((lane & 15) >> 2);
}

// Two words at p (16-byte aligned) where `in`, else 0.
__device__ __forceinline__ void ld2_if(const uint64_t* p, bool in, uint64_t& x, uint64_t& y) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %3, 0;\n\t"
      "mov.u64 %0, 0;\n\t"
      "mov.u64 %1, 0;\n\t"
      "@p ld.global.nc.v2.u64 {%0, %1}, [%2];\n\t}"
      : "=&l"(x), "=&l"(y)
      : "l"(p), "r"(static_cast<int>(in)));
}

// *p where `in`, else 0: a word of a buffer that the same kernel writes (ld_if's
// loads are for memory that nothing writes while the kernel runs).
__device__ __forceinline__ uint64_t ld_written_if(const uint64_t* p, bool in) {
  uint64_t v;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %2, 0;\n\t"
      "mov.u64 %0, 0;\n\t"
      "@p ld.global.u64 %0, [%1];\n\t}"
      : "=l"(v)
      : "l"(p), "r"(static_cast<int>(in))
      : "memory");
  return v;
}

// The cached operand's byte planes.  KEYS: block (128-key tile, chunk of 32
// words), rows = keys; else block (32 keys, 128-word tile), rows = words of
// the head.  Out-of-range rows and depths are zero.
template <bool KEYS>
__global__ void __launch_bounds__(256) cache_planes_kernel(const __grid_constant__ AttnTc a) {
  pdl_trigger();
  __shared__ int64_t s_key[kTM];
  const AttnSeqs& s = a.s;
  constexpr int kPer = KEYS ? kTM : kTK;
  const int t = threadIdx.x, kh = blockIdx.z;
  const bool places = s.d_plane_keys != nullptr;
  const int b = block_seq(places ? s.d_plane_keys : s.d_cu_ctx, s.batch, 1, kPer, blockIdx.x, places ? 0 : 1);
  SeqInfo q;
  if (!seq_info(s, b, a.o.status, q) || s.q_heads / s.kv_heads * q.n <= a.o.few) return;
  const int64_t plane = plane_first(s, b, q, kPer, a.o.status), first = blockIdx.x - plane;  // this block in its sequence
  if (plane < 0 || first < 0 || first * kPer >= q.L) return;
  const int j0 = static_cast<int>(first) * kPer;
  for (int e = t; e < kPer; e += 256) s_key[e] = j0 + e < q.L ? key_off(s, b, kh, j0 + e, a.o.status) : -1;
  __syncthreads();
  const int64_t block = ((kh * a.tiles + blockIdx.x) * a.chunks + blockIdx.y) * 2;
  uint8_t* dst = a.planes + block * kAStage;
  // two units of four words at a time: their loads before the first use
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    uint64_t e[2][4], w[2][4], v[2][4];
#pragma unroll
    for (int y = 0; y < 2; y++) {
      const int u = t + 256 * (i + y), deep = 16 * (u >> 9) + 4 * (u & 3), r = (u >> 2) & (kTM - 1);
      if (KEYS) {  // four words of a key; the head's size is even
        const int64_t at = s_key[r];
        const int word = static_cast<int>(blockIdx.y) * kTK + deep;
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          const bool in = at >= 0 && word + j < s.head_dim;
          ld2_if(a.o.e + at + word + j, in, e[y][j], e[y][j + 1]);
          ld2_if(a.o.b[0] + at + word + j, in, w[y][j], w[y][j + 1]);
          ld2_if(a.o.b[1] + at + word + j, in, v[y][j], v[y][j + 1]);
        }
      } else {  // a word of four keys
        const int word = static_cast<int>(blockIdx.y) * kTM + r;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int64_t at = s_key[deep + j];
          const bool in = at >= 0 && word < s.head_dim;
          e[y][j] = ld_if(a.o.e + at + word, in);
          w[y][j] = ld_if(a.o.b[0] + at + word, in);
          v[y][j] = ld_if(a.o.b[1] + at + word, in);
        }
      }
    }
#pragma unroll
    for (int y = 0; y < 2; y++) {
      const int u = t + 256 * (i + y);
      uint8_t* at = dst + core_off((u >> 2) & (kTM - 1), u >> 9) + 4 * (u & 3);
#pragma unroll
      for (int j = 0; j < 4; j++) w[y][j] += v[y][j];
      put4(at, kPlaneX, e[y]);
      put4(at + kAStage, kPlaneX, w[y]);
    }
  }
}

// True in one lane of the (converged) warp, always the same one.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// The mbarriers and flags behind the stages.
struct Ctrl {
  uint32_t afull, aempty, bfull, bempty, tfull, tempty, done, slot;
  volatile uint32_t* err;
  uint32_t* tmem_slot;
  int64_t* row;  // [64] scores: first word of a row; values: its first packed word
  int* len;      // [64] its keys
};

__device__ __forceinline__ Ctrl ctrl_at(uint8_t* smem, uint32_t off) {
  Ctrl c;
  const uint32_t base = smem_u32(smem) + off;
  c.afull = base;
  c.aempty = base + 8 * kAStages;
  c.bfull = base + 16 * kAStages;
  c.bempty = c.bfull + 8 * kBStages;
  c.tfull = c.bempty + 8 * kBStages;
  c.tempty = c.tfull + 8;
  c.done = c.tempty + 8;
  c.slot = c.done + 8;
  uint8_t* p = smem + off + (c.slot - base);
  c.tmem_slot = reinterpret_cast<uint32_t*>(p);
  c.err = reinterpret_cast<volatile uint32_t*>(p + 4);
  c.row = reinterpret_cast<int64_t*>(smem + off + 512);
  c.len = reinterpret_cast<int*>(smem + off + 512 + 8 * kTN);
  return c;
}
static_assert(16 * kAStages + 16 * kBStages + 32 <= 512 && 512 + 12 * kTN <= kCtrlBytes, "control block");

// Tensor memory and barriers; every thread of the CTA.  A CTA takes all 512
// columns, so they start at column 0 and the accumulators' addresses are
// constants; false (and *err set) should they not.
__device__ __forceinline__ bool start(const Ctrl& c, int warp, int t, int bwarps) {
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(c.slot), "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (t == 0) {
    for (int i = 0; i < kAStages; i++) {
      mbar_init(c.afull + 8 * i, 1);
      mbar_init(c.aempty + 8 * i, 1);
    }
    for (int i = 0; i < kBStages; i++) {
      mbar_init(c.bfull + 8 * i, bwarps);
      mbar_init(c.bempty + 8 * i, 1);
    }
    mbar_init(c.tfull, 1);
    mbar_init(c.tempty, kWorkers / 32);
    mbar_init(c.done, 1);
    mbar_init_fence();
    *c.err = 0;
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (*c.tmem_slot != 0) *c.err = 1;
  return *c.tmem_slot == 0;
}

// All threads: report a wait that gave up, let what was issued finish (again
// with a limit) and free the tensor memory.  `copies` = A copies issued.
__device__ __forceinline__ void stop(const Ctrl& c, uint32_t* status, int warp, int lane, int copies) {
  __syncthreads();
  if (*c.err) {
    if (warp == 0 && lane == 0) {
      atomicOr(status, kStatusTimeout);
      for (int i = copies > kAStages ? copies - kAStages : 0; i < copies; i++)
        mbar_wait(c.afull + 8 * (i % kAStages), static_cast<uint32_t>((i / kAStages) & 1));
    }
    if (warp == 1) {
      if (elect_one()) umma_commit(c.done);
      __syncwarp();
      mbar_wait(c.done, 0);
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 0) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*c.tmem_slot), "r"(kTmemCols) : "memory");
  }
}

// Lane 0 of the producer warp: the A planes of one step into the ring.
__device__ __forceinline__ bool load_a(const Ctrl& c, uint32_t sbase, int li, const uint8_t* src) {
  const int st = li % kAStages;
  if (li >= kAStages && !mbar_wait(c.aempty + 8 * st, static_cast<uint32_t>(((li / kAStages) - 1) & 1))) return false;
  mbar_expect_tx(c.afull + 8 * st, kAStage);
  bulk_copy(sbase + static_cast<uint32_t>(st) * kAStage, src, kAStage, c.afull + 8 * st);
  return true;
}

// 4 columns of this warp's 32 lanes; the registers are valid after tmem_wait4.
__device__ __forceinline__ void tmem_ld4(uint32_t taddr, uint32_t (&v)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(taddr));
}

__device__ __forceinline__ void tmem_wait4(uint32_t (&v)[4]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]) : : "memory");
}

// sum_s (P_s mod 2^32) << 8s of 16 columns from `col` on, for this thread's
// lane; four columns at a time (all eight diagonals of more would spill).
__device__ __forceinline__ void fold16(int quarter, int col, uint64_t (&z)[16]) {
#pragma unroll
  for (int cb = 0; cb < 4; cb++) {
    uint32_t v[8][4];
#pragma unroll
    for (int sd = 0; sd < 8; sd++)
      tmem_ld4((static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(sd * kTN + col + cb * 4), v[sd]);
#pragma unroll
    for (int sd = 0; sd < 8; sd++) tmem_wait4(v[sd]);
#pragma unroll
    for (int x = 0; x < 4; x++) {
      uint64_t lo = v[0][x];
#pragma unroll
      for (int sd = 1; sd < 4; sd++) lo += static_cast<uint64_t>(v[sd][x]) << (8 * sd);
      const uint32_t hi = v[4][x] + (v[5][x] << 8) + (v[6][x] << 16) + (v[7][x] << 24);
      z[cb * 4 + x] = lo + (static_cast<uint64_t>(hi) << 32);
    }
  }
}

// The twelve MMAs of one step (the products of ring_gemm_tc.cu's mma_step in
// another order) on the A planes at shared address a and the B planes at b:
// x_i times [y_j ...] for N = 256, accumulated at column 64 (i + j), lands every
// product (i, j) on its diagonal i + j.  The tensor core's queue
// is short: it runs dry whenever the issuing warp is held up for longer than
// the last MMAs it was given take, and a wait for the next step's planes holds
// it up by about 200 cycles even when they are there.  So a step is issued in
// two parts, 416 cycles of MMAs in the last, and the
// next step's wait stands between them (a step took 0.90 us with the wait in
// front, 0.63 us of it MMAs).  For the same reason accumulators, shapes and the
// descriptors' high words are constants; only two 32-bit bases vary.
__device__ __forceinline__ uint64_t plane_desc(uint32_t base_lo, uint32_t planes_off) {
  return static_cast<uint64_t>(base_lo + (planes_off >> 4)) | (static_cast<uint64_t>((1u << 14) | (256u >> 4)) << 32);
}
__device__ __forceinline__ uint32_t desc_base(uint32_t saddr) { return (saddr >> 4) | ((128u >> 4) << 16); }

// x_i times [y_j ...] for N = 256, fewer where the 512 columns end.
__device__ __forceinline__ void issue_one(uint32_t al, uint32_t bl, int i, int j, uint32_t accumulate) {
  const int n = 64 * (8 - i - j);
  umma_i8((i + j) * kTN, plane_desc(al, i * kPlaneX), plane_desc(bl, j * kPlaneY), idesc_n(n < 256 ? n : 256), accumulate);
}

__device__ __forceinline__ void issue_first(uint32_t a, uint32_t b, uint32_t accumulate) {
  const uint32_t al = desc_base(a), bl = desc_base(b);
  issue_one(al, bl, 0, 0, accumulate);  // these two write all 512 columns
  issue_one(al, bl, 0, 4, accumulate);
  issue_one(al, bl, 7, 0, 1u);
  issue_one(al, bl, 6, 0, 1u);
  issue_one(al, bl, 5, 0, 1u);
  issue_one(al, bl, 4, 0, 1u);
  issue_one(al, bl, 3, 4, 1u);
  issue_one(al, bl, 3, 0, 1u);
}

__device__ __forceinline__ void issue_last(uint32_t a, uint32_t b) {
  const uint32_t al = desc_base(a), bl = desc_base(b);
  issue_one(al, bl, 2, 4, 1u);
  issue_one(al, bl, 2, 0, 1u);
  issue_one(al, bl, 1, 4, 1u);
  issue_one(al, bl, 1, 0, 1u);
}

// Row tile `tile` of the call: its sequence and its first row, rho0 = -1 when
// there is none.  From the list of tiles, or counting through the sequences,
// each from its last (longest) rows on.
struct TileOf {
  SeqInfo q;
  int b, R, rho0;
};

__device__ __forceinline__ TileOf tile_of(const AttnTc& a, int tile) {
  const AttnSeqs& s = a.s;
  const int group = s.q_heads / s.kv_heads;
  TileOf t{};
  t.rho0 = -1;
  const bool list = s.d_tiles != nullptr;
  t.b = list ? s.d_tiles[2 * tile] : block_seq(s.d_cu_q, s.batch, group, kTN, tile);
  if (t.b < 0 || t.b >= s.batch) {
    atomicOr(a.o.status, kStatusBadArgument);
    return t;
  }
  if (!seq_info(s, t.b, a.o.status, t.q) || group * t.q.n <= a.o.few) return t;
  t.R = group * t.q.n;
  const int64_t tiles = (t.R + kTN - 1) / kTN;
  const int64_t i = list ? s.d_tiles[2 * tile + 1] : tiles - 1 - (tile - first_block(static_cast<int64_t>(group) * t.q.t0, t.b, kTN));
  if (i >= 0 && i < tiles) t.rho0 = static_cast<int>(i) * kTN;
  return t;
}

// Row tiles a launch enumerates.
int64_t row_tiles(const AttnSeqs& s) {
  return s.d_tiles ? s.n_tiles : blocks_of(s.q_heads / s.kv_heads * s.tokens, s.batch, kTN);
}

// FIRST: the head's first part, which adds C and r; else its second part, which
// adds to the first one's words in o.out.
template <bool FIRST>
__global__ void __launch_bounds__(kThreads, 1) scores_tc_kernel(const __grid_constant__ AttnTc a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const AttnSeqs& s = a.s;
  const AttnOperands& o = a.o;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, dh = s.head_dim, group = s.q_heads / s.kv_heads;
  const int kh = blockIdx.x % s.kv_heads;
  const TileOf tile = tile_of(a, blockIdx.x / s.kv_heads);
  const SeqInfo& q = tile.q;
  const int b = tile.b, R = tile.R, rho0 = tile.rho0;
  const int last = (rho0 + kTN < R ? rho0 + kTN : R) - 1;
  const int len = rho0 >= 0 && rho0 < R ? row_len(q.n, q.L, s.causal, last / group) : 0;
  const int nt = (len + kTM - 1) / kTM, tile0 = blockIdx.y * a.span;
  const int tiles = nt - tile0 < a.span ? nt - tile0 : a.span;
  const int64_t plane = tiles > 0 ? plane_first(s, b, q, kTM, o.status) : -1;
  if (plane < 0) {
    pdl_wait();
    return;
  }
  const int steps = 2 * a.part;
  const uint32_t sbase = smem_u32(smem);
  const Ctrl c = ctrl_at(smem, kBOff + static_cast<uint32_t>(steps) * kBStage);
  if (t < kTN) {
    const int rho = rho0 + t;
    c.row[t] = rho < R ? (static_cast<int64_t>(q.t0 + rho / group) * s.q_heads + kh * group + rho % group) * dh : -1;
  }
  const bool ready = start(c, warp, t, kThreads / 32 - 2);
  int copies = 0;

  if (!ready) {
  } else if (warp == 0) {  // A planes: every step of every key tile
    pdl_wait();  // written by the pre-pass
    const int64_t next = 2 * static_cast<int64_t>(a.chunks) * kAStage;  // from a key tile to the one after
    const uint8_t* src = a.planes + (kh * a.tiles + plane + tile0) * next + 2 * a.chunk0 * kAStage;
    int go = 1;
    for (int tl = 0; tl < tiles && go; tl++, src += next)
      for (int st = 0; st < steps && go; st++) {
        if (lane == 0) {
          go = load_a(c, sbase, copies, src + static_cast<int64_t>(st) * kAStage);
          if (!go) *c.err = 1;
        }
        go = __shfl_sync(0xffffffffu, go, 0);
        copies += go;
      }
  } else if (warp == 1) {  // MMAs
    // The whole warp waits and steps, one elected lane issues: step, stage and
    // descriptors stay warp-uniform.
    const auto landed = [&](int li) {
      const bool ok = mbar_wait(c.afull + 8 * (li % kAStages), static_cast<uint32_t>((li / kAStages) & 1));
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      return __all_sync(0xffffffffu, ok) != 0;
    };
    bool go = __all_sync(0xffffffffu, mbar_wait(c.bfull, 0)) && landed(0);  // the rows' planes, the first keys'
    for (int tl = 0, li = 0; tl < tiles && go; tl++) {
      if (tl > 0) {  // the last tile is out of tensor memory
        go = __all_sync(0xffffffffu, mbar_wait(c.tempty, static_cast<uint32_t>((tl - 1) & 1)));
        if (!go) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      }
      for (int st = 0; st < steps && go; st++, li++) {
        const int as = li % kAStages;
        const uint32_t at = sbase + static_cast<uint32_t>(as) * kAStage, bt = sbase + kBOff + static_cast<uint32_t>(st) * kBStage;
        if (elect_one()) issue_first(at, bt, st > 0 ? 1u : 0u);
        __syncwarp();
        if (li + 1 < tiles * steps) go = landed(li + 1);
        if (elect_one()) {
          issue_last(at, bt);
          umma_commit(c.aempty + 8 * as);
          if (st + 1 == steps) umma_commit(c.tfull);
        }
        __syncwarp();
      }
    }
    if (!go && lane == 0) *c.err = 1;
  } else {
    // the rows' planes [U | D]: the loads of two units, then their splitting
    const int units = a.part * (kTN / 4);
    for (int u0 = warp - 2; u0 < units; u0 += 2 * (kThreads / 32 - 2)) {
      uint64_t d[2][4], w[2][4], x[2][4];
#pragma unroll
      for (int y = 0; y < 2; y++) {
        const int u = u0 + y * (kThreads / 32 - 2), k = (a.chunk0 + u / (kTN / 4)) * kTK + 16 * (u & 1) + (lane & 15);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int64_t row = c.row[u % (kTN / 4) / 2 * 8 + 2 * j + (lane >> 4)];
          const bool in = row >= 0 && u < units && k < dh;
          d[y][j] = ld_if(o.x[0] + row + k, in);
          w[y][j] = ld_if(o.a[0] + row + k, in);
          x[y][j] = ld_if(o.a[1] + row + k, in);
        }
      }
#pragma unroll
      for (int y = 0; y < 2; y++) {
        const int u = u0 + y * (kThreads / 32 - 2);
        if (u >= units) break;
#pragma unroll
        for (int j = 0; j < 4; j++) w[y][j] += d[y][j] + x[y][j];
        turn4(w[y], lane);
        turn4(d[y], lane);
        uint8_t* at = smem + kBOff + static_cast<uint32_t>(2 * (u / (kTN / 4))) * kBStage +
                      turned_off(u % (kTN / 4) / 2 * 8, u & 1, lane);
        put4(at, kPlaneY, w[y]);
        put4(at + kBStage, kPlaneY, d[y]);
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // generic writes -> tensor core reads
    __syncwarp();
    if (lane == 0) mbar_arrive(c.bfull);
  }
  if (ready && warp >= 4) {  // epilogue: while the next tile's MMAs run
    // The MMAs take most of the shared-memory bandwidth and every multiply of
    // an address would stand in this warp's chain, so the rows' places are
    // stepped from one row to the next (row_off, row_len by differences).  C is
    // fetched eight rows ahead of the stores, the first eight while the tile's
    // MMAs still run (four rows ahead: 16 heads of 64 402 us, eight 384; more in
    // flight would spill).
    const int quarter = warp & 3, col = ((warp - 4) >> 2) * 16;
    const int i0 = (rho0 + col) / group, g0 = (rho0 + col) % group;  // the first row's query and head of the group
    const int rows = R - rho0 - col;                                 // rows there are, from there on
    const int64_t at0 = q.base + static_cast<int64_t>(kh * group) * q.blk + row_off(q.n, q.L, s.causal, i0);
    const int len0 = s.causal ? q.L - q.n + i0 + 1 : q.L;
    for (int tl = 0; tl < tiles; tl++) {
      const int key = (tile0 + tl) * kTM + quarter * 32 + lane;
      // this query's row of the group's first head, and this row: one walk for
      // the loads of C, eight rows ahead, one for the stores
      int lg = g0, llen = len0, sg = g0, slen = len0;
      int64_t lrow = at0 + key, lat = lrow + g0 * q.blk, srow = lrow, sat = lat;
      const auto next = [&](int& g, int& len, int64_t& row, int64_t& at) {
        at += q.blk;
        if (++g == group) {
          g = 0;
          row += len > 0 ? len : 0;
          at = row;
          len += s.causal ? 1 : 0;
        }
      };
      uint64_t c0[2][4], c1[2][4];
      const auto fetch = [&](int x0) {
#pragma unroll
        for (int x = 0; x < 4; x++) {
          const bool in = x0 + x < rows && key < llen;
          c0[(x0 >> 2) & 1][x] = FIRST ? ld_if(o.c[0] + lat, in) : ld_written_if(o.out + lat, in);
          c1[(x0 >> 2) & 1][x] = FIRST ? ld_if(o.c[1] + lat, in) : 0;
          next(lg, llen, lrow, lat);
        }
      };
      fetch(0);
      fetch(4);
      int go = 1;
      if (lane == 0) go = mbar_wait(c.tfull, static_cast<uint32_t>(tl & 1));
      if (!__shfl_sync(0xffffffffu, go, 0)) {
        if (lane == 0) *c.err = 1;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      uint64_t z[16];
      fold16(quarter, col, z);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(c.tempty);
#pragma unroll
      for (int x0 = 0; x0 < 16; x0 += 4) {
#pragma unroll
        for (int x = 0; x < 4; x++) {
          if (x0 + x < rows && key < slen) o.out[sat] = z[x0 + x] + c0[(x0 >> 2) & 1][x] + c1[(x0 >> 2) & 1][x] + (FIRST ? o.r : 0);
          next(sg, slen, srow, sat);
        }
        if (x0 < 8) fetch(x0 + 8);
      }
    }
  }
  stop(c, o.status, warp, lane, copies);
}

// SOLO: one CTA has all keys of a row tile and stores; else the ranges add to
// out, which holds C_0 + C_1 + r.
template <bool SOLO>
__global__ void __launch_bounds__(kThreads, 1) values_tc_kernel(const __grid_constant__ AttnTc a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const AttnSeqs& s = a.s;
  const AttnOperands& o = a.o;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, dh = s.head_dim, group = s.q_heads / s.kv_heads;
  const int kh = blockIdx.x % s.kv_heads, dt0 = blockIdx.x / s.kv_heads % a.chunks;
  const TileOf tile = tile_of(a, blockIdx.x / s.kv_heads / a.chunks);
  const SeqInfo& q = tile.q;
  const int b = tile.b, R = tile.R, rho0 = tile.rho0;
  const int last = (rho0 + kTN < R ? rho0 + kTN : R) - 1;
  const int len = rho0 >= 0 && rho0 < R ? row_len(q.n, q.L, s.causal, last / group) : 0;
  const int beg = blockIdx.y * a.span, end = len < beg + a.span ? len : beg + a.span;
  const int nch = end > beg ? (end - beg + kTK - 1) / kTK : 0;
  const int word0 = dt0 * kTM;
  // word `word` of the output of row rho
  const auto place = [&](int rho, int word) {
    return (static_cast<int64_t>(q.t0 + rho / group) * s.q_heads + kh * group + rho % group) * dh + word;
  };
  if (nch == 0) {
    pdl_wait();
    if (SOLO && rho0 >= 0 && rho0 < R)  // rows without keys: C_0 + C_1 + r
      for (int e = t; e < kTN * kTM; e += kThreads) {
        const int rho = rho0 + e / kTM, word = word0 + e % kTM;
        if (rho < R && word < dh) o.out[place(rho, word)] = o.c[0][place(rho, word)] + o.c[1][place(rho, word)] + o.r;
      }
    return;
  }
  const int64_t plane = plane_first(s, b, q, kTK, o.status);
  if (plane < 0) {
    pdl_wait();
    return;
  }
  const uint32_t sbase = smem_u32(smem);
  const Ctrl c = ctrl_at(smem, kBOff + kBStages * kBStage);
  if (t < kTN) {
    const int rho = rho0 + t, i = rho / group;
    const int m = rho < R ? row_len(q.n, q.L, s.causal, i) : 0;
    c.row[t] = rho < R ? q.base + (kh * group + rho % group) * q.blk + row_off(q.n, q.L, s.causal, i) : 0;
    c.len[t] = m < end ? m : end;
  }
  const bool ready = start(c, warp, t, kWorkers / 32);
  int copies = 0;

  if (!ready) {
  } else if (warp == 0) {
    pdl_wait();
    const int64_t block0 = kh * a.tiles + plane + beg / kTK;
    for (int li = 0; li < 2 * nch; li++) {
      int go = 1;
      if (lane == 0) {
        go = load_a(c, sbase, li, a.planes + (((block0 + li / 2) * a.chunks + dt0) * 2 + (li & 1)) * kAStage);
        if (!go) *c.err = 1;
      }
      if (!__shfl_sync(0xffffffffu, go, 0)) break;
      copies++;
    }
  } else if (warp == 1) {
    const auto landed = [&](int li) {
      const bool ok = mbar_wait(c.afull + 8 * (li % kAStages), static_cast<uint32_t>((li / kAStages) & 1)) &&
                      mbar_wait(c.bfull + 8 * (li % kBStages), static_cast<uint32_t>((li / kBStages) & 1));
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      return __all_sync(0xffffffffu, ok) != 0;
    };
    bool go = landed(0);
    for (int li = 0; li < 2 * nch && go; li++) {
      const int as = li % kAStages, bs = li % kBStages;
      const uint32_t at = sbase + static_cast<uint32_t>(as) * kAStage, bt = sbase + kBOff + static_cast<uint32_t>(bs) * kBStage;
      if (elect_one()) issue_first(at, bt, li > 0 ? 1u : 0u);
      __syncwarp();
      if (li + 1 < 2 * nch) go = landed(li + 1);
      if (elect_one()) {
        issue_last(at, bt);
        umma_commit(c.aempty + 8 * as);
        umma_commit(c.bempty + 8 * bs);
        if (li + 1 == 2 * nch) umma_commit(c.tfull);
      }
      __syncwarp();
    }
    if (!go && lane == 0) *c.err = 1;
  } else if (warp >= 4) {
    // A worker warp has one unit of every chunk.  The next chunk's shares are in
    // flight while this one's are split.
    const int r0 = ((warp - 4) >> 1) * 8, h = warp & 1;
    int64_t row[4];
    int m[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      row[j] = c.row[r0 + 2 * j + (lane >> 4)];
      m[j] = c.len[r0 + 2 * j + (lane >> 4)];
    }
    uint64_t p0[4], p1[4], a0[4], a1[4];
    const auto fetch = [&](int ch) {
      const int key = beg + ch * kTK + 16 * h + (lane & 15);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const bool in = key < m[j];
        p0[j] = ld_if(o.x[0] + row[j] + key, in);
        p1[j] = ld_if(o.x[1] + row[j] + key, in);
        a0[j] = ld_if(o.a[0] + row[j] + key, in);
        a1[j] = ld_if(o.a[1] + row[j] + key, in);
      }
    };
    fetch(0);
    int go = 1;
    const uint32_t mine = turned_off(r0, h, lane);
    for (int ch = 0; ch < nch; ch++) {
      uint64_t d[4], u[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        d[j] = (p0[j] - a0[j]) + (p1[j] - a1[j]);
        u[j] = d[j] + a0[j] + a1[j];
      }
      if (ch + 1 < nch) fetch(ch + 1);
      turn4(u, lane);
      turn4(d, lane);
      const int su = (2 * ch) % kBStages, sd = su + 1;
      if (lane == 0 && 2 * ch >= kBStages)
        go = mbar_wait(c.bempty + 8 * su, static_cast<uint32_t>(((2 * ch / kBStages) - 1) & 1)) &&
             mbar_wait(c.bempty + 8 * sd, static_cast<uint32_t>(((2 * ch / kBStages) - 1) & 1));
      if (!__shfl_sync(0xffffffffu, go, 0)) {
        if (lane == 0) *c.err = 1;
        break;
      }
      uint8_t* at = smem + kBOff + static_cast<uint32_t>(su) * kBStage + mine;
      put4(at, kPlaneY, u);
      put4(at + kBStage, kPlaneY, d);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // generic writes -> tensor core reads
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(c.bfull + 8 * su);
        mbar_arrive(c.bfull + 8 * sd);
      }
    }
    const int quarter = warp & 3, col = ((warp - 4) >> 2) * 16;
    const int word = word0 + quarter * 32 + lane, left = R - rho0 - col;  // rows there are from column 0 on
    int g = (rho0 + col) % group;
    int64_t at = left > 0 ? place(rho0 + col, word) : 0;
    const auto next = [&] {  // the row after: the group's next head, or the next token's first
      at += dh;
      if (++g == group) {
        g = 0;
        at += static_cast<int64_t>(s.q_heads - group) * dh;
      }
    };
    uint64_t c0[8], c1[8];
    const auto fetch_c = [&](int x0) {  // C of eight rows; leaves the walk where it was
      const int g1 = g;
      const int64_t at1 = at;
#pragma unroll
      for (int x = 0; x < 8; x++) {
        const bool in = x0 + x < left && word < dh;
        c0[x] = ld_if(o.c[0] + at, in);
        c1[x] = ld_if(o.c[1] + at, in);
        next();
      }
      g = g1;
      at = at1;
    };
    if (SOLO) fetch_c(0);  // while the last MMAs run
    if (lane == 0 && go) go = mbar_wait(c.tfull, 0);
    if (__shfl_sync(0xffffffffu, go, 0)) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      uint64_t z[16];
      fold16(quarter, col, z);
      if (SOLO) {
#pragma unroll
        for (int x0 = 0; x0 < 16; x0 += 8) {
          if (x0 > 0) fetch_c(x0);
#pragma unroll
          for (int x = 0; x < 8; x++) {
            if (x0 + x < left && word < dh) o.out[at] = z[x0 + x] + c0[x] + c1[x] + o.r;
            next();
          }
        }
      } else {
#pragma unroll
        for (int x = 0; x < 16; x++) {
          if (x < left && word < dh)
            atomicAdd(reinterpret_cast<unsigned long long*>(o.out + at), static_cast<unsigned long long>(z[x]));
          next();
        }
      }
    } else if (lane == 0) {
      *c.err = 1;
    }
  }
  stop(c, o.status, warp, lane, copies);
}

// Launch, as the pre-pass's programmatic dependent if `after_planes`; the kernel
// may take all shared memory, said once per kernel and device.
template <int WHICH>
cudaError_t launch(const sufb200_ctx_s* ctx, void (*kernel)(AttnTc), dim3 grid, size_t smem, cudaStream_t st,
                   const AttnTc& a, bool after_planes = true) {
  constexpr int kMaxDevices = 64;
  static std::atomic<bool> ready[kMaxDevices];
  const bool known = ctx->device < kMaxDevices;
  if (!known || !ready[ctx->device].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e != cudaSuccess) return e;
    if (known) ready[ctx->device].store(true, std::memory_order_release);
  }
  if (after_planes) return launch_pdl(kernel, grid, dim3(kThreads), smem, st, a);
  kernel<<<grid, kThreads, smem, st>>>(a);
  return cudaGetLastError();
}

// Most chunks of the head whose row planes stay in shared memory beside three A
// stages; wider heads take a second launch that adds to the first one's words
// (2,048 tokens, 16 / 4 heads of 256: 646 us, 6,527 on the integer pipes).
constexpr int kMostChunks = 4;

}  // namespace

cudaError_t launch_scores_tc(const sufb200_ctx_s* ctx, const AttnSeqs& s, const AttnOperands& o, cudaStream_t st) {
  const int64_t rts = row_tiles(s);
  const int nt = (long_ctx(s) + kTM - 1) / kTM;
  AttnTc a{s, o, nullptr, plane_blocks(s, kTM), (s.head_dim + kTK - 1) / kTK, 0, 0, 0};
  const int64_t bytes = a.tiles * s.kv_heads * a.chunks * 2 * static_cast<int64_t>(kAStage);
  cudaError_t e = cudaMallocFromPoolAsync(reinterpret_cast<void**>(&a.planes), bytes, ctx->pool, st);
  if (e != cudaSuccess) return e;
  // key tiles per CTA, by the longest of these sequences' own contexts (by the
  // batch's, 64 tokens behind 4,096 beside a single one with 65,536 cached, 32 / 8
  // heads, took 717 us, 457 now; the values 703 and 449): long runs reuse the rows' planes and hide the epilogue
  // behind the next tile; two CTAs an SM in all even out, more cost more set-ups
  // (16 / 4 heads of 128, 1,024 tokens: 112 us, 141 by four an SM; 256 behind
  // 4,096: 192 and 224 us; 64 behind 8,000, 32 / 8 heads: 214 and 259 us)
  const int64_t all = nt * rts * s.kv_heads, two = static_cast<int64_t>(ctx->sm_count) * 2;
  a.span = static_cast<int>((all + two - 1) / two < nt ? (all + two - 1) / two : nt);
  cache_planes_kernel<true><<<dim3(static_cast<unsigned>(a.tiles), a.chunks, s.kv_heads), 256, 0, st>>>(a);
  e = cudaGetLastError();
  const dim3 grid(static_cast<unsigned>(rts * s.kv_heads), (nt + a.span - 1) / a.span);
  for (a.chunk0 = 0; a.chunk0 < a.chunks && e == cudaSuccess; a.chunk0 += a.part) {
    a.part = a.chunks - a.chunk0 < kMostChunks ? a.chunks - a.chunk0 : kMostChunks;
    const size_t smem = kBOff + static_cast<size_t>(2 * a.part) * kBStage + kCtrlBytes;
    e = a.chunk0 == 0 ? launch<0>(ctx, scores_tc_kernel<true>, grid, smem, st, a)
                      : launch<3>(ctx, scores_tc_kernel<false>, grid, smem, st, a, false);
  }
  const cudaError_t f = cudaFreeAsync(a.planes, st);
  return e == cudaSuccess ? f : e;
}

// Keys per CTA of the values form, and whether one CTA takes whole rows.
int values_span(const sufb200_ctx_s* ctx, const AttnSeqs& s) {
  const int nch = (long_ctx(s) + kTK - 1) / kTK, words = (s.head_dim + kTM - 1) / kTM;
  const int64_t units = row_tiles(s) * words * s.kv_heads;
  // whole rows where there is more than one row tile an SM (no pass that starts
  // the output from C: 16 / 4 heads of 128, 1,024 tokens 83 us, 94 split), else
  // two CTAs an SM in all, of eight chunks at least (256 behind 4,096: 154 us, 162
  // by equal parts, 180 by four CTAs an SM); at most the exact depth
  const int64_t two = static_cast<int64_t>(ctx->sm_count) * 2, even = (units * nch + two - 1) / two;
  const int64_t want = two / units < 2 ? nch : (even < 8 ? 8 : even);
  const int span = static_cast<int>(want < nch ? want : nch) * kTK;
  return span > kMaxDepthKeys ? kMaxDepthKeys : span;
}

bool values_tc_solo(const sufb200_ctx_s* ctx, const AttnSeqs& s) { return values_span(ctx, s) >= long_ctx(s); }

cudaError_t launch_values_tc(const sufb200_ctx_s* ctx, const AttnSeqs& s, const AttnOperands& o, cudaStream_t st) {
  AttnTc a{s, o, nullptr, plane_blocks(s, kTK), (s.head_dim + kTM - 1) / kTM, 0, 0, values_span(ctx, s)};
  const int64_t bytes = a.tiles * s.kv_heads * a.chunks * 2 * static_cast<int64_t>(kAStage);
  cudaError_t e = cudaMallocFromPoolAsync(reinterpret_cast<void**>(&a.planes), bytes, ctx->pool, st);
  if (e != cudaSuccess) return e;
  cache_planes_kernel<false><<<dim3(static_cast<unsigned>(a.tiles), a.chunks, s.kv_heads), 256, 0, st>>>(a);
  e = cudaGetLastError();
  const size_t smem = kBOff + kBStages * kBStage + kCtrlBytes;
  const dim3 grid(static_cast<unsigned>(row_tiles(s) * a.chunks * s.kv_heads), (long_ctx(s) + a.span - 1) / a.span);
  if (e == cudaSuccess)
    e = a.span >= long_ctx(s) ? launch<1>(ctx, values_tc_kernel<true>, grid, smem, st, a)
                            : launch<2>(ctx, values_tc_kernel<false>, grid, smem, st, a);
  const cudaError_t f = cudaFreeAsync(a.planes, st);
  return e == cudaSuccess ? f : e;
}

}  // namespace sufb200

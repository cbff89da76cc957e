// Products of e4m3 operands with one fp32 scale for each block of 128, on sm_100a tensor cores.
//
//   y[r, n] = sum_b xs[r, b] * ws[e, n / 128, b] * sum_{j in block b} xq[r, j] * wq[e, n, j]
//
// x has a scale for each row and 128 columns, the weights [E, N, K] one for each 128 x 128 block
// (the layout of 8-bit checkpoints); rows come in segments, each with its stack entry e.  The
// scales differ from one 128-wide step of the reduction to the next, so a tensor-core accumulator
// may only span one step: each step's MMAs start a fresh TMEM accumulator, and the epilogue warps
// read it back, multiply by the step's scales and add into fp32 registers while the tensor cores
// work on the next step in another accumulator.
//
// Gated form (the gate/up half of an expert): h = act(x Wg^T) * (x Wu^T) leaves as e4m3 codes
// with a scale for each row and 128 columns, made from the fp32 accumulators in the epilogue; it
// is the input of the down product, which is the plain form.
//
// Two kernels of one shape, x as the MMA's M and 256 weight rows as its N:
//   pair    256 rows of x on two SMs (tcgen05 cta_group::2): many rows a segment, bound by the tensor
//           cores.
//   single  a row tile of 32, 64 or 128 rows on one SM: few rows a segment, bound by reading the
//           weights.  With few tiles the reduction is split over a cluster and joined through
//           distributed shared memory, in the order of the ranks.
// The weights are never the M operand, although they have more rows than a decode batch: an MMA takes
// 123 cycles to load its 128 rows of M whatever N is (128 for N = 256), so 256 weight rows a step
// cost 4 x 128 cycles as N and 8 x 123 as M.  For the same reason an accumulator is 256 columns, and
// TMEM holds two: a step's MMAs (512 cycles) and its way through the epilogue (about 1,000: commit, wake,
// 128 columns a warp read and added, hand-back) overlap with the next step's and no further.
//
// What bounds them, measured on a B200: many rows, the way of an accumulator from its first MMA to its
// hand-back, about 1,400 cycles, which two accumulators share: a step takes 700-720 cycles where its MMAs
// take 512 (4096 x 14336 x 4096 in 216-230 us, 2.1-2.2 PFLOP/s, against 174 us for the same loop without
// scales, one read-back a tile; long runs meet the power cap besides); few rows, HBM (512 rows over 32
// experts of 7168/2048: gate/up 939 MB in 160 us, down 470 MB in 85 us, 5.5-5.9 TB/s); one token
// through 14336 x 4096, 59 MB in 16 us: 1.3 us to set up, 11 us of memory, 2.7 us to join and leave.
#include <cuda_fp8.h>

#include "dmoe_common.cuh"
#include "tcgen05.cuh"

namespace dmoe {
namespace {

constexpr int kBlk = 128;          // scale block; also bytes of one swizzle row of codes
constexpr int kMaxSegs = 1024;     // device segment tables
constexpr int kMaxHostSegs = 256;  // host tables travel in the launch parameters
constexpr int kEpiWarps = 8;

struct BlkSegs {
  int n_seg, m_rows, e_stack;
  const int32_t* dev_expert;
  const int32_t* dev_end;
  int32_t expert[kMaxHostSegs];
  int32_t end[kMaxHostSegs];
};

struct BlkArgs {
  const float* xs;  // row scales: [row * xs_ld + kb]
  int64_t xs_ld;
  const float* ws0;  // [e][n_blk][k_blk] scales of the (gate) weights, and of the up weights
  const float* ws1;
  int n_out;      // valid output columns (weight rows)
  int K;          // reduction length
  int n_tiles_n;  // output column tiles
  int n_blk, k_blk;
  int act;
  void* out;  // plain: rows of out_dtype; gated: e4m3 codes
  int64_t ldo;
  int out_dtype;
  float* out_scale;  // gated: [row * os_ld + column block]
  int64_t os_ld;
  int32_t* status;
  // plain only: store row r at scatter_base[code >> 27] + (code & 0x7ffffff) rows with
  // code = scatter_map[r] (negative: not stored) instead of at row r of `out`; the bases may be
  // other GPUs' memory.
  // The kernel before this one in the stream is the gate/up product of the same call: it writes
  // nothing but this one's x and its scales, so the weights and the segment table are read before
  // it has ended (it waited for its own predecessors before it let this one start).
  int early;
  int scatter;
  const int32_t* scatter_map;
  char* scatter_base[DMOE_EP_MAX_RANKS];
};

// Segment table in shared memory: rows [start, end) of stack entry `expert`, first row tile `tile`.
struct SegTable {
  int32_t* start;
  int32_t* end;
  int32_t* expert;
  int32_t* tile;  // [n_seg + 1]
};
constexpr int kSegTableBytes = 4 * (kMaxSegs + 4) * 4;

__device__ __forceinline__ SegTable seg_table_at(void* p) {
  int32_t* b = reinterpret_cast<int32_t*>(p);
  return SegTable{b, b + (kMaxSegs + 4), b + 2 * (kMaxSegs + 4), b + 3 * (kMaxSegs + 4)};
}

// The whole CTA fetches the table at once (one trip to memory), ...
__device__ __forceinline__ void fetch_segments(const BlkSegs& segs, const SegTable& t) {
  for (int i = threadIdx.x; i < segs.n_seg; i += blockDim.x) {
    t.end[i] = segs.dev_end ? segs.dev_end[i] : segs.end[i];
    t.expert[i] = segs.dev_expert ? segs.dev_expert[i] : segs.expert[i];
  }
}

// ... and one warp makes tiles of it, a run of segments in each lane: ends are clamped to [previous
// end, m_rows] (reported in *status where that changes one), entries outside the stack are left out.
__device__ __forceinline__ void read_segments(const BlkSegs& segs, const SegTable& t, int tile_m, int32_t* status) {
  const int lane = threadIdx.x & 31;
  const int n = segs.n_seg;
  const int run = (n + 31) >> 5;
  const int i0 = min(lane * run, n), i1 = min(i0 + run, n);
  int top = 0;  // running maximum of the clamped ends, over this lane's run, then over those before
  for (int i = i0; i < i1; ++i) top = max(top, min(t.end[i], segs.m_rows));
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, top, o);
    if (lane >= o) top = max(top, v);
  }
  int prev = __shfl_up_sync(0xffffffffu, top, 1);
  if (lane == 0) prev = 0;
  int tiles = 0, bad = 0;
  for (int i = i0; i < i1; ++i) {
    const int given = t.end[i], e = t.expert[i];
    const int en = max(min(given, segs.m_rows), prev);
    const bool in_stack = e >= 0 && e < segs.e_stack;
    bad |= given != en || !in_stack;
    t.start[i] = prev;
    t.end[i] = in_stack ? en : prev;
    t.expert[i] = in_stack ? e : 0;
    t.tile[i] = tiles;
    if (in_stack) tiles += (en - prev + tile_m - 1) / tile_m;
    prev = en;
  }
  int before = tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += v;
  }
  if (lane == 31) t.tile[n] = before;
  before -= tiles;
  for (int i = i0; i < i1; ++i) t.tile[i] += before;
  if (__any_sync(0xffffffffu, bad) && lane == 0 && blockIdx.x == 0) atomicOr(status, DMOE_DEVERR_BAD_SEGMENT);
}

struct BlkTile {
  int row0, row_end, expert, nt;
};

// Tiles go segment by segment, row tiles fastest: those in flight together share one expert's
// weight rows, which come from memory once and then from L2.
__device__ __forceinline__ BlkTile blk_tile(int tile, int n_tiles_n, int n_seg, int tile_m, const SegTable& t) {
  int lo = 0, hi = n_seg - 1;  // last segment whose first tile is <= tile (skips empty segments)
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((int64_t)t.tile[mid] * n_tiles_n <= tile) lo = mid; else hi = mid - 1;
  }
  const int m_tiles = t.tile[lo + 1] - t.tile[lo];
  const int local = tile - t.tile[lo] * n_tiles_n;
  const int nt = local / m_tiles;
  return BlkTile{t.start[lo] + (local - nt * m_tiles) * tile_m, t.end[lo], t.expert[lo], nt};
}

// acc += v * s on two lanes of packed fp32.
__device__ __forceinline__ void fma2(uint64_t& acc, uint32_t v0, uint32_t v1, uint64_t s2) {
  asm("{\n\t.reg .b64 v;\n\tmov.b64 v, {%1, %2};\n\tfma.rn.f32x2 %0, v, %3, %0;\n\t}" : "+l"(acc) : "r"(v0), "r"(v1), "l"(s2));
}
__device__ __forceinline__ uint64_t pack_f2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(__float_as_uint(a)), "r"(__float_as_uint(b)));
  return r;
}
__device__ __forceinline__ float2 unpack_f2(uint64_t v) {
  uint32_t a, b;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
  return make_float2(__uint_as_float(a), __uint_as_float(b));
}

constexpr float kFinite = 3.402823466e38f;

// silu(g) = g / (1 + 2^(-g log2 e)) or relu(g), by the two approximate instructions (2 ulp each; a
// sigmoid below 2^-126 is 0).  Without flushing, the subnormals that cannot matter here cost as many
// instructions again.
template <int ACT>
__device__ __forceinline__ float blk_act(float g) {
  if constexpr (ACT != DMOE_ACT_SILU) return relu_fn(g);
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.442695041f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return g * r;
}

// Scale of a block with this largest finite magnitude.
__device__ __forceinline__ float block_scale(float amax) {
  return amax > 0.f ? fmaxf(__fdiv_rn(amax, 448.f), 1.17549435e-38f) : 1.f;
}

__device__ __forceinline__ float finite_abs(float v) { return fabsf(v) <= kFinite ? fabsf(v) : 0.f; }

// Four codes of h * inv (NaN stays NaN).
__device__ __forceinline__ uint32_t codes4(const float* h, float inv) {
  const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(h[0] * inv, h[1] * inv), __NV_SATFINITE, __NV_E4M3);
  const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(h[2] * inv, h[3] * inv), __NV_SATFINITE, __NV_E4M3);
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

// Where row `row` of a plain product goes (nullptr: not stored).
__device__ __forceinline__ char* blk_out_row(const BlkArgs& a, int row, int esz) {
  if (!a.scatter) return reinterpret_cast<char*>(a.out) + (int64_t)row * a.ldo * esz;
  const int32_t code = a.scatter_map[row];
  if (code < 0) return nullptr;
  char* base = a.scatter_base[(uint32_t)code >> 27];
  return base == nullptr ? nullptr : base + (int64_t)(code & 0x7ffffff) * a.ldo * esz;
}

// 32 lanes x 16 or 32 fp32 columns in two halves: the registers hold their values after the second,
// which waits for every load this warp has started.
__device__ __forceinline__ void tmem_ld_start(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : DMOE_R8(0), DMOE_R8(8)
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_start(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : DMOE_R8(0), DMOE_R8(8), DMOE_R8(16), DMOE_R8(24)
      : "r"(taddr)
      : "memory");
}
#define BLK_RW8(b) "+r"(r[b + 0]), "+r"(r[b + 1]), "+r"(r[b + 2]), "+r"(r[b + 3]), "+r"(r[b + 4]), "+r"(r[b + 5]), \
                   "+r"(r[b + 6]), "+r"(r[b + 7])
__device__ __forceinline__ void tmem_ld_finish(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : BLK_RW8(0), BLK_RW8(8)::"memory");
}
__device__ __forceinline__ void tmem_ld_finish(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : BLK_RW8(0), BLK_RW8(8), BLK_RW8(16), BLK_RW8(24)::"memory");
}
#undef BLK_RW8

// kind::f8f6f4, D fp32, A and B e4m3 (format 0), both K-major.
__host__ __device__ constexpr uint32_t blk_idesc(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// mbar_wait without a call: the sums held in registers would be spilled around one.  REMOTE: the
// arrivals come from the other CTA too, by mbar_arrive_remote.
template <bool REMOTE = false>
__device__ __forceinline__ bool wait_in_line(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int32_t* status,
                                             int code) {
  auto done = [&] { return REMOTE ? mbar_try_wait_remote(bar, parity) : mbar_try_wait(bar, parity); };
  if (done()) return true;
  const uint64_t t0 = global_timer_ns();
  while (!done()) {
    if (*abort_flag) return false;
    if (global_timer_ns() - t0 > kWaitTimeoutNs) {
      *abort_flag = 1;
      atomicOr(status, code);
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ void wait_or_report(uint64_t* bar, uint32_t parity, int32_t* status) {
  if (mbar_try_wait(bar, parity)) return;
  const uint64_t t0 = global_timer_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (global_timer_ns() - t0 > kWaitTimeoutNs) {
      atomicOr(status, DMOE_DEVERR_TIMEOUT_TEARDOWN);
      break;
    }
  }
}

// Programmatic dependent launch: a product starts while the kernel before it in the stream drains,
// sets itself up, and waits here for that kernel's results.  The next kernel may be launched once
// every CTA has passed its own wait.
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_kernel_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// --------------------------------------------------------------------- the epilogue of both kernels
// Eight epilogue warps: warp pairs share a lane quadrant (rows of x), each takes half of the 256
// columns (gated: 64 gate and the matching 64 up columns), 128 fp32 sums a thread.  The sums need more
// registers than 65,536 / 384 threads: the first warpgroup (TMA, MMA, segment table, one idle warp)
// hands its own to the other two.
constexpr int kN = 256;                // weight rows of a tile: gated 128 gate and 128 up rows
constexpr int kThreadsBlk = 128 + 32 * kEpiWarps;
// Registers a thread after the hand-over; both sides of the split have to hold their own without
// spills (the issuing warps spilled at 40: 224 -> 377 us for 4096 x 14336 x 4096).
struct RegSplit {
  int issue, sums;
};
constexpr RegSplit kWide{56, 224}, kEven{72, 216};
static_assert(128 * kWide.issue + 256 * kWide.sums == kThreadsBlk * 168 &&
                  128 * kEven.issue + 256 * kEven.sums == kThreadsBlk * 168,
              "a split hands out the registers the block was launched with");
constexpr int kOpBytes = 128 * kBlk;             // one step of 128 operand rows
constexpr int kBarBytes = 256;
constexpr int kXchBytes = 2 * 2 * 128 * 4;
constexpr int kOutBytes = kEpiWarps * 32 * 128;  // 128 bytes of 32 rows for each epilogue warp

template <bool GATED>
__device__ __forceinline__ int tmem_col(int half, int c) {  // column c of this warp's 128
  return GATED ? (c < 64 ? half * 64 + c : 64 + half * 64 + c) : half * 128 + c;
}

// Reads back this warp's 32 rows and 128 columns of an accumulator and adds them, scaled; `release`
// hands the accumulator back as soon as the last columns are in registers.
// C columns are loaded at a time, the next C while these are added: 32 where the registers allow it.
template <bool GATED, int C, class F>
__device__ __forceinline__ void add_step(uint64_t (&sum)[64], uint32_t tbase, int half, float s0, float s1, F&& release) {
  const uint64_t s0p = pack_f2(s0, s0), s1p = pack_f2(s1, s1);
  uint32_t v[2][C];
  tmem_ld_start(tbase + tmem_col<GATED>(half, 0), v[0]);
#pragma unroll
  for (int j = 0; j < 128 / C; ++j) {
    tmem_ld_finish(v[j & 1]);
    if (j < 128 / C - 1)
      tmem_ld_start(tbase + tmem_col<GATED>(half, (j + 1) * C), v[(j + 1) & 1]);
    else
      release();
#pragma unroll
    for (int i = 0; i < C / 2; ++i)
      fma2(sum[j * (C / 2) + i], v[j & 1][2 * i], v[j & 1][2 * i + 1], j * C < 64 ? s0p : s1p);
  }
}

__device__ __forceinline__ bool normal(float s) { return fabsf(s) >= 1.17549435e-38f && fabsf(s) <= kFinite; }

// x = significand * 2^e with 1 <= |significand| < 2, x finite and not 0.
__device__ __forceinline__ float significand(float x, int& e) {
  const bool sub = !normal(x);
  const int b = __float_as_int(sub ? x * 16777216.f : x);
  e = ((b >> 23) & 255) - (sub ? 127 + 24 : 127);
  return __int_as_float((b & 0x807fffff) | 0x3f800000);
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

// Factors c1 * c2 = x * w where the product is no normal number (else 0 * 0), although the sum of a step's
// codes (a multiple of 2^-18 below 2^26) times it may be one: c1 has the significands and as much of the
// exponent as keeps sum * c1 normal, c2 is a power of two (past its range every result is 0 or infinite in
// fp32).  Zeros, infinities and NaN are taken as they are.
__device__ __forceinline__ float2 two_factors(float x, float w) {
  const float s = x * w;
  if (normal(s)) return make_float2(0.f, 0.f);
  if (!(fabsf(x) <= kFinite && fabsf(w) <= kFinite) || x == 0.f || w == 0.f) return make_float2(s, 1.f);
  int ex, ew;
  const float m = significand(x, ex) * significand(w, ew);
  const int e = ex + ew, e1 = min(max(e, -96), 96);
  return make_float2(m * power_of_two(e1), power_of_two(min(max(e - e1, -126), 127)));
}

// A scale.  Not by the read-only path: this kernel may have started before the one ahead of it in the stream,
// which may be writing these, had ended, and that path takes only what no one writes while a kernel runs.
__device__ __forceinline__ float scale_at(const float* p) { return *p; }

// add_step where the product of two scales is no normal number in some lane: sums times the normal products
// as there, then the others as (sum * c1) * c2.  x, w0, w1: the step's scales, read once more.
template <bool GATED, class F>
__device__ __forceinline__ void add_step_any(uint64_t (&sum)[64], uint32_t tbase, int half, const float* x, const float* w0,
                                             const float* w1, F&& release) {
  const float xs = scale_at(x);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float w = scale_at(!GATED || j < 4 ? w0 : w1), s = normal(xs * w) ? xs * w : 0.f;
    const float2 c = two_factors(xs, w);
    const uint64_t sp = pack_f2(s, s), p1 = pack_f2(c.x, c.x), p2 = pack_f2(c.y, c.y);
    uint32_t v[16];
    tmem_ld_start(tbase + tmem_col<GATED>(half, j * 16), v);
    tmem_ld_finish(v);
    if (j == 7) release();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint64_t t = 0;
      fma2(t, v[2 * i], v[2 * i + 1], p1);
      const float2 f = unpack_f2(t);
      fma2(sum[j * 8 + i], v[2 * i], v[2 * i + 1], sp);
      fma2(sum[j * 8 + i], __float_as_uint(f.x), __float_as_uint(f.y), p2);
    }
  }
}

// Results of a tile, the row `row` in each lane.  They go through shared memory (`st`: this warp's
// 4 KB), so that a store instruction writes runs of 64 or 128 bytes of a few rows rather than 16
// bytes of 32: 6,300 cycles a tile before, at 256 columns of bf16.

template <int ACT>
__device__ __forceinline__ void gated_values(const uint64_t (&sum)[64], float (&h)[64], float& top) {
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const float2 g = unpack_f2(sum[i]), u = unpack_f2(sum[32 + i]);
    h[2 * i] = blk_act<ACT>(g.x) * u.x;
    h[2 * i + 1] = blk_act<ACT>(g.y) * u.y;
    top = fmaxf(top, fmaxf(fabsf(h[2 * i]), fabsf(h[2 * i + 1])));
  }
}

// h = act(gate) * up as codes, with the scale of the row's 128 columns; the other 64 of them are in
// the warp that shares this quadrant (`xch`: both warps' largest magnitudes).
__device__ __forceinline__ void store_codes(const uint64_t (&sum)[64], const BlkArgs& a, int row, int row_end, bool ok,
                                            int nt, int half, int q, uint32_t* xch, uint4* st) {
  const int lane = threadIdx.x & 31;
  float h[64];
  float top = 0.f;  // fmaxf prefers a number to NaN, so only an infinity shows in it
  if (a.act == DMOE_ACT_SILU)
    gated_values<DMOE_ACT_SILU>(sum, h, top);
  else
    gated_values<DMOE_ACT_RELU>(sum, h, top);
  if (top > kFinite) {  // infinities become NaN codes and leave the scale alone
    top = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) {
      top = fmaxf(top, finite_abs(h[i]));
      if (fabsf(h[i]) > kFinite) h[i] = __int_as_float(0x7fffffff);
    }
  }
  xch[half * 128 + q * 32 + lane] = __float_as_uint(top);
  named_sync(1 + q, 64);
  const float s = block_scale(fmaxf(top, __uint_as_float(xch[(half ^ 1) * 128 + q * 32 + lane])));
  const float inv = __frcp_rn(s);
  if (half == 0 && ok && row < row_end) a.out_scale[(int64_t)row * a.os_ld + nt] = s;
#pragma unroll
  for (int v = 0; v < 4; ++v)
    st[lane * 4 + (v ^ ((lane >> 1) & 3))] = make_uint4(codes4(h + v * 16, inv), codes4(h + v * 16 + 4, inv),
                                                        codes4(h + v * 16 + 8, inv), codes4(h + v * 16 + 12, inv));
  __syncwarp();
  const int col = nt * 128 + half * 64 + (lane & 3) * 16;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + (lane >> 2);
    const uint4 v = st[r * 4 + ((lane & 3) ^ ((r >> 1) & 3))];
    const int64_t orow = row - lane + r;
    if (ok && orow < row_end && col < a.n_out)
      *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(a.out) + orow * a.ldo + col) = v;
  }
  __syncwarp();
}

// A plain product's columns, rounded to the output type.
__device__ __forceinline__ void store_rows(const uint64_t (&sum)[64], const BlkArgs& a, int row, bool valid, int nt,
                                           int half, uint4* st) {
  const int lane = threadIdx.x & 31;
  const bool f32 = a.out_dtype == DMOE_F32;
  const int esz = f32 ? 4 : 2;
  const int col0 = nt * kN + half * 128;
  char* const dst = valid ? blk_out_row(a, row, esz) : nullptr;
  const int vec = 16 / esz;  // columns of 16 bytes
#pragma unroll
  for (int p = 0; p < 4; ++p) {  // 32 columns a thread; 128 bytes of each row at a time
    if (f32) {
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        const float2 x = unpack_f2(sum[p * 16 + 2 * v]), y = unpack_f2(sum[p * 16 + 2 * v + 1]);
        st[lane * 8 + (v ^ (lane & 7))] =
            make_uint4(__float_as_uint(x.x), __float_as_uint(x.y), __float_as_uint(y.x), __float_as_uint(y.y));
      }
    } else {
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        uint32_t pk[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 x = unpack_f2(sum[p * 16 + 4 * v + i]);
          pk[i] = a.out_dtype == DMOE_BF16 ? pack2<DMOE_BF16>(x.x, x.y) : pack2<DMOE_F16>(x.x, x.y);
        }
        st[lane * 8 + (((p & 1) * 4 + v) ^ (lane & 7))] = make_uint4(pk[0], pk[1], pk[2], pk[3]);
      }
      if ((p & 1) == 0) continue;
    }
    __syncwarp();
    const int col = col0 + (f32 ? p * 32 : (p >> 1) * 64) + (lane & 7) * vec;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = i * 4 + (lane >> 3);
      char* to = reinterpret_cast<char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), r));
      const uint4 v = st[r * 8 + ((lane & 7) ^ (r & 7))];
      if (to != nullptr && col < a.n_out) *reinterpret_cast<uint4*>(to + (int64_t)col * esz) = v;
    }
    __syncwarp();
  }
}

// Scales of the steps of one row and of the two column blocks of a tile, each fetched a step ahead.
struct StepScales {
  const float *x, *w0, *w1;
  float xn, an, bn;
  template <bool GATED>
  __device__ __forceinline__ void start(const BlkArgs& a, const BlkTile& t, int row, bool valid, int half, int kb) {
    x = a.xs + (int64_t)(valid ? row : t.row0) * a.xs_ld;
    // Gated: this column block of both stacks; plain: this half's block (the last tile's second half
    // may lie past the last block: its sums are never stored).
    const int nb = GATED ? t.nt : min(t.nt * 2 + half, a.n_blk - 1);
    const int64_t at = ((int64_t)t.expert * a.n_blk + nb) * a.k_blk;
    w0 = a.ws0 + at;
    w1 = GATED ? a.ws1 + at : w0;
    xn = scale_at(x + kb);
    an = scale_at(w0 + kb);
    bn = GATED ? scale_at(w1 + kb) : an;
  }
  template <bool GATED>
  __device__ __forceinline__ void take(int kb, int end, float& s0, float& s1) {
    s0 = xn * an;
    s1 = xn * bn;
    if (kb + 1 < end) {
      xn = scale_at(x + kb + 1);
      an = scale_at(w0 + kb + 1);
      bn = GATED ? scale_at(w1 + kb + 1) : an;
    }
  }
};

// ------------------------------------------------------------------------------- pair kernel
// A CTA pair computes 256 rows x 256 weight rows.  Each CTA loads its 128 rows of x and its 128 weight
// rows (gated: CTA 0 the gate rows, CTA 1 the up rows); its TMEM holds its 128 rows of x by all 256
// columns, twice.
constexpr int kPM = 256;
constexpr int kPStages = 5;
constexpr int kPStageBytes = 2 * kOpBytes;
constexpr int kPSmemBytes = 1024 + kPStages * kPStageBytes + kOutBytes + kBarBytes + kXchBytes + kSegTableBytes;

template <bool GATED>
__global__ void __launch_bounds__(kThreadsBlk, 1)
    blk_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w0,
                    const __grid_constant__ CUtensorMap tm_w1, const __grid_constant__ BlkSegs segs,
                    const __grid_constant__ BlkArgs args) {
  constexpr RegSplit kSplit = GATED ? kEven : kWide;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* out_buf = smem + kPStages * kPStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(out_buf + kOutBytes);
  uint64_t* empty = full + kPStages;
  uint64_t* accf = empty + kPStages;
  uint64_t* acce = accf + 2;
  uint64_t* fin = acce + 2;
  uint64_t* bye = fin + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bye + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* xch = reinterpret_cast<uint32_t*>(out_buf + kOutBytes + kBarBytes);
  const SegTable tab = seg_table_at(out_buf + kOutBytes + kBarBytes + kXchBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1;
  const int n_pairs = gridDim.x >> 1;

  if (threadIdx.x == 64) {
    tma_prefetch_map(&tm_x);
    tma_prefetch_map(GATED && rank == 1 ? &tm_w1 : &tm_w0);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < kPStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&accf[a], 1);
      mbar_init(&acce[a], 2 * kEpiWarps);
    }
    mbar_init(fin, 1);
    mbar_init(bye, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 2 * kN);
    tmem_relinquish_pair();
  }
  wait_for_previous_kernel();
  let_next_kernel_start();
  fetch_segments(segs, tab);
  tc_fence_before();
  __syncthreads();
  if (warp == 2) read_segments(segs, tab, kPM, args.status);
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers exist before any remote arrive or TMA signal
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int total = tab.tile[segs.n_seg] * args.n_tiles_n;
  const int nk = args.k_blk;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kSplit.issue));
  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer (both CTAs)
    if (lane == 0) {
      const uint32_t full_leader0 = map_to_cta(smem_u32(&full[0]), 0);
      int stage = 0;
      uint32_t ph = 0, armed = 0, armed_ph = 0;
      bool ok = true;
      for (int tile = pair; tile < total && ok; tile += n_pairs) {
        const BlkTile ti = blk_tile(tile, args.n_tiles_n, segs.n_seg, kPM, tab);
        const int xrow = ti.row0 + (int)rank * 128;
        const int wrow = GATED ? ti.nt * 128 : ti.nt * kN + (int)rank * 128;
        const CUtensorMap* tw = (GATED && rank == 1) ? &tm_w1 : &tm_w0;
        for (int kb = 0; kb < nk; ++kb) {
          if (!mbar_wait(&empty[stage], ph ^ 1u, abort_flag, args.status, DMOE_DEVERR_TIMEOUT_PRODUCER)) {
            ok = false;
            break;
          }
          uint8_t* sx = smem + stage * kPStageBytes;
          const uint32_t fbar = full_leader0 + (uint32_t)(stage * sizeof(uint64_t));
          if (leader) mbar_arrive_expect_tx(&full[stage], 2 * kPStageBytes);
          tma_load_2d_pair(sx, &tm_x, fbar, kb * kBlk, xrow);
          tma_load_3d_pair(sx + kOpBytes, tw, fbar, kb * kBlk, wrow, ti.expert);
          armed |= 1u << stage;
          armed_ph = (armed_ph & ~(1u << stage)) | (ph << stage);
          if (++stage == kPStages) {
            stage = 0;
            ph ^= 1u;
          }
        }
      }
      // The leader's full barriers count both CTAs' bytes: wait for every phase it armed.
      if (leader)
        for (int s = 0; s < kPStages; ++s)
          if (armed >> s & 1u) wait_or_report(&full[s], armed_ph >> s & 1u, args.status);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (leader CTA)
    // The whole warp walks the steps and one lane issues: with uniform control flow around it an
    // issue takes a fraction of what it does inside a branch of one lane.
    if (leader) {
      constexpr uint32_t idesc = blk_idesc(kPM, kN);
      const uint64_t xd0 = sdesc_sw128(smem_u32(smem)), wd0 = sdesc_sw128(smem_u32(smem + kOpBytes));
      int stage = 0, acc = 0;
      uint32_t ph = 0, acc_ph = 0;
      bool ok = true;
      for (int tile = pair; tile < total && ok; tile += n_pairs) {
        for (int kb = 0; kb < nk; ++kb) {
          ok = wait_in_line(&full[stage], ph, abort_flag, args.status, DMOE_DEVERR_TIMEOUT_MMA) &&
               wait_in_line<true>(&acce[acc], acc_ph ^ 1u, abort_flag, args.status, DMOE_DEVERR_TIMEOUT_MMA);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t off = (uint64_t)(stage * (kPStageBytes >> 4));
#pragma unroll
            for (int k = 0; k < 4; ++k)  // 32 codes of K per MMA; the first starts a fresh sum
              umma_f16_pair<DMOE_E4M3>(tmem_base + (uint32_t)(acc * kN), xd0 + off + 2 * k, wd0 + off + 2 * k, idesc,
                                       k != 0);
            umma_commit_both(&empty[stage]);
            umma_commit_both(&accf[acc]);
          }
          __syncwarp();
          if (++stage == kPStages) {
            stage = 0;
            ph ^= 1u;
          }
          acc ^= 1;
          if (acc == 0) acc_ph ^= 1u;
        }
      }
      if (elect_one()) umma_commit_both(fin);
      __syncwarp();
    }
    // Every MMA of the pair (issued by the leader) has completed once `fin` fires in this CTA.
    if (lane == 0) wait_or_report(fin, 0, args.status);
  }
  } else {
    // ------------------------------------------------------------------ epilogue (both CTAs)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSplit.sums));
    const int q = warp & 3;  // TMEM lane quadrant this warp may access
    const int half = (warp - 4) >> 2;
    const uint32_t acce_leader0 = map_to_cta(smem_u32(&acce[0]), 0);
    uint4* st = reinterpret_cast<uint4*>(out_buf + (warp - 4) * 32 * 128);
    int acc = 0, flip = 0;
    uint32_t acc_ph = 0;
    bool ok = true;
    for (int tile = pair; tile < total; tile += n_pairs, flip ^= 1) {
      const BlkTile ti = blk_tile(tile, args.n_tiles_n, segs.n_seg, kPM, tab);
      const int row = ti.row0 + (int)rank * 128 + q * 32 + lane;
      const bool valid = row < ti.row_end;
      StepScales sc;
      sc.start<GATED>(args, ti, row, valid, half, 0);
      uint64_t sum[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) sum[i] = 0;
      for (int kb = 0; kb < nk && ok; ++kb) {
        float s0, s1;
        sc.take<GATED>(kb, nk, s0, s1);
        const uint32_t at = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * kN);
        auto release = [&] {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_remote(acce_leader0 + (uint32_t)(acc * sizeof(uint64_t)));
        };
        ok = wait_in_line(&accf[acc], acc_ph, abort_flag, args.status, DMOE_DEVERR_TIMEOUT_EPILOGUE);
        // One vote for the wait and the scales: of a large product it costs 2 %, a vote and a branch more 5 %.
        if (__all_sync(0xffffffffu, ok && normal(s0) && (!GATED || normal(s1)))) {
          tc_fence_after();
          add_step<GATED, 32>(sum, at, half, s0, s1, release);
        } else {
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          add_step_any<GATED>(sum, at, half, sc.x + kb, sc.w0 + kb, sc.w1 + kb, release);
        }
        acc ^= 1;
        if (acc == 0) acc_ph ^= 1u;
      }
      // After a wait that ran out nothing is stored, but the warps that share a quadrant still meet.
      if constexpr (GATED)
        store_codes(sum, args, row, ti.row_end, ok, ti.nt, half, q, xch + flip * 256, st);
      else
        store_rows(sum, args, row, valid && ok, ti.nt, half, st);
    }
  }

  if (args.scatter) __threadfence_system();  // scattered rows may live in other GPUs' memory
  tc_fence_before();
  __syncthreads();
  // Exit handshake: tell the peer this CTA is done with the pair's shared state, then wait
  // (bounded) until the peer says the same.
  if (threadIdx.x == 0) {
    mbar_arrive_cluster(map_to_cta(smem_u32(bye), rank ^ 1u));
    wait_or_report(bye, 0, args.status);
  }
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 2 * kN);
  }
}

// ----------------------------------------------------------------------------- single-SM kernel
// Row tiles of tile_m rows (32, 64 or 128) x 256 weight rows.  The MMA's M is 128: the rows past the
// tile come from whatever lies behind it in shared memory, give rows of D that nobody reads, and
// the warps of their quadrants only pass the accumulators on.
// With SPLIT the CTAs of a cluster take parts of the reduction of the same tile where whole tiles would
// leave SMs idle (few tiles, or the last wave of many); each leaves its sums in its own shared memory
// (where the operands were) and finishes some of the rows, adding the ranks' sums in order.
__host__ __device__ constexpr int single_stage_bytes(int tile_m) { return tile_m * kBlk + 2 * kOpBytes; }
constexpr int kSingleFixed = 1024 + kOutBytes + kBarBytes + kXchBytes + kSegTableBytes;
__host__ __device__ constexpr int single_stages(int tile_m) {
  return (227 * 1024 - kSingleFixed) / single_stage_bytes(tile_m);
}
static_assert(single_stages(32) <= 8 && single_stages(128) >= 3, "stages of the single-SM kernel");
// Sums of a split tile, 256 fp32 a row, fit where the operands were.
static_assert(32 * kN * 4 <= single_stages(32) * single_stage_bytes(32) &&
                  64 * kN * 4 <= single_stages(64) * single_stage_bytes(64) &&
                  128 * kN * 4 <= single_stages(128) * single_stage_bytes(128),
              "sums of a split tile");

__device__ __forceinline__ float4 ld_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

template <bool GATED, bool SPLIT>
__global__ void __launch_bounds__(kThreadsBlk, 1)
    blk_single_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w0,
                      const __grid_constant__ CUtensorMap tm_w1, const __grid_constant__ BlkSegs segs,
                      const __grid_constant__ BlkArgs args, const int tile_m, const int stages, const int ranks) {
  constexpr RegSplit kSplit = GATED || SPLIT ? kEven : kWide;
  constexpr int kCols = GATED || SPLIT ? 16 : 32;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  // Rows of x first: an MMA reads 128 of them from the start of a stage's tile_m.
  uint8_t* wbuf = smem + stages * tile_m * kBlk;
  uint8_t* out_buf = wbuf + stages * 2 * kOpBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(out_buf + kOutBytes);
  uint64_t* empty = full + 8;
  uint64_t* accf = empty + 8;
  uint64_t* acce = accf + 2;
  uint64_t* fin = acce + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(fin + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* xch = reinterpret_cast<uint32_t*>(out_buf + kOutBytes + kBarBytes);
  const SegTable tab = seg_table_at(out_buf + kOutBytes + kBarBytes + kXchBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 64) {
    tma_prefetch_map(&tm_w0);
    if (GATED) tma_prefetch_map(&tm_w1);
    tma_prefetch_map(&tm_x);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&accf[a], 1);
      mbar_init(&acce[a], tile_m / 32 * 2);  // the warps of the quadrants that a tile can reach
    }
    mbar_init(fin, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 2 * kN);
    tmem_relinquish();
  }
  const bool early = !GATED && args.early;
  if (!early) {
    wait_for_previous_kernel();
    let_next_kernel_start();
  }
  fetch_segments(segs, tab);
  tc_fence_before();
  __syncthreads();
  if (warp == 2) read_segments(segs, tab, tile_m, args.status);
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int total = tab.tile[segs.n_seg] * args.n_tiles_n;
  // Tiles [0, whole) go to one CTA each, in waves of the grid; with SPLIT the last ones, where they
  // would leave SMs idle, go to a cluster each.  A tile costs its steps and about two more, a split
  // one its part of them, about eight for the two meetings and more with its rows.
  const int grid = (int)gridDim.x;
  int whole = total, rank = 0;
  if constexpr (SPLIT) {
    const int clusters = grid / ranks, left = total % grid;
    const int part = args.k_blk / ranks + 8 + tile_m / 8;
    if (left > 0 && (int64_t)((left + clusters - 1) / clusters) * part <= args.k_blk + 2) whole = total - left;
    rank = (int)cluster_ctarank();
  }
  const int whole_here = whole > (int)blockIdx.x ? (whole - (int)blockIdx.x + grid - 1) / grid : 0;
  struct Item {
    int tile, kb0, kb1;
    bool parts;
  };
  auto item = [&](int it) {  // tile >= total: no more
    if (!SPLIT || it < whole_here) return Item{it < whole_here ? (int)blockIdx.x + it * grid : total, 0, args.k_blk, false};
    return Item{whole + (int)blockIdx.x / ranks + (it - whole_here) * (grid / ranks),
                (int)((int64_t)args.k_blk * rank / ranks), (int)((int64_t)args.k_blk * (rank + 1) / ranks), true};
  };

  // Every role walks the same tiles; at a split one all warps of the cluster's CTAs meet twice (sums
  // written; sums read), which also keeps the next tile's operands off the sums.
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kSplit.issue));
    int stage = 0, acc = 0;
    uint32_t ph = 0, acc_ph = 0, armed = 0, armed_ph = 0;
    bool ok = true;
    const uint64_t xd0 = sdesc_sw128(smem_u32(smem)), wd0 = sdesc_sw128(smem_u32(wbuf));
    auto load_w = [&](const BlkTile& ti, int kb, int at) {
      uint8_t* sw = wbuf + at * 2 * kOpBytes;
      mbar_arrive_expect_tx(&full[at], single_stage_bytes(tile_m));
      if constexpr (GATED) {
        tma_load_3d(sw, &tm_w0, &full[at], kb * kBlk, ti.nt * 128, ti.expert);
        tma_load_3d(sw + kOpBytes, &tm_w1, &full[at], kb * kBlk, ti.nt * 128, ti.expert);
      } else {
        tma_load_3d(sw, &tm_w0, &full[at], kb * kBlk, ti.nt * kN, ti.expert);
      }
    };
    int ahead = 0;  // steps of the first tile whose weights were asked for early
    if (early && warp == 0) {
      const Item first = item(0);
      if (first.tile < total) {
        const BlkTile ti = blk_tile(first.tile, args.n_tiles_n, segs.n_seg, tile_m, tab);
        ahead = min(stages, first.kb1 - first.kb0);
        if (elect_one())
          for (int i = 0; i < ahead; ++i) load_w(ti, first.kb0 + i, i);
        __syncwarp();
      }
      wait_for_previous_kernel();
      let_next_kernel_start();
    } else if (early && warp == 1) {
      wait_for_previous_kernel();  // before its waits for x are timed
    }
    for (int it = 0;; ++it) {
      const Item now = item(it);
      if (now.tile >= total) break;
      const int kb0 = now.kb0, kb1 = now.kb1;
      const BlkTile ti = blk_tile(now.tile, args.n_tiles_n, segs.n_seg, tile_m, tab);
      if (warp == 0) {
        // -------------------------------------------------------------- TMA producer
        for (int kb = kb0; kb < kb1 && ok; ++kb) {
          ok = wait_in_line(&empty[stage], ph ^ 1u, abort_flag, args.status, DMOE_DEVERR_TIMEOUT_PRODUCER);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (elect_one()) {
            if (ahead == 0) load_w(ti, kb, stage);
            tma_load_2d(smem + stage * tile_m * kBlk, &tm_x, &full[stage], kb * kBlk, ti.row0);
          }
          __syncwarp();
          if (ahead > 0) --ahead;
          armed |= 1u << stage;
          armed_ph = (armed_ph & ~(1u << stage)) | (ph << stage);
          if (++stage == stages) {
            stage = 0;
            ph ^= 1u;
          }
        }
      } else if (warp == 1) {
        // -------------------------------------------------------------- MMA issuer
        for (int kb = kb0; kb < kb1 && ok; ++kb) {
          ok = wait_in_line(&full[stage], ph, abort_flag, args.status, DMOE_DEVERR_TIMEOUT_MMA) &&
               wait_in_line(&acce[acc], acc_ph ^ 1u, abort_flag, args.status, DMOE_DEVERR_TIMEOUT_MMA);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t xd = xd0 + (uint64_t)(stage * (tile_m * kBlk >> 4));
            const uint64_t wd = wd0 + (uint64_t)(stage * (2 * kOpBytes >> 4));
#pragma unroll
            for (int k = 0; k < 4; ++k)  // 32 codes of K per MMA; the first starts a fresh sum
              umma_f16<DMOE_E4M3>(tmem_base + (uint32_t)(acc * kN), xd + 2 * k, wd + 2 * k, blk_idesc(128, kN), k != 0);
            umma_commit(&empty[stage]);
            umma_commit(&accf[acc]);
          }
          __syncwarp();
          if (++stage == stages) {
            stage = 0;
            ph ^= 1u;
          }
          acc ^= 1;
          if (acc == 0) acc_ph ^= 1u;
        }
      }
      if (SPLIT && now.parts) {
        __syncwarp();
        cluster_sync_all();
        cluster_sync_all();
      }
    }
    // The epilogue has waited for every step's MMAs, and those for every copy, unless some wait ran
    // out: then copies in flight land and MMAs complete before the CTA's shared memory and TMEM go.
    named_sync(7, kThreadsBlk);
    if (*abort_flag) {
      if (warp == 0 && lane == 0) {
        for (int s = 0; s < stages; ++s)
          if (armed >> s & 1u) wait_or_report(&full[s], armed_ph >> s & 1u, args.status);
      } else if (warp == 1) {
        if (elect_one()) {
          umma_commit(fin);
          wait_or_report(fin, 0, args.status);
        }
        __syncwarp();
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSplit.sums));
    if (early) wait_for_previous_kernel();
    const int q = warp & 3, half = (warp - 4) >> 2;
    uint4* st = reinterpret_cast<uint4*>(out_buf + (warp - 4) * 32 * 128);
    int acc = 0, flip = 0;
    uint32_t acc_ph = 0;
    bool ok = true;
    for (int it = 0;; ++it) {
      const Item now = item(it);
      if (now.tile >= total) break;
      const int kb0 = now.kb0, kb1 = now.kb1;
      const BlkTile ti = blk_tile(now.tile, args.n_tiles_n, segs.n_seg, tile_m, tab);
      const int rows = min(tile_m, ti.row_end - ti.row0);
      const bool reached = q * 32 < tile_m, active = q * 32 < rows;  // some row of this quadrant belongs to the tile
      const int row = ti.row0 + q * 32 + lane;
      const bool valid = q * 32 + lane < rows;
      StepScales sc;
      if (active) sc.start<GATED>(args, ti, row, valid, half, kb0);
      uint64_t sum[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) sum[i] = 0;
      for (int kb = kb0; kb < kb1 && ok && reached; ++kb) {
        float s0 = 0.f, s1 = 0.f;
        if (active) sc.take<GATED>(kb, kb1, s0, s1);
        const uint32_t at = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * kN);
        auto release = [&] {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acce[acc]);
        };
        ok = wait_in_line(&accf[acc], acc_ph, abort_flag, args.status, DMOE_DEVERR_TIMEOUT_EPILOGUE);
        if (__all_sync(0xffffffffu, ok && active && normal(s0) && (!GATED || normal(s1)))) {  // one vote, as above
          tc_fence_after();
          add_step<GATED, kCols>(sum, at, half, s0, s1, release);
        } else {
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (active) {
            tc_fence_after();
            add_step_any<GATED>(sum, at, half, sc.x + kb, sc.w0 + kb, sc.w1 + kb, release);
          } else if (lane == 0) {
            mbar_arrive(&acce[acc]);
          }
        }
        acc ^= 1;
        if (acc == 0) acc_ph ^= 1u;
      }
      // After a wait that ran out nothing is stored, but warps that meet below still do.
      if (!(SPLIT && now.parts)) {
        if (active) {
          if constexpr (GATED)
            store_codes(sum, args, row, ti.row0 + rows, ok, ti.nt, half, q, xch + flip * 256, st);
          else
            store_rows(sum, args, row, valid && ok, ti.nt, half, st);
        }
        flip ^= 1;
      } else {
        // Sums as [row][256 columns], 16-byte units exchanged within a row against bank conflicts.
        float4* red = reinterpret_cast<float4*>(smem);
        if (valid) {
#pragma unroll
          for (int v = 0; v < 32; ++v) {
            const float2 x = unpack_f2(sum[2 * v]), y = unpack_f2(sum[2 * v + 1]);
            const int unit = tmem_col<GATED>(half, v * 4) >> 2;
            red[(q * 32 + lane) * 64 + (unit ^ (lane & 7))] = make_float4(x.x, x.y, y.x, y.y);
          }
        }
        __syncwarp();
        cluster_sync_all();
        const uint32_t red0 = smem_u32(smem);
        auto total_of = [&](int r, int unit) {  // the ranks' sums of four columns, in order
          const uint32_t at = red0 + (uint32_t)((r * 64 + (unit ^ (r & 7))) * 16);
          float4 part[8];
#pragma unroll
          for (int g = 0; g < 8; ++g)
            part[g] = g < ranks ? ld_cluster(map_to_cta(at, (uint32_t)g)) : make_float4(0.f, 0.f, 0.f, 0.f);
          float4 v = part[0];
#pragma unroll
          for (int g = 1; g < 8; ++g) {
            v.x += part[g].x;
            v.y += part[g].y;
            v.z += part[g].z;
            v.w += part[g].w;
          }
          return v;
        };
        // Rank g finishes rows g, g + ranks, ... of the tile, a warp a row.
        for (int r = rank + ranks * (warp - 4); r < rows; r += ranks * kEpiWarps) {
          const int orow = ti.row0 + r;
          if constexpr (GATED) {
            const float4 g4 = total_of(r, lane), u4 = total_of(r, 32 + lane);
            float h[4] = {g4.x, g4.y, g4.z, g4.w};
            const float u[4] = {u4.x, u4.y, u4.z, u4.w};
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              h[i] = (args.act == DMOE_ACT_SILU ? blk_act<DMOE_ACT_SILU>(h[i]) : blk_act<DMOE_ACT_RELU>(h[i])) * u[i];
              top = fmaxf(top, finite_abs(h[i]));
              if (fabsf(h[i]) > kFinite) h[i] = __int_as_float(0x7fffffff);
            }
            // non-negative floats order as their bits
            const float s = block_scale(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top))));
            const int col = ti.nt * 128 + lane * 4;
            if (ok && col < args.n_out)
              *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(args.out) + (int64_t)orow * args.ldo + col) =
                  codes4(h, __frcp_rn(s));
            if (ok && lane == 0) args.out_scale[(int64_t)orow * args.os_ld + ti.nt] = s;
          } else {
            const bool f32 = args.out_dtype == DMOE_F32;
            const float4 y[2] = {total_of(r, lane), total_of(r, 32 + lane)};
            char* dst = blk_out_row(args, orow, f32 ? 4 : 2);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int col = ti.nt * kN + i * 128 + lane * 4;
              if (!ok || dst == nullptr || col >= args.n_out) continue;
              if (f32)
                *reinterpret_cast<float4*>(dst + (int64_t)col * 4) = y[i];
              else if (args.out_dtype == DMOE_BF16)
                *reinterpret_cast<uint2*>(dst + (int64_t)col * 2) =
                    make_uint2(pack2<DMOE_BF16>(y[i].x, y[i].y), pack2<DMOE_BF16>(y[i].z, y[i].w));
              else
                *reinterpret_cast<uint2*>(dst + (int64_t)col * 2) =
                    make_uint2(pack2<DMOE_F16>(y[i].x, y[i].y), pack2<DMOE_F16>(y[i].z, y[i].w));
            }
          }
        }
        // The next tile's copies write where the sums were read.
        asm volatile("fence.proxy.async;" ::: "memory");
        __syncwarp();
        cluster_sync_all();
      }
    }
    named_sync(7, kThreadsBlk);
  }
  if (args.scatter) __threadfence_system();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * kN);
  }
}

// ------------------------------------------------------------------------------------- host
// Row-major e4m3 tensor map, dims innermost first, rows ld bytes apart, 128-byte swizzle.
int code_map(CUtensorMap* map, const void* base, int rank, uint64_t cols, uint64_t rows, uint64_t stack, uint64_t ld,
             uint32_t box_rows) {
  PFN_encodeTiled enc = get_encode_fn();
  DMOE_REQUIRE(enc != nullptr, "cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[3] = {cols, rows, stack};
  const cuuint64_t strides[2] = {ld, ld * rows};
  const cuuint32_t box[3] = {(cuuint32_t)kBlk, box_rows, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, (cuuint32_t)rank, const_cast<void*>(base), dims, strides,
                         box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed (%d)", (int)r);
    return DMOE_ERR_CUDA;
  }
  return DMOE_OK;
}

// One product: x [m_rows, K] codes against the stack(s) [E, N, K].
struct Product {
  const void* x;
  int64_t x_ld;
  const void* w0;
  const void* w1;  // up weights of the gated form, else null
  int E, N, K;
  BlkArgs args;
};

template <bool GATED>
int n_tiles_of(int N) {
  return GATED ? (N + 127) / 128 : (N + kN - 1) / kN;
}

template <bool GATED>
int launch_pair(const Product& p, const BlkSegs& segs, int m_tiles, cudaStream_t stream) {
  static PerDeviceOnce once;
  static int max_clusters[64];
  int dev = 0;
  DMOE_CUDA(cudaGetDevice(&dev));
  DMOE_REQUIRE(dev >= 0 && dev < 64, "block-scaled product: device index %d out of range", dev);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.blockDim = dim3(kThreadsBlk);
  cfg.dynamicSmemBytes = kPSmemBytes;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const int r = once_per_device(once, dev, [&] {
    DMOE_CUDA(cudaFuncSetAttribute(blk_pair_kernel<GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPSmemBytes));
    cfg.gridDim = dim3(2 * 74);
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, blk_pair_kernel<GATED>, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = 64;
    }
    max_clusters[dev] = n;
    return DMOE_OK;
  });
  if (r) return r;
  CUtensorMap tx, t0, t1;
  if (int e = code_map(&tx, p.x, 2, p.K, segs.m_rows, 1, p.x_ld, 128)) return e;
  if (int e = code_map(&t0, p.w0, 3, p.K, p.N, p.E, p.K, 128)) return e;
  t1 = t0;
  if (GATED)
    if (int e = code_map(&t1, p.w1, 3, p.K, p.N, p.E, p.K, 128)) return e;
  BlkArgs a = p.args;
  a.n_tiles_n = n_tiles_of<GATED>(p.N);
  int pairs = max_clusters[dev] - (gemm_sm_reserve() + 1) / 2;
  const int64_t tiles = (int64_t)m_tiles * a.n_tiles_n;
  if (tiles < pairs) pairs = (int)tiles;
  if (pairs < 1) pairs = 1;
  cfg.gridDim = dim3(2 * pairs);
  DMOE_CUDA(cudaLaunchKernelEx(&cfg, blk_pair_kernel<GATED>, tx, t0, t1, segs, a));
  DMOE_LAUNCH_CHECK();
  return DMOE_OK;
}

// Clusters of `ranks` CTAs of the single-SM kernel that fit on the device at once.
template <bool GATED>
int max_split_clusters(int dev, int ranks, int* out) {
  static PerDeviceOnce once;
  static int fit[64][9];
  DMOE_REQUIRE(dev >= 0 && dev < 64, "block-scaled product: device index %d out of range", dev);
  const int r = once_per_device(once, dev, [&] {
    DMOE_CUDA(cudaFuncSetAttribute(blk_single_kernel<GATED, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    for (int n = 2; n <= 8; ++n) {
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = n;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.gridDim = dim3(n * 74);
      cfg.blockDim = dim3(kThreadsBlk);
      cfg.dynamicSmemBytes = kSingleFixed + single_stages(32) * single_stage_bytes(32);
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int got = 0;
      if (cudaOccupancyMaxActiveClusters(&got, blk_single_kernel<GATED, true>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        got = 0;
      }
      fit[dev][n] = got;
    }
    return DMOE_OK;
  });
  *out = r == DMOE_OK ? fit[dev][ranks] : 0;
  return r;
}

template <bool GATED, bool SPLIT>
int launch_single(const Product& p, const BlkSegs& segs, int tile_m, int m_tiles, int ranks, cudaStream_t stream) {
  static PerDeviceOnce once;
  int dev = 0;
  DMOE_CUDA(cudaGetDevice(&dev));
  const int r = once_per_device(once, dev, [] {
    DMOE_CUDA(cudaFuncSetAttribute(blk_single_kernel<GATED, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    return DMOE_OK;
  });
  if (r) return r;
  CUtensorMap tx, t0, t1;
  if (int e = code_map(&tx, p.x, 2, p.K, segs.m_rows, 1, p.x_ld, tile_m)) return e;
  if (int e = code_map(&t0, p.w0, 3, p.K, p.N, p.E, p.K, GATED ? 128 : kN)) return e;
  t1 = t0;
  if (GATED)
    if (int e = code_map(&t1, p.w1, 3, p.K, p.N, p.E, p.K, 128)) return e;
  BlkArgs a = p.args;
  a.n_tiles_n = n_tiles_of<GATED>(p.N);
  const int64_t tiles = (int64_t)m_tiles * a.n_tiles_n;
  int groups = gemm_usable_sms() / ranks;
  if (tiles < groups) groups = (int)tiles;
  if (groups < 1) groups = 1;
  const int stages = single_stages(tile_m);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ranks;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3(groups * ranks);
  cfg.blockDim = dim3(kThreadsBlk);
  cfg.dynamicSmemBytes = kSingleFixed + stages * single_stage_bytes(tile_m);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = SPLIT ? 2 : 1;
  DMOE_CUDA(cudaLaunchKernelEx(&cfg, blk_single_kernel<GATED, SPLIT>, tx, t0, t1, segs, a, tile_m, stages, ranks));
  DMOE_LAUNCH_CHECK();
  return DMOE_OK;
}

// Rows of x that a segment is expected to have: what the caller says, else the mean over the
// segments that can have any.
int expected_rows(const BlkSegs& segs, int hint) {
  if (hint > 0) return hint < segs.m_rows ? hint : segs.m_rows;
  const int used = segs.n_seg < segs.m_rows ? segs.n_seg : segs.m_rows;
  return used > 0 ? (segs.m_rows + used - 1) / used : 0;
}

// Row tiles of `tile_m` rows: counted for a host table, for a device table the most that
// m_rows rows in n_seg segments can make.
int row_tiles(const BlkSegs& segs, int tile_m) {
  if (segs.dev_end == nullptr) {
    int prev = 0, n = 0;
    for (int i = 0; i < segs.n_seg; ++i) {
      n += (segs.end[i] - prev + tile_m - 1) / tile_m;
      prev = segs.end[i];
    }
    return n;
  }
  const int64_t most = (int64_t)segs.m_rows / tile_m + segs.n_seg;
  return (int)(most < segs.m_rows ? most : segs.m_rows);
}

template <bool GATED>
int run_product(Product& p, const BlkSegs& segs, int hint, cudaStream_t stream) {
  p.args.n_out = p.N;
  p.args.K = p.K;
  p.args.n_blk = (p.N + kBlk - 1) / kBlk;
  p.args.k_blk = (p.K + kBlk - 1) / kBlk;
  const int rows = expected_rows(segs, hint);
  const int n_tiles = n_tiles_of<GATED>(p.N);
  const int used = segs.n_seg < segs.m_rows ? segs.n_seg : segs.m_rows;
  // Row tiles of the single-SM kernel: room for segments half again as long as expected, since a
  // segment that needs a second tile reads its weights twice.
  const int tile_m = rows <= 20 ? 32 : rows <= 40 ? 64 : 128;
  const int m_tiles = row_tiles(segs, tile_m);
  if (m_tiles == 0) return DMOE_OK;  // a host table without rows
  const int64_t likely = (int64_t)(segs.dev_end ? used * ((rows + tile_m - 1) / tile_m) : m_tiles) * n_tiles;
  const int sms = gemm_usable_sms();
  if (likely * 2 <= sms) {
    // Few tiles: split the reduction over as many SMs of a cluster as leave all clusters room at
    // once, at least two steps each.
    int dev = 0, ranks = (int)(sms / likely);
    DMOE_CUDA(cudaGetDevice(&dev));
    if (ranks > 8) ranks = 8;
    if (ranks > p.args.k_blk / 2) ranks = p.args.k_blk / 2;
    for (; ranks > 1; --ranks) {
      int fit = 0;
      if (int r = max_split_clusters<GATED>(dev, ranks, &fit)) return r;
      if (fit >= likely) return launch_single<GATED, true>(p, segs, tile_m, m_tiles, ranks, stream);
    }
  }
  // Rows that the tiles of each kernel cover, the padding of each segment's last tile included (half
  // a tile on average where the table is not at hand).  A pair does a row in about 0.93 of the time
  // of a single SM twice: 4096 x 14336 x 4096 in 223 us against 238, 8192 x 8192 x 8192 in 549
  // against 611; on ragged segments the finer tiles win (32 of 256 rows on average at 2048 x 7168: 172 us
  // against 184).
  const int64_t by_pair = segs.dev_end ? (int64_t)(rows + kPM / 2) * used : (int64_t)row_tiles(segs, kPM) * kPM;
  const int64_t by_single = segs.dev_end ? (int64_t)(rows + 64) * used : (int64_t)row_tiles(segs, 128) * 128;
  if (tile_m == 128 && by_pair * 93 < by_single * 100) return launch_pair<GATED>(p, segs, row_tiles(segs, kPM), stream);
  // Long reductions: the tiles of a last, partly empty wave are split over two SMs each.  The kernel's rule
  // lets 128-row tiles go to two from 44 blocks of K on (k_blk / 2 + 24 <= k_blk + 2); below, the cluster
  // launch alone is left (1002 rows over 8 experts, N = 4096, whole -> split: 32 blocks 41.0 -> 41.7 us, 40
  // 49.3 -> 49.9, 44 53.9 -> 51.5, 48 57.6 -> 53.8, 56 65.9 -> 60.9; 8192 rows over 32, N = 2048: 32 103.4 ->
  // 104.6, 48 164.6 -> 156.7, 56 174.1 -> 169.3; 500 rows over 8, whose last wave is too full for it: 32
  // 28.6 -> 29.0, 56 46.3 -> 46.6).
  if (p.args.k_blk >= 48) return launch_single<GATED, true>(p, segs, tile_m, m_tiles, 2, stream);
  return launch_single<GATED, false>(p, segs, tile_m, m_tiles, 1, stream);
}

int fill_blk_segs(const char* name, BlkSegs& s, const int32_t* seg_expert, const int32_t* seg_end, int n_seg,
                  int seg_on_device, int m_rows, int E_stack) {
  s.n_seg = n_seg;
  s.m_rows = m_rows;
  s.e_stack = E_stack;
  if (seg_on_device) {
    DMOE_REQUIRE(n_seg <= kMaxSegs, "%s: n_seg=%d > %d", name, n_seg, kMaxSegs);
    s.dev_expert = seg_expert;
    s.dev_end = seg_end;
    return DMOE_OK;
  }
  DMOE_REQUIRE(n_seg <= kMaxHostSegs, "%s: n_seg=%d > %d for host segment tables", name, n_seg, kMaxHostSegs);
  s.dev_expert = s.dev_end = nullptr;
  int prev = 0;
  for (int i = 0; i < n_seg; ++i) {
    DMOE_REQUIRE(seg_end[i] >= prev && seg_end[i] <= m_rows, "%s: segment %d end %d invalid", name, i, seg_end[i]);
    DMOE_REQUIRE(seg_expert[i] >= 0 && seg_expert[i] < E_stack, "%s: segment %d expert %d", name, i, seg_expert[i]);
    s.expert[i] = seg_expert[i];
    s.end[i] = seg_end[i];
    prev = seg_end[i];
  }
  return DMOE_OK;
}

// Row and tile numbers are 32-bit: rows leave room for a tile past the last one, tiles for a step of
// the grid.
constexpr int64_t kMostRows = INT32_MAX - 1024;
bool too_many_tiles(int64_t rows, int64_t n_seg, int64_t N) {
  return (rows / 32 + n_seg) * ((N + 127) / 128) > INT32_MAX - 1024;
}

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

int64_t blocks_of(int64_t n) { return (n + kBlk - 1) / kBlk; }

// Gate/up product into codes and scales of h in the workspace, then the down product.
int run_blk_mlp(const void* x, int64_t x_ld, const float* xs, int64_t xs_ld, const void* wg, const float* gs,
                const void* wu, const float* us, const void* wd, const float* ds, int E, int d, int I,
                const BlkSegs& segs, int hint, int act, void* Y, const int32_t* scatter_map, char* const* scatter_base,
                void* workspace, int32_t* status, cudaStream_t stream) {
  uint8_t* h = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
  float* hs = reinterpret_cast<float*>(h + (((int64_t)segs.m_rows * I + 255) & ~int64_t(255)));
  Product g{x, x_ld, wg, wu, E, I, d, {}};
  g.args.xs = xs;
  g.args.xs_ld = xs_ld;
  g.args.ws0 = gs;
  g.args.ws1 = us;
  g.args.act = act;
  g.args.out = h;
  g.args.ldo = I;
  g.args.out_dtype = DMOE_E4M3;
  g.args.out_scale = hs;
  g.args.os_ld = blocks_of(I);
  g.args.status = status;
  if (int r = run_product<true>(g, segs, hint, stream)) return r;
  Product dn{h, I, wd, nullptr, E, d, I, {}};
  dn.args.xs = hs;
  dn.args.xs_ld = blocks_of(I);
  dn.args.ws0 = ds;
  dn.args.out = Y;
  dn.args.early = 1;
  dn.args.ldo = d;
  dn.args.out_dtype = DMOE_BF16;
  dn.args.status = status;
  if (scatter_map != nullptr) {
    dn.args.scatter = 1;
    dn.args.scatter_map = scatter_map;
    for (int g2 = 0; g2 < DMOE_EP_MAX_RANKS; ++g2) dn.args.scatter_base[g2] = scatter_base[g2];
  }
  return run_product<false>(dn, segs, hint, stream);
}

}  // namespace
}  // namespace dmoe

using namespace dmoe;

extern "C" int dmoe_grouped_matmul_fp8_blocks(const void* Xq, int64_t x_ld, const float* x_scale, int64_t xs_ld,
                                              const void* w_q, const float* w_scale, int E_stack, int N, int K,
                                              const int32_t* seg_expert, const int32_t* seg_end, int n_seg,
                                              int seg_on_device, int m_rows, int rows_hint, void* Y, int64_t y_ld,
                                              int out_dtype, int32_t* dev_status, void* stream) {
  clear_error();
  const char* name = "dmoe_grouped_matmul_fp8_blocks";
  DMOE_REQUIRE(dtype_ok(out_dtype), "%s: output dtype must be f32, f16 or bf16", name);
  DMOE_REQUIRE(N > 0 && K > 0 && N % 8 == 0 && K % 16 == 0, "%s: N=%d must be a multiple of 8, K=%d of 16", name, N, K);
  DMOE_REQUIRE(E_stack >= 1 && m_rows >= 0 && n_seg >= 0 && rows_hint >= 0, "%s: bad E_stack/m_rows/n_seg/rows_hint",
               name);
  DMOE_REQUIRE(x_ld >= K && x_ld % 16 == 0 && xs_ld >= blocks_of(K), "%s: x_ld=%lld, xs_ld=%lld too small or odd", name,
               (long long)x_ld, (long long)xs_ld);
  DMOE_REQUIRE(y_ld >= N && y_ld % 8 == 0, "%s: y_ld=%lld must be >= N and a multiple of 8", name, (long long)y_ld);
  if (n_seg == 0 || m_rows == 0) return DMOE_OK;
  DMOE_REQUIRE(Xq && x_scale && w_q && w_scale && Y && dev_status && seg_expert && seg_end, "%s: null pointer", name);
  DMOE_REQUIRE(aligned16(Xq) && aligned16(w_q) && aligned16(Y), "%s: tensors must be 16-byte aligned", name);
  DMOE_REQUIRE(aligned4(x_scale) && aligned4(w_scale), "%s: scales must be 4-byte aligned", name);
  DMOE_REQUIRE(m_rows <= kMostRows && !too_many_tiles(m_rows, n_seg, N), "%s: too many rows or tiles", name);
  static thread_local BlkSegs segs;
  if (int r = fill_blk_segs(name, segs, seg_expert, seg_end, n_seg, seg_on_device, m_rows, E_stack)) return r;
  Product p{Xq, x_ld, w_q, nullptr, E_stack, N, K, {}};
  p.args.xs = x_scale;
  p.args.xs_ld = xs_ld;
  p.args.ws0 = w_scale;
  p.args.out = Y;
  p.args.ldo = y_ld;
  p.args.out_dtype = out_dtype;
  p.args.status = dev_status;
  return run_product<false>(p, segs, rows_hint, as_stream(stream));
}

extern "C" size_t dmoe_grouped_mlp_fp8_blocks_workspace_size(int m_rows, int I) {
  if (m_rows < 0 || I < 0) return 0;
  return (size_t)m_rows * (size_t)I + (size_t)m_rows * (size_t)blocks_of(I) * 4 + 1024;
}

namespace dmoe {
namespace {
int check_blk_mlp(const char* name, const void* x, const void* wg, const float* gs, const void* wu, const float* us,
                  const void* wd, const float* ds, int d, int I, int n_seg, const int32_t* seg_expert,
                  const int32_t* seg_end, int64_t m_rows, const void* workspace, size_t workspace_bytes,
                  const int32_t* dev_status) {
  DMOE_REQUIRE(x && wg && gs && wu && us && wd && ds && workspace && dev_status && seg_expert && seg_end,
               "%s: null pointer", name);
  DMOE_REQUIRE(aligned16(x) && aligned16(wg) && aligned16(wu) && aligned16(wd) && aligned16(workspace),
               "%s: tensors must be 16-byte aligned", name);
  DMOE_REQUIRE(aligned4(gs) && aligned4(us) && aligned4(ds), "%s: scales must be 4-byte aligned", name);
  DMOE_REQUIRE(workspace_bytes >= dmoe_grouped_mlp_fp8_blocks_workspace_size((int)m_rows, I), "%s: workspace %zu < %zu bytes",
               name, workspace_bytes, dmoe_grouped_mlp_fp8_blocks_workspace_size((int)m_rows, I));
  DMOE_REQUIRE(m_rows <= kMostRows && !too_many_tiles(m_rows, n_seg, d > I ? d : I), "%s: too many rows or tiles", name);
  return DMOE_OK;
}
}  // namespace
}  // namespace dmoe

extern "C" int dmoe_grouped_gated_mlp_fp8_blocks(const void* Xq, int64_t x_ld, const float* x_scale, int64_t xs_ld,
                                                 const void* wg_q, const float* wg_scale, const void* wu_q,
                                                 const float* wu_scale, const void* wd_q, const float* wd_scale,
                                                 int E_stack, int d, int I, const int32_t* seg_expert,
                                                 const int32_t* seg_end, int n_seg, int seg_on_device, int m_rows,
                                                 int rows_hint, int act, void* Y, void* workspace,
                                                 size_t workspace_bytes, int32_t* dev_status, void* stream) {
  clear_error();
  const char* name = "dmoe_grouped_gated_mlp_fp8_blocks";
  DMOE_REQUIRE(act == DMOE_ACT_RELU || act == DMOE_ACT_SILU, "%s: bad activation %d", name, act);
  DMOE_REQUIRE(d > 0 && I > 0 && d % 16 == 0 && I % 16 == 0, "%s: d=%d and I=%d must be multiples of 16", name, d, I);
  DMOE_REQUIRE(E_stack >= 1 && m_rows >= 0 && n_seg >= 0 && rows_hint >= 0, "%s: bad E_stack/m_rows/n_seg/rows_hint",
               name);
  DMOE_REQUIRE(x_ld >= d && x_ld % 16 == 0 && xs_ld >= blocks_of(d), "%s: x_ld=%lld, xs_ld=%lld too small or odd", name,
               (long long)x_ld, (long long)xs_ld);
  if (n_seg == 0 || m_rows == 0) return DMOE_OK;
  DMOE_REQUIRE(x_scale && Y, "%s: null pointer", name);
  DMOE_REQUIRE(aligned4(x_scale) && aligned16(Y), "%s: misaligned scales or output", name);
  if (int r = check_blk_mlp(name, Xq, wg_q, wg_scale, wu_q, wu_scale, wd_q, wd_scale, d, I, n_seg, seg_expert, seg_end,
                            m_rows, workspace, workspace_bytes, dev_status))
    return r;
  static thread_local BlkSegs segs;
  if (int r = fill_blk_segs(name, segs, seg_expert, seg_end, n_seg, seg_on_device, m_rows, E_stack)) return r;
  return run_blk_mlp(Xq, x_ld, x_scale, xs_ld, wg_q, wg_scale, wu_q, wu_scale, wd_q, wd_scale, E_stack, d, I, segs,
                     rows_hint, act, Y, nullptr, nullptr, workspace, dev_status, as_stream(stream));
}

extern "C" int dmoe_ep_expert_mlp_fp8_blocks(const dmoe_ep_window* win, const void* wg_q, const float* wg_scale,
                                             const void* wu_q, const float* wu_scale, const void* wd_q,
                                             const float* wd_scale, int E_stack, int d, int I,
                                             const int32_t* seg_expert, const int32_t* seg_end, int n_seg, int64_t cap,
                                             int rows_hint, int act, void* workspace, size_t workspace_bytes,
                                             int32_t* dev_status, void* stream) {
  clear_error();
  const char* name = "dmoe_ep_expert_mlp_fp8_blocks";
  DMOE_REQUIRE(win != nullptr && win->world >= 1 && win->world <= DMOE_EP_MAX_RANKS && win->rank >= 0 &&
                   win->rank < win->world,
               "%s: bad window table", name);
  DMOE_REQUIRE(act == DMOE_ACT_RELU || act == DMOE_ACT_SILU, "%s: bad activation %d", name, act);
  DMOE_REQUIRE(d > 0 && I > 0 && d % 16 == 0 && I % 16 == 0, "%s: d=%d and I=%d must be multiples of 16", name, d, I);
  DMOE_REQUIRE(E_stack >= 1 && n_seg >= 0 && n_seg <= kMaxSegs && rows_hint >= 0, "%s: bad E_stack/n_seg/rows_hint", name);
  DMOE_REQUIRE(cap >= 0 && cap < (1ll << 31), "%s: bad capacity", name);
  if (n_seg == 0 || cap == 0) return DMOE_OK;
  const char* X = reinterpret_cast<const char*>(win->recv[win->rank]);
  DMOE_REQUIRE(win->back[win->rank] != nullptr, "%s: null pointer", name);
  if (int r = check_blk_mlp(name, X, wg_q, wg_scale, wu_q, wu_scale, wd_q, wd_scale, d, I, n_seg, seg_expert, seg_end,
                            cap, workspace, workspace_bytes, dev_status))
    return r;
  char* base[DMOE_EP_MAX_RANKS] = {};
  for (int g = 0; g < win->world; ++g) {
    DMOE_REQUIRE(win->rows[g] != nullptr && aligned16(win->rows[g]), "%s: rank %d has no return rows", name, g);
    base[g] = reinterpret_cast<char*>(win->rows[g]);
  }
  static thread_local BlkSegs segs;
  if (int r = fill_blk_segs(name, segs, seg_expert, seg_end, n_seg, 1, (int)cap, E_stack)) return r;
  const int64_t rec = d + ((blocks_of(d) * 4 + 15) & ~int64_t(15));
  return run_blk_mlp(X, rec, reinterpret_cast<const float*>(X + d), rec / 4, wg_q, wg_scale, wu_q, wu_scale, wd_q,
                     wd_scale, E_stack, d, I, segs, rows_hint, act, nullptr,
                     reinterpret_cast<const int32_t*>(win->back[win->rank]), base, workspace, dev_status,
                     as_stream(stream));
}

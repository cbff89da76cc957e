// Row-wise e4m3 quantisation for the 8-bit expert GEMM.
//
// Each row r of x [rows, cols] (f16/bf16/f32) becomes q[r, :] = rn_satfinite(x[r, :] / s[r]) in
// e4m3 with s[r] = amax(|x[r, :]|) / 448 (448 = the largest finite e4m3), s[r] = 1 for an
// all-zero row.  q's rows are q_ld bytes apart and the scales scale_ld floats apart, so a row
// and its scale can share one record (d codes, then the scale: the receive rows of an 8-bit
// exchange window).  Rows of activations give per-token scales; rows of an expert's gate or
// up weight [E, I, d] viewed as [E * I, d] give per-output-channel scales.  The reference's
// benchmark casts the whole layer to an 8-bit float with no scale (precision "fp8",
// src/python/MoE/benchmarks/bench.py:184-185); per-row scales keep the 8-bit storage and the
// 8-bit tensor-core kind while the products stay within a few percent of 16-bit ones.
//
// One warp per row, 16-byte loads: the first pass finds amax, the second (an L1/L2 hit)
// converts.  HBM-bound: (input bytes + 1) per element.

#include <cuda_fp8.h>

#include "dmoe_common.cuh"

namespace dmoe {
namespace {

constexpr int kQuantWarps = 8;

template <int DT>
__device__ __forceinline__ void load8(const void* base, int64_t i, float* f) {
  if constexpr (DT == DMOE_F32) {
    const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + i);
    const float4 a = __ldg(p), b = __ldg(p + 1);
    f[0] = a.x;
    f[1] = a.y;
    f[2] = a.z;
    f[3] = a.w;
    f[4] = b.x;
    f[5] = b.y;
    f[6] = b.z;
    f[7] = b.w;
  } else {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(base) + i * 2));
    unpack8<DT>(v, f);
  }
}

template <int DT>
__global__ void __launch_bounds__(kQuantWarps * 32)
    quantize_rows_e4m3_kernel(const void* __restrict__ x, int64_t rows, int cols, uint8_t* __restrict__ q,
                              int64_t q_ld, float* __restrict__ scale, int64_t scale_ld) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * kQuantWarps + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int64_t base = row * cols;
  float amax = 0.f;
  for (int c = lane * 8; c < cols; c += 256) {
    float f[8];
    load8<DT>(x, base + c, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(f[i]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  // fmaxf prefers a number to NaN: a row of NaN gets scale 1 and NaN codes.
  const float s = amax > 0.f ? amax / 448.f : 1.f;
  if (lane == 0) scale[row * scale_ld] = s;
  for (int c = lane * 8; c < cols; c += 256) {
    float f[8];
    load8<DT>(x, base + c, f);
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(
          make_float2(__fdiv_rn(f[4 * h], s), __fdiv_rn(f[4 * h + 1], s)), __NV_SATFINITE, __NV_E4M3);
      const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(
          make_float2(__fdiv_rn(f[4 * h + 2], s), __fdiv_rn(f[4 * h + 3], s)), __NV_SATFINITE, __NV_E4M3);
      w[h] = (uint32_t)lo | ((uint32_t)hi << 16);
    }
    *reinterpret_cast<uint2*>(q + row * q_ld + c) = make_uint2(w[0], w[1]);
  }
}

}  // namespace
}  // namespace dmoe

using namespace dmoe;

extern "C" int dmoe_quantize_rows_e4m3(const void* x, int dtype, int64_t rows, int cols, void* q, int64_t q_ld,
                                       float* scale, int64_t scale_ld, void* stream) {
  clear_error();
  DMOE_REQUIRE(dtype_ok(dtype), "dmoe_quantize_rows_e4m3: dtype must be f32, f16 or bf16");
  DMOE_REQUIRE(rows >= 0 && cols > 0 && cols % 16 == 0, "dmoe_quantize_rows_e4m3: cols=%d must be a multiple of 16",
               cols);
  if (rows == 0) return DMOE_OK;
  DMOE_REQUIRE(x && q && scale, "dmoe_quantize_rows_e4m3: null pointer");
  DMOE_REQUIRE(aligned16(x) && aligned16(q), "dmoe_quantize_rows_e4m3: x and q must be 16-byte aligned");
  DMOE_REQUIRE(q_ld >= cols && q_ld % 16 == 0 && scale_ld >= 1,
               "dmoe_quantize_rows_e4m3: q_ld=%lld must be >= cols and a multiple of 16, scale_ld=%lld >= 1",
               (long long)q_ld, (long long)scale_ld);
  DMOE_REQUIRE((reinterpret_cast<uintptr_t>(scale) & 3u) == 0, "dmoe_quantize_rows_e4m3: scale must be 4-byte aligned");
  DMOE_REQUIRE(rows <= (int64_t)INT32_MAX * kQuantWarps, "dmoe_quantize_rows_e4m3: %lld rows", (long long)rows);
  const unsigned grid = (unsigned)((rows + kQuantWarps - 1) / kQuantWarps);
  cudaStream_t s = as_stream(stream);
  uint8_t* qb = reinterpret_cast<uint8_t*>(q);
  if (dtype == DMOE_BF16)
    quantize_rows_e4m3_kernel<DMOE_BF16><<<grid, kQuantWarps * 32, 0, s>>>(x, rows, cols, qb, q_ld, scale, scale_ld);
  else if (dtype == DMOE_F16)
    quantize_rows_e4m3_kernel<DMOE_F16><<<grid, kQuantWarps * 32, 0, s>>>(x, rows, cols, qb, q_ld, scale, scale_ld);
  else
    quantize_rows_e4m3_kernel<DMOE_F32><<<grid, kQuantWarps * 32, 0, s>>>(x, rows, cols, qb, q_ld, scale, scale_ld);
  DMOE_LAUNCH_CHECK();
  return DMOE_OK;
}

// ------------------------------------------------------------------------ blocks of 128 columns
// Scales for blocks of 1 x 128 (activations) or 128 x 128 (weights): s = max(amax / 448, 2^-126),
// 1 for an all-zero block, q = e4m3(x / s) with the quotient rounded to fp32 first, as above.  The
// lower bound keeps the scale a normal number (a subnormal one could not be divided by).  A value
// that is not finite becomes a NaN code and leaves its block's scale alone.
//
// Each thread holds the eight neighbouring values of one 16-byte load (two for fp32); 16 lanes make
// a row of 128, so the row's amax is four shuffles and x is read once.
namespace dmoe {
namespace {

constexpr float kFiniteMax = 3.402823466e38f;

__device__ __forceinline__ float finite_max8(const float* f) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(f[i]) <= kFiniteMax ? fabsf(f[i]) : 0.f);
  return m;
}

__device__ __forceinline__ float scale_of(float amax) {
  return amax > 0.f ? fmaxf(__fdiv_rn(amax, 448.f), 1.17549435e-38f) : 1.f;
}

// Codes of eight values by a block's scale and its rounded reciprocal.  x / s as a product with the
// reciprocal and one correction by the residual, which the fused steps compute exactly (Markstein,
// 1990): the value before the last rounding is within 1.5 x 2^-24 ulp of the quotient, so it rounds
// as the quotient does unless that lies so near the middle between two fp32 numbers.  `fast` must be
// false for scales below 2^-90, where the residual could be subnormal, and where infinities have
// to become NaN codes (the conversion saturates them); those take the division.
__device__ __forceinline__ uint2 codes8(const float* f, float s, float inv, bool fast) {
  float v[8];
  if (fast) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float r = __fmul_rn(f[i], inv);
      v[i] = __fmaf_rn(__fmaf_rn(-r, s, f[i]), inv, r);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = fabsf(f[i]) <= kFiniteMax ? __fdiv_rn(f[i], s) : __int_as_float(0x7fffffff);
  }
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * h], v[4 * h + 1]), __NV_SATFINITE, __NV_E4M3);
    const __nv_fp8x2_storage_t hi =
        __nv_cvt_float2_to_fp8x2(make_float2(v[4 * h + 2], v[4 * h + 3]), __NV_SATFINITE, __NV_E4M3);
    w[h] = (uint32_t)lo | ((uint32_t)hi << 16);
  }
  return make_uint2(w[0], w[1]);
}
constexpr float kFastScale = 8.0779357e-28f;  // 2^-90

// Eight neighbouring values as they lie in memory (a 16-bit value widened early would take twice the
// registers), their largest magnitude and the values as numbers.
template <int DT>
struct Raw8 {
  static constexpr int kVecs = DT == DMOE_F32 ? 2 : 1;
  // Magnitudes order as their bits; from this one on they are not finite.
  static constexpr uint32_t kInf = DT == DMOE_F32 ? 0x7f800000u : (DT == DMOE_BF16 ? 0x7f80u : 0x7c00u);
  uint4 v[kVecs];
  __device__ __forceinline__ void load(const void* base, int64_t i) {
    const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(base) + i * (DT == DMOE_F32 ? 4 : 2));
#pragma unroll
    for (int j = 0; j < kVecs; ++j) v[j] = __ldcs(p + j);  // read once
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < kVecs; ++j) v[j] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void numbers(float* f) const {
    if constexpr (DT == DMOE_F32) {
      const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(w[j]);
    } else {
      unpack8<DT>(v[0], f);
    }
  }
  __device__ __forceinline__ uint32_t top() const {
    if constexpr (DT == DMOE_F32) {
      const uint32_t m = 0x7fffffffu;
      const uint4 a = v[0], b = v[1];
      return max(max(max(a.x & m, a.y & m), max(a.z & m, a.w & m)), max(max(b.x & m, b.y & m), max(b.z & m, b.w & m)));
    } else {
      const uint32_t m = 0x7fff7fffu;
      const uint32_t t = __vmaxu2(__vmaxu2(v[0].x & m, v[0].y & m), __vmaxu2(v[0].z & m, v[0].w & m));
      return max(t & 0xffffu, t >> 16);
    }
  }
  static __device__ __forceinline__ float value(uint32_t bits) {
    if constexpr (DT == DMOE_F32) return __uint_as_float(bits);
    if constexpr (DT == DMOE_BF16) return __uint_as_float(bits << 16);
    return __half2float(__ushort_as_half((unsigned short)bits));
  }
};

// 1 x 128: a warp takes kRowLoads x 256 consecutive columns of one row, two blocks per load, with all
// its loads in flight at once.  A scale costs two divisions, some 35 instructions: lane i of each
// half-warp does those of load i and hands them round, rather than all lanes for every load (8192 x
// 7168 bf16: 34 us, 5.2 TB/s, against 44, with 76 % of the issue slots taken and DRAM at 46 %: instructions
// bound it; f32 46 us, 6.4 TB/s, HBM's rate).
template <int DT>
constexpr int kRowLoads = DT == DMOE_F32 ? 4 : 8;
constexpr int kRowWarps = 4, kRowCtas = 8;  // warps of a CTA, CTAs an SM: 32 warps at 64 registers (24 at 72: 36 us)

template <int DT>
__global__ void __launch_bounds__(kRowWarps * 32, kRowCtas)
    quantize_row_blocks_kernel(const void* __restrict__ x, int64_t rows, int cols, uint8_t* __restrict__ q,
                               int64_t q_ld, float* __restrict__ scale, int64_t scale_ld) {
  // The product that follows may set itself up meanwhile; it waits for this kernel's end.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int NL = kRowLoads<DT>;
  const int lane = threadIdx.x & 31, at = lane & 15;
  const int64_t row = (int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int c0 = blockIdx.y * (NL * 256) + lane * 8;
  Raw8<DT> raw[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    if (c0 + i * 256 < cols)
      raw[i].load(x, row * cols + c0 + i * 256);
    else
      raw[i].clear();
  }
  uint32_t bits = 0;  // of the block whose scale this lane makes
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    uint32_t t = raw[i].top();
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) t = max(t, __shfl_xor_sync(0xffffffffu, t, o));
    if (at == i) bits = t;
  }
  const bool finite = bits < Raw8<DT>::kInf;
  float m = Raw8<DT>::value(bits);
  if (!__all_sync(0xffffffffu, finite)) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      float f[8];
      raw[i].numbers(f);
      float t = finite_max8(f);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
      if (at == i) m = t;
    }
  }
  const float s = scale_of(m), inv = __frcp_rn(s);
  const uint32_t fast = __ballot_sync(0xffffffffu, finite && s >= kFastScale);
  const int block = blockIdx.y * (NL * 2) + at * 2 + (lane >> 4);
  if (at < NL && block * 128 < cols) scale[row * scale_ld + block] = s;
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int from = (lane & 16) | i;
    const float si = __shfl_sync(0xffffffffu, s, from), ri = __shfl_sync(0xffffffffu, inv, from);
    const int c = c0 + i * 256;
    if (c < cols) {
      float f[8];
      raw[i].numbers(f);
      *reinterpret_cast<uint2*>(q + row * q_ld + c) = codes8(f, si, ri, fast >> from & 1u);
    }
  }
}

// 128 x 128: a CTA takes one block of one matrix of the batch, 64 values a thread, all loads in
// flight at once (14336 x 4096 f32: 47 us, 6.3 TB/s, HBM's rate; bf16 and f16 34 us, 5.2 TB/s).
template <int DT>
__global__ void __launch_bounds__(256)
    quantize_square_blocks_kernel(const void* __restrict__ x, int64_t rows, int cols, int col_blocks,
                                  int64_t row_blocks, uint8_t* __restrict__ q, float* __restrict__ scale) {
  __shared__ uint32_t tops[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t rb_all = blockIdx.x / col_blocks;  // row block within the whole batch
  const int cb = (int)(blockIdx.x - rb_all * col_blocks);
  const int64_t mat = rb_all / row_blocks;
  const int64_t r0 = (rb_all - mat * row_blocks) * 128 + warp * 2 + (lane >> 4);
  const int c = cb * 128 + (lane & 15) * 8;
  const int64_t base = mat * rows * cols;
  Raw8<DT> raw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = r0 + i * 16;
    if (r < rows && c < cols)
      raw[i].load(x, base + r * cols + c);
    else
      raw[i].clear();
  }
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) bits = max(bits, raw[i].top());
  bits = __reduce_max_sync(0xffffffffu, bits);
  if (lane == 0) tops[warp] = bits;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) bits = max(bits, tops[w]);
  const bool finite = bits < Raw8<DT>::kInf;  // of the whole block
  float m = Raw8<DT>::value(bits);
  if (!finite) {
    m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float f[8];
      raw[i].numbers(f);
      m = fmaxf(m, finite_max8(f));
    }
    bits = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
    __syncthreads();
    if (lane == 0) tops[warp] = bits;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) bits = max(bits, tops[w]);
    m = __uint_as_float(bits);
  }
  const float s = scale_of(m), inv = __frcp_rn(s);
  const bool fast = finite && s >= kFastScale;
  if (threadIdx.x == 0) scale[rb_all * col_blocks + cb] = s;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = r0 + i * 16;
    if (r < rows && c < cols) {
      float f[8];
      raw[i].numbers(f);
      *reinterpret_cast<uint2*>(q + base + r * cols + c) = codes8(f, s, inv, fast);
    }
  }
}

template <int DT>
int run_quantize_blocks(const void* x, int64_t batch, int64_t rows, int cols, int block_rows, uint8_t* q, int64_t q_ld,
                        float* scale, int64_t scale_ld, cudaStream_t s) {
  if (block_rows == 1) {
    const int parts = (cols + kRowLoads<DT> * 256 - 1) / (kRowLoads<DT> * 256);
    const int64_t grid = (batch * rows + kRowWarps - 1) / kRowWarps;
    DMOE_REQUIRE(grid <= INT32_MAX, "dmoe_quantize_blocks_e4m3: %lld rows", (long long)(batch * rows));
    DMOE_REQUIRE(parts <= 65535, "dmoe_quantize_blocks_e4m3: cols=%d, at most 2^26 - 1024 f32 columns", cols);  // grid.y
    quantize_row_blocks_kernel<DT><<<dim3((unsigned)grid, parts), kRowWarps * 32, 0, s>>>(x, batch * rows, cols, q,
                                                                                            q_ld, scale, scale_ld);
  } else {
    const int64_t row_blocks = (rows + 127) / 128;
    const int col_blocks = (cols + 127) / 128;
    const int64_t grid = batch * row_blocks * col_blocks;
    DMOE_REQUIRE(grid <= INT32_MAX, "dmoe_quantize_blocks_e4m3: %lld blocks", (long long)grid);
    quantize_square_blocks_kernel<DT><<<(unsigned)grid, 256, 0, s>>>(x, rows, cols, col_blocks, row_blocks, q, scale);
  }
  DMOE_LAUNCH_CHECK();
  return DMOE_OK;
}

}  // namespace
}  // namespace dmoe

extern "C" int dmoe_quantize_blocks_e4m3(const void* x, int dtype, int64_t batch, int64_t rows, int cols,
                                         int block_rows, void* q, int64_t q_ld, float* scale, int64_t scale_ld,
                                         void* stream) {
  clear_error();
  const char* name = "dmoe_quantize_blocks_e4m3";
  DMOE_REQUIRE(dtype_ok(dtype), "%s: dtype must be f32, f16 or bf16", name);
  DMOE_REQUIRE(block_rows == 1 || block_rows == 128, "%s: block_rows=%d must be 1 or 128", name, block_rows);
  DMOE_REQUIRE(batch >= 0 && rows >= 0 && cols > 0 && cols <= (1 << 26) && cols % 16 == 0,
               "%s: cols=%d must be a multiple of 16 up to 2^26", name, cols);
  if (batch == 0 || rows == 0) return DMOE_OK;
  DMOE_REQUIRE(batch <= (INT64_MAX >> 24) / rows, "%s: %lld x %lld rows", name, (long long)batch, (long long)rows);
  DMOE_REQUIRE(x && q && scale, "%s: null pointer", name);
  DMOE_REQUIRE(aligned16(x) && aligned16(q) && (reinterpret_cast<uintptr_t>(scale) & 3u) == 0,
               "%s: x and q must be 16-byte aligned, scale 4-byte", name);
  const int col_blocks = (cols + 127) / 128;
  DMOE_REQUIRE(q_ld >= cols && q_ld % 16 == 0 && scale_ld >= (block_rows == 1 ? col_blocks : 0),
               "%s: q_ld=%lld must be >= cols and a multiple of 16, scale_ld=%lld >= %d", name, (long long)q_ld,
               (long long)scale_ld, col_blocks);
  DMOE_REQUIRE(block_rows == 1 || (q_ld == cols && scale_ld == col_blocks), "%s: 128 x 128 blocks take packed q and scale",
               name);
  uint8_t* qb = reinterpret_cast<uint8_t*>(q);
  cudaStream_t s = as_stream(stream);
  if (dtype == DMOE_BF16)
    return run_quantize_blocks<DMOE_BF16>(x, batch, rows, cols, block_rows, qb, q_ld, scale, scale_ld, s);
  if (dtype == DMOE_F16)
    return run_quantize_blocks<DMOE_F16>(x, batch, rows, cols, block_rows, qb, q_ld, scale, scale_ld, s);
  return run_quantize_blocks<DMOE_F32>(x, batch, rows, cols, block_rows, qb, q_ld, scale, scale_ld, s);
}

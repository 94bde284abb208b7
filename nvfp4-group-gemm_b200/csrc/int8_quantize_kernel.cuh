// Rows of 16-bit activations to int8 codes with one fp32 scale per row.
//
//   scale = max_k |x[k]| / 127        code[k] = rne(127 * x[k] / max|x|)
//
// (rne: nearest integer, ties to even; a row of zeros has scale 0 and zero codes; a row that
// holds an infinity or a NaN has scale NaN and zero codes, so that whatever the row is
// multiplied into is NaN as well).
//
// The codes are those of the exact quotient. 127 x is exact in fp32 for bf16 and fp16 x. With
// t = x * (127 / max|x|), rounded twice, |t - exact| <= 2^-23 |t|. Where the exact quotient T
// is not half-way between two integers it is at least |T| / (254 * 2047) > 2^-19 |T| away from
// such a point (both are ratios of integers of at most 11 bits times 127), so rne(t) is right;
// where it is half-way, the residual r = 127 x - q max|x| (exact: a product of 7 and 11 bits)
// has 2 |r| = max|x|, and an odd q is moved to its even neighbour. Rows with maxima far from 1
// are scaled by 2^+-64 first, so that 127 / max|x| and 127 x stay in range.
//
// Bound by memory: each row is read once and kept in registers between the maximum and the
// codes (rows above kInt8RegCols columns are read again, from L2 by then).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "sm100_ptx.cuh"

namespace nvfp4 {

constexpr int kInt8QuantThreads = 256;
constexpr int kInt8Chunk = 16;         // columns a thread handles at once: 32 bytes in, 16 out
constexpr int kInt8ChunksPerThread = 2;  // chunks kept in registers
constexpr int kInt8RegCols = kInt8QuantThreads * kInt8Chunk * kInt8ChunksPerThread;

struct Int8QuantParams {
  const uint16_t* x;     // bf16 or fp16 bits
  int64_t ld;            // elements between rows
  int32_t rows;
  int32_t cols;
  int32_t vec;           // x and its rows are 16-byte aligned
  const int32_t* row_mask;  // nullptr, or rows with row_mask[r] < 0 are left out
  const int32_t* dest;   // nullptr: row r goes to row r; else to rows dest[r * topk + j]
  int32_t topk;
  int32_t out_rows;      // destinations outside [0, out_rows) are dropped
  int8_t* codes;
  int64_t codes_ld;      // bytes, a multiple of 16
  float* scales;
};

template <typename T>
__device__ __forceinline__ uint32_t int8_absmax2(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t int8_absmax2<__nv_bfloat16>(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                       __habs2(*reinterpret_cast<const __nv_bfloat162*>(&b)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <>
__device__ __forceinline__ uint32_t int8_absmax2<__half>(uint32_t a, uint32_t b) {
  const __half2 r = __hmax2_nan(*reinterpret_cast<const __half2*>(&a),
                                __habs2(*reinterpret_cast<const __half2*>(&b)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

template <typename T>
__device__ __forceinline__ float2 int8_unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 int8_unpack2<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 int8_unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// The 16 columns from c0 of a row as eight pairs; columns past the end read as 0.
__device__ __forceinline__ void int8_load_chunk(const uint16_t* __restrict__ row, int c0, int cols,
                                                bool vec, uint32_t (&v)[8]) {
  if (vec && c0 + kInt8Chunk <= cols) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(row + c0));
    const uint4 b = __ldg(reinterpret_cast<const uint4*>(row + c0) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = c0 + 2 * i;
    const uint32_t lo = c < cols ? __ldg(row + c) : 0u;
    const uint32_t hi = c + 1 < cols ? __ldg(row + c + 1) : 0u;
    v[i] = lo | (hi << 16);
  }
}

// Code of one scaled value (low byte of the result). xs = x * s, inv = 127 / (max|x| * s).
__device__ __forceinline__ uint32_t int8_code(float xs, float inv, float amax_s) {
  const float magic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer, ties to even
  const float m = __fadd_rn(__fmul_rn(xs, inv), magic);
  const float q = __fsub_rn(m, magic);
  const float r = __fmaf_rn(-q, amax_s, __fmul_rn(xs, 127.0f));
  uint32_t bits = __float_as_uint(m);
  if (__fmul_rn(fabsf(r), 2.0f) == amax_s && (bits & 1u)) bits += r > 0.0f ? 1u : 0xffffffffu;
  return bits;
}

template <typename T>
__device__ __forceinline__ uint4 int8_codes16(const uint32_t (&v)[8], float s, float inv,
                                              float amax_s) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = int8_unpack2<T>(v[2 * i]);
    const float2 b = int8_unpack2<T>(v[2 * i + 1]);
    const uint32_t q0 = int8_code(__fmul_rn(a.x, s), inv, amax_s);
    const uint32_t q1 = int8_code(__fmul_rn(a.y, s), inv, amax_s);
    const uint32_t q2 = int8_code(__fmul_rn(b.x, s), inv, amax_s);
    const uint32_t q3 = int8_code(__fmul_rn(b.y, s), inv, amax_s);
    w[i] = __byte_perm(__byte_perm(q0, q1, 0x0040), __byte_perm(q2, q3, 0x0040), 0x5410);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 16 codes at column c0; the bytes behind the row's last column are not written.
__device__ __forceinline__ void int8_store_chunk(int8_t* row, int c0, int cols, const uint4& q) {
  if (c0 + kInt8Chunk <= cols) {
    *reinterpret_cast<uint4*>(row + c0) = q;
    return;
  }
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < kInt8Chunk; ++i)
    if (c0 + i < cols) row[c0 + i] = static_cast<int8_t>(w[i / 4] >> (8 * (i % 4)));
}

// G threads per row, kInt8QuantThreads / G rows per block. The group is the smallest that
// holds the row in registers: few threads per row keep many rows in flight per SM.
template <typename T, int G>
__global__ void __launch_bounds__(kInt8QuantThreads)
    nvfp4_quantize_int8_kernel(const __grid_constant__ Int8QuantParams p) {
  constexpr int kRows = kInt8QuantThreads / G;
  __shared__ uint32_t warp_max[kInt8QuantThreads / 32];
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int group = threadIdx.x / G;
  const int gt = threadIdx.x % G;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * kRows + group;
  const bool active = r < p.rows && (p.row_mask == nullptr || __ldg(p.row_mask + r) >= 0);
  const uint16_t* row = p.x + r * p.ld;
  const int cols = active ? p.cols : 0;
  uint32_t v[kInt8ChunksPerThread][8];
  uint32_t m2 = 0u;
#pragma unroll
  for (int u = 0; u < kInt8ChunksPerThread; ++u) {
    const int c0 = (gt + u * G) * kInt8Chunk;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[u][i] = 0u;
    if (c0 < cols) int8_load_chunk(row, c0, cols, p.vec != 0, v[u]);
  }
#pragma unroll
  for (int u = 0; u < kInt8ChunksPerThread; ++u)
#pragma unroll
    for (int i = 0; i < 8; ++i) m2 = int8_absmax2<T>(m2, v[u][i]);
  for (int c0 = (gt + kInt8ChunksPerThread * G) * kInt8Chunk; c0 < cols; c0 += G * kInt8Chunk) {
    uint32_t t[8];
    int8_load_chunk(row, c0, cols, p.vec != 0, t);
#pragma unroll
    for (int i = 0; i < 8; ++i) m2 = int8_absmax2<T>(m2, t[i]);
  }
  // Non-negative fp32 values order like their bits, with every NaN above infinity.
  const float2 mf = int8_unpack2<T>(m2);
  uint32_t mb = max(__float_as_uint(mf.x) & 0x7fffffffu, __float_as_uint(mf.y) & 0x7fffffffu);
  mb = __reduce_max_sync(0xffffffffu, mb);
  if (G > 32) {
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = mb;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < G / 32; ++i) mb = max(mb, warp_max[group * (G / 32) + i]);
  }
  if (!active) return;
  const bool finite = mb < 0x7f800000u;
  const float amax = __uint_as_float(mb);
  const float s = !finite || mb == 0u ? 0.0f
                  : amax < 5.42101086e-20f ? 18446744073709551616.0f
                  : amax > 18446744073709551616.0f ? 5.42101086e-20f : 1.0f;  // 2^+-64
  const float amax_s = __fmul_rn(amax, s);
  const float inv = s == 0.0f ? 0.0f : __fdiv_rn(127.0f, amax_s);
  const float scale = finite ? __fdiv_rn(amax, 127.0f) : __uint_as_float(0x7fc00000u);
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  uint4 q[kInt8ChunksPerThread];
#pragma unroll
  for (int u = 0; u < kInt8ChunksPerThread; ++u)
    q[u] = s == 0.0f ? zero : int8_codes16<T>(v[u], s, inv, amax_s);
  const int copies = p.dest == nullptr ? 1 : p.topk;
  for (int j = 0; j < copies; ++j) {
    const int64_t d = p.dest == nullptr ? r : __ldg(p.dest + r * p.topk + j);
    if (d < 0 || d >= p.out_rows) continue;
    int8_t* out = p.codes + d * p.codes_ld;
    if (gt == 0) p.scales[d] = scale;
#pragma unroll
    for (int u = 0; u < kInt8ChunksPerThread; ++u) {
      const int c0 = (gt + u * G) * kInt8Chunk;
      if (c0 < cols) int8_store_chunk(out, c0, cols, q[u]);
    }
  }
  for (int c0 = (gt + kInt8ChunksPerThread * G) * kInt8Chunk; c0 < cols; c0 += G * kInt8Chunk) {
    uint32_t t[8];
    int8_load_chunk(row, c0, cols, p.vec != 0, t);
    const uint4 qt = s == 0.0f ? zero : int8_codes16<T>(t, s, inv, amax_s);
    for (int j = 0; j < copies; ++j) {
      const int64_t d = p.dest == nullptr ? r : __ldg(p.dest + r * p.topk + j);
      if (d >= 0 && d < p.out_rows) int8_store_chunk(p.codes + d * p.codes_ld, c0, cols, qt);
    }
  }
}

}  // namespace nvfp4

// Rows of 16-bit activations to int8 codes with one fp32 scale per row.
//
//   scale = max_k |x[k]| / 127        code[k] = rne(127 * x[k] / max|x|)
//
// (rne: nearest integer, ties to even; a row of zeros has scale 0 and zero codes; a row that
// holds an infinity or a NaN has scale NaN and zero codes, so that whatever the row is
// multiplied into is NaN as well).
//
// The codes are those of the exact quotient T = 127 x / max|x|. With inv = 127 / max|x| rounded
// once, x * inv is within 2^-24 |T| of T, and a fused multiply-add of 1.5 * 2^23 rounds it to an
// integer q, ties to even. Where T is not half-way between two integers it is at least
// |T| / (254 * 2047) > 2^-19 |T| away from such a point (both are ratios of integers of at most
// 11 bits times 127), so q is right. Only quotients within 2e-5 of a half-way point (more than
// 127 * 2^-24 and the rounding of their distance) are looked at again: 127 x - q' max|x| is
// exact in fp32 (7 and 11 bits), twice its size is max|x| at a tie, and an odd q' is moved to its
// even neighbour there. Rows with maxima far from 1 are scaled by 2^+-64 first, so that 127 / max
// and 127 x stay in range.
//
// Each row is read once and kept in registers between the maximum and the codes (wider rows than
// a group's registers hold are read again, from L2 by then).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "sm100_ptx.cuh"

namespace nvfp4 {

constexpr int kInt8Chunk = 8;  // columns a thread handles at once: a warp loads 512 bytes in a row

struct Int8QuantParams {
  const uint16_t* x;     // bf16 or fp16 bits
  int64_t ld;            // elements between rows
  int32_t rows;
  int32_t cols;
  int32_t align;         // rows of x start on 16-byte (16) or 4-byte (4) boundaries, or any (2)
  const int32_t* row_list;  // nullptr: every row; else `listed` rows (outside [0, rows): none)
  int32_t listed;
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

// The 8 columns from c0 of a row as four pairs; columns past the end read as 0.
__device__ __forceinline__ void int8_load_chunk(const uint16_t* __restrict__ row, int c0, int cols,
                                                int align, uint32_t (&v)[4]) {
  if (align == 16 && c0 + kInt8Chunk <= cols) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(row + c0));
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  } else if (align >= 4 && c0 + kInt8Chunk <= cols) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __ldg(reinterpret_cast<const uint32_t*>(row + c0) + i);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = c0 + 2 * i;
      const uint32_t lo = c < cols ? __ldg(row + c) : 0u;
      const uint32_t hi = c + 1 < cols ? __ldg(row + c + 1) : 0u;
      v[i] = lo | (hi << 16);
    }
  }
}

// A row's constants: x * s is in range, amax_s = max|x| * s, inv = 127 / amax_s; s = 0 for rows
// whose codes are all zero.
struct Int8RowScale {
  float s, amax_s, inv;
};

constexpr float kInt8Magic = 12582912.0f;  // 1.5 * 2^23: the sum's low byte is the integer's
constexpr float kInt8NearTie = 0.49998f;

// The codes (low bytes) of four values. SCALED: s is not 1.
template <bool SCALED>
__device__ __forceinline__ uint32_t int8_codes4(float (&x)[4], const Int8RowScale& k) {
  float m[4], d[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (SCALED) x[e] = __fmul_rn(x[e], k.s);
    m[e] = __fmaf_rn(x[e], k.inv, kInt8Magic);
    d[e] = __fmaf_rn(x[e], k.inv, __fsub_rn(kInt8Magic, m[e]));
  }
  const float off = fmaxf(fmaxf(fabsf(d[0]), fabsf(d[1])), fmaxf(fabsf(d[2]), fabsf(d[3])));
  uint32_t q[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) q[e] = __float_as_uint(m[e]);
  if (off > kInt8NearTie) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (fabsf(d[e]) > kInt8NearTie) {
        const float r = __fmaf_rn(__fsub_rn(kInt8Magic, m[e]), k.amax_s, __fmul_rn(x[e], 127.0f));
        if (__fmul_rn(fabsf(r), 2.0f) == k.amax_s && (q[e] & 1u))
          q[e] += r > 0.0f ? 1u : 0xffffffffu;
      }
    }
  }
  return __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
}

template <typename T>
__device__ __forceinline__ uint2 int8_codes8(const uint32_t (&v)[4], const Int8RowScale& k) {
  float x[2][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = int8_unpack2<T>(v[i]);
    x[i / 2][2 * (i % 2)] = a.x;
    x[i / 2][2 * (i % 2) + 1] = a.y;
  }
  if (k.s == 1.0f) return make_uint2(int8_codes4<false>(x[0], k), int8_codes4<false>(x[1], k));
  if (k.s == 0.0f) return make_uint2(0u, 0u);
  return make_uint2(int8_codes4<true>(x[0], k), int8_codes4<true>(x[1], k));
}

// 8 codes at column c0; the bytes behind the row's last column are not written.
__device__ __forceinline__ void int8_store_chunk(int8_t* row, int c0, int cols, const uint2& q) {
  if (c0 + kInt8Chunk <= cols) {
    *reinterpret_cast<uint2*>(row + c0) = q;
    return;
  }
#pragma unroll
  for (int i = 0; i < kInt8Chunk; ++i)
    if (c0 + i < cols) row[c0 + i] = static_cast<int8_t>((i < 4 ? q.x : q.y) >> (8 * (i % 4)));
}

// G threads on a row, each with V chunks of it in registers; blocks of one row, or of 128 threads
// where fewer hold one. DISPATCH: a row goes to the rows dest names, else to its own. Small blocks
// start and end without waiting for one another: 69,632 rows of 4096 columns took 149 us (0.88 of
// the measured copy rate) in blocks of 128, 159 in blocks of 256, and 198 with the exact check on
// every element.
template <int G>
__host__ __device__ constexpr int int8_quant_threads() { return G < 128 ? 128 : G; }

template <typename T, int G, int V, bool DISPATCH>
__global__ void __launch_bounds__(int8_quant_threads<G>(), 1536 / int8_quant_threads<G>())
    nvfp4_quantize_int8_kernel(const __grid_constant__ Int8QuantParams p) {
  constexpr int kRows = int8_quant_threads<G>() / G;
  __shared__ uint32_t warp_max[int8_quant_threads<G>() / 32];
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int group = threadIdx.x / G;
  const int gt = threadIdx.x % G;
  int64_t r = static_cast<int64_t>(blockIdx.x) * kRows + group;
  if (!DISPATCH && p.row_list != nullptr) r = r < p.listed ? __ldg(p.row_list + r) : -1;
  const bool active = r >= 0 && r < p.rows;
  const uint16_t* row = p.x + r * p.ld;
  const int cols = active ? p.cols : 0;
  uint32_t v[V][4];
  uint32_t m2 = 0u;
#pragma unroll
  for (int u = 0; u < V; ++u) {
    const int c0 = (gt + u * G) * kInt8Chunk;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[u][i] = 0u;
    if (c0 < cols) int8_load_chunk(row, c0, cols, p.align, v[u]);
  }
#pragma unroll
  for (int u = 0; u < V; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) m2 = int8_absmax2<T>(m2, v[u][i]);
  for (int c0 = (gt + V * G) * kInt8Chunk; c0 < cols; c0 += G * kInt8Chunk) {
    uint32_t t[4];
    int8_load_chunk(row, c0, cols, p.align, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) m2 = int8_absmax2<T>(m2, t[i]);
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
  Int8RowScale k;
  k.s = s;
  k.amax_s = __fmul_rn(amax, s);
  k.inv = s == 0.0f ? 0.0f : __fdiv_rn(127.0f, k.amax_s);
  float scale = 0.0f;  // the group's first thread stores it
  if (gt == 0) scale = finite ? __fdiv_rn(amax, 127.0f) : __uint_as_float(0x7fc00000u);
  uint2 q[V];
#pragma unroll
  for (int u = 0; u < V; ++u) q[u] = int8_codes8<T>(v[u], k);
  // Every destination of the row (row index, or -1), four looked up at a time.
  auto for_rows = [&](auto&& store) {
    if constexpr (!DISPATCH) {
      store(static_cast<int32_t>(r));
    } else {
      for (int j0 = 0; j0 < p.topk; j0 += 4) {
        int32_t d[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          d[j] = j0 + j < p.topk ? __ldg(p.dest + r * p.topk + j0 + j) : -1;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (d[j] >= 0 && d[j] < p.out_rows) store(d[j]);
      }
    }
  };
  for_rows([&](int32_t d) {
    int8_t* out = p.codes + d * p.codes_ld;
    if (gt == 0) p.scales[d] = scale;
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const int c0 = (gt + u * G) * kInt8Chunk;
      if (c0 < cols) int8_store_chunk(out, c0, cols, q[u]);
    }
  });
  for (int c0 = (gt + V * G) * kInt8Chunk; c0 < cols; c0 += G * kInt8Chunk) {
    uint32_t t[4];
    int8_load_chunk(row, c0, cols, p.align, t);
    const uint2 qt = int8_codes8<T>(t, k);
    for_rows([&](int32_t d) { int8_store_chunk(p.codes + d * p.codes_ld, c0, cols, qt); });
  }
}

}  // namespace nvfp4

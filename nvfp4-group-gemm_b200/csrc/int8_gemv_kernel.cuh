// The int8 product for a few tokens and few weight tiles: sums of byte products on the CUDA
// cores (dp4a).
//
// A tensor-core tile takes 128 weight rows at 64 bytes per cycle at best, so a weight matrix of
// fewer tiles than SMs (N = 4096: 32) cannot be streamed at the memory's rate (one token, us on
// a B200: N 4096, K 7168 11.5; N 1024, K 8192 12.1). Here every warp of the GPU streams rows of
// its own: a lane loads 16 bytes of K of each of its R rows, several in flight, multiplies them
// with the codes of up to TB tokens, which all warps of an SM share in L1, and the warp adds up.
// Where that leaves too few warps, KS warps share rows and K, and add their sums in shared
// memory: 7.4 us with two (4.0 TB/s; 8.8 with one) and 4.3 with four (7.5 with one) for these
// sizes. A launch that does nothing takes 2.5.
//
// Segments of more than TB rows are taken in several passes over the (cached) weights.
#pragma once

#include "int8_gemm_kernel.cuh"

namespace nvfp4 {

constexpr int kInt8GemvThreads = 256;

// 16 bytes at byte c of a row, zeros where they do not end within its first k bytes.
template <bool STREAM>
__device__ __forceinline__ uint4 int8_load16(const uint8_t* __restrict__ row, int c, int k) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (c + 16 <= k) {
    if (STREAM)
      asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                   : "l"(row + c));
    else
      v = __ldg(reinterpret_cast<const uint4*>(row + c));
  }
  return v;
}

__device__ __forceinline__ int32_t int8_dot16(const uint4& a, const uint4& b, int32_t acc) {
  acc = __dp4a(static_cast<int>(a.x), static_cast<int>(b.x), acc);
  acc = __dp4a(static_cast<int>(a.y), static_cast<int>(b.y), acc);
  acc = __dp4a(static_cast<int>(a.z), static_cast<int>(b.z), acc);
  return __dp4a(static_cast<int>(a.w), static_cast<int>(b.w), acc);
}

struct Int8GemvParams {
  Int8GemmParams p;
  const uint8_t* a;
  const uint8_t* b;
  const uint8_t* b2;
  int64_t lda, ldb;
  int32_t k;
};

// The bound on blocks leaves 64 registers a thread up to TB = 4 (left to itself the compiler took
// 32 to 48, with fewer loads in flight: 4099 x 2011 4.9 us instead of 4.0) and 128 above.
template <int TB, int R, int KS, bool GATED>
__global__ void __launch_bounds__(kInt8GemvThreads, TB <= 4 ? 4 : 2)
    nvfp4_int8_gemv_kernel(const __grid_constant__ Int8GemvParams q) {
  constexpr int kWarps = kInt8GemvThreads / 32;
  constexpr int kGroups = kWarps / KS;        // groups of KS warps that share channels
  constexpr int kRows = R * (GATED ? 2 : 1);  // weight rows of a warp
  constexpr int kAhead = 8 / kRows;           // 16-byte loads in flight per row
  static_assert(kRows * TB <= 32, "one lane per sum");
  const Int8GemmParams& p = q.p;
  __shared__ int32_t used[kInt8MaxExperts];  // experts with rows
  __shared__ int32_t num_used;
  __shared__ int32_t parts[kWarps][kRows * TB];
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int part = warp % KS;
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  if (warp == 0) {
    int n = 0;
    for (int base = 0; base < p.num_experts; base += 32) {
      const int e = base + lane;
      bool has = false;
      if (e < p.num_experts) {
        int32_t off = 0, cnt = p.rows;
        if (p.seg_offsets != nullptr) {
          off = __ldg(p.seg_offsets + e);
          cnt = __ldg(p.seg_counts + e);
        }
        if (cnt < 0 || off < 0 || static_cast<int64_t>(off) + cnt > p.rows)
          atomicOr(p.error_bits, kDevErrBadSegment);
        else
          has = cnt > 0;
      }
      const uint32_t mask = __ballot_sync(0xffffffffu, has);
      if (has) used[n + __popc(mask & ((1u << lane) - 1u))] = e;
      n += __popc(mask);
    }
    if (lane == 0) num_used = n;
  }
  __syncthreads();
  constexpr int kChannels = kGroups * R;  // of a block
  const int blocks = (p.n + kChannels - 1) / kChannels;
  const int64_t units = static_cast<int64_t>(num_used) * blocks;
  for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int e = used[unit / blocks];
    const int n0 = static_cast<int>(unit % blocks) * kChannels + warp / KS * R;
    const int32_t row0 = p.seg_offsets != nullptr ? __ldg(p.seg_offsets + e) : 0;
    const int32_t cnt = p.seg_counts != nullptr ? __ldg(p.seg_counts + e) : p.rows;
    const uint8_t* w[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int64_t row = static_cast<int64_t>(e) * p.n + min(n0 + i % R, p.n - 1);
      w[i] = (i < R ? q.b : q.b2) + row * q.ldb;
    }
    for (int t0 = 0; t0 < cnt; t0 += TB) {
      const uint8_t* x[TB];
#pragma unroll
      for (int t = 0; t < TB; ++t)
        x[t] = q.a + (static_cast<int64_t>(row0) + min(t0 + t, cnt - 1)) * q.lda;
      int32_t acc[kRows][TB];
#pragma unroll
      for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int t = 0; t < TB; ++t) acc[i][t] = 0;
      for (int c0 = 16 * lane + 512 * part; c0 < q.k; c0 += 512 * KS * kAhead) {
        uint4 wv[kRows][kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
          for (int i = 0; i < kRows; ++i)
            wv[i][u] = int8_load16<true>(w[i], c0 + 512 * KS * u, q.k);
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
          for (int t = 0; t < TB; ++t) {
            const uint4 xv = int8_load16<false>(x[t], c0 + 512 * KS * u, q.k);
#pragma unroll
            for (int i = 0; i < kRows; ++i) acc[i][t] = int8_dot16(wv[i][u], xv, acc[i][t]);
          }
      }
      // The last k % 16 bytes, one per lane.
      const int tail = q.k & 15;
      if (part == 0 && lane < tail) {
        const int c = q.k - tail + lane;
        int32_t xb[TB];
#pragma unroll
        for (int t = 0; t < TB; ++t) xb[t] = static_cast<int8_t>(__ldg(x[t] + c));
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const int32_t wb = static_cast<int8_t>(__ldg(w[i] + c));
#pragma unroll
          for (int t = 0; t < TB; ++t) acc[i][t] += wb * xb[t];
        }
      }
      // Lane i of the group's first warp gets sum i (i = r + R t, the second set's behind the
      // first's), of all its warps.
      int32_t sum = 0;
#pragma unroll
      for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int t = 0; t < TB; ++t) {
          const int32_t s = __reduce_add_sync(0xffffffffu, acc[i][t]);
          if (lane == i % R + R * t + (i / R) * R * TB) sum = s;
        }
      if (KS > 1) {
        if (t0 > 0) __syncthreads();  // the previous sums are read
        if (lane < kRows * TB) parts[warp][lane] = sum;
        __syncthreads();
        if (part == 0 && lane < kRows * TB)
#pragma unroll
          for (int k = 1; k < KS; ++k) sum += parts[warp + k][lane];
      }
      if (part != 0) continue;
      const int32_t h = GATED ? __shfl_sync(0xffffffffu, sum, (lane + R * TB) & 31) : 0;
      const int n = n0 + lane % R;
      const int tok = t0 + lane / R;
      if (lane < R * TB && n < p.n && tok < cnt) {
        const int64_t row = static_cast<int64_t>(row0) + tok;
        const int64_t chan = static_cast<int64_t>(e) * p.n + n;
        const float as = __ldg(p.a_scale + row);
        float y = __fmul_rn(__fmul_rn(__int2float_rn(sum), as), __ldg(p.b_scale + chan));
        if (GATED) {
          const float g[1] = {y};
          const float u[1] = {__fmul_rn(__fmul_rn(__int2float_rn(h), as),
                                        __ldg(p.b2_scale + chan))};
          float z[1];
          int8_gate(p.out_dtype, g, u, z);
          y = z[0];
        } else {
          y = __fadd_rn(y, p.bias != nullptr ? __ldg(p.bias + n) : 0.0f);
        }
        const int64_t at = row * p.ldo + n;
        if (p.out_dtype == kInt8OutBf16)
          static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(y);
        else if (p.out_dtype == kInt8OutFp16)
          static_cast<__half*>(p.out)[at] = __float2half_rn(y);
        else
          static_cast<float*>(p.out)[at] = y;
      }
    }
    if (KS > 1) __syncthreads();  // the sums are read before the next unit writes its own
  }
}

}  // namespace nvfp4

// Tokens sorted by expert and back, in bf16, fp16 or fp32, with their gradients.
//
//   dispatch    y[dest[t, j]] = x[t] for every kept pair (t, j), 0 on padding rows
//   combine     out[t] = sum_j w[t, j] * y[dest[t, j]]   (without weights: the gradient of
//               dispatch), slot order, fp32 products and sums, rounded once at the end
//   combine's gradients   dy[dest[t, j]] = w[t, j] * dout[t], 0 on padding rows;
//                         dw[t, j] = sum_c dout[t, c] * y[dest[t, j], c] in fp32
//
// All three work by token, not by sorted row: a token's own row is read once however many
// experts it goes to, and no pair's row is written by two threads, so there are no atomics and
// results do not depend on timing. Pairs whose row is outside [0, rows) are dropped pairs.
// They are bound by memory.
//
// Columns move in pieces of 16 bytes (VEC elements) where every row involved starts on a
// 16-byte boundary, one element at a time otherwise.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "sm100_ptx.cuh"

namespace nvfp4 {

struct TokenSortParams {
  const void* x;       // dispatch: x; combine: y; gradients: dout [tokens, cols]
  const void* y;       // gradients: y [rows, cols] (nullptr: no weight gradient)
  void* out;           // dispatch: y; combine: out; gradients: dy (nullptr: not wanted)
  const int32_t* dest;
  const int32_t* src_rows;  // < 0 marks padding rows (dispatch, gradients)
  const float* weights;     // nullptr: all ones
  float* grad_w;            // nullptr: not wanted
  int64_t ldx, ldy, ldo;
  int32_t tokens, topk, cols, rows;
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Piece {
  T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ Piece<T, VEC> load_piece(const T* p) {
  Piece<T, VEC> r;
  if constexpr (VEC == 1) {
    r.v[0] = *p;
  } else {
    *reinterpret_cast<uint4*>(&r) = __ldg(reinterpret_cast<const uint4*>(p));
  }
  return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void store_piece(T* p, const Piece<T, VEC>& r) {
  if constexpr (VEC == 1) {
    *p = r.v[0];
  } else {
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ Piece<T, VEC> zero_piece() {
  Piece<T, VEC> r;
#pragma unroll
  for (int i = 0; i < VEC; ++i) r.v[i] = T(0.0f);
  return r;
}
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

constexpr int kSortThreads = 256;
constexpr int kSortPieces = 4;  // pieces a lane moves per task, all loaded before the first store

// Zero columns [c0, c0 + span) of the padding rows among rows [32 g, 32 g + 32). Warp-wide.
template <typename T, int VEC>
__device__ __forceinline__ void zero_padding(const TokenSortParams& p, int64_t g, int c0, int span,
                                             int lane) {
  const int64_t r = g * 32 + lane;
  uint32_t pad = __ballot_sync(0xffffffffu, r < p.rows && __ldg(p.src_rows + r) < 0);
  const int c1 = min(p.cols, c0 + span);
  const Piece<T, VEC> z = zero_piece<T, VEC>();
  while (pad != 0u) {
    const int i = __ffs(pad) - 1;
    pad &= pad - 1;
    T* row = static_cast<T*>(p.out) + (g * 32 + i) * p.ldo;
    for (int c = c0 + lane * VEC; c < c1; c += 32 * VEC) store_piece<T, VEC>(row + c, z);
  }
}

// One warp per (token, 32 * VEC * kSortPieces columns), then one per (32 rows, as many columns)
// for the padding.
template <typename T, int VEC>
__global__ void __launch_bounds__(kSortThreads)
    nvfp4_dispatch_tokens_kernel(const __grid_constant__ TokenSortParams p) {
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  constexpr int kSpan = 32 * VEC * kSortPieces;
  const int lane = threadIdx.x & 31;
  const int chunks = (p.cols + kSpan - 1) / kSpan;
  const int64_t task = (static_cast<int64_t>(blockIdx.x) * kSortThreads + threadIdx.x) >> 5;
  const int64_t t = task / chunks;
  const int c0 = static_cast<int>(task % chunks) * kSpan;
  if (t >= p.tokens) {
    const int64_t g = t - p.tokens;
    if (g * 32 < p.rows) zero_padding<T, VEC>(p, g, c0, kSpan, lane);
    return;
  }
  const T* row = static_cast<const T*>(p.x) + t * p.ldx;
  Piece<T, VEC> v[kSortPieces];
#pragma unroll
  for (int u = 0; u < kSortPieces; ++u) {
    const int c = c0 + (u * 32 + lane) * VEC;
    v[u] = c < p.cols ? load_piece<T, VEC>(row + c) : zero_piece<T, VEC>();
  }
  for (int j = 0; j < p.topk; ++j) {
    const int64_t d = __ldg(p.dest + t * p.topk + j);
    if (d < 0 || d >= p.rows) continue;
    T* out = static_cast<T*>(p.out) + d * p.ldo;
#pragma unroll
    for (int u = 0; u < kSortPieces; ++u) {
      const int c = c0 + (u * 32 + lane) * VEC;
      if (c < p.cols) store_piece<T, VEC>(out + c, v[u]);
    }
  }
}

// One warp per (token, 32 * VEC columns); up to eight slots' rows are loaded before the first
// is added.
template <typename T, int VEC>
__global__ void __launch_bounds__(kSortThreads)
    nvfp4_combine_tokens_kernel(const __grid_constant__ TokenSortParams p) {
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  constexpr int kSpan = 32 * VEC;
  const int lane = threadIdx.x & 31;
  const int chunks = (p.cols + kSpan - 1) / kSpan;
  const int64_t task = (static_cast<int64_t>(blockIdx.x) * kSortThreads + threadIdx.x) >> 5;
  const int64_t t = task / chunks;
  const int c = static_cast<int>(task % chunks) * kSpan + lane * VEC;
  if (t >= p.tokens || c >= p.cols) return;
  const T* y = static_cast<const T*>(p.x);
  float acc[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
  for (int j0 = 0; j0 < p.topk; j0 += 8) {
    int64_t d[8];
    Piece<T, VEC> v[8];
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      d[j] = j0 + j < p.topk ? __ldg(p.dest + t * p.topk + j0 + j) : -1;
      if (d[j] >= p.rows) d[j] = -1;
      w[j] = d[j] >= 0 && p.weights != nullptr ? __ldg(p.weights + t * p.topk + j0 + j) : 1.0f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (d[j] >= 0) v[j] = load_piece<T, VEC>(y + d[j] * p.ldx + c);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (d[j] < 0) continue;
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        acc[i] = __fadd_rn(acc[i], __fmul_rn(w[j], to_f32(v[j].v[i])));
    }
  }
  Piece<T, VEC> o;
#pragma unroll
  for (int i = 0; i < VEC; ++i) o.v[i] = from_f32<T>(acc[i]);
  store_piece<T, VEC>(static_cast<T*>(p.out) + t * p.ldo + c, o);
}

// One block per token; blocks behind the tokens zero the padding of 32 rows each.
template <typename T, int VEC>
__global__ void __launch_bounds__(kSortThreads)
    nvfp4_combine_tokens_backward_kernel(const __grid_constant__ TokenSortParams p) {
  constexpr int kWarps = kSortThreads / 32;
  __shared__ float part[kWarps][8];
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int64_t t = blockIdx.x;
  if (t >= p.tokens) {
    const int span = ((p.cols + kWarps - 1) / kWarps + 32 * VEC - 1) / (32 * VEC) * (32 * VEC);
    if (warp * span < p.cols) zero_padding<T, VEC>(p, t - p.tokens, warp * span, span, lane);
    return;
  }
  const T* g = static_cast<const T*>(p.x) + t * p.ldx;
  const T* y = static_cast<const T*>(p.y);
  T* dy = static_cast<T*>(p.out);
  for (int j0 = 0; j0 < p.topk; j0 += 8) {
    int64_t d[8];
    float w[8], acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      d[j] = j0 + j < p.topk ? __ldg(p.dest + t * p.topk + j0 + j) : -1;
      if (d[j] >= p.rows) d[j] = -1;
      w[j] = d[j] >= 0 && p.weights != nullptr ? __ldg(p.weights + t * p.topk + j0 + j) : 1.0f;
      acc[j] = 0.0f;
    }
    for (int c = threadIdx.x * VEC; c < p.cols; c += kSortThreads * VEC) {
      const Piece<T, VEC> gv = load_piece<T, VEC>(g + c);
      if (p.grad_w != nullptr) {
        Piece<T, VEC> v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (d[j] >= 0) v[j] = load_piece<T, VEC>(y + d[j] * p.ldy + c);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (d[j] < 0) continue;
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[j] += to_f32(gv.v[i]) * to_f32(v[j].v[i]);
        }
      }
      if (dy != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (d[j] < 0) continue;
          Piece<T, VEC> o;
#pragma unroll
          for (int i = 0; i < VEC; ++i) o.v[i] = from_f32<T>(__fmul_rn(w[j], to_f32(gv.v[i])));
          store_piece<T, VEC>(dy + d[j] * p.ldo + c, o);
        }
      }
    }
    if (p.grad_w != nullptr) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], s);
        if (lane == 0) part[warp][j] = acc[j];
      }
      __syncthreads();
      if (threadIdx.x < 8 && j0 + static_cast<int>(threadIdx.x) < p.topk) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) sum += part[i][threadIdx.x];
        p.grad_w[t * p.topk + j0 + threadIdx.x] = sum;
      }
      __syncthreads();
    }
  }
}

}  // namespace nvfp4

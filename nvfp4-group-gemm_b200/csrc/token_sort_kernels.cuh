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
// Columns move in pieces of 16, 8 or 4 bytes (VEC elements), the largest on whose boundaries
// every row involved starts and that divides the row, or one element at a time (bf16, 8192 x 8
// pairs of 4095 columns: 0.6 - 0.7 of the copy rate instead of 0.92 and more at 4096).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

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

template <int BYTES>
struct PieceWords;
template <>
struct PieceWords<16> { using type = uint4; };
template <>
struct PieceWords<8> { using type = uint2; };
template <>
struct PieceWords<4> { using type = uint32_t; };

// VEC consecutive elements: one element, or 4 to 16 bytes kept as words until they are used (as
// arrays of bf16 they took twice the registers).
template <typename T, int VEC>
struct Piece {
  using Words = typename PieceWords<VEC * sizeof(T)>::type;
  static constexpr int kWords = VEC * sizeof(T) / 4;
  Words w;
  __device__ __forceinline__ uint32_t word(int k) const {
    if constexpr (kWords == 1) return w;
    else if constexpr (kWords == 2) return k ? w.y : w.x;
    else return k < 2 ? (k ? w.y : w.x) : (k == 2 ? w.z : w.w);
  }
  __device__ __forceinline__ void put(const uint32_t (&k)[kWords]) {
    if constexpr (kWords == 1) w = k[0];
    else if constexpr (kWords == 2) w = make_uint2(k[0], k[1]);
    else w = make_uint4(k[0], k[1], k[2], k[3]);
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(word(i));
    } else {
      const uint32_t v = word(i / 2);
      if constexpr (std::is_same<T, __half>::value)
        return __half2float(__ushort_as_half(static_cast<uint16_t>(i & 1 ? v >> 16 : v & 0xffffu)));
      else
        return __uint_as_float(i & 1 ? v & 0xffff0000u : v << 16);
    }
  }
  __device__ __forceinline__ void set(const float (&f)[VEC]) {
    uint32_t words[kWords];
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      if constexpr (sizeof(T) == 4) {
        words[k] = __float_as_uint(f[k]);
      } else if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(f[2 * k], f[2 * k + 1]);
        words[k] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * k], f[2 * k + 1]);
        words[k] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    put(words);
  }
  __device__ __forceinline__ void load(const T* p) { w = __ldg(reinterpret_cast<const Words*>(p)); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Words*>(p) = w; }
  __device__ __forceinline__ void clear() {
    uint32_t zero[kWords];
#pragma unroll
    for (int k = 0; k < kWords; ++k) zero[k] = 0u;
    put(zero);
  }
};
template <typename T>
struct Piece<T, 1> {
  T v;
  __device__ __forceinline__ float get(int) const { return to_f32(v); }
  __device__ __forceinline__ void set(const float (&f)[1]) { v = from_f32<T>(f[0]); }
  __device__ __forceinline__ void load(const T* p) { v = __ldg(p); }
  __device__ __forceinline__ void store(T* p) const { *p = v; }
  __device__ __forceinline__ void clear() { v = from_f32<T>(0.0f); }
};

constexpr int kSortThreads = 256;
constexpr int kSortPieces = 4;  // pieces a lane moves per task, all loaded before the first store

// The row and weight of up to eight slots of a token, from slot j0 on; row -1: dropped or past
// the last slot.
struct Slots {
  int32_t row[8];
  float w[8];
};
__device__ __forceinline__ Slots load_slots(const TokenSortParams& p, int64_t t, int j0) {
  Slots s;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool in = t < p.tokens && j0 + j < p.topk;
    s.row[j] = in ? __ldg(p.dest + t * p.topk + j0 + j) : -1;
    s.w[j] = in && p.weights != nullptr ? __ldg(p.weights + t * p.topk + j0 + j) : 1.0f;
    if (s.row[j] >= p.rows) s.row[j] = -1;
  }
  return s;
}

constexpr int kPadRows = 16;  // rows whose padding one task clears (32: 7.4 us for 300 x 4 pairs)

// Zero columns [c0, c0 + span) of the padding rows among rows [kPadRows g, kPadRows (g + 1)).
// Warp-wide.
template <typename T, int VEC>
__device__ __forceinline__ void zero_padding(const TokenSortParams& p, int64_t g, int c0, int span,
                                             int lane) {
  const int64_t r = g * kPadRows + lane;
  uint32_t pad = __ballot_sync(0xffffffffu,
                               lane < kPadRows && r < p.rows && __ldg(p.src_rows + r) < 0);
  const int c1 = min(p.cols, c0 + span);
  Piece<T, VEC> z;
  z.clear();
  while (pad != 0u) {
    const int i = __ffs(pad) - 1;
    pad &= pad - 1;
    T* row = static_cast<T*>(p.out) + (g * kPadRows + i) * p.ldo;
    for (int c = c0 + lane * VEC; c < c1; c += 32 * VEC) z.store(row + c);
  }
}

// One warp per (kPadRows rows, 32 * VEC * kSortPieces columns) for the padding, then one per
// (token, as many columns).
template <typename T, int VEC>
__global__ void __launch_bounds__(kSortThreads)
    nvfp4_dispatch_tokens_kernel(const __grid_constant__ TokenSortParams p) {
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  constexpr int kSpan = 32 * VEC * kSortPieces;
  const int lane = threadIdx.x & 31;
  const int chunks = (p.cols + kSpan - 1) / kSpan;
  const int64_t groups = (static_cast<int64_t>(p.rows) + kPadRows - 1) / kPadRows;
  const int64_t task = (static_cast<int64_t>(blockIdx.x) * kSortThreads + threadIdx.x) >> 5;
  const int64_t t = task / chunks - groups;
  const int c0 = static_cast<int>(task % chunks) * kSpan;
  if (t < 0) {
    zero_padding<T, VEC>(p, t + groups, c0, kSpan, lane);
    return;
  }
  if (t >= p.tokens) return;
  const T* row = static_cast<const T*>(p.x) + t * p.ldx;
  Piece<T, VEC> v[kSortPieces];
#pragma unroll
  for (int u = 0; u < kSortPieces; ++u) {
    const int c = c0 + (u * 32 + lane) * VEC;
    v[u].clear();
    if (c < p.cols) v[u].load(row + c);
  }
  for (int j0 = 0; j0 < p.topk; j0 += 8) {
    const Slots s = load_slots(p, t, j0);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (s.row[j] < 0) continue;
      T* out = static_cast<T*>(p.out) + s.row[j] * p.ldo;
#pragma unroll
      for (int u = 0; u < kSortPieces; ++u) {
        const int c = c0 + (u * 32 + lane) * VEC;
        if (c < p.cols) v[u].store(out + c);
      }
    }
  }
}

// Combine and its gradients: small blocks, one token each. A lane holds kTokenPieces pieces of
// every one of eight slots' rows at once, so a warp has 8 KB in flight, and short-lived blocks
// keep the SMs evenly loaded: at 8192 tokens x 8 slots x 4096 bf16 columns the gradients took
// 180 us like this (0.99 of the measured copy rate), 225 with as many persistent blocks as fit,
// 201 with blocks of 128 and one piece per lane, 235 with blocks of 256.
constexpr int kTokenThreads = 64;
constexpr int kTokenPieces = 2;

// Block b works on token b / parts, on every parts-th chunk of its columns.
template <typename T, int VEC>
__global__ void __launch_bounds__(kTokenThreads)
    nvfp4_combine_tokens_kernel(const __grid_constant__ TokenSortParams p, int parts) {
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  constexpr int P = kTokenPieces;
  constexpr int kSpan = kTokenThreads * VEC * P;  // columns of a chunk
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int64_t t = blockIdx.x / parts;
  const T* y = static_cast<const T*>(p.x);
  const Slots first = load_slots(p, t, 0);
  for (int c0 = static_cast<int>(blockIdx.x % parts) * kSpan + (warp * 32 * P + lane) * VEC;
       c0 < p.cols; c0 += parts * kSpan) {
    float acc[P][VEC];
#pragma unroll
    for (int u = 0; u < P; ++u)
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[u][i] = 0.0f;
    for (int j0 = 0; j0 < p.topk; j0 += 8) {
      const Slots s = j0 == 0 ? first : load_slots(p, t, j0);
      Piece<T, VEC> v[8][P];
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int u = 0; u < P; ++u) {
          const int c = c0 + u * 32 * VEC;
          if (s.row[j] >= 0 && c < p.cols) v[j][u].load(y + s.row[j] * p.ldx + c);
        }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (s.row[j] < 0) continue;
#pragma unroll
        for (int u = 0; u < P; ++u)
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            acc[u][i] = __fadd_rn(acc[u][i], __fmul_rn(s.w[j], v[j][u].get(i)));
      }
    }
#pragma unroll
    for (int u = 0; u < P; ++u) {
      const int c = c0 + u * 32 * VEC;
      if (c < p.cols) {
        Piece<T, VEC> o;
        o.set(acc[u]);
        o.store(static_cast<T*>(p.out) + t * p.ldo + c);
      }
    }
  }
}

// The first blocks clear the padding, kPadRows rows each; the others take one token each.
template <typename T, int VEC>
__global__ void __launch_bounds__(kTokenThreads)
    nvfp4_combine_tokens_backward_kernel(const __grid_constant__ TokenSortParams p) {
  constexpr int kWarps = kTokenThreads / 32;
  constexpr int P = kTokenPieces;
  constexpr int kSpan = kTokenThreads * VEC * P;
  __shared__ float part[kWarps][8];
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const T* y = static_cast<const T*>(p.y);
  T* dy = static_cast<T*>(p.out);
  const int64_t groups =
      dy != nullptr ? (static_cast<int64_t>(p.rows) + kPadRows - 1) / kPadRows : 0;
  const int64_t t = static_cast<int64_t>(blockIdx.x) - groups;
  if (t < 0) {
    const int span = ((p.cols + kWarps - 1) / kWarps + 32 * VEC - 1) / (32 * VEC) * (32 * VEC);
    zero_padding<T, VEC>(p, t + groups, warp * span, span, lane);
    return;
  }
  const T* g = static_cast<const T*>(p.x) + t * p.ldx;
  for (int j0 = 0; j0 < p.topk; j0 += 8) {
    const Slots s = load_slots(p, t, j0);
    float acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = 0.0f;
    for (int c0 = (warp * 32 * P + lane) * VEC; c0 < p.cols; c0 += kSpan) {
      Piece<T, VEC> gv[P];
      Piece<T, VEC> v[8][P];
#pragma unroll
      for (int u = 0; u < P; ++u) {
        const int c = c0 + u * 32 * VEC;
        gv[u].clear();
        if (c < p.cols) gv[u].load(g + c);
      }
      if (p.grad_w != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int u = 0; u < P; ++u) {
            const int c = c0 + u * 32 * VEC;
            if (s.row[j] >= 0 && c < p.cols) v[j][u].load(y + s.row[j] * p.ldy + c);
          }
      }
      if (dy != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (s.row[j] < 0) continue;
#pragma unroll
          for (int u = 0; u < P; ++u) {
            const int c = c0 + u * 32 * VEC;
            float f[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] = __fmul_rn(s.w[j], gv[u].get(i));
            Piece<T, VEC> o;
            o.set(f);
            if (c < p.cols) o.store(dy + s.row[j] * p.ldo + c);
          }
        }
      }
      if (p.grad_w != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (s.row[j] < 0) continue;
#pragma unroll
          for (int u = 0; u < P; ++u) {
            if (c0 + u * 32 * VEC >= p.cols) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[j] += gv[u].get(i) * v[j][u].get(i);
          }
        }
      }
    }
    if (p.grad_w != nullptr) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], d);
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

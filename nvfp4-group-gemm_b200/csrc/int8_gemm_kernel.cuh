// int8 matrix product with a scale per token and per channel, over one or many row segments.
//
//   out[t, n] = a_scale[t] * b_scale[e, n] * sum_k a[t, k] * b[e, n, k]  (+ bias[n])
//   gated:      g, u the same with b and b2;  out = g / (1 + exp(-g)) * u
//
// for every row t of expert e's segment [offset_e, offset_e + count_e). The sums are exact:
// tcgen05.mma kind::i8 accumulates in int32, and K <= 131071 keeps 128 * 128 * K below 2^31.
// They are converted to fp32 once, scaled there, and rounded once more to the output type.
//
// Weight rows are the MMA's M operand, tokens its N operand, so a decode step of a few tokens
// computes no padding beyond 16 columns, and a TMEM lane holds one output channel: the 32
// lanes of a warp store 32 consecutive channels of one token, coalesced for any width,
// alignment or row stride of the output, and no row outside a segment is touched.
//
// Persistent CTAs walk tiles (expert, channel tile, token tile), token tiles fastest so that
// tiles which share weights run together:
//   warp 0     computes the tile ranges of the segments, then loads tiles by TMA (128-byte
//              swizzle, zero fill past K and past the last row) into a ring of stages
//   warp 1     TMEM allocation and the single-thread MMA issue (4 x K = 32 per stage)
//   warps 2..  epilogue: TMEM -> registers -> scales -> global (4 warps, or 8 for tiles of 64
//              or more tokens, the second four taking the upper half of the tokens: with 4
//              the stores of a tile took longer than its MMAs at K = 1536)
// Accumulators are double-buffered in TMEM. Every wait is bounded in time (wait_phase).
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "grouped_gemm_kernel.cuh"
#include "sm100_ptx.cuh"

namespace nvfp4 {

constexpr int kInt8MaxExperts = 1024;
constexpr int kInt8MaxK = 131071;
constexpr int kInt8StageK = 128;  // bytes of K per stage: one 128-byte swizzle row
constexpr int kInt8SegBytes = 3 * kInt8MaxExperts * 4;

enum : int { kInt8OutBf16 = 0, kInt8OutFp16 = 1, kInt8OutFp32 = 2 };

struct Int8GemmParams {
  const float* a_scale;
  const float* b_scale;
  const float* b2_scale;
  const float* bias;  // nullptr: none
  void* out;
  int64_t ldo;  // elements
  const int32_t* seg_offsets;  // nullptr: one segment of all rows
  const int32_t* seg_counts;
  uint32_t* error_bits;
  int32_t rows;
  int32_t n;
  int32_t ktiles;
  int32_t num_experts;
  int32_t out_dtype;
  int32_t pair_rows;  // CTA pairs: most tokens of a tile, a multiple of 32 from 64 to 256
  uint32_t pair_inv;  // and 2^32 / (pair_rows / 32), rounded up
};

// Outputs of 32 channels (one per lane) x M tokens: y[i] is row i's, the first `count` rows are
// stored, a row's 32 channels at a time. (Turned in shared memory first and stored in 16-byte
// pieces, with this as the path of unaligned rows, 65,536 expert rows at N 4096, K 1536 took
// 370 - 390 us instead of 325.)
template <typename T, int M>
__device__ __forceinline__ void int8_store_rows_as(T* out, int64_t ldo, const float (&y)[M],
                                                   int count) {
#pragma unroll
  for (int i = 0; i < M; ++i) {
    if (i < count) {
      if constexpr (sizeof(T) == 4) *out = y[i];
      else if constexpr (std::is_same<T, __half>::value) *out = __float2half_rn(y[i]);
      else *out = __float2bfloat16_rn(y[i]);
    }
    out += ldo;
  }
}
// row0: first token row; n: this lane's channel (nothing is stored past the last one).
template <int M>
__device__ __forceinline__ void int8_store_rows(const Int8GemmParams& p, int64_t row0, int n,
                                                const float (&y)[M], int count) {
  if (n >= p.n) return;
  const int64_t at = row0 * p.ldo + n;
  if (p.out_dtype == kInt8OutBf16)
    int8_store_rows_as(static_cast<__nv_bfloat16*>(p.out) + at, p.ldo, y, count);
  else if (p.out_dtype == kInt8OutFp16)
    int8_store_rows_as(static_cast<__half*>(p.out) + at, p.ldo, y, count);
  else
    int8_store_rows_as(static_cast<float*>(p.out) + at, p.ldo, y, count);
}

// g / (1 + exp(-g)) * u. With e = exp(-|g|) the divisor lies in [1, 2]: written with exp(-g) it
// passes 2^126 for g in (-88.7, -87.3), where the fast division returns 0. FULL, for outputs of 32
// bits, is within 8 * 2^-24; otherwise the fast exponential and division are taken, within
// (5 + 1.2 |g|) * 2^-23, far below the rounding to 16 bits that follows.
template <bool FULL>
__device__ __forceinline__ float int8_silu_mul(float g, float u) {
  const float e = FULL ? expf(-fabsf(g)) : __expf(-fabsf(g));
  const float x = g < 0.0f ? g * e : g;
  return (FULL ? __fdiv_rn(x, 1.0f + e) : __fdividef(x, 1.0f + e)) * u;
}
// y[i] = silu(g[i]) * u[i]
template <int M>
__device__ __forceinline__ void int8_gate(int out_dtype, const float (&g)[M], const float (&u)[M],
                                          float (&y)[M]) {
  if (out_dtype == kInt8OutFp32) {
#pragma unroll
    for (int i = 0; i < M; ++i) y[i] = int8_silu_mul<true>(g[i], u[i]);
  } else {
#pragma unroll
    for (int i = 0; i < M; ++i) y[i] = int8_silu_mul<false>(g[i], u[i]);
  }
}

// Most token rows of a tile, and the tiles that hold `count` rows. Of CTA pairs these rows are the
// host's choice: a multiplication instead of the division that every warp would wait for per tile
// (exact: inv is off by less than 8 / 2^32, the dividend is below 2^27).
template <int ROWS>
struct Int8FixedRows {
  static constexpr int most = ROWS;
  __host__ __device__ __forceinline__ int tiles(int count) const {
    return (count + ROWS - 1) / ROWS;
  }
};
struct Int8PairRows {
  int most;
  uint32_t inv;
  __host__ __device__ __forceinline__ int tiles(int count) const {
    const uint32_t v = (static_cast<uint32_t>(count) + most - 1) / 32;
    return static_cast<int>(static_cast<uint64_t>(v) * inv >> 32);
  }
};

// Rows of each of `tiles` equal tiles of `count` >= 1 rows (a multiple of 32), the last one aside;
// no sum passes 2^31, whatever the count.
__host__ __device__ __forceinline__ int int8_equal_rows(int count, int tiles) {
  return ((count - 1) / tiles + 32) / 32 * 32;
}

// Segments of the launch in shared memory: first row, rows, and the end of each expert's tile
// range. Warp-wide; a segment outside the slab is skipped and reported, and so is one with which
// the segments hold more rows than the slab (they share some), so that the tiles stay within
// the host's bound.
template <typename Rows>
__device__ __forceinline__ void int8_stage_segments(const Int8GemmParams& p, Rows tile_rows,
                                                    int n_tiles, int32_t* seg_row,
                                                    int32_t* seg_cnt, int32_t* seg_end, int lane) {
  int32_t carry = 0;
  int64_t rows_before = 0;
  for (int base = 0; base < p.num_experts; base += 32) {
    const int e = base + lane;
    int32_t off = 0, cnt = 0;
    if (e < p.num_experts) {
      if (p.seg_offsets == nullptr) {
        cnt = p.rows;
      } else {
        off = __ldg(p.seg_offsets + e);
        cnt = __ldg(p.seg_counts + e);
        if (cnt < 0 || off < 0 || static_cast<int64_t>(off) + cnt > p.rows) {
          atomicOr(p.error_bits, kDevErrBadSegment);
          off = cnt = 0;
        }
      }
    }
    long long sum = cnt;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long t = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += t;
    }
    if (rows_before + sum > p.rows && cnt > 0) {
      atomicOr(p.error_bits, kDevErrBadSegment);
      off = cnt = 0;
    }
    rows_before += __shfl_sync(0xffffffffu, sum, 31);
    int32_t v = tile_rows.tiles(cnt) * n_tiles;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int32_t t = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v += t;
    }
    if (e < p.num_experts) {
      seg_row[e] = off;
      seg_cnt[e] = cnt;
      seg_end[e] = carry + v;
    }
    carry += __shfl_sync(0xffffffffu, v, 31);
  }
}

struct Int8Tile {
  int expert, row, rows, nt;  // rows: valid token rows of the tile
};

// Tile `tile` of the launch. BALANCED: an expert's tiles have equal rows (a multiple of 32, at
// tile_rows.most), the last one the remainder.
template <bool BALANCED, typename Rows>
__device__ __forceinline__ Int8Tile int8_find_tile(int tile, Rows tile_rows, int n_tiles,
                                                   int num_experts, const int32_t* seg_row,
                                                   const int32_t* seg_cnt,
                                                   const int32_t* seg_end) {
  int lo = 0, hi = num_experts - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (seg_end[mid] > tile) hi = mid;
    else lo = mid + 1;
  }
  const int cnt = seg_cnt[lo];
  const int tiles_m = tile_rows.tiles(cnt);
  const int local = tile - (seg_end[lo] - tiles_m * n_tiles);
  const int mt = local % tiles_m;
  const int rows = BALANCED ? int8_equal_rows(cnt, tiles_m) : tile_rows.most;
  return {lo, seg_row[lo] + mt * rows, min(rows, cnt - mt * rows), local / tiles_m};
}

template <int TN, bool GATED>
struct Int8Config {
  static constexpr int kSets = GATED ? 2 : 1;
  static constexpr int kEpiWarps = TN >= 64 ? 8 : 4;
  static constexpr int kThreads = 64 + 32 * kEpiWarps;
  static constexpr int kWBytes = 128 * kInt8StageK;
  static constexpr int kXBytes = TN * kInt8StageK;
  static constexpr int kStageBytes = kSets * kWBytes + kXBytes;
  static constexpr int kFixedBytes = 1024 + kInt8SegBytes + 512;
  static constexpr int kFit = (232448 - kFixedBytes) / kStageBytes;
  static constexpr int kStages = kFit > 12 ? 12 : kFit;
  static constexpr int kSmemBytes = kFixedBytes + kStages * kStageBytes;
  static constexpr int kAccCols = TN * kSets;
  static constexpr int kTmemColumns = 2 * kAccCols < 32 ? 32 : 2 * kAccCols;
  static_assert(kStages >= 3 && 8 * (2 * kStages + 5) + 16 <= 512, "shared memory layout");
  static_assert((kTmemColumns & (kTmemColumns - 1)) == 0 && kTmemColumns <= 512, "TMEM columns");
};

template <int TN, bool GATED>
__global__ void __launch_bounds__(Int8Config<TN, GATED>::kThreads, 1)
    nvfp4_int8_gemm_kernel(const __grid_constant__ CUtensorMap map_a,
                           const __grid_constant__ CUtensorMap map_a32,
                           const __grid_constant__ CUtensorMap map_b,
                           const __grid_constant__ CUtensorMap map_b2,
                           const __grid_constant__ Int8GemmParams p) {
  using Cfg = Int8Config<TN, GATED>;
  constexpr int kStages = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  int32_t* seg_row = reinterpret_cast<int32_t*>(smem + kStages * Cfg::kStageBytes);
  int32_t* seg_cnt = seg_row + kInt8MaxExperts;
  int32_t* seg_end = seg_cnt + kInt8MaxExperts;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(seg_end + kInt8MaxExperts);
  uint64_t* empty_bar = full_bar + kStages;
  uint64_t* accf_bar = empty_bar + kStages;
  uint64_t* acce_bar = accf_bar + 2;
  uint64_t* drain_bar = acce_bar + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile uint32_t* abort_flag = tmem_holder + 1;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      ptx::mbar_init(&full_bar[s], 1);
      ptx::mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(&accf_bar[a], 1);
      ptx::mbar_init(&acce_bar[a], Cfg::kEpiWarps);
    }
    ptx::mbar_init(drain_bar, 1);
    *abort_flag = 0u;
    ptx::fence_mbarrier_init();
    ptx::tma_prefetch_desc(&map_a);
    ptx::tma_prefetch_desc(&map_b);
    if (GATED) ptx::tma_prefetch_desc(&map_b2);
  }
  if (warp == 1) {
    ptx::tmem_alloc(tmem_holder, Cfg::kTmemColumns);
    ptx::tmem_relinquish_alloc_permit();
  }
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int n_tiles = (p.n + 127) / 128;
  constexpr Int8FixedRows<TN> kRows;
  if (warp == 0) int8_stage_segments(p, kRows, n_tiles, seg_row, seg_cnt, seg_end, lane);
  ptx::tcgen05_fence_before_sync();
  __syncthreads();
  ptx::tcgen05_fence_after_sync();
  const uint32_t tmem_base = *tmem_holder;
  const int total = seg_end[p.num_experts - 1];
  const int first = static_cast<int>(blockIdx.x);
  const int step = static_cast<int>(gridDim.x);

  if (warp == 0) {
    if (ptx::elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      uint32_t issued = 0;
      bool ok = true;
      for (int tile = first; ok && tile < total; tile += step) {
        const Int8Tile t =
            int8_find_tile<false>(tile, kRows, n_tiles, p.num_experts, seg_row, seg_cnt, seg_end);
        const int wrow = t.expert * p.n + t.nt * 128;
        // Tokens come in one box of TN rows, or in boxes of 32 where half the rows are enough.
        const int boxes = (t.rows + 31) / 32;
        const bool small = 64 * boxes <= TN;
        const uint32_t bytes =
            Cfg::kSets * Cfg::kWBytes + (small ? 32 * boxes * kInt8StageK : Cfg::kXBytes);
        for (int kt = 0; kt < p.ktiles; ++kt) {
          if (!wait_phase(&empty_bar[stage], phase ^ 1u, abort_flag, p.error_bits,
                          kDevErrProducerTimeout)) {
            ok = false;
            break;
          }
          uint8_t* sW = smem + stage * Cfg::kStageBytes;
          ptx::mbar_arrive_expect_tx(&full_bar[stage], bytes);
          ptx::tma_load_2d(sW, &map_b, &full_bar[stage], kt * kInt8StageK, wrow);
          if (GATED)
            ptx::tma_load_2d(sW + Cfg::kWBytes, &map_b2, &full_bar[stage], kt * kInt8StageK, wrow);
          uint8_t* sX = sW + Cfg::kSets * Cfg::kWBytes;
          if (small)
            for (int b = 0; b < boxes; ++b)
              ptx::tma_load_2d(sX + 32 * b * kInt8StageK, &map_a32, &full_bar[stage],
                               kt * kInt8StageK, t.row + 32 * b);
          else
            ptx::tma_load_2d(sX, &map_a, &full_bar[stage], kt * kInt8StageK, t.row);
          ++issued;
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // The most recent fill of each stage completes before the CTA may exit.
      const uint32_t recent = issued < static_cast<uint32_t>(kStages) ? issued : kStages;
      for (uint32_t i = 0; i < recent; ++i) {
        const uint32_t n = issued - 1 - i;
        const uint64_t t0 = ptx::globaltimer_ns();
        while (!ptx::mbar_try_wait(&full_bar[n % kStages], (n / kStages) & 1u)) {
          if (ptx::globaltimer_ns() - t0 > kWaitTimeoutNs) {
            atomicOr(p.error_bits, kDevErrDrainTimeout);
            break;
          }
        }
      }
    }
  } else if (warp == 1) {
    if (ptx::elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      uint32_t acc_parity = 0x3u;
      uint32_t local = 0;
      bool ok = true;
      for (int tile = first; ok && tile < total; tile += step, ++local) {
        const int acc = static_cast<int>(local & 1u);
        if (!wait_phase(&acce_bar[acc], (acc_parity >> acc) & 1u, abort_flag, p.error_bits,
                        kDevErrAccTimeout))
          break;
        acc_parity ^= 1u << acc;
        ptx::tcgen05_fence_after_sync();
        const uint32_t d_tmem = tmem_base + acc * Cfg::kAccCols;
        const Int8Tile t =
            int8_find_tile<false>(tile, kRows, n_tiles, p.num_experts, seg_row, seg_cnt, seg_end);
        const uint32_t idesc = ptx::make_idesc_i8(128, (t.rows + 15) / 16 * 16);
        for (int kt = 0; kt < p.ktiles; ++kt) {
          if (!wait_phase(&full_bar[stage], phase, abort_flag, p.error_bits, kDevErrMmaTimeout)) {
            ok = false;
            break;
          }
          ptx::tcgen05_fence_after_sync();
          const uint32_t sW = ptx::smem_u32(smem + stage * Cfg::kStageBytes);
          const uint64_t w_desc = ptx::make_sw128_kmajor_desc(sW);
          const uint64_t x_desc = ptx::make_sw128_kmajor_desc(sW + Cfg::kSets * Cfg::kWBytes);
#pragma unroll
          for (int kb = 0; kb < 4; ++kb)
            ptx::mma_i8(d_tmem, w_desc + 2 * kb, x_desc + 2 * kb, idesc,
                        (kt | kb) != 0 ? 1u : 0u);
          if (GATED) {
            const uint64_t w2_desc = ptx::make_sw128_kmajor_desc(sW + Cfg::kWBytes);
#pragma unroll
            for (int kb = 0; kb < 4; ++kb)
              ptx::mma_i8(d_tmem + TN, w2_desc + 2 * kb, x_desc + 2 * kb, idesc,
                          (kt | kb) != 0 ? 1u : 0u);
          }
          ptx::tcgen05_commit(&empty_bar[stage]);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        ptx::tcgen05_commit(&accf_bar[acc]);
      }
      ptx::tcgen05_commit(drain_bar);
      const uint64_t t0 = ptx::globaltimer_ns();
      while (!ptx::mbar_try_wait(drain_bar, 0)) {
        if (ptx::globaltimer_ns() - t0 > kWaitTimeoutNs) {
          atomicOr(p.error_bits, kDevErrDrainTimeout);
          break;
        }
      }
    }
  } else {
    const int quarter = warp & 3;
    // This warp's tokens of a tile: all of them, or one half.
    constexpr int kToks = TN / (Cfg::kEpiWarps / 4);
    const int tok0 = (warp - kEpilogueWarp0) / 4 * kToks;
    uint32_t full_parity = 0;
    uint32_t local = 0;
    for (int tile = first; tile < total; tile += step, ++local) {
      const Int8Tile t =
          int8_find_tile<false>(tile, kRows, n_tiles, p.num_experts, seg_row, seg_cnt, seg_end);
      const int n = t.nt * 128 + 32 * quarter + lane;
      const bool in = n < p.n;
      const int64_t chan = static_cast<int64_t>(t.expert) * p.n + n;
      const float bs = in ? __ldg(p.b_scale + chan) : 0.0f;
      const float bs2 = GATED && in ? __ldg(p.b2_scale + chan) : 0.0f;
      const float bias = !GATED && in && p.bias != nullptr ? __ldg(p.bias + n) : 0.0f;
      // Token scales, one per lane, handed out by shuffles.
      float as[(kToks + 31) / 32];
#pragma unroll
      for (int i = 0; i < (kToks + 31) / 32; ++i) {
        const int tok = tok0 + 32 * i + lane;
        as[i] = tok < t.rows ? __ldg(p.a_scale + t.row + tok) : 0.0f;
      }
      auto scaled = [](uint32_t sum, float a, float b) {
        return __fmul_rn(__fmul_rn(__int2float_rn(static_cast<int32_t>(sum)), a), b);
      };
      const int acc = static_cast<int>(local & 1u);
      if (!warp_wait_phase(&accf_bar[acc], (full_parity >> acc) & 1u, abort_flag, p.error_bits,
                           kDevErrEpilogueTimeout, lane))
        break;
      full_parity ^= 1u << acc;
      ptx::tcgen05_fence_after_sync();
      const uint32_t t_acc =
          tmem_base + (static_cast<uint32_t>(32 * quarter) << 16) + acc * Cfg::kAccCols + tok0;
      const int toks = min(kToks, t.rows - tok0);
      auto load16 = [&](int c, uint32_t(&v)[16], uint32_t(&u)[16]) {
        ptx::tmem_ld_32x32b_x16(t_acc + c, v);
        if (GATED) ptx::tmem_ld_32x32b_x16(t_acc + TN + c, u);
        ptx::tmem_ld_wait();
        ptx::reg_fence(v);
        if (GATED) ptx::reg_fence(u);
      };
#pragma unroll
      for (int c = 0; c < kToks; c += 16) {
        if (c >= toks) break;  // uniform over the warp
        uint32_t v[16], u[16];
        load16(c, v, u);
        float y[16], w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float a = __shfl_sync(0xffffffffu, as[c / 32], (c + i) & 31);
          y[i] = scaled(v[i], a, bs);
          if (GATED) w[i] = scaled(u[i], a, bs2);
          else y[i] = __fadd_rn(y[i], bias);
        }
        if constexpr (GATED) int8_gate(p.out_dtype, y, w, y);
        int8_store_rows(p, static_cast<int64_t>(t.row) + tok0 + c, n, y, toks - c);
      }
      ptx::tcgen05_fence_before_sync();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&acce_bar[acc]);
    }
  }
  ptx::tcgen05_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    ptx::tcgen05_fence_after_sync();
    ptx::tmem_dealloc(tmem_base, Cfg::kTmemColumns);
  }
}

}  // namespace nvfp4

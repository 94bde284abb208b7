// The int8 product on CTA pairs (cta_group::2), for segments of many rows (gated: and long K).
//
// A cluster of two CTAs computes 256 weight rows x up to pair_rows (at most 256) tokens per tile:
// each CTA loads its 128 weight rows and half of the tokens, so a token byte is brought to one SM
// only, and the even CTA issues MMAs of M = 256 that read both CTAs' shared memory and leave each
// CTA's 128 rows in its own TMEM. All 512 TMEM columns hold two accumulators, so a tile's
// epilogue runs under the next tile's MMAs.
//
// As in the single-CTA kernel, weight rows are TMEM lanes and tokens are columns. The MMA's N is
// the tile's own token count (a multiple of 32), and an expert's tiles share its rows equally:
// with tokens as the 256-row operand a ragged expert computed up to 255 rows of padding (64
// experts of 128 +- 11 rows, gated, N 1536, K 4096: 168 us against 149; of 64 +- 8 rows, N 4096,
// K 1536: 84 against 71). 8192 x 4096 x 7168 takes 151 us (3.2 POP/s, 0.97 of twice the measured
// bf16 rate), and 182 to 197 us from one GPU to the next in seconds-long runs under the power cap
// (0.89 to 0.96 of that rate there).
//
// Gated: a CTA's 128 rows are 64 of each weight set, so a channel's gate and up sums are 64
// lanes apart, in two epilogue warps. Per 16 tokens each of the two hands the other its scaled
// values of 8 tokens through shared memory and finishes the other 8.
//
// Barriers as in the NVFP4 pair kernel: full[s] on the even CTA takes the bytes of both CTAs'
// loads; the MMAs' commit frees a stage (and hands over an accumulator) in both CTAs; the
// epilogue warps of the pair release accumulators on the even CTA. Every wait is bounded.
#pragma once

#include "int8_gemm_kernel.cuh"

namespace nvfp4 {

constexpr int kInt8PairTokens = 256;

// WARPS: of the epilogue, 8 or 16 (a tile's epilogue is a chain of latencies: with 8 warps 256
// tokens took 3.9 us, gated 6.4, as long as the MMAs of K = 1300 and 2200; with 16 warps 3.6 and
// 4.7, but long K ran 3 % slower beside them).
template <bool GATED, int WARPS>
struct Int8PairConfig {
  static constexpr int kOutN = GATED ? 128 : 256;   // channels of a tile
  static constexpr int kWBox = GATED ? 64 : 128;    // weight rows per load
  static constexpr int kWBytes = 128 * kInt8StageK;
  static constexpr int kXBytes = kInt8PairTokens / 2 * kInt8StageK;
  static constexpr int kStageBytes = kWBytes + kXBytes;
  static constexpr int kThreads = 64 + 32 * WARPS;
  static constexpr int kStages = GATED && WARPS > 8 ? 5 : 6;
  // Exchange of two warps: two buffers of 2 directions x 8 tokens x 32 channels.
  static constexpr int kPairBytes = 2 * 2 * 8 * 32 * 4;
  static constexpr int kExchangeBytes = GATED ? WARPS / 2 * kPairBytes : 0;
  static constexpr int kSmemBytes =
      1024 + kStages * kStageBytes + kExchangeBytes + kInt8SegBytes + 512;
  static_assert(kSmemBytes <= 232448, "exceeds 227 KB of shared memory per CTA");
};

template <bool GATED, int WARPS>
__global__ void __launch_bounds__(64 + 32 * WARPS, 1)
    nvfp4_int8_gemm_pair_kernel(const __grid_constant__ CUtensorMap map_a,
                                const __grid_constant__ CUtensorMap map_a32,
                                const __grid_constant__ CUtensorMap map_b,
                                const __grid_constant__ CUtensorMap map_b2,
                                const __grid_constant__ Int8GemmParams p) {
  using Cfg = Int8PairConfig<GATED, WARPS>;
  constexpr int kStages = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* exchange = reinterpret_cast<float*>(smem + kStages * Cfg::kStageBytes);
  int32_t* seg_row = reinterpret_cast<int32_t*>(smem + kStages * Cfg::kStageBytes +
                                                Cfg::kExchangeBytes);
  int32_t* seg_cnt = seg_row + kInt8MaxExperts;
  int32_t* seg_end = seg_cnt + kInt8MaxExperts;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(seg_end + kInt8MaxExperts);
  uint64_t* empty_bar = full_bar + kStages;
  uint64_t* accf_bar = empty_bar + kStages;
  uint64_t* acce_bar = accf_bar + 2;
  uint64_t* drain_bar = acce_bar + 2;
  uint64_t* swap_bar = drain_bar + 1;  // one per two warps that exchange
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(swap_bar + WARPS / 2);
  volatile uint32_t* abort_flag = tmem_holder + 1;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const bool leader = rank == 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      ptx::mbar_init(&full_bar[s], 1);
      ptx::mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(&accf_bar[a], 1);
      ptx::mbar_init(&acce_bar[a], 2 * WARPS);
    }
    for (int i = 0; i < WARPS / 2; ++i) ptx::mbar_init(&swap_bar[i], 2);
    ptx::mbar_init(drain_bar, 1);
    *abort_flag = 0u;
    ptx::fence_mbarrier_init();
    ptx::tma_prefetch_desc(&map_a);
    ptx::tma_prefetch_desc(&map_b);
    if (GATED) ptx::tma_prefetch_desc(&map_b2);
  }
  if (warp == 1) {
    ptx::tmem_alloc_pair(tmem_holder, kTmemCols);
    ptx::tmem_relinquish_alloc_permit_pair();
  }
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int n_tiles = (p.n + Cfg::kOutN - 1) / Cfg::kOutN;
  const Int8PairRows tile_rows = {p.pair_rows, p.pair_inv};
  if (warp == 0)
    int8_stage_segments(p, tile_rows, n_tiles, seg_row, seg_cnt, seg_end, lane);
  ptx::tcgen05_fence_before_sync();
  ptx::cluster_sync_all();
  ptx::tcgen05_fence_after_sync();
  const uint32_t tmem_base = *tmem_holder;
  const int total = seg_end[p.num_experts - 1];
  const int first = static_cast<int>(blockIdx.x >> 1);
  const int step = static_cast<int>(gridDim.x >> 1);
  auto find = [&](int tile) {
    return int8_find_tile<true>(tile, tile_rows, n_tiles, p.num_experts, seg_row, seg_cnt, seg_end);
  };
  // N of a tile's MMAs: its tokens, 16 at a time from each CTA.
  auto mma_n = [](const Int8Tile& t) { return (t.rows + 31) / 32 * 32; };

  if (warp == 0) {
    if (ptx::elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      uint32_t issued = 0;
      bool ok = true;
      for (int tile = first; ok && tile < total; tile += step) {
        const Int8Tile t = find(tile);
        const int half = mma_n(t) / 2;  // this CTA's tokens
        const int xrow = t.row + rank * half;
        // In one box of pair_rows / 2 rows, or in boxes of 32 where half of them are enough.
        const int boxes = (half + 31) / 32;
        const bool small = 128 * boxes <= p.pair_rows;
        const uint32_t bytes =
            Cfg::kWBytes + (small ? 32 * boxes : p.pair_rows / 2) * kInt8StageK;
        const int wrow = t.expert * p.n + t.nt * Cfg::kOutN + rank * Cfg::kWBox;
        for (int kt = 0; kt < p.ktiles; ++kt) {
          if (!wait_phase(&empty_bar[stage], phase ^ 1u, abort_flag, p.error_bits,
                          kDevErrProducerTimeout)) {
            ok = false;
            break;
          }
          const uint32_t full = ptx::mapa_shared(ptx::smem_u32(&full_bar[stage]), 0);
          if (leader) ptx::mbar_arrive_expect_tx(&full_bar[stage], 2u * bytes);
          uint8_t* sW = smem + stage * Cfg::kStageBytes;
          uint8_t* sX = sW + Cfg::kWBytes;
          const int kx = kt * kInt8StageK;
          ptx::tma_load_2d_pair(sW, &map_b, full, kx, wrow);
          if (GATED)
            ptx::tma_load_2d_pair(sW + Cfg::kWBox * kInt8StageK, &map_b2, full, kx, wrow);
          if (small)
            for (int b = 0; b < boxes; ++b)
              ptx::tma_load_2d_pair(sX + 32 * b * kInt8StageK, &map_a32, full, kx, xrow + 32 * b);
          else
            ptx::tma_load_2d_pair(sX, &map_a, full, kx, xrow);
          ++issued;
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (leader) {
        // Every load of both CTAs completes on these barriers: the most recent fill of each
        // stage completes before the cluster may exit.
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
    }
  } else if (warp == 1) {
    if (leader && ptx::elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      uint32_t acc_parity = 0x3u;
      uint32_t local = 0;
      bool ok = true;
      for (int tile = first; ok && tile < total; tile += step, ++local) {
        const uint32_t idesc = ptx::make_idesc_i8(256, mma_n(find(tile)));
        const int acc = static_cast<int>(local & 1u);
        if (!wait_phase(&acce_bar[acc], (acc_parity >> acc) & 1u, abort_flag, p.error_bits,
                        kDevErrAccTimeout))
          break;
        acc_parity ^= 1u << acc;
        ptx::tcgen05_fence_after_sync();
        const uint32_t d_tmem = tmem_base + acc * kInt8PairTokens;
        for (int kt = 0; kt < p.ktiles; ++kt) {
          if (!wait_phase(&full_bar[stage], phase, abort_flag, p.error_bits, kDevErrMmaTimeout)) {
            ok = false;
            break;
          }
          ptx::tcgen05_fence_after_sync();
          const uint32_t sW = ptx::smem_u32(smem + stage * Cfg::kStageBytes);
          const uint64_t w_desc = ptx::make_sw128_kmajor_desc(sW);
          const uint64_t x_desc = ptx::make_sw128_kmajor_desc(sW + Cfg::kWBytes);
#pragma unroll
          for (int kb = 0; kb < 4; ++kb)
            ptx::mma_i8_pair(d_tmem, w_desc + 2 * kb, x_desc + 2 * kb, idesc,
                             (kt | kb) != 0 ? 1u : 0u);
          ptx::tcgen05_commit_pair_both(&empty_bar[stage]);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        ptx::tcgen05_commit_pair_both(&accf_bar[acc]);
      }
      ptx::tcgen05_commit_pair(drain_bar);
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
    constexpr int kStep = 4 * WARPS;  // tokens between a warp's chunks of 16
    constexpr int kChunks = kInt8PairTokens / kStep;
    const int turn = (warp - kEpilogueWarp0) / 4;  // its first chunk
    const bool up = GATED && quarter >= 2;
    const int group = GATED ? quarter & 1 : quarter;  // 32 channels of the CTA's
    float* swap = exchange + (2 * turn + group) * (Cfg::kPairBytes / 4) + lane;
    uint32_t full_parity = 0;
    uint32_t local = 0;
    uint32_t swaps = 0;
    bool ok = true;
    for (int tile = first; ok && tile < total; tile += step, ++local) {
      const Int8Tile t = find(tile);
      const int n = t.nt * Cfg::kOutN + rank * Cfg::kWBox + 32 * group + lane;
      const bool in = n < p.n;
      const int64_t chan = static_cast<int64_t>(t.expert) * p.n + n;
      const float bs = in ? __ldg((up ? p.b2_scale : p.b_scale) + chan) : 0.0f;
      const float bias = !GATED && in && p.bias != nullptr ? __ldg(p.bias + n) : 0.0f;
      // Token scales: lane l of as[j] holds that of token l % 16 of the warp's chunk 2 j + l / 16.
      float as[kChunks / 2];
#pragma unroll
      for (int j = 0; j < kChunks / 2; ++j) {
        const int tok = kStep * (2 * j + (lane >> 4)) + 16 * turn + (lane & 15);
        as[j] = tok < t.rows ? __ldg(p.a_scale + t.row + tok) : 0.0f;
      }
      const int acc = static_cast<int>(local & 1u);
      if (!warp_wait_phase(&accf_bar[acc], (full_parity >> acc) & 1u, abort_flag, p.error_bits,
                           kDevErrEpilogueTimeout, lane))
        break;
      full_parity ^= 1u << acc;
      ptx::tcgen05_fence_after_sync();
      const uint32_t t_acc = tmem_base + (static_cast<uint32_t>(32 * quarter) << 16) +
                             acc * kInt8PairTokens + 16 * turn;
#pragma unroll
      for (int j = 0; j < kChunks; ++j) {
        const int tok = kStep * j + 16 * turn;
        if (tok >= t.rows) break;  // uniform over the warp (and the two that exchange)
        uint32_t v[16];
        ptx::tmem_ld_32x32b_x16(t_acc + kStep * j, v);
        ptx::tmem_ld_wait();
        ptx::reg_fence(v);
        float y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          y[i] = __fmul_rn(__fmul_rn(__int2float_rn(static_cast<int32_t>(v[i])),
                                     __shfl_sync(0xffffffffu, as[j / 2], 16 * (j & 1) + i)),
                           bs);
        if (!GATED) {
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i] = __fadd_rn(y[i], bias);
          int8_store_rows(p, static_cast<int64_t>(t.row) + tok, n, y, t.rows - tok);
        } else {
          // The gate warp finishes tokens 0-7 of the chunk, the up warp tokens 8-15.
          float* to = swap + (2 * (swaps & 1u) + (up ? 1 : 0)) * 256;
          const float* from = swap + (2 * (swaps & 1u) + (up ? 0 : 1)) * 256;
#pragma unroll
          for (int i = 0; i < 8; ++i) to[32 * i] = up ? y[i] : y[8 + i];
          __syncwarp();
          uint64_t* bar = &swap_bar[2 * turn + group];
          if (lane == 0) ptx::mbar_arrive(bar);
          if (!warp_wait_phase(bar, swaps & 1u, abort_flag, p.error_bits, kDevErrEpilogueTimeout,
                               lane)) {
            ok = false;
            break;
          }
          ++swaps;
          float g[8], w[8], z[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float other = from[32 * i];
            g[i] = up ? other : y[i];
            w[i] = up ? y[8 + i] : other;
          }
          int8_gate(p.out_dtype, g, w, z);
          const int first8 = tok + (up ? 8 : 0);
          int8_store_rows(p, static_cast<int64_t>(t.row) + first8, n, z, t.rows - first8);
        }
      }
      ptx::tcgen05_fence_before_sync();
      __syncwarp();
      if (lane == 0)
        ptx::mbar_arrive_cluster(ptx::mapa_shared(ptx::smem_u32(&acce_bar[acc]), 0));
    }
  }
  // Both CTAs stay until every arrive, load and MMA that touches the other one is done.
  __syncwarp();
  ptx::tcgen05_fence_before_sync();
  ptx::cluster_sync_all();
  if (warp == 1) {
    ptx::tcgen05_fence_after_sync();
    ptx::tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

}  // namespace nvfp4

// Host entry points of the int8 operators: the row quantiser and its dispatching form
// (nvfp4_quantize_int8, nvfp4_moe_dispatch_int8) and the matrix product (nvfp4_int8_gemm).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>

#include "../../include/nvfp4_group_gemm.h"
#include "host_common.cuh"
#include "int8_gemm_kernel.cuh"
#include "int8_gemm_pair_kernel.cuh"
#include "int8_gemv_kernel.cuh"
#include "int8_quantize_kernel.cuh"

namespace nvfp4 {

// Why a product gave up on a wait or skipped a segment (kDevErr* bits): in the caller's word, or
// in this one of the device, which all callers without a word of their own share.
// A product needs no workspace: its tensor maps travel as kernel parameters and nothing else of
// one call is left for the next, so calls on any streams and in any graphs may overlap.
__device__ uint32_t g_int8_error_bits;

// Reads and clears an error word in one step: bits that another stream sets meanwhile are in this
// report or in the next.
__device__ uint32_t g_int8_taken_bits;
__global__ void nvfp4_int8_take_errors_kernel(uint32_t* word) {
  g_int8_taken_bits = atomicExch(word, 0u);
}

namespace {

struct Int8Device {
  std::once_flag once;
  cudaError_t status = cudaSuccess;
  uint32_t* error_bits = nullptr;
  uint32_t* taken_bits = nullptr;
  std::mutex taking;  // one check at a time uses taken_bits
};
Int8Device g_int8_dev[kMaxDevices];

template <int TN, bool GATED>
cudaError_t allow_smem() {
  return cudaFuncSetAttribute(nvfp4_int8_gemm_kernel<TN, GATED>,
                              cudaFuncAttributeMaxDynamicSharedMemorySize,
                              Int8Config<TN, GATED>::kSmemBytes);
}
template <bool GATED, int WARPS>
cudaError_t allow_smem_pair() {
  return cudaFuncSetAttribute(nvfp4_int8_gemm_pair_kernel<GATED, WARPS>,
                              cudaFuncAttributeMaxDynamicSharedMemorySize,
                              Int8PairConfig<GATED, WARPS>::kSmemBytes);
}

template <bool GATED>
cudaError_t allow_smem_all() {
  cudaError_t e = allow_smem<16, GATED>();
  if (e == cudaSuccess) e = allow_smem<32, GATED>();
  if (e == cudaSuccess) e = allow_smem<64, GATED>();
  if (e == cudaSuccess) e = allow_smem<128, GATED>();
  if (e == cudaSuccess) e = allow_smem_pair<GATED, 8>();
  if (e == cudaSuccess) e = allow_smem_pair<GATED, 16>();
  return e;
}

// Once per device. The look-up may load the module, which a stream capture under way on this
// thread would otherwise forbid.
void init_int8_device(Int8Device& d) {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  cudaThreadExchangeStreamCaptureMode(&mode);
  void* p = nullptr;
  cudaError_t e = cudaGetSymbolAddress(&p, g_int8_error_bits);
  d.error_bits = static_cast<uint32_t*>(p);
  if (e == cudaSuccess) e = cudaGetSymbolAddress(&p, g_int8_taken_bits);
  d.taken_bits = static_cast<uint32_t*>(p);
  if (e == cudaSuccess) e = allow_smem_all<false>();
  if (e == cudaSuccess) e = allow_smem_all<true>();
  d.status = e;
  cudaThreadExchangeStreamCaptureMode(&mode);
}

int int8_device(Int8Device** out, DeviceState** state) {
  const int st = current_device_state(state);
  if (st != NVFP4_OK) return st;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  Int8Device& d = g_int8_dev[dev];
  std::call_once(d.once, init_int8_device, std::ref(d));
  if (d.status != cudaSuccess) return cuda_fail(d.status, "int8 kernel set-up");
  *out = &d;
  return NVFP4_OK;
}

int int8_ktiles(const nvfp4_int8_product* g) { return (g->k + kInt8StageK - 1) / kInt8StageK; }

// What a product launches: one of NVFP4_INT8_*, the most tokens that a tile (or a pass over the
// weights) takes, the warps that share K or drain the accumulators, and the most tiles there can be.
struct Int8Plan {
  int kernel, tokens, warps;
  int64_t tiles;
};
Int8PairRows int8_pair_tile(int most) {
  return {most, static_cast<uint32_t>(((int64_t{1} << 32) + most / 32 - 1) / (most / 32))};
}

// int8 rows [rows, k], `ld` bytes apart, in boxes of 128 bytes x box_rows, 128-byte swizzle,
// zero fill past the last column and row.
bool int8_map(CUtensorMap* m, const void* addr, int64_t rows, int k, int64_t ld, int box_rows) {
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
  cuuint32_t box[2] = {kInt8StageK, static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  return encode_tiled_map(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(addr), dims,
                          strides, box, estr, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}

// Tensor maps of a product: tokens in boxes of `x_box` and of 32 rows, weights in boxes of `w_box`.
struct Int8Maps {
  CUtensorMap a, a32, b, b2;
};
bool int8_maps(const nvfp4_int8_product* g, int x_box, int w_box, Int8Maps* m) {
  const int64_t wrows = static_cast<int64_t>(g->num_experts) * g->n;
  if (!int8_map(&m->a, g->a, g->rows, g->k, g->lda, x_box) ||
      !int8_map(&m->a32, g->a, g->rows, g->k, g->lda, 32) ||
      !int8_map(&m->b, g->b, wrows, g->k, g->ldb, w_box))
    return false;
  if (g->b2 == nullptr) {
    m->b2 = m->b;
    return true;
  }
  return int8_map(&m->b2, g->b2, wrows, g->k, g->ldb, w_box);
}

// Most tiles of a launch: a persistent CTA's next tile number, the grid added to it, fits 31 bits.
constexpr int64_t kInt8MaxTiles = 0x7fffffff - 65536;

// The most tiles any segments can need: every row tile full, and one ragged tile each.
int64_t int8_max_tiles(const nvfp4_int8_product* g, int tile_rows, int tile_n) {
  return ((g->rows + tile_rows - 1) / tile_rows + (g->num_experts - 1)) *
         ((g->n + tile_n - 1) / tile_n);
}

template <int TN, bool GATED>
int launch_int8(const nvfp4_int8_product* g, const Int8GemmParams& p, int64_t tiles, int num_sms,
                cudaStream_t s) {
  using Cfg = Int8Config<TN, GATED>;
  Int8Maps m;
  if (!int8_maps(g, TN, 128, &m)) return fail(NVFP4_ERR_DRIVER, "cuTensorMapEncodeTiled failed");
  const cudaError_t e =
      launch_dependent(&nvfp4_int8_gemm_kernel<TN, GATED>, std::min<int64_t>(tiles, num_sms),
                       Cfg::kThreads, Cfg::kSmemBytes, s, m.a, m.a32, m.b, m.b2, p);
  return e == cudaSuccess ? NVFP4_OK : cuda_fail(e, "int8 product launch");
}

// Channels (R) of a group of warps: two, four where more tokens' codes have to be loaded for them
// (four tokens, N 2048, K 2048: 4.0 us against 4.6).
constexpr int int8_gemv_channels(int tokens, bool gated) { return tokens <= 2 || gated ? 2 : 4; }

template <int TB, int R, int KS, bool GATED>
int launch_int8_gemv(const nvfp4_int8_product* g, const Int8GemmParams& p, int num_sms,
                     cudaStream_t s) {
  Int8GemvParams q = {};
  q.p = p;
  q.a = static_cast<const uint8_t*>(g->a);
  q.b = static_cast<const uint8_t*>(g->b);
  q.b2 = static_cast<const uint8_t*>(g->b2);
  q.lda = g->lda;
  q.ldb = g->ldb;
  q.k = g->k;
  const int channels = kInt8GemvThreads / 32 / KS * R;  // of a block
  const int64_t blocks = (static_cast<int64_t>(g->n) + channels - 1) / channels * g->num_experts;
  const cudaError_t e =
      launch_dependent(&nvfp4_int8_gemv_kernel<TB, R, KS, GATED>,
                       std::min<int64_t>(blocks, num_sms * 4), kInt8GemvThreads, 0, s, q);
  return e == cudaSuccess ? NVFP4_OK : cuda_fail(e, "int8 product launch");
}

template <int TB, bool GATED>
int launch_int8_gemv_split(const nvfp4_int8_product* g, const Int8GemmParams& p, int warps,
                           int num_sms, cudaStream_t s) {
  constexpr int R = int8_gemv_channels(TB, GATED);
  if (warps == 8) return launch_int8_gemv<TB, R, 8, GATED>(g, p, num_sms, s);
  if (warps == 4) return launch_int8_gemv<TB, R, 4, GATED>(g, p, num_sms, s);
  // Eight tokens are taken where tiles are fewer than a ninth of the SMs and K is 2048 or more: two
  // warps always fit.
  if (TB == 8 || warps == 2) return launch_int8_gemv<TB, R, 2, GATED>(g, p, num_sms, s);
  if constexpr (TB < 8) return launch_int8_gemv<TB, R, 1, GATED>(g, p, num_sms, s);
}

template <bool GATED, int WARPS>
int launch_int8_pair(const nvfp4_int8_product* g, Int8GemmParams p, const Int8Plan& plan,
                     int clusters, cudaStream_t s) {
  using Cfg = Int8PairConfig<GATED, WARPS>;
  Int8Maps m;
  const Int8PairRows rows = int8_pair_tile(plan.tokens);
  p.pair_rows = rows.most;
  p.pair_inv = rows.inv;
  if (!int8_maps(g, plan.tokens / 2, Cfg::kWBox, &m))
    return fail(NVFP4_ERR_DRIVER, "cuTensorMapEncodeTiled failed");
  const cudaError_t e =
      launch_clusters(&nvfp4_int8_gemm_pair_kernel<GATED, WARPS>,
                      std::min<int64_t>(plan.tiles, clusters) * 2, 2, Cfg::kThreads,
                      Cfg::kSmemBytes, s, m.a, m.a32, m.b, m.b2, p);
  return e == cudaSuccess ? NVFP4_OK : cuda_fail(e, "int8 product launch");
}

// Most tokens of a CTA pair's tile, for one segment: those whose waves of tiles end soonest. In
// units of one token's MMAs over a stage, a stage takes the larger of its MMAs (tokens + 16) and
// its loads (96 + tokens / 2), and a tile no less than its epilogue (8 per token and 1024), which
// is not hidden behind the last tile. Fitted to 8192 x 4096 x 7168 (23.3 us a wave with 256
// tokens, 15.1 with 160, 13.7 with 128, 12.3 with 96) and to short K. Against 256 tokens: 2537 x
// 1806 x 7296 with 160 39.2 -> 30.2 us, 1536 x 1598 x 5253 with 160 22.3 -> 19.7, 700 x 4096 x
// 7168 with 192 24.0 -> 19.6, 1453 x 4224 x 577 with 192 12.6 -> 11.0; 2048 x 4096 x 4096 keeps
// 256 (26.8; 160 takes 27.6). Segments of several
// experts keep 256, as their rows are not known here (by the average, 64 experts of 1024 +- 32
// rows would lose 2 % and 64 of 128 +- 11 gain as much).
int int8_pair_rows(const nvfp4_int8_product* g, bool gated, int ktiles, int clusters) {
  const int kOutN = gated ? Int8PairConfig<true, 8>::kOutN : Int8PairConfig<false, 8>::kOutN;
  const int64_t n_tiles = (g->n + kOutN - 1) / kOutN;
  int64_t best_cost = 0;
  int best = 0;
  for (int most = kInt8PairTokens; most >= 96; most -= 32) {
    const int64_t row_tiles = (g->rows + most - 1) / most;
    const int64_t equal = ((g->rows + row_tiles - 1) / row_tiles + 31) / 32 * 32;
    const int64_t waves = (row_tiles * n_tiles + clusters - 1) / clusters;
    const int64_t stage = std::max(equal + 16, 96 + equal / 2);
    const int64_t cost = waves * std::max(ktiles * stage, 8 * equal + 1024) + 8 * equal;
    if (best != 0 && 13 * cost >= 12 * best_cost) continue;  // a clear gain only
    best_cost = cost;
    best = static_cast<int>(equal);
  }
  return best;
}

// Kernel and tile of a product, from the rows that the segments are expected to hold. Times in us
// on a B200, one launch of many, weights not in L2.
//
// Few tiles (fewer 128-channel tiles than SMs): a launch takes as long as one CTA's K loop, so
// the smallest token tile that still runs in one wave is taken. Dense, N 4096, K 7168: 256 rows
// 13.2 with tiles of 64, 16.5 with 128; 512 rows 16.9 with 128, 21.4 with 64.
//
// With at most 8 rows at once and few tiles the weights are streamed by all SMs without
// tiles (int8_gemv_kernel.cuh), against these tiles: one row 7.4 and 11.6 us (N 4096, K 7168),
// 13.7 and 15.6 (N 18432, K 4096); two rows 7.6 and 11.6, 14.1 and 15.4; four rows 10.2 and
// 11.5, 6.6 and 7.0 (N 7168, K 2048), but 17.5 and 15.5 (N 18432); eight rows 6.4 and 12.1 (N
// 1024, K 8192), 3.8 and 5.9 (N 2048, K 2048), but 16 and 11.5 (N 4096, K 7168). Of several experts
// with a row each on average (64 experts, N 128, K 4096, in passes of one and of two rows, and in
// tiles of 16): one token's 8 pairs 4.5, 4.5 and 9.6; 32 pairs, skewed, 8.1, 6.4 and 9.8; 64 pairs,
// even, 9.9, 8.5 and 10.1, skewed 16.7, 12.6 and 9.9 (gated, N 256: 33.7, 26.3 and 16.3).
//
// Many tiles: bound by the weights' bytes while an expert's rows fit one tile, so tiles are
// chosen to hold them with a quarter to spare (64 experts of 64 +- 8 rows, N 4096, K 1536:
// 70.5 with 128 tokens, 75.6 with 64); above 80 rows the MMAs decide and CTA pairs are faster
// (128 rows: 81 against 97 with 128-token tiles, gated N 1536, K 4096 155 against 159;
// 64 rows: 141 against 137). Gated sums of short K stay on single CTAs, whose epilogue has both
// sums of a channel in one lane (16 experts of 2048 rows, N 1024, single and pair: K 512 57 and
// 75 us, K 1024 65 and 78, K 1536 88 and 87, K 2048 110 and 102). Pairs take 16 epilogue warps up
// to the K at which a tile's MMAs hide what 8 of them do (8 and 16 warps: these experts, K 1536
// 104 and 88, K 2048 115 and 104, K 3000 146 and 149; plain N 2048, K 512 62.5 and 56, K 1024 69.6
// and 65.9, K 2048 100.7 and 102.8).
Int8Plan plan_int8(const nvfp4_int8_product* g, int num_sms, int clusters) {
  const bool gated = g->b2 != nullptr;
  const int ktiles = int8_ktiles(g);
  const int64_t expected = g->expected_rows > 0 ? std::min(g->expected_rows, g->rows) : g->rows;
  const int64_t active = std::min<int64_t>(g->num_experts, expected);  // experts with rows
  const int64_t rows = (expected + active - 1) / active;
  const int64_t n_tiles = (g->n + 127) / 128;
  const int64_t tiles = active * n_tiles;
  // Warps of a group (KS): as many as keep the warps within one wave (32 per SM) and leave each
  // two loads of 512 bytes of K.
  auto bytes = [&](int tokens) {
    const int r = int8_gemv_channels(tokens, gated);
    const int64_t groups = (static_cast<int64_t>(g->n) + r - 1) / r * active;
    int warps = 8;
    while (warps > 1 && (groups * warps > num_sms * 32 || g->k < 1024 * warps)) warps /= 2;
    return Int8Plan{NVFP4_INT8_BYTES, tokens, warps, 0};
  };
  // Experts' counts vary: twice the average. An average of one is one row each for a single token
  // (up to eight experts) only; more pairs crowd into popular experts, whose weights would be read
  // once per row.
  const int64_t at_once = g->num_experts == 1 ? rows
                          : rows > 1          ? 2 * rows
                          : expected <= 8     ? 1
                          : expected <= 32    ? 2 : 16;
  if (at_once == 1 && tiles < num_sms) return bytes(1);
  if (at_once == 2 && tiles < num_sms) return bytes(2);
  if (at_once <= 4 && (gated ? 4 : 2) * tiles < num_sms && g->k >= 1024) return bytes(4);
  if (at_once <= 8 && 9 * tiles < num_sms && g->k >= 2048) return bytes(8);
  auto one_wave = [&](int tn) { return active * ((rows + tn - 1) / tn) * n_tiles <= num_sms; };
  const bool many = !one_wave(128);
  if (many && rows > 80 && (!gated || ktiles > 10)) {
    const int tile_rows = g->seg_offsets == nullptr ? int8_pair_rows(g, gated, ktiles, clusters)
                                                    : kInt8PairTokens;
    return {NVFP4_INT8_PAIRS, tile_rows, ktiles <= (gated ? 18 : 8) ? 16 : 8,
            int8_max_tiles(g, tile_rows, gated ? 128 : 256)};
  }
  auto fits = [&](int tn) { return many ? 4 * tn >= 5 * rows : one_wave(tn); };
  int tn = 16;
  while (tn < 128 && !fits(tn)) tn *= 2;
  return {NVFP4_INT8_TILES, tn, tn >= 64 ? 8 : 4, int8_max_tiles(g, tn, 128)};
}

template <bool GATED>
int launch_plan_int8(const Int8Plan& plan, const nvfp4_int8_product* g, const Int8GemmParams& p,
                     const DeviceState& ds, cudaStream_t s) {
  const int sms = ds.num_sms;
  const int tokens = plan.tokens;
  if (plan.kernel == NVFP4_INT8_BYTES)
    return tokens == 1   ? launch_int8_gemv_split<1, GATED>(g, p, plan.warps, sms, s)
           : tokens == 2 ? launch_int8_gemv_split<2, GATED>(g, p, plan.warps, sms, s)
           : tokens == 4 ? launch_int8_gemv_split<4, GATED>(g, p, plan.warps, sms, s)
                         : launch_int8_gemv_split<8, GATED>(g, p, plan.warps, sms, s);
  if (plan.kernel == NVFP4_INT8_PAIRS)
    return plan.warps == 16 ? launch_int8_pair<GATED, 16>(g, p, plan, ds.pair_clusters, s)
                            : launch_int8_pair<GATED, 8>(g, p, plan, ds.pair_clusters, s);
  return tokens == 16   ? launch_int8<16, GATED>(g, p, plan.tiles, sms, s)
         : tokens == 32 ? launch_int8<32, GATED>(g, p, plan.tiles, sms, s)
         : tokens == 64 ? launch_int8<64, GATED>(g, p, plan.tiles, sms, s)
                        : launch_int8<128, GATED>(g, p, plan.tiles, sms, s);
}

template <typename T, int G, int V>
cudaError_t launch_quantize_rows(const Int8QuantParams& p, cudaStream_t s) {
  constexpr int kThreads = int8_quant_threads<G>();
  const int64_t per_block = kThreads / G;
  const int64_t rows = p.row_list != nullptr ? p.listed : p.rows;
  const int64_t blocks = (rows + per_block - 1) / per_block;
  return p.dest == nullptr
             ? launch_dependent(&nvfp4_quantize_int8_kernel<T, G, V, false>, blocks, kThreads, 0, s, p)
             : launch_dependent(&nvfp4_quantize_int8_kernel<T, G, V, true>, blocks, kThreads, 0, s, p);
}

// The fewest threads that hold a row at four chunks each, or at three where that is as many or
// fewer (1536 columns: 64 threads, all with columns).
template <typename T>
cudaError_t launch_quantize_int8(const Int8QuantParams& p, cudaStream_t s) {
  const int chunks = (p.cols + kInt8Chunk - 1) / kInt8Chunk;
  if (chunks <= 3 * 32) return launch_quantize_rows<T, 32, 3>(p, s);
  if (chunks <= 4 * 32) return launch_quantize_rows<T, 32, 4>(p, s);
  if (chunks <= 3 * 64) return launch_quantize_rows<T, 64, 3>(p, s);
  if (chunks <= 4 * 64) return launch_quantize_rows<T, 64, 4>(p, s);
  if (chunks <= 3 * 128) return launch_quantize_rows<T, 128, 3>(p, s);
  if (chunks <= 4 * 128) return launch_quantize_rows<T, 128, 4>(p, s);
  if (chunks <= 3 * 256) return launch_quantize_rows<T, 256, 3>(p, s);
  if (chunks <= 4 * 256) return launch_quantize_rows<T, 256, 4>(p, s);
  return launch_quantize_rows<T, 512, 4>(p, s);
}

int quantize_int8_impl(const void* x, int64_t rows, int cols, int64_t ld, int dtype,
                       const int32_t* row_list, int64_t listed, const int32_t* dest, int topk,
                       int64_t out_rows,
                       void* codes, int64_t codes_ld, float* scales, void* stream) {
  if (dtype != NVFP4_DTYPE_BF16 && dtype != NVFP4_DTYPE_FP16)
    return fail(NVFP4_ERR_INVALID_ARGUMENT, "dtype=%d (expected NVFP4_DTYPE_BF16 or _FP16)", dtype);
  if (rows < 0 || rows > 0x7fffffff || out_rows < 0 || out_rows > 0x7fffffff || cols <= 0 ||
      cols > NVFP4_MAX_ROW_COLUMNS)
    return fail(NVFP4_ERR_BAD_SHAPE, "rows=%lld out_rows=%lld cols=%d", static_cast<long long>(rows),
                static_cast<long long>(out_rows), cols);
  if (listed < 0 || listed > 0x7fffffff)
    return fail(NVFP4_ERR_BAD_SHAPE, "listed=%lld", static_cast<long long>(listed));
  if (rows == 0 || out_rows == 0 || (row_list != nullptr && listed == 0)) return NVFP4_OK;
  if (x == nullptr || codes == nullptr || scales == nullptr)
    return fail(NVFP4_ERR_NULL_POINTER, "x, codes or scales is NULL");
  if (ld < cols || codes_ld < cols)
    return fail(NVFP4_ERR_INVALID_ARGUMENT, "ld=%lld codes_ld=%lld too small for cols=%d",
                static_cast<long long>(ld), static_cast<long long>(codes_ld), cols);
  if (!aligned16(codes) || codes_ld % 16 != 0)
    return fail(NVFP4_ERR_MISALIGNED, "codes must be 16-byte aligned, codes_ld a multiple of 16");
  DeviceState* ds = nullptr;
  const int st = current_device_state(&ds);
  if (st != NVFP4_OK) return st;
  Int8QuantParams p = {};
  p.x = static_cast<const uint16_t*>(x);
  p.ld = ld;
  p.rows = static_cast<int32_t>(rows);
  p.cols = cols;
  const uintptr_t at = reinterpret_cast<uintptr_t>(x);
  p.align = at % 16 == 0 && ld % 8 == 0 ? 16 : at % 4 == 0 && ld % 2 == 0 ? 4 : 2;
  p.row_list = row_list;
  p.listed = static_cast<int32_t>(listed);
  p.dest = dest;
  p.topk = topk;
  p.out_rows = static_cast<int32_t>(out_rows);
  p.codes = static_cast<int8_t*>(codes);
  p.codes_ld = codes_ld;
  p.scales = scales;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == NVFP4_DTYPE_BF16
                            ? launch_quantize_int8<__nv_bfloat16>(p, s)
                            : launch_quantize_int8<__half>(p, s);
  return e == cudaSuccess ? NVFP4_OK : cuda_fail(e, "int8 quantiser launch");
}

// Checks of a product's record that need no GPU.
int check_product(const nvfp4_int8_product* g) {
  if (g == nullptr) return fail(NVFP4_ERR_NULL_POINTER, "product is NULL");
  if (g->num_experts <= 0 || g->num_experts > kInt8MaxExperts)
    return fail(NVFP4_ERR_INVALID_ARGUMENT, "num_experts=%d must be in [1, %d]", g->num_experts,
                kInt8MaxExperts);
  if (g->out_dtype != NVFP4_DTYPE_BF16 && g->out_dtype != NVFP4_DTYPE_FP16 &&
      g->out_dtype != NVFP4_DTYPE_FP32)
    return fail(NVFP4_ERR_INVALID_ARGUMENT,
                "out_dtype=%d (expected NVFP4_DTYPE_BF16, _FP16 or _FP32)", g->out_dtype);
  if (g->rows < 0 || g->rows > 0x7fffffff - 256 || g->n <= 0 || g->k <= 0 || g->k > kInt8MaxK ||
      static_cast<int64_t>(g->num_experts) * g->n > 0x7fffffff - 256)
    return fail(NVFP4_ERR_BAD_SHAPE, "rows=%lld n=%d k=%d (k in [1, %d])",
                static_cast<long long>(g->rows), g->n, g->k, kInt8MaxK);
  if ((g->seg_offsets == nullptr) != (g->seg_counts == nullptr))
    return fail(NVFP4_ERR_NULL_POINTER, "seg_offsets and seg_counts must both be given or NULL");
  if (g->seg_offsets == nullptr && g->num_experts != 1)
    return fail(NVFP4_ERR_NULL_POINTER, "several experts need seg_offsets and seg_counts");
  if ((g->b2 == nullptr) != (g->b2_scale == nullptr))
    return fail(NVFP4_ERR_NULL_POINTER, "b2 and b2_scale must both be given or NULL");
  const bool gated = g->b2 != nullptr;
  if (g->bias != nullptr && (gated || g->num_experts != 1))
    return fail(NVFP4_ERR_INVALID_ARGUMENT, "bias is for plain products of one weight matrix");
  if (g->lda < g->k || g->ldb < g->k || g->ldo < g->n)
    return fail(NVFP4_ERR_INVALID_ARGUMENT, "lda/ldb < k or ldo < n");
  if (g->rows == 0) return NVFP4_OK;
  if (g->a == nullptr || g->a_scale == nullptr || g->b == nullptr || g->b_scale == nullptr ||
      g->out == nullptr)
    return fail(NVFP4_ERR_NULL_POINTER, "an operand, scale or output is NULL");
  if (!aligned16(g->a) || !aligned16(g->b) || !aligned16(g->b2) || g->lda % 16 != 0 ||
      g->ldb % 16 != 0)
    return fail(NVFP4_ERR_MISALIGNED,
                "operands must be 16-byte aligned, lda and ldb multiples of 16 bytes");
  return NVFP4_OK;
}

}  // namespace
}  // namespace nvfp4

using namespace nvfp4;

extern "C" {

NVFP4_API int nvfp4_quantize_int8(const void* x, int64_t rows, int cols, int64_t ld, int dtype,
                                  const int32_t* row_list, int64_t listed, void* codes,
                                  int64_t codes_ld, float* scales, void* stream) {
  g_last_error.clear();
  return quantize_int8_impl(x, rows, cols, ld, dtype, row_list, row_list != nullptr ? listed : 0,
                            nullptr, 1, rows, codes, codes_ld, scales, stream);
}

NVFP4_API int nvfp4_moe_dispatch_int8(const void* x, int tokens, int cols, int64_t ld, int dtype,
                                      const int32_t* dest, int topk, int64_t rows, void* codes,
                                      int64_t codes_ld, float* scales, void* stream) {
  g_last_error.clear();
  if (topk <= 0 || static_cast<int64_t>(tokens) * topk > (int64_t{1} << 30))
    return fail(NVFP4_ERR_BAD_SHAPE, "tokens=%d topk=%d", tokens, topk);
  if (tokens > 0 && dest == nullptr) return fail(NVFP4_ERR_NULL_POINTER, "dest is NULL");
  return quantize_int8_impl(x, tokens, cols, ld, dtype, nullptr, 0, dest, topk, rows, codes, codes_ld,
                            scales, stream);
}

NVFP4_API int nvfp4_int8_plan(const nvfp4_int8_product* g, int num_sms, int cta_pairs,
                              nvfp4_int8_launch* launch) {
  g_last_error.clear();
  const int bad = check_product(g);
  if (bad != NVFP4_OK) return bad;
  if (launch == nullptr) return fail(NVFP4_ERR_NULL_POINTER, "launch is NULL");
  if (num_sms <= 0 || cta_pairs <= 0)
    return fail(NVFP4_ERR_INVALID_ARGUMENT, "num_sms=%d cta_pairs=%d", num_sms, cta_pairs);
  *launch = {};
  if (g->rows == 0) return NVFP4_OK;
  const Int8Plan plan = plan_int8(g, num_sms, cta_pairs);
  if (plan.tiles > kInt8MaxTiles) return fail(NVFP4_ERR_BAD_SHAPE, "too many tiles");
  launch->kernel = plan.kernel;
  launch->tokens = plan.tokens;
  launch->warps = plan.warps;
  launch->rows = std::min<int64_t>(g->rows, plan.tokens);
  if (plan.kernel == NVFP4_INT8_PAIRS)
    launch->rows = int8_equal_rows(static_cast<int>(g->rows),
                                   int8_pair_tile(plan.tokens).tiles(static_cast<int>(g->rows)));
  return NVFP4_OK;
}

NVFP4_API int nvfp4_int8_gemm(const nvfp4_int8_product* g, void* stream) {
  return nvfp4_int8_gemm_reporting(g, nullptr, stream);
}

NVFP4_API int nvfp4_int8_gemm_reporting(const nvfp4_int8_product* g, unsigned int* error_word,
                                        void* stream) {
  g_last_error.clear();
  const int bad = check_product(g);
  if (bad != NVFP4_OK || g->rows == 0) return bad;
  Int8Device* d = nullptr;
  DeviceState* ds = nullptr;
  const int st = int8_device(&d, &ds);
  if (st != NVFP4_OK) return st;
  Int8GemmParams p = {};
  p.a_scale = g->a_scale;
  p.b_scale = g->b_scale;
  p.b2_scale = g->b2_scale;
  p.bias = g->bias;
  p.out = g->out;
  p.ldo = g->ldo;
  p.seg_offsets = g->seg_offsets;
  p.seg_counts = g->seg_counts;
  p.error_bits = error_word != nullptr ? error_word : d->error_bits;
  p.rows = static_cast<int32_t>(g->rows);
  p.n = g->n;
  p.ktiles = int8_ktiles(g);
  p.num_experts = g->num_experts;
  p.out_dtype = g->out_dtype == NVFP4_DTYPE_BF16   ? kInt8OutBf16
                : g->out_dtype == NVFP4_DTYPE_FP16 ? kInt8OutFp16
                                                   : kInt8OutFp32;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Int8Plan plan = plan_int8(g, ds->num_sms, ds->pair_clusters);
  if (plan.tiles > kInt8MaxTiles) return fail(NVFP4_ERR_BAD_SHAPE, "too many tiles");
  return g->b2 != nullptr ? launch_plan_int8<true>(plan, g, p, *ds, s)
                          : launch_plan_int8<false>(plan, g, p, *ds, s);
}

NVFP4_API int nvfp4_int8_check(void* stream, unsigned int* device_error_bits) {
  return nvfp4_int8_check_word(nullptr, stream, device_error_bits);
}

NVFP4_API int nvfp4_int8_check_word(unsigned int* error_word, void* stream,
                                    unsigned int* device_error_bits) {
  g_last_error.clear();
  if (device_error_bits) *device_error_bits = 0;
  Int8Device* d = nullptr;
  DeviceState* ds = nullptr;
  const int st = int8_device(&d, &ds);
  if (st != NVFP4_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaStreamSynchronize(s);
  if (e != cudaSuccess) return cuda_fail(e, "cudaStreamSynchronize");
  uint32_t bits = 0;
  {
    std::lock_guard<std::mutex> lock(d->taking);
    nvfp4_int8_take_errors_kernel<<<1, 1, 0, s>>>(error_word != nullptr ? error_word
                                                                        : d->error_bits);
    e = cudaGetLastError();
    if (e == cudaSuccess)
      e = cudaMemcpyAsync(&bits, d->taken_bits, sizeof(bits), cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  }
  if (e != cudaSuccess) return cuda_fail(e, "read error word");
  if (device_error_bits) *device_error_bits = bits;
  if (bits & kDevErrTimeouts)
    return fail(NVFP4_ERR_DEVICE_TIMEOUT, "device error bits 0x%x", bits);
  if (bits != 0)
    return fail(NVFP4_ERR_BAD_SHAPE,
                "device error bits 0x%x: a device-side row segment was out of range (skipped)",
                bits);
  return NVFP4_OK;
}

}  // extern "C"

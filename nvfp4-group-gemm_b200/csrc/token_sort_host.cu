// Host entry points of the token sort and its gradients (nvfp4_moe_dispatch_tokens,
// nvfp4_moe_combine_tokens, nvfp4_moe_combine_tokens_backward).
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/nvfp4_group_gemm.h"
#include "host_common.cuh"
#include "token_sort_kernels.cuh"

namespace nvfp4 {
namespace {

int element_size(int dtype) {
  return dtype == NVFP4_DTYPE_FP32 ? 4 : dtype == NVFP4_DTYPE_BF16 || dtype == NVFP4_DTYPE_FP16 ? 2 : 0;
}

// Whether rows of `cols` elements move in pieces of `bytes`.
bool rows_in_pieces(const TokenSortParams& p, int es, int bytes) {
  auto starts = [&](const void* at, int64_t ld) {
    return reinterpret_cast<uintptr_t>(at) % bytes == 0 && ld * es % bytes == 0;
  };
  return static_cast<int64_t>(p.cols) * es % bytes == 0 && starts(p.x, p.ldx) &&
         starts(p.y, p.ldy) && starts(p.out, p.ldo);
}

int check_sizes(int tokens, int topk, int cols, int64_t rows, int dtype, const void* dest) {
  if (element_size(dtype) == 0)
    return fail(NVFP4_ERR_INVALID_ARGUMENT, "dtype=%d (expected NVFP4_DTYPE_BF16, _FP16 or _FP32)",
                dtype);
  // The kernels' column counters step past the last column by as much as a block's span.
  if (tokens < 0 || topk <= 0 || cols <= 0 || cols > NVFP4_MAX_ROW_COLUMNS || rows < 0 ||
      rows > 0x7fffffff - 32)
    return fail(NVFP4_ERR_BAD_SHAPE, "tokens=%d topk=%d cols=%d rows=%lld", tokens, topk, cols,
                static_cast<long long>(rows));
  if (static_cast<int64_t>(tokens) * topk > (int64_t{1} << 30))
    return fail(NVFP4_ERR_BAD_SHAPE, "too many pairs");
  if (tokens > 0 && dest == nullptr) return fail(NVFP4_ERR_NULL_POINTER, "dest is NULL");
  return NVFP4_OK;
}

enum class SortOp { kDispatch, kCombine, kBackward };

template <typename T, int VEC>
cudaError_t launch(SortOp op, const TokenSortParams& p, int num_sms, cudaStream_t s) {
  const int64_t groups =
      p.out != nullptr ? (static_cast<int64_t>(p.rows) + kPadRows - 1) / kPadRows : 0;
  if (op == SortOp::kBackward)
    return launch_dependent(&nvfp4_combine_tokens_backward_kernel<T, VEC>, groups + p.tokens,
                            kTokenThreads, 0, s, p);
  if (op == SortOp::kDispatch) {
    const int warps = kSortThreads / 32;
    const int64_t chunks = (p.cols + 32 * VEC * kSortPieces - 1) / (32 * VEC * kSortPieces);
    return launch_dependent(&nvfp4_dispatch_tokens_kernel<T, VEC>,
                            ((groups + p.tokens) * chunks + warps - 1) / warps, kSortThreads, 0, s,
                            p);
  }
  // A whole row per block where the tokens alone fill the GPU, parts of it where they do not.
  const int span = kTokenThreads * VEC * kTokenPieces;
  const int64_t chunks = (p.cols + span - 1) / span;
  const int64_t parts = std::min<int64_t>(
      chunks, std::max<int64_t>(1, static_cast<int64_t>(num_sms) * 8 / p.tokens));
  return launch_dependent(&nvfp4_combine_tokens_kernel<T, VEC>, p.tokens * parts, kTokenThreads, 0, s,
                          p, static_cast<int>(parts));
}

template <typename T>
cudaError_t by_piece(SortOp op, int bytes, const TokenSortParams& p, int num_sms, cudaStream_t s) {
  if (bytes == 16) return launch<T, 16 / sizeof(T)>(op, p, num_sms, s);
  if (bytes == 8) return launch<T, 8 / sizeof(T)>(op, p, num_sms, s);
  if constexpr (sizeof(T) == 2)
    if (bytes == 4) return launch<T, 2>(op, p, num_sms, s);
  return launch<T, 1>(op, p, num_sms, s);
}

int run(SortOp op, int dtype, const TokenSortParams& p, void* stream) {
  DeviceState* ds = nullptr;
  const int st = current_device_state(&ds);
  if (st != NVFP4_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int es = element_size(dtype);
  const int bytes = rows_in_pieces(p, es, 16) ? 16
                    : rows_in_pieces(p, es, 8) ? 8
                    : rows_in_pieces(p, es, 4) ? 4 : 2;
  const cudaError_t e = dtype == NVFP4_DTYPE_FP32   ? by_piece<float>(op, bytes, p, ds->num_sms, s)
                        : dtype == NVFP4_DTYPE_FP16 ? by_piece<__half>(op, bytes, p, ds->num_sms, s)
                                                    : by_piece<__nv_bfloat16>(op, bytes, p, ds->num_sms, s);
  return e == cudaSuccess ? NVFP4_OK : cuda_fail(e, "token sort launch");
}

}  // namespace
}  // namespace nvfp4

using namespace nvfp4;

extern "C" {

NVFP4_API int nvfp4_moe_dispatch_tokens(const void* x, int64_t ldx, int dtype, const int32_t* dest,
                                        const int32_t* src_rows, int tokens, int topk, int cols,
                                        int64_t rows, void* y, int64_t ldy, void* stream) {
  g_last_error.clear();
  const int st = check_sizes(tokens, topk, cols, rows, dtype, dest);
  if (st != NVFP4_OK) return st;
  if (rows == 0) return NVFP4_OK;
  if ((tokens > 0 && x == nullptr) || src_rows == nullptr || y == nullptr)
    return fail(NVFP4_ERR_NULL_POINTER, "x, src_rows or y is NULL");
  if (ldx < cols || ldy < cols) return fail(NVFP4_ERR_INVALID_ARGUMENT, "ldx/ldy < cols");
  TokenSortParams p = {};
  p.x = x; p.ldx = ldx; p.out = y; p.ldo = ldy; p.dest = dest; p.src_rows = src_rows;
  p.tokens = tokens; p.topk = topk; p.cols = cols; p.rows = static_cast<int32_t>(rows);
  return run(SortOp::kDispatch, dtype, p, stream);
}

NVFP4_API int nvfp4_moe_combine_tokens(const void* y, int64_t ldy, int dtype, const int32_t* dest,
                                       const float* weights, int tokens, int topk, int cols,
                                       int64_t rows, void* out, int64_t ldo, void* stream) {
  g_last_error.clear();
  const int st = check_sizes(tokens, topk, cols, rows, dtype, dest);
  if (st != NVFP4_OK) return st;
  if (tokens == 0) return NVFP4_OK;
  if ((rows > 0 && y == nullptr) || out == nullptr)
    return fail(NVFP4_ERR_NULL_POINTER, "y or out is NULL");
  if (ldy < cols || ldo < cols) return fail(NVFP4_ERR_INVALID_ARGUMENT, "ldy/ldo < cols");
  TokenSortParams p = {};
  p.x = y; p.ldx = ldy; p.out = out; p.ldo = ldo; p.dest = dest; p.weights = weights;
  p.tokens = tokens; p.topk = topk; p.cols = cols; p.rows = static_cast<int32_t>(rows);
  return run(SortOp::kCombine, dtype, p, stream);
}

NVFP4_API int nvfp4_moe_combine_tokens_backward(const void* grad_out, int64_t ldg, const void* y,
                                                int64_t ldy, int dtype, const int32_t* dest,
                                                const int32_t* src_rows, const float* weights,
                                                int tokens, int topk, int cols, int64_t rows,
                                                void* grad_y, int64_t ldo, float* grad_w,
                                                void* stream) {
  g_last_error.clear();
  const int st = check_sizes(tokens, topk, cols, rows, dtype, dest);
  if (st != NVFP4_OK) return st;
  if (grad_y == nullptr && grad_w == nullptr) return NVFP4_OK;
  if (tokens == 0 && rows == 0) return NVFP4_OK;
  if ((tokens > 0 && grad_out == nullptr) || (grad_w != nullptr && rows > 0 && y == nullptr) ||
      (grad_y != nullptr && rows > 0 && src_rows == nullptr))
    return fail(NVFP4_ERR_NULL_POINTER, "grad_out, y or src_rows is NULL");
  if (ldg < cols || (grad_w != nullptr && ldy < cols) || (grad_y != nullptr && ldo < cols))
    return fail(NVFP4_ERR_INVALID_ARGUMENT, "ldg/ldy/ldo < cols");
  TokenSortParams p = {};
  p.x = grad_out; p.ldx = ldg; p.dest = dest; p.src_rows = src_rows; p.weights = weights;
  if (grad_w != nullptr) { p.y = y; p.ldy = ldy; p.grad_w = grad_w; }
  if (grad_y != nullptr) { p.out = grad_y; p.ldo = ldo; }
  p.tokens = tokens; p.topk = topk; p.cols = cols; p.rows = static_cast<int32_t>(rows);
  return run(SortOp::kBackward, dtype, p, stream);
}

}  // extern "C"

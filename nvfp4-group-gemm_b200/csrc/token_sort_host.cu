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

bool vector_rows(const void* p, int64_t ld, int es) {
  return p == nullptr || (aligned16(p) && ld * es % 16 == 0);
}

int check_sizes(int tokens, int topk, int cols, int64_t rows, int dtype, const void* dest) {
  if (element_size(dtype) == 0)
    return fail(NVFP4_ERR_INVALID_ARGUMENT, "dtype=%d (expected NVFP4_DTYPE_BF16, _FP16 or _FP32)",
                dtype);
  if (tokens < 0 || topk <= 0 || cols <= 0 || rows < 0 || rows > 0x7fffffff - 32)
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

int run(SortOp op, int dtype, const TokenSortParams& p, void* stream) {
  DeviceState* ds = nullptr;
  const int st = current_device_state(&ds);
  if (st != NVFP4_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int es = element_size(dtype);
  const bool vec = static_cast<int64_t>(p.cols) * es % 16 == 0 && vector_rows(p.x, p.ldx, es) &&
                   vector_rows(p.y, p.ldy, es) && vector_rows(p.out, p.ldo, es);
  cudaError_t e;
  if (dtype == NVFP4_DTYPE_FP32)
    e = vec ? launch<float, 4>(op, p, ds->num_sms, s) : launch<float, 1>(op, p, ds->num_sms, s);
  else if (dtype == NVFP4_DTYPE_FP16)
    e = vec ? launch<__half, 8>(op, p, ds->num_sms, s) : launch<__half, 1>(op, p, ds->num_sms, s);
  else
    e = vec ? launch<__nv_bfloat16, 8>(op, p, ds->num_sms, s) : launch<__nv_bfloat16, 1>(op, p, ds->num_sms, s);
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

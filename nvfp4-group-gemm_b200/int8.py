"""int8 operators: activations to codes with a scale per token, and the matrix product of
codes with scales per token and per channel, dense or over the rows of every expert.

    codes, scale = quantize_int8(x)                      # int8 [M, K], fp32 [M]
    y = int8_gemm(codes, scale, w_codes, w_scale)        # bf16 [M, N]
    y = int8_gemm_segments(a, a_scale, w, w_scale, offsets, counts)   # experts' rows of a slab

Code matrices are int8 with unit inner stride and rows a multiple of 16 bytes apart, which is
how :func:`quantize_int8` allocates them for any number of columns. The products need no
workspace and keep nothing between calls but their errors, so calls may overlap on any streams
and be captured in any CUDA graphs. Errors go to one word per GPU, which all calls share, or to
an ``error_word`` of the caller's. The reference has no 8-bit form of its product.
"""
from __future__ import annotations

import ctypes

import torch

from . import _native

_IN_DTYPES = {torch.bfloat16: _native.DTYPE_BF16, torch.float16: _native.DTYPE_FP16}
_OUT_DTYPES = {**_IN_DTYPES, torch.float32: _native.DTYPE_FP32}


def _launch_on(tensors, stream: torch.cuda.Stream | None) -> tuple:
    """``(raw stream, context)`` of a call on ``tensors`` (None entries left out; the first gives
    the device, the others must be on it). The context, None where nothing has to change, makes
    device and stream current, so that what is allocated inside belongs to the stream. Tensors
    used on another stream than the current one are recorded there, so that freeing them early
    does not hand their memory out while the call runs."""
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != index or index < 0:
            raise ValueError("all tensors must be CUDA tensors on one device")
    raw = torch._C._cuda_getCurrentRawStream(index)
    if stream is None or (stream.cuda_stream == raw and stream.device.index == index):
        return raw, None if torch._C._cuda_getDevice() == index else torch.cuda.device(index)
    if stream.device.index != index:
        raise ValueError(f"stream is on {stream.device}, the tensors are on cuda:{index}")
    for t in tensors:
        if t is not None:
            t.record_stream(stream)
    return stream.cuda_stream, torch.cuda.stream(stream)


def _within(where, call, *args):
    """``call(*args)`` inside the context of :func:`_launch_on`."""
    if where is None:
        return call(*args)
    with where:
        return call(*args)


def _row_stride(t: torch.Tensor) -> int:
    """Elements between rows (a single row has none of its own)."""
    return int(t.stride(0)) if t.shape[0] > 1 else max(int(t.stride(0)), int(t.shape[1]))


def _unit_inner(t: torch.Tensor) -> bool:
    return t.stride(-1) == 1 or t.shape[-1] == 1


def _check_activations(x: torch.Tensor) -> None:
    if not isinstance(x, torch.Tensor):
        raise ValueError("x must be a CUDA tensor")
    if x.dtype not in _IN_DTYPES:
        raise ValueError(f"x must be bfloat16 or float16, got {x.dtype}")
    if x.dim() != 2 or x.shape[1] < 1 or not _unit_inner(x):
        raise ValueError("x must be 2-D with unit stride along the last dimension")
    if x.shape[1] > _native.MAX_ROW_COLUMNS:
        raise ValueError(f"x has {x.shape[1]} columns, at most {_native.MAX_ROW_COLUMNS}")
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor")
    if x.shape[0] > 1 and x.stride(0) < x.shape[1]:
        raise ValueError("rows of x must not overlap (expanded tensors: call .contiguous())")


def _codes_stride(t: torch.Tensor, name: str) -> int:
    """Bytes between the rows of an int8 code matrix [rows, k] (checked)."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int8 or t.dim() != 2:
        raise ValueError(f"{name} must be a 2-D CUDA int8 tensor")
    rows, cols = t.shape
    ld, inner = t.stride()
    if cols < 1 or (inner != 1 and cols != 1):
        raise ValueError(f"{name} must have unit stride along the last dimension")
    if rows <= 1:
        ld = (cols + 15) // 16 * 16
    if ld % 16 or ld < cols or t.data_ptr() % 16:
        raise ValueError(f"rows of {name} must start on 16-byte boundaries "
                         "(quantize_int8 allocates them so)")
    return ld


def _check_word(t) -> None:
    if t is not None and (not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.numel() != 1):
        raise ValueError("error_word must be a CUDA int32 tensor of one entry (zero at first)")


def _check_scale(t: torch.Tensor, shape: tuple, name: str) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.shape != shape or \
            not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous CUDA float32 tensor of shape {list(shape)}")


def empty_codes(rows: int, cols: int, device) -> torch.Tensor:
    """Uninitialised int8 codes [rows, cols] whose rows are a multiple of 16 bytes apart."""
    ld = (cols + 15) // 16 * 16
    return torch.empty((rows, ld), dtype=torch.int8, device=device)[:, :cols]


def _check_code_outputs(codes, scales, rows: int, cols: int) -> None:
    if codes is not None:
        _codes_stride(codes, "codes")
        if tuple(codes.shape) != (rows, cols):
            raise ValueError(f"codes must be [{rows}, {cols}]")
    if scales is not None:
        _check_scale(scales, (rows,), "scales")


def quantize_int8(x: torch.Tensor, codes: torch.Tensor | None = None,
                  scales: torch.Tensor | None = None, row_list: torch.Tensor | None = None,
                  stream: torch.cuda.Stream | None = None) -> tuple:
    """Quantise the rows of ``x`` (bf16 or fp16 [rows, cols]) to int8: ``(codes, scales)`` with
    ``scales[r] = max|x[r]| / 127`` and ``codes = 127 * x / max|x[r]|`` rounded to nearest, ties
    to even (of the exact quotient), so ``x ~= codes * scales[:, None]``.

    A row of zeros gets scale 0; a row that holds an infinity or a NaN gets scale NaN and zero
    codes. ``row_list`` (1-D int32, e.g. a routing's ``dest`` for a dispatched buffer): only these
    rows are quantised, each in its place (entries outside ``[0, rows)`` are none); the others are
    neither read nor written. ``codes`` / ``scales`` write in place.
    """
    _check_activations(x)
    rows, cols = int(x.shape[0]), int(x.shape[1])
    _check_code_outputs(codes, scales, rows, cols)
    if row_list is not None and (row_list.dtype != torch.int32 or row_list.dim() != 1 or
                                 not row_list.is_contiguous()):
        raise ValueError("row_list must be a contiguous 1-D int32 tensor")
    raw, where = _launch_on((x, codes, scales, row_list), stream)
    return _within(where, _quantize, x, rows, cols, codes, scales, row_list, raw)


def _quantize(x, rows, cols, codes, scales, row_list, raw):
    if codes is None:
        codes = empty_codes(rows, cols, x.device)
    if scales is None:
        scales = x.new_empty(rows, dtype=torch.float32)
    listed = 0
    if row_list is not None:
        listed = row_list.numel()
        if listed == 0:
            return codes, scales
    lib = _native.load_library()
    _native.check(lib.nvfp4_quantize_int8(
        x.data_ptr(), rows, cols, _row_stride(x), _IN_DTYPES[x.dtype],
        row_list.data_ptr() if listed else None, listed, codes.data_ptr(),
        _codes_stride(codes, "codes"), scales.data_ptr(), raw), lib)
    return codes, scales


def _check_out(out, out_dtype, rows: int, n: int) -> None:
    if out is None:
        return
    if not isinstance(out, torch.Tensor) or not out.is_cuda or out.dtype not in _OUT_DTYPES or \
            tuple(out.shape) != (rows, n) or not _unit_inner(out) or \
            (rows > 1 and out.stride(0) < n):
        raise ValueError(f"out must be a CUDA bf16, fp16 or fp32 tensor [{rows}, {n}] with unit "
                         "inner stride")
    if out_dtype is not None and out.dtype != out_dtype:
        raise ValueError(f"out is {out.dtype}, out_dtype is {out_dtype}")


def _product(a, lda, a_scale, b, ldb, b_scale, b2, b2_scale, bias, out, out_dtype, n, k, experts,
             offsets, counts, expected_rows, error_word, raw):
    rows = a.shape[0]
    if out is None:
        dtype = torch.bfloat16 if out_dtype is None else out_dtype
        if dtype not in _OUT_DTYPES:
            raise ValueError(f"out_dtype must be bfloat16, float16 or float32, got {dtype}")
        out, ldo = a.new_empty((rows, n), dtype=dtype), n
    else:
        dtype, ldo = out.dtype, _row_stride(out)
    product = _native.pack_int8_product(
        a.data_ptr(), b.data_ptr(), b2.data_ptr() if b2 is not None else 0, a_scale.data_ptr(),
        b_scale.data_ptr(), b2_scale.data_ptr() if b2 is not None else 0,
        bias.data_ptr() if bias is not None else 0, out.data_ptr(),
        offsets.data_ptr() if offsets is not None else 0,
        counts.data_ptr() if counts is not None else 0, rows, lda, ldb, ldo, expected_rows, n, k,
        experts, _OUT_DTYPES[dtype])
    lib = _native.load_library()
    word = error_word.data_ptr() if error_word is not None else None
    _native.check(lib.nvfp4_int8_gemm_reporting(product, word, raw), lib)
    return out


def int8_gemm(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
              bias: torch.Tensor | None = None, out: torch.Tensor | None = None,
              out_dtype: torch.dtype | None = None, stream: torch.cuda.Stream | None = None,
              error_word: torch.Tensor | None = None) -> torch.Tensor:
    """``out[m, n] = a_scale[m] * b_scale[n] * sum_k a[m, k] * b[n, k] (+ bias[n])``.

    ``a`` int8 [M, K] (codes of tokens), ``b`` int8 [N, K] (codes of weight rows), scales fp32
    [M] and [N], ``bias`` fp32 [N]. The sums are exact; they are multiplied with ``a_scale``, then
    with ``b_scale`` in fp32 (a product past its range is an infinity), and the result is rounded
    once, to ``out_dtype`` (bf16 by default; fp16, fp32). Any M, N and K up to 131071; ``out`` may have
    any row stride and alignment. ``error_word``: where a wait that timed out is reported (see
    :func:`check_int8_errors`).
    """
    _check_word(error_word)
    lda, ldb = _codes_stride(a, "a"), _codes_stride(b, "b")
    m, k = a.shape
    n = b.shape[0]
    if b.shape[1] != k or n < 1:
        raise ValueError(f"b must be [N >= 1, {k}], got {list(b.shape)}")
    if n > _native.INT8_MAX_CHANNELS:
        raise ValueError(f"b has {n} channels, at most {_native.INT8_MAX_CHANNELS}")
    if k > _native.INT8_MAX_K:
        raise ValueError(f"K={k} is above {_native.INT8_MAX_K}: sums could leave int32")
    _check_scale(a_scale, (m,), "a_scale")
    _check_scale(b_scale, (n,), "b_scale")
    if bias is not None:
        _check_scale(bias, (n,), "bias")
    _check_out(out, out_dtype, m, n)
    raw, where = _launch_on((a, a_scale, b, b_scale, bias, out, error_word), stream)
    return _within(where, _product, a, lda, a_scale, b, ldb, b_scale, None, None, bias, out,
                   out_dtype, n, k, 1, None, None, 0, error_word, raw)


def _expert_weights(b: torch.Tensor, b_scale: torch.Tensor, k: int, name: str) -> int:
    """Checks expert weights [E, N, k] (experts N rows apart) and their scales; the row stride."""
    if not isinstance(b, torch.Tensor) or b.dim() != 3 or b.shape[0] < 1 or b.shape[1] < 1 or \
            b.shape[2] != k:
        raise ValueError(f"{name} must be an int8 tensor [experts, N, {k}]")
    experts, n = int(b.shape[0]), int(b.shape[1])
    if experts > 1 and n > 1 and b.stride(0) != n * b.stride(1):
        raise ValueError(f"the experts of {name} must follow one another ([experts * N, K] rows)")
    _check_scale(b_scale, (experts, n), f"{name}_scale")
    if n > 1:
        return _codes_stride(b[0], name)
    rows = b[:, 0]
    return _codes_stride(rows, name)


def int8_gemm_segments(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor,
                       b_scale: torch.Tensor, seg_offsets: torch.Tensor,
                       seg_counts: torch.Tensor, b2: torch.Tensor | None = None,
                       b2_scale: torch.Tensor | None = None, out: torch.Tensor | None = None,
                       out_dtype: torch.dtype | None = None, expected_rows: int = 0,
                       stream: torch.cuda.Stream | None = None,
                       error_word: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`int8_gemm` over row segments of one slab, read on the GPU.

    ``a`` int8 [R, K] with scales [R]; expert e multiplies rows ``[seg_offsets[e],
    seg_offsets[e] + seg_counts[e])`` by its weights ``b[e]`` (int8 [E, N, K], scales [E, N])
    into the same rows of ``out`` [R, N]. With ``b2`` / ``b2_scale`` (same shapes) the result is
    ``silu(product with b) * (product with b2)``, fp32 until its one rounding (with the fast
    exponential and division where that is to 16 bits). ``seg_offsets``
    and ``seg_counts`` are int32 CUDA tensors (a routing's offsets and counts): nothing is read
    back, so the call can be captured in a CUDA graph. Segments may start anywhere; rows outside
    all of them are left as they were (undefined where ``out`` is allocated here). A segment
    outside the slab is skipped and :func:`check_int8_errors` raises; segments that share rows
    are not supported (their rows hold either result; segments past the slab's number of rows in
    all may be skipped and reported). ``expected_rows`` (the host's estimate of all segments'
    rows, e.g. tokens x top-k) picks the tile shape only. ``error_word`` (int32 CUDA tensor of one
    entry, zero at first; it has to outlive the call and any graph that holds it) takes the reports
    in place of the device's word, which all other calls share.
    """
    _check_word(error_word)
    lda = _codes_stride(a, "a")
    rows, k = int(a.shape[0]), int(a.shape[1])
    if k > _native.INT8_MAX_K:
        raise ValueError(f"K={k} is above {_native.INT8_MAX_K}: sums could leave int32")
    ldb = _expert_weights(b, b_scale, k, "b")
    experts, n = int(b.shape[0]), int(b.shape[1])
    if experts > _native.INT8_MAX_EXPERTS:
        raise ValueError(f"at most {_native.INT8_MAX_EXPERTS} experts")
    if experts * n > _native.INT8_MAX_CHANNELS:
        raise ValueError(f"b has {experts * n} channels, at most {_native.INT8_MAX_CHANNELS}")
    if (b2 is None) != (b2_scale is None):
        raise ValueError("b2 and b2_scale must both be given")
    if b2 is not None:
        if tuple(b2.shape) != tuple(b.shape) or _expert_weights(b2, b2_scale, k, "b2") != ldb:
            raise ValueError("b2 must have the shape and row stride of b")
    _check_scale(a_scale, (rows,), "a_scale")
    for name, t in (("seg_offsets", seg_offsets), ("seg_counts", seg_counts)):
        if t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous() or t.numel() < experts:
            raise ValueError(f"{name} must be a contiguous CUDA int32 tensor of >= {experts} entries")
    _check_out(out, out_dtype, rows, n)
    raw, where = _launch_on((a, a_scale, b, b_scale, b2, b2_scale, seg_offsets, seg_counts, out,
                             error_word), stream)
    return _within(where, _product, a, lda, a_scale, b, ldb, b_scale, b2, b2_scale, None, out,
                   out_dtype, n, k, experts, seg_offsets, seg_counts, int(expected_rows),
                   error_word, raw)


def check_int8_errors(device: torch.device | int | None = None,
                      stream: torch.cuda.Stream | None = None,
                      error_word: torch.Tensor | None = None) -> int:
    """Synchronise ``stream`` (the current one by default) and read and clear, in one step, the
    error bits of the int8 products in ``error_word``: raises Nvfp4Error when a segment was out of
    range or a wait timed out, else returns 0. Without ``error_word``: the device's, of all calls
    that were given none (whoever made them)."""
    _check_word(error_word)
    if error_word is not None:
        if not error_word.is_cuda:
            raise ValueError("error_word must be on a CUDA device")
        device = error_word.device
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else \
        torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
    s = stream or torch.cuda.current_stream(dev)
    lib = _native.load_library()
    bits = ctypes.c_uint(0)
    with torch.cuda.device(dev):
        _native.check(lib.nvfp4_int8_check_word(
            error_word.data_ptr() if error_word is not None else None, s.cuda_stream,
            ctypes.byref(bits)), lib)
    return int(bits.value)

"""What the int8 operators and the token sort refuse, before anything is launched (CPU only)."""
from __future__ import annotations

import ctypes

import pytest
import torch


def _product(N, **kw):
    p = N.Int8Product()
    base = dict(a=0x10000, b=0x20000, a_scale=0x30000, b_scale=0x40000, out=0x50000, rows=16, n=64,
                k=100, lda=112, ldb=112, ldo=64, num_experts=1, out_dtype=0)
    base.update(kw)
    for k, v in base.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,status", [
    (dict(k=0), 2), (dict(k=131072, lda=131072, ldb=131072), 2), (dict(n=0), 2), (dict(rows=-1), 2),
    (dict(rows=2 ** 31), 2), (dict(n=2 ** 30, num_experts=4, ldo=2 ** 30, seg_offsets=0x100, seg_counts=0x200), 2),
    (dict(num_experts=0), 1), (dict(num_experts=1025), 1), (dict(out_dtype=3), 1), (dict(out_dtype=-1), 1),
    (dict(num_experts=2), 4), (dict(seg_offsets=0x100), 4), (dict(b2=0x60000), 4),
    (dict(a=0), 4), (dict(b_scale=0), 4), (dict(out=0), 4),
    (dict(bias=0x100, b2=0x60000, b2_scale=0x70000), 1),
    (dict(lda=96), 1), (dict(ldb=96), 1), (dict(ldo=63), 1),
    (dict(lda=120), 3), (dict(ldb=104), 3), (dict(a=0x10008), 3), (dict(b=0x20001), 3),
])
def test_product_statuses(pkg, kw, status):
    lib = pkg.load_library()
    assert lib.nvfp4_int8_gemm(ctypes.byref(_product(pkg._native, **kw)), None) == status
    assert lib.nvfp4_last_error_detail()


def test_product_of_no_rows_and_null(pkg):
    lib = pkg.load_library()
    assert lib.nvfp4_int8_gemm(ctypes.byref(_product(pkg._native, rows=0)), None) == 0
    assert lib.nvfp4_int8_gemm(None, None) == 4


def test_product_struct_layout(pkg):
    P = pkg._native.Int8Product
    assert ctypes.sizeof(P) == 10 * 8 + 5 * 8 + 4 * 4
    assert P.rows.offset == 80 and P.n.offset == 120


def test_quantiser_statuses(pkg):
    lib = pkg.load_library()

    def call(x=0x1000, rows=4, cols=33, ld=33, dtype=0, listed=None, n=0, codes=0x2000, codes_ld=48,
             scales=0x3000):
        return lib.nvfp4_quantize_int8(x, rows, cols, ld, dtype, listed, n, codes, codes_ld, scales, None)

    assert call(dtype=2) == 1 and call(dtype=-1) == 1
    assert call(cols=0) == 2 and call(rows=-1) == 2 and call(rows=2 ** 31) == 2
    assert call(x=None) == 4 and call(codes=None) == 4 and call(scales=None) == 4
    assert call(ld=32) == 1 and call(codes_ld=32) == 1
    assert call(codes=0x2008) == 3 and call(codes_ld=40) == 3
    assert call(rows=0) == 0
    assert call(listed=0x4000, n=0) == 0 and call(listed=0x4000, n=-1) == 2 and call(listed=0x4000, n=2 ** 31) == 2

    def dispatch(tokens=4, topk=2, dest=0x4000, rows=128, cols=33):
        return lib.nvfp4_moe_dispatch_int8(0x1000, tokens, cols, 33, 0, dest, topk, rows, 0x2000, 48, 0x3000, None)

    assert dispatch(topk=0) == 2 and dispatch(tokens=2 ** 30) == 2 and dispatch(rows=-1) == 2
    assert dispatch(dest=None) == 4 and dispatch(tokens=0) == 0 and dispatch(rows=0) == 0


def test_token_sort_statuses(pkg):
    lib = pkg.load_library()

    def disp(x=0x1000, ldx=8, dtype=0, dest=0x2000, src=0x3000, tokens=4, topk=2, cols=8, rows=128, y=0x4000, ldy=8):
        return lib.nvfp4_moe_dispatch_tokens(x, ldx, dtype, dest, src, tokens, topk, cols, rows, y, ldy, None)

    assert disp(dtype=3) == 1 and disp(ldx=7) == 1 and disp(ldy=7) == 1
    assert disp(tokens=-1) == 2 and disp(topk=0) == 2 and disp(cols=0) == 2 and disp(rows=2 ** 31) == 2
    assert disp(x=None) == 4 and disp(dest=None) == 4 and disp(src=None) == 4 and disp(y=None) == 4
    assert disp(rows=0) == 0

    def comb(y=0x1000, ldy=8, dtype=0, dest=0x2000, w=None, tokens=4, topk=2, cols=8, rows=128, out=0x4000, ldo=8):
        return lib.nvfp4_moe_combine_tokens(y, ldy, dtype, dest, w, tokens, topk, cols, rows, out, ldo, None)

    assert comb(dtype=-1) == 1 and comb(ldy=7) == 1 and comb(ldo=7) == 1 and comb(rows=-1) == 2
    assert comb(y=None) == 4 and comb(out=None) == 4 and comb(tokens=0) == 0

    def back(g=0x1000, ldg=8, y=0x2000, ldy=8, dtype=0, dest=0x3000, src=0x4000, w=None, tokens=4, topk=2, cols=8,
             rows=128, gy=0x5000, ldo=8, gw=0x6000):
        return lib.nvfp4_moe_combine_tokens_backward(g, ldg, y, ldy, dtype, dest, src, w, tokens, topk, cols, rows,
                                                     gy, ldo, gw, None)

    assert back(dtype=7) == 1 and back(ldg=7) == 1 and back(ldy=7) == 1 and back(ldo=7) == 1
    assert back(g=None) == 4 and back(y=None) == 4 and back(src=None) == 4
    assert back(gy=None, gw=None) == 0 and back(cols=-1) == 2


def test_python_checks_refuse_cpu_tensors_and_bad_types(pkg):
    x = torch.zeros((4, 32), dtype=torch.bfloat16)
    q = torch.zeros((4, 32), dtype=torch.int8)
    s = torch.zeros(4)
    for call in (lambda: pkg.quantize_int8(x), lambda: pkg.int8_gemm(q, s, q, s),
                 lambda: pkg.int8_gemm_segments(q, s, q[None], s[None], s.int(), s.int())):
        with pytest.raises(ValueError):
            call()
    r = pkg.moe.Routing(4, 1, 1, [4], [0, 128], torch.zeros(4, dtype=torch.int32),
                        torch.zeros(128, dtype=torch.int32))
    for call in (lambda: pkg.moe.dispatch_tokens(x, r), lambda: pkg.moe.combine_tokens(x, r),
                 lambda: pkg.moe.dispatch_int8(x, r), lambda: pkg.moe.combine_tokens_backward(x, x, r)):
        with pytest.raises(ValueError):
            call()


def test_block_refuses_bad_sizes(pkg):
    w = pkg.moe.Int8ExpertWeights(*(torch.zeros(s, dtype=t) for s, t in (
        ((2, 8, 16), torch.int8), ((2, 8), torch.float32), ((2, 8, 16), torch.int8), ((2, 8), torch.float32),
        ((2, 16, 9), torch.int8), ((2, 16), torch.float32))))
    with pytest.raises(ValueError, match="w_down"):
        pkg.moe.Int8MoEBlock(w, 4, 2)
    with pytest.raises(ValueError, match="positive"):
        pkg.moe.Int8MoEBlock(w, 0, 2)
    with pytest.raises(ValueError, match="dtype"):
        pkg.moe.Int8MoEBlock(w, 4, 2, dtype=torch.float32)


WIDE = 2 ** 30 + 8  # columns past the operators' limit


def test_columns_past_the_kernels_index_range(pkg):
    """Column counters step past the last column by up to a block's span: counts near 2^31 are refused."""
    lib = pkg.load_library()
    for cols in (WIDE, 2 ** 31 - 1):
        ld = (cols + 15) // 16 * 16
        assert lib.nvfp4_quantize_int8(0x1000, 1, cols, ld, 0, None, 0, 0x2000, ld, 0x3000, None) == 2
        assert lib.nvfp4_moe_dispatch_int8(0x1000, 1, cols, ld, 0, 0x4000, 1, 128, 0x2000, ld, 0x3000, None) == 2
        assert lib.nvfp4_moe_dispatch_tokens(0x1000, ld, 0, 0x2000, 0x3000, 1, 1, cols, 128, 0x4000, ld, None) == 2
        assert lib.nvfp4_moe_combine_tokens(0x1000, ld, 0, 0x2000, None, 1, 1, cols, 128, 0x4000, ld, None) == 2
        assert lib.nvfp4_moe_combine_tokens_backward(0x1000, ld, 0x2000, ld, 0, 0x3000, 0x4000, None, 1, 1, cols, 128,
                                                     0x5000, ld, 0x6000, None) == 2


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("cols", [WIDE, 2 ** 32 + 5])
def test_python_refuses_wide_rows(pkg, cols):
    """... and none is cut to its low 32 bits on the way."""
    r = pkg.moe.Routing(1, 1, 1, [1], [0, 128], torch.zeros(1, dtype=torch.int32), torch.zeros(128, dtype=torch.int32))
    for call in (lambda: pkg.quantize_int8(_meta(1, cols)), lambda: pkg.moe.dispatch_int8(_meta(1, cols), r),
                 lambda: pkg.moe.dispatch_tokens(_meta(1, cols), r), lambda: pkg.moe.combine_tokens(_meta(128, cols), r),
                 lambda: pkg.moe.dispatch_tokens_backward(_meta(128, cols), r),
                 lambda: pkg.moe.combine_tokens_backward(_meta(1, cols), _meta(128, cols), r)):
        with pytest.raises(ValueError, match="columns"):
            call()


def test_python_refuses_more_pairs_or_channels_than_32_bits_hold(pkg):
    many = 2 ** 32 + 1
    r = pkg.moe.Routing(many, 1, 1, [1], [0, 128], _meta(many, dtype=torch.int32), _meta(128, dtype=torch.int32))
    for call in (lambda: pkg.moe.dispatch_tokens(_meta(many, 8), r), lambda: pkg.moe.combine_tokens(_meta(128, 8), r),
                 lambda: pkg.moe.dispatch_int8(_meta(many, 8), r),
                 lambda: pkg.moe.combine_tokens_backward(_meta(many, 8), _meta(128, 8), r)):
        with pytest.raises(ValueError, match="pairs"):
            call()
    i8, f32 = dict(dtype=torch.int8), dict(dtype=torch.float32)
    a, sa = _meta(4, 16, **i8), _meta(4, **f32)
    with pytest.raises(ValueError, match="channels"):
        pkg.int8_gemm(a, sa, _meta(2 ** 31, 16, **i8), _meta(2 ** 31, **f32))
    with pytest.raises(ValueError, match="channels"):
        pkg.int8_gemm_segments(a, sa, _meta(4, 2 ** 29, 16, **i8), _meta(4, 2 ** 29, **f32),
                               torch.zeros(4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))


def test_error_words_are_checked(pkg):
    q, s = torch.zeros((4, 32), dtype=torch.int8), torch.zeros(4)
    for word in (torch.zeros(2, dtype=torch.int32), torch.zeros(1), 5):
        for call in (lambda: pkg.int8_gemm(q, s, q, s, error_word=word),
                     lambda: pkg.int8_gemm_segments(q, s, q[None], s[None], s.int(), s.int(), error_word=word),
                     lambda: pkg.check_int8_errors(error_word=word)):
            with pytest.raises(ValueError, match="error_word"):
                call()
    with pytest.raises(ValueError, match="CUDA"):
        pkg.check_int8_errors(error_word=torch.zeros(1, dtype=torch.int32))

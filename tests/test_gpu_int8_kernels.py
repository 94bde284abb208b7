"""Every kernel of the int8 products that a rule on sizes chooses, at the sizes of int8_cases.py, against
64-bit restatements (tolerances: test_gpu_int8.py)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import int8_cases as C
import test_gpu_int8 as T

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("counts,n,k,warps", C.GATED_PAIRS)
def test_gated_pairs(pkg, counts, n, k, warps, dtype):
    """CTA pairs that hand gate and up sums to one another, with 16 and with 8 epilogue warps."""
    offs, rows = C.offsets(counts)
    T._segments_case(pkg, offs, counts, rows, n, k, True, dtype, sum(counts), seed=k)
    assert pkg.check_int8_errors() == 0


@pytest.mark.parametrize("gated,k,warps", C.EIGHT_ROWS)
def test_byte_products_of_eight_rows(pkg, gated, k, warps):
    offs, rows = C.offsets(C.EIGHT_COUNTS, gap=3)
    T._segments_case(pkg, offs, C.EIGHT_COUNTS, rows, C.EIGHT_N, k, gated, torch.bfloat16, C.EIGHT_EXPECTED, seed=k)
    assert pkg.check_int8_errors() == 0


@pytest.mark.parametrize("rows,k,warps", C.ONE_EXPERT)
def test_byte_products_of_one_expert(pkg, rows, k, warps):
    """Segments of one expert whose estimate is right, and below what it holds."""
    for count in (rows, 2 * rows + 1):
        T._segments_case(pkg, [2], [count], count + 5, C.ONE_EXPERT_N, k, True, torch.float16, rows, seed=k)
    assert pkg.check_int8_errors() == 0


def _gated(pkg, rows, n, k, gate, up, dtype):
    """One expert whose gate and up sums are exactly `gate` (a multiple of 1/64 above -129) and `up`
    (a power of two) in every row; the output, and the kernel that made it."""
    a = torch.zeros((rows, (k + 15) // 16 * 16), dtype=torch.int8)
    a[:, 0], a[:, 1] = 64, 1
    s = (gate * 64).round().long()
    hi = torch.div(s, 64, rounding_mode="floor")
    w = [torch.zeros((1, n, (k + 15) // 16 * 16), dtype=torch.int8) for _ in range(2)]
    w[0][0, :, 0], w[0][0, :, 1] = hi.to(torch.int8), (s - 64 * hi).to(torch.int8)
    w[1][0, :, 1] = 1
    one = torch.ones(rows, device="cuda")
    sw = [torch.full((1, n), v, device="cuda") for v in (1 / 64, up)]
    off, cnt = (torch.tensor([v], dtype=torch.int32, device="cuda") for v in (0, rows))
    out = pkg.int8_gemm_segments(a.cuda()[:, :k], one, w[0].cuda()[:, :, :k], sw[0], off, cnt, b2=w[1].cuda()[:, :, :k],
                                 b2_scale=sw[1], out_dtype=dtype, expected_rows=rows)
    return out.double().cpu(), C.plan(pkg, rows, n, k, 1, True, rows, True)[0]


GATED_OF_EACH_KERNEL = [(1, 300, 64, C.BYTES), (130, 300, 64, C.TILES), (600, 5000, 1300, C.PAIRS)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,n,k,kernel", GATED_OF_EACH_KERNEL)
def test_gates_whose_exponential_is_next_to_the_largest_float(pkg, rows, n, k, kernel, dtype):
    """silu of -88.7 .. -87.3: exp(-g) is finite but above 2^126. With a large up sum the result is an
    ordinary number. Tolerance: as in test_gpu_int8.py, and half a step of the subnormal exp(g) (at
    most 2^-150 / 3e-39 = 4 u)."""
    gate = -87.3125 - torch.arange(n).remainder(90).double() / 64
    got, used = _gated(pkg, rows, n, k, gate, 2.0 ** 40, dtype)
    assert used == kernel
    want = (gate / (1 + torch.exp(-gate)) * 2.0 ** 40).expand(rows, n)
    tol = ((20 + 5.4 * 88.8) * T.U + T.HALF[dtype]) * want.abs()
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / want.abs()).max())


@pytest.mark.parametrize("rows,n,k,kernel", GATED_OF_EACH_KERNEL)
def test_gated_fp32_outputs_have_32_bits(pkg, rows, n, k, kernel):
    """Gate and up sums are exact here, so what is left is silu's own error. e = exp(-|g|) within 2 ulp
    (4 u), g e, 1 + e and the quotient within half an ulp each (u); the up sum is a power of two: 7 u."""
    gate = -80 + (torch.arange(n).double() * (160 * 64) / n).floor() / 64
    got, used = _gated(pkg, rows, n, k, gate, 2.0 ** 10, torch.float32)
    assert used == kernel
    want = (gate / (1 + torch.exp(-gate)) * 2.0 ** 10).expand(rows, n)
    err = (got - want).abs()
    assert bool((err <= 7 * T.U * want.abs()).all()), float((err / want.abs()).nan_to_num(0).max() / T.U)


@pytest.mark.parametrize("rows,n,k,kernel,tokens,warps", C.DENSE_GATED)
def test_dense_gated_products_of_the_c_entry(pkg, rows, n, k, kernel, tokens, warps):
    """b2 without segments: every kernel and tile, all of them ragged; what surrounds the output stays."""
    dtype = (torch.bfloat16, torch.float16, torch.float32)[(rows + k) % 3]
    a, sa = T._codes(rows, k, rows), T._scale(rows, 2, 0.01)
    w, sw = [T._codes(n, k, 3 + i) for i in range(2)], [T._scale(n, 5 + i, 0.002) for i in range(2)]
    big = torch.full((rows + 2, n + 3), 7.0, dtype=dtype, device="cuda")
    out = big[1:rows + 1, 1:n + 1]
    N = pkg._native
    p = N.Int8Product(a=a.data_ptr(), b=w[0].data_ptr(), b2=w[1].data_ptr(), a_scale=sa.data_ptr(),
                      b_scale=sw[0].data_ptr(), b2_scale=sw[1].data_ptr(), out=out.data_ptr(), rows=rows,
                      lda=a.stride(0), ldb=w[0].stride(0), ldo=big.stride(0), n=n, k=k, num_experts=1,
                      out_dtype=[torch.bfloat16, torch.float16, torch.float32].index(dtype))
    lib = pkg.load_library()
    N.check(lib.nvfp4_int8_gemm(ctypes.byref(p), torch.cuda.current_stream().cuda_stream), lib)
    assert pkg.check_int8_errors() == 0
    g, up = (T.O.product(T._np(a), T._np(sa), T._np(b), T._np(s)) for b, s in zip(w, sw))
    want = T.O.silu(g) * up
    tol = (16 + 5.4 * np.abs(g)) * T.U * np.abs(want) + 1e-30 * np.abs(up)
    T._close(out, want, 1.01 * (tol + T.HALF[dtype] * np.abs(want)) + T.TINY[dtype])
    out.fill_(7.0)
    assert bool((big == 7).all())


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("expected,kernel,tokens", C.ONE_ROW_EACH)
def test_one_expected_row_each_and_all_of_them_in_one_expert(pkg, expected, kernel, tokens, gated):
    for counts in ([1] * expected + [0] * (64 - expected), [0] * 7 + [expected] + [0] * 56):
        offs, rows = C.offsets(counts)
        T._segments_case(pkg, offs, counts, rows, C.ONE_ROW_N, 1100, gated, torch.bfloat16, expected, seed=expected)
    assert pkg.check_int8_errors() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k,kernel", [(100, 200, 1, C.TILES), (40, 3000, 15, C.TILES), (600, 10000, 3, C.PAIRS),
                                          (300, 20000, 16, C.PAIRS)])
def test_sums_shorter_than_a_load(pkg, m, n, k, kernel, dtype):
    assert C.plan(pkg, m, n, k)[0] == kernel
    a, b = T._codes(m, k, 1), T._codes(n, k, 2)
    sa, sb = T._scale(m, 3, 0.01), T._scale(n, 4, 0.01)
    T._check_product(pkg.int8_gemm(a, sa, b, sb, out_dtype=dtype), a, sa, b, sb)
    assert pkg.check_int8_errors() == 0

"""int8 quantiser and products on the GPU against 64-bit restatements.

Tolerances, counted from the kernels' roundings (u = 2^-24, h = eps / 2 of the output type):
a product converts its exact sum to fp32 and multiplies twice (3 u of the product), adds the
bias (u of the result) and rounds (h). Gated: both projections carry 3 u, which silu passes on
times at most 1 + |g|; __expf is within 2 + 1.173 |g| ulp, __fdividef within 2 ulp, the sum
and the last product within half an ulp each, together (16 + 5.4 |g|) u.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import int8_oracle as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: U}
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}


def _codes(rows, cols, seed, pad=0, fill=None):
    """int8 codes on the GPU with rows a multiple of 16 bytes apart (plus `pad` * 16)."""
    g = torch.Generator().manual_seed(seed)
    ld = (cols + 15) // 16 * 16 + 16 * pad
    buf = torch.randint(-127, 128, (rows, ld), generator=g, dtype=torch.int8)
    if fill is not None:
        buf.fill_(fill)
    return buf.cuda()[:, :cols]


def _scale(shape, seed, level):
    g = torch.Generator().manual_seed(seed)
    return ((0.25 + torch.rand(shape, generator=g)) * level).cuda()


def _np(t):
    return t.detach().double().cpu().numpy()


def _close(got, want, tol):
    err = np.abs(_np(got) - want)
    assert np.all(err <= tol), (float((err - tol).max()), np.argwhere(err > tol)[:5])


def _check_product(got, a, sa, b, sb, bias=None):
    want = O.product(_np(a), _np(sa), _np(b), _np(sb), None if bias is None else _np(bias))
    part = np.abs(O.product(_np(a), _np(sa), _np(b), _np(sb)))
    h = HALF[got.dtype]
    _close(got, want, 1.01 * (3 * U * part + U * np.abs(want) + h * np.abs(want)) + TINY[got.dtype])


# ------------------------------------------------------------------ quantiser
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 17), (5, 16), (9, 1023), (4, 1024), (7, 2050),
                                       (6, 4096), (3, 8192), (2, 20011), (0, 64), (300, 96), (3, 1300), (5, 2000)])
def test_quantize_codes_are_those_of_the_exact_quotient(pkg, rows, cols, dtype):
    g = torch.Generator().manual_seed(rows * 7 + cols)
    x = torch.randn((rows, cols), generator=g) * torch.exp(2 * torch.randn((rows, 1), generator=g))
    x = x.to(dtype)
    if rows:
        x[0, cols // 2] = 2 * x[0].float().abs().max()  # halves of the maximum: ties
        x[0, cols // 3] = x[0].float().abs().max() / 2
    codes, scales = pkg.quantize_int8(x.cuda())
    want, ws = O.quantize_int8(x.double().numpy())
    assert np.array_equal(codes.cpu().numpy(), want)
    assert np.all(np.abs(_np(scales) - ws) <= U * ws)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantize_every_ratio_of_ties(pkg, dtype):
    """Rows whose quotients are half-integers: x = (2k + 1) max / 254 with max = 254 2^e."""
    k = torch.arange(-127, 127, dtype=torch.float64)
    rows = []
    for e in (-14, -3, 0, 4) + ((-126, 90) if dtype == torch.bfloat16 else ()):
        rows.append(torch.cat([(2 * k + 1) * 2.0 ** e, torch.tensor([254.0 * 2.0 ** e])]))
    x = torch.stack(rows).to(dtype)
    codes, _ = pkg.quantize_int8(x.cuda())
    assert np.array_equal(codes.cpu().numpy(), O.quantize_int8(x.double().numpy())[0])


@pytest.mark.parametrize("rows,cols", [(2400, 513), (2368, 4096), (2500, 4100), (2371, 8200), (2370, 20000)])
def test_quantize_many_rows(pkg, rows, cols):
    """Row counts at which fewer threads share a row."""
    g = torch.Generator().manual_seed(cols)
    x = (torch.randn((rows, cols), generator=g) * 3).to(torch.bfloat16)
    codes, scales = pkg.quantize_int8(x.cuda())
    xd = x.double()
    amax = xd.abs().amax(1, keepdim=True)
    assert torch.equal(codes.cpu(), torch.round(127 * xd / amax).to(torch.int8))
    assert float(((scales.cpu().double() - amax[:, 0] / 127).abs() / amax[:, 0] * 127).max()) <= U


def test_quantize_extreme_rows(pkg):
    x = torch.zeros((8, 40), dtype=torch.bfloat16)
    x[1, 3] = float("inf")
    x[2, 39] = float("nan")
    x[3] = torch.finfo(torch.bfloat16).max
    x[3, 1:5] = -torch.finfo(torch.bfloat16).max / 2
    x[4, 7] = 2.0 ** -133  # the smallest bf16
    x[5, 0], x[5, 1] = 2.0 ** -130, -(2.0 ** -131)
    x[6, 0], x[6, 1] = float("-inf"), float("nan")
    x[7, 0] = -1.0
    codes, scales = pkg.quantize_int8(x.cuda())
    want, ws = O.quantize_int8(x.double().numpy())
    assert np.array_equal(codes.cpu().numpy(), want)
    assert np.array_equal(np.isnan(_np(scales)), np.isnan(ws))
    ok = ~np.isnan(ws)
    assert np.all(np.abs(_np(scales)[ok] - ws[ok]) <= U * ws[ok] + 2.0 ** -149)


def test_quantize_strided_input_listed_rows_and_untouched_bytes(pkg):
    base = torch.randn((33, 301), generator=torch.Generator().manual_seed(4)).to(torch.float16).cuda()
    x = base[:, 5:5 + 203]  # rows 301 elements apart, odd start
    buf = torch.full((33, 256), 77, dtype=torch.int8, device="cuda")
    scales = torch.full((33,), -1.0, device="cuda")
    rows = torch.tensor([4, -1, 32, 0, 33, 4, 17, 2 ** 31 - 1, -5], dtype=torch.int32, device="cuda")
    pkg.quantize_int8(x, codes=buf[:, :203], scales=scales, row_list=rows)
    want, ws = O.quantize_int8(_np(x))
    keep = np.zeros(33, dtype=bool)
    keep[[4, 32, 0, 17]] = True
    assert np.array_equal(buf.cpu().numpy()[keep, :203], want[keep])
    assert np.all(np.abs(_np(scales)[keep] - ws[keep]) <= U * ws[keep])
    assert np.all(buf.cpu().numpy()[~keep] == 77) and np.all(buf.cpu().numpy()[:, 203:] == 77)
    assert np.all(_np(scales)[~keep] == -1.0)
    pkg.quantize_int8(x, codes=buf[:, :203], scales=scales, row_list=rows[:0])  # none
    assert np.all(_np(scales)[~keep] == -1.0)


# ------------------------------------------------------------------ dense product
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 128), (1, 1000, 2048), (2, 129, 144),
                                   (16, 256, 512), (17, 77, 1000), (33, 130, 31), (65, 384, 256),
                                   (128, 128, 640), (129, 257, 127), (300, 515, 1111)])
def test_product(pkg, m, n, k, dtype):
    a, b = _codes(m, k, 1 + m), _codes(n, k, 2 + n)
    sa, sb = _scale(m, 3, 0.01), _scale(n, 4, 0.002)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(5)).cuda() if m % 2 else None
    out = pkg.int8_gemm(a, sa, b, sb, bias=bias, out_dtype=dtype)
    assert out.dtype == dtype and tuple(out.shape) == (m, n)
    _check_product(out, a, sa, b, sb, bias)
    assert pkg.check_int8_errors() == 0


@pytest.mark.parametrize("m,n,k", [(1, 4096, 7168), (83, 4099, 2011), (512, 384, 4096),
                                   (1000, 1025, 520), (2500, 640, 384)])
def test_product_larger(pkg, m, n, k):
    a, b = _codes(m, k, 11), _codes(n, k, 12)
    sa, sb = _scale(m, 13, 0.01), _scale(n, 14, 0.002)
    _check_product(pkg.int8_gemm(a, sa, b, sb), a, sa, b, sb)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(2, 300, 1000), (1, 4099, 17), (1300, 2050, 520),
                                   (1100, 2304, 300), (3000, 1111, 257), (700, 2048, 1024)])
def test_product_of_every_kernel(pkg, m, n, k, dtype):
    """Sizes at which one or two rows, few tiles, many tiles and CTA pairs are chosen."""
    a, b = _codes(m, k, 21), _codes(n, k, 22)
    sa, sb = _scale(m, 23, 0.01), _scale(n, 24, 0.002)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(5)).cuda()
    _check_product(pkg.int8_gemm(a, sa, b, sb, bias=bias, out_dtype=dtype), a, sa, b, sb, bias)
    assert pkg.check_int8_errors() == 0


@pytest.mark.parametrize("m,n,k", [(993, 3090, 532), (861, 4811, 507), (858, 2859, 256),
                                   (1291, 2418, 714), (1161, 2908, 960), (1001, 3934, 1398),
                                   (97, 20000, 65), (600, 4200, 300), (1453, 4224, 577)])
def test_product_on_cta_pairs_with_tiles_of_every_size(pkg, m, n, k):
    """Rows and channels whose waves end soonest with tiles of 96, 128, ... 256 tokens, all of
    them ragged; what surrounds the output is left as it was."""
    a, b = _codes(m, k, 41), _codes(n, k, 42)
    sa, sb = _scale(m, 43, 0.01), _scale(n, 44, 0.002)
    out = torch.full((m + 2, n + 3), 7.0, dtype=torch.float16, device="cuda")
    pkg.int8_gemm(a, sa, b, sb, out=out[:m, :n])
    _check_product(out[:m, :n], a, sa, b, sb)
    assert bool((out[m:] == 7).all()) and bool((out[:, n:] == 7).all())
    assert pkg.check_int8_errors() == 0


@pytest.mark.parametrize("n,k", [(2000, 8200), (300, 500), (1100, 4096), (500, 2047), (33, 1025)])
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 8])
def test_product_of_few_rows(pkg, m, n, k):
    """Few rows and tiles: one to eight tokens at once, K shared by one to eight warps."""
    a, b = _codes(m, k, 31 + m), _codes(n, k, 32)
    sa, sb = _scale(m, 33, 0.01), _scale(n, 34, 0.002)
    _check_product(pkg.int8_gemm(a, sa, b, sb, out_dtype=torch.float16), a, sa, b, sb)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("per,k", [(1, 8192), (2, 4100), (3, 2047), (4, 500), (6, 8192), (8, 1030)])
def test_segments_of_few_rows(pkg, per, k, gated):
    """The same over experts whose real counts differ from the estimate (one far above it)."""
    _segments_case(pkg, [40, 0, 7, 30], [per, max(per - 1, 0), 19, 0], 60, 410, k, gated,
                   torch.bfloat16, 4 * per, seed=per)
    assert pkg.check_int8_errors() == 0


def test_product_sums_are_exact_at_the_largest_k(pkg):
    """Sums next to the edge of int32, and codes of -128."""
    k = pkg._native.INT8_MAX_K
    a, b = _codes(3, k, 0, fill=-128), _codes(5, k, 0, fill=-128)
    one = torch.ones(5, device="cuda")
    out = pkg.int8_gemm(a, one[:3].contiguous(), b, one, out_dtype=torch.float32)
    assert torch.all(out == float(np.float32(128 * 128 * k)))
    b = _codes(5, k, 0, fill=127)
    out = pkg.int8_gemm(a, one[:3].contiguous(), b, one, out_dtype=torch.float32)
    assert torch.all(out == float(np.float32(-128 * 127 * k)))


def test_product_strides_and_untouched_output(pkg):
    a, b = _codes(37, 200, 1, pad=2), _codes(150, 200, 2, pad=1)
    sa, sb = _scale(37, 3, 0.01), _scale(150, 4, 0.01)
    big = torch.full((40, 333), 5.0, dtype=torch.float16, device="cuda")
    out = big[2:39, 7:157]  # odd start, rows 333 apart
    assert pkg.int8_gemm(a, sa, b, sb, out=out) is out
    _check_product(out, a, sa, b, sb)
    big[2:39, 7:157] = 5.0
    assert torch.all(big == 5.0)


def test_product_scales_of_nan_and_zero(pkg):
    a, b = _codes(4, 64, 1), _codes(9, 64, 2)
    sa, sb = _scale(4, 3, 0.01), _scale(9, 4, 0.01)
    sa[1], sa[2] = float("nan"), 0.0
    out = pkg.int8_gemm(a, sa, b, sb).float().cpu()
    assert torch.isnan(out[1]).all() and torch.all(out[2] == 0)
    assert torch.isfinite(out[[0, 3]]).all()


def test_product_of_no_rows(pkg):
    b = _codes(9, 64, 2)
    out = pkg.int8_gemm(_codes(0, 64, 1), _scale(0, 1, 1.0), b, _scale(9, 4, 0.01))
    assert tuple(out.shape) == (0, 9)


# ------------------------------------------------------------------ segments
def _segments_case(pkg, offs, cnts, rows, n, k, gated, dtype, expected, seed=0):
    E = len(cnts)
    a, sa = _codes(rows, k, seed + 1), _scale(rows, seed + 2, 0.01)
    w = [_codes(E * n, k, seed + 3 + i).unflatten(0, (E, n)) for i in range(2)]
    sw = [_scale((E, n), seed + 5 + i, 0.002) for i in range(2)]
    off = torch.tensor(offs, dtype=torch.int32, device="cuda")
    cnt = torch.tensor(cnts, dtype=torch.int32, device="cuda")
    out = torch.full((rows, n), 3.0, dtype=dtype, device="cuda")
    pkg.int8_gemm_segments(a, sa, w[0], sw[0], off, cnt, b2=w[1] if gated else None,
                           b2_scale=sw[1] if gated else None, out=out, expected_rows=expected)
    touched = np.zeros(rows, dtype=bool)
    h = HALF[dtype]
    for e in range(E):
        o, c = offs[e], cnts[e]
        if c <= 0 or o < 0 or o + c > rows:
            continue
        touched[o:o + c] = True
        g = O.product(_np(a[o:o + c]), _np(sa[o:o + c]), _np(w[0][e]), _np(sw[0][e]))
        tol = 4 * U * np.abs(g)
        if gated:
            up = O.product(_np(a[o:o + c]), _np(sa[o:o + c]), _np(w[1][e]), _np(sw[1][e]))
            want = O.silu(g) * up
            tol = (16 + 5.4 * np.abs(g)) * U * np.abs(want) + 1e-30 * np.abs(up)
        else:
            want = g
        _close(out[o:o + c], want, 1.01 * (tol + h * np.abs(want)) + TINY[dtype])
    assert torch.all(out[torch.from_numpy(~touched).cuda()] == 3.0)
    return out


@pytest.mark.parametrize("k", [700, 1025, 2304, 2305])
@pytest.mark.parametrize("gated", [False, True])
def test_segments_on_cta_pairs_with_short_and_long_sums(pkg, gated, k):
    """CTA pairs with 16 epilogue warps (short K) and with 8: counts that leave warps without
    tokens in a tile, and an expert without rows."""
    cnts = [17, 256, 0, 289, 513, 33, 241]
    offs = np.concatenate([[1], 1 + np.cumsum(cnts)[:-1] + np.arange(1, 7)]).tolist()
    _segments_case(pkg, offs, cnts, offs[-1] + cnts[-1] + 3, 1701, k, gated, torch.bfloat16,
                   sum(cnts), seed=k)
    assert pkg.check_int8_errors() == 0


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("offs,cnts,expected", [
    ([0], [1], 1),
    ([0, 128, 256, 256], [5, 100, 0, 16], 121),
    ([0, 7, 40], [7, 33, 201], 241),           # segments that start anywhere
    ([300, 0, 150], [41, 129, 64], 0),          # any order, gaps
    ([0, 0, 0, 0, 0], [0, 0, 0, 0, 0], 10),     # nothing routed
    ([0, 16, 32, 33], [16, 15, 1, 255], 40),    # an estimate far below the rows
])
def test_segments(pkg, offs, cnts, expected, gated):
    _segments_case(pkg, offs, cnts, 345, 200, 208, gated, torch.bfloat16, expected)
    assert pkg.check_int8_errors() == 0


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("per", [3, 20, 50, 130, 260])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_segments_of_every_tile_shape(pkg, per, gated, dtype):
    E = 5
    cnts = [per, 0, per + 9, max(per - 2, 0), 1]
    offs = np.concatenate([[0], np.cumsum([(c + 127) // 128 * 128 for c in cnts])])[:E].tolist()
    rows = offs[-1] + 128
    _segments_case(pkg, offs, cnts, rows, 301, 333, gated, dtype, per * E, seed=per)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("per,n", [(1, 300), (2, 333), (8, 4000), (20, 2000), (40, 5000),
                                   (50, 2500), (60, 5000), (130, 1300), (130, 3000), (260, 3008),
                                   (520, 2048)])
def test_segments_of_every_kernel(pkg, per, n, gated, dtype):
    """Rows per expert and widths at which each kernel and token tile is chosen; the real counts
    differ from the estimate, some far above it."""
    E = 5
    cnts = [per, 0, per + 9, max(per - 2, 0), 2 * per]
    offs = np.concatenate([[0], np.cumsum([c + 3 for c in cnts])])[:E].tolist()
    _segments_case(pkg, offs, cnts, offs[-1] + cnts[-1] + 2, n, 180, gated, dtype, per * E, seed=per)
    assert pkg.check_int8_errors() == 0


def test_many_experts(pkg):
    E = pkg._native.INT8_MAX_EXPERTS
    rng = np.random.default_rng(3)
    cnts = rng.integers(0, 4, E)
    offs = np.concatenate([[0], np.cumsum(cnts)])[:E].tolist()
    _segments_case(pkg, offs, cnts.tolist(), int(cnts.sum()), 40, 48, True, torch.bfloat16, 1500)


def test_segment_outside_the_slab_is_skipped_and_reported(pkg):
    offs, cnts = [0, -1, 10, 90, 2 ** 31 - 8], [5, 4, -3, 50, 100]
    _segments_case(pkg, offs, cnts, 100, 64, 64, False, torch.bfloat16, 60)
    with pytest.raises(pkg.Nvfp4Error, match="segment"):
        pkg.check_int8_errors()
    assert pkg.check_int8_errors() == 0


@pytest.mark.parametrize("expected", [8, 2000])
def test_segments_that_share_rows_stay_in_bounds(pkg, expected):
    """Many segments that all claim the whole slab: no row outside them is written, and the
    excess is reported (few tiles and many)."""
    rows, n, k, E = 300, 2100, 64, 40
    a, sa = _codes(rows, k, 1), _scale(rows, 2, 0.01)
    b, sb = _codes(E * n, k, 3).unflatten(0, (E, n)), _scale((E, n), 4, 0.01)
    big = torch.full((rows + 20, n), 3.0, dtype=torch.bfloat16, device="cuda")
    off = torch.zeros(E, dtype=torch.int32, device="cuda")
    cnt = torch.full((E,), rows, dtype=torch.int32, device="cuda")
    pkg.int8_gemm_segments(a, sa, b, sb, off, cnt, out=big[10:10 + rows], expected_rows=expected * E)
    with pytest.raises(pkg.Nvfp4Error, match="segment"):
        pkg.check_int8_errors()
    assert torch.all(big[:10] == 3.0) and torch.all(big[10 + rows:] == 3.0)


def test_outputs_past_32_bits(pkg):
    """2.4e9 output elements: the last rows are where they belong."""
    m, n, k = 600_000, 4000, 16
    a, sa = _codes(m, k, 1), _scale(m, 2, 0.01)
    b, sb = _codes(n, k, 3), _scale(n, 4, 0.01)
    out = pkg.int8_gemm(a, sa, b, sb)
    for rows in (slice(0, 3), slice(536_869, 536_875), slice(m - 3, m)):
        _check_product(out[rows], a[rows], sa[rows], b, sb)
    codes, scales = pkg.quantize_int8(out)
    want, ws = O.quantize_int8(_np(out[m - 2:]))
    assert np.array_equal(codes[m - 2:].cpu().numpy(), want)


def test_two_streams_and_a_graph(pkg):
    """Calls on two streams at once and two captured graphs, replayed in turn: no shared state."""
    k, n = 512, 384
    xs = [_codes(m, k, m) for m in (5, 200)]
    b, sb = _codes(n, k, 9), _scale(n, 10, 0.01)
    ss = [_scale(x.shape[0], 11, 0.01) for x in xs]
    want = [pkg.int8_gemm(x, s, b, sb) for x, s in zip(xs, ss)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        got = [pkg.int8_gemm(x, s, b, sb, stream=st) for x, s, st in zip(xs, ss, streams)]
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g, w)
    outs = [torch.zeros_like(w) for w in want]
    graphs = []
    for x, s, o in zip(xs, ss, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            pkg.int8_gemm(x, s, b, sb, out=o)
        graphs.append(g)
    for st, g in zip(streams, graphs):
        with torch.cuda.stream(st):
            g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)

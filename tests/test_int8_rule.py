"""The rule that chooses an int8 product's kernel and tile, as the host reports it (CPU only)."""
from __future__ import annotations

import ctypes

import pytest

import int8_cases as C


@pytest.mark.parametrize("counts,n,k,warps", C.GATED_PAIRS)
def test_gated_pairs(pkg, counts, n, k, warps):
    _, rows = C.offsets(counts)
    assert C.plan(pkg, rows, n, k, len(counts), True, sum(counts), True) == (C.PAIRS, 256, warps)


@pytest.mark.parametrize("gated,k,warps", C.EIGHT_ROWS)
def test_byte_products_of_eight_rows(pkg, gated, k, warps):
    _, rows = C.offsets(C.EIGHT_COUNTS)
    got = C.plan(pkg, rows, C.EIGHT_N, k, len(C.EIGHT_COUNTS), gated, C.EIGHT_EXPECTED, True)
    assert got == (C.BYTES, 8, warps)


@pytest.mark.parametrize("rows,k,warps", C.ONE_EXPERT)
def test_byte_products_of_one_expert(pkg, rows, k, warps):
    assert C.plan(pkg, rows, C.ONE_EXPERT_N, k, 1, True, rows, True) == (C.BYTES, rows, warps)


def test_short_gated_sums_stay_on_single_ctas(pkg):
    _, rows = C.offsets(C.RAGGED)
    for k, kernel in ((1280, C.TILES), (1281, C.PAIRS)):
        assert C.plan(pkg, rows, 1701, k, len(C.RAGGED), True, sum(C.RAGGED), True)[0] == kernel
        assert C.plan(pkg, rows, 3402, k, len(C.RAGGED), False, sum(C.RAGGED), True)[0] == C.PAIRS


@pytest.mark.parametrize("rows,n,k,kernel,tokens,warps", C.DENSE_GATED)
def test_dense_gated_products(pkg, rows, n, k, kernel, tokens, warps):
    assert C.plan(pkg, rows, n, k, gated=True) == (kernel, tokens, warps)


def test_dense_products(pkg):
    assert C.plan(pkg, 1, 4096, 7168) == (C.BYTES, 1, 2)
    assert C.plan(pkg, 83, 4099, 2011) == (C.TILES, 32, 4)
    assert C.plan(pkg, 8192, 4096, 7168) == (C.PAIRS, 256, 8)
    assert C.plan(pkg, 8192, 2048, 512)[::2] == (C.PAIRS, 16)
    assert C.plan(pkg, 2537, 1806, 7296)[:2] == (C.PAIRS, 160)


def test_of_no_rows_and_refusals(pkg):
    assert C.plan(pkg, 0, 64, 64) == (0, 0, 0)
    lib, N = pkg.load_library(), pkg._native
    out = N.Int8Launch()
    assert lib.nvfp4_int8_plan(None, 148, 74, ctypes.byref(out)) == 4
    with pytest.raises(pkg.Nvfp4Error):
        C.plan(pkg, 4, 64, 131072)
    with pytest.raises(pkg.Nvfp4Error):
        C.plan(pkg, 4, 64, 64, sms=0)


MOST_ROWS = 2 ** 31 - 1 - 256


@pytest.mark.parametrize("rows", [MOST_ROWS, MOST_ROWS - 1, 2_139_127_681, 2_139_127_680, 2 ** 30, 193, 8192, 8193])
def test_rows_of_a_tile_up_to_the_largest_count(pkg, rows):
    """Equal tiles hold all rows, none more than the kernel's accumulators, for counts whose sum with the
    number of tiles passes 2^31 as well."""
    got = C.launch(pkg, rows, 20000, 16)
    assert got.kernel == C.PAIRS
    tiles = -(-rows // got.tokens)
    assert got.rows % 32 == 0 and 0 < got.rows <= got.tokens <= 256
    assert (tiles - 1) * got.rows < rows <= tiles * got.rows


def test_tile_numbers_stay_below_2_to_31_with_a_stride_added(pkg):
    """Persistent CTAs add the grid to a tile's number: the sum has to fit as well."""
    rows, n = 2 ** 15 * 256, 65535 * 256
    with pytest.raises(pkg.Nvfp4Error, match="too many tiles"):
        C.launch(pkg, rows, n, 16)
    assert C.launch(pkg, rows, n // 2, 16).kernel == C.PAIRS


@pytest.mark.parametrize("gated", [False, True])
def test_byte_products_of_eight_rows_always_share_k(pkg, gated):
    """No kernel of eight tokens and one warp per channel exists: the rule never asks for it."""
    seen = set()
    for sms in (8, 80, 132, 148, 160):
        for experts in (1, 2, 3, 5, 8, 16):
            for n in (1, 127, 128, 129, 300, 410, 1000, 2048, 2100):
                for k in (1024, 2047, 2048, 4096, 8192, 20000):
                    for per in (3, 4, 5, 8):
                        kernel, tokens, warps = C.plan(pkg, 2 * per * experts, n, k, experts, gated, per * experts,
                                                       True, sms=sms, pairs=max(sms // 2, 1))
                        if kernel == C.BYTES and tokens == 8:
                            seen.add(warps)
    assert seen == {2, 4, 8}


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("expected,kernel,tokens", C.ONE_ROW_EACH)
def test_one_expected_row_each_is_certain_for_one_token_only(pkg, expected, kernel, tokens, gated):
    """As many pairs as experts average one row, but a popular expert has several: the weights must not be
    read once for each of them."""
    got = C.plan(pkg, 64 * 128, C.ONE_ROW_N, 1100, 64, gated, expected, True)
    assert got[:2] == (kernel, tokens)

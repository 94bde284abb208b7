"""Every kernel of the int8 products that a rule on sizes chooses, at the sizes of int8_cases.py, against
64-bit restatements (tolerances: test_gpu_int8.py)."""
from __future__ import annotations

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

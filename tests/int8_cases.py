"""Sizes at which each kernel of the int8 products is chosen, with what the rule has to say of them
on a B200 (148 SMs, 74 CTA pairs at once). The CPU tests hold the rule to this table and the GPU tests
run it, so that a threshold cannot move the tests away from a kernel unnoticed."""
from __future__ import annotations

import ctypes

BYTES, TILES, PAIRS = 1, 2, 3  # NVFP4_INT8_*
SMS, CTA_PAIRS = 148, 74

# Segments over gated CTA pairs: (counts, n, k, epilogue warps). Every n and k leaves a remainder of
# the tiles (128 channels) and of the stages (128 bytes), counts leave warps without tokens.
RAGGED = (17, 256, 0, 289, 513, 33, 241)
FEW = (300, 97, 1, 180)
GATED_PAIRS = [(RAGGED, 1701, 1281, 16), (FEW, 2433, 1300, 16), (RAGGED, 1665, 2011, 16), (FEW, 2500, 3000, 8)]

# Segments over byte products of eight rows: (gated, k, warps that share K).
EIGHT_COUNTS = (3, 2, 19, 0)  # three expected per expert, one far above it
EIGHT_N, EIGHT_EXPECTED = 410, 12
EIGHT_ROWS = [(False, 2048, 2), (False, 4111, 4), (False, 8200, 8), (True, 2100, 2), (True, 4111, 4)]

# One expert's segment over byte products of one, two and four rows, gated: (rows, k, warps).
ONE_EXPERT_N = 410
ONE_EXPERT = [(1, 1000, 1), (1, 2100, 2), (2, 1030, 1), (2, 4111, 4), (4, 1030, 1), (4, 8200, 8)]

# At most one expected row per expert, of 64: (expected rows, kernel, tokens).
ONE_ROW_N = 250
ONE_ROW_EACH = [(1, BYTES, 1), (8, BYTES, 1), (9, BYTES, 2), (32, BYTES, 2), (33, TILES, 16), (64, TILES, 16)]

# Gated products of one weight pair without segments (the C entry): (rows, n, k, kernel, tokens, warps).
DENSE_GATED = [(1, 410, 1000, BYTES, 1, 1), (2, 410, 2100, BYTES, 2, 2), (4, 410, 1030, BYTES, 4, 1),
               (7, 410, 4111, BYTES, 8, 4), (7, 2050, 300, TILES, 16, 4), (60, 5000, 200, TILES, 32, 4),
               (102, 4778, 1300, TILES, 64, 8), (275, 3725, 1300, TILES, 128, 8), (93, 19500, 1290, PAIRS, 96, 16),
               (971, 3084, 2011, PAIRS, 128, 16), (389, 4747, 1281, PAIRS, 160, 16), (487, 4772, 2400, PAIRS, 192, 8),
               (804, 3728, 2305, PAIRS, 224, 8), (693, 4789, 1300, PAIRS, 256, 16)]


def launch(pkg, rows, n, k, experts=1, gated=False, expected=0, segments=False, sms=SMS, pairs=CTA_PAIRS):
    """What a product of these sizes launches (nvfp4_int8_launch)."""
    N = pkg._native
    p = N.Int8Product(a=0x10000, b=0x20000, a_scale=0x30000, b_scale=0x40000, out=0x50000, rows=rows, n=n, k=k,
                      lda=(k + 15) // 16 * 16, ldb=(k + 15) // 16 * 16, ldo=n, num_experts=experts, out_dtype=0,
                      expected_rows=expected)
    if gated:
        p.b2, p.b2_scale = 0x60000, 0x70000
    if segments:
        p.seg_offsets, p.seg_counts = 0x80000, 0x90000
    got = N.Int8Launch()
    lib = pkg.load_library()
    N.check(lib.nvfp4_int8_plan(ctypes.byref(p), sms, pairs, ctypes.byref(got)), lib)
    return got


def plan(pkg, *args, **kw):
    """(kernel, tokens, warps) of a product."""
    got = launch(pkg, *args, **kw)
    return got.kernel, got.tokens, got.warps


def offsets(counts, gap=1):
    """Starts of segments `gap` rows apart, the first at row 1; the rows of the slab."""
    at, out = 1, []
    for c in counts:
        out.append(at)
        at += c + gap
    return out, at + 2

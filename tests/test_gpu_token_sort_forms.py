"""Forms of the token sort that callers meet beside the plain ones: one gradient only, weights shared by
the slots, one row for all, recomputation, mixed precision."""
from __future__ import annotations

import pytest
import torch

import test_gpu_token_sort as S

pytestmark = pytest.mark.gpu
TOKENS, TOPK, EXPERTS = 41, 3, 8


def _routing(pkg, seed):
    r = pkg.moe.route(S._ids(TOKENS, TOPK, EXPERTS, seed), EXPERTS)
    dest = r.dest.view(TOKENS, TOPK).long()
    return r, dest, dest >= 0


@pytest.mark.parametrize("dtype", list(S.HALF))
@pytest.mark.parametrize("cols", [1, 2, 130, 515])
def test_one_gradient_only(pkg, cols, dtype):
    """Rows without a gradient under weights with one, and each gradient asked for by itself."""
    r, dest, keep = _routing(pkg, cols)
    y, g = S._randn((r.rows, cols), 1, dtype), S._randn((TOKENS, cols), 2, dtype)
    w = S._randn((TOKENS, TOPK), 3, torch.float32).requires_grad_(True)
    (gw,) = torch.autograd.grad(pkg.moe.combine_tokens(y, r, w), w, g)
    want = (y[dest.clamp(min=0)].double() * g.double()[:, None]).sum(2) * keep
    mag = (y[dest.clamp(min=0)].double() * g.double()[:, None]).abs().sum(2) * keep
    assert bool(((gw.double() - want).abs() <= 1.01 * (cols + 1) * S.U * mag).all())
    gy, none = pkg.moe.combine_tokens_backward(g, None, r, w.detach(), want_weights=False)
    no, alone = pkg.moe.combine_tokens_backward(g, y, r, w.detach(), want_y=False)
    assert none is None and no is None and torch.equal(alone, gw)
    rows = torch.zeros_like(y)
    rows[dest[keep]] = (w.detach()[:, :, None] * g.float()[:, None]).to(dtype)[keep]
    assert torch.equal(gy, rows)


def test_shared_weights_and_one_row_for_all(pkg):
    """Gradients of expanded inputs are the sums over what they were expanded to. A token's sum has TOPK
    terms of cols products, the row's one of at most TOKENS * TOPK: as many roundings of the magnitudes'
    sum, and torch's own in its sums over the expanded dimension."""
    cols = 130
    r, _, keep = _routing(pkg, 7)
    n = keep.sum(1, keepdim=True)
    w = torch.rand((TOKENS, 1), generator=torch.Generator().manual_seed(1)).cuda().requires_grad_(True)
    y = S._randn((1, cols), 2, torch.float32).requires_grad_(True)
    g = S._randn((TOKENS, cols), 3, torch.float32)
    gw, gy = torch.autograd.grad(pkg.moe.combine_tokens(y.expand(r.rows, -1), r, w.expand(-1, TOPK)), (w, y), g)
    yd, gd, wd = y.detach().double(), g.double(), w.detach().double()
    mag = (gd * yd).abs().sum(1, keepdim=True) * n
    assert bool(((gw - (gd * yd).sum(1, keepdim=True) * n).abs() <= 1.01 * (cols + TOPK + 1) * S.U * mag).all())
    mag = (gd * wd * n).abs().sum(0, keepdim=True)
    assert bool(((gy - (gd * wd * n).sum(0, keepdim=True)).abs() <= 1.01 * (r.rows + 1) * S.U * mag).all())


def test_recomputed_and_repeated_backward(pkg):
    from torch.utils.checkpoint import checkpoint

    r, _, _ = _routing(pkg, 5)
    x = S._randn((TOKENS, 64), 1, torch.float32).requires_grad_(True)
    w = torch.rand((TOKENS, TOPK), device="cuda").requires_grad_(True)

    def step(x, w):
        return pkg.moe.combine_tokens(torch.tanh(pkg.moe.dispatch_tokens(x, r)), r, w).sum()

    loss = step(x, w)
    first = torch.autograd.grad(loss, (x, w), retain_graph=True)
    for again in (torch.autograd.grad(loss, (x, w)),
                  torch.autograd.grad(checkpoint(step, x, w, use_reentrant=False), (x, w))):
        assert all(torch.equal(a, b) for a, b in zip(first, again))

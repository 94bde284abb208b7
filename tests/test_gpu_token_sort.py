"""Token sort, its way back and their gradients on the GPU against 64-bit restatements.

Tolerances (u = 2^-24, h = eps / 2 of the rows' type): combine rounds a product and a sum per
slot (topk + 1 roundings of the sum of magnitudes) and the result once (h); a row gradient is
one product (u) rounded once (h); a weight gradient is a sum of `cols` products, at most
(cols + 1) u of the sum of their magnitudes.
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
CASES = [(1, 1, 1, 8), (1, 1, 1, 1), (45, 3, 6, 1030), (21, 2, 4, 260), (37, 2, 8, 515), (64, 4, 16, 512), (5, 9, 12, 96),
         (130, 3, 5, 2056), (40, 8, 64, 4096), (6, 17, 20, 33)]


def _ids(tokens, topk, experts, seed, drop=0.1):
    rng = np.random.default_rng(seed)
    ids = np.stack([rng.choice(experts, topk, replace=False) for _ in range(tokens)]) if tokens \
        else np.zeros((0, topk))
    ids[rng.random(ids.shape) < drop] = -1
    return torch.from_numpy(ids.astype(np.int32)).cuda()


def _np(t):
    return t.detach().double().cpu().numpy()


def _close(got, want, tol):
    err = np.abs(_np(got) - want)
    assert np.all(err <= tol), float((err - tol).max())


def _randn(shape, seed, dtype):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("tokens,topk,experts,cols", CASES)
def test_dispatch_and_gradient(pkg, tokens, topk, experts, cols, dtype):
    r = pkg.moe.route(_ids(tokens, topk, experts, tokens + cols), experts)
    dest = r.dest.cpu().numpy()
    x = _randn((tokens, cols), 1, dtype).requires_grad_(True)
    y = pkg.moe.dispatch_tokens(x, r)
    assert np.array_equal(_np(y), O.dispatch(_np(x), dest, r.rows, topk))
    gy = _randn((r.rows, cols), 2, dtype)
    (gx,) = torch.autograd.grad(y, x, gy)
    want = O.combine(_np(gy), dest, None, tokens, topk)
    mag = O.combine(np.abs(_np(gy)), dest, None, tokens, topk)
    _close(gx, want, 1.01 * ((topk + 1) * U * mag + HALF[dtype] * np.abs(want)) + TINY[dtype])
    assert torch.equal(gx, pkg.moe.dispatch_tokens_backward(gy, r))


@pytest.mark.parametrize("weights", ["fp32", "bf16", None])
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("tokens,topk,experts,cols", CASES)
def test_combine_and_gradients(pkg, tokens, topk, experts, cols, dtype, weights):
    r = pkg.moe.route(_ids(tokens, topk, experts, tokens + cols + 1), experts)
    dest = r.dest.cpu().numpy()
    y = _randn((r.rows, cols), 3, dtype).requires_grad_(True)
    w = None
    if weights is not None:
        w = _randn((tokens, topk), 4, torch.float32 if weights == "fp32" else torch.bfloat16)
        w.requires_grad_(True)
    out = pkg.moe.combine_tokens(y, r, w)
    wn = None if w is None else _np(w)
    h = HALF[dtype]
    want = O.combine(_np(y), dest, wn, tokens, topk)
    mag = O.combine(np.abs(_np(y)), dest, None if wn is None else np.abs(wn), tokens, topk)
    _close(out, want, 1.01 * ((topk + 1) * U * mag + h * np.abs(want)) + TINY[dtype])
    g = _randn((tokens, cols), 5, dtype)
    got = torch.autograd.grad(out, (y,) if w is None else (y, w), g)
    gy, gw = O.combine_backward(_np(g), _np(y), dest, wn, topk)
    _close(got[0], gy, 1.01 * (U + h) * np.abs(gy) + TINY[dtype])
    if w is not None:
        _, mag = O.combine_backward(np.abs(_np(g)), np.abs(_np(y)), dest, np.abs(wn), topk)
        assert got[1].dtype == w.dtype
        _close(got[1], gw, 1.01 * ((cols + 1) * U * mag + HALF[w.dtype] * np.abs(gw)) + 1e-37)


def test_gradients_against_differences(pkg):
    """combine is linear in the rows and in the weights: a central difference over a unit step
    is its derivative, up to the roundings of the two passes."""
    tokens, topk, experts, cols = 21, 3, 6, 136
    r = pkg.moe.route(_ids(tokens, topk, experts, 8), experts)
    y = _randn((r.rows, cols), 1, torch.float32).requires_grad_(True)
    w = _randn((tokens, topk), 2, torch.float32).requires_grad_(True)
    c = _randn((tokens, cols), 3, torch.float32)
    gy, gw = torch.autograd.grad(pkg.moe.combine_tokens(y, r, w), (y, w), c)
    dy, dw = _randn(tuple(y.shape), 4, torch.float32), _randn(tuple(w.shape), 5, torch.float32)

    def loss(yy, ww):
        return float((pkg.moe.combine_tokens(yy, r, ww).double() * c.double()).sum())

    size = float((pkg.moe.combine_tokens(y.detach().abs() + dy.abs(), r, w.detach().abs() + dw.abs())
                  .double() * c.double().abs()).sum())
    tol = 16 * (topk + cols) * U * size
    num = (loss(y.detach() + dy, w.detach()) - loss(y.detach() - dy, w.detach())) / 2
    assert abs(num - float((gy.double() * dy.double()).sum())) <= tol
    num = (loss(y.detach(), w.detach() + dw) - loss(y.detach(), w.detach() - dw)) / 2
    assert abs(num - float((gw.double() * dw.double()).sum())) <= tol


def test_rows_past_32_bits(pkg):
    """2.4e9 sorted elements: the last expert's rows and their gradients are where they belong."""
    tokens, cols = 150_000, 8000
    ids = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda").repeat(tokens, 1)
    r = pkg.moe.route(ids, 2)
    x = torch.arange(tokens, device="cuda", dtype=torch.float32)[:, None].expand(-1, cols)
    x = (x % 251).to(torch.bfloat16)
    y = pkg.moe.dispatch_tokens(x, r)
    for t in (0, 131_072, tokens - 1):
        for j in range(2):
            assert torch.equal(y[int(r.dest[2 * t + j])], x[t])
    w = torch.ones((tokens, 2), device="cuda")
    gy, gw = pkg.moe.combine_tokens_backward(x, y, r, w)
    assert torch.equal(gy[int(r.dest[2 * tokens - 1])], x[tokens - 1])
    t = tokens - 1
    want = float((x[t].double() ** 2).sum())
    assert abs(float(gw[t, 1]) - want) <= (cols + 1) * U * want
    del gy, gw
    out = pkg.moe.combine_tokens(y, r)
    assert torch.equal(out[t], (2 * x[t].float()).to(torch.bfloat16))


def test_same_expert_twice_and_everything_dropped(pkg):
    ids = torch.tensor([[1, 1], [-1, 7], [0, 1]], dtype=torch.int32, device="cuda")
    r = pkg.moe.route(ids, 2)
    x = _randn((3, 40), 1, torch.bfloat16).requires_grad_(True)
    y = pkg.moe.dispatch_tokens(x, r)
    (gx,) = torch.autograd.grad(y.sum(), x)  # an expanded gradient
    assert torch.equal(gx[:, 0].float().cpu(), torch.tensor([2.0, 0.0, 2.0]))
    r0 = pkg.moe.route(torch.full((3, 2), -1, dtype=torch.int32, device="cuda"), 2)
    assert r0.rows == 0
    y0 = pkg.moe.dispatch_tokens(x, r0)
    assert tuple(y0.shape) == (0, 40)
    w = _randn((3, 2), 2, torch.float32).requires_grad_(True)
    out = pkg.moe.combine_tokens(y0.detach().requires_grad_(True), r0, w)
    assert torch.all(out == 0)
    (gw,) = torch.autograd.grad(out.sum(), w)
    assert torch.all(gw == 0)
    assert torch.all(torch.autograd.grad(y0.sum(), x)[0] == 0)


def test_infinities_reach_only_their_token(pkg):
    ids = _ids(20, 2, 4, 3, drop=0.0)
    r = pkg.moe.route(ids, 4)
    y = _randn((r.rows, 64), 1, torch.float16)
    pad = r.src_rows[:r.rows] < 0
    y[pad] = float("nan")  # padding rows may hold anything
    w = _randn((20, 2), 2, torch.float32)
    out = pkg.moe.combine_tokens(y, r, w)
    assert torch.isfinite(out).all()
    gy, gw = pkg.moe.combine_tokens_backward(_randn((20, 64), 3, torch.float16), y, r, w)
    assert torch.isfinite(gw).all() and torch.all(gy[pad] == 0)
    y[int(r.dest[0])] = float("inf")
    out = pkg.moe.combine_tokens(y, r, w)
    assert torch.isfinite(out[1:]).all() and not torch.isfinite(out[0]).any()


def test_strides_streams_and_repeatability(pkg):
    r = pkg.moe.route(_ids(50, 4, 8, 1), 8)
    base = _randn((50, 300), 1, torch.bfloat16)
    x = base[:, 3:203]
    want = pkg.moe.dispatch_tokens(x.contiguous(), r)
    assert torch.equal(pkg.moe.dispatch_tokens(x, r), want)
    assert torch.equal(pkg.moe.dispatch_tokens(base.t()[3:203].t(), r), want)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    xs = x.contiguous().requires_grad_(True)
    torch.cuda.synchronize()
    y = pkg.moe.dispatch_tokens(xs, r, stream=side)
    out = pkg.moe.combine_tokens(y, r, stream=side)
    side.synchronize()
    assert torch.equal(y, want)
    (g,) = torch.autograd.grad(out, xs, torch.ones_like(out))
    torch.cuda.synchronize()
    kept = (r.dest.view(50, 4) >= 0).sum(1)
    assert torch.equal(g[:, 0].float(), kept.float())
    w = torch.rand((50, 4), generator=torch.Generator().manual_seed(1)).cuda()
    first = pkg.moe.combine_tokens_backward(x, want, r, w)
    for _ in range(3):
        again = pkg.moe.combine_tokens_backward(x, want, r, w)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_forward_and_gradients_in_a_graph(pkg):
    """Captured with the gradient functions, replayed on new contents."""
    r = pkg.moe.route(_ids(30, 2, 4, 5), 4)
    x, w, g = _randn((30, 72), 1, torch.bfloat16), torch.rand((30, 2), device="cuda"), _randn((30, 72), 2, torch.bfloat16)

    def step():
        y = pkg.moe.dispatch_tokens(x, r)
        out = pkg.moe.combine_tokens(y, r, w)
        gy, gw = pkg.moe.combine_tokens_backward(g, y, r, w)
        return out, gw, pkg.moe.dispatch_tokens_backward(gy, r)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (3, 4):
        x.copy_(_randn((30, 72), seed, torch.bfloat16))
        g.copy_(_randn((30, 72), seed + 10, torch.bfloat16))
        graph.replay()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_autograd_captured_in_a_graph(pkg):
    """A whole training step (forward and autograd backward) in a graph, as torch asks for it:
    leaves whose first eager graph is gone, warm-up on a side stream."""
    r = pkg.moe.route(_ids(30, 2, 4, 5), 4)
    x = _randn((30, 72), 1, torch.float32).requires_grad_(True)
    w = torch.rand((30, 2), device="cuda").requires_grad_(True)

    def step():
        out = pkg.moe.combine_tokens(torch.tanh(pkg.moe.dispatch_tokens(x, r)), r, w)
        return torch.autograd.grad(out.square().sum(), (x, w))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_second_gradients(pkg):
    """Without weights both operators are linear and differentiable again; with weights the
    second gradient is refused."""
    r = pkg.moe.route(_ids(12, 2, 4, 5), 4)
    x = _randn((12, 24), 1, torch.float32).requires_grad_(True)
    y = pkg.moe.dispatch_tokens(x, r)
    gy = _randn(tuple(y.shape), 2, torch.float32).requires_grad_(True)
    (gx,) = torch.autograd.grad(y, x, gy, create_graph=True)
    c = _randn((12, 24), 3, torch.float32)
    (ggy,) = torch.autograd.grad(gx, gy, c)
    assert torch.equal(ggy, pkg.moe.dispatch_tokens(c, r))
    out = pkg.moe.combine_tokens(gy, r)
    (g1,) = torch.autograd.grad(out, gy, c.requires_grad_(True), create_graph=True)
    (g2,) = torch.autograd.grad(g1, c, gy.detach())
    assert torch.equal(g2, out)
    w = torch.rand((12, 2), device="cuda").requires_grad_(True)
    (g3,) = torch.autograd.grad(pkg.moe.combine_tokens(gy, r, w), gy, c, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g3.sum().backward()

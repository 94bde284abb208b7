"""The int8 operators together: the MoE block against its stages and a dense restatement, and a
training step through the token sort."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _setup(pkg, tokens, topk, E, H, I, dtype, seed, drop=0.05):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((tokens, H), generator=g).to(dtype).cuda()
    gate, up = ((torch.randn((E, I, H), generator=g) * H ** -0.5).to(dtype).cuda() for _ in range(2))
    down = (torch.randn((E, H, I), generator=g) * I ** -0.5).to(dtype).cuda()
    rng = np.random.default_rng(seed)
    ids = np.stack([rng.choice(E, topk, replace=False) for _ in range(tokens)])
    ids[rng.random(ids.shape) < drop] = -1
    w = torch.softmax(torch.randn((tokens, topk), generator=g), 1).cuda()
    return x, gate, up, down, torch.from_numpy(ids.astype(np.int32)).cuda(), w


@pytest.mark.parametrize("tokens,topk,E,H,I,dtype", [
    (1, 2, 4, 64, 48, torch.bfloat16), (37, 2, 6, 200, 136, torch.float16),
    (64, 8, 64, 512, 192, torch.bfloat16), (600, 4, 8, 515, 333, torch.bfloat16)])
def test_block_equals_its_stages_and_follows_the_dense_form(pkg, tokens, topk, E, H, I, dtype):
    x, gate, up, down, ids, w = _setup(pkg, tokens, topk, E, H, I, dtype, tokens + H)
    W = pkg.moe.quantize_expert_weights_int8(list(gate), list(up), list(down))
    blk = pkg.moe.Int8MoEBlock(W, tokens, topk, dtype)
    out = blk.run(x, ids, w).clone()
    assert blk.check_device_errors() == 0
    r = pkg.moe.route(ids, E)
    a, sa = pkg.moe.dispatch_int8(x, r)
    # Dispatching codes is quantising the dispatched rows (padding rows aside).
    q2, s2 = pkg.quantize_int8(pkg.moe.dispatch_tokens(x, r))
    real = r.src_rows[:r.rows] >= 0
    assert torch.equal(a[real], q2[real]) and torch.equal(sa[real], s2[real])
    off = torch.tensor(r.offsets[:E], dtype=torch.int32, device="cuda")
    cnt = torch.tensor(r.counts, dtype=torch.int32, device="cuda")
    h = torch.zeros((r.rows, I), dtype=dtype, device="cuda")
    pkg.int8_gemm_segments(a, sa, W.w_gate, W.s_gate, off, cnt, b2=W.w_up, b2_scale=W.s_up, out=h,
                           expected_rows=tokens * topk)
    a2, sa2 = pkg.quantize_int8(h)
    y = pkg.int8_gemm_segments(a2, sa2, W.w_down, W.s_down, off, cnt, out_dtype=dtype,
                               expected_rows=tokens * topk)
    assert torch.equal(pkg.moe.combine_tokens(y, r, w), out)
    # The dense computation in 64 bits. Each quantisation is off by at most half a step of the
    # row's 127 (relative to its largest value): the whole stays within a few percent.
    ref = torch.zeros((tokens, H), dtype=torch.float64, device="cuda")
    for t_slot in range(topk):
        for e in range(E):
            sel = (ids[:, t_slot] == e).nonzero().flatten()
            if sel.numel():
                xs = x[sel].double()
                hh = torch.nn.functional.silu(xs @ gate[e].double().t()) * (xs @ up[e].double().t())
                ref[sel] += w[sel, t_slot, None].double() * (hh @ down[e].double().t())
    rel = float(torch.linalg.norm(out.double() - ref) / torch.linalg.norm(ref))
    assert rel < 0.05, rel


def test_block_captured_and_replayed_on_new_inputs(pkg):
    x, gate, up, down, ids, w = _setup(pkg, 40, 4, 8, 256, 128, torch.bfloat16, 3)
    W = pkg.moe.quantize_expert_weights_int8(gate, up, down)
    a, b = pkg.moe.Int8MoEBlock(W, 40, 4), pkg.moe.Int8MoEBlock(W, 40, 4)
    graphs = [blk.capture(x, ids, w) for blk in (a, b)]
    for seed in (5, 6):
        x2, _, _, _, ids2, w2 = _setup(pkg, 40, 4, 8, 256, 128, torch.bfloat16, seed)
        x.copy_(x2), ids.copy_(ids2), w.copy_(w2)
        want = pkg.moe.Int8MoEBlock(W, 40, 4).run(x2, ids2, w2)
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for st, g in zip(streams, graphs):  # both graphs at once
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(a.out, want) and torch.equal(b.out, want)


def test_training_step_through_the_token_sort(pkg):
    """Experts in torch between dispatch and combine: gradients of the tokens, the experts'
    weights and the routing weights equal those of the dense formula in 64 bits."""
    T, K, E, H = 33, 2, 4, 48
    x, _, _, _, ids, w = _setup(pkg, T, K, E, H, 8, torch.bfloat16, 9)
    x = x.float().requires_grad_(True)
    w = w.clone().requires_grad_(True)
    experts = (torch.randn((E, H, H), generator=torch.Generator().manual_seed(1)) * H ** -0.5).cuda()
    experts.requires_grad_(True)
    r = pkg.moe.route(ids, E)
    rows = pkg.moe.dispatch_tokens(x, r)
    parts = [torch.tanh(rows[r.offsets[e]:r.offsets[e + 1]].double() @ experts[e].double()).float()
             for e in range(E)]
    out = pkg.moe.combine_tokens(torch.cat(parts), r, w)
    got = torch.autograd.grad(out.double().square().sum(), (x, experts, w))
    xd, ed, wd = (t.detach().double().requires_grad_(True) for t in (x, experts, w))
    keep = (ids >= 0).double()
    eid = ids.clamp(min=0).long()
    y = torch.tanh(torch.einsum("th,tkhj->tkj", xd, ed[eid]))
    ref = ((wd * keep)[:, :, None] * y).sum(1)
    want = torch.autograd.grad(ref.square().sum(), (xd, ed, wd))
    u = 2.0 ** -24
    # A dozen fp32 roundings lie between the inputs and each gradient, each of a sum of at most
    # T * H terms: their norms stay together within 16 u sqrt(T H).
    for a, b in zip(got, want):
        rel = float(torch.linalg.norm(a.double() - b) / torch.linalg.norm(b))
        assert rel <= 16 * u * (T * H) ** 0.5, rel


def test_block_with_everything_dropped_and_one_expert_twice(pkg):
    x, gate, up, down, ids, w = _setup(pkg, 20, 2, 4, 64, 32, torch.bfloat16, 2, drop=0.0)
    W = pkg.moe.quantize_expert_weights_int8(gate, up, down)
    blk = pkg.moe.Int8MoEBlock(W, 20, 2)
    first = blk.run(x, ids, w).clone()
    assert torch.all(blk.run(x, torch.full_like(ids, -1), w) == 0)
    assert torch.equal(blk.run(x, ids, w), first)  # nothing of the empty run stays
    twice = ids[:, :1].repeat(1, 2).contiguous()
    half = torch.full((20, 2), 0.5, device="cuda")
    both = blk.run(x, twice, half).clone()
    once = blk.run(x, torch.cat([ids[:, :1], torch.full_like(ids[:, :1], -1)], 1).contiguous(),
                   torch.ones((20, 2), device="cuda"))
    assert torch.equal(both, once)  # 0.5 y + 0.5 y is exact
    assert blk.check_device_errors() == 0


def test_block_on_a_stream_of_its_own(pkg):
    """The caller's stream differs from the current one; weights in another type are converted on it."""
    x, gate, up, down, ids, w = _setup(pkg, 30, 2, 4, 96, 64, torch.float16, 4)
    W = pkg.moe.quantize_expert_weights_int8(gate, up, down)
    blk = pkg.moe.Int8MoEBlock(W, 30, 2, torch.float16)
    want = blk.run(x, ids, w.to(torch.bfloat16)).clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        blk.out.zero_()
        side.wait_stream(torch.cuda.current_stream())
        out = blk.run(x, ids, w.to(torch.bfloat16), stream=side)
        side.synchronize()
        assert torch.equal(out, want)


def test_operators_on_two_streams_at_once(pkg):
    """Quantiser, dispatch, products and combine hold no state that two streams could share."""
    cases = []
    for seed, (T, H) in enumerate(((500, 512), (33, 1024))):
        x, gate, up, down, ids, w = _setup(pkg, T, 2, 4, H, 128, torch.bfloat16, seed)
        W = pkg.moe.quantize_expert_weights_int8(gate, up, down)
        r = pkg.moe.route(ids, 4)
        off = torch.tensor(r.offsets[:4], dtype=torch.int32, device="cuda")
        cnt = torch.tensor(r.counts, dtype=torch.int32, device="cuda")
        cases.append((x, W, r, off, cnt, w))

    def chain(case, st):
        x, W, r, off, cnt, w = case
        a, sa = pkg.moe.dispatch_int8(x, r, stream=st)
        h = pkg.int8_gemm_segments(a, sa, W.w_gate, W.s_gate, off, cnt, b2=W.w_up, b2_scale=W.s_up,
                                   stream=st)
        a2, sa2 = pkg.quantize_int8(h, row_list=r.dest, stream=st)
        y = pkg.int8_gemm_segments(a2, sa2, W.w_down, W.s_down, off, cnt, stream=st)
        return pkg.moe.combine_tokens(y, r, w, stream=st)

    want = [chain(c, None) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        got = [chain(c, st) for c, st in zip(cases, streams)]
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_rows_outside_segments_may_hold_anything(pkg):
    """Padding rows with NaN scales and any codes neither reach a result nor are written."""
    x, gate, up, down, ids, w = _setup(pkg, 50, 2, 4, 160, 96, torch.bfloat16, 8)
    W = pkg.moe.quantize_expert_weights_int8(gate, up, down)
    r = pkg.moe.route(ids, 4)
    off = torch.tensor(r.offsets[:4], dtype=torch.int32, device="cuda")
    cnt = torch.tensor(r.counts, dtype=torch.int32, device="cuda")
    a, sa = pkg.moe.dispatch_int8(x, r)
    pad = r.src_rows[:r.rows] < 0
    outs = []
    for fill, scale in ((0, 0.0), (127, float("nan")), (-128, float("inf"))):
        a[pad] = fill
        sa[pad] = scale
        out = torch.full((r.rows, 96), 7.0, dtype=torch.bfloat16, device="cuda")
        pkg.int8_gemm_segments(a, sa, W.w_gate, W.s_gate, off, cnt, b2=W.w_up, b2_scale=W.s_up, out=out)
        assert torch.all(out[pad] == 7.0) and torch.isfinite(out).all()
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])

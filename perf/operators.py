"""The int8 and token-sorting operators: their cases, inputs, plain forms and work.

Five operators are measured, over the sizes that an MoE layer gives them (hidden 4096 or 7168,
experts' intermediate 1536 or 2048, up to 8192 tokens with top-8 routing over 64 experts):

  quantise   rows of activations to int8 codes with one scale per token; with ``topk`` > 0 the
             codes go straight to every expert's rows (the serving form of the dispatch)
  product    ``a_scale[m] * b_scale[n] * sum_k a[m, k] b[n, k] + bias[n]`` of int8 operands
  experts    the same product over the rows of every expert, their counts read on the GPU;
             gated: ``silu(gate) * up`` of two weight sets
  dispatch   tokens sorted by expert (padding rows zero) and the gradient of the tokens
  combine    expert rows back to tokens with weights applied, and the gradients of rows and weights

``run`` computes the plain form of a case where ``own`` is false and calls the framework where
it is true; both take what ``prepare`` gives.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# --------------------------------------------------------------------------- cases
def listed():
    """The listed cases."""
    return [
        # A decode step of eight sequences: the activations of a layer before its projection.
        dict(name="quantise_decode", op="quantise", tokens=8, cols=7168, dtype="bf16", topk=0, experts=0, skew=0.0, drop=0.0),
        # A prompt batch sent to its experts as codes (64 experts, top-8).
        dict(name="quantise_dispatch_prompt", op="quantise", tokens=8192, cols=4096, dtype="bf16", topk=8, experts=64, skew=0.0, drop=0.0),
        # One token through a projection: bound by the stream of the weights.
        dict(name="product_one_token", op="product", m=1, n=4096, k=7168, dtype="bf16", bias=False),
        # A small ragged batch; no size is a multiple of a tile, rows of the output are unaligned.
        dict(name="product_odd", op="product", m=83, n=4099, k=2011, dtype="fp16", bias=True),
        # A prompt of 8192 tokens through the same projection: bound by the tensor cores.
        dict(name="product_prompt", op="product", m=8192, n=4096, k=7168, dtype="bf16", bias=False),
        # Gate and up projections of a decode step: 64 tokens, top-8 of 64 experts, skewed routing.
        dict(name="experts_decode_gated", op="experts", tokens=64, topk=8, experts=64, n=1536, k=4096, dtype="bf16", gated=True, skew=1.2, drop=0.0),
        # Down projection of a middling batch with skewed routing.
        dict(name="experts_down", op="experts", tokens=512, topk=8, experts=64, n=4096, k=1536, dtype="fp16", gated=False, skew=1.2, drop=0.0),
        # Gate and up projections of a prompt batch.
        dict(name="experts_prompt_gated", op="experts", tokens=8192, topk=8, experts=64, n=1536, k=4096, dtype="bf16", gated=True, skew=0.0, drop=0.0),
        # Training: a small batch in fp32 whose row length no vector divides, with dropped pairs.
        dict(name="dispatch_odd", op="dispatch", tokens=37, topk=2, experts=8, cols=515, dtype="fp32", skew=1.1, drop=0.1),
        # Training: a batch of 8192 tokens.
        dict(name="dispatch_train", op="dispatch", tokens=8192, topk=8, experts=64, cols=4096, dtype="bf16", skew=0.0, drop=0.0),
        # Training: a middling fp16 batch with skewed routing and dropped pairs.
        dict(name="combine_skewed", op="combine", tokens=300, topk=4, experts=16, cols=1536, dtype="fp16", skew=1.2, drop=0.05),
        # Training: a batch of 8192 tokens.
        dict(name="combine_train", op="combine", tokens=8192, topk=8, experts=64, cols=4096, dtype="bf16", skew=0.0, drop=0.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the ranges that the listed ones stand for."""
    op = rng.choice(["quantise", "product", "experts", "dispatch", "combine"])
    if op == "product":
        c = dict(op=op, m=_log_int(rng, 1, 8192), n=_log_int(rng, 64, 8192), k=_log_int(rng, 64, 8192),
                 dtype=rng.choice(["bf16", "fp16", "fp32"]), bias=rng.random() < 0.5)
        while c["m"] * c["n"] * c["k"] > 8192 * 4096 * 7168:
            c["m"] = c["m"] // 2 + 1
        return c
    experts = _log_int(rng, 2, 64)
    route = dict(topk=rng.randint(1, min(8, experts)), experts=experts, skew=rng.choice([0.0, 0.8, 1.2]),
                 drop=rng.choice([0.0, 0.05]))
    if op == "experts":
        c = dict(op=op, tokens=_log_int(rng, 1, 8192), n=_log_int(rng, 64, 4096), k=_log_int(rng, 64, 4096),
                 dtype=rng.choice(["bf16", "fp16", "fp32"]), gated=rng.random() < 0.5, **route)
        # The plain form pads every expert to the longest: keep that, too, within the largest case.
        while c["tokens"] * c["experts"] * c["n"] * c["k"] > 8192 * 8 * 3 * 1536 * 4096:
            c["tokens"] = c["tokens"] // 2 + 1
            c["n"] = max(64, c["n"] * 7 // 8)
        return c
    if op == "quantise":
        if rng.random() < 0.5:
            route = dict(topk=0, experts=0, skew=0.0, drop=0.0)
        return dict(op=op, tokens=_log_int(rng, 1, 8192), cols=_log_int(rng, 64, 4096 if route["topk"] else 8192),
                    dtype=rng.choice(["bf16", "fp16"]), **route)
    c = dict(op=op, tokens=_log_int(rng, 1, 8192), cols=_log_int(rng, 64, 4096),
             dtype=rng.choice(["bf16", "fp16", "fp32"]), **route)
    if c["dtype"] == "fp32":
        c["cols"] = min(c["cols"], 2047)
    return c


# --------------------------------------------------------------------------- inputs
def _round_up(v, q):
    return (v + q - 1) // q * q


def _gen(case, seed):
    return torch.Generator(device="cuda").manual_seed(1009 * seed + 17)


def _codes(gen, rows, cols, spread=40.0):
    """int8 codes [rows, cols] as a quantiser leaves them: bell-shaped, rows a multiple of 16 bytes apart."""
    buf = torch.randn((rows, _round_up(cols, 16)), generator=gen, device="cuda")
    return (buf * spread).round_().clamp_(-127, 127).to(torch.int8)[:, :cols]


def _scales(gen, n, level):
    return (0.25 + torch.rand(n, generator=gen, device="cuda")) * level


def _routing(gen, tokens, topk, experts, skew, drop):
    """Routing metadata of a random batch: every token picks ``topk`` different experts, popular
    ones more often (``skew``); a share ``drop`` of the pairs is dropped. Each expert's rows start
    on a multiple of 128, in token order; ``src`` is -1 on padding rows. The picks are the case's
    (outputs of every seed have one shape); the seed says which token made which."""
    pairs = tokens * topk
    order = torch.randperm(tokens, generator=gen, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(7919 * tokens + 31 * experts + topk)
    logits = -skew * torch.log(torch.arange(1, experts + 1, device="cuda", dtype=torch.float32))
    gumbel = -torch.log(-torch.log(torch.rand((tokens, experts), generator=gen, device="cuda").clamp_(1e-7, 1 - 1e-6)))
    ids = torch.topk(logits + gumbel, topk, dim=1).indices
    ids = torch.where(torch.rand((tokens, topk), generator=gen, device="cuda") < drop, experts, ids)[order].flatten()
    order = torch.argsort(ids, stable=True)
    counts = torch.bincount(ids, minlength=experts + 1)[:experts]
    first = torch.cumsum(counts, 0) - counts
    padded = (counts + 127) // 128 * 128
    ends = torch.cumsum(padded, 0)
    offsets = torch.cat([ends.new_zeros(1), ends])
    rows = int(offsets[-1])
    expert = ids[order]
    inside = expert < experts
    e = expert.clamp(max=experts - 1)
    row = torch.where(inside, offsets[e] + torch.arange(pairs, device="cuda") - first[e], -1)
    dest = torch.empty(pairs, dtype=torch.int32, device="cuda")
    dest[order] = row.to(torch.int32)
    src = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    src[row[inside]] = (order[inside] // topk).to(torch.int32)
    return dict(tokens=tokens, topk=topk, experts=experts, rows=rows, counts=counts.to(torch.int32),
                offsets=offsets.to(torch.int32), dest=dest, src=src, host_counts=counts.tolist(),
                host_offsets=offsets.tolist())


def _activations(gen, tokens, cols, dtype):
    """Activations with tokens of different size and a few channels far above the rest."""
    x = torch.randn((tokens, cols), generator=gen, device="cuda")
    x *= torch.exp(torch.randn((tokens, 1), generator=gen, device="cuda"))
    x *= 1.0 + 9.0 * (torch.rand((1, cols), generator=gen, device="cuda") < 0.002)
    return x.to(_DTYPES[dtype])


def prepare(case, seed):
    """Inputs of a case, from the seed alone."""
    gen = _gen(case, seed)
    op = case["op"]
    s = dict(case=case)
    if op == "product":
        s["a"], s["b"] = _codes(gen, case["m"], case["k"]), _codes(gen, case["n"], case["k"])
        s["a_scale"] = _scales(gen, case["m"], 1.0 / 40)
        s["b_scale"] = _scales(gen, case["n"], 1.0 / (40 * math.sqrt(case["k"])))
        s["bias"] = torch.randn(case["n"], generator=gen, device="cuda") if case["bias"] else None
        return s
    if case["topk"]:
        s["routing"] = _routing(gen, case["tokens"], case["topk"], case["experts"], case["skew"], case["drop"])
    rows = s["routing"]["rows"] if case["topk"] else case["tokens"]
    if op == "experts":
        n, k, e = case["n"], case["k"], case["experts"]
        s["a"], s["a_scale"] = _codes(gen, rows, k), _scales(gen, rows, 1.0 / 40)
        level = 1.0 / (40 * math.sqrt(k))
        for name in ("b", "b2") if case["gated"] else ("b",):
            buf = torch.empty((e, n, _round_up(k, 16)), dtype=torch.int8, device="cuda")
            for i in range(e):  # one expert at a time: no wide temporary of all the weights
                buf[i, :, :k] = _codes(gen, n, k)
            s[name], s[name + "_scale"] = buf[:, :, :k], _scales(gen, e * n, level).view(e, n)
        s["out"] = torch.zeros((rows, n), dtype=_DTYPES[case["dtype"]], device="cuda")
    elif op == "quantise":
        s["x"] = _activations(gen, case["tokens"], case["cols"], case["dtype"])
        s["codes"] = torch.zeros((rows, _round_up(case["cols"], 16)), dtype=torch.int8, device="cuda")[:, :case["cols"]]
        s["scales"] = torch.zeros(rows, dtype=torch.float32, device="cuda")
    elif op == "dispatch":
        s["x"] = _activations(gen, case["tokens"], case["cols"], case["dtype"]).requires_grad_(True)
        s["grad"] = torch.randn((rows, case["cols"]), generator=gen, device="cuda").to(_DTYPES[case["dtype"]])
    else:
        s["y"] = torch.randn((rows, case["cols"]), generator=gen, device="cuda").to(_DTYPES[case["dtype"]]).requires_grad_(True)
        w = torch.softmax(torch.randn((case["tokens"], case["topk"]), generator=gen, device="cuda"), dim=1)
        s["weights"] = w.requires_grad_(True)
        s["grad"] = torch.randn((case["tokens"], case["cols"]), generator=gen, device="cuda").to(_DTYPES[case["dtype"]])
    return s


# --------------------------------------------------------------------------- one pass
def run(s):
    """One pass of the case's operator and its outputs."""
    if own:
        return _own(s)
    with torch.no_grad():
        return {"quantise": _plain_quantise, "product": _plain_product, "experts": _plain_experts,
                "dispatch": _plain_dispatch, "combine": _plain_combine}[s["case"]["op"]](s)


def _own(s):
    import submission

    nv = submission.load_package()
    case, r = s["case"], s.get("routing")
    op, dtype = case["op"], _DTYPES[case["dtype"]]
    if op == "product":
        return nv.int8_gemm(s["a"], s["a_scale"], s["b"], s["b_scale"], bias=s["bias"], out_dtype=dtype)
    if op == "experts":
        return nv.int8_gemm_segments(s["a"], s["a_scale"], s["b"], s["b_scale"], r["offsets"], r["counts"],
                                     b2=s.get("b2"), b2_scale=s.get("b2_scale"), out=s["out"],
                                     expected_rows=r["tokens"] * r["topk"])
    routing = None
    if r is not None:
        routing = nv.moe.Routing(r["tokens"], r["topk"], r["experts"], r["host_counts"], r["host_offsets"],
                                 r["dest"], r["src"])
    if op == "quantise":
        if routing is None:
            return nv.quantize_int8(s["x"], codes=s["codes"], scales=s["scales"])
        return nv.moe.dispatch_int8(s["x"], routing, codes=s["codes"], scales=s["scales"])
    if op == "dispatch":
        y = nv.moe.dispatch_tokens(s["x"], routing)
        return y.detach(), *torch.autograd.grad(y, s["x"], s["grad"])
    out = nv.moe.combine_tokens(s["y"], routing, s["weights"])
    return out.detach(), *torch.autograd.grad(out, (s["y"], s["weights"]), s["grad"])


def _plain_quantise(s):
    x = s["x"].float()
    amax = x.abs().amax(dim=1, keepdim=True)
    # x * 127 is exact in 32 bits for 16-bit inputs, so the quotient is rounded once before it is
    # rounded to a code: ties of the definition stay ties.
    codes = torch.where(amax > 0, torch.round(x * 127.0 / amax), 0.0).to(torch.int8)
    scales = (amax / 127.0).flatten()
    if "routing" in s:
        src = s["routing"]["src"].long()
        real, at = src >= 0, src.clamp(min=0)
        codes = torch.where(real[:, None], codes[at], 0)
        scales = torch.where(real, scales[at], 0.0)
    return codes, scales


def _plain_product(s):
    out = (s["a"].float() @ s["b"].float().t()) * s["a_scale"][:, None] * s["b_scale"]
    if s["bias"] is not None:
        out = out + s["bias"]
    return out.to(_DTYPES[s["case"]["dtype"]])


def _plain_experts(s):
    r = s["routing"]
    longest = max(r["host_counts"])
    at = torch.arange(longest, device="cuda")
    real = at < r["counts"][:, None]                                      # [experts, longest]
    row = torch.where(real, r["offsets"][:-1, None] + at, r["rows"])      # the row past the end: dropped
    read = row.clamp(max=max(r["rows"] - 1, 0))
    a, a_scale = s["a"].float()[read], s["a_scale"][read][:, :, None]
    y = torch.bmm(a, s["b"].float().transpose(1, 2)) * a_scale * s["b_scale"][:, None, :]
    if "b2" in s:
        up = torch.bmm(a, s["b2"].float().transpose(1, 2)) * a_scale * s["b2_scale"][:, None, :]
        y = y / (1.0 + torch.exp(-y)) * up
    out = torch.zeros((r["rows"] + 1, y.shape[2]), dtype=_DTYPES[s["case"]["dtype"]], device="cuda")
    out[row.flatten().long()] = y.to(out.dtype).flatten(0, 1)
    return out[:r["rows"]]


def _by_token(s, rows):
    """``rows`` of every (token, slot) pair in 32 bits, zero for dropped pairs: [tokens, topk, cols]."""
    r = s["routing"]
    dest = r["dest"].long().view(r["tokens"], r["topk"])
    return torch.where((dest >= 0)[:, :, None], rows[dest.clamp(min=0)].float(), 0.0)


def _plain_dispatch(s):
    src = s["routing"]["src"].long()
    y = torch.where((src >= 0)[:, None], s["x"][src.clamp(min=0)], 0.0)
    return y, _by_token(s, s["grad"]).sum(dim=1).to(y.dtype)


def _plain_combine(s):
    r, w, grad = s["routing"], s["weights"], s["grad"]
    rows = _by_token(s, s["y"])
    out = (rows * w[:, :, None]).sum(dim=1).to(s["y"].dtype)
    grad_w = (rows * grad.float()[:, None, :]).sum(dim=2)
    dest = r["dest"].long()
    grad_y = torch.zeros((r["rows"] + 1, grad.shape[1]), dtype=grad.dtype, device="cuda")
    pair = (w[:, :, None] * grad.float()[:, None, :]).to(grad.dtype).flatten(0, 1)
    grad_y[torch.where(dest >= 0, dest, r["rows"])] = pair
    return out, grad_y[:r["rows"]], grad_w


# --------------------------------------------------------------------------- work
def _route_sizes(case):
    """Expected (kept pairs, experts with a row, padding rows) of a case's routing."""
    pairs = case["tokens"] * case["topk"] * (1.0 - case["drop"])
    weights = [(i + 1) ** -case["skew"] for i in range(case["experts"])]
    top = sum(weights)
    used = sum(1.0 - math.exp(-pairs * w / top) for w in weights)
    return pairs, used, 63.5 * used


def work(case):
    """Bytes and operations that one pass cannot do without (expected values where the routing decides)."""
    op, es = case["op"], _BYTES[case["dtype"]]
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * (m + n) + (4 * n if case["bias"] else 0) + m * n * es, "flops": 2 * m * n * k}
    t, k = case["tokens"], case["topk"]
    if op == "quantise" and not k:
        return {"bytes": t * case["cols"] * (es + 1) + 4 * t, "flops": 3 * t * case["cols"]}
    pairs, used, padding = _route_sizes(case)
    if op == "experts":
        sets = 2 if case["gated"] else 1
        size = case["n"] * case["k"]
        return {"bytes": pairs * (case["k"] + 4) + used * sets * (size + 4 * case["n"]) + pairs * case["n"] * es,
                "flops": 2 * sets * pairs * size}
    cols = case["cols"]
    if op == "quantise":
        return {"bytes": t * cols * es + pairs * (cols + 4) + 4 * t * k, "flops": 3 * t * cols}
    if op == "dispatch":  # tokens and gradient rows read; rows with their padding and token gradients written
        return {"bytes": es * cols * (t + pairs + padding + pairs + t) + 8 * t * k, "flops": pairs * cols}
    # Rows read for the sum and, with the sum's gradient, again for the weights' gradient; sums and row gradients written.
    return {"bytes": es * cols * (pairs + t + t + pairs + pairs + padding) + 16 * t * k, "flops": 5 * pairs * cols}


# --------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    """The outputs from the operators' definitions in 64 bits."""
    s = prepare(case, seed)
    f64 = torch.float64
    op = case["op"]
    if op == "product":
        out = torch.einsum("mk,nk->mn", s["a"].to(f64), s["b"].to(f64))
        out = out * torch.outer(s["a_scale"].to(f64), s["b_scale"].to(f64))
        return out if s["bias"] is None else out + s["bias"].to(f64)
    r = s.get("routing")
    if op == "quantise":
        x = s["x"].to(f64)
        scale = x.abs().max(dim=1).values / 127
        q = (x * 127) / torch.clamp(x.abs().max(dim=1).values, min=1e-300)[:, None]
        low = torch.floor(q)  # nearest code, ties to the even one
        gap = q - low
        up = (gap > 0.5) | ((gap == 0.5) & (low.remainder(2) == 1))
        codes = (low + up.to(f64)).to(torch.int8)
        if r is None:
            return codes, scale
        rows, row_scales = torch.zeros((r["rows"], case["cols"]), dtype=torch.int8, device="cuda"), torch.zeros(r["rows"], dtype=f64, device="cuda")
        for j in range(case["topk"]):
            d = r["dest"].long().view(-1, case["topk"])[:, j]
            keep = d >= 0
            rows[d[keep]], row_scales[d[keep]] = codes[keep], scale[keep]
        return rows, row_scales
    if op == "experts":
        out = torch.zeros((r["rows"], case["n"]), dtype=f64, device="cuda")
        for e, count in enumerate(r["host_counts"]):
            if count:
                part = slice(r["host_offsets"][e], r["host_offsets"][e] + count)
                a = s["a"][part].to(f64) * s["a_scale"][part].to(f64)[:, None]
                y = a @ (s["b"][e].to(f64) * s["b_scale"][e].to(f64)[:, None]).t()
                if case["gated"]:
                    y = y * torch.sigmoid(y) * (a @ (s["b2"][e].to(f64) * s["b2_scale"][e].to(f64)[:, None]).t())
                out[part] = y
        return out
    with torch.no_grad():
        grad = s["grad"].to(f64)
        dest = r["dest"].long().view(case["tokens"], case["topk"])
        if op == "dispatch":
            y = torch.zeros((r["rows"], case["cols"]), dtype=f64, device="cuda")
            gx = torch.zeros((case["tokens"], case["cols"]), dtype=f64, device="cuda")
            for j in range(case["topk"]):
                keep = dest[:, j] >= 0
                y[dest[keep, j]] = s["x"].to(f64)[keep]
                gx[keep] += grad[dest[keep, j]]
            return y, gx
        y, w = s["y"].to(f64), s["weights"].to(f64)
        out = torch.zeros((case["tokens"], case["cols"]), dtype=f64, device="cuda")
        gy, gw = torch.zeros_like(y), torch.zeros_like(w)
        for j in range(case["topk"]):
            keep = dest[:, j] >= 0
            d = dest[keep, j]
            out[keep] += w[keep, j, None] * y[d]
            gy[d] = w[keep, j, None] * grad[keep]
            gw[keep, j] = (grad[keep] * y[d]).sum(dim=1)
        return out, gy, gw

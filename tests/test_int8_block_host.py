"""Host side of the int8 MoE block, with tensors, streams and the library replaced (CPU only)."""
from __future__ import annotations

import contextlib
import types

import torch


class _Tensor:
    """What the block's host code asks of a tensor, and the streams it was recorded on."""

    def __init__(self, shape, dtype):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, torch.device("cuda", 0)
        self.recorded = []

    def stride(self, i):
        return 1 if i == len(self.shape) - 1 else self.shape[-1]

    def get_device(self):
        return 0

    def data_ptr(self):
        return 0x1000

    def is_contiguous(self):
        return True

    def record_stream(self, stream):
        self.recorded.append(stream)

    def copy_(self, _):
        return self


def _block(pkg, monkeypatch, tokens=3, topk=2, E=4, hidden=16, inter=8):
    moe = pkg.moe
    device, current = torch.device("cuda", 0), types.SimpleNamespace(cuda_stream=7, device=torch.device("cuda", 0))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: current)
    monkeypatch.setattr(torch.cuda, "device", lambda *a: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "stream", lambda *a: contextlib.nullcontext())
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 7, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(moe, "int8_gemm_segments", lambda *a, **k: None)
    monkeypatch.setattr(moe, "quantize_int8", lambda *a, **k: None)
    blk = object.__new__(moe.Int8MoEBlock)
    blk.tokens, blk.topk, blk.num_experts, blk.hidden, blk.intermediate = tokens, topk, E, hidden, inter
    blk.dtype, blk.device = torch.bfloat16, device
    cap = blk.capacity = tokens * topk + 127 * E
    i32, bf = torch.int32, torch.bfloat16
    for name, shape, dtype in (("_meta", (2 * E + 1,), i32), ("counts", (E,), i32), ("offsets", (E + 1,), i32),
                               ("dest", (tokens * topk,), i32), ("src_rows", (cap,), i32),
                               ("_route_ws", (64,), torch.uint8), ("_a", (cap, 16), torch.int8),
                               ("_a_scale", (cap,), torch.float32), ("_h", (cap, inter), bf),
                               ("_a2", (cap, 16), torch.int8), ("_a2_scale", (cap,), torch.float32),
                               ("_y", (cap, hidden), bf), ("_w", (tokens, topk), torch.float32),
                               ("out", (tokens, hidden), bf), ("_errors", (1,), i32)):
        setattr(blk, name, _Tensor(shape, dtype))
    blk._route_ws_bytes = 64
    blk._weights = types.SimpleNamespace(**{k: _Tensor((E, 8, 16), torch.int8) for k in (
        "w_gate", "w_up", "w_down", "s_gate", "s_up", "s_down")})
    blk._lib = types.SimpleNamespace(**{k: lambda *a: 0 for k in (
        "nvfp4_moe_route", "nvfp4_moe_dispatch_int8", "nvfp4_moe_combine_tokens")})
    args = (_Tensor((tokens, hidden), bf), _Tensor((tokens, topk), i32), _Tensor((tokens, topk), bf))
    return blk, args


def test_inputs_and_buffers_are_recorded_on_the_stream_that_uses_them(pkg, monkeypatch):
    """Freed right after the call, their memory must not be handed out while the block still reads it."""
    blk, args = _block(pkg, monkeypatch)
    side = types.SimpleNamespace(cuda_stream=9, device=torch.device("cuda", 0))
    blk.run(*args, stream=side)
    for t in (*args, blk._meta, blk.dest, blk.src_rows, blk._route_ws, blk._a, blk._a_scale, blk._h, blk._a2,
              blk._a2_scale, blk._y, blk._w, blk.out):
        assert side in t.recorded


def test_nothing_is_recorded_on_the_current_stream(pkg, monkeypatch):
    blk, args = _block(pkg, monkeypatch)
    blk.run(*args)
    assert not any(t.recorded for t in (*args, blk.out))

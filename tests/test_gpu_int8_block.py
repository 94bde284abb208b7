"""The int8 MoE block as programs use it: streams, temporaries, several blocks."""
from __future__ import annotations

import pytest
import torch

import test_gpu_int8_moe as M

pytestmark = pytest.mark.gpu


def test_temporaries_freed_while_the_block_waits(pkg):
    """Inputs dropped right after a call on a busy stream: tensors that the current stream makes of
    the same sizes get other memory."""
    x, gate, up, down, ids, w = M._setup(pkg, 300, 2, 4, 256, 96, torch.bfloat16, 4)
    blk = pkg.moe.Int8MoEBlock(pkg.moe.quantize_expert_weights_int8(gate, up, down), 300, 2)
    want = blk.run(x, ids, w.to(torch.bfloat16)).clone()
    side = torch.cuda.Stream()
    busy = torch.randn((4096, 4096), device="cuda")
    for _ in range(3):
        blk.out.zero_()
        x2, ids2, w2 = x.clone(), ids.clone(), w.to(torch.bfloat16)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(20):  # some milliseconds before the block starts
                busy = torch.tanh(busy @ busy)
        out = blk.run(x2, ids2, w2, stream=side)
        del x2, ids2, w2
        kept = [torch.zeros_like(t) for t in (x, ids, w.to(torch.bfloat16)) for _ in range(4)]
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        del kept

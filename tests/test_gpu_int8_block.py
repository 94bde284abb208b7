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


def _bad_segment(pkg, error_word=None):
    a, sa = torch.zeros((8, 16), dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda")
    off = torch.tensor([4], dtype=torch.int32, device="cuda")
    cnt = torch.tensor([5], dtype=torch.int32, device="cuda")
    pkg.int8_gemm_segments(a, sa, a[None], sa[None], off, cnt, error_word=error_word)


def test_errors_stay_with_their_owner(pkg):
    """A bad segment of one caller is neither reported as another's nor cleared by it."""
    words = [torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2)]
    x, gate, up, down, ids, w = M._setup(pkg, 20, 2, 4, 64, 32, torch.bfloat16, 2)
    blk = pkg.moe.Int8MoEBlock(pkg.moe.quantize_expert_weights_int8(gate, up, down), 20, 2)
    blk.run(x, ids, w)
    _bad_segment(pkg)  # nobody's: the device's word
    assert blk.check_device_errors() == 0
    with pytest.raises(pkg.Nvfp4Error, match="segment"):
        pkg.check_int8_errors()
    _bad_segment(pkg, words[0])
    assert pkg.check_int8_errors() == 0 and blk.check_device_errors() == 0
    assert pkg.check_int8_errors(error_word=words[1]) == 0
    with pytest.raises(pkg.Nvfp4Error, match="segment"):
        pkg.check_int8_errors(error_word=words[0])
    assert pkg.check_int8_errors(error_word=words[0]) == 0


def test_a_block_reports_its_own_errors(pkg):
    """Two blocks, one with an error in its word: the other one checks clean before and after."""
    x, gate, up, down, ids, w = M._setup(pkg, 20, 2, 4, 64, 32, torch.bfloat16, 2)
    W = pkg.moe.quantize_expert_weights_int8(gate, up, down)
    a, b = pkg.moe.Int8MoEBlock(W, 20, 2), pkg.moe.Int8MoEBlock(W, 20, 2)
    for blk in (a, b):
        blk.run(x, ids, w)
    _bad_segment(pkg, a._errors)
    assert b.check_device_errors() == 0
    with pytest.raises(pkg.Nvfp4Error, match="segment"):
        a.check_device_errors()
    assert a.check_device_errors() == 0 and b.check_device_errors() == 0


def test_a_check_waits_for_the_run_on_its_stream(pkg):
    """The stream of the run is busy and not the current one: the check sees the run's end."""
    x, gate, up, down, ids, w = M._setup(pkg, 20, 2, 4, 64, 32, torch.bfloat16, 2)
    blk = pkg.moe.Int8MoEBlock(pkg.moe.quantize_expert_weights_int8(gate, up, down), 20, 2)
    side = torch.cuda.Stream()
    busy = torch.randn((4096, 4096), device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            busy = torch.tanh(busy @ busy)
        _bad_segment(pkg, blk._errors)
    blk.run(x, ids, w, stream=side)
    done = torch.cuda.Event()
    done.record(side)
    with pytest.raises(pkg.Nvfp4Error, match="segment"):
        blk.check_device_errors()
    assert done.query()


def test_checks_of_many_threads_lose_no_report(pkg):
    """Every bad segment is reported by one check: threads that set and check words at once."""
    import threading

    found = []

    def work(i):
        word = torch.zeros(1, dtype=torch.int32, device="cuda")
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        for _ in range(20):
            with torch.cuda.stream(st):
                _bad_segment(pkg, word)
                try:
                    pkg.check_int8_errors(error_word=word)
                except pkg.Nvfp4Error:
                    found.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert sorted(found) == sorted(list(range(4)) * 20)

"""Calls of the expert-layer operators as programs make them: from several threads, with results in given memory, repeated."""
import ctypes
import threading

import pytest
import torch

from kquant_b200 import _native, experts
from tests.expert_cases import offsets_of

pytestmark = pytest.mark.gpu


def test_threads_with_calls_of_different_sizes(cuda_device):
    """Threads whose calls differ in the shared memory that they ask for do not disturb one another."""
    g = torch.Generator(device=cuda_device).manual_seed(31)
    w = (torch.randn((8, 64, 256), generator=g, device=cuda_device) / 8).bfloat16()
    L, calls = _native.load(), []
    for each in (1, 16):                                   # rows an expert
        x = torch.randn((8 * each, 64), generator=g, device=cuda_device).bfloat16()
        off = offsets_of([each] * 8, cuda_device)
        calls.append((x, off, experts.expert_linear(x, w, off, activation="silu", gated=True)))
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        x, off, want = calls[i % 2]
        out, stream = torch.empty_like(want), torch.cuda.Stream(cuda_device)
        stream.wait_stream(torch.cuda.current_stream(cuda_device))
        p = experts._product(x, w, off, None, "silu", True)
        p.y, p.ldy = out.data_ptr(), out.stride(0)
        for _ in range(5000):                              # the C entry itself: ctypes lets the other threads run meanwhile
            if L.kq_expert_linear(ctypes.byref(p), None, 0, stream.cuda_stream):
                wrong.append(L.kq_last_error())
                break
        stream.synchronize()
        if not torch.equal(out, want):
            wrong.append("values")

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
    _native.check_wait_errors(cuda_device)

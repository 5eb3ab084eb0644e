"""Calls of the expert-layer operators as programs make them: from several threads, with results in given memory, repeated."""
import ctypes
import threading

import pytest
import torch

from kquant_b200 import _native, capture, experts
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


def test_a_wait_that_ran_out_is_not_silent(cuda_device):
    """A kernel reports it in a flag that the next call sees; here the flag is set by hand."""
    bf16 = lambda *s: torch.ones(s, device=cuda_device).bfloat16()  # noqa: E731
    half = lambda *s: torch.ones(s, device=cuda_device).half()  # noqa: E731
    off = offsets_of([1, 2], cuda_device)
    t = torch.zeros((2, 8, 8, 48), dtype=torch.int16, device=cuda_device)
    calls = [lambda: experts.expert_linear(bf16(3, 128), bf16(2, 128, 64), off),
             lambda: experts.linear(bf16(3, 128), bf16(128, 64)),
             lambda: experts.expert_linear_grad(bf16(3, 64), bf16(3, 128), bf16(2, 128, 64), off),
             lambda: experts.expert_linear_grad(bf16(3, 64), bf16(3, 128), bf16(2, 128, 64), off, bias=bf16(2, 64), need_dx=False,
                                                need_dw=False),
             lambda: experts.trellis_linear(bf16(3, 128), t, half(2, 128), half(2, 128), off),
             lambda: experts.trellis_linear(bf16(900, 128), t, half(2, 128), half(2, 128), offsets_of([400, 500], cuda_device)),
             lambda: capture.accumulate_expert_hessians(bf16(3, 128), off)]
    want = [c() for c in calls]
    experts.check_wait_errors(cuda_device)
    torch.cuda.synchronize()
    flag = ctypes.POINTER(ctypes.c_int32)()
    with torch.cuda.device(cuda_device):
        assert _native.load().kq_wait_error_flag(ctypes.byref(flag)) == 0
    assert flag[0] == 0
    flag[0] = 1
    for c in calls:
        with pytest.raises(_native.KQError, match="ran out"):
            c()
    with pytest.raises(_native.KQError, match="timed out"):
        experts.check_wait_errors(cuda_device)
    assert flag[0] == 0
    experts.check_wait_errors(cuda_device)
    for c, w in zip(calls, want):
        for a, b in zip(*((r if isinstance(r, tuple) else (r,)) for r in (c(), w))):
            assert a is b or torch.equal(a, b)

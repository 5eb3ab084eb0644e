"""Calls of the expert-layer operators as programs make them: from several threads, with results in given memory, repeated."""
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
    calls = []
    for each in (1, 16):                                   # rows an expert
        x = torch.randn((8 * each, 64), generator=g, device=cuda_device).bfloat16()
        off = offsets_of([each] * 8, cuda_device)
        calls.append((x, off, experts.expert_linear(x, w, off, activation="silu", gated=True)))
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        x, off, want = calls[i % 2]
        out = torch.empty_like(want)
        try:
            with torch.cuda.stream(torch.cuda.Stream(cuda_device)):
                for _ in range(2000):
                    experts.expert_linear(x, w, off, activation="silu", gated=True, out=out)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(out, want):
                    wrong.append("values")
        except Exception as error:                         # noqa: BLE001
            wrong.append(error)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
    _native.check_wait_errors(cuda_device)

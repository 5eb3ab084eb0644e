"""kquant_b200.experts.trellis_linear: the same call gives the same result whichever kernel its size selects."""
import pytest
import torch

from kquant_b200 import _native, experts
from tests.expert_cases import check, groups, offsets_of
from tests.test_trellis_linear_gpu import expect, make, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("book", ["mcg", "e4m3", "labels"])
@pytest.mark.parametrize("counts,n", [([8, 30], 256), ([8, 30], 4224), ([8, 100], 4224), ([300, 100], 4224)])
def test_scales_of_rows_in_every_kernel(cuda_device, book, counts, n):
    """Rows whose sums before the output scales leave the fp32 range, next to small ones: few rows, tens, decoded once."""
    x, t, suh, svh, off = make(counts, 256, n, 4, torch.bfloat16, cuda_device, seed=41)
    x[0], x[1], x[2], x[3] = 0, x[1] * 2.0 ** -60, x[2] * 2.0 ** 60, x[3] * 2.0 ** 20
    x[4, 17], x[9, 200] = 3e4, -2e5
    x[5] = torch.sign(x[5]) * 1e38
    x[6] = torch.sign(x[6]) * 3e38
    suh[0] *= 0.5
    svh[0] *= 2.0 ** -10
    cb = tables(cuda_device)[book]
    y = experts.trellis_linear(x, t, suh, svh, off, codebook=cb)
    want, bound = expect(x, t, suh, svh, off, cb)
    assert float(want.abs().max()) < 2.0 ** 127
    check(y, want, bound)
    assert not y[0].any()
    _native.check_wait_errors(cuda_device)


@pytest.mark.parametrize("counts,n", [([8, 30], 256), ([8, 100], 4224), ([300, 100], 4224)])
def test_result_over_its_own_rows(cuda_device, counts, n):
    """x is read before the first result is written, in every kernel."""
    x, t, suh, svh, off = make(counts, n, n, 3, torch.bfloat16, cuda_device, seed=42, spare=2)
    want = experts.trellis_linear(x, t, suh, svh, off)
    rows = x.clone()
    assert experts.trellis_linear(rows, t, suh, svh, off, out=rows) is rows
    assert torch.equal(rows[: sum(counts)], want[: sum(counts)]) and torch.equal(rows[sum(counts):], x[sum(counts):])
    _native.check_wait_errors(cuda_device)


@pytest.mark.parametrize("book", ["mcg", "labels"])
def test_more_experts_than_are_decoded_at_a_time(cuda_device, book):
    """Two experts of this size fit the decoded matrices' memory: three rounds, and what each expert gives alone."""
    g = torch.Generator(device=cuda_device).manual_seed(43)
    counts, k, n = [300, 0, 250, 200, 260], 16384, 16384
    rows, E = sum(counts), len(counts)
    x = torch.randn((rows + 5, k), generator=g, device=cuda_device).bfloat16()
    t = torch.randint(-32768, 32768, (E, k // 16, n // 16, 16), generator=g, device=cuda_device, dtype=torch.int16)
    suh, svh = (torch.rand((E, k), generator=g, device=cuda_device) + 0.5).half(), (torch.rand((E, n), generator=g, device=cuda_device) + 0.5).half()
    cb, off = tables(cuda_device)[book], offsets_of(counts, cuda_device, first=3)
    run = lambda: experts.trellis_linear(x, t, suh, svh, off, codebook=cb)  # noqa: E731
    y = run()
    assert not y[:3].any() and not y[rows + 3:].any()
    for e, r in enumerate(groups(off)):
        if r.stop > r.start:
            alone = experts.trellis_linear(x[r], t[e], suh[e], svh[e], codebook=cb)
            assert alone.abs().max() > 0 and torch.equal(y[r], alone), e
    keep = torch.full_like(y, 7.0)
    experts.trellis_linear(x, t, suh, svh, off, codebook=cb, out=keep)
    assert torch.equal(keep[3: rows + 3], y[3: rows + 3]) and (keep[:3] == 7).all() and (keep[rows + 3:] == 7).all()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for new in (counts, [0, 0, 0, 0, rows], [rows, 0, 0, 0, 0], [1, 2, 3, 4, 5]):
        off.copy_(offsets_of(new, cuda_device))
        graph.replay()
        assert torch.equal(got, run())
    _native.check_wait_errors(cuda_device)

"""kquant_b200.capture.accumulate_expert_hessians against 64-bit sums."""
import pytest
import torch

from kquant_b200 import _native
from kquant_b200.capture import accumulate_expert_hessians
from tests.expert_cases import check, groups, offsets_of

pytestmark = pytest.mark.gpu

# Operand terms left out are below 2^-24 of a product each side; the tensor accumulator holds at most 8 steps of 16
# rows before a rounded fp32 add (a truncation of at most 2^-23 a step and product, six products at most in two
# steps), and the fp32 adds of s segments round by s 2^-24.
def slack(rows):
    return 16 * 2.0 ** -23 + (rows / 32 + 4) * 2.0 ** -24


def expect(x, offsets, index, weights):
    d = x.shape[1]
    E = offsets.numel() - 1
    H = torch.zeros((E, d, d), dtype=torch.float64, device=x.device)
    B, den = torch.zeros_like(H), torch.zeros(E, dtype=torch.float64, device=x.device)
    slots = x.shape[0] if index is None else index.numel()
    pick = torch.arange(slots, device=x.device) if index is None else index
    w = torch.ones(slots, dtype=torch.float64, device=x.device) if weights is None else weights.double()
    ok = (pick >= 0) & (pick < x.shape[0])
    w = w * ok
    X = x.double()[pick.clamp(0, x.shape[0] - 1)]
    for e, r in enumerate(groups(offsets)):
        H[e] = (X[r] * w[r, None]).T @ X[r]
        # w x is rounded to fp32 before it is split
        B[e] = (X[r] * w[r, None]).abs().T @ X[r].abs() * (slack(r.stop - r.start) + 2.0 ** -24) + 1e-38
        den[e] = w[r].sum()
    return H, B, den


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("counts,d,tokens", [([1], 1, 1), ([3, 0, 40], 7, 20), ([64, 1, 130], 300, 512), ([0, 500], 256, 64),
                                             ([33], 1000, 33), ([31, 32, 33, 95, 96, 97, 0], 72, 400)])
def test_hessians(cuda_device, dtype, weighted, counts, d, tokens):
    g = torch.Generator(device=cuda_device).manual_seed(d + tokens)
    x = (torch.randn((tokens, d), generator=g, device=cuda_device) * torch.exp(torch.randn(d, generator=g, device=cuda_device))).to(dtype)
    rows = sum(counts)
    index = torch.randint(tokens, (rows + 3,), generator=g, device=cuda_device)
    w = torch.rand(rows + 3, generator=g, device=cuda_device) - 0.3 if weighted else None      # signs of both kinds
    off = offsets_of(counts, cuda_device, first=1)
    H, den = accumulate_expert_hessians(x, off, index=index, weights=w)
    want, bound, wden = expect(x, off, index, w)
    check(H, want, bound)
    assert torch.equal(H, H.transpose(1, 2))
    assert torch.allclose(den, wden, rtol=1e-13, atol=1e-13)
    assert H.stride(1) % 32 == 0 or d == 1
    _native.check_wait_errors(cuda_device)


def test_without_index_and_added(cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(1)
    x = torch.randn((200, 130), generator=g, device=cuda_device)
    off = offsets_of([60, 0, 140], cuda_device)
    want, bound, _ = expect(x, off, None, None)
    H, den = accumulate_expert_hessians(x, off)
    check(H, want, bound)
    start = torch.randn((3, 130, 130), generator=g, device=cuda_device)
    start = start + start.transpose(1, 2)
    out = start.clone()
    got, den2 = accumulate_expert_hessians(x, off, out=out)
    assert got is out and torch.equal(den, den2) and torch.equal(out, out.transpose(1, 2))
    assert torch.equal(out[1], start[1])
    check(out, want + start.double(), bound + (want + start.double()).abs() * 2.0 ** -23)
    # A wider output, an odd row stride, a base off the 16-byte grid.
    wide = torch.zeros((3, 130, 133), device=cuda_device)
    accumulate_expert_hessians(x, off, out=wide[:, :, 1:131])
    assert torch.equal(wide[:, :, 1:131], H) and not wide[:, :, 0].any() and not wide[:, :, 131:].any()
    xs = torch.zeros((200, 135), device=cuda_device)
    xs[:, 3:133] = x
    assert torch.equal(accumulate_expert_hessians(xs[:, 3:133], off)[0], H)


def test_long_sums_keep_fp32_accuracy(cuda_device):
    """Positive values: the diagonal and off-diagonal sums grow with the rows, where truncation would show."""
    g = torch.Generator(device=cuda_device).manual_seed(2)
    for dtype in (torch.bfloat16, torch.float32):
        x = (torch.rand((20000, 64), generator=g, device=cuda_device) + 0.5).to(dtype)
        off = offsets_of([20000], cuda_device)
        H, _ = accumulate_expert_hessians(x, off)
        want, bound, _ = expect(x, off, None, None)
        check(H, want, bound)
        assert float((H.double() - want).norm() / want.norm()) < 1e-6


def test_wild_indexes_count_for_nothing(cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(3)
    x = torch.randn((10, 40), generator=g, device=cuda_device).bfloat16()
    index = torch.tensor([0, -1, 3, 10, 1 << 40, 9, -(1 << 40)], device=cuda_device)
    off = torch.tensor([0, 3, 99], device=cuda_device)
    H, den = accumulate_expert_hessians(x, off, index=index)
    want, bound, wden = expect(x, torch.tensor([0, 3, 7], device=cuda_device), index, None)
    check(H, want, bound)
    assert torch.equal(den, wden) and den.tolist() == [2.0, 1.0]


def test_experts_do_not_mix_and_replay(cuda_device):
    """NaN rows of one expert stay its own; a captured call follows new offsets, indexes and values."""
    g = torch.Generator(device=cuda_device).manual_seed(4)
    x = torch.randn((100, 96), generator=g, device=cuda_device).bfloat16()
    off = offsets_of([40, 5, 50], cuda_device)
    x[40:45] = float("nan")
    H, _ = accumulate_expert_hessians(x, off)
    assert H[1].isnan().all() and not H[0].isnan().any() and not H[2].isnan().any()
    index = torch.arange(100, device=cuda_device)
    w = torch.rand(100, generator=g, device=cuda_device)
    run = lambda: accumulate_expert_hessians(x, off, index=index, weights=w)  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for counts in ([95, 0, 0], [1, 2, 3], [30, 30, 40]):
        off.copy_(offsets_of(counts, cuda_device))
        x.copy_(torch.randn((100, 96), generator=g, device=cuda_device))
        index.copy_(torch.randint(100, (100,), generator=g, device=cuda_device))
        graph.replay()
        for a, b in zip(got, run()):
            assert torch.equal(a, b)


def test_nothing_to_add(cuda_device):
    x = torch.zeros((0, 40), device=cuda_device)
    off = offsets_of([0, 0], cuda_device)
    H, den = accumulate_expert_hessians(x, off)
    assert H.shape == (2, 40, 40) and not H.any() and not den.any()
    start = torch.ones((2, 40, 40), device=cuda_device)
    assert (accumulate_expert_hessians(x, off, out=start)[0] == 1).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts", [[300, 5, 0, 140, 1, 130, 20, 129, 2, 257, 40, 0, 400, 64, 128, 3, 90, 131, 60, 33],
                                    [129] * 3 + [1] * 17, [200] * 11 + [2] * 9, [1, 500, 1, 260, 1, 130] + [7] * 14])
def test_uneven_experts(cuda_device, dtype, counts):
    """Experts of one to several segments of rows in turn, every CTA with several tiles of each."""
    E, d, tokens, rows = len(counts), 901, 333, sum(counts)
    g = torch.Generator(device=cuda_device).manual_seed(3)
    x = torch.randn((tokens, d), generator=g, device=cuda_device).to(dtype)
    index = torch.randint(tokens, (rows,), generator=g, device=cuda_device)
    off = offsets_of(counts, cuda_device)
    first = None
    for _ in range(10):
        H, den = accumulate_expert_hessians(x, off, index=index)
        first = H if first is None else first
        assert torch.equal(H, first)
    assert den.tolist() == counts
    added, _ = accumulate_expert_hessians(x, off, index=index, out=H.clone())
    for e, r in enumerate(groups(off)):
        X = x[index[r]].double()
        want, mass = X.T @ X, X.abs().T @ X.abs()
        assert ((H[e].double() - want).abs() <= mass * slack(counts[e]) + 1e-38).all(), e
        assert ((added[e].double() - 2 * want).abs() <= 2 * mass * slack(2 * counts[e]) + 1e-38).all(), e
    _native.check_wait_errors(cuda_device)

"""The grouped and dense products of kquant_b200.experts, and their gradients, against 64-bit results."""
import pytest
import torch

from kquant_b200 import _native, experts
from tests.expert_cases import check, forward64, grad64, groups, offsets_of

pytestmark = pytest.mark.gpu

# rows of each expert, k, n
SHAPES = [
    ([1], 1, 1),
    ([1], 64, 128),
    ([5], 331, 517),
    ([128, 128], 64, 256),
    ([0, 3, 0, 130, 1, 0], 200, 264),
    ([17, 300, 64], 513, 130),
    ([129, 0, 255], 96, 1030),
    ([2000], 40, 24),
    ([1] * 40, 72, 80),
    ([0, 0], 64, 64),
]


def make(counts, k, n, dtype, layout, dev, seed=0, spare=0, first=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    E, rows = len(counts), sum(counts) + spare + first
    rnd = lambda *s: torch.randn(s, generator=g, device=dev).to(dtype)  # noqa: E731
    x = rnd(rows, k)
    w = rnd(E, n, k).transpose(1, 2) if layout == "hf" else rnd(E, k, n)
    w = w * 0.5
    if layout == "hf":
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    return x, w, rnd(E, n), offsets_of(counts, dev, first), rnd


def expect(x, w, offsets, bias, act, gated, residual):
    n_out = w.shape[2] // 2 if gated else w.shape[2]
    y = torch.zeros((x.shape[0], n_out), dtype=torch.float64, device=x.device)
    b = torch.zeros_like(y)
    for e, r in enumerate(groups(offsets)):
        y[r], b[r] = forward64(x[r], w[e], None if bias is None else bias[e], act, gated,
                               None if residual is None else residual[r])
    return y, b


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["exl", "hf"])
@pytest.mark.parametrize("counts,k,n", SHAPES)
def test_plain_product(cuda_device, dtype, layout, counts, k, n):
    x, w, bias, off, rnd = make(counts, k, n, dtype, layout, cuda_device, spare=2)
    y = experts.expert_linear(x, w, off)
    check(y, *expect(x, w, off, None, None, False, None))
    _native.check_wait_errors(cuda_device)


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("layout", ["exl", "hf"])
@pytest.mark.parametrize("counts,k,n", [([3, 0, 140], 136, 264), ([37], 65, 70), ([2, 9], 128, 30)])
def test_epilogue(cuda_device, act, gated, layout, counts, k, n):
    for dtype in (torch.bfloat16, torch.float16):
        x, w, bias, off, rnd = make(counts, k, n, dtype, layout, cuda_device, seed=3)
        res = rnd(x.shape[0], n // 2 if gated else n)
        y = experts.expert_linear(x, w, off, bias=bias, activation=act, gated=gated, residual=res)
        check(y, *expect(x, w, off, bias, act, gated, res))
    _native.check_wait_errors(cuda_device)


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("layout", ["exl", "hf"])
@pytest.mark.parametrize("counts,k,n", [([3, 0, 140, 64], 136, 264), ([37], 65, 70), ([2, 9], 300, 30), ([1], 8, 2)])
def test_gradients(cuda_device, act, gated, layout, counts, k, n):
    for dtype in (torch.bfloat16, torch.float16):
        x, w, bias, off, rnd = make(counts, k, n, dtype, layout, cuda_device, seed=5, spare=3)
        dy = rnd(x.shape[0], n // 2 if gated else n)
        dx, dw, db = experts.expert_linear_grad(dy, x, w, off, bias=bias, activation=act, gated=gated)
        assert dw.shape == w.shape and not dx[sum(counts):].any()
        for e, r in enumerate(groups(off)):
            gx, gw, gb = grad64(dy[r], x[r], w[e], bias[e], act, gated)
            check(dx[r], *gx, what=f"dx {e}")
            check(dw[e], *gw, what=f"dw {e}")
            check(db[e], *gb, what=f"db {e}")
    _native.check_wait_errors(cuda_device)


@pytest.mark.parametrize("act,gated", [("silu", True), ("gelu", False)])
def test_gradients_are_slopes(cuda_device, act, gated):
    """The gradients against differences of a 64-bit forward pass along random directions."""
    x, w, bias, off, rnd = make([5, 0, 9], 24, 16, torch.float16, "exl", cuda_device, seed=8)
    n_out = 8 if gated else 16
    dy = rnd(x.shape[0], n_out)
    grads = experts.expert_linear_grad(dy, x, w, off, bias=bias, activation=act, gated=gated)

    def loss(x, w, bias):
        total = 0.0
        for e, r in enumerate(groups(off)):
            total += float((forward64(x[r], w[e], bias[e], act, gated, None)[0] * dy[r].double()).sum())
        return total

    for i, g in enumerate(grads):
        base = [x.double(), w.double(), bias.double()]
        d = torch.sign(g.double())                 # the direction in which every term of the slope is positive
        for t in base:
            t.requires_grad_(False)
        h = 2.0 ** -14
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + h * d, base[i] - h * d
        from tests import expert_cases
        expert_cases.HALF_STEP[torch.float64], expert_cases.TINY[torch.float64] = 2.0 ** -53, 0.0
        slope = (loss(*up) - loss(*down)) / (2 * h)
        # Two fp16 roundings on the way (dz and the result): 2^-10 of the sum of absolute terms.
        # The difference itself is off by h^2 / 6 of a third derivative along d, far below.
        assert abs(slope - float(g.double().abs().sum())) <= 2.0 ** -9 * float(g.double().abs().sum()) + 2.0 ** -9 * float(
            dy.double().abs().sum())


def test_dense_linear_and_views(cuda_device):
    """Sliced operands: odd strides, a base off the 16-byte grid, a transposed matrix, an output with a wider row."""
    g = torch.Generator(device=cuda_device).manual_seed(2)
    rnd = lambda *s: torch.randn(s, generator=g, device=cuda_device).bfloat16()  # noqa: E731
    wide_x, wide_w = rnd(77, 205), rnd(203, 311)
    res = rnd(77, 307)[:, 3:303]
    out = torch.full((77, 305), 7.0, dtype=torch.bfloat16, device=cuda_device)
    for x, w in ((wide_x[:, 1:201], wide_w[3:, 5:305]), (wide_x[:, :200], wide_w[:200, :300]),
                 (wide_x[:, 3:203], rnd(300, 207)[:, 4:204].T), (wide_x[::2, :200], wide_w[:200, :300])):
        r = res[: x.shape[0]]
        y = experts.linear(x, w, activation="gelu", residual=r, out=out[: x.shape[0], 2:302])
        check(y, *forward64(x, w, None, "gelu", False, r))
        assert (out[:, :2] == 7).all() and (out[:, 302:] == 7).all()
    y = experts.linear(wide_x, rnd(205, 300))
    assert y.shape == (77, 300)
    _native.check_wait_errors(cuda_device)


def test_broadcast_operands(cuda_device):
    """Experts that share one matrix (stride 0), one row for all, one bias for all."""
    x, w, bias, off, rnd = make([4, 70], 64, 48, torch.bfloat16, "exl", cuda_device, seed=4)
    ws, bs, xs = w[:1].expand(2, -1, -1), bias[:1].expand(2, -1), x[:1].expand(74, -1)
    y = experts.expert_linear(xs, ws, off, bias=bs, activation="silu")
    check(y, *expect(xs, ws, off, bs, "silu", False, None))
    dx, dw, db = experts.expert_linear_grad(rnd(74, 48), xs, ws, off, bias=bs)
    assert dw.shape == (2, 64, 48) and dw.is_contiguous() and db.shape == (2, 48)


def test_rows_of_no_expert_and_out(cuda_device):
    x, w, bias, off, rnd = make([3, 5], 64, 32, torch.bfloat16, "exl", cuda_device, seed=6, spare=4, first=2)
    y = experts.expert_linear(x, w, off)
    assert not y[:2].any() and not y[10:].any()
    check(y, *expect(x, w, off, None, None, False, None))
    keep = rnd(14, 32)
    out = keep.clone()
    assert experts.expert_linear(x, w, off, out=out) is out
    assert torch.equal(out[:2], keep[:2]) and torch.equal(out[10:], keep[10:]) and torch.equal(out[2:10], y[2:10])
    # In place on the residual.
    both = experts.expert_linear(x, w, off, residual=keep)
    out = keep.clone()
    experts.expert_linear(x, w, off, residual=out, out=out)
    assert torch.equal(out[2:10], both[2:10]) and torch.equal(out[:2], keep[:2])


@pytest.mark.parametrize("layout", ["exl", "hf"])
def test_other_experts_values_stay_out(cuda_device, layout):
    """NaN and infinity in one expert's rows or matrix reach no other expert's results."""
    counts = [70, 3, 130]
    x, w, bias, off, rnd = make(counts, 100, 72, torch.bfloat16, layout, cuda_device, seed=7, spare=5)
    dy = rnd(x.shape[0], 72)
    clean = experts.expert_linear(x, w, off), *experts.expert_linear_grad(dy, x, w, off, bias=bias, activation="silu")
    x2, dy2, w2 = x.clone(), dy.clone(), w.clone()
    x2[70:73], dy2[70:73], w2[1] = float("nan"), float("inf"), float("nan")
    x2[203:], dy2[203:] = float("nan"), float("nan")
    y, (dx, dw, db) = experts.expert_linear(x2, w2, off), experts.expert_linear_grad(dy2, x2, w2, off, bias=bias, activation="silu")
    keep = torch.ones(208, dtype=torch.bool, device=cuda_device)
    keep[70:73] = False
    for a, b in ((y, clean[0]), (dx, clean[1])):
        assert torch.equal(a[keep], b[keep])
    for a, b in ((dw, clean[2]), (db, clean[3])):
        assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
    assert dw[1].isnan().any()


def test_wild_offsets_stay_in_bounds(cuda_device):
    """Offsets beyond the rows are clamped: nothing outside is read or written."""
    x, w, bias, off, rnd = make([4, 4], 64, 32, torch.bfloat16, "exl", cuda_device, seed=9)
    off = torch.tensor([-5, 6, 1 << 40], device=cuda_device)
    y = experts.expert_linear(x, w, off)
    fixed = torch.tensor([0, 6, 8], device=cuda_device)
    assert torch.equal(y, experts.expert_linear(x, w, fixed))
    _native.check_wait_errors(cuda_device)


def test_captured_call_follows_new_offsets(cuda_device):
    x, w, bias, off, rnd = make([30, 2, 40], 64, 96, torch.bfloat16, "exl", cuda_device, seed=10)
    dy = rnd(72, 96)
    run = lambda: (experts.expert_linear(x, w, off, bias=bias, activation="silu"),  # noqa: E731
                   *experts.expert_linear_grad(dy, x, w, off, bias=bias, activation="silu"))
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for counts in ([30, 2, 40], [0, 72, 0], [71, 0, 1], [1, 1, 3]):
        off.copy_(offsets_of(counts, cuda_device))
        x.copy_(rnd(72, 64))
        graph.replay()
        for a, b in zip(got, run()):
            assert torch.equal(a, b)


def test_streams_and_repeats(cuda_device):
    """Calls on two streams at once give what they give alone, every time the same bits."""
    x, w, bias, off, rnd = make([300, 40, 500], 205, 301, torch.bfloat16, "exl", cuda_device, seed=11)
    dy = rnd(840, 301)
    want = experts.expert_linear_grad(dy, x, w, off, bias=bias, activation="gelu")
    streams = [torch.cuda.Stream(cuda_device) for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(experts.expert_linear_grad(dy, x, w, off, bias=bias, activation="gelu"))
    torch.cuda.synchronize()
    for g in got:
        for a, b in zip(g, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("counts,k,n", [([700, 1, 1200, 300], 512, 2048), ([3000], 264, 4104)])
def test_many_tiles(cuda_device, counts, k, n):
    """More tiles than SMs: the accumulators and stages wrap several times."""
    x, w, bias, off, rnd = make(counts, k, n, torch.bfloat16, "hf", cuda_device, seed=12)
    y = experts.expert_linear(x, w, off, activation="silu", gated=True)
    check(y, *expect(x, w, off, None, "silu", True, None))
    dx, dw, _ = experts.expert_linear_grad(rnd(x.shape[0], n), x, w, off)
    assert dw.stride() == w.stride()
    _native.check_wait_errors(cuda_device)


def test_empty_calls(cuda_device):
    x, w, bias, off, rnd = make([0, 0], 64, 32, torch.float16, "exl", cuda_device)
    assert experts.expert_linear(x, w, off).shape == (0, 32)
    dx, dw, db = experts.expert_linear_grad(x.new_empty((0, 32)), x, w, off, bias=bias, activation="silu")
    assert dx.shape == (0, 64) and not dw.any() and not db.any()

"""Every choice of kernel and tile of the expert-layer products, at the sizes that take it, against 64-bit results."""
import pytest
import torch

from kquant_b200 import _native, experts
from tests.expert_cases import check, grad64, groups
from tests.test_expert_linear_gpu import expect, make

pytestmark = pytest.mark.gpu


def check_gradients(dy, x, w, off, bias, act, gated, **needs):
    dx, dw, db = experts.expert_linear_grad(dy, x, w, off, bias=bias, activation=act, gated=gated, **needs)
    for e, r in enumerate(groups(off)):
        gx, gw, gb = grad64(dy[r], x[r], w[e], None if bias is None else bias[e], act, gated)
        for what, got, want in (("dx", None if dx is None else dx[r], gx), ("dw", None if dw is None else dw[e], gw),
                                ("db", None if db is None else db[e], gb)):
            if got is not None:
                check(got, *want, what=f"{what} {e}")
    _native.check_wait_errors(x.device)


@pytest.mark.parametrize("layout", ["exl", "hf"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("counts,k,n", [([45, 3, 40], 2056, 2 * 77), ([33], 2050, 2 * 5), ([120, 1], 4100, 2 * 131)])
def test_ragged_features(cuda_device, layout, gated, counts, k, n):
    """Lanes without a feature beside lanes with one, in warps that go on to collective instructions: more than 32 rows a
    tile, k split over a cluster."""
    x, w, bias, off, rnd = make(counts, k, n, torch.bfloat16, layout, cuda_device, seed=21)
    res = rnd(x.shape[0], n // 2 if gated else n)
    for _ in range(3):
        y = experts.expert_linear(x, w, off, bias=bias, activation="silu", gated=gated, residual=res)
        check(y, *expect(x, w, off, bias, "silu", gated, res))
    _native.check_wait_errors(cuda_device)


@pytest.mark.parametrize("layout", ["exl", "hf"])
@pytest.mark.parametrize("counts,k,n", [([100, 7], 40, 40), ([300], 264, 1000), ([1, 90, 2], 8, 520), ([70], 1000, 16)])
def test_ragged_lines_of_the_weight_gradient(cuda_device, layout, counts, k, n):
    """Lines that are no multiple of 32, several chunks of columns: lanes without a line beside lanes with one."""
    x, w, bias, off, rnd = make(counts, k, n, torch.float16, layout, cuda_device, seed=22)
    check_gradients(rnd(x.shape[0], n), x, w, off, None, None, False, need_dx=False)


# The few-row kernel takes row tiles of 32, 64 and 128 (a mean of 9 to 16, 17 to 32, 33 to 48 rows an expert, and however many
# where tiles are scarce), k split over up to eight CTAs, and one long ring instead of two short ones (gated).
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["exl", "hf"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("counts,k,n", [
    ([30, 1, 0, 17, 9], 136, 264),            # tiles of 32, k not split
    ([20, 2, 16], 2050, 2 * 129),             # tiles of 32
    ([60, 17, 0, 5, 66], 2050, 2 * 129),      # tiles of 64, one of two tiles an expert
    ([130, 3, 1, 40], 2056, 2 * 70),          # tiles of 128, the second of two rows
    ([257, 30], 4104, 2 * 33),                # three tiles of 128
    ([47] * 12, 2048, 2 * 1030),              # as many tiles as leave little or no split
])
def test_few_row_tiles(cuda_device, dtype, layout, gated, counts, k, n):
    x, w, bias, off, rnd = make(counts, k, n, dtype, layout, cuda_device, seed=23, spare=3)
    res = rnd(x.shape[0], n // 2 if gated else n)
    y = experts.expert_linear(x, w, off, bias=bias, activation="gelu", gated=gated, residual=res)
    check(y[: sum(counts)], *(t[: sum(counts)] for t in expect(x, w, off, bias, "gelu", gated, res)))
    assert not y[sum(counts):].any()
    check_gradients(rnd(x.shape[0], n // 2 if gated else n), x, w, off, bias, "silu", gated)


@pytest.mark.parametrize("layout", ["exl", "hf"])
@pytest.mark.parametrize("counts", [[20, 2, 16], [60, 17, 40], [130, 3, 1, 40]])
def test_few_row_tiles_of_the_input_gradient(cuda_device, layout, counts):
    """dz W^T contracts over n: long enough here to be the few-row kernel's."""
    x, w, bias, off, rnd = make(counts, 72, 2050, torch.bfloat16, layout, cuda_device, seed=24)
    check_gradients(rnd(x.shape[0], 2050), x, w, off, None, None, False)


def test_few_row_tiles_follow_new_offsets(cuda_device):
    """Captured with even experts and replayed with every row on one: more tiles of an expert than its share."""
    x, w, bias, off, rnd = make([47, 47, 47], 2056, 264, torch.bfloat16, "exl", cuda_device, seed=25)
    run = lambda: experts.expert_linear(x, w, off, bias=bias, activation="silu", gated=True)  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for edges in ([0, 141, 141, 141], [0, 0, 1, 141], [7, 50, 99, 133], [0, 0, 0, 0]):
        off.copy_(torch.tensor(edges))
        graph.replay()
        check(got, *expect(x, w, off, bias, "silu", True, None))
    _native.check_wait_errors(cuda_device)


# Two accumulators a tile: 512 features, from three tiles for every pair of SMs on; with rows to read (residual, dy) from a k
# above 2048 on.  Row tiles of more than 128 rows alternate the halves of the tensor memory, smaller ones share one.
@pytest.mark.parametrize("layout", ["exl", "hf"])
@pytest.mark.parametrize("counts,k,n,residual", [([1500, 0, 130, 2200], 200, 7100, False), ([2000, 1, 127, 1400], 2100, 7000, True),
                                                 ([4000], 72, 7177, False)])
def test_two_accumulators(cuda_device, layout, counts, k, n, residual):
    x, w, bias, off, rnd = make(counts, k, n, torch.bfloat16, layout, cuda_device, seed=26)
    res = rnd(x.shape[0], n) if residual else None
    y = experts.expert_linear(x, w, off, bias=bias, activation="silu", residual=res)
    check(y, *expect(x, w, off, bias, "silu", False, res))
    if residual:                                           # the gradient in z reads dy as this reads the residual
        check_gradients(rnd(x.shape[0], n), x, w, off, bias, "gelu", False)
    _native.check_wait_errors(cuda_device)


@pytest.mark.parametrize("layout", ["exl", "hf"])
@pytest.mark.parametrize("counts,k,n", [
    ([1000, 400], 4700, 2992),                # lines on 32 bytes; a last tile of one accumulator
    ([643, 1, 1300], 5000, 2040),             # lines on 16 bytes, an expert of one row
    ([1341, 0], 4000, 4003),                  # by column; an expert without rows
    ([64 * 11], 7168, 4096),                  # no tail behind the last stage
])
def test_two_accumulators_of_the_weight_gradient(cuda_device, layout, counts, k, n):
    """More than 640 rows an expert and enough tiles."""
    x, w, bias, off, rnd = make(counts, k, n, torch.bfloat16, layout, cuda_device, seed=27, spare=5)
    x[sum(counts):] = float("nan")                         # behind the last expert: in no sum
    dy = rnd(x.shape[0], n)
    dy[sum(counts):] = float("nan")
    check_gradients(dy, x, w, off, None, None, False, need_dx=False)

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

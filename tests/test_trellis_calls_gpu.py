"""kquant_b200.experts.trellis_linear: the same call gives the same result whichever kernel its size selects."""
import pytest
import torch

from kquant_b200 import _native, experts
from tests.expert_cases import check
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

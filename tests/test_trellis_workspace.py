"""Memory that the products with encoded experts take, computed on the host."""
import ctypes

import pytest

from kquant_b200 import _native


def workspace(rows, k, n, experts, codebook=_native.KQ_CB_MCG):
    p = _native.TrellisProduct(x=64, trellis=64, suh=64, svh=64, offsets=64, table=64, y=64, rows=rows, k=k, n=n, experts=experts,
                               ldx=k, ldy=n, suh_stride_e=k, svh_stride_e=n, bits=3, codebook=codebook)
    return _native.load().kq_trellis_linear_workspace_bytes(ctypes.byref(p))


@pytest.mark.parametrize("rows,k,n,experts,codebook", [
    (80000, 7168, 4096, 384, _native.KQ_CB_MCG), (200000, 2048, 7168, 1024, _native.KQ_CB_SQG), (16000, 7168, 4096, 384, _native.KQ_CB_LABELS),
    (2048, 2048, 7168, 8, _native.KQ_CB_MCG), (1000, 16384, 16384, 5, _native.KQ_CB_MCG)])
def test_decoded_matrices_are_bounded(rows, k, n, experts, codebook):
    """Beside the rotated rows: 1 GiB of decoded matrices at most, whatever the number of experts."""
    assert 0 < workspace(rows, k, n, experts, codebook) <= (1 << 30) + rows * (2 * k + 4) + 256


def test_one_matrix_larger_than_the_bound():
    assert workspace(2000, 1 << 15, 1 << 15, 4) <= (1 << 31) + 2000 * ((1 << 16) + 4) + 256

"""What the expert-layer operators refuse, checked on the host before any launch."""
import ctypes

import pytest
import torch

from kquant_b200 import _native, experts


class FakeCuda(torch.Tensor):
    """A CPU tensor that says it is on a GPU: the argument checks run, no kernel is reached."""
    is_cuda = True


def fake(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype).as_subclass(FakeCuda)


@pytest.mark.parametrize("change,error,match", [
    (dict(x=torch.zeros(4, 8, dtype=torch.bfloat16)), _native.KQError, "CUDA"),
    (dict(x=fake(4, 8, dtype=torch.float32)), TypeError, "bfloat16 or torch.float16"),
    (dict(w=fake(2, 8, 6, dtype=torch.float16)), TypeError, "w must be"),
    (dict(w=fake(8, 6)), ValueError, "3 dimensions"),
    (dict(w=fake(2, 9, 6)), ValueError, "x must be"),
    (dict(w=fake(2, 8, 0)), ValueError, "empty"),
    (dict(w=fake(2, 16, 12)[:, ::2, ::2]), ValueError, "unit stride"),
    (dict(x=fake(4, 16)[:, ::2]), ValueError, "unit stride"),
    (dict(offsets=None), ValueError, "offsets"),
    (dict(offsets=torch.zeros(2, dtype=torch.int64).as_subclass(FakeCuda)), ValueError, "3 contiguous"),
    (dict(offsets=torch.zeros(3, dtype=torch.int32).as_subclass(FakeCuda)), TypeError, "int64"),
    (dict(offsets=torch.zeros(3, dtype=torch.int64)), _native.KQError, "CUDA"),
    (dict(activation="tanh"), ValueError, "activation"),
    (dict(w=fake(2, 8, 7), gated=True), ValueError, "even"),
    (dict(bias=fake(2, 5)), ValueError, "bias"),
    (dict(bias=fake(6)), ValueError, "2 dimensions"),
    (dict(residual=fake(4, 5)), ValueError, "residual"),
    (dict(residual=fake(4, 6), gated=True), ValueError, "residual"),
    (dict(out=fake(3, 6)), ValueError, "out"),
    (dict(out=fake(4, 6, dtype=torch.float32)), TypeError, "out"),
])
def test_expert_linear_refuses(change, error, match):
    args = dict(x=fake(4, 8), w=fake(2, 8, 6), offsets=torch.zeros(3, dtype=torch.int64).as_subclass(FakeCuda))
    args.update(change)
    with pytest.raises(error, match=match):
        experts.expert_linear(**args)


def test_linear_and_gradient_refuse():
    with pytest.raises(ValueError, match="2 dimensions"):
        experts.linear(fake(4, 8), fake(1, 8, 6))
    with pytest.raises(ValueError, match="1 dimension"):
        experts.linear(fake(4, 8), fake(8, 6), bias=fake(1, 6))
    with pytest.raises(ValueError, match="dy"):
        experts.expert_linear_grad(fake(4, 5), fake(4, 8), fake(1, 8, 6), None)


def test_overlapping_results_are_refused():
    buf = fake(64)
    wide = fake(6, 24)
    w = fake(8, 8)
    for x, residual, out in ((buf[:32].view(4, 8), None, buf[8:40].view(4, 8)), (wide[:4, :8], None, wide[:4, 4:12]),
                             (wide[:4, :8], None, wide[1:5, :8]), (buf[:32].view(4, 8), None, buf[:32].view(4, 8)),
                             (fake(4, 8), buf[:32].view(4, 8), buf[8:40].view(4, 8)), (w[:4], None, w[4:]),
                             (fake(4, 8), None, w[:4])):
        with pytest.raises(ValueError, match="overlap"):
            experts.linear(x, w, residual=residual, out=out)
    with pytest.raises(ValueError, match="overlap bias"):
        experts.linear(fake(4, 8), w, bias=buf[20:28], out=buf[:32].view(4, 8))
    for x, residual, out in ((wide[:4, :8], None, wide[:4, 8:16]), (wide[:4, 16:], None, wide[:4, 8:16]),
                             (buf[:32].view(4, 8), None, buf[32:].view(4, 8)), (wide[:1, :8], None, wide[1:2, 2:10]),
                             (wide[:4, :8], wide[:4, 8:16], wide[:4, 8:16]), (wide[:4, 8:16], None, wide[1:5, 16:])):
        experts._refuse_overlap(out, x, "x")
        if residual is not None:
            with pytest.raises(ValueError, match="overlap"):
                experts._refuse_overlap(out, residual, "residual")


def _product(**kw):
    p = _native.ExpertProduct(x=64, w=64, y=64, rows=4, k=8, n=6, experts=1, ldx=8, w_stride_e=48, w_stride_k=6, w_stride_n=1,
                              ldy=6)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,status", [
    (dict(rows=-1), -1), (dict(k=0), -1), (dict(n=0), -1), (dict(experts=0), -1), (dict(experts=1025, offsets=64), -1),
    (dict(experts=2), -1), (dict(dtype=2), -1), (dict(activation=4), -1), (dict(gated=1, n=7), -1), (dict(w_stride_n=2), -1),
    (dict(x=None), -1), (dict(y=None), -1), (dict(ldy=5), -1), (dict(rows=1 << 31), -1), (dict(w=65), -4),
    (dict(), -2),        # 6 columns are not a multiple of 16 bytes: a workspace is needed
])
def test_c_entry_refuses(change, status):
    """Status codes of the C entry points; the pointers are never followed."""
    L, p = _native.load(), _product(**change)
    assert L.kq_expert_linear(ctypes.byref(p), None, 0, None) == status
    assert L.kq_last_error()


def test_c_entries_refuse_null():
    L = _native.load()
    assert L.kq_expert_linear(None, None, 0, None) == -1
    assert L.kq_expert_linear_grad_z(None, None, 0, None, 0, None) == -1
    assert L.kq_expert_weight_grad(None, None, 0, None, None, 0, None) == -1
    assert L.kq_expert_weight_grad(ctypes.byref(_product()), None, 0, 64, None, 0, None) == -1
    assert L.kq_expert_bias_grad(None, None, 0, None, 4, 8, 1, 0, None, 0, None) == -1
    assert L.kq_wait_errors(None, None) == -1
    assert L.kq_expert_linear_workspace_bytes(None) == 0
    # Nothing to do: no pointer is needed.
    assert L.kq_expert_linear(ctypes.byref(_product(rows=0, x=None, y=None)), None, 0, None) == 0


@pytest.mark.parametrize("change,error,match", [
    (dict(rows=fake(4, 8, dtype=torch.float64)), TypeError, "rows must be"),
    (dict(rows=torch.zeros(4, 8)), _native.KQError, "CUDA"),
    (dict(rows=fake(4, 16)[:, ::2]), ValueError, "unit stride"),
    (dict(rows=fake(4, 0)), ValueError, "at least one column"),
    (dict(offsets=fake(1, dtype=torch.int64)), ValueError, "experts"),
    (dict(offsets=fake(3, dtype=torch.int32)), TypeError, "int64"),
    (dict(index=fake(4, dtype=torch.int32)), TypeError, "int64"),
    (dict(index=fake(8, dtype=torch.int64)[::2]), ValueError, "contiguous"),
    (dict(weights=fake(3, dtype=torch.float32)), ValueError, "4 values"),
    (dict(weights=fake(4)), TypeError, "float32"),
    (dict(out=fake(2, 8, 7, dtype=torch.float32)), ValueError, "out must be"),
    (dict(out=fake(2, 8, 8)), TypeError, "out must be"),
])
def test_expert_hessians_refuse(change, error, match):
    from kquant_b200.capture import accumulate_expert_hessians
    args = dict(rows=fake(4, 8), offsets=fake(3, dtype=torch.int64))
    args.update(change)
    with pytest.raises(error, match=match):
        accumulate_expert_hessians(**args)


@pytest.mark.parametrize("change,status", [
    (dict(tokens=-1), -1), (dict(dim=0), -1), (dict(ldx=7), -1), (dict(dtype=3), -1), (dict(offsets=None), -1), (dict(rows=5), -1),
    (dict(experts=0), -1), (dict(experts=2000), -1), (dict(H=None), -1), (dict(h_stride=63), -1), (dict(ldh=7), -1), (dict(den=None), -1),
    (dict(), -2), (dict(ws=200, size=1 << 20), -4), (dict(x=None), -1),
])
def test_expert_hessian_c_entry_refuses(change, status):
    a = dict(x=64, tokens=4, dim=8, ldx=8, dtype=0, index=None, w=None, offsets=64, rows=4, experts=2, H=64, h_stride=64, ldh=8, add=0,
             den=64, ws=None, size=0, stream=None)
    a.update(change)
    assert _native.load().kq_accumulate_expert_hessians(*a.values()) == status


@pytest.mark.parametrize("change,error,match", [
    (dict(x=torch.zeros(4, 128, dtype=torch.bfloat16)), _native.KQError, "CUDA"),
    (dict(x=fake(4, 128, dtype=torch.float32)), TypeError, "bfloat16"),
    (dict(x=fake(4, 256)), ValueError, "x must be"),
    (dict(trellis=fake(2, 8, 8, 48, dtype=torch.int32)), TypeError, "int16"),
    (dict(trellis=fake(2, 8, 8, 40, dtype=torch.int16)), ValueError, "16 K"),
    (dict(trellis=fake(2, 8, 8, 144, dtype=torch.int16)), ValueError, "K in 1..8"),
    (dict(trellis=fake(2, 8, 16, 48, dtype=torch.int16)[:, :, ::2]), ValueError, "contiguous"),
    (dict(trellis=fake(2, 8, 9, 48, dtype=torch.int16)), ValueError, "multiples of 128"),
    (dict(suh=fake(2, 128)), TypeError, "suh"),
    (dict(svh=fake(2, 64, dtype=torch.float16)), ValueError, "svh"),
    (dict(offsets=None), ValueError, "offsets"),
    (dict(codebook=fake(65536, dtype=torch.int32)), TypeError, "codebook"),
    (dict(codebook=fake(4096, dtype=torch.uint8)), ValueError, "65,536"),
    (dict(out=fake(4, 64)), ValueError, "out"),
])
def test_trellis_linear_refuses(change, error, match):
    args = dict(x=fake(4, 128), trellis=fake(2, 8, 8, 48, dtype=torch.int16), suh=fake(2, 128, dtype=torch.float16),
                svh=fake(2, 128, dtype=torch.float16), offsets=fake(3, dtype=torch.int64))
    args.update(change)
    with pytest.raises(error, match=match):
        experts.trellis_linear(**args)


@pytest.mark.parametrize("change,status", [
    (dict(rows=-1), -1), (dict(k=64), -1), (dict(n=130), -1), (dict(experts=0), -1), (dict(bits=0), -1), (dict(bits=9), -1),
    (dict(experts=2, offsets=None), -1), (dict(dtype=2), -1), (dict(codebook=2), -1), (dict(ldx=100), -1), (dict(x=None), -1),
    (dict(codebook=4), -1), (dict(trellis=72), -4), (dict(), -2),
])
def test_trellis_c_entry_refuses(change, status):
    p = _native.TrellisProduct(x=64, trellis=64, suh=64, svh=64, offsets=64, y=64, rows=4, k=128, n=128, experts=1, ldx=128, ldy=128,
                               suh_stride_e=128, svh_stride_e=128, bits=3, codebook=1)
    for k, v in change.items():
        setattr(p, k, v)
    assert _native.load().kq_trellis_linear(ctypes.byref(p), None, 0, None) == status
    assert _native.load().kq_trellis_linear(None, None, 0, None) == -1

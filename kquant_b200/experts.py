"""The expert layer around the encode: products with the experts' matrices, and their gradients.

Rows are sorted by expert: rows ``offsets[e] .. offsets[e + 1]`` of ``x`` belong to expert e (``offsets``: int64
[experts + 1], non-decreasing, on the GPU).  The kernels read the offsets, the host never does, so no call waits for
the GPU and a call captured into a graph follows new offsets at replay.  Rows before ``offsets[0]`` and from
``offsets[-1]`` on belong to no expert: a fresh output holds zeros there, an ``out`` given by the caller keeps what
it had.

Matrices are [in, out] (EXL orientation), as the encoder takes and reconstructs them; a transposed view of the HF
orientation ([out, in]) is taken as it is.  Operands are bf16 or fp16, sums are fp32, each result is rounded once.
Bases, strides and widths that are not multiples of 16 bytes are accepted and cost one more pass over that operand.

The results carry no autograd history; :func:`expert_linear_grad` computes the gradients.
"""

from __future__ import annotations

import torch

from . import _native

# Every wait inside the kernels is bounded.  Should one run out, later calls on that device raise until this has been called.
check_wait_errors = _native.check_wait_errors

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3}


def _operand(t: torch.Tensor, name: str, dims: int, dtype: torch.dtype, device: torch.device) -> None:
    if t.is_cuda and t.dtype is dtype and t.ndim == dims and t.device == device:
        return
    if not t.is_cuda:
        raise _native.KQError(f"{name} must be a CUDA tensor (kquant_b200 has no CPU path)")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    raise ValueError(f"{name} must have {dims} dimensions, got {t.ndim}")


def _rows_operand(t: torch.Tensor, name: str, rows: int, width: int, dtype: torch.dtype, device: torch.device) -> int:
    """The row stride of a [rows, width] operand."""
    _operand(t, name, 2, dtype, device)
    if t.shape != (rows, width):
        raise ValueError(f"{name} must be [{rows}, {width}], got {list(t.shape)}")
    ld, unit = t.stride()
    if unit != 1 and width > 1:
        raise ValueError(f"{name} needs unit stride along its last dimension")
    return ld


def _check_offsets(offsets: torch.Tensor | None, experts: int, device: torch.device) -> None:
    if offsets is None:
        if experts != 1:
            raise ValueError("several experts need offsets")
        return
    _operand(offsets, "offsets", 1, torch.int64, device)
    if offsets.numel() != experts + 1 or not offsets.is_contiguous():
        raise ValueError(f"offsets must be {experts + 1} contiguous values for {experts} experts")


def _span(t: torch.Tensor) -> tuple[int, int]:
    """First byte and end of what a tensor's elements lie in."""
    return t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _refuse_overlap(out: torch.Tensor, t: torch.Tensor | None, name: str) -> None:
    """The kernels read operands while others write results; columns of one buffer beside each other are apart."""
    if t is None or not t.numel() or not out.numel():
        return
    (a, a_end), (b, b_end) = _span(out), _span(t)
    if a_end <= b or b_end <= a:
        return
    if t.ndim == out.ndim == 2 and t.element_size() == out.element_size() and t.stride(0) == out.stride(0) > 0 and name != "bias":
        ld, by = out.stride(0), (b - a) // out.element_size() % out.stride(0)      # where t's rows begin among out's
        if by >= out.shape[1] and by + t.shape[1] <= ld:
            return
    raise ValueError(f"out must not overlap {name}")


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _product(x, w, offsets, bias, activation, gated, dense=False) -> _native.ExpertProduct:
    """The checked operands that every product of these shares; ``dense``: one matrix [k, n] and its bias [n]."""
    if not isinstance(x, torch.Tensor) or not isinstance(w, torch.Tensor):
        raise TypeError("x and w must be tensors")
    dt, dev = x.dtype, x.device
    if dt not in _DTYPES:
        raise TypeError(f"x must be torch.bfloat16 or torch.float16, got {dt}")
    _operand(x, "x", 2, dt, dev)
    p = _native.ExpertProduct()
    if dense:
        _operand(w, "w", 2, dt, dev)
        E, (k, n) = 1, w.shape
        p.w_stride_k, p.w_stride_n = sk, sn = w.stride()
    else:
        _operand(w, "w", 3, dt, dev)
        E, k, n = w.shape
        p.w_stride_e, p.w_stride_k, p.w_stride_n = _, sk, sn = w.stride()
    if E < 1 or k < 1 or n < 1:
        raise ValueError(f"w must not be empty, got {list(w.shape)}")
    rows = x.shape[0]
    p.rows, p.k, p.n, p.experts = rows, k, n, E
    p.ldx = _rows_operand(x, "x", rows, k, dt, dev)
    if sk != 1 and sn != 1 and k > 1 and n > 1:
        raise ValueError("w needs unit stride along its in or its out dimension")
    _check_offsets(offsets, E, dev)
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {[a for a in _ACTIVATIONS]}, got {activation!r}")
    if gated and n % 2:
        raise ValueError("a gated product needs an even out dimension (gate, then up)")
    if bias is not None:
        _operand(bias, "bias", 1 if dense else 2, dt, dev)
        if bias.shape != ((n,) if dense else (E, n)) or (n > 1 and bias.stride(-1) != 1):
            raise ValueError(f"bias must be [{'' if dense else f'{E}, '}{n}] with unit stride along its last dimension, got {list(bias.shape)}")
        p.bias = bias.data_ptr()
        if not dense:
            p.bias_stride_e = bias.stride(0)
    p.x, p.w = x.data_ptr(), w.data_ptr()
    if offsets is not None:
        p.offsets = offsets.data_ptr()
    p.dtype, p.activation, p.gated = _DTYPES[dt], _ACTIVATIONS[activation], 1 if gated else 0
    return p


def _linear(p: _native.ExpertProduct, x, w, offsets, bias, residual, out) -> torch.Tensor:
    """The forward product behind checked operands."""
    n_out, rows, dt, dev = p.n // 2 if p.gated else p.n, p.rows, x.dtype, x.device
    if residual is not None:
        p.ld_residual = _rows_operand(residual, "residual", rows, n_out, dt, dev)
        p.residual = residual.data_ptr()
    if out is None:
        out = torch.empty((rows, n_out), dtype=dt, device=dev)
        p.ldy, p.zero_rest = n_out, 1
    else:
        p.ldy = _rows_operand(out, "out", rows, n_out, dt, dev)
        _refuse_overlap(out, x, "x")
        _refuse_overlap(out, w, "w")
        _refuse_overlap(out, bias, "bias")
        _refuse_overlap(out, offsets, "offsets")
        if residual is not None and (residual.data_ptr(), residual.stride()) != (out.data_ptr(), out.stride()):
            _refuse_overlap(out, residual, "residual other than as the same view")
    if rows:
        p.y = out.data_ptr()
        _native.expert_linear(p, dev)
    return out


def expert_linear(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor | None, *, bias: torch.Tensor | None = None,
                  activation: str | None = None, gated: bool = False, residual: torch.Tensor | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """y[r] = act(x[r] w[e] + bias[e]) + residual[r] for the rows r of each expert e.

    x [rows, k], w [experts, k, n], bias [experts, n], residual and y [rows, n].  ``gated``: w holds the gate's
    columns and then the up projection's, y = act(gate) * up + residual has n / 2 columns.  ``activation``: None,
    "relu", "silu" or "gelu" (the error-function form).  ``out`` may be the residual itself, and overlaps no operand otherwise.
    """
    return _linear(_product(x, w, offsets, bias, activation, gated), x, w, offsets, bias, residual, out)


def linear(x: torch.Tensor, w: torch.Tensor, *, bias: torch.Tensor | None = None, activation: str | None = None,
           gated: bool = False, residual: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """act(x w + bias) + residual with one matrix w [k, n] and bias [n]; see :func:`expert_linear`."""
    return _linear(_product(x, w, None, bias, activation, gated, dense=True), x, w, None, bias, residual, out)


def expert_linear_grad(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor | None, *,
                       bias: torch.Tensor | None = None, activation: str | None = None, gated: bool = False,
                       need_dx: bool = True, need_dw: bool = True):
    """Gradients (dx, dw, dbias) of :func:`expert_linear` for dy, the gradient of its result.

    The pre-activation z = x w + bias is recomputed where the activation needs it; dz (one rounding to the operands'
    type) then feeds dx = dz w^T and dw[e] = x_e^T dz_e; dbias[e] = sum dz_e is taken of it unrounded.  dw has w's layout; an expert without
    rows gets zeros.  dbias is None without a bias, dx and dw where they are not asked for.  The residual's gradient
    is dy itself.
    """
    p = _product(x, w, offsets, bias, activation, gated)
    dev, dt = x.device, x.dtype
    _rows_operand(dy, "dy", p.rows, p.n // 2 if gated else p.n, dt, dev)
    E, k, n = w.shape
    dz, low = dy, None
    if p.rows and (gated or activation is not None):
        dz = torch.empty((p.rows, -(-n // 8) * 8), dtype=dt, device=dev)[:, :n]
        p.y, p.ldy = dz.data_ptr(), dz.stride(0)
        if bias is not None:
            low = torch.empty((p.rows, p.ldy), dtype=dt, device=dev)     # laid out as dz: the sums of db take dz as it was before its rounding
            p.y_low = low.data_ptr()
        _native.expert_linear_grad_z(p, dy, dev)
    elif gated:
        dz = dy.new_empty((0, n))
    dx = dw = db = None
    if need_dx:
        dx = torch.empty((p.rows, k), dtype=dt, device=dev)
        if p.rows:                                  # dz w^T: the product with in and out exchanged
            q = _native.ExpertProduct(x=dz.data_ptr(), w=p.w, offsets=p.offsets, y=dx.data_ptr(), rows=p.rows, k=n, n=k, experts=E,
                                      ldx=dz.stride(0), w_stride_e=p.w_stride_e, w_stride_k=p.w_stride_n, w_stride_n=p.w_stride_k,
                                      ldy=k, dtype=p.dtype, zero_rest=1)
            _native.expert_linear(q, dev)
    if need_dw:
        n_major = not (w.stride(2) != 1 and w.stride(1) == 1)
        dw = torch.empty((E, k, n), dtype=dt, device=dev) if n_major else \
            torch.empty((E, n, k), dtype=dt, device=dev).transpose(1, 2)
        p.w_stride_e, p.w_stride_k, p.w_stride_n = k * n, n if n_major else 1, 1 if n_major else k
        p.gated, p.activation = 0, 0
        _native.expert_weight_grad(p, dz, dw, dev)
    if bias is not None:
        db = torch.empty((E, n), dtype=dt, device=dev)
        _native.expert_bias_grad(dz, low, offsets, db, p.dtype)
    return dx, dw, db


def trellis_linear(x: torch.Tensor, trellis: torch.Tensor, suh: torch.Tensor, svh: torch.Tensor,
                   offsets: torch.Tensor | None = None, *, codebook: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """x[r] times the encoded matrix of each row's expert, decoded from its packed payload on the way.

    x [rows, k] bf16 or fp16, trellis [experts, k/16, n/16, 16 K] int16 as the encoder packs it, suh [experts, k] and
    svh [experts, n] fp16: ``{"suh", "svh", "trellis"}`` of the encoder's results, stacked over the experts of one
    rate K.  One encoded matrix goes without the experts dimension and without offsets.  ``codebook``: None for MCG,
    the 65,536 E4M3 bytes of an SQG table, or 65,536 binary16 labels (int16 bits, ``_native.build_labels``).
    ``out`` may lie over x, which is read before the first result is written; it overlaps no other operand.
    """
    if not isinstance(x, torch.Tensor) or x.dtype not in _DTYPES:
        raise TypeError("x must be a torch.bfloat16 or torch.float16 tensor")
    dev = x.device
    if isinstance(trellis, torch.Tensor) and trellis.ndim == 3 and offsets is None:
        trellis, suh, svh = trellis[None], suh[None], svh[None]
    _operand(x, "x", 2, x.dtype, dev)
    _operand(trellis, "trellis", 4, torch.int16, dev)
    E, k, n, K = trellis.shape[0], 16 * trellis.shape[1], 16 * trellis.shape[2], trellis.shape[3] // 16
    if not trellis.is_contiguous() or trellis.shape[3] % 16 or not 1 <= K <= 8:
        raise ValueError("trellis must be contiguous [experts, k/16, n/16, 16 K] words with K in 1..8")
    if E < 1 or k < 1 or n < 1 or k % 128 or n % 128:
        raise ValueError(f"trellis must hold at least one matrix with k and n multiples of 128, got {E} of [{k}, {n}]")
    rows = x.shape[0]
    ldx = _rows_operand(x, "x", rows, k, x.dtype, dev)
    _check_offsets(offsets, E, dev)
    for name, t, size in (("suh", suh, k), ("svh", svh, n)):
        _operand(t, name, 2, torch.float16, dev)
        if t.shape != (E, size) or t.stride(1) != 1:
            raise ValueError(f"{name} must be [{E}, {size}] with unit stride along its last dimension")
    p = _native.TrellisProduct()
    p.codebook = _native.KQ_CB_MCG
    if codebook is not None:
        if not isinstance(codebook, torch.Tensor) or codebook.dtype not in (torch.uint8, torch.int16):
            raise TypeError("codebook must be None, uint8 E4M3 bytes or int16 binary16 labels")
        _operand(codebook, "codebook", 1, codebook.dtype, dev)
        if codebook.numel() != 65536 or not codebook.is_contiguous():
            raise ValueError("codebook must hold 65,536 contiguous values")
        p.codebook = _native.KQ_CB_SQG if codebook.dtype == torch.uint8 else _native.KQ_CB_LABELS
        p.table = codebook.data_ptr()
    if out is None:
        out = torch.empty((rows, n), dtype=x.dtype, device=dev)
        p.ldy, p.zero_rest = n, 1
    else:
        p.ldy = _rows_operand(out, "out", rows, n, x.dtype, dev)
        for name, t in (("trellis", trellis), ("suh", suh), ("svh", svh), ("offsets", offsets), ("codebook", codebook)):
            _refuse_overlap(out, t, name)
    p.x, p.trellis, p.suh, p.svh, p.offsets, p.y = (x.data_ptr(), trellis.data_ptr(), suh.data_ptr(), svh.data_ptr(),
                                                    _ptr(offsets), out.data_ptr())
    p.rows, p.k, p.n, p.experts = rows, k, n, E
    p.ldx, p.suh_stride_e, p.svh_stride_e = ldx, suh.stride(0), svh.stride(0)
    p.bits, p.dtype = K, _DTYPES[x.dtype]
    if rows:
        _native.trellis_linear(p, dev)
    return out

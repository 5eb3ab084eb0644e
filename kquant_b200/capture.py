"""Hessian accumulation H = sum_t w_t x_t x_t^T on the tensor cores.

Mirrors kquant/capture.py:713-730 (``_accumulate_hessian``): rows [T, d]
and weights [T] stream in chunks of ``chunk_rows``; returns (accumulator
[d, d] fp32, denominator = sum of weights).  Each chunk is one call of
``kq_accumulate_hessian``: an operand kernel (transpose, weighting, TF32
hi/lo split) and one tcgen05 GEMM over the upper-triangle tiles, mirrored.
Precision ``"3xtf32"`` (default) accumulates hi*hi + hi*lo + lo*hi and
drains the tensor-core accumulator into fp32 registers every 128 samples,
which matches the accuracy of the reference's FP32 addmm; ``"tf32"``
issues the single TF32 product.  The result is exactly symmetric.
"""

from __future__ import annotations

import torch

from . import _native, experts

_SPLIT = {"3xtf32": 3, "tf32": 1}


def accumulate_hessian(rows: torch.Tensor, weights: torch.Tensor, *, device: torch.device, chunk_rows: int,
                       precision: str = "3xtf32", out: torch.Tensor | None = None) -> tuple[torch.Tensor, float]:
    if rows.ndim != 2 or weights.ndim != 1 or rows.shape[0] != weights.shape[0]:
        raise ValueError("invalid Hessian sample shapes")
    if precision not in _SPLIT:
        raise ValueError("precision must be '3xtf32' or 'tf32'")
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError("accumulate_hessian requires a CUDA device (kquant_b200 has no CPU path)")
    dim = int(rows.shape[1])
    acc = out if out is not None else torch.zeros((dim, dim), dtype=torch.float32, device=device)
    den = torch.zeros((), dtype=torch.float64, device=device)
    step = max(int(chunk_rows), 1)
    ws = None
    for start in range(0, int(rows.shape[0]), step):
        x = rows[start:start + step].to(device=device, dtype=torch.float32).contiguous()
        w = weights[start:start + step].to(device=device, dtype=torch.float32).contiguous()
        den += w.double().sum()
        ws = _native.accumulate_hessian(x, w, acc, _SPLIT[precision], ws)
    _native.check_trace_errors()
    return acc, float(den.item())


_ROW_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def accumulate_expert_hessians(rows: torch.Tensor, offsets: torch.Tensor, *, index: torch.Tensor | None = None,
                               weights: torch.Tensor | None = None,
                               out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The Hessians of all experts of a layer in one call: H[e] = sum_t w_t x_t x_t^T over the slots
    ``offsets[e] .. offsets[e + 1]``.

    ``rows`` [tokens, d] bf16, fp16 or fp32 on the GPU.  ``index`` (int64) names the row of each slot, as routing
    gives it (a row may serve several experts, and an index outside the rows counts for nothing); without it slot t
    is row t.  ``weights`` fp32, one per slot.  Returns (H [experts, d, d] fp32, denominators [experts] fp64, the
    sums of the weights), both on the GPU: nothing waits for the device.  A fresh H whose d is not a multiple of 32 is a
    view with rows padded to one.  With ``out`` the sums are added to it,
    which is how samples stream in (it overlaps no operand); the denominators are this call's alone.  fp32 accuracy for every type.
    Infinity or NaN in a row that counts makes infinity or NaN of that row's share of H (NaN also where the products alone would be
    infinite, with weights or fp32 rows).
    """
    if not isinstance(rows, torch.Tensor) or rows.dtype not in _ROW_DTYPES:
        raise TypeError("rows must be a torch.bfloat16, torch.float16 or torch.float32 tensor")
    dev = rows.device
    experts._operand(rows, "rows", 2, rows.dtype, dev)
    experts._operand(offsets, "offsets", 1, torch.int64, dev)
    if offsets.numel() < 2 or not offsets.is_contiguous():
        raise ValueError("offsets must be experts + 1 contiguous values")
    E, (tokens, d) = offsets.numel() - 1, rows.shape
    if d < 1 or (d > 1 and rows.stride(1) != 1):
        raise ValueError("rows needs at least one column and unit stride along its last dimension")
    slots = tokens
    if index is not None:
        experts._operand(index, "index", 1, torch.int64, dev)
        slots = index.numel()
    if weights is not None:
        experts._operand(weights, "weights", 1, torch.float32, dev)
        if weights.numel() != slots:
            raise ValueError(f"weights must have {slots} values, got {weights.numel()}")
    for name, t in (("index", index), ("weights", weights)):
        if t is not None and not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    if out is not None:
        experts._operand(out, "out", 3, torch.float32, dev)
        if out.shape != (E, d, d) or (d > 1 and out.stride(2) != 1):
            raise ValueError(f"out must be [{E}, {d}, {d}] with unit stride along its last dimension")
        for name, t in (("rows", rows), ("offsets", offsets), ("index", index), ("weights", weights)):
            experts._refuse_overlap(out, t, name)
    if tokens > 1 and rows.stride(0) < d:
        rows = rows.contiguous()
    # Rows of a fresh H start on 128-byte lines: with d floats a row, an odd d splits every line that is written.
    H = out if out is not None else torch.empty((E, d, -(-d // 32) * 32), dtype=torch.float32, device=dev)[:, :, :d]
    den = torch.empty(E, dtype=torch.float64, device=dev)
    _native.accumulate_expert_hessians(rows, _ROW_DTYPES[rows.dtype], index, weights, offsets, slots, H, out is not None, den)
    return H, den


def expert_layer_hessians(tokens: torch.Tensor, index: torch.Tensor, offsets: torch.Tensor, w13: torch.Tensor, *,
                          weights: torch.Tensor | None = None, activation: str | None = "silu",
                          bias: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Both calibration Hessians of every expert of a layer from its routed tokens, on the GPU throughout.

    tokens [T, k] bf16 or fp16; ``index`` (int64) the token of each routed slot, slots sorted by expert behind
    ``offsets``; w13 [experts, k, 2 I] the gate's columns and then the up projection's (``weights``, ``activation`` and
    ``bias`` as in :func:`accumulate_expert_hessians` and ``experts.expert_linear``).  Returns (H13 [experts, k, k] of
    the inputs of gate and up, H2 [experts, I, I] of act(gate) * up, the inputs of the down projection, and the
    denominators): the (x13, x2) pair of kquant/capture.py:1268-1273 for a whole layer.  Slots whose index is outside
    the tokens count for nothing in either.
    """
    if index is None:
        raise ValueError("index must name the token of each slot")
    H13, den = accumulate_expert_hessians(tokens, offsets, index=index, weights=weights)
    valid = (index >= 0) & (index < tokens.shape[0])
    rows = tokens.index_select(0, index.clamp(0, max(tokens.shape[0] - 1, 0))) if tokens.shape[0] else \
        tokens.new_zeros((index.numel(), tokens.shape[1]))
    hidden = experts.expert_linear(rows, w13, offsets, bias=bias, activation=activation, gated=True)
    slot = torch.where(valid, torch.arange(index.numel(), device=index.device), -1)
    H2, _ = accumulate_expert_hessians(hidden, offsets, index=slot, weights=weights)
    return H13, H2, den


# the reference's private name, for callers that import it directly
_accumulate_hessian = accumulate_hessian

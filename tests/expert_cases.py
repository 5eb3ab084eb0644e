"""Inputs, 64-bit results and error bounds shared by the expert-layer tests.

A bound is built from what the operators document: products of 16-bit values are exact in fp32, a sum of k of them
is taken 16 at a time into an fp32 accumulator that may truncate (at most (k / 16 + 16) 2^-23 of the sum of the
absolute products), exp is good to 2^-20 relative, and every result is rounded once (half a step of its type).
"""
import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -149}


def sum_slack(k):
    return (k / 16 + 16) * 2.0 ** -23


def offsets_of(counts, device, first=0):
    edge = [first]
    for c in counts:
        edge.append(edge[-1] + c)
    return torch.tensor(edge, dtype=torch.int64, device=device)


def groups(offsets):
    o = offsets.tolist()
    return [slice(a, b) for a, b in zip(o, o[1:])]


def act64(name, z):
    if name == "relu":
        return z.clamp_min(0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
    return z


def slope64(name, z):
    if name == "relu":
        return (z > 0).double()
    if name == "silu":
        p = torch.sigmoid(z)
        return p * (1 + z * (1 - p))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z / math.sqrt(2))) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def forward64(x, w, bias, act, gated, residual):
    """(y, bound) of one expert's rows in 64 bits; w [k, n]."""
    dt = x.dtype
    k, n = w.shape
    z = x.double() @ w.double()
    dz = (x.double().abs() @ w.double().abs()) * sum_slack(k)
    if bias is not None:
        z = z + bias.double()
        dz = dz + z.abs() * 2.0 ** -23
    if gated:
        g, u, dg, du = z[:, : n // 2], z[:, n // 2:], dz[:, : n // 2], dz[:, n // 2:]
        a = act64(act, g)
        y, e = a * u, u.abs() * (1.13 * dg + a.abs() * 2.0 ** -19) + a.abs() * du + dg * du
    else:
        y, e = act64(act, z), 1.13 * dz + act64(act, z).abs() * 2.0 ** -19
    if act in ("silu", "gelu"):                   # 1 + exp and 1 + erf cancel or round at 2^-23 of 1
        s = z[:, : n // 2] if gated else z
        e = e + s.abs() * 2.0 ** -22 * (z[:, n // 2:].abs() if gated else 1)
    if residual is not None:
        y = y + residual.double()
        e = e + y.abs() * 2.0 ** -23
    return y, e + (y.abs() + e) * HALF_STEP[dt] + TINY[dt]


def grad64(dy, x, w, bias, act, gated):
    """(dx, bound), (dw, bound), (db, bound) of one expert."""
    dt = x.dtype
    k, n = w.shape
    X, W, D = x.double(), w.double(), dy.double()
    if not gated and act is None:
        dz, e = D, torch.zeros_like(D)
        e_sum = e
    else:
        z = X @ W + (0 if bias is None else bias.double())
        ez = (X.abs() @ W.abs()) * sum_slack(k) + z.abs() * 2.0 ** -23
        if gated:
            g, u, eg, eu = z[:, : n // 2], z[:, n // 2:], ez[:, : n // 2], ez[:, n // 2:]
            a, s = act64(act, g), slope64(act, g)
            dz = torch.cat((D * u * s, D * a), 1)
            es = eg + (1 + g.abs()) * 2.0 ** -19          # |second derivative| of silu and gelu is below 1
            e = torch.cat((D.abs() * (u.abs() * es + 1.13 * eu + es * eu), D.abs() * (1.13 * eg + (1 + g.abs()) * 2.0 ** -19)), 1)
        else:
            dz = D * slope64(act, z)
            e = D.abs() * (ez + (1 + z.abs()) * 2.0 ** -19)
        if act == "relu":                                  # a step: where z may lie on either side, either slope is right
            s = (z[:, : n // 2] if gated else z)
            near = s.abs() <= (ez[:, : n // 2] if gated else ez)
            full = D.abs() * (z[:, n // 2:].abs() if gated else 1)
            if gated:
                e[:, : n // 2] += near * full
            else:
                e += near * full
        e_sum = e + (dz.abs() + e) * HALF_STEP[dt] ** 2 + TINY[dt]     # db: of dz in two terms
        e = e + (dz.abs() + e) * HALF_STEP[dt] + TINY[dt]

    def rounded(v, b):
        return v, b + (v.abs() + b) * HALF_STEP[dt] + TINY[dt]

    rows = x.shape[0]
    dx = rounded(dz @ W.T, e @ W.abs().T + (dz.abs() @ W.abs().T) * sum_slack(n))
    dw = rounded(X.T @ dz, X.abs().T @ e + (X.abs().T @ dz.abs()) * sum_slack(rows))
    db = rounded(dz.sum(0), e_sum.sum(0) + dz.abs().sum(0) * (rows + 8) * 2.0 ** -24)
    return dx, dw, db


def check(got, want, bound, what=""):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    if bool(bad.any()):
        i = int((off / bound.clamp_min(1e-300)).nan_to_num(nan=math.inf).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; worst at {i}: got {got.flatten()[i].item()!r}, "
                             f"want {want.flatten()[i].item()!r}, bound {bound.flatten()[i].item()!r}")

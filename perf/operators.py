"""The operators of an expert layer around its encode, measured case by case.

Five operators, each on rows that are sorted by expert (rows ``offsets[e] .. offsets[e + 1]`` belong to expert e):

* ``linear``: one matrix product with bias, activation and residual in its epilogue;
* ``expert_linear``: the same grouped by expert, ragged, with the gated form act(x Wg) * (x Wu);
* ``expert_linear_grad``: its gradients in x, w and bias;
* ``hessians``: the calibration Hessians sum_t w_t x_t x_t^T of every expert at once, rows picked by index;
* ``trellis_linear``: the product with the packed trellis payload of encoded experts.

With ``own`` false ``run`` computes them from elementary torch operations in 32 bits; with ``own`` true it calls
the framework's operators.
"""

import math
import random

import torch

own = False  # whether run() calls the framework's operators

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MCG_MULTIPLIER = 0xCBAC1FED
STATES = 1 << 16
BLOCK = 128  # channels of one Hadamard block


# ------------------------------------------------------------------ cases


def listed():
    return [
        # Serving: eight experts see one token each (gate and up projections of a 7168-channel layer).
        dict(name="gated, one token an expert", op="expert_linear", rows=8, experts=8, split=0, skew=0.0, k=7168, n=4096,
             gated=True, act="silu", bias=False, residual=False, dtype="bf16", layout="hf", spare=0),
        # Calibration: about 64 routed tokens an expert through gate and up, the inputs of the down Hessians.
        dict(name="gated, calibration tokens", op="expert_linear", rows=512, experts=8, split=1, skew=0.5, k=7168, n=4096,
             gated=True, act="silu", bias=False, residual=False, dtype="bf16", layout="exl", spare=3),
        # A prompt through the down projections, unevenly routed, added to the residual stream.
        dict(name="down, prompt", op="expert_linear", rows=8192, experts=16, split=2, skew=1.0, k=2048, n=7168,
             gated=False, act=None, bias=False, residual=True, dtype="fp16", layout="exl", spare=0),
        # The smallest call: a few rows of a small odd matrix, where latency counts.
        dict(name="linear, small and odd", op="linear", rows=5, experts=1, split=0, skew=0.0, k=331, n=517,
             gated=False, act="gelu", bias=True, residual=True, dtype="bf16", layout="exl", spare=0),
        # An attention projection over 8192 calibration tokens.
        dict(name="linear, 8192 tokens", op="linear", rows=8192, experts=1, split=0, skew=0.0, k=1536, n=12288,
             gated=False, act="silu", bias=True, residual=False, dtype="bf16", layout="hf", spare=0),
        # A training step of gate and up on 4096 routed rows.
        dict(name="gated gradients, 4096 rows", op="expert_linear_grad", rows=4096, experts=8, split=3, skew=0.7, k=7168,
             n=4096, gated=True, act="silu", bias=False, residual=False, dtype="bf16", layout="hf", spare=0),
        # A small odd layer's gradients, one expert without rows.
        dict(name="gradients, small and odd", op="expert_linear_grad", rows=299, experts=5, split=4, skew=1.0, k=264, n=136,
             gated=False, act="gelu", bias=True, residual=False, dtype="fp16", layout="exl", spare=2),
        # Calibration of eight experts from routed bf16 activations: 64 rows an expert out of 8192 tokens' rows.
        dict(name="hessians, routed bf16", op="hessians", rows=512, experts=8, split=5, skew=0.5, tokens=1024, k=7168,
             weighted=False, dtype="bf16"),
        # The down projections' Hessians from many weighted fp32 rows.
        dict(name="hessians, weighted fp32", op="hessians", rows=8192, experts=4, split=6, skew=0.5, tokens=8192, k=2048,
             weighted=True, dtype="fp32"),
        # A small odd calibration, where latency counts.
        dict(name="hessians, small and odd", op="hessians", rows=77, experts=3, split=7, skew=1.0, tokens=50, k=300,
             weighted=True, dtype="bf16"),
        # Serving from the packed payload: eight experts, one token each.
        dict(name="trellis, one token an expert", op="trellis_linear", rows=8, experts=8, split=0, skew=0.0, k=7168, n=2048,
             bits=3, table=True, dtype="bf16"),
        # A prompt on the packed payload.
        dict(name="trellis, prompt", op="trellis_linear", rows=2048, experts=8, split=8, skew=0.7, k=2048, n=7168,
             bits=4, table=False, dtype="fp16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.4e12, w["flops"] / 6e13)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["expert_linear", "linear", "expert_linear_grad", "hessians", "trellis_linear"])
        experts = 1 if op == "linear" else _log_uniform(rng, 1, 32)
        case = dict(op=op, rows=_log_uniform(rng, 1, 8192), experts=experts, split=rng.randrange(1 << 20),
                    skew=rng.choice([0.0, 0.5, 1.0, 2.0]))
        case["dtype"] = rng.choice(["bf16", "fp16"])
        if op == "hessians":
            case["dtype"] = rng.choice(["bf16", "fp16", "fp32"])
            case.update(tokens=_log_uniform(rng, 1, 8192), k=_log_uniform(rng, 16, 7168), weighted=rng.random() < 0.5)
        elif op == "trellis_linear":
            case.update(k=BLOCK * _log_uniform(rng, 1, 56), n=BLOCK * _log_uniform(rng, 1, 56), bits=rng.choice([1, 2, 3, 3, 4, 4, 5, 6, 8]),
                        table=rng.random() < 0.6)
        else:
            gated = op != "linear" and rng.random() < 0.4
            # Half of the widths are multiples of 8 as models have them, half are any number.
            step = rng.choice([1, 8])
            case.update(k=step * _log_uniform(rng, max(1, 32 // step), 7168 // step), gated=gated,
                        n=(2 if gated else 1) * step * _log_uniform(rng, max(1, 32 // step), (4096 if gated else 8192) // step),
                        act=rng.choice(["silu", "gelu", "relu"]) if gated else rng.choice([None, "silu", "gelu", "relu"]),
                        bias=rng.random() < 0.4, residual=op != "expert_linear_grad" and rng.random() < 0.4,
                        layout=rng.choice(["exl", "hf"]), spare=0 if op == "linear" else rng.choice([0, 0, 7]))
        if _cost(case) <= most and _weights(case) <= 6e8:
            return case


def _weights(case):
    return case["experts"] * case["k"] * (case["k"] if case["op"] == "hessians" else case["n"])


def _counts(case):
    """Rows of each expert: shares u^skew of the rows, every expert alike for skew 0."""
    rng, e = random.Random(case["split"]), case["experts"]
    share = [(rng.random() + 1e-3) ** (3.0 * case["skew"]) for _ in range(e)]
    total, edge, acc = sum(share), [0], 0.0
    for s in share:
        acc += s
        edge.append(min(case["rows"], int(round(case["rows"] * acc / total))))
    edge[-1] = case["rows"]
    return [b - a for a, b in zip(edge, edge[1:])]


def work(case):
    es, rows, k = torch.finfo(DTYPES[case["dtype"]]).bits // 8, case["rows"], case["k"]
    busy = sum(c > 0 for c in _counts(case))
    e = case["experts"]
    if case["op"] == "hessians":
        # Each picked row once, the matrices written whole; the products of one triangle.
        return {"bytes": min(rows, case["tokens"]) * k * es + 8 * rows + (4 * rows if case["weighted"] else 0) + 4 * e * k * k + 8 * e,
                "flops": rows * k * (k + 1)}
    n = case["n"]
    if case["op"] == "trellis_linear":
        return {"bytes": busy * (k * n * case["bits"] // 8 + 2 * (k + n)) + es * rows * (k + n), "flops": 2 * rows * k * n}
    n_out = n // 2 if case["gated"] else n
    if case["op"] == "expert_linear_grad":
        products = 3 if case["act"] else 2  # the pre-activation is not kept by the forward pass
        return {"bytes": es * (busy * k * n + e * k * n + 2 * rows * k + rows * n_out + (2 * e * n if case["bias"] else 0)),
                "flops": 2 * products * rows * k * n}
    extra = rows * n_out if case["residual"] else 0
    return {"bytes": es * (busy * (k * n + (n if case["bias"] else 0)) + rows * k + rows * n_out + extra), "flops": 2 * rows * k * n}


# ------------------------------------------------------------------ inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, rows, k = DTYPES[case["dtype"]], case["rows"], case["k"]
    randn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    counts = _counts(case)
    edges = [0]
    for c in counts:
        edges.append(edges[-1] + c)
    s = dict(case=case, offsets=torch.tensor(edges, device="cuda"), most=max(counts), groups=[slice(a, b) for a, b in zip(edges, edges[1:])],
             expert=torch.repeat_interleave(torch.arange(case["experts"], device="cuda"), torch.tensor(counts, device="cuda")),
             place=torch.cat([torch.arange(c) for c in counts]).cuda())
    if case["op"] == "hessians":
        # Activations with channel scales that differ by a log-normal factor; tokens may be picked more than once.
        s["x"] = (randn(case["tokens"], k) * torch.exp(randn(k))).to(dt)
        s["index"] = torch.randint(case["tokens"], (rows,), generator=g, device="cuda")
        s["weights"] = torch.rand(rows, generator=g, device="cuda") + 0.1 if case["weighted"] else None
        return s
    n, e = case["n"], case["experts"]
    if case["op"] == "trellis_linear":
        s["x"] = randn(rows, k).to(dt)
        s["trellis"] = torch.randint(-(1 << 15), 1 << 15, (e, k // 16, n // 16, 16 * case["bits"]), generator=g, device="cuda", dtype=torch.int16)
        s["suh"] = (torch.sign(randn(e, k)) * (0.5 + torch.rand((e, k), generator=g, device="cuda")) * k ** -0.5).half()
        s["svh"] = (torch.sign(randn(e, n)) * (0.5 + torch.rand((e, n), generator=g, device="cuda"))).half()
        s["table"] = None
        if case["table"]:
            # E4M3 bytes by state: normal quantiles, dealt to the states at random.
            q = 1.5 * torch.special.ndtri((torch.arange(STATES, device="cuda", dtype=torch.float64) + 0.5) / STATES)
            s["table"] = q[torch.randperm(STATES, generator=g, device="cuda")].float().to(torch.float8_e4m3fn).view(torch.uint8)
        return s
    total = rows + case["spare"]
    n_out = n // 2 if case["gated"] else n
    s["x"] = randn(total, k).to(dt)
    w = torch.empty((e, n, k) if case["layout"] == "hf" else (e, k, n), dtype=dt, device="cuda").normal_(0.0, k ** -0.5, generator=g)
    s["w"] = w.transpose(1, 2) if case["layout"] == "hf" else w  # [e, k, n] either way
    s["bias"] = randn(e, n).to(dt) if case["bias"] else None
    s["residual"] = randn(total, n_out).to(dt) if case["residual"] else None
    if case["op"] == "expert_linear_grad":
        s["dy"] = randn(total, n_out).to(dt)
    return s


# ------------------------------------------------------------------ plain forms, 32 bits


def _padded(s, t):
    """Rows sorted by expert -> [experts, most, width], zeros behind each expert's rows."""
    out = torch.zeros((s["case"]["experts"], s["most"], t.shape[1]), device=t.device)
    out[s["expert"], s["place"]] = t
    return out


def _fits(s):
    """Whether one batched product over padded rows costs less than twice the ragged ones."""
    return s["case"]["experts"] * s["most"] <= 2 * s["case"]["rows"]


def _products(s, x, w):
    """x[rows of e] @ w[e] for every expert."""
    if _fits(s):
        return torch.bmm(_padded(s, x), w)[s["expert"], s["place"]]
    return torch.cat([x[r] @ w[e] for e, r in enumerate(s["groups"])])


def _sums(s, x, y):
    """x[rows of e].T @ y[rows of e] for every expert."""
    if _fits(s):
        return torch.bmm(_padded(s, x).transpose(1, 2), _padded(s, y))
    return torch.stack([x[r].T @ y[r] for r in s["groups"]])


def _whole(s, t):
    """The rows of t with zeros behind the last expert's."""
    return torch.cat((t, torch.zeros((s["x"].shape[0] - t.shape[0], t.shape[1]), device=t.device)))


def _activate(z, name):
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return torch.clamp_min(z, 0) if name == "relu" else z


def _slope(z, name):
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * math.sqrt(0.5 / math.pi)
    return (z > 0).to(z.dtype) if name == "relu" else torch.ones_like(z)


def _pre(s):
    z = _products(s, s["x"][: s["case"]["rows"]].float(), s["w"].float())
    return z if s["bias"] is None else z + s["bias"].float()[s["expert"]]


def _plain_linear(s):
    c, z = s["case"], _pre(s)
    if c["gated"]:
        gate, up = z.chunk(2, dim=1)
        z = _activate(gate, c["act"]) * up
    else:
        z = _activate(z, c["act"])
    if s["residual"] is not None:
        z = z + s["residual"][: c["rows"]].float()
    return _whole(s, z).to(s["x"].dtype)


def _plain_grad(s):
    c, dt = s["case"], s["x"].dtype
    x, w, dz = s["x"][: c["rows"]].float(), s["w"].float(), s["dy"][: c["rows"]].float()
    if c["gated"]:
        gate, up = _pre(s).chunk(2, dim=1)
        dz = torch.cat((dz * up * _slope(gate, c["act"]), dz * _activate(gate, c["act"])), dim=1)
    elif c["act"]:
        dz = dz * _slope(_pre(s), c["act"])
    dx = _whole(s, _products(s, dz, w.transpose(1, 2))).to(dt)
    dw = _sums(s, x, dz).to(dt)
    if not c["bias"]:
        return dx, dw
    return dx, dw, torch.zeros((c["experts"], c["n"]), device=dz.device).index_add_(0, s["expert"], dz).to(dt)


def _plain_hessians(s):
    x = s["x"][s["index"]].float()
    w = torch.ones(s["case"]["rows"], device=x.device) if s["weights"] is None else s["weights"]
    den = torch.zeros(s["case"]["experts"], dtype=torch.float64, device=x.device).index_add_(0, s["expert"], w.double())
    return _sums(s, x, x * w[:, None]), den


def _hadamard(dtype):
    i = torch.arange(BLOCK, device="cuda")
    both, ones = i[:, None] & i[None, :], 0
    for b in range(7):
        ones = ones + ((both >> b) & 1)
    return (1 - 2 * (ones & 1)).to(dtype) * BLOCK ** -0.5


def _blocks(t, h):
    return (t.unflatten(-1, (-1, BLOCK)) @ h).flatten(-2)


def _states(trellis, bits):
    """Packed words (adjacent ones swapped, MSB first) -> the 16-bit window that ends with each of the 256 symbols."""
    words = trellis.unflatten(-1, (-1, 2)).flip(-1).flatten(-2).int() & 0xFFFF
    first = (torch.arange(1, 257, device=words.device) * bits - 16) % (256 * bits)
    word, bit = first >> 4, first & 15
    pair = (words[..., word] << 16) | words[..., (word + 1) % (16 * bits)]
    return (pair >> (16 - bit)) & 0xFFFF


def _labels(table):
    """fp32 value of every state: E4M3 bytes, or the procedural sum of two binary16 halves of a product."""
    if table is not None:
        return table.view(torch.float8_e4m3fn).float()
    y = ((torch.arange(STATES, device="cuda") * MCG_MULTIPLIER) & 0x8FFF8FFF) ^ 0x3B603B60
    half = lambda v: (((v & 0xFFFF) ^ 0x8000) - 0x8000).to(torch.int16).view(torch.float16)  # noqa: E731
    return (half(y) + half(y >> 16)).float()


def _tile_order():
    """Row-major place in a 16 x 16 tile of each trellis position."""
    j = torch.arange(256, device="cuda")
    m, t = j >> 3, j & 7
    return (2 * (m % 4) + (t & 1) + 8 * ((t >> 1) & 1)) * 16 + (m >> 2) + 8 * (t >> 2)


def _plain_trellis(s):
    c, h = s["case"], _hadamard(torch.float32)
    q = _labels(s["table"])[_states(s["trellis"], c["bits"])][..., torch.argsort(_tile_order())]
    q = q.unflatten(-1, (16, 16)).transpose(2, 3).reshape(c["experts"], c["k"], c["n"])
    y = _products(s, _blocks(s["x"].float() * s["suh"].float()[s["expert"]], h), q)
    return (_blocks(y, h) * s["svh"].float()[s["expert"]]).to(s["x"].dtype)


def run(state):
    s, op = state, state["case"]["op"]
    c = s["case"]
    if own:
        from kquant_b200 import capture, experts
        if op == "linear":
            return experts.linear(s["x"], s["w"][0], bias=None if s["bias"] is None else s["bias"][0], activation=c["act"], residual=s["residual"])
        if op == "expert_linear":
            return experts.expert_linear(s["x"], s["w"], s["offsets"], bias=s["bias"], activation=c["act"], gated=c["gated"], residual=s["residual"])
        if op == "expert_linear_grad":
            dx, dw, db = experts.expert_linear_grad(s["dy"], s["x"], s["w"], s["offsets"], bias=s["bias"], activation=c["act"], gated=c["gated"])
            return (dx, dw) if db is None else (dx, dw, db)
        if op == "hessians":
            return capture.accumulate_expert_hessians(s["x"], s["offsets"], index=s["index"], weights=s["weights"])
        return experts.trellis_linear(s["x"], s["trellis"], s["suh"], s["svh"], s["offsets"], codebook=s["table"])
    if op in ("linear", "expert_linear"):
        return _plain_linear(s)
    if op == "expert_linear_grad":
        return _plain_grad(s)
    return _plain_hessians(s) if op == "hessians" else _plain_trellis(s)


# ------------------------------------------------------------------ the definitions, 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    groups = list(enumerate(s["groups"]))
    x = s["x"].double()
    if case["op"] == "hessians":
        x = x[s["index"]]
        w = torch.ones(case["rows"], dtype=torch.float64, device="cuda") if s["weights"] is None else s["weights"].double()
        return torch.stack([(x[r] * w[r, None]).T @ x[r] for _, r in groups]), torch.stack([w[r].sum() for _, r in groups])
    if case["op"] == "trellis_linear":
        return _exact_trellis(case, s, x, groups)
    grad = case["op"] == "expert_linear_grad"
    act = {None: lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[case["act"]]
    n_out = case["n"] // 2 if case["gated"] else case["n"]
    y = torch.zeros((x.shape[0], n_out), dtype=torch.float64, device="cuda")
    dx, dw = (torch.zeros_like(x), torch.zeros(s["w"].shape, dtype=torch.float64, device="cuda")) if grad else (None, None)
    db = torch.zeros((case["experts"], case["n"]), dtype=torch.float64, device="cuda")
    for e, r in groups:
        with torch.enable_grad() if grad else torch.no_grad():
            leaf = [x[r].clone(), s["w"][e].double(), (s["bias"][e].double() if case["bias"] else torch.zeros(case["n"], dtype=torch.float64, device="cuda"))]
            if grad:
                leaf = [t.requires_grad_() for t in leaf]
            z = leaf[0] @ leaf[1] + leaf[2]
            z = act(z[:, :n_out]) * z[:, n_out:] if case["gated"] else act(z)
            if grad:
                dx[r], dw[e], db[e] = torch.autograd.grad(z, leaf, s["dy"][r].double())
            else:
                y[r] = z if s["residual"] is None else z + s["residual"][r].double()
    if grad:
        return (dx, dw, db) if case["bias"] else (dx, dw)
    return y


def _exact_trellis(case, s, x, groups):
    bits, k, n = case["bits"], case["k"], case["n"]
    had = torch.ones((1, 1), dtype=torch.float64, device="cuda")
    while had.shape[0] < BLOCK:
        had = torch.cat((torch.cat((had, had), 1), torch.cat((had, -had), 1)), 0)
    had = had / math.sqrt(BLOCK)
    left, right = torch.block_diag(*[had] * (k // BLOCK)), torch.block_diag(*[had] * (n // BLOCK))
    if case["table"]:
        b = s["table"].long()
        expo, frac = (b >> 3) & 15, (b & 7).double()
        value = torch.where(expo > 0, (8 + frac) * torch.pow(2.0, (expo - 10).double()), frac * 2.0 ** -9) * (1 - 2 * (b >> 7)).double()
    else:
        y = ((torch.arange(STATES, device="cuda") * MCG_MULTIPLIER) % (1 << 32) & 0x8FFF8FFF) ^ 0x3B603B60
        parts = []
        for v in (y & 0xFFFF, y >> 16):
            expo, frac = (v >> 10) & 31, (v & 1023).double()
            parts.append(torch.where(expo > 0, (1024 + frac) * torch.pow(2.0, (expo - 25).double()), frac * 2.0 ** -24) * (1 - 2 * (v >> 15)).double())
        value = (parts[0] + parts[1]).half().double()  # the codebook rounds the sum to binary16
    out = torch.zeros((case["rows"], n), dtype=torch.float64, device="cuda")
    for e, r in groups:
        if r.start == r.stop:
            continue
        words = s["trellis"][e].long() & 0xFFFF
        words = torch.stack((words[..., 1::2], words[..., 0::2]), -1).flatten(-2)
        stream = torch.stack([(words >> (15 - b)) & 1 for b in range(16)], -1).flatten(-2)  # bits in stream order
        edge = sum(stream[..., b::bits] << (bits - 1 - b) for b in range(bits))
        state = torch.zeros_like(edge)
        for lag in range(-(-16 // bits)):
            state |= torch.roll(edge, lag, -1) << (lag * bits)
        weight = torch.empty((k // 16, 16, n // 16, 16), dtype=torch.float64, device="cuda")
        for lane in range(32):
            for slot in range(8):
                row, col = 2 * (lane % 4) + slot % 2 + 8 * (slot // 2 % 2), lane // 4 + 8 * (slot // 4)
                weight[:, row, :, col] = value[state[..., 8 * lane + slot] & 0xFFFF]
        full = s["suh"][e].double()[:, None] * (left @ weight.reshape(k, n)) @ right * s["svh"][e].double()
        out[r] = x[r] @ full
    return out

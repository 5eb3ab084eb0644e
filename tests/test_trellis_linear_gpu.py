"""kquant_b200.experts.trellis_linear against the 64-bit product with the decoded, reconstructed weights."""
import numpy as np
import pytest
import torch

from kquant_b200 import _native, codebooks, experts
from tests.expert_cases import HALF_STEP, TINY, check, groups, offsets_of, sum_slack

pytestmark = pytest.mark.gpu

RATES = [1, 2, 3, 4, 5, 6, 7, 8]


def had64(dev):
    h = torch.ones((1, 1), dtype=torch.float64, device=dev)
    while h.shape[0] < 128:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)), 0)
    return h / 128 ** 0.5


def labels64(codebook, dev):
    if codebook is None:
        return _native.build_labels(_native.KQ_CB_MCG, None, dev).view(torch.float16).double()
    return codebook.view(torch.float8_e4m3fn if codebook.dtype == torch.uint8 else torch.float16).double()


def decode64(trellis, codebook):
    """What [experts, k, n]: the framework's own unpack, labels by state, tensor-core order undone."""
    from kquant_b200.exl3_encoder_backend import tensor_core_perm_i
    K = trellis.shape[-1] // 16
    states = _native.unpack_trellis_states(trellis, K).long() & 0xFFFF
    v = labels64(codebook, trellis.device)[states][..., tensor_core_perm_i(trellis.device)]
    E, kt, nt, _ = v.shape
    return v.reshape(E, kt, nt, 16, 16).transpose(2, 3).reshape(E, 16 * kt, 16 * nt)


def expect(x, trellis, suh, svh, offsets, codebook):
    h, What = had64(x.device), decode64(trellis, codebook)
    E, k, n = What.shape
    y = torch.zeros((x.shape[0], n), dtype=torch.float64, device=x.device)
    b = torch.zeros_like(y)
    for e, r in enumerate(groups(offsets)):
        v = x[r].double() * suh[e].double()
        xr = (v.unflatten(1, (-1, 128)) @ h).flatten(1)
        # Half a binary16 step of x'; before it seven fp32 butterfly stages, 7 sqrt(128) 2^-24 of the largest value.
        big = v.abs().amax(1, keepdim=True) if v.numel() else v.new_zeros((v.shape[0], 1))
        ex = xr.abs() * 2.0 ** -11 + big * 2.0 ** -17
        z = xr @ What[e]
        ez = ex @ What[e].abs() + (xr.abs() @ What[e].abs()) * sum_slack(k)
        s = svh[e].double()
        y[r] = (z.unflatten(1, (-1, 128)) @ h).flatten(1) * s
        b[r] = ((ez + z.abs() * 2.0 ** -21).unflatten(1, (-1, 128)) @ h.abs()).flatten(1) * s.abs()
    return y, b + (y.abs() + b) * HALF_STEP[x.dtype] + TINY[x.dtype]


def make(counts, k, n, K, dtype, dev, seed=0, spare=0, first=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    E, rows = len(counts), sum(counts) + spare + first
    x = torch.randn((rows, k), generator=g, device=dev).to(dtype)
    t = torch.randint(-32768, 32768, (E, k // 16, n // 16, 16 * K), generator=g, device=dev, dtype=torch.int16)
    sign = lambda m: torch.sign(torch.randn((E, m), generator=g, device=dev))  # noqa: E731
    suh = (sign(k) * (0.5 + torch.rand((E, k), generator=g, device=dev))).half()
    svh = (sign(n) * (0.5 + torch.rand((E, n), generator=g, device=dev))).half()
    return x, t, suh, svh, offsets_of(counts, dev, first)


def tables(dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    q = 1.5 * torch.randn(65536, generator=g, device=dev)
    return {"mcg": None, "e4m3": q.to(torch.float8_e4m3fn).view(torch.uint8), "labels": q.half().view(torch.int16)}


def near(got, want):
    """Two independent roundings, of x' and of y, whose rms is at most 0.41 of their half steps."""
    rel = float((got.double() - want).norm() / want.norm().clamp_min(1e-300))
    assert rel <= 0.6 * (HALF_STEP[got.dtype] ** 2 + 2.0 ** -22) ** 0.5, rel


@pytest.mark.parametrize("K", RATES)
@pytest.mark.parametrize("book", ["mcg", "e4m3", "labels"])
@pytest.mark.parametrize("counts,k,n", [([1], 128, 128), ([1, 0, 2], 256, 384), ([40, 3, 150], 384, 256), ([16, 17], 128, 1152)])
def test_products(cuda_device, K, book, counts, k, n):
    for dtype in (torch.bfloat16, torch.float16):
        x, t, suh, svh, off = make(counts, k, n, K, dtype, cuda_device, seed=K)
        cb = tables(cuda_device)[book]
        y = experts.trellis_linear(x, t, suh, svh, off, codebook=cb)
        want, bound = expect(x, t, suh, svh, off, cb)
        check(y, want, bound)
        near(y, want)
    _native.check_wait_errors(cuda_device)


@pytest.mark.parametrize("rows", [1, 2, 7, 15, 16, 17, 31, 33, 64, 65, 127, 129, 300])
def test_every_row_count(cuda_device, rows):
    x, t, suh, svh, off = make([rows, 0, 1], 512, 256, 3, torch.bfloat16, cuda_device, seed=rows)
    cb = tables(cuda_device)["e4m3"]
    y = experts.trellis_linear(x, t, suh, svh, off, codebook=cb)
    check(y, *expect(x, t, suh, svh, off, cb))
    _native.check_wait_errors(cuda_device)


def test_matches_the_encoder(cuda_device):
    """A matrix encoded by the framework: the product from its payload is the product with its reconstruction."""
    from kquant_b200 import exl3_encoder_backend as backend
    from kquant_b200.ldlq import make_shared_h
    g = torch.Generator(device=cuda_device).manual_seed(3)
    W = torch.randn((256, 128), generator=g, device=cuda_device) * 0.02
    X = torch.randn((512, 256), generator=g, device=cuda_device)
    for K, lut in ((3, codebooks.sqg_xor_cheb_t12_bytes(3)), (5, None)):
        args = {"K": K, "seed": 7, "sv_seed": 11, "sigma_reg": 0.025, "devices": [str(cuda_device)], "apply_out_scales": False,
                "tailbite_context": 128, **({"mcg": True} if lut is None else {"sqg_e4m3_luts_by_bits": {K: lut}})}
        wq, proxy, out = backend.quantize_qsrt(W.clone(), make_shared_h(256, cuda_device, X.T @ X / 512), args, True)
        x = torch.randn((9, 256), generator=g, device=cuda_device).half()
        book = None if lut is None else lut.to(cuda_device)
        y = experts.trellis_linear(x, out["trellis"], out["suh"], out["svh"], codebook=book)
        want, bound = expect(x, out["trellis"][None], out["suh"][None], out["svh"][None], offsets_of([9], cuda_device), book)
        check(y, want, bound)
        # The reconstruction has the scales in fp32, the payload in binary16 (half a step each), and is itself good to
        # 2e-6 of its largest weight.
        full = x.double() @ wq.double()
        slack = (x.double().abs() @ wq.double().abs()) * 1.01 * 2.0 ** -10 + 4e-6 * wq.abs().max() * x.double().abs().sum(1, keepdim=True)
        check(want, full, slack)


def test_scales_of_rows(cuda_device):
    """Rows of very different size, an all-zero row and one with a large outlier keep their relative accuracy."""
    x, t, suh, svh, off = make([8, 30], 256, 256, 4, torch.bfloat16, cuda_device, seed=6)
    x[0], x[1], x[2], x[3] = 0, x[1] * 2.0 ** -60, x[2] * 2.0 ** 60, x[3] * 2.0 ** 20
    x[4, 17], x[9, 200] = 3e4, -2e5
    x[5] = torch.sign(x[5]) * 1e38                     # the transform of these would leave the fp32 range
    suh[0] *= 0.5
    svh[0] *= 2.0 ** -10
    y = experts.trellis_linear(x, t, suh, svh, off)
    want, bound = expect(x, t, suh, svh, off, None)
    check(y, want, bound)
    assert not y[0].any()


def test_rows_of_no_expert_views_and_nan(cuda_device):
    x, t, suh, svh, off = make([3, 40], 256, 128, 3, torch.float16, cuda_device, seed=7, spare=3, first=2)
    x[:2], x[45:] = float("nan"), float("nan")
    want, bound = expect(x, t, suh, svh, off, None)
    y = experts.trellis_linear(x, t, suh, svh, off)
    assert not y[:2].any() and not y[45:].any()
    check(y[2:45], want[2:45], bound[2:45])
    wide = torch.full((48, 133), 5.0, dtype=torch.float16, device=cuda_device)
    xs = torch.zeros((48, 259), dtype=torch.float16, device=cuda_device)
    xs[:, 1:257] = x
    assert torch.equal(experts.trellis_linear(xs[:, 1:257], t, suh, svh, off, out=wide[:, 3:131])[2:45], y[2:45])
    assert (wide[:2] == 5).all() and (wide[45:] == 5).all() and (wide[:, :3] == 5).all() and (wide[:, 131:] == 5).all()
    x[2] = float("inf")
    z = experts.trellis_linear(x, t, suh, svh, off)
    assert torch.equal(z[3:45], y[3:45]) and not z[2].isfinite().all()


def test_replay_and_streams(cuda_device):
    for counts in ([5, 1, 3], [100, 2, 60]):
        x, t, suh, svh, off = make(counts, 256, 384, 3, torch.bfloat16, cuda_device, seed=8)
        rows = x.shape[0]
        run = lambda: experts.trellis_linear(x, t, suh, svh, off)  # noqa: E731
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run()
        for new in (counts, [0, rows, 0], [rows - 1, 0, 1], [1, 1, 1]):
            off.copy_(offsets_of(new, cuda_device))
            x.copy_(torch.randn_like(x))
            graph.replay()
            assert torch.equal(got, run())
        want = run()
        streams = [torch.cuda.Stream(cuda_device) for _ in range(2)]
        torch.cuda.synchronize()
        outs = []
        for i in range(6):
            with torch.cuda.stream(streams[i % 2]):
                outs.append(run())
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


def test_no_rows(cuda_device):
    x, t, suh, svh, off = make([0, 0], 128, 128, 3, torch.bfloat16, cuda_device)
    assert experts.trellis_linear(x, t, suh, svh, off).shape == (0, 128)
    x = torch.randn((4, 128), device=cuda_device).bfloat16()
    assert not experts.trellis_linear(x, t, suh, svh, off).any()


@pytest.mark.parametrize("K", RATES)
@pytest.mark.parametrize("book", ["mcg", "e4m3"])
@pytest.mark.parametrize("counts,k,n", [([300, 0, 1, 70, 129, 256], 256, 1920), ([9, 17, 1] * 11, 384, 256), ([12], 128, 8320)])
def test_middling_rows(cuda_device, K, book, counts, k, n):
    """More than a few rows an expert and enough columns: decoded into the tensor core's tiles."""
    for dtype in (torch.bfloat16, torch.float16):
        x, t, suh, svh, off = make(counts, k, n, K, dtype, cuda_device, seed=10 + K)
        cb = tables(cuda_device)[book]
        y = experts.trellis_linear(x, t, suh, svh, off, codebook=cb)
        want, bound = expect(x, t, suh, svh, off, cb)
        check(y, want, bound)
        near(y, want)
    _native.check_wait_errors(cuda_device)


def test_middling_rows_views_replay_and_nan(cuda_device):
    """Rows of no expert kept or zeroed, odd strides and bases, NaN confined to its row, new offsets at replay."""
    counts, k, n = [40, 0, 33, 260, 5], 384, 1792
    x, t, suh, svh, off = make(counts, k, n, 4, torch.float16, cuda_device, seed=3, spare=5, first=3)
    wide = torch.full((x.shape[0], k + 7), float("nan"), dtype=x.dtype, device=cuda_device)
    wide[:, 3:3 + k].copy_(x)
    x = wide[:, 3:3 + k]
    x[off[1] - 2, 5] = float("nan")
    x[-2, 7] = float("inf")                                # behind the last expert
    buf = torch.full((x.shape[0], n + 9), 7.0, dtype=x.dtype, device=cuda_device)
    out = buf[:, 1:1 + n]
    assert experts.trellis_linear(x, t, suh, svh, off, out=out) is out
    fresh = experts.trellis_linear(x, t, suh, svh, off)
    a, b = int(off[0]), int(off[-1])
    keep = torch.ones(x.shape[0], dtype=torch.bool, device=cuda_device)
    keep[off[1] - 2] = False
    assert torch.isnan(fresh[~keep]).all()
    clean = x.clone()
    clean[~keep] = 0
    want, bound = expect(clean, t, suh, svh, off, None)
    want[a:b][~keep[a:b]] = float("nan")
    inside = keep.clone()
    inside[:a], inside[b:] = False, False
    check(fresh[inside], want[inside], bound[inside])
    assert torch.equal(out[inside], fresh[inside])
    assert not fresh[:a].any() and not fresh[b:].any()
    assert (buf[:, 0] == 7).all() and (buf[:, 1 + n:] == 7).all() and (out[:a] == 7).all() and (out[b:] == 7).all()

    x = torch.randn((64, k), device=cuda_device).half()
    off = offsets_of([20, 14, 10, 12, 8], cuda_device)
    run = lambda: experts.trellis_linear(x, t, suh, svh, off)  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for new in ([64, 0, 0, 0, 0], [0, 0, 0, 0, 0], [1, 1, 1, 1, 1], [0, 30, 0, 34, 0]):
        off.copy_(offsets_of(new, cuda_device))
        graph.replay()
        assert torch.equal(got, run())
        want, bound = expect(x, t, suh, svh, off, None)
        check(got[:sum(new)], want[:sum(new)], bound[:sum(new)])
    _native.check_wait_errors(cuda_device)


def test_every_way_gives_the_same_sums(cuda_device):
    """Row counts on both sides of each choice of kernel."""
    for book, counts, n in (("mcg", [8, 8], 4224), ("mcg", [9, 9], 4224), ("e4m3", [192, 192], 4224), ("e4m3", [193, 193], 4224),
                            ("mcg", [96], 8192), ("mcg", [97], 8192), ("labels", [40, 40], 4224), ("labels", [41, 41], 4224)):
        x, t, suh, svh, off = make(counts, 256, n, 3, torch.bfloat16, cuda_device, seed=5)
        cb = tables(cuda_device)[book]
        y = experts.trellis_linear(x, t, suh, svh, off, codebook=cb)
        check(y, *expect(x, t, suh, svh, off, cb))

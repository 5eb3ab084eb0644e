"""The expert-layer operators together: calibrate a layer's experts, encode them, run what was encoded."""
import pytest
import torch

from kquant_b200 import _native, codebooks, experts
from kquant_b200 import exl3_encoder_backend as backend
from kquant_b200.capture import accumulate_expert_hessians, expert_layer_hessians
from kquant_b200.ldlq import make_shared_h
from tests.expert_cases import check, forward64, groups, offsets_of
from tests.test_trellis_linear_gpu import expect

pytestmark = pytest.mark.gpu


def layer(dev, E=3, k=256, inter=128, tokens=96, counts=(70, 0, 33), seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    x = (rnd(tokens, k) * torch.exp(0.5 * rnd(k))).bfloat16()
    w13, w2 = (rnd(E, k, 2 * inter) * k ** -0.5).bfloat16(), (rnd(E, inter, k) * inter ** -0.5).bfloat16()
    index = torch.randint(tokens, (sum(counts),), generator=g, device=dev)
    return x, w13, w2, index, offsets_of(counts, dev), torch.rand(sum(counts), generator=g, device=dev) + 0.1


@pytest.mark.parametrize("weighted", [False, True])
def test_layer_hessians(cuda_device, weighted):
    x, w13, w2, index, off, w = layer(cuda_device)
    index[3], index[80] = -7, 1 << 40                   # slots that count for nothing
    w = w if weighted else None
    H13, H2, den = expert_layer_hessians(x, index, off, w13, weights=w)
    ok = (index >= 0) & (index < x.shape[0])
    h = experts.expert_linear(x[index.clamp(0, 95)], w13, off, activation="silu", gated=True)
    for e, r in enumerate(groups(off)):
        keep = ok[r]
        weight = (torch.ones(keep.numel(), device=cuda_device) if w is None else w[r])[keep].double()
        for H, rows in ((H13, x[index.clamp(0, 95)][r][keep].double()), (H2, h[r][keep].double())):
            want = (rows * weight[:, None]).T @ rows
            bound = (rows * weight[:, None]).abs().T @ rows.abs() * 2.0 ** -18 + 1e-30
            check(H[e], want, bound)
        assert float(den[e]) == pytest.approx(float(weight.sum()), rel=1e-14)


def test_calibrate_encode_and_run(cuda_device):
    """The encoder takes the Hessians, and the layer run from the payloads is the layer run from what they decode to."""
    x, w13, w2, index, off, _ = layer(cuda_device)
    E, k, inter = 3, 256, 128
    H13, H2, den = expert_layer_hessians(x, index, off, w13)
    lut = codebooks.sqg_xor_cheb_t12_bytes(3)
    args = lambda: {"K": 3, "seed": 7, "sv_seed": 11, "sigma_reg": 0.025, "devices": [str(cuda_device)],  # noqa: E731
                    "apply_out_scales": False, "tailbite_context": 128, "sqg_e4m3_luts_by_bits": {3: lut}}
    parts, full = {"w13": [], "w2": []}, {"w13": [], "w2": []}
    for e in range(E):
        for name, W, H in (("w13", w13[e], H13[e]), ("w2", w2[e], H2[e])):
            h = H / max(float(den[e]), 1.0) if float(den[e]) else torch.eye(W.shape[0], device=cuda_device)
            wq, proxy, out = backend.quantize_qsrt(W.float().clone(), make_shared_h(W.shape[0], cuda_device, h), args(), True)
            assert 0 <= proxy < 1
            parts[name].append(out)
            full[name].append(wq)
    stack = lambda name, key: torch.stack([p[key] for p in parts[name]])  # noqa: E731
    book = lut.to(cuda_device)
    rows = x[index]
    z = experts.trellis_linear(rows, stack("w13", "trellis"), stack("w13", "suh"), stack("w13", "svh"), off, codebook=book)
    gate, up = z.float().chunk(2, 1)
    hidden = (torch.nn.functional.silu(gate) * up).bfloat16()
    y = experts.trellis_linear(hidden, stack("w2", "trellis"), stack("w2", "suh"), stack("w2", "svh"), off, codebook=book)
    # The dense operators on the reconstructed weights in bf16: both sides round inputs, z, hidden and y to bf16 (half a
    # step 2^-8 each, the weights once more on the dense side); over sums of independent errors their rms stays below.
    dense13, dense2 = torch.stack(full["w13"]).bfloat16(), torch.stack(full["w2"]).bfloat16()
    h2 = experts.expert_linear(rows, dense13, off, activation="silu", gated=True)
    y2 = experts.expert_linear(h2, dense2, off)
    assert float((hidden.float() - h2.float()).norm() / h2.float().norm()) < 4 * 2.0 ** -8
    assert float((y.float() - y2.float()).norm() / y2.float().norm()) < 6 * 2.0 ** -8
    # And the dense side is what 64 bits make of it.
    for e, r in enumerate(groups(off)):
        if r.stop > r.start:
            check(y2[r], *forward64(h2[r], dense2[e], None, None, False, None))
    # A training step on what the layer computed: gradients come back for every expert.
    dh, dw2, _ = experts.expert_linear_grad(torch.ones_like(y2), h2, dense2, off)
    dx, dw13, _ = experts.expert_linear_grad(dh, rows, dense13, off, activation="silu", gated=True)
    assert dx.shape == rows.shape and dw13.shape == dense13.shape and not dw13[1].any() and not dw2[1].any()
    assert dx.isfinite().all() and dw13.isfinite().all() and dw2.isfinite().all()
    _native.check_wait_errors(cuda_device)


def test_layer_in_one_graph(cuda_device):
    """The whole calibration captured once and replayed on new tokens and routing."""
    x, w13, w2, index, off, w = layer(cuda_device)
    run = lambda: expert_layer_hessians(x, index, off, w13, weights=w)  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for counts in ((70, 0, 33), (1, 101, 1), (0, 0, 5)):
        off.copy_(offsets_of(counts, cuda_device))
        x.copy_(torch.randn_like(x))
        index.copy_(torch.randint(96, (103,), device=cuda_device))
        graph.replay()
        for a, b in zip(got, run()):
            assert torch.equal(a, b)


def test_two_graphs_side_by_side(cuda_device):
    """Two captured calls share no workspace: replayed at once on two streams, each gives its own result."""
    made = []
    for seed in (1, 2):
        x, w13, w2, index, off, w = layer(cuda_device, seed=seed)
        x = x[:, :255].contiguous()                      # odd rows: the call needs workspace
        w13 = w13[:, :255].contiguous()
        run = lambda x=x, w13=w13, off=off, index=index: (experts.expert_linear(x[index], w13, off, activation="silu", gated=True),  # noqa: E731
                                                          *accumulate_expert_hessians(x, off, index=index))
        want = run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run()
        made.append((graph, got, want, torch.cuda.Stream(cuda_device), run))    # run keeps the graph's operands alive
    for _ in range(5):
        for graph, _, _, stream, _ in made:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, got, want, _, _ in made:
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_many_experts(cuda_device):
    """As many experts as there may be, most of them without rows."""
    g = torch.Generator(device=cuda_device).manual_seed(9)
    E = 1024
    counts = [0] * E
    for e in (0, 1, 31, 32, 511, 700, 1023):
        counts[e] = 1 + e % 5
    counts[512] = 70
    off, rows = offsets_of(counts, cuda_device), sum(counts)
    x = torch.randn((rows, 128), generator=g, device=cuda_device).half()
    w = torch.randn((E, 128, 128), generator=g, device=cuda_device).half()
    y = experts.expert_linear(x, w, off)
    dx, dw, _ = experts.expert_linear_grad(y, x, w, off)
    H, den = accumulate_expert_hessians(x, off)
    t = torch.randint(-32768, 32768, (E, 8, 8, 48), generator=g, device=cuda_device, dtype=torch.int16)
    one = torch.ones((E, 128), device=cuda_device).half()
    z = experts.trellis_linear(x, t, one, one, off)
    assert not dw[2].any() and not H[2].any() and den.sum() == rows
    for e, r in enumerate(groups(off)):
        if r.stop > r.start:
            check(y[r], *forward64(x[r], w[e], None, None, False, None), what=e)
            assert torch.equal(H[e], accumulate_expert_hessians(x[r], offsets_of([r.stop - r.start], cuda_device))[0][0])
    want, bound = expect(x, t, one, one, off, None)
    check(z, want, bound)
    _native.check_wait_errors(cuda_device)


def test_first_call_captured(cuda_device):
    """A process whose first call of each operator is a captured one."""
    import subprocess
    import sys
    code = """
import torch
from kquant_b200 import capture, experts
x, w = torch.randn(20, 64, device='cuda').bfloat16(), torch.randn(2, 64, 128, device='cuda').bfloat16()
off = torch.tensor([0, 5, 20], device='cuda')
t = torch.randint(-9, 9, (2, 8, 8, 48), device='cuda', dtype=torch.int16)
one = torch.ones(2, 128, device='cuda').half()
big = torch.randn(20, 128, device='cuda').bfloat16()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
run = lambda: (experts.expert_linear(x, w, off, activation='silu', gated=True), *experts.expert_linear_grad(big, x, w, off)[:2],
               *capture.accumulate_expert_hessians(x, off), experts.trellis_linear(big, t, one, one, off))
with torch.cuda.graph(graph):
    got = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, run()))
print('captured first')
"""
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert "captured first" in out.stdout, out.stderr[-2000:]


def test_threads(cuda_device):
    """Calls from several host threads, each on a stream of its own."""
    import threading
    x, w13, w2, index, off, w = layer(cuda_device)
    want = expert_layer_hessians(x, index, off, w13, weights=w)
    torch.cuda.synchronize()
    got, streams = [None] * 4, [torch.cuda.Stream(cuda_device) for _ in range(4)]

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(5):
                got[i] = expert_layer_hessians(x, index, off, w13, weights=w)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for g in got:
        for a, b in zip(g, want):
            assert torch.equal(a, b)


def test_operands_of_more_than_two_to_the_32_elements(cuda_device):
    """The last rows of a long x, of long results and of a long list of slots are where they should be."""
    free = torch.cuda.mem_get_info(cuda_device)[0]
    if free < 60 << 30:
        pytest.skip("needs 60 GB free")
    g = torch.Generator(device=cuda_device).manual_seed(4)
    rows, k = (1 << 22) + 77, 1024
    x = torch.zeros((rows, k), dtype=torch.bfloat16, device=cuda_device)
    x[:40].copy_(torch.randn((40, k), generator=g, device=cuda_device))
    x[-300:].copy_(torch.randn((300, k), generator=g, device=cuda_device))
    w = torch.randn((2, k, 128), generator=g, device=cuda_device).bfloat16()
    off = torch.tensor([0, 40, rows], device=cuda_device)
    tail, toff = x[-300:].clone(), torch.tensor([0, 0, 300], device=cuda_device)
    y = experts.expert_linear(x, w, off)
    check(y[-300:], *forward64(tail, w[1], None, None, False, None))
    check(y[:40], *forward64(x[:40], w[0], None, None, False, None))
    assert not y[40:-300].any()
    up = torch.randn((1, 128, k), generator=g, device=cuda_device).bfloat16()
    z = experts.expert_linear(y, up, None)
    check(z[-300:], *forward64(y[-300:], up[0], None, None, False, None))
    del z
    _, dw, _ = experts.expert_linear_grad(y, x, w, off, need_dx=False)
    want = experts.expert_linear_grad(y[-300:].contiguous(), tail, w, toff, need_dx=False)[1]
    assert torch.allclose(dw[1].float(), want[1].float(), rtol=2.0 ** -7, atol=1e-2)       # one bf16 step each; sums of 300
    H, den = accumulate_expert_hessians(x, off)
    want, _ = accumulate_expert_hessians(tail, toff)
    assert den.tolist() == [40.0, rows - 40.0]
    assert torch.allclose(H[1], want[1], rtol=0, atol=300 * 2.0 ** -22 * 16)
    t = torch.randint(-32768, 32768, (2, k // 16, 8, 48), generator=g, device=cuda_device, dtype=torch.int16)
    su, sv = torch.ones((2, k), device=cuda_device).half(), torch.ones((2, 128), device=cuda_device).half()
    q = experts.trellis_linear(x, t, su, sv, off)
    want, bound = expect(tail, t, su, sv, toff, None)
    check(q[-300:], want, bound)
    assert not q[40:-300].any()
    _native.check_wait_errors(cuda_device)

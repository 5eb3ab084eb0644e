"""Results that would be written over operands while kernels still read them are refused, on the host, before any launch."""
import pytest
import torch

from kquant_b200 import experts
from kquant_b200.capture import accumulate_expert_hessians
from tests.test_expert_refusals import FakeCuda, fake


def as_fake(t):
    return t.as_subclass(FakeCuda)


def trellis_args(**change):
    args = dict(x=fake(4, 128), trellis=fake(2, 8, 8, 48, dtype=torch.int16), suh=fake(2, 128, dtype=torch.float16),
                svh=fake(2, 128, dtype=torch.float16), offsets=fake(3, dtype=torch.int64))
    args.update(change)
    return args


def test_trellis_linear_refuses():
    memory = torch.zeros(1 << 17, dtype=torch.uint8)
    out = lambda at, dtype=torch.bfloat16: as_fake(memory[at: at + 1024].view(dtype).view(4, 128))  # noqa: E731
    half = lambda at: as_fake(memory[at: at + 512].view(torch.float16).view(2, 128))  # noqa: E731
    # The encoded operands and the offsets are read until the last result is written.
    for name, t in (("svh", half(1000)), ("suh", half(1000)), ("offsets", as_fake(memory[1016:1040].view(torch.int64))),
                    ("trellis", as_fake(memory[: 2 * 8 * 8 * 96].view(torch.int16).view(2, 8, 8, 48))),
                    ("codebook", as_fake(memory[: 1 << 16])), ("codebook", as_fake(memory.view(torch.int16)))):
        with pytest.raises(ValueError, match=f"out must not overlap {name}"):
            experts.trellis_linear(**trellis_args(**{name: t}), out=out(512))
    # One matrix without offsets.
    with pytest.raises(ValueError, match="out must not overlap svh"):
        experts.trellis_linear(fake(4, 128, dtype=torch.float16), fake(8, 8, 48, dtype=torch.int16), fake(128, dtype=torch.float16),
                               as_fake(memory[:256].view(torch.float16)), out=out(0, torch.float16))


def test_expert_hessians_refuse():
    memory = torch.zeros(4096, dtype=torch.uint8)
    args = dict(rows=fake(4, 8), offsets=fake(3, dtype=torch.int64), index=fake(4, dtype=torch.int64), weights=fake(4, dtype=torch.float32))
    H = as_fake(memory[:512].view(torch.float32).view(2, 8, 8))
    for name, t in (("offsets", as_fake(memory[504:528].view(torch.int64))), ("index", as_fake(memory[:32].view(torch.int64))),
                    ("weights", as_fake(memory[496:512].view(torch.float32))), ("rows", as_fake(memory[448:576].view(torch.float32).view(4, 8)))):
        with pytest.raises(ValueError, match=f"out must not overlap {name}"):
            accumulate_expert_hessians(**{**args, name: t}, out=H)
    # Rows as far apart as two matrices are still inside them.
    rows = as_fake(memory[:512].view(torch.float32).as_strided((2, 8), (64, 1), 16))
    with pytest.raises(ValueError, match="out must not overlap rows"):
        accumulate_expert_hessians(rows, fake(3, dtype=torch.int64), out=H)


def test_expert_linear_refuses_its_offsets():
    memory = torch.zeros(256, dtype=torch.uint8)
    with pytest.raises(ValueError, match="out must not overlap offsets"):
        experts.expert_linear(fake(4, 8), fake(2, 8, 6), as_fake(memory[40:64].view(torch.int64)),
                              out=as_fake(memory[:48].view(torch.bfloat16).view(4, 6)))


def test_memory_shared_without_a_common_storage():
    """Tensors that came from one buffer through another library know nothing of each other."""
    memory = torch.zeros(64, dtype=torch.bfloat16)
    x = torch.utils.dlpack.from_dlpack(torch.utils.dlpack.to_dlpack(memory[:32])).view(4, 8)
    out = torch.utils.dlpack.from_dlpack(torch.utils.dlpack.to_dlpack(memory[8:40])).view(4, 8)
    with pytest.raises(ValueError, match="out must not overlap x"):
        experts.linear(as_fake(x), fake(8, 8), out=as_fake(out))
    experts._refuse_overlap(as_fake(memory[32:].view(4, 8)), as_fake(x), "x")

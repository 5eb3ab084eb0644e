"""The bounded waits inside the tensor-core kernels."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "kquant_b200" / "csrc"


def test_limit_of_the_waits():
    """Every kernel takes its limit from one place, 2^24 polls: the trace, the Hessian and the expert-layer kernels."""
    found = {p.name: int(m) for p in sorted(CSRC.glob("*.cu*")) for m in re.findall(r"kSpinLimit\s*=\s*1u\s*<<\s*(\d+)", p.read_text())}
    assert found == {"kq_umma.cuh": 24}

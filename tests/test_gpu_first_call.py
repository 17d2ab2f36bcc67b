"""A process whose first layer call is part of a capture."""

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

FIRST_IN_A_CAPTURE = """
import sys, torch
sys.path.insert(0, {root!r})
import oztt_b200 as oz
x, w = (torch.randn(64, 128, device="cuda").bfloat16() for _ in range(2))
graph = torch.cuda.CUDAGraph()
try:
    with torch.cuda.graph(graph):
        y = oz.linear(x, w)
    graph.replay()
    torch.cuda.synchronize()
    print("captured", float((y.double() - x.double() @ w.double().t()).abs().max()) < 0.5)
except Exception as e:
    print("not captured:", e)
del graph
torch.cuda.synchronize()
print("later", float((oz.linear(x, w).double() - x.double() @ w.double().t()).abs().max()) < 0.5)
"""


def test_first_call_in_a_capture(oztt, cuda):
    """A process whose first product is captured has it captured, and its later products run."""
    r = subprocess.run([sys.executable, "-c", FIRST_IN_A_CAPTURE.format(root=str(ROOT))], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and r.stdout.split("\n")[:2] == ["captured True", "later True"], r.stdout + r.stderr

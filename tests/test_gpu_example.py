"""The training example runs, learns, and serves what it trained."""

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


def test_train_mlp(cuda):
    r = subprocess.run([sys.executable, str(ROOT / "examples" / "train_mlp.py"), "--steps", "60", "--width", "256",
                        "--tokens", "1024"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.strip().endswith("ok")

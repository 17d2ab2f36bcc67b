"""The layer calls' status where no product has run (on any machine)."""

import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def test_refusal(oztt):
    with pytest.raises(ValueError, match="device_id"):
        oztt.layer_status(-1)


def test_nothing_has_run():
    r = subprocess.run([sys.executable, "-c", f"import sys; sys.path.insert(0, {str(ROOT)!r}); import oztt_b200 as oz; "
                        "oz.layer_status(); oz.layer_status(100); assert 'torch' not in sys.modules"])
    assert r.returncode == 0

"""The package without torch: everything but the calls on torch's tensors, which say what they lack."""

import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def run(code):
    r = subprocess.run([sys.executable, "-c", f"import sys; sys.path.insert(0, {str(ROOT)!r}); sys.modules['torch'] = None\n{code}"],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_star_import():
    run("from oztt_b200 import *\nassert Context and Options and layer_status")


def test_names_that_need_torch():
    run("import oztt_b200 as oz\n"
        "for name in ('linear', 'linear_backward', 'AdamW'):\n"
        "    try:\n        getattr(oz, name)\n"
        "    except ImportError as e:\n        assert 'torch' in str(e)\n"
        "    else:\n        raise AssertionError(name)")


def test_star_import_with_torch():
    r = subprocess.run([sys.executable, "-c", f"import sys; sys.path.insert(0, {str(ROOT)!r})\nfrom oztt_b200 import *\n"
                        "assert Context and linear and linear_backward and AdamW"])
    assert r.returncode == 0

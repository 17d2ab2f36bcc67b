"""What needs no torch is built without it."""

import importlib.util

from oztt_b200 import build


def test_the_binding_is_left_out(monkeypatch):
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    ran = []
    monkeypatch.setattr(build, "_run", ran.append)
    assert build.build_torch_binding(force=True) is None and not ran


def test_the_rest_is_built(monkeypatch):
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    steps = []
    for name in ("build_library", "build_programs", "build_oracle"):
        monkeypatch.setattr(build, name, lambda *a, name=name: steps.append(name))
    build.build()
    assert steps == ["build_library", "build_programs", "build_oracle"]

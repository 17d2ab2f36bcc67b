"""Orderings that the kernels' sources have to state, since no result shows for certain that one is missing."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "oztt_b200" / "csrc"
SOURCES = sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh"))


def without_comments(path):
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", path.read_text(), flags=re.S)


def statements(text):
    """The asm statements of a source, whole."""
    for at in re.finditer(r"\basm\b(?:\s+volatile)?\s*\(", text):
        depth, end = 1, at.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[end], 0)
            end += 1
        yield text[at.start():end]


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_loads_from_tensor_memory_are_waited_for(path):
    """A load from tensor memory writes its registers until tcgen05.wait::ld: the wait names every one of them as its
    own, in the same function and behind the load, or the compiler may use one before it."""
    asm = list(statements(without_comments(path)))
    loads = [i for i, s in enumerate(asm) if "tcgen05.ld." in s]
    for i in loads:
        regs = re.findall(r'"=r"\((\w+\[\d+\])\)', asm[i])
        assert len(regs) == int(re.search(r"\.x(\d+)\.b32", asm[i]).group(1))
        wait = asm[i] if "tcgen05.wait::ld" in asm[i] else asm[i + 1]
        assert "tcgen05.wait::ld" in wait
        assert wait is asm[i] or re.findall(r'"\+r"\((\w+\[\d+\])\)', wait) == regs, asm[i][:80]
    assert len([s for s in asm if "tcgen05.wait::ld" in s]) == len(loads)


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_overlapped_kernels_do_not_call_their_inputs_constant(path):
    """A kernel that starts while the one before it ends (overlap_launches) may read what that one is still writing: its
    inputs do change while it runs, so none is `const __restrict__`, which would let loads move ahead of its wait or
    take the path of data that nobody writes."""
    text = without_comments(path)
    for at in re.finditer(r"__global__", text):
        end = text.index("{", at.start())
        body = text[end:text.index("\n}", end)]
        if "overlap_launches" in body:
            assert not re.search(r"\bconst\s+\w+\s*\*\s*__restrict__", text[at.start():end])


@pytest.mark.parametrize("name", ["linear.cu", "adamw.cu", "launch.cuh"])
def test_the_layers_rules_ask_the_device_for_its_size(name):
    """No rule of the layer calls has an SM count of its own (148, half, a quarter or twice as many), and what a device
    was asked once is kept for that device."""
    text = without_comments(CSRC / name)
    assert not re.search(r"\b(148|296|74|37)\b", text.replace("* 6 / 37", "").replace("* 13 / 37", ""))
    for kept in re.findall(r"static std::atomic<int> \w+(\[[^;]*\])?;", text):
        assert "KNOWN_DEVICES" in kept

"""The C ABI's products with scratch memory from the caller."""

import ctypes
import struct

import pytest
import torch

pytestmark = pytest.mark.gpu
ALLOCATOR = ctypes.CFUNCTYPE(ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t)


def views(*tensors):
    return struct.pack("=" + "Qqq" * len(tensors), *(v for t in tensors for v in (
        (0, 0, 0) if t is None else (t.data_ptr(), t.stride(0) if t.dim() == 2 else 0, t.stride(-1)))))


def calls(oztt, odd):
    """(name, arguments, the results' buffers, what the calls on tensors give) of a forward and a backward product."""
    m, n, k = 100, 200, 264 + odd
    x, w, dy = (torch.randn(*s, device="cuda").bfloat16() for s in ((m, k), (n, k), (m, n)))
    y, dx, dw, db = (torch.empty_like(t) for t in (dy, x, w, dy[0]))
    yield ("oztt_linear_forward_in", struct.pack("=ii3Q", 0, 0, m, n, k) + views(x, w, None, None, y, None), [y],
           [oztt.linear(x, w)], odd)
    yield ("oztt_linear_backward_in", struct.pack("=ii3Q", 0, 1, m, n, k) + views(dy, dy, x, w, dx, dw, db), [dx, dw, db],
           oztt.linear_backward(dy, x, w, pre=dy, activation="relu"), 1)


@pytest.mark.parametrize("odd", [0, 1])
def test_memory_from_the_caller(oztt, cuda, odd):
    for name, args, got, want, needs in calls(oztt, odd):
        held = []

        def alloc(context, size):
            held.append(torch.empty(size, dtype=torch.uint8, device="cuda"))
            return held[-1].data_ptr()

        oztt.call(name, 0, args, ALLOCATOR(alloc), None, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert len(held) == needs and all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_memory(oztt, cuda):
    for name, args, got, want, needs in calls(oztt, 1):
        for t in got:
            t.fill_(7)
        with pytest.raises(MemoryError):
            oztt.call(name, 0, args, ALLOCATOR(lambda context, size: None), None, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert all(bool((t == 7).all()) for t in got)


def test_memory_off_its_boundary(oztt, cuda):
    room = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
    for name, args, got, want, needs in calls(oztt, 1):
        for t in got:
            t.fill_(7)
        for off in (1, 8, 16, 128):
            with pytest.raises(ValueError, match="256"):
                oztt.call(name, 0, args, ALLOCATOR(lambda context, size: room.data_ptr() + off), None,
                          torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert all(bool((t == 7).all()) for t in got)


def test_refusals(oztt, cuda):
    for name in ("oztt_linear_forward_in", "oztt_linear_backward_in"):
        with pytest.raises(ValueError, match="no arguments"):
            oztt.call(name, 0, None, None, None, None)

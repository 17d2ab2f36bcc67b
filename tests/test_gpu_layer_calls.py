"""The layer calls in captures, on several streams and from several threads."""

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def training_step(oztt, x, w, b, dy, opt, grads):
    pre = oztt.linear(x, w, b, activation="silu", save_pre=True)[1]
    dx, dw, db = oztt.linear_backward(dy, x, w, pre=pre, activation="silu")
    grads[0].copy_(dw)
    grads[1].copy_(db)
    opt.step(grads)
    return dx


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("odd", [0, 1])
def test_captured_training_step(oztt, cuda, bits, odd):
    """Forward, backward and the optimiser's step from a graph are those of the calls (a graph repeats its step's
    number: one replay)."""
    runs = []
    for captured in (False, True):
        g = torch.Generator(device="cuda").manual_seed(1)
        r = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()  # noqa: E731
        x, w, b, dy = r(300, 256 + odd), r(200 + odd, 256 + odd) / 16, r(200 + odd), r(300, 200 + odd)
        opt = oztt.AdamW([w, b], masters=True, state_bits=bits, seed=4)
        grads = [torch.zeros_like(w), torch.zeros_like(b)]
        if captured:
            oztt.linear(x, w, b)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                dx = training_step(oztt, x, w, b, dy, opt, grads)
            graph.replay()
        else:
            dx = training_step(oztt, x, w, b, dy, opt, grads)
        torch.cuda.synchronize()
        runs.append([dx.clone(), w.clone(), b.clone(), opt.m.clone(), opt.v.clone(), *[t.clone() for t in opt.masters]])
    assert all(torch.equal(a, c) for a, c in zip(*runs))


def products(oztt, seed):
    """Calls of every path, and what each gives."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()  # noqa: E731
    out = []
    for m, n, k in ((1, 520, 1024), (4, 264, 512), (16, 256, 4096), (200, 300, 777), (1300, 2064, 264)):
        x, w, b, dy = r(m, k), r(n, k) / 16, r(n), r(m, n)
        y, pre = oztt.linear(x, w, b, activation="gelu", save_pre=True)
        out += [y, pre, *oztt.linear_backward(dy, x, w, pre=pre, activation="gelu"),
                *oztt.linear_backward(dy, x, w)]
    return out


def test_from_two_streams_and_threads(oztt, cuda):
    want = [products(oztt, seed) for seed in (1, 2)]
    torch.cuda.synchronize()
    got, failed = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[i] = products(oztt, i + 1)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))

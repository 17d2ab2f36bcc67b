"""States that are refused, and states that are loaded."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_states_of_other_tensors_are_refused(oztt, cuda):
    """Sizes whose blocks add up alike, masters of another shape, buffers of another kind: refused, and nothing is
    loaded."""
    def make(sizes, **kw):
        opt = oztt.AdamW([torch.randn(n, device="cuda").bfloat16() for n in sizes], masters=True, state_bits=8, **kw)
        opt.step([torch.randn(n, device="cuda") for n in sizes])
        return opt

    a, b = make([300, 700]), make([700, 300], seed=9)
    kept = [t.clone() for t in (a.m, a.v, a.m_exp, a.v_exp, *a.masters)]
    good = a.state_dict()
    bad = [b.state_dict(), {**good, "masters": [a.masters[0][:1], a.masters[1]]},
           {**good, "masters": [a.masters[1], a.masters[0]]}, {**good, "masters": good["masters"][:1]},
           {**good, "m": good["m"].float() + 1}, {**good, "m_exp": good["m_exp"][:1]}]
    for d in bad:
        with pytest.raises(ValueError):
            a.load_state_dict(d)
        assert all(torch.equal(x, y) for x, y in zip(kept, (a.m, a.v, a.m_exp, a.v_exp, *a.masters)))
        assert a.t == 1 and a.seed == 0
    with pytest.raises(ValueError):
        a.load_state_dict({k: v for k, v in good.items() if k != "v"})
    c = oztt.AdamW([torch.zeros(n, device="cuda").bfloat16() for n in (300, 700)], masters=True, state_bits=8)
    c.load_state_dict(a.state_dict())
    assert torch.equal(c.m, a.m) and torch.equal(c.masters[1], a.masters[1])

"""AdamW's bookkeeping, with the step itself replaced: what counts as a step, what a copy is."""
import pytest
import torch


@pytest.fixture
def adamw(monkeypatch):
    """an AdamW over three CPU parameters in two groups; calls are written down, those with a tensor of `refused` are refused"""
    from vc3d import ops, optim
    from vc3d.capi import Vc3dError
    calls, refused = [], []

    def step(params, *moments, **hyper):
        if any(p is q for p in params for q in refused):
            raise Vc3dError("refused")
        calls.append((list(params), hyper["step"]))
    monkeypatch.setattr(ops, "adamw_step", step)
    monkeypatch.setattr(optim.AdamW, "_new_state", lambda self, p: {"step": 0, "exp_avg": torch.zeros_like(p), "exp_avg_sq": torch.zeros_like(p)})
    ps = [torch.nn.Parameter(torch.zeros(k + 1)) for k in range(3)]
    for p in ps:
        p.grad = torch.ones_like(p)
    return optim.AdamW([dict(params=ps[:2]), dict(params=ps[2:], lr=0.1)]), ps, calls, refused


def counts(opt, ps):
    return [opt.state[p]["step"] if opt.state[p] else 0 for p in ps]


def test_a_refused_step_does_not_count(adamw):
    from vc3d.capi import Vc3dError
    opt, ps, calls, refused = adamw
    opt.step()
    assert counts(opt, ps) == [1, 1, 1] and [c[1] for c in calls] == [1, 1]
    refused.append(ps[1])
    for _ in range(3):
        with pytest.raises(Vc3dError):
            opt.step()
    assert counts(opt, ps) == [1, 1, 1]
    refused[:] = [ps[2]]  # the first group has been stepped when the second is refused
    with pytest.raises(Vc3dError):
        opt.step()
    assert counts(opt, ps) == [2, 2, 1]
    refused.clear()
    ps[0].grad = None
    opt.step()
    assert counts(opt, ps) == [2, 3, 2] and [c[1] for c in calls[-2:]] == [3, 2]

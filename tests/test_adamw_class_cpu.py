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


@pytest.mark.parametrize("bits", [32, 8])
def test_a_copy_holds_its_moments_in_as_many_bits(bits):
    import copy
    import pickle

    from vc3d.optim import AdamW
    opt = AdamW([torch.nn.Parameter(torch.zeros(3))], lr=0.5, state_bits=bits)
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert other.state_bits == bits and other.param_groups[0]["lr"] == 0.5
        assert other.state_dict()["state_bits"] == bits


def test_moments_that_torch_held_in_the_parameters_type_are_widened():
    """torch.optim.AdamW holds the moments of a bf16 parameter in bf16; here they are fp32 whatever the parameter's type"""
    from vc3d.optim import AdamW
    p = torch.nn.Parameter(torch.randn(40).bfloat16())
    theirs = torch.optim.AdamW([p], lr=1e-2)
    for _ in range(2):
        p.grad = torch.randn(40).bfloat16()
        theirs.step()
    mine = AdamW([p], lr=1e-2)
    mine.load_state_dict(theirs.state_dict())
    for k in ("exp_avg", "exp_avg_sq"):
        assert theirs.state[p][k].dtype == torch.bfloat16 and mine.state[p][k].dtype == torch.float32
        assert torch.equal(mine.state[p][k], theirs.state[p][k].float())
    assert mine.state[p]["step"] == 2


def test_eight_bits_that_there_are_not_are_refused():
    """without a GPU 'adamw' is torch's, whose moments have no other width"""
    from helpers import make_config
    from utils.utils import create_optimizer
    cfg = make_config(18, 10, OPTIMIZER="adamw", STATE_BITS=8)
    with pytest.raises(ValueError, match="STATE_BITS"):
        create_optimizer(cfg, torch.nn.Linear(4, 2))


def test_a_parameter_that_is_listed_twice_is_stepped_twice(monkeypatch):
    """as torch does (with a warning): two steps, one after the other, each with its own count"""
    import warnings

    from vc3d import ops, optim
    calls = []
    monkeypatch.setattr(ops, "adamw_step", lambda params, *a, **k: calls.append((len(params), k["step"])))
    monkeypatch.setattr(optim.AdamW, "_new_state", lambda self, p: {"step": 0, "exp_avg": torch.zeros_like(p), "exp_avg_sq": torch.zeros_like(p)})
    p, q = torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(2))
    p.grad, q.grad = torch.ones(3), torch.ones(2)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        opt = optim.AdamW([p, q, p])
    opt.step()
    assert calls == [(2, 1), (1, 2)] and opt.state[p]["step"] == 2 and opt.state[q]["step"] == 1

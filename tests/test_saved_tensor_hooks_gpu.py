"""The backward of the scan and of the linear cross-entropy where a caller's hooks hold what autograd saves and hand back copies at
other addresses and strides, as offloading does; tensors that are others are refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def moved(t, shift=1):
    """a copy that begins `shift` elements into its storage"""
    flat = torch.empty(t.numel() + shift, dtype=t.dtype, device=t.device)
    return flat[shift:].view(t.shape).copy_(t)


def spread(t):
    """a copy whose last dimension is strided"""
    wide = torch.empty(t.shape + (2,), dtype=t.dtype, device=t.device)
    return wide[..., 0].copy_(t)


def offloaded(t):
    return t.cpu().to("cuda")


def hooks(change):
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: change(t))


def scan():
    import vc3d
    g = torch.Generator().manual_seed(1)
    gates = torch.randn(3, 700, 2 * 37, generator=g).cuda().bfloat16().requires_grad_()
    h0, lengths = torch.randn(3, 37, generator=g).cuda().requires_grad_(), torch.tensor([700, 0, 333]).cuda()
    return lambda: vc3d.gated_scan(gates, h0, lengths=lengths), (gates, h0)


def loss(D, keep, shift, bias):
    import vc3d
    g = torch.Generator().manual_seed(2)
    x, w = (moved((torch.randn(n, D, generator=g) / 4).bfloat16().cuda(), shift) for n in (70, 900))
    b = torch.randn(900, generator=g).bfloat16().cuda() if bias else None
    y = torch.randint(0, 900, (70,), generator=g).cuda()
    leaves = [t.requires_grad_() for t in (x, w, b) if t is not None]
    return lambda: (vc3d.linear_cross_entropy(x, w, y, b, keep_bytes=keep),), tuple(leaves)


CASES = [("scan", scan)] + [("lce-%d-%d-%d" % (D, keep, shift), lambda D=D, keep=keep, shift=shift: loss(D, keep, shift, D == 64))
                            for D in (64, 61) for keep in (0, 1 << 30) for shift in (0, 1)]


def grads(case, change):
    call, leaves = case()
    if change is None:
        outs = call()
    else:
        with hooks(change):
            outs = call()
    return torch.autograd.grad([o.float().square().sum() for o in outs], leaves)


@pytest.mark.parametrize("change", [offloaded, moved, spread, lambda t: moved(t, 3)], ids=["offloaded", "moved", "spread", "moved3"])
@pytest.mark.parametrize("case", [c for _, c in CASES], ids=[n for n, _ in CASES])
def test_what_comes_back_elsewhere_gives_the_same_bits(case, change):
    want = grads(case, None)
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(grads(case, change), want))


@pytest.mark.parametrize("change", [lambda t: t.cpu(), lambda t: t[:-1], lambda t: t.double() if t.is_floating_point() else t.short()],
                         ids=["cpu", "shorter", "type"])
@pytest.mark.parametrize("case", [CASES[0][1], CASES[1][1], CASES[4][1]], ids=["scan", "lce", "lce-kept"])
def test_what_comes_back_as_another_tensor_is_refused(case, change):
    with pytest.raises(RuntimeError, match="came back"):
        grads(case, change)

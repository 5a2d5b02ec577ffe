"""Sizes whose work does not fit one launch (2^32 lanes)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_scan_in_two_launches():
    """65535 sequences of one step, 8193 channels: the step form and the formula of its gradients on the same inputs"""
    import vc3d
    B, H = 65535, 8193
    g = torch.Generator(device="cuda").manual_seed(1)
    gates = torch.randn(B, 1, 2 * H, device="cuda", generator=g, dtype=torch.bfloat16).requires_grad_()
    h0 = torch.randn(B, H, device="cuda", generator=g).requires_grad_()
    lengths = torch.ones(B, dtype=torch.int32, device="cuda")
    lengths[::7] = 0
    h, last = vc3d.gated_scan(gates, h0, lengths=lengths)
    with torch.no_grad():
        state = h0.detach().clone()
        out = vc3d.gated_scan_step(gates[:, 0].detach(), state)
        there = lengths[:, None] > 0
        assert torch.equal(h[:, 0], torch.where(there, out, torch.zeros_like(out)))
        assert torch.equal(last, torch.where(there, state, h0))
    # the last state's gradient: dh0 = f up, dv = (1 - f) up; up = 1.  f is off by 2^-21 (exp2 and rcp: 1 ulp each, a few roundings)
    dg, dh0 = torch.autograd.grad(last.sum(), (gates, h0))
    for b in (0, 1, 2, 64526, 64527, 64528, 65533, 65534):
        f = torch.sigmoid(gates[b, 0, :H].detach().double()) if lengths[b] else torch.ones(H, dtype=torch.float64, device="cuda")
        assert bool(((dh0[b].double() - f).abs() <= 2.0 ** -21 * f).all())
        q = torch.sigmoid(-gates[b, 0, :H].detach().double()) * float(lengths[b] > 0)
        assert bool(((dg[b, 0, H:].double() - q).abs() <= (2.0 ** -8 + 2.0 ** -20) * q).all())


def test_a_loss_in_two_pieces():
    """524291 rows of 1048576 words: row losses, each off by twice a logit's error, the sum's and its own rounding"""
    import vc3d
    N, V, D = (1 << 19) + 3, 1 << 20, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(N, D, device="cuda", generator=g, dtype=torch.bfloat16)
    w = torch.randn(V, D, device="cuda", generator=g, dtype=torch.bfloat16) / 4
    y = torch.randint(0, V, (N,), device="cuda", generator=g)
    y[-1], y[0] = V - 1, 1047808  # in the second piece: its last word, its first
    loss = vc3d.linear_cross_entropy(x, w, y, reduction="none")
    rows = torch.tensor([0, 1, 255, 256, 262143, N - 4, N - 2, N - 1], device="cuda")
    z = x[rows].double() @ w.double().t()
    want = torch.logsumexp(z, 1) - z.gather(1, y[rows, None])[:, 0]
    dz = (D + 8) * 2.0 ** -24 * (x[rows].double().abs() @ w.double().abs().t()).amax(1)
    off = 2 * dz + (64 + V / 16) * 2.0 ** -24 + want * 2.0 ** -24
    assert bool(((loss[rows].double() - want).abs() <= off).all())
    assert bool((loss > 0).all())

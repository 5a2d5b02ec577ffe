"""What the gated scan, the linear cross-entropy and AdamW refuse on the GPU, or answer in a way of their own."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_step_that_would_lose_a_gradient_is_refused():
    import vc3d
    from vc3d.capi import Vc3dError
    gates, state = torch.randn(3, 16, device="cuda"), torch.randn(3, 8, device="cuda")
    before = state.clone()
    wants = [(gates.clone().requires_grad_(), state), (gates, state.clone().requires_grad_()), ((gates.clone().requires_grad_() * 2), state)]
    for g, s in wants:
        with pytest.raises(Vc3dError, match="gradient"):
            vc3d.gated_scan_step(g, s)
        assert torch.equal(s.detach(), before)
    want = vc3d.gated_scan(gates[:, None], before)[1]
    for g, s in wants[:2]:
        with torch.no_grad():  # serving a model whose parameters want gradients elsewhere
            h = vc3d.gated_scan_step(g, s)
        assert torch.equal(h, want) and torch.equal(s.detach(), want) and not h.requires_grad
        state.copy_(before)
    assert torch.equal(vc3d.gated_scan_step(gates, state), want)


def test_a_state_of_another_shape_is_refused():
    import vc3d
    from vc3d.capi import Vc3dError
    gates = torch.randn(3, 16, device="cuda")
    for shape in ((8, 3), (24,), (3, 1, 8), (1, 3, 8), (3, 7)):
        with pytest.raises(Vc3dError):
            vc3d.gated_scan_step(gates, torch.zeros(shape, device="cuda"))

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


class limited:
    """torch's allocator may hold `more` bytes beside what it holds now; the holes in that (other tests' work leaves some, of any size) are
    filled"""

    def __init__(self, more):
        self.more, self.total = more, torch.cuda.get_device_properties(0).total_memory

    def most(self, n):
        torch.cuda.set_per_process_memory_fraction(n / self.total)

    def __enter__(self):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        self.most(torch.cuda.memory_reserved())
        self.holes, size = [], 1 << 32
        while size >= 4 << 20:
            try:
                self.holes.append(torch.empty(size, dtype=torch.uint8, device="cuda"))
            except torch.OutOfMemoryError:
                size //= 2
        self.most(torch.cuda.memory_reserved() + self.more)

    def __exit__(self, *exc):
        self.most(self.total)
        del self.holes


def test_memory_that_runs_out_is_torchs_error():
    """callers that catch torch.OutOfMemoryError, to free memory or take a smaller batch, see it"""
    import vc3d
    gates = torch.zeros(64, 1024, 2048, device="cuda")  # 512 MB; h: 256
    x, w, y = torch.zeros(65536, 8, device="cuda"), torch.zeros(8192, 8, device="cuda"), torch.zeros(65536, dtype=torch.int64, device="cuda")
    for call in (lambda: vc3d.gated_scan(gates), lambda: vc3d.linear_cross_entropy(x.requires_grad_(), w, y, keep_bytes=4 << 30)):
        with limited(32 << 20):
            with pytest.raises(torch.OutOfMemoryError):
                call()
    assert not vc3d.gated_scan(gates)[0].any()


def test_what_a_hook_raises_reaches_the_caller():
    import vc3d

    class Mine(Exception):
        pass

    def pack(t):
        raise Mine("from the hook")
    gates = torch.zeros(2, 3, 8, device="cuda", requires_grad=True)
    x, w, y = torch.zeros(4, 8, device="cuda", requires_grad=True), torch.zeros(10, 8, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    for call in (lambda: vc3d.gated_scan(gates), lambda: vc3d.linear_cross_entropy(x, w, y)):
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            with pytest.raises(Mine, match="from the hook"):
                call()


@pytest.mark.parametrize("engine", [False, True])
def test_nothing_is_kept_where_there_is_no_room(engine):
    """8192 x 65536 bf16 logits are 1 GB: with less the step runs as with keep_bytes=0, to the same bits; what the caller asked to be
    kept is not dropped"""
    import vc3d
    from vc3d.linear_ce import _EngineHeadFn
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(8192, 1024, device="cuda", generator=g).bfloat16().requires_grad_()
    w = (torch.randn(65536, 1024, device="cuda", generator=g) / 32).bfloat16().requires_grad_()
    y = torch.randint(0, 65536, (8192,), device="cuda", generator=g)

    def step(keep):
        if engine and keep == -1:
            loss = _EngineHeadFn.apply(x, w, None, y, type("Engine", (), dict(flat_grad=None)))
        else:
            loss = vc3d.linear_cross_entropy(x, w, y, keep_bytes=keep)
        return (loss.detach(),) + torch.autograd.grad(loss, (x, w))
    want = step(0)
    with limited(1000 << 20):
        got = step(-1)
        with pytest.raises(torch.OutOfMemoryError):
            step(2 << 30)
    assert all(torch.equal(a, b) for a, b in zip(got, want))

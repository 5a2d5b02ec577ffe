"""Gated linear recurrence (vc3d.gated_scan, gated_scan_step) against the step-by-step recurrence in 64 bits, on the CPU, of the
same (rounded) inputs.

Tolerances.  Per step the kernels round the gate (exp, reciprocal and the products around them: under 8 half steps of 2^-24,
the argument of exp adds |z| 2^-24) and the affine map (3 half steps), each relative to at most M = max(|h0|, |v|), which bounds
every state.  A state forgets: f < 1, so errors of the steps before only shrink; composing maps instead of applying them adds as
many roundings again.  So |h - exact| <= T * C * M with C = 2 * (11 + max|z|) 2^-24, plus half a step of h's type.  Backward:
lam is the same recurrence with dy for u (bounded by L = max |lam| of the exact run); dv = q lam, dz = lam (h - v) f q with
f q <= 1/4 and |h - v| <= 2 M: errors T * C * L and T * C * 2 M L (both factors), plus half a step of the type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def reference(gates, h0, lengths, reverse, dy=None, dlast=None):
    """everything in 64 bits, one step after the other -> h, last, dgates, dh0, max |lam|"""
    B, T, H2 = gates.shape
    H = H2 // 2
    z, v = gates[..., :H].double().cpu(), gates[..., H:].double().cpu()
    f, q = torch.sigmoid(z), torch.sigmoid(-z)
    h, last = torch.zeros(B, T, H, dtype=torch.float64), torch.zeros(B, H, dtype=torch.float64)
    dg, dh0, top = torch.zeros(B, T, H2, dtype=torch.float64), torch.zeros(B, H, dtype=torch.float64), 0.0
    for b in range(B):
        n = T if lengths is None else int(lengths[b])
        order = list(range(n - 1, -1, -1)) if reverse else list(range(n))
        s = torch.zeros(H, dtype=torch.float64) if h0 is None else h0[b].double().cpu()
        before = {}
        for t in order:
            before[t] = s
            s = f[b, t] * s + q[b, t] * v[b, t]
            h[b, t] = s
        last[b] = s
        mu = torch.zeros(H, dtype=torch.float64) if dlast is None else dlast[b].double().cpu()
        for t in reversed(order):
            lam = mu if dy is None else mu + dy[b, t].double().cpu()
            top = max(top, float(lam.abs().max()))
            dg[b, t, H:] = q[b, t] * lam
            dg[b, t, :H] = lam * (before[t] - v[b, t]) * f[b, t] * q[b, t]
            mu = f[b, t] * lam
        dh0[b] = mu
    return h, last, dg, dh0, top


def make(B, T, H, dtype, seed=0, shift=1.0):
    g = torch.Generator().manual_seed(seed)
    gates = torch.randn(B, T, 2 * H, generator=g)
    gates[..., :H] += shift
    return (gates.to(dtype).cuda(), torch.randn(B, H, generator=g).cuda(), torch.randn(B, T, H, generator=g).to(dtype).cuda(),
            torch.randn(B, H, generator=g).cuda())


def check(got, want, tol, half, what):
    want = want.to(got.device)
    err = (got.double() - want).abs()
    assert bool(torch.isfinite(got).all()), what
    over = err - (tol + half * want.abs())
    assert float(over.max()) <= 0, "%s: off by %.3e, %.3e allowed" % (what, float(err.max()), float((tol + half * want.abs()).max()))


def run_and_check(gates, h0, lengths, reverse, dy, dlast):
    import vc3d
    gates_l = gates.detach().requires_grad_()
    h0_l = None if h0 is None else h0.detach().requires_grad_()
    dev_len = None if lengths is None else torch.tensor(lengths, device="cuda", dtype=torch.int32)
    h, last = vc3d.gated_scan(gates_l, h0_l, lengths=dev_len, reverse=reverse)
    wrt = (gates_l,) if h0 is None else (gates_l, h0_l)
    grads = torch.autograd.grad((h, last), wrt, (dy, dlast))
    torch.cuda.synchronize()
    # what counts for the bounds: nothing behind a sequence's end
    clean, dyc = gates.detach().clone(), dy.clone()
    if lengths is not None:
        for b, n in enumerate(lengths):
            clean[b, n:], dyc[b, n:] = 0, 0
    eh, el, eg, e0, L = reference(clean, h0, lengths, reverse, dyc, dlast)
    H, T = h.shape[2], h.shape[1]
    M = max(float(clean[..., H:].abs().max()) if clean.numel() else 0.0, float(h0.abs().max()) if h0 is not None else 0.0)
    z = float(clean[..., :H].abs().max()) if clean.numel() else 0.0
    C = max(T, 1) * 2 * (11 + z) * 2.0 ** -24
    half = HALF[gates.dtype]
    check(h, eh, C * M, half, "h")
    check(last, el, C * M, 2.0 ** -24, "last")
    check(grads[0][..., H:], eg[..., H:], C * L, half, "dv")
    check(grads[0][..., :H], eg[..., :H], C * 4 * M * L, half, "dz")
    if h0 is not None:
        check(grads[1], e0, C * L, 2.0 ** -24, "dh0")
    if lengths is not None:  # exactly 0 behind the end
        for b, n in enumerate(lengths):
            assert not bool(h[b, n:].any()) and not bool(grads[0][b, n:].any())
    return h, last, grads


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,H", [(1, 1, 1), (2, 1, 64), (1, 2, 3), (3, 15, 130), (2, 63, 128), (2, 64, 127), (1, 65, 256), (2, 127, 20),
                                   (1, 128, 128), (2, 129, 33), (1, 700, 130), (5, 257, 64), (1, 4100, 20)])
def test_matches_the_recurrence(B, T, H, dtype):
    gates, h0, dy, dlast = make(B, T, H, dtype, seed=B * 1000 + T + H)
    run_and_check(gates, h0, None, False, dy, dlast)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,lengths,reverse", [(1, [4500, 0, 2049], False), (2, [1, 2048, 4097], True), (5, [2047, 16, 3000], False), (16, [4200, 129, 2048], False),
                                               (15, [1025, 1023, 17], True), (17, [2100, 8, 1024], False), (32, [1024, 1040, 2050], True), (31, [7, 2000, 513], False),
                                               (33, [1300, 512, 0], False), (63, [511, 513, 1024], True), (64, [1100, 256, 255], False), (65, [300, 257, 1], True)])
def test_few_channels_share_a_wave_with_later_steps(H, lengths, reverse, dtype):
    """the borders of groups, waves and tiles for every number of lanes that hold channels, odd numbers of channels"""
    gates, h0, dy, dlast = make(3, max(lengths) + 3, H, dtype, seed=H)
    run_and_check(gates, h0, lengths, reverse, dy, dlast)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reverse", [False, True])
def test_lengths_direction_and_what_lies_behind_the_end(dtype, reverse):
    lengths = [0, 1, 300, 63, 64, 65, 129, 299]
    gates, h0, dy, dlast = make(8, 300, 70, dtype, seed=3)
    for b, n in enumerate(lengths):  # padding holds anything
        gates[b, n:] = float("nan")
        dy[b, n:] = float("inf")
    _, last, grads = run_and_check(gates, h0, lengths, reverse, dy, dlast)
    assert torch.equal(last[0], h0[0]) and torch.equal(grads[1][0], dlast[0])  # a sequence without steps


def test_reverse_without_lengths_and_without_a_first_state():
    gates, _, dy, dlast = make(2, 200, 96, torch.bfloat16, seed=4)
    run_and_check(gates, None, None, True, dy, dlast)


def test_lengths_of_int64_and_out_of_range_are_clamped():
    import vc3d
    gates, h0, _, _ = make(3, 70, 16, torch.float32, seed=5)
    want = vc3d.gated_scan(gates, h0, lengths=torch.tensor([0, 70, 7], device="cuda", dtype=torch.int32))
    for dt in (torch.int32, torch.int64):
        got = vc3d.gated_scan(gates, h0, lengths=torch.tensor([-5, 2 ** 31 - 1, 7], device="cuda", dtype=dt))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gates_that_are_saturated_or_infinite(dtype):
    """f = 0 and f = 1 exactly at +-inf and far out; nothing turns into NaN, also in the gradients"""
    import vc3d
    H = 64
    gates, h0, dy, dlast = make(2, 150, H, dtype, seed=6)
    far = torch.tensor([float("inf"), -float("inf"), 200.0, -200.0, 88.0, -88.0, torch.finfo(dtype).min, torch.finfo(dtype).max])
    gates[:, :, :H] = far.to(dtype).cuda().repeat(H // 8)[torch.randperm(H, generator=torch.Generator().manual_seed(1)).cuda()]
    gates.requires_grad_()
    h0.requires_grad_()
    h, last = vc3d.gated_scan(gates, h0)
    grads = torch.autograd.grad((h, last), (gates, h0), (dy, dlast))
    eh, el, eg, e0, L = reference(gates.detach(), h0.detach(), None, False, dy, dlast)
    M = 8.0
    for got, want in ((h, eh), (last, el), (grads[0][..., H:], eg[..., H:]), (grads[0][..., :H], eg[..., :H]), (grads[1], e0)):
        check(got, want, 150 * 2 * 11 * 2.0 ** -24 * M * max(L, 1.0), HALF[dtype], "saturated")


def test_layouts():
    """slices of a wider tensor at odd offsets, time-major storage, an expanded batch: the same bits as from a contiguous copy"""
    import vc3d
    g = torch.Generator().manual_seed(7)
    wide = torch.randn(3, 140, 2 * 40 + 5, generator=g).to(torch.bfloat16).cuda()
    views = [wide[..., 3:83], wide[..., 1:79], torch.randn(140, 3, 64, generator=g).cuda().transpose(0, 1),
             torch.randn(1, 140, 64, generator=g).cuda().expand(3, 140, 64), wide[:, 1::2, 2:82]]
    for v in views:
        want, got = vc3d.gated_scan(v.contiguous()), vc3d.gated_scan(v)
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
        a, b = v.detach().contiguous().requires_grad_(), v.detach().requires_grad_()
        dy = torch.randn(want[0].shape, generator=g).to(v.dtype).cuda()
        ga, = torch.autograd.grad(vc3d.gated_scan(a)[0], a, dy)
        odd = torch.empty(dy.numel() + 1, dtype=dy.dtype, device="cuda")[1:].view(dy.shape).copy_(dy)  # an upstream gradient at an odd offset
        gb, = torch.autograd.grad(vc3d.gated_scan(b)[0], b, odd)
        assert torch.equal(ga, gb)


def test_only_one_output_has_a_gradient():
    import vc3d
    gates, h0, dy, dlast = make(2, 130, 32, torch.float32, seed=8)
    zero, zl = torch.zeros_like(dy), torch.zeros_like(dlast)
    gates.requires_grad_(), h0.requires_grad_()
    full = lambda a, b: torch.autograd.grad(vc3d.gated_scan(gates, h0), (gates, h0), (a, b))  # noqa: E731
    for pick, (a, b) in ((0, (dy, zl)), (1, (zero, dlast))):
        want = full(a, b)
        got = torch.autograd.grad(vc3d.gated_scan(gates, h0)[pick], (gates, h0), (a, b)[pick])
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    # a sum hands an expanded gradient down
    got, = torch.autograd.grad(vc3d.gated_scan(gates, h0)[0].sum(), gates)
    assert torch.equal(got, full(torch.ones_like(dy), zl)[0])


def test_gradient_against_differences():
    """central differences of a weighted sum of the outputs along a random direction, fp32.  h is smooth: the third derivative
    along a unit-size direction is below 1 per unit of weight, so the truncation is under eps^2 = 2^-14 of the sum's scale
    S = sum |weights| M; the outputs' rounding (T C M each) divides by eps = 2^-7"""
    import vc3d
    B, T, H = 2, 100, 16
    gates, h0, dy, dlast = make(B, T, H, torch.float32, seed=9)
    g = torch.Generator().manual_seed(10)
    d, d0 = torch.randn(gates.shape, generator=g).cuda(), torch.randn(h0.shape, generator=g).cuda()

    def value(s):
        h, last = vc3d.gated_scan(gates + s * d, h0 + s * d0)
        return float((h.double() * dy).sum() + (last.double() * dlast).sum())
    gl, hl = gates.clone().requires_grad_(), h0.clone().requires_grad_()
    dg, dh = torch.autograd.grad(vc3d.gated_scan(gl, hl), (gl, hl), (dy, dlast))
    slope = float((dg.double() * d).sum() + (dh.double() * d0).sum())
    eps = 2.0 ** -7
    S = float(dy.abs().sum() + dlast.abs().sum())
    M = float(gates[..., H:].abs().max())
    # errors of the outputs are independent over them: their sum grows with the root of their number
    noise = (B * T * H) ** 0.5 * 16 * 2.0 ** -24 * M * float(dy.abs().max()) / eps
    assert abs((value(eps) - value(-eps)) / (2 * eps) - slope) <= eps ** 2 * S * M + noise


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H", [(1, 1), (3, 33), (64, 2048), (5000, 8)])
def test_step_is_the_scan_of_one_step(B, H, dtype):
    import vc3d
    gates, h0, _, _ = make(B, 1, H, dtype, seed=11)
    want, last = vc3d.gated_scan(gates, h0)
    state = h0.clone()
    version = state._version
    got = vc3d.gated_scan_step(gates[:, 0], state)
    assert torch.equal(got, want[:, 0]) and torch.equal(state, last) and state._version > version
    # rows of a wider buffer
    wide = torch.zeros(B, 2 * H + 3, dtype=dtype, device="cuda")
    wide[:, 1:2 * H + 1] = gates[:, 0]
    state = h0.clone()
    assert torch.equal(vc3d.gated_scan_step(wide[:, 1:2 * H + 1], state), got) and torch.equal(state, last)


def test_steps_continue_a_scan():
    """a prompt scanned at once, then steps: the same states as one scan over all of it, to the bound of its steps"""
    import vc3d
    gates, h0, _, _ = make(4, 90, 48, torch.float32, seed=12)
    h, last = vc3d.gated_scan(gates, h0)
    _, state = vc3d.gated_scan(gates[:, :70], h0)
    outs = [vc3d.gated_scan_step(gates[:, t], state) for t in range(70, 90)]
    tol = 90 * 2 * (11 + float(gates.abs().max())) * 2.0 ** -24 * float(gates.abs().max())
    assert float((torch.stack(outs, 1) - h[:, 70:]).abs().max()) <= tol and float((state - last).abs().max()) <= tol


def test_empty_inputs():
    import vc3d
    h0 = torch.randn(2, 8, device="cuda", requires_grad=True)
    for B, T in ((2, 0), (0, 5)):
        gates = torch.randn(B, T, 16, device="cuda", requires_grad=True)
        h, last = vc3d.gated_scan(gates, h0[:B])
        assert h.shape == (B, T, 8) and torch.equal(last, h0[:B])
        dg, dh = torch.autograd.grad((h.sum() + (last * 2).sum()), (gates, h0))
        assert dg.shape == gates.shape and torch.equal(dh[:B], torch.full((B, 8), 2.0, device="cuda"))


def test_runs_repeat_bit_for_bit_and_on_other_streams():
    import vc3d
    gates, h0, dy, dlast = make(2, 5000, 160, torch.bfloat16, seed=13)
    gates.requires_grad_(), h0.requires_grad_()

    def once():
        h, last = vc3d.gated_scan(gates, h0)
        return (h.detach(), last.detach()) + torch.autograd.grad((h, last), (gates, h0), (dy, dlast))
    want = once()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(once())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(want, g))


def test_two_captured_graphs_replay():
    """forward and backward captured twice (two graphs of their own), replayed several times with eager work in between and new
    inputs in the captured buffers"""
    import vc3d
    gates, h0, dy, dlast = make(2, 700, 96, torch.float32, seed=14)

    def once(gates):
        h, last, states = vc3d.ops.gated_scan_fwd(gates, h0, want_states=True)
        dg, dh0 = vc3d.ops.gated_scan_bwd(gates, None, states, dy, dlast)
        return h, last, dg, dh0
    ins = [gates.clone(), gates.flip(1).contiguous()]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for x in ins:
            once(x)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in ins:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(once(x))
        graphs.append(graph)
    for rep in range(3):
        for x in ins:
            x.mul_(-1.0)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for x, out in zip(ins, outs):
            assert all(torch.equal(a, b) for a, b in zip(once(x), out))


def test_more_than_2_31_elements():
    """one sequence whose gates pass 2^31 elements: its ends, against 400 steps around them (what lies further off is forgotten:
    a product of 300 gates is below 2^-100)"""
    import vc3d
    T, H, near = 140000, 8192, 100
    torch.manual_seed(41)
    gates = torch.randn(1, T, 2 * H, dtype=torch.bfloat16, device="cuda")
    gates[..., :H] += 1
    dy = torch.randn(1, T, H, dtype=torch.bfloat16, device="cuda")
    gates.requires_grad_()
    h, last = vc3d.gated_scan(gates)
    dgates, = torch.autograd.grad((h, last), gates, (dy, torch.ones_like(last)))
    g = gates.detach()
    M, z = 8.0, 8.0  # (normal values of 8 bits' mantissa: below)
    half = HALF[torch.bfloat16]
    for first in (True, False):
        at = slice(0, 400) if first else slice(T - 400, T)
        eh, el, eg, _, L = reference(g[:, at].clone(), None, None, False, dy[:, at], torch.zeros(1, H) if first else torch.ones(1, H))
        part = slice(0, near) if first else slice(400 - near, 400)
        C = 400 * 2 * (11 + z) * 2.0 ** -24
        assert float(g[:, at].float().abs().max()) < M
        check(h[:, at][:, part], eh[:, part], C * M, half, "h")
        check(dgates[:, at][:, part, H:], eg[:, part, H:], C * L, half, "dv")
        check(dgates[:, at][:, part, :H], eg[:, part, :H], C * 4 * M * L, half, "dz")
    check(last, el, C * M, 2.0 ** -24, "last")

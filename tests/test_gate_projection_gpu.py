"""The gate projection's packed operands where calls share them: streams, graphs, weights that change in between."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def cell_of(F, H, seed):
    from models.recurrence import GatedScan
    torch.manual_seed(seed)
    return GatedScan(F, H).cuda()


def expected(cell, x):
    """what a module without any history computes"""
    with torch.no_grad():
        out = copy.deepcopy(cell).sequence(x)
    torch.cuda.synchronize()
    return out


def equal(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


def test_sequences_on_two_streams_after_a_change_of_weights():
    """the first call packs behind 50 ms of other work on its stream; the second, on another stream, may not overtake it"""
    cell, g = cell_of(128, 64, 1), torch.Generator().manual_seed(2)
    xs = [torch.randn(3, 40, 128, generator=g).cuda() for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for step in range(3):
        with torch.no_grad():
            cell.gates.weight.normal_()
        want = [expected(cell, x) for x in xs]
        with torch.no_grad():
            with torch.cuda.stream(streams[step % 2]):
                torch.cuda._sleep(100_000_000)
                first = cell.sequence(xs[0])
            with torch.cuda.stream(streams[1 - step % 2]):
                second = cell.sequence(xs[1])
        torch.cuda.synchronize()
        assert equal(first, want[0]) and equal(second, want[1]), step


@pytest.mark.parametrize("warm", [True, False])
def test_a_captured_sequence_follows_the_weights(warm):
    """replays with what the weights hold then, eager calls between the replays, the graph's memory its own"""
    cell, g = cell_of(128, 64, 3), torch.Generator().manual_seed(4)
    x = torch.randn(3, 40, 128, generator=g).cuda()
    expected(cell_of(128, 64, 5), x)  # (kernels loaded)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        if warm:
            with torch.cuda.stream(side):
                cell.sequence(x)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            out = cell.sequence(x)
        want = expected(cell, x)
        assert equal(cell.sequence(x), want)  # before the first replay
        for k in range(4):
            graph.replay()
            torch.cuda.synchronize()
            assert equal(out, want), k
            cell.gates.weight.normal_()
            want = expected(cell, x)
            if k % 2:
                assert equal(cell.sequence(x), want)  # packs anew: what it replaces is not the graph's
                junk = [torch.full((256, 128), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(64)]
                torch.cuda.synchronize()
                del junk


def operands(N, F, C, seed):
    """bf16-exact x and weight, a bias that takes each column's first product away again: what is left is small beside both"""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(1, F, generator=g) + 2.0 ** -6 * torch.randn(N, F, generator=g)).bfloat16().float()
    w = (torch.randn(C, F, generator=g) * 4.0).bfloat16().float()
    b = -(x[0].double() @ w.double().t()).float()
    return x, w, b


@pytest.mark.parametrize("N,F,C", [(1, 64, 64), (5, 64, 128), (64, 512, 1024), (64, 2048, 1024), (33, 2048, 2048), (1000, 192, 320)])
def test_gates_are_rounded_once(N, F, C):
    """gates = bf16(x W^T + b): operands are exact, the sum of F + 3 products runs in fp32, and one rounding (half a step: 2^-8)
    follows it"""
    from vc3d.scan import PackedGateWeight, gate_projection
    x, w, b = operands(N, F, C, N + F)
    got = gate_projection(x.cuda(), w.cuda(), b.cuda(), PackedGateWeight())
    assert got.dtype == torch.bfloat16
    want = x.double() @ w.double().t() + b.double()
    off = (F + 8) * 2.0 ** -24 * (x.double().abs() @ w.double().abs().t() + b.double().abs())
    assert bool(((got.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + (1 + 2.0 ** -8) * off).all())


def test_gradients_of_a_projection_with_a_bias():
    """dx = dg W, dW = dg^T x, db = sum dg: fp32 sums of exact products (dx rounds to bf16, 2^-8)"""
    from vc3d.scan import PackedGateWeight, gate_projection
    N, F, C = 300, 128, 192
    x, w, b = operands(N, F, C, 9)
    dg = torch.randn(N, C, generator=torch.Generator().manual_seed(10)).bfloat16()
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    gate_projection(*leaves, PackedGateWeight()).backward(dg.cuda())
    d, e = dg.double(), 2.0 ** -24
    want = [d @ w.double(), d.t() @ x.double(), d.sum(0)]
    size = [d.abs() @ w.double().abs(), d.abs().t() @ x.double().abs(), d.abs().sum(0)]
    for t, v, s, terms, half in zip(leaves, want, size, (C, N, N), (2.0 ** -8, e, e)):
        off = (terms + 8) * e * s
        assert t.grad.shape == t.shape and t.grad.dtype == torch.float32
        assert bool(((t.grad.cpu().double() - v).abs() <= half * v.abs() + (1 + half) * off).all())


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), 3.3895e38, 1e-39, 0.0])
def test_a_bias_at_the_ends_of_its_range(value):
    """a gate that is held open or shut by its bias; the other columns do not see it"""
    from vc3d.scan import PackedGateWeight, gate_projection
    x, w, b = operands(7, 64, 64, 11)
    plain = gate_projection(x.cuda(), w.cuda(), b.cuda(), PackedGateWeight()).cpu()
    b[5] = value
    got = gate_projection(x.cuda(), w.cuda(), b.cuda(), PackedGateWeight()).cpu()
    others = torch.arange(64) != 5
    assert torch.equal(got[:, others], plain[:, others]) and not bool(got.isnan().any())
    if abs(value) > 1e38:
        assert bool((got[:, 5].double() * (1 if value > 0 else -1) >= 3.3e38).all())


@pytest.mark.parametrize("B,T", [(0, 7), (3, 0), (0, 0)])
@pytest.mark.parametrize("h0", [False, True])
def test_an_empty_sequence(B, T, h0):
    """no sequences, or none with a step: empty h, the state as it was, gradients of zero"""
    cell, g = cell_of(64, 64, 12), torch.Generator().manual_seed(13)
    x = torch.randn(B, T, 64, generator=g).cuda().requires_grad_()
    start = torch.randn(B, 64, generator=g).cuda().requires_grad_() if h0 else None
    h, last = cell.sequence(x, h0=start)
    assert h.shape == (B, T, 64) and torch.equal(last, torch.zeros(B, 64, device="cuda") if start is None else start)
    (h.sum() + (2.0 * last).sum()).backward()
    assert not x.grad.any() and not cell.gates.weight.grad.any() and not cell.gates.bias.grad.any()
    assert start is None or bool((start.grad == 2.0).all())


def test_a_step_of_no_sequences():
    cell = cell_of(64, 64, 14)
    x = torch.zeros(0, 64, device="cuda")
    assert cell(x).shape == (0, 64)
    with torch.no_grad():
        assert cell(x).shape == (0, 64)


def test_a_captured_sequence_with_its_backward():
    """forward and backward in one graph, replayed with new inputs and new weights between eager work on a copy of the module"""
    cell, g = cell_of(128, 192, 15), torch.Generator().manual_seed(16)
    x = torch.randn(6, 150, 128, generator=g).cuda().requires_grad_()
    up = torch.randn(6, 150, 192, generator=g).cuda()

    def once(c, x):
        h, last = c.sequence(x)
        return (h.detach(), last.detach()) + torch.autograd.grad((h, last), (x, c.gates.weight, c.gates.bias), (up, last.detach()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once(cell, x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once(cell, x)
    for rep in range(4):
        with torch.no_grad():
            for t in (x, cell.gates.weight, cell.gates.bias):
                t.copy_(torch.randn(t.shape, generator=g) * (0.5 + rep) / 8)
        want = once(copy.deepcopy(cell), x.detach().clone().requires_grad_())
        graph.replay()
        torch.cuda.synchronize()
        assert equal(out, want), rep


@pytest.mark.parametrize("rows,D", [(1, 4), (3, 64), (5, 60), (1000, 512), (300000, 64)])
def test_bias_columns(rows, D):
    """x and W with the columns of a bias, exactly: the bias's three parts are bf16 numbers and sum to it"""
    from vc3d import ops
    g = torch.Generator().manual_seed(rows)
    big = torch.randn(rows * D + 1, generator=g).cuda()
    for t in (big[:-1].view(rows, D), big[1:].view(rows, D)):  # (any alignment)
        b = (torch.randn(rows, generator=g) * 10.0 ** torch.randint(-20, 20, (rows,), generator=g)).cuda()
        b[0] = 0.0
        ones = ops.bias_columns(t)
        assert ones.dtype == torch.bfloat16 and torch.equal(ones[:, :D], t.bfloat16())
        assert bool((ones[:, D:D + 3] == 1).all()) and not ones[:, D + 3:].any()
        for dtype in (torch.float32, torch.bfloat16):
            out = ops.bias_columns(t, b, dtype)
            parts = out[:, D:D + 3]
            assert out.dtype == dtype and torch.equal(out[:, :D], t.to(dtype)) and not out[:, D + 3:].any()
            assert torch.equal(parts.bfloat16().to(dtype), parts) and torch.equal(parts.double().sum(1), b.double())


def test_bias_columns_refuses():
    from vc3d import ops
    from vc3d.capi import Vc3dError
    t = torch.zeros(4, 64, device="cuda")
    for args in ((t.cpu(),), (t.bfloat16(),), (t[:, :62],), (t[:, :32],), (t[0],), (t, t[0]), (t, t[:, 0].double()), (t, t[:, 0].cpu()),
                 (t, None, torch.float64)):
        with pytest.raises(Vc3dError):
            ops.bias_columns(*args)
    assert ops.bias_columns(t[:0]).shape == (0, 128)

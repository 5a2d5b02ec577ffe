"""AdamW over a list of tensors (ops.adamw_step, optim.AdamW) against the formula.

Every operation of the step rounds by itself in fp32, so numpy's elementary operations, in the same order, give the same bits:
parameters, 32-bit moments, 8-bit codes and scales are compared for equality with them.  (Not torch's on the CPU: they are not
the correctly rounded ones on every processor -- one parameter of 768 differed from numpy's, and from the kernel's, by 2^-24.)  Apart from that the
update is compared with the formula in 64 bits: under 12 roundings of half a step (2^-24) each of which is relative to the
parameter or to the move lr |m' / ...|; the step's own half step of the parameter's type on top.  A code is off by half a step of
e4m3, 2^-4 of the value, or by half of the least code 2^-9 (times the scale); roots get up to the whole least code."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HYPER = dict(lr=3e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1)
BLOCK = 256
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def rows(t):
    t = t.reshape(-1)
    return torch.nn.functional.pad(t, (0, -t.numel() % BLOCK)).view(-1, BLOCK)


def encode(r, n, floor=0.0):
    """rows of BLOCK fp32 values -> e4m3 codes of the first n, scale of each row"""
    r, f = r.numpy(), np.float32
    with np.errstate(all="ignore"):
        top = np.abs(r).max(1, keepdims=True)
        some = ~(top < f(2.0 ** -100))
        code = r * np.where(some, (f(1) / top) * f(448), f(0))
        if floor:
            code = np.where(some & (r > 0), np.maximum(code, f(floor)), code)
        scale = np.where(some, top * f(1.0 / 448.0), f(0))
    assert code.dtype == f and scale.dtype == f
    return torch.from_numpy(code).to(torch.float8_e4m3fn).view(-1)[:n], torch.from_numpy(scale.reshape(-1).copy())


def plain_step(p, g, m, v, ms, vs, step, lr, beta1, beta2, eps, weight_decay, scale=1.0):
    """fp32 on the CPU, every operation rounded by itself -> new p, m, v, ms, vs and the unrounded moments"""
    n, f = p.numel(), np.float32
    arr = lambda t: t.reshape(-1).float().numpy()  # noqa: E731
    m, v = arr(m), arr(v)
    with np.errstate(all="ignore"):
        if ms is not None:
            m = (rows(torch.from_numpy(m)).numpy() * ms.numpy()[:, None]).reshape(-1)[:n]
            v = (rows(torch.from_numpy(v)).numpy() * vs.numpy()[:, None]).reshape(-1)[:n]
            v = v * v
        g = arr(g) * f(scale)
        m1 = m * f(beta1) + g * f(1.0 - beta1)
        v1 = v * f(beta2) + (g * f(1.0 - beta2)) * g
        r1 = np.sqrt(v1)
        move = (m1 / (r1 * f(1.0 / (1.0 - beta2 ** step) ** 0.5) + f(eps))) * f(lr / (1.0 - beta1 ** step))
        p1 = arr(p) * f(1.0 - lr * weight_decay) - move
    assert all(x.dtype == f for x in (m1, v1, r1, p1))
    m1, v1, r1, p1 = (torch.from_numpy(x) for x in (m1, v1, r1, p1))
    p1 = p1.to(p.dtype)
    if ms is None:
        return p1, m1, v1, None, None, m1, r1
    qm, am = encode(rows(m1), n)
    qv, av = encode(rows(r1), n, 2.0 ** -9)
    return p1, qm, qv, am, av, m1, r1


def make(sizes, dtype, bits, seed=0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        p, gr = torch.randn(n, generator=g).to(dtype), (torch.randn(n, generator=g) * torch.rand(n, generator=g) ** 4 * 1e-2).to(dtype)
        m, v = torch.randn(n, generator=g) * 1e-3, torch.rand(n, generator=g) ** 6 * 1e-5
        if bits == 8:
            (m, ms), (v, vs) = encode(rows(m), n), encode(rows(v.sqrt()), n, 2.0 ** -9)
        else:
            ms = vs = None
        out.append([p, gr, m, v, ms, vs])
    return out


def same(a, b):
    a, b = a.cpu(), b.cpu()
    if a.dtype == torch.float8_e4m3fn:
        a, b = a.view(torch.uint8), b.view(torch.uint8)
    return torch.equal(a.view(-1), b.view(-1))


def step_and_check(ts, step, bits, shift=0, scale=None, hyper=HYPER):
    from vc3d import ops

    def place(t):  # on the device, `shift` elements into its storage
        if t is None:
            return None
        buf = torch.empty(t.numel() + shift, dtype=t.dtype, device="cuda")
        return buf[shift:].copy_(t.cuda())
    dev = [[place(t) for t in x] for x in ts]
    cols = list(zip(*dev)) if dev else [()] * 6
    ops.adamw_step(*[list(c) for c in cols[:4]], *([list(c) for c in cols[4:]] if bits == 8 else []), step=step, grad_scale=scale, **hyper)
    torch.cuda.synchronize()
    sc = 1.0 if scale is None else float(scale)
    for i, (x, d) in enumerate(zip(ts, dev)):
        want = plain_step(*x, step, scale=sc, **hyper)
        for k, name in ((0, "p"), (2, "m"), (3, "v")) + (((4, "m scale"), (5, "v scale")) if bits == 8 else ()):
            assert same(d[k], want[(0, None, 1, 2, 3, 4)[k]]), "tensor %d (%d elements): %s" % (i, x[0].numel(), name)
        # against the formula in 64 bits
        h = hyper
        m0, v0 = x[2].double(), x[3].double()
        n = x[0].numel()
        if bits == 8:
            m0, v0 = (rows(m0) * x[4].double()[:, None]).view(-1)[:n], (rows(v0) * x[5].double()[:, None]).view(-1)[:n] ** 2
        g = x[1].double() * sc
        m1, v1 = h["beta1"] * m0 + (1 - h["beta1"]) * g, h["beta2"] * v0 + (1 - h["beta2"]) * g * g
        den = (v1 / (1 - h["beta2"] ** step)).sqrt() + h["eps"]
        move = h["lr"] * (m1 / (1 - h["beta1"] ** step)) / den
        size = h["lr"] * ((h["beta1"] * m0).abs() + ((1 - h["beta1"]) * g).abs()) / (1 - h["beta1"] ** step) / den
        p1 = (1 - h["lr"] * h["weight_decay"]) * x[0].double() - move
        tol = 12 * 2.0 ** -24 * (x[0].double().abs() + size) + HALF[x[0].dtype] * p1.abs()
        # (where v' itself is below the normal fp32 numbers its root has no relative precision: with an eps that does not cover
        # that, sqrt(2 2^-149) = 2^-74 of the root against the denominator, the formula in 64 bits says nothing)
        known = (v1 >= 2.0 ** -120) | (den >= 2.0 ** -48)
        assert bool((((d[0].cpu().double() - p1).abs() <= tol) | ~known).all()), "tensor %d: parameters" % i
        if bits == 8:
            # (v is held in fp32 before its root is taken: two products that underflow by up to 2^-149 each are up to
            # sqrt(2 2^-149) < 2^-73 of the root; a block of m below 2^-100 is held as zeros)
            for k, s, exact, least, tiny in ((2, 4, m1, 0.5, 2.0 ** -100), (3, 5, v1.sqrt(), 1.0, 2.0 ** -73)):
                sc8 = rows(torch.ones(n, dtype=torch.float64)) * d[s].cpu().double()[:, None]
                sc8 = sc8.view(-1)[:n]
                off = (d[k].cpu().double() * sc8 - exact).abs()
                assert bool((off <= exact.abs() * (2.0 ** -4 + 2.0 ** -20) + least * 2.0 ** -9 * sc8 * (1 + 2.0 ** -20) + tiny).all())
    return dev


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", [[1], [255, 256, 257], [4096, 4095, 4097, 1, 3], [100003], [17 * (i + 1) for i in range(130)]])
def test_matches_the_formula_bit_for_bit(sizes, bits, dtype):
    step_and_check(make(sizes, dtype, bits, seed=sum(sizes)), step=5, bits=bits)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("shift", [1, 2, 3])
def test_any_alignment(shift, bits, dtype):
    step_and_check(make([1000, 4099], dtype, bits, seed=shift), step=1, bits=bits, shift=shift)


@pytest.mark.parametrize("bits", [32, 8])
def test_roots_and_quotients_of_every_mantissa(bits):
    """2^22 parameters of 0 that a step of size 1 moves to the quotient itself: gradients of every second mantissa over
    [2^-20, 2^-19) (their squares run through [1, 4) 2^-40), moments that make the quotient another one in every element; the
    last blocks hold zeros and values outside the range that has shorter sequences"""
    n = 1 << 22
    g = torch.from_numpy((np.arange(n, dtype=np.int32) * 2 + (107 << 23)).view(np.float32).copy())
    gen = torch.Generator().manual_seed(21)
    m, v = torch.randn(n, generator=gen) * 1e-6, torch.rand(n, generator=gen) * 1e-12
    g[-8 * BLOCK:-6 * BLOCK] *= 2.0 ** -60
    g[-6 * BLOCK:-4 * BLOCK] *= 2.0 ** 60
    g[-4 * BLOCK:] = 0
    m[-8 * BLOCK:], v[-8 * BLOCK:] = 0, 0
    ms = vs = None
    if bits == 8:
        (m, ms), (v, vs) = encode(rows(m), n), encode(rows(v.sqrt()), n, 2.0 ** -9)
    step_and_check([[torch.zeros(n), g, m, v, ms, vs]], 1, bits, hyper=dict(lr=0.5, beta1=0.5, beta2=0.75, eps=1e-30, weight_decay=0.0))


@pytest.mark.parametrize("bits", [32, 8])
def test_gradient_scale_from_the_host_and_from_the_device(bits):
    ts = make([3000], torch.float32, bits, seed=1)
    a = step_and_check(ts, 3, bits, scale=0.25)
    b = step_and_check(ts, 3, bits, scale=torch.tensor([0.25], device="cuda"))
    assert same(a[0][0], b[0][0])


@pytest.mark.parametrize("bits", [32, 8])
def test_zeros_and_vanishing_moments(bits):
    """no gradient yet (0 / eps), moments too small for a scale, a block with one value in it"""
    ts = make([BLOCK * 4], torch.float32, bits, seed=2)
    p, g, m, v, ms, vs = ts[0]
    g[:BLOCK * 3] = 0
    g[BLOCK] = 1e-3
    g[BLOCK * 2] = 1e-22
    if bits == 8:
        m[:BLOCK * 3], v[:BLOCK * 3] = 0, 0
        ms[:3], vs[:3] = 0, 0
    else:
        m[:BLOCK * 3], v[:BLOCK * 3] = 0, 0
        m[:BLOCK] = 1e-39
    step_and_check(ts, 1, bits)


def test_a_gradient_that_is_not_finite_poisons_its_block_and_no_other():
    from vc3d import ops
    for bad in (float("nan"), float("inf")):
        ts = make([BLOCK * 3], torch.float32, 8, seed=3)
        ts[0][1][BLOCK + 7] = bad
        dev = [[t.cuda() for t in x] for x in ts]
        ops.adamw_step(*[[c] for c in dev[0]], step=2, **HYPER)
        want = plain_step(*ts[0], 2, **HYPER)
        p, m = dev[0][0].cpu(), (rows(dev[0][2].float().cpu()) * dev[0][4].cpu()[:, None])
        ok = torch.tensor([True, False, True])
        assert torch.equal(torch.isfinite(m).all(1), ok) and not bool(torch.isfinite(m[1]).any())
        keep = torch.isfinite(p)
        assert int((~keep).sum()) == 1 and torch.equal(p[keep], want[0][keep])


def test_no_tensor_and_tensors_without_elements():
    from vc3d import ops
    ops.adamw_step([], [], [], [], step=1, **HYPER)
    ts = make([0, 5, 0], torch.float32, 32, seed=4)
    step_and_check(ts, 1, 32)


def test_dense_orders_and_refusals():
    from vc3d import ops
    from vc3d.capi import Vc3dError
    g = torch.Generator().manual_seed(5)
    p = torch.randn(4, 6, 3, 5, 7, generator=g).to(memory_format=torch.channels_last_3d)
    gr = torch.randn(4, 6, 3, 5, 7, generator=g).to(memory_format=torch.channels_last_3d)
    m, v = torch.zeros_like(p), torch.zeros_like(p)
    dev = [t.cuda() for t in (p, gr, m, v)]
    ops.adamw_step(*[[t] for t in dev], step=1, **HYPER)
    want = plain_step(p.permute(0, 2, 3, 4, 1), gr.permute(0, 2, 3, 4, 1), m.permute(0, 2, 3, 4, 1), v.permute(0, 2, 3, 4, 1), None, None, 1, **HYPER)
    assert same(dev[0].permute(0, 2, 3, 4, 1).contiguous(), want[0])
    x = [torch.zeros(8, 8, device="cuda") for _ in range(7)]
    call = lambda *a, **k: ops.adamw_step(*a, **{"step": 1, **HYPER, **k})  # noqa: E731
    ok = [[t] for t in x[:4]]
    half = torch.zeros(8, 8, device="cuda", dtype=torch.float16)
    for bad in ([[x[0]], [x[1].t()], [x[2]], [x[3]]], [[x[0][:, :4]], [x[1][:, :4]], [x[2][:, :4]], [x[3][:, :4]]],
                [[x[0], x[0]], [x[1], x[1]], [x[2], x[2]], [x[3], x[3]]], [[x[0]], [x[1].cpu()], [x[2]], [x[3]]],
                [[x[0]], [x[1].bfloat16()], [x[2]], [x[3]]], [[half], [half], [x[2]], [x[3]]], [[x[0]], [x[1][0]], [x[2]], [x[3]]],
                [[x[0]], [], [x[2]], [x[3]]], [x[:2], x[2:4], [x[4], x[4]], [x[5], x[6]]], [[x[0]], [x[1]], [x[2]], [x[2]]]):
        with pytest.raises(Vc3dError):
            call(*bad)
    for k in (dict(step=0), dict(beta1=1.0), dict(lr=-1.0), dict(eps=-1e-9), dict(weight_decay=-0.1)):
        with pytest.raises(Vc3dError):
            call(*ok, **k)
    codes = [torch.zeros(8, 8, device="cuda").to(torch.float8_e4m3fn) for _ in range(2)]
    with pytest.raises(Vc3dError):  # codes without scales, scales of the wrong length
        call([x[0]], [x[1]], [codes[0]], [codes[1]])
    with pytest.raises(Vc3dError):
        call([x[0]], [x[1]], [codes[0]], [codes[1]], [torch.zeros(2, device="cuda")], [torch.zeros(1, device="cuda")])
    torch.cuda.synchronize()


def test_a_captured_step_replays():
    """the tensors travel as kernel arguments: a captured step needs nothing from the host when it is replayed"""
    from vc3d import ops
    ts = make([5000, 3], torch.float32, 8, seed=6)
    dev = [[t.cuda() for t in x] for x in ts]
    twin = [[t.clone() for t in x] for x in dev]
    cols, tcols = ([list(c) for c in zip(*d)] for d in (dev, twin))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.adamw_step(*cols, step=4, **HYPER)
    for _ in range(3):
        for a, b in zip(cols[1], tcols[1]):
            a.mul_(-0.5), b.mul_(-0.5)
        graph.replay()
        ops.adamw_step(*tcols, step=4, **HYPER)
        torch.cuda.synchronize()
        assert all(same(a, b) for x, y in zip(dev, twin) for a, b in zip(x, y))


@pytest.mark.parametrize("bits", [32, 8])
def test_more_than_2_31_elements(bits):
    """the end of a long tensor moves as a short tensor of the same values does"""
    import vc3d
    n, tail = (1 << 31) + 300, 300  # (2^31 is whole blocks)
    g = torch.Generator().manual_seed(61)
    ends = [torch.randn(tail, generator=g).bfloat16().cuda() for _ in range(2)]
    out = []
    for size in (tail, n):
        p, gr = (torch.zeros(size, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        p[-tail:], gr[-tail:] = ends[0], ends[1]
        kind = torch.float32 if bits == 32 else torch.float8_e4m3fn
        m, v = (torch.zeros(size, dtype=kind, device="cuda") for _ in range(2))
        ms, vs = ([torch.zeros((size + 255) // 256, device="cuda")] if bits == 8 else None for _ in range(2))
        for step in (1, 2):
            vc3d.ops.adamw_step([p], [gr], [m], [v], ms, vs, lr=1e-2, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1, step=step)
        out.append([p[-tail:].clone(), m[-tail:].float(), v[-tail:].float()] + ([ms[0][-2:].clone(), vs[0][-2:].clone()] if bits == 8 else []))
        assert not bool(p[:-tail].any())
        del p, gr, m, v, ms, vs
    assert all(torch.equal(a, b) for a, b in zip(*out))

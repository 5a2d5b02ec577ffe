"""Linear classifier + cross-entropy (vc3d.linear_cross_entropy) against the definition in 64 bits, on the same (rounded) inputs.

Tolerances, element by element, from the roundings on the way.  A logit is a sum of D + 1 products in fp32: it is off by at most
dz = (D + 8) 2^-24 (|x| |w|^T + |b|), its largest value over a row taken.  The row's lse is off by as much, plus the rounding of
exp, of the sum over V terms and of log: de = (64 + V / 16) 2^-24 (the sum runs in 16 or more partial sums).  So the loss is off
by 2 dz + de + |loss| 2^-24, and a probability relatively by 2 dz + de.  P is rounded to the operands' type (half a step: h)
before the products dw = P^T x and dx = P w, whose sums run in fp32 over K terms: with Pa = |p| + onehot, a gradient is off by
  Pa^T |x| (2 dz + de + h + (K + 8) 2^-24) + h |gradient|      (h = 2^-8 for bf16, 2^-24 for fp32).
Where the forward keeps exponentials for the backward (keep_bytes), P is rounded twice (2 h + h^2), and is a product of two
exponentials, each off by its argument times 2^-24: below 64 each in these tests wherever p is not below 2^-90.  db then sums the
kept ones, rounded once, where it otherwise sums what no rounding has touched: h + h^2 beside the rest.
What underflows: exp and the matrix instructions take values below 2^-126 for 0, so a probability may be off by 2^-126 beside
all that, a gradient by K 2^-126 max|x| and itself by 2^-126 (words of a probability of 1e-39 show it)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
E = 2.0 ** -24
UNDER = 2.0 ** -126


def make(N, D, V, dtype, bias, seed=0, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, D, generator=g).to(dtype).cuda()
    w = (torch.randn(V, D, generator=g) * scale / D ** 0.5).to(dtype).cuda()
    b = (torch.randn(V, generator=g) * 0.5).to(dtype).cuda() if bias else None
    return x, w, b, torch.randint(0, V, (N,), generator=g).cuda()


def check(got, want, tol, what):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), "%s: %d elements off, worst %.3e where %.3e is allowed" % (
        what, int(bad.sum()), float(err[bad].max()), float(tol.expand_as(err)[bad][err[bad].argmax()]))


ALL = 1 << 40


def run_and_check(*args, keep=(0, ALL), **kw):
    """without and with kept exponentials"""
    for k in keep:
        out = run_and_check_one(*args, keep_bytes=k, **kw)
    return out


def run_and_check_one(x, w, b, y, reduction="mean", ignore=-100, dloss=None, keep_bytes=0):
    import vc3d
    leaves = [t.detach().requires_grad_() for t in (x, w) + ((b,) if b is not None else ())]
    loss = vc3d.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2] if b is not None else None, ignore_index=ignore, reduction=reduction,
                                     keep_bytes=keep_bytes)
    if dloss is None:
        dloss = torch.ones_like(loss)
    grads = torch.autograd.grad(loss, leaves, dloss)
    torch.cuda.synchronize()
    X, W, N, V, D = x.double(), w.double(), x.shape[0], w.shape[0], x.shape[1]
    keep = y != ignore
    X = torch.where(keep[:, None], X, torch.zeros_like(X))  # what an ignored row holds is nobody's business
    z, S = X @ W.t(), X.abs() @ W.abs().t()
    if b is not None:
        z, S = z + b.double(), S + torch.where(torch.isfinite(b), b, torch.zeros_like(b)).double().abs()
    dz = ((D + 8) * E * S).amax(1)
    de = (64 + V / 16) * E
    logp = torch.log_softmax(z, 1)
    at = torch.where(keep, y, torch.zeros_like(y))
    rows = torch.where(keep, -logp.gather(1, at[:, None])[:, 0], torch.zeros_like(dz))
    tol_rows = torch.where(keep, 2 * dz + de + rows.abs() * E, torch.zeros_like(dz))
    n = max(1, int(keep.sum()))
    if reduction == "none":
        check(loss, rows, tol_rows, "loss")
        gn = dloss.double()
    else:
        k = n if reduction == "mean" else 1
        check(loss, rows.sum() / k, tol_rows.sum() / k + rows.abs().sum() / k * E, "loss")
        gn = dloss.double().expand(N) / k
    gn = torch.where(keep, gn, torch.zeros_like(gn))
    p = logp.exp()
    hot = torch.zeros_like(p).scatter_(1, at[:, None], 1.0)
    P, Pa, rel = (p - hot) * gn[:, None], (p + hot) * gn.abs()[:, None], (2 * dz + de + 4 * E)[:, None]
    h = HALF[x.dtype]
    hp = h
    if keep_bytes:
        hp, rel = 2 * h + h * h, rel + 128 * E
    dx, dw = P @ W, P.t() @ X
    check(grads[0], dx, (Pa * (rel + hp + (V + 8) * E)) @ W.abs() + h * dx.abs() + UNDER * (1 + V * float(W.abs().max())), "dx")
    check(grads[1], dw, (Pa * (rel + hp + (N + 8) * E)).t() @ X.abs() + h * dw.abs() + UNDER * (1 + N * float(X.abs().max())), "dw")
    assert not bool(grads[0][~keep].any())
    if b is not None:
        db = P.sum(0)
        check(grads[2], db, (Pa * (rel + hp - h + (N + 8) * E)).sum(0) + h * db.abs() + UNDER * (1 + N), "db")
    return loss, grads


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,D,V,bias", [(1, 1, 1, True), (1, 64, 2, False), (2, 3, 5, True), (64, 512, 400, True), (7, 33, 129, False),
                                        (130, 65, 1000, True), (127, 128, 128, False), (128, 64, 127, True), (129, 96, 1025, False),
                                        (300, 200, 3001, True), (16, 2048, 5000, False), (1, 256, 20011, True), (513, 72, 257, True)])
def test_matches_the_definition(N, D, V, bias, dtype):
    x, w, b, y = make(N, D, V, dtype, bias, seed=N + D + V)
    run_and_check(x, w, b, y)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_reductions_ignored_rows_and_upstream_gradients(reduction, dtype):
    x, w, b, y = make(300, 96, 700, dtype, True, seed=1)
    g = torch.Generator().manual_seed(2)
    y[torch.rand(300, generator=g).cuda() < 0.4] = -100
    y[0] = y[299] = -100
    x[y == -100] = float("nan")  # padding holds anything
    d = torch.randn(300, generator=g).cuda() if reduction == "none" else torch.tensor(-3.5, device="cuda")
    run_and_check(x, w, b, y, reduction, dloss=d)


def test_another_ignore_index_and_leading_dimensions():
    import vc3d
    x, w, b, y = make(60, 32, 50, torch.float32, False, seed=3)
    y[::3] = 7
    run_and_check(x, w, b, y, "none", ignore=7)
    want = vc3d.linear_cross_entropy(x, w, y, reduction="none")
    got = vc3d.linear_cross_entropy(x.view(4, 15, 32), w, y.view(4, 15), reduction="none")
    assert got.shape == (4, 15) and torch.equal(got.view(-1), want)
    one = vc3d.linear_cross_entropy(x[1], w, y[1], reduction="none")  # a row by itself
    assert one.shape == () and abs(float(one) - float(want[1])) <= 64 * E * (1 + abs(float(want[1])))


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_no_row_counts(reduction):
    import vc3d
    x, w, b, y = make(70, 64, 300, torch.bfloat16, True, seed=4)
    y.fill_(-100)
    x.fill_(float("nan"))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    loss = vc3d.linear_cross_entropy(x, w, y, b, reduction=reduction)
    grads = torch.autograd.grad(loss.sum(), leaves)
    assert not bool(loss.any()) and not any(bool(g.any()) for g in grads)
    # and no row at all
    empty = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    loss = vc3d.linear_cross_entropy(empty, w, y[:0], b, reduction=reduction)
    grads = torch.autograd.grad(loss.sum(), [empty, w, b])
    assert grads[0].shape == (0, 64) and not any(bool(g.any()) for g in grads) and not bool(loss.any())


def test_labels_that_are_no_class_give_nan_in_their_row_alone():
    import vc3d
    x, w, b, y = make(40, 64, 300, torch.float32, False, seed=5)
    y[3], y[5] = 300, -1
    loss = vc3d.linear_cross_entropy(x, w, y, reduction="none")
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[3] = bad[5] = True
    assert torch.equal(torch.isnan(loss), bad)
    assert bool(torch.isnan(vc3d.linear_cross_entropy(x, w, y)))
    x.requires_grad_()
    dx, = torch.autograd.grad(loss_of(x, w, y), x)
    assert torch.equal(torch.isnan(dx).all(1), bad) and torch.equal(torch.isnan(dx).any(1), bad)


def loss_of(x, w, y):
    import vc3d
    return vc3d.linear_cross_entropy(x, w, y, reduction="none").sum()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_classes_masked_by_their_bias(dtype):
    """a bias of -inf or of the type's lowest value takes a class out: probability and gradients 0, whole tiles of them too"""
    for low in (-float("inf"), torch.finfo(dtype).min):
        x, w, b, y = make(50, 64, 700, dtype, True, seed=6)
        b[100:600] = low
        y = torch.where((y >= 100) & (y < 600), y % 100, y)
        _, grads = run_and_check(x, w, b, y)
        assert not bool(grads[1][100:600].any()) and not bool(grads[2][100:600].any())


def test_large_logits():
    """logits of +-1e4: the largest term is 1 and nothing overflows"""
    import vc3d
    x, w, b, y = make(33, 64, 500, torch.float32, False, seed=7, scale=1e4)
    loss = vc3d.linear_cross_entropy(x, w, y, reduction="none")
    z = x.double() @ w.double().t()
    want = torch.logsumexp(z, 1) - z.gather(1, y[:, None])[:, 0]
    tol = 2 * ((64 + 8) * E * (x.double().abs() @ w.double().abs().t())).amax(1) + (64 + 32) * E + want.abs() * E
    assert bool(((loss - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(dtype):
    """rows of wider buffers, odd offsets, columns first: the same values as from contiguous copies, to the bound"""
    import vc3d
    g = torch.Generator().manual_seed(8)
    big = torch.randn(200, 150, generator=g).to(dtype).cuda()
    y = torch.randint(0, 90, (60,), generator=g).cuda()
    for x, w in ((big[:60, 3:131], big[60:150, 1:129]), (big[:60, :128], big[60:150, :128]), (big[:128, :60].t(), big[:128, 60:150].t()),
                 (big[:120:2, 4:100], big[110:200, 20:116]), (big[:1, :64].expand(60, 64), big[:90, :64])):
        run_and_check(x, w, None, y)
    x, w = big[:60, :128], big[60:150, :128]
    b = torch.randn(90, generator=g).to(dtype).cuda()
    for keep in (0, ALL):
        for pick in range(3):  # gradients of one input alone
            leaves = [t.detach().clone().requires_grad_(i == pick) for i, t in enumerate((x, w, b))]
            both = [t.detach().clone().requires_grad_() for t in (x, w, b)]
            got, = torch.autograd.grad(vc3d.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2], keep_bytes=keep), leaves[pick])
            want = torch.autograd.grad(vc3d.linear_cross_entropy(both[0], both[1], y, both[2], keep_bytes=keep), both)[pick]
            assert torch.equal(got, want)


def test_the_plain_operators_refuse_layouts_that_they_cannot_read():
    import vc3d
    from vc3d.capi import Vc3dError
    x, w, b, y = make(40, 64, 90, torch.float32, True, seed=22)
    for bad in (dict(x=x.t()[:, :40].t()[:, ::2], w=w[:, :32]), dict(x=x[:1].expand(40, 64)), dict(w=w.t().contiguous().t()),
                dict(y=torch.stack((y, y), 1)[:, 0]), dict(b=torch.stack((b, b), 1)[:, 0])):
        a = {**dict(x=x, w=w, y=y, b=b), **bad}
        with pytest.raises(Vc3dError):
            vc3d.ops.linear_ce_fwd(a["x"], a["w"], a["y"], a["b"])
    loss, saved = vc3d.ops.linear_ce_fwd(x, w, y, b)
    for bad in (dict(saved=saved[:-1]), dict(dloss=loss.double()), dict(dloss=loss.cpu())):
        a = {**dict(saved=saved, dloss=loss), **bad}
        with pytest.raises(Vc3dError):
            vc3d.ops.linear_ce_bwd(x, w, y, b, a["saved"], a["dloss"])


def test_more_than_one_piece_of_the_vocabulary():
    """a batch long enough that the vocabulary goes by in several pieces (P of a piece is bounded)"""
    x, w, b, y = make(8192, 64, 40000, torch.bfloat16, True, seed=9)
    y[::5] = -100
    run_and_check(x, w, b, y)


def test_gradient_against_differences():
    """central differences along a random direction, fp32: truncation under eps^2 times the third derivative (softmax: below
    |dlogits|^3 / 4 < 2 with |dlogits| < 2 here), rounding of the loss (dz + de of the module's head) over eps"""
    import vc3d
    x, w, b, y = make(50, 32, 300, torch.float32, True, seed=10)
    g = torch.Generator().manual_seed(11)
    dirs = [torch.randn(t.shape, generator=g).cuda() * s for t, s in ((x, 0.1), (w, 0.02), (b, 0.1))]
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(vc3d.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2]), leaves)
    slope = sum(float((a.double() * d).sum()) for a, d in zip(grads, dirs))
    eps = 2.0 ** -5

    def value(s):
        return float(vc3d.linear_cross_entropy(x + s * dirs[0], w + s * dirs[1], y, b + s * dirs[2]))
    noise = (2 * 40 * E * float((x.abs() @ w.abs().t() + b.abs()).max()) + 96 * E) / eps
    assert abs((value(eps) - value(-eps)) / (2 * eps) - slope) <= 2 * eps ** 2 + noise


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["sum", "mean"])
def test_kept_exponentials_that_do_not_fit_their_type(reduction, dtype):
    """labels 44 nats and more behind another word, far enough that exp(z - z_label) overflows in one row: nothing of it is used"""
    for far in (60.0, 300.0):
        x, w, b, y = make(150, 64, 700, dtype, True, seed=20)
        b[:] = torch.where(torch.arange(700, device="cuda") == 650, torch.tensor(far, dtype=dtype, device="cuda"), b)
        y = torch.where(y == 650, y * 0, y)
        run_and_check(x, w, b, y, reduction)
        b[650] = 0
        x[77], x[:, 0] = 0, 0
        x[77, 0], w[650], w[650, 0], w[y[77], 0] = 8, 0, far / 8, 0  # one row alone
        run_and_check(x, w, b, y, reduction)
    y[3] = -100
    y[4] = 5
    b[5] = -float("inf")  # a label that is masked: loss inf, as torch has it
    import vc3d
    assert float(vc3d.linear_cross_entropy(x, w, y, b, reduction="sum", keep_bytes=ALL)) == float("inf")


def test_bad_labels_and_values_with_kept_exponentials():
    import vc3d
    x, w, b, y = make(40, 64, 300, torch.bfloat16, False, seed=5)
    y[3], y[5], y[7] = 300, -1, -100
    x[9, 3], x[7] = float("inf"), float("nan")
    got = []
    for keep in (0, ALL):
        leaves = [t.detach().clone().requires_grad_() for t in (x, w)]
        loss = vc3d.linear_cross_entropy(leaves[0], leaves[1], y, reduction="sum", keep_bytes=keep)
        bad = torch.zeros(40, dtype=torch.bool, device="cuda")
        bad[3] = bad[5] = bad[9] = True
        assert bool(torch.isnan(loss))
        dx, dw = torch.autograd.grad(loss, leaves)
        assert torch.equal(torch.isnan(dx).any(1), bad) and not bool(dx[7].any())
        got.append((dx, dw))
    assert all(torch.equal(torch.isnan(a), torch.isnan(b)) for a, b in zip(*got))


def test_what_is_kept():
    """the rule, the limit, nothing without a backward; a backward that is called twice"""
    import vc3d
    x, w, b, y = make(512, 512, 1 << 14, torch.bfloat16, False, seed=21)
    size = [vc3d.ops.linear_ce_fwd(x, w, y, keep_bytes=k)[1].numel() for k in (0, -1, 1 << 24, (1 << 24) - 1)]
    assert size[1] == size[2] == size[0] + (1 << 24) + (1 << 18) + 2 * 2048 and size[3] == size[0]
    assert vc3d.ops.linear_ce_fwd(x[:, :128], w[:, :128], y)[1].numel() < 1 << 20  # short rows: quicker computed again
    # rows that are no whole chunks: w is copied, and the copy kept where there is room for it too
    xo, wo = x[:, :511].contiguous(), w[:, :511].contiguous()
    one = torch.ones(1, device="cuda")
    got = []
    for k in (1 << 24, ALL):
        loss, saved = vc3d.ops.linear_ce_fwd(xo, wo, y, keep_bytes=k)
        got.append((saved.numel(), loss) + vc3d.ops.linear_ce_bwd(xo, wo, y, None, saved, one, keep_bytes=k))
    assert got[1][0] == got[0][0] + (1 << 14) * 1024 and all(torch.equal(a, b) for a, b in zip(got[0][1:4], got[1][1:4]))
    leaves = [t.requires_grad_() for t in (x, w)]
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    with torch.no_grad():
        loss = vc3d.linear_cross_entropy(x, w, y)
    torch.cuda.reset_peak_memory_stats()
    with torch.no_grad():
        loss = vc3d.linear_cross_entropy(x, w, y)
    assert torch.cuda.max_memory_allocated() - before < 1 << 22
    loss = vc3d.linear_cross_entropy(x, w, y)
    first = torch.autograd.grad(loss, leaves, retain_graph=True)
    again = torch.autograd.grad(loss, leaves)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("keep", [0, ALL])
def test_streams_and_repeats_bit_for_bit(keep):
    import vc3d
    x, w, b, y = make(700, 128, 3000, torch.bfloat16, True, seed=12)
    y[::7] = -100
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def once():
        loss = vc3d.linear_cross_entropy(x, w, y, b, keep_bytes=keep)
        return (loss.detach(),) + torch.autograd.grad(loss, leaves)
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


@pytest.mark.parametrize("keep", [0, ALL])
def test_captured_graphs_replay(keep):
    import vc3d
    x, w, b, y = make(300, 128, 1500, torch.bfloat16, True, seed=13)
    one = torch.ones(1, device="cuda")

    def once(y):
        loss, saved = vc3d.ops.linear_ce_fwd(x, w, y, b, keep_bytes=keep)
        return (loss,) + vc3d.ops.linear_ce_bwd(x, w, y, b, saved, one, keep_bytes=keep)
    ins = [y.clone(), y.flip(0).contiguous()]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for t in ins:
            once(t)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for t in ins:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(once(t))
        graphs.append(graph)
    for rep in range(3):
        for k, t in enumerate(ins):  # another number of rows that count in every replay
            t[rep * 50 + k:rep * 50 + 90] = -100
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for t, out in zip(ins, outs):
            assert all(torch.equal(a, b) for a, b in zip(once(t), out))


@pytest.mark.parametrize("keep", [0, ALL])
def test_more_than_2_31_logits(keep):
    """33000 rows of 66000 words: offsets into the kept gradient of the logits pass 2^31 elements; the last rows and words"""
    import vc3d
    N, D, V, last = 33000, 64, 66000, 50
    x, w, b, y = make(N, D, V, torch.bfloat16, True, seed=51, scale=1.0)
    y[::9] = -100
    leaves = [t.requires_grad_() for t in (x, w, b)]
    loss = vc3d.linear_cross_entropy(x, w, y, b, keep_bytes=keep)
    dx, dw, db = torch.autograd.grad(loss, leaves)
    X, W, B = x.detach().double(), w.detach().double(), b.detach().double()
    kept = y != -100
    at = torch.where(kept, y, torch.zeros_like(y))
    n = int(kept.sum())
    lse = torch.cat([torch.logsumexp(X[i:i + 3000] @ W.t() + B, 1) for i in range(0, N, 3000)])
    rows = torch.where(kept, lse - ((X * W[at]).sum(1) + B[at]), torch.zeros_like(lse))
    S = float((X.abs().amax(0) * W.abs().amax(0)).sum() + B.abs().max())  # of |x| |w| + |b|, over all
    rel = 2 * (D + 8) * E * S + (64 + V / 16) * E + 128 * E
    check(loss, rows.sum() / n, torch.tensor(rel, device="cuda") + rows.abs().sum() / n * E, "loss")
    h = HALF[torch.bfloat16]
    hp = 2 * h + h * h
    for what, got, r, v in (("dx", dx[-last:], slice(N - last, N), slice(0, V)), ("dw", dw[-last:], slice(0, N), slice(V - last, V))):
        p = (X[r] @ W[v].t() + B[v] - lse[r, None]).exp()
        hot = at[r, None] == torch.arange(V, device="cuda")[v]
        P, Pa = [torch.where(kept[r, None], q / n, torch.zeros_like(p)) for q in (p - hot.double(), p + hot.double())]
        want = P @ W[v] if what == "dx" else P.t() @ X[r]
        size = Pa @ W[v].abs() if what == "dx" else Pa.t() @ X[r].abs()
        check(got, want, size * (rel + hp + (max(N, V) + 8) * E) + h * want.abs() + UNDER * max(N, V) * 8, what)
        if what == "dw":
            want = P.sum(0)
            check(db[-last:], want, Pa.sum(0) * (rel + hp + (N + 8) * E) + h * want.abs() + UNDER * N, "db")

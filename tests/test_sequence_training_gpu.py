"""The gated scan, the linear cross-entropy and AdamW as they are used: a recurrent classifier over sequences trained for a step,
the model's recurrent head and fused head loss, the optimizer class.

Tolerances: bf16 operands, gates and gradients round by up to 2^-8 each (2^-9.8 on average); along the longest path (input,
weight, gates, h, logits' operands, P, dgates and the projection's operands) eight such roundings add up, independent of each
other, to sqrt(8) 2^-9.8 = 3.2e-3 of a gradient's 2-norm; what is compared is below 1e-2.  fp32 paths: sums of up to 2^11 terms
in another order, 2^-24 sqrt(2^11) < 3e-6 of the 2-norm; 1e-5."""
import numpy as np
import pytest
import torch

from helpers import make_config, rel_l2
from test_adamw_gpu import plain_step, same

pytestmark = pytest.mark.gpu


def reference(x, W, b, h0, head, hb, y, lengths):
    """the classifier in 64 bits on the CPU -> loss, gradients of (W, b, head, hb)"""
    leaves = [t.detach().double().cpu().requires_grad_() for t in (W, b, head, hb)]
    x, h0 = x.detach().double().cpu(), h0.detach().double().cpu()
    z = x @ leaves[0].t() + leaves[1]
    H = z.shape[2] // 2
    hs = []
    h = h0
    for t in range(x.shape[1]):
        f = torch.sigmoid(z[:, t, :H])
        h = torch.where((t < lengths)[:, None], f * h + (1 - f) * z[:, t, H:], h)
        hs.append(h)
    h = torch.stack(hs, 1)
    logits = h @ leaves[2].t() + leaves[3]
    loss = torch.nn.functional.cross_entropy(logits.reshape(-1, logits.shape[2]), y.cpu().reshape(-1), ignore_index=-100)
    return float(loss.detach()), torch.autograd.grad(loss, leaves)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_training_step_of_a_recurrent_classifier(bits):
    """gate projection -> scan over padded sequences -> cross-entropy over 5000 classes without logits -> AdamW"""
    import vc3d
    from models.recurrence import GatedScan
    from vc3d.optim import AdamW
    B, T, F, H, V = 6, 150, 128, 192, 5000
    g = torch.Generator().manual_seed(1)
    torch.manual_seed(2)
    cell = GatedScan(F, H).cuda()
    head = torch.nn.Linear(H, V).cuda()
    with torch.no_grad():
        for p in (cell.gates.weight, head.weight):
            p.copy_(p.bfloat16().float())
    x = torch.randn(B, T, F, generator=g).bfloat16().float().cuda()
    h0 = torch.randn(B, H, generator=g).cuda()
    lengths = torch.tensor([150, 1, 77, 128, 0, 64])
    y = torch.randint(0, V, (B, T), generator=g)
    y[torch.arange(T)[None, :] >= lengths[:, None]] = -100
    y = y.cuda()
    params = [cell.gates.weight, cell.gates.bias, head.weight, head.bias]
    opt = AdamW(params, lr=1e-2, weight_decay=0.1, state_bits=bits)
    for step in (1, 2):
        before = [p.detach().clone() for p in params]
        held = [{k: v.clone() for k, v in opt.state[p].items() if torch.is_tensor(v)} if opt.state[p] else None for p in params]
        opt.zero_grad()
        h, last = cell.sequence(x, lengths.cuda(), h0)
        loss = vc3d.linear_cross_entropy(h.bfloat16(), head.weight.bfloat16(), y, head.bias.bfloat16())
        loss.backward()
        versions = [p._version for p in params]
        opt.step()
        torch.cuda.synchronize()
        assert all(p._version > v for p, v in zip(params, versions))  # what caches weights by version sees the step
        if step == 1:
            want, grads = reference(x, before[0], before[1], h0, before[2], before[3], y, lengths)
            assert abs(float(loss.detach()) - want) <= 1e-2 * want
            for p, e in zip(params, grads):
                assert rel_l2(p.grad, e) <= 1e-2
        # the step itself, bit for bit, from the gradients that it was given
        for p, b4, st in zip(params, before, held):
            n = p.numel()
            if st is None:
                zero = torch.zeros(n)
                m = v = zero if bits == 32 else zero.to(torch.float8_e4m3fn)
                ms = vs = None if bits == 32 else torch.zeros((n + 255) // 256)
            else:
                m, v = st["exp_avg"].cpu().view(-1), st["exp_avg_sq"].cpu().view(-1)
                ms, vs = (st[k].cpu() if bits == 8 else None for k in ("exp_avg_scale", "exp_avg_sq_scale"))
            want = plain_step(b4.cpu().view(-1), p.grad.cpu().view(-1), m, v, ms, vs, step, 1e-2, 0.9, 0.999, 1e-8, 0.1)
            assert same(p.detach(), want[0]) and same(opt.state[p]["exp_avg"], want[1]) and same(opt.state[p]["exp_avg_sq"], want[2])


def test_sequence_is_the_steps_and_steps_keep_the_state():
    from models.recurrence import GatedScan
    torch.manual_seed(3)
    cell = GatedScan(64, 64).cuda()
    x = torch.randn(5, 20, 64, device="cuda")
    with torch.no_grad():
        h, last = cell.sequence(x)
        cell.reset(5)
        outs = []
        for t in range(20):
            outs.append(cell(x[:, t]))
    # one state in fp32 either way; sequence() rounds its h to the gates' bf16
    assert float((outs[-1] - last).abs().max()) <= 20 * 32 * 2.0 ** -24 * float(last.abs().max() + 1)
    assert rel_l2(h, torch.stack(outs, 1)) <= 2.0 ** -8
    assert not torch.equal(outs[0], outs[1])  # a step does not write into what the step before returned
    # with gradients: a step's loss reaches the parameters, the state that is kept is detached
    cell.reset(5)
    out = cell(x[:, 0])
    out.sum().backward()
    assert cell.gates.weight.grad is not None and not cell.h.requires_grad and rel_l2(out, outs[0]) <= 1e-6


def test_fused_head_loss_is_the_plain_one():
    """HeadScores and Loss on the same features: the same loss and gradients as scores and Loss, to fp32's order of sums"""
    import vc3d
    from core.loss import Loss
    criterion = Loss(make_config(18, 37))
    torch.manual_seed(4)
    head = torch.nn.Linear(512, 37).cuda()
    feat, y = torch.randn(6, 512, device="cuda", requires_grad=True), torch.tensor([3, 36, 0, 3, 9, 20], device="cuda")
    got = []
    for fused in (False, True):
        score = vc3d.HeadScores(feat, head.weight, head.bias)
        if not fused:
            score = score.scores()
        loss = criterion(score, y, None, None)
        got.append((loss.detach(),) + torch.autograd.grad(loss * 3.0, (feat, head.weight, head.bias)))
    for a, b in zip(*got):
        assert rel_l2(b, a) <= 1e-5


@pytest.mark.parametrize("use_lstm", [False, True])
def test_fused_head_loss_in_the_model(use_lstm, det_mode):
    """MODEL.FUSED_HEAD_LOSS through create_model, both heads: gradients of all parameters arrive where the plain loss's do;
    eval gives scores.  (BatchNorm's sums are taken relative to the previous forward's mean, so a forward repeats an earlier
    one's features up to bf16 roundings only: loss and gradients are compared to the bar of those, 3e-2; the operator itself is
    compared above.)"""
    from core.loss import Loss
    from models.model import create_model
    cfg = make_config(18, 37)
    cfg.MODEL.USE_LSTM, cfg.MODEL.LSTM_OUTDIM = use_lstm, 128
    cfg.MODEL.RECURRENT_CELL = "scan"
    torch.manual_seed(4)
    model = create_model(cfg, True).cuda().train()
    x, y = torch.randn(4, 3, 8, 64, 64, device="cuda"), torch.tensor([3, 36, 0, 3], device="cuda")
    criterion = Loss(cfg)
    got = []
    for fused in (False, False, True):
        model.fused_head_loss = fused
        model.zero_grad(set_to_none=True)
        if use_lstm:
            model.lstm.reset(4)
        action, score, value = model(x)
        assert torch.is_tensor(score) != fused
        loss = criterion(score, y, None, None)
        loss.backward()
        got.append({"loss": loss.detach().clone(), **{k: p.grad.clone() for k, p in model.named_parameters() if p.grad is not None}})
    assert set(got[1]) == set(got[2]) and len(got[1]) > 60
    head = {k for k in got[1] if not k.startswith("backbone")}
    assert all(rel_l2(got[2][k], got[1][k]) <= 3e-2 for k in head), {k: rel_l2(got[2][k], got[1][k]) for k in head}
    model.eval()
    with torch.no_grad():
        assert torch.is_tensor(model(x)[1])


@pytest.mark.parametrize("opt_name,bits", [("adamw", 8), ("adamw", 32), ("adam", 32), ("sgd", 32)])
def test_train_loop_with_the_new_options(opt_name, bits):
    """core.function.train with the fused head loss and each optimizer: parameters of head and backbone move, all finite"""
    from core.function import train
    from core.loss import Loss
    from models.model import create_model
    from utils.utils import create_optimizer
    from vc3d.optim import AdamW
    cfg = make_config(18, 11, OPTIMIZER=opt_name, LR=1e-3, TRAIN_STEP=3, PRINT_EVERY=100, STATE_BITS=bits)
    cfg.MODEL.FUSED_HEAD_LOSS = True
    torch.manual_seed(5)
    model = create_model(cfg, True).cuda()
    opt = create_optimizer(cfg, model)
    assert isinstance(opt, AdamW) == (opt_name == "adamw")
    before = {k: v.detach().clone() for k, v in model.named_parameters()}
    x, y = torch.randn(4, 3, 8, 64, 64), torch.tensor([1, 2, 10, 0])
    train(cfg, [(x, y)], model, Loss(cfg), opt, 0)
    torch.cuda.synchronize()
    for k, p in model.named_parameters():
        assert bool(torch.isfinite(p).all()) and not torch.equal(p, before[k]), k


def test_adamw_class_matches_torch_adamw():
    """32-bit moments, several groups, a parameter without a gradient, weights in channels_last order, a changed learning rate:
    torch.optim.AdamW in 64 bits; per step 12 roundings of half a step (tests/test_adamw_gpu.py), 5 steps"""
    from vc3d.optim import AdamW
    g = torch.Generator().manual_seed(6)
    ps = [torch.randn(33, 7, generator=g), torch.randn(5, generator=g), torch.randn(8, 6, 3, 3, 3, generator=g).to(memory_format=torch.channels_last_3d),
          torch.randn((), generator=g), torch.randn(4, 4, generator=g)]
    mine = [torch.nn.Parameter(p.cuda()) for p in ps]
    ref = [torch.nn.Parameter(p.double()) for p in ps]
    groups = lambda q: [dict(params=q[:2], lr=1e-2, weight_decay=0.1), dict(params=q[2:])]  # noqa: E731
    a, b = AdamW(groups(mine), lr=1e-3), torch.optim.AdamW(groups(ref), lr=1e-3)
    for step in range(5):
        for m, r in zip(mine[:4], ref[:4]):
            gr = torch.randn(m.shape, generator=g)
            m.grad, r.grad = gr.cuda(), gr.double()  # (contiguous, also for the channels_last parameter)
        a.step(), b.step()
        for o in (a, b):
            o.param_groups[0]["lr"] *= 0.5
    for m, r, p in zip(mine, ref, ps):
        assert float((m.detach().cpu().double() - r.detach()).abs().max()) <= 5 * 12 * 2.0 ** -24 * (float(p.abs().max()) + 1)
    assert torch.equal(mine[4].detach().cpu(), ps[4]) and not a.state[mine[4]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_state_survives_saving(bits, dtype, tmp_path):
    """a run that is saved, loaded into a new optimizer and continued gives the bits of one that was not interrupted"""
    from vc3d.capi import Vc3dError
    from vc3d.optim import AdamW
    g = torch.Generator().manual_seed(7)
    start = [torch.randn(300, 5, generator=g).to(dtype), torch.randn(77, generator=g).to(dtype)]
    grads = [[torch.randn(p.shape, generator=g).to(dtype).cuda() for p in start] for _ in range(4)]

    def run(ps, opt, steps):
        for k in steps:
            for p, gr in zip(ps, grads[k]):
                p.grad = gr.clone()
            opt.step()
    one = [torch.nn.Parameter(p.cuda()) for p in start]
    oa = AdamW(one, lr=1e-2, state_bits=bits)
    run(one, oa, range(4))
    two = [torch.nn.Parameter(p.cuda()) for p in start]
    ob = AdamW(two, lr=1e-2, state_bits=bits)
    run(two, ob, range(2))
    torch.save(ob.state_dict(), tmp_path / "opt.pth")
    three = [torch.nn.Parameter(p.detach().clone()) for p in two]
    oc = AdamW(three, lr=1e-2, state_bits=bits)
    oc.load_state_dict(torch.load(tmp_path / "opt.pth", weights_only=True))
    run(three, oc, range(2, 4))
    for p, q in zip(one, three):
        assert torch.equal(p.detach(), q.detach())
        assert all(same(oa.state[p][k], oc.state[q][k]) and oa.state[p][k].dtype == oc.state[q][k].dtype for k in oa.state[p] if k != "step")
    with pytest.raises(Vc3dError):
        AdamW(three, state_bits=40 - bits).load_state_dict(ob.state_dict())


def test_a_run_begun_with_torch_adamw_goes_on():
    """torch.optim.AdamW's state is taken over (fp32 moments, its step count); one step on: torch's own, to its roundings"""
    from vc3d.capi import Vc3dError
    from vc3d.optim import AdamW
    g = torch.Generator().manual_seed(17)
    p = [torch.nn.Parameter(torch.randn(40, 7, generator=g).cuda()), torch.nn.Parameter(torch.randn(5, generator=g).cuda())]
    theirs = torch.optim.AdamW(p, lr=1e-2)
    for _ in range(3):
        for q in p:
            q.grad = torch.randn(q.shape, generator=g).cuda()
        theirs.step()
    mine_p = [torch.nn.Parameter(q.detach().clone()) for q in p]
    mine = AdamW(mine_p, lr=1e-2)
    mine.load_state_dict(theirs.state_dict())
    assert all(mine.state[q]["step"] == 3 for q in mine_p)
    for q, r in zip(p, mine_p):
        q.grad = torch.randn(q.shape, generator=g).cuda()
        r.grad = q.grad.clone()
    theirs.step()
    mine.step()
    for q, r in zip(p, mine_p):
        # both round each of some ten operations on values of at most |p| + 2 lr (|m'| <= 2 r at step 4)
        assert bool(((q - r).abs() <= 10 * 2.0 ** -24 * (q.abs() + 0.02)).all())
    with pytest.raises(Vc3dError):
        AdamW(mine_p, lr=1e-2, state_bits=8).load_state_dict(theirs.state_dict())
    with pytest.raises(Vc3dError):
        mine.load_state_dict(torch.optim.AdamW(p, amsgrad=True).state_dict())


def test_adamw_refuses_to_be_captured():
    from vc3d.capi import Vc3dError
    from vc3d.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    p.grad = torch.ones_like(p)
    opt = AdamW([p])
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = torch.zeros(8, device="cuda") + 1
        with pytest.raises(Vc3dError):
            opt.step()
    graph.replay()
    torch.cuda.synchronize()
    assert opt.state[p]["step"] == 1 and bool((q == 1).all())
    p.grad = torch.sparse_coo_tensor(torch.tensor([[1]]), torch.tensor([1.0]), (8,)).cuda()
    with pytest.raises(Vc3dError):
        opt.step()


def test_clipping_by_a_scale_on_the_device():
    """a clipping factor that never visits the host: the same bits as scaling by the number"""
    from vc3d.optim import AdamW
    g = torch.Generator().manual_seed(8)
    start, gr = torch.randn(1000, generator=g), torch.randn(1000, generator=g)
    out = []
    for kind in range(2):
        p = torch.nn.Parameter(start.cuda())
        p.grad = gr.cuda()
        scale = (1.0 / p.grad.norm()).float().reshape(1)
        AdamW([p], lr=1e-2).step(grad_scale=scale if kind else float(scale))
        out.append(p.detach())
    assert torch.equal(out[0], out[1])


@pytest.mark.parametrize("op", ["scan", "lce"])
def test_public_entries_captured_with_their_backward(op):
    """forward and backward through autograd in one graph, replayed with new inputs between eager work on other leaves.  (The
    leaves' own eager graphs are gone when the capture begins.)"""
    import vc3d
    g = torch.Generator().manual_seed(31)
    lengths = torch.tensor([500, 0, 700], dtype=torch.int32).cuda()
    if op == "scan":
        leaves = [torch.randn(3, 700, 160, generator=g).cuda(), torch.randn(3, 80, generator=g).cuda()]
        up = torch.randn(3, 700, 80, generator=g).cuda()

        def once(a, b):
            h, last = vc3d.gated_scan(a, b, lengths=lengths)
            return (h.detach(), last.detach()) + torch.autograd.grad((h, last), (a, b), (up, last.detach()))
    else:
        leaves = [torch.randn(600, 512, generator=g).bfloat16().cuda(), (torch.randn(16000, 512, generator=g) / 16).bfloat16().cuda()]
        y = torch.randint(0, 16000, (600,), generator=g).cuda()

        def once(a, b):
            loss = vc3d.linear_cross_entropy(a, b, y)
            return (loss.detach(),) + torch.autograd.grad(loss, (a, b))
    leaves = [t.requires_grad_() for t in leaves]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            once(*leaves)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once(*leaves)
    for rep in range(3):
        with torch.no_grad():
            for t in leaves:
                t.copy_(torch.randn(t.shape, generator=g) * (0.5 + rep) / (1 if op == "scan" else 4))
        want = once(*[t.detach().clone().requires_grad_() for t in leaves])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("op", ["scan", "lce"])
def test_a_gradient_of_a_gradient_is_refused(op):
    import vc3d
    x = torch.randn(4, 6, 8, device="cuda", requires_grad=True)
    if op == "scan":
        out = vc3d.gated_scan(x)[0].sum()
    else:
        out = vc3d.linear_cross_entropy(x, torch.randn(10, 8, device="cuda"), torch.zeros(4, 6, dtype=torch.int64, device="cuda"))
    first, = torch.autograd.grad(out, x, create_graph=True)
    assert bool(torch.isfinite(first).all())
    with pytest.raises(RuntimeError, match="once"):
        first.sum().backward(retain_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), x)


def test_errors_reach_the_caller_as_this_package_s():
    import vc3d
    from vc3d.capi import Vc3dError
    g = torch.zeros(2, 3, 8, device="cuda")
    x, w, y = torch.zeros(4, 8, device="cuda"), torch.zeros(10, 8, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    for call in (lambda: vc3d.gated_scan(g.half()), lambda: vc3d.gated_scan(g[0]), lambda: vc3d.gated_scan(g[..., :7]),
                 lambda: vc3d.gated_scan(g, torch.zeros(2, 3, device="cuda")), lambda: vc3d.gated_scan(g, torch.zeros(2, 4)),
                 lambda: vc3d.gated_scan(g, torch.zeros(2, 4, device="cuda").bfloat16()), lambda: vc3d.gated_scan(g, lengths=[1, 2]),
                 lambda: vc3d.gated_scan(g, lengths=torch.zeros(3, dtype=torch.int32, device="cuda")),
                 lambda: vc3d.gated_scan(g, lengths=torch.zeros(2, dtype=torch.int32)), lambda: vc3d.gated_scan(3),
                 lambda: vc3d.gated_scan_step(g[0], torch.zeros(3, 3, device="cuda")), lambda: vc3d.gated_scan_step(g[0].t(), torch.zeros(8, 1, device="cuda")),
                 lambda: vc3d.gated_scan_step(g[0], torch.zeros(3, 8, device="cuda")[:, ::2]),
                 lambda: vc3d.linear_cross_entropy(x, w.bfloat16(), y), lambda: vc3d.linear_cross_entropy(x, w[:, :4], y),
                 lambda: vc3d.linear_cross_entropy(x, w, y[:3]), lambda: vc3d.linear_cross_entropy(x, w, y.int()),
                 lambda: vc3d.linear_cross_entropy(x, w, y.cpu()), lambda: vc3d.linear_cross_entropy(x, w[:0], y),
                 lambda: vc3d.linear_cross_entropy(x, w, y, torch.zeros(9, device="cuda")), lambda: vc3d.linear_cross_entropy(x, w, y, reduction="avg"),
                 lambda: vc3d.linear_cross_entropy(x.requires_grad_(), w, y, keep_bytes=-2), lambda: vc3d.linear_cross_entropy(x.half(), w.half(), y)):
        with pytest.raises(Vc3dError):
            call()

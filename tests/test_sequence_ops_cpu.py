"""What the gated scan, the linear cross-entropy and the multi-tensor AdamW refuse, and what they answer without a GPU: the
Python side's checks, the C entries' argument checks (each is refused before any launch), workspace sizes, the config keys and
the optimizer factory."""
import ctypes
import os
import sys

import pytest
import torch

from helpers import make_config

PTR = 0x10000  # never read on the host


def _capi():
    from vc3d import capi
    return capi


def test_there_is_no_cpu_path():
    import vc3d
    from vc3d import ops
    from vc3d.capi import Vc3dError
    from vc3d.optim import AdamW
    from vc3d.scan import PackedGateWeight, gate_projection
    x, w, y = torch.zeros(4, 8), torch.zeros(16, 8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: vc3d.gated_scan(torch.zeros(1, 2, 4)), lambda: vc3d.gated_scan_step(torch.zeros(1, 4), torch.zeros(1, 2)),
                 lambda: vc3d.linear_cross_entropy(x, w, y), lambda: ops.linear_ce_fwd(x, w, y), lambda: ops.gated_scan_fwd(torch.zeros(1, 2, 4)),
                 lambda: gate_projection(torch.zeros(2, 64), torch.zeros(64, 64), None, PackedGateWeight()),
                 lambda: ops.adamw_step([x], [x], [x], [x], lr=1, beta1=0, beta2=0, eps=0, weight_decay=0, step=1)):
        with pytest.raises(Vc3dError):
            call()
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    with pytest.raises(Vc3dError):
        AdamW([p]).step()
    for bad in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-1.0)):
        with pytest.raises(Vc3dError):
            AdamW([p], **bad)


def test_c_entry_of_the_scan_refuses():
    c = _capi()
    ok = lambda **k: c.ScanDesc(**{**dict(B=2, T=100, H=8, is_bf16=1, reverse=0, pad_=0, stride_b=1600, stride_t=16), **k})  # noqa: E731
    need = c.lib.vc_gated_scan_workspace_bytes
    assert need(ok(), 0) == 0 and need(ok(T=100000), 0) > 0 and need(ok(T=100000), 1) > need(ok(T=10000), 1) > 0
    assert need(None, 0) == 0 and need(ok(H=0), 0) == 0
    fwd = lambda d, g=PTR, h=PTR, last=PTR, ws=None, n=0: c.lib.vc_gated_scan_fwd(d, g, None, None, h, last, None, ws, n, None)  # noqa: E731
    bwd = lambda d, g=PTR, st=PTR, dy=PTR, dg=PTR, ws=None, n=0: c.lib.vc_gated_scan_bwd(d, g, None, st, dy, None, dg, None, ws, n, None)  # noqa: E731
    for bad in (None, ok(B=0), ok(T=0), ok(H=0), ok(T=-1), ok(B=65536), ok(T=(1 << 30) + 1), ok(B=65535, T=1 << 30, H=1 << 24)):
        assert fwd(bad) == -2 and bwd(bad) == -2
        assert c.lib.vc_last_error()
    for bad in (dict(g=None), dict(h=None), dict(last=None), dict(h=PTR + 2)):
        assert fwd(ok(), **bad) == -2
    for bad in (dict(g=None), dict(st=None), dict(dg=None), dict(dg=PTR + 2), dict(dy=PTR + 2)):
        assert bwd(ok(), **bad) == -2
    assert fwd(ok(is_bf16=0), h=PTR + 4) == -2
    long = ok(T=100000)
    for run, op in ((fwd, 0), (bwd, 1)):  # no workspace, a short one, one at an odd address
        n = need(long, op)
        assert run(long) == -2 and run(long, ws=PTR, n=n - 1) == -2 and run(long, ws=PTR + 8, n=n) == -2
        assert b"workspace" in c.lib.vc_last_error()
    for bad in ((None, PTR, PTR, 1, 8), (PTR, None, PTR, 1, 8), (PTR, PTR, None, 1, 8), (PTR, PTR, PTR, 0, 8), (PTR, PTR, PTR, 1, 0)):
        g, st, h, B, H = bad
        assert c.lib.vc_gated_scan_step(g, 16, 1, st, h, B, H, None) == -2


def test_c_entry_of_the_linear_cross_entropy_refuses():
    c = _capi()
    base = dict(N=100, D=64, V=1000, is_bf16=1, reduction=1, w_align=0, ldx=64, ldw=64, ignore_index=-100, keep_bytes=-1)
    ok = lambda **k: c.LinearCeDesc(**{**base, **k})  # noqa: E731
    need = c.lib.vc_linear_ce_workspace_bytes
    big = 1 << 30
    fwd = lambda d, x=PTR, w=PTR, y=PTR, loss=PTR, saved=PTR, ws=PTR, n=big: c.lib.vc_linear_ce_fwd(  # noqa: E731
        d, x, w, None, y, loss, saved, ws, n, None)
    bwd = lambda d, x=PTR, w=PTR, b=None, y=PTR, saved=PTR, g=PTR, dx=PTR, dw=PTR, db=None, ws=PTR, n=big: c.lib.vc_linear_ce_bwd(  # noqa: E731
        d, x, w, b, y, saved, g, dx, dw, db, ws, n, None)
    for bad in (None, ok(N=0), ok(D=0), ok(V=0), ok(N=(1 << 23) + 1), ok(V=(1 << 23) + 1), ok(ldx=63), ok(ldw=63), ok(reduction=3),
                ok(reduction=-1), ok(w_align=16), ok(w_align=-1), ok(keep_bytes=-2)):
        assert fwd(bad) == -2 and bwd(bad) == -2 and need(bad, 0) == 0 and c.lib.vc_linear_ce_saved_bytes(bad) == 0
    for bad in (dict(x=None), dict(w=None), dict(y=None), dict(saved=None), dict(saved=PTR + 16), dict(ws=None), dict(ws=PTR + 16), dict(n=16)):
        assert fwd(ok(), **bad) == -2 and bwd(ok(), **bad) == -2
    assert bwd(ok(), dx=PTR + 8) == -2 and bwd(ok(), dw=PTR + 2) == -2 and b"aligned" in c.lib.vc_last_error()
    assert fwd(ok(), loss=None) == -2 and bwd(ok(), g=None) == -2 and bwd(ok(), db=PTR) == -2
    assert fwd(ok(), w=PTR + 2) == -2 and b"modulo 16" in c.lib.vc_last_error()  # the descriptor says that w is aligned
    # what is left for the backward: a few words a row, copies of x while they are small
    assert c.lib.vc_linear_ce_saved_bytes(ok()) >= 100 * 8 + 100 * 128 and c.lib.vc_linear_ce_saved_bytes(ok(N=1 << 20, D=512, ldx=512, ldw=512, keep_bytes=0)) < 16 << 20
    assert c.lib.vc_linear_ce_saved_bytes(ok(keep_bytes=1 << 20)) >= 100 * 1000 * 2
    # no N x V block: one piece's P, sums of dx, a pair for every row and tile
    n = need(ok(N=8192, D=2048, V=1 << 20, ldx=2048, ldw=2048), 1)
    assert n < 1.2e9 and n < 8192 * (1 << 20) * 2 / 10
    assert need(ok(N=8192, D=2048, V=1 << 20, ldx=2048, ldw=2048), 0) < 8192 * (1 << 20) * 2 / 40
    # rows that are no whole 16-byte chunks: room for the copies of a piece
    assert need(ok(D=63), 0) > need(ok(), 0) and need(ok(ldw=65), 1) > need(ok(), 1) and need(ok(w_align=2), 1) > need(ok(), 1)


def test_c_entry_of_adamw_refuses():
    c = _capi()
    step = c.lib.vc_adamw_step
    h = lambda **k: c.AdamwHyper(**{**dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, grad_scale=1.0, step=1), **k})  # noqa: E731
    t = lambda *a: (ctypes.c_int64 * 7)(*a)  # noqa: E731
    good = t(PTR, PTR, PTR, PTR, PTR, PTR, 10)
    assert step(None, 0, 0, 32, h(), None, None) == 0  # nothing to do
    assert step(t(0, 0, 0, 0, 0, 0, 0), 1, 0, 8, h(), None, None) == 0
    assert step(good, 1, 0, 32, None, None, None) == -2 and step(None, 1, 0, 32, h(), None, None) == -2 and step(good, -1, 0, 32, h(), None, None) == -2
    assert step(good, 1, 0, 16, h(), None, None) == -2
    for bad in (dict(step=0), dict(lr=-1.0), dict(beta1=1.0), dict(beta2=1.0), dict(beta1=-0.1), dict(eps=-1.0), dict(weight_decay=-1.0), dict(lr=float("nan"))):
        assert step(good, 1, 0, 32, h(**bad), None, None) == -2
    for k in range(4):
        bad = list(good)
        bad[k] = 0
        assert step(t(*bad), 1, 0, 32, h(), None, None) == -2
    assert step(t(PTR, PTR, PTR, PTR, 0, PTR, 10), 1, 0, 8, h(), None, None) == -2  # no scales
    assert step(t(PTR, PTR, PTR, PTR, PTR, PTR, -1), 1, 0, 32, h(), None, None) == -2


def test_config_and_factory():
    from core.config import config
    from models.lstm import LSTM, getLSTM
    from models.recurrence import GatedScan
    from utils.utils import create_optimizer
    assert (config.MODEL.RECURRENT_CELL, config.MODEL.FUSED_HEAD_LOSS, config.TRAIN.STATE_BITS) == ("lstm", False, 32)
    cfg = make_config(18, 10, OPTIMIZER="adamw", LR=0.01, WD=0.1)
    opt = create_optimizer(cfg, torch.nn.Linear(4, 2))
    assert isinstance(opt, torch.optim.AdamW) and (opt.param_groups[0]["lr"], opt.param_groups[0]["weight_decay"]) == (0.01, 0.1)
    cfg.MODEL.LSTM_OUTDIM = 64
    assert isinstance(getLSTM(cfg, in_dim=128), LSTM)
    cfg.MODEL.RECURRENT_CELL = "scan"
    cell = getLSTM(cfg, in_dim=128)
    assert isinstance(cell, GatedScan) and set(cell.state_dict()) == {"gates.weight", "gates.bias"} and cell.gates.weight.shape == (128, 128)
    cfg.MODEL.RECURRENT_CELL = "gru"
    with pytest.raises(ValueError):
        getLSTM(cfg, in_dim=128)


def test_the_measured_work_is_well_formed():
    """perf/operators.py: case names, the spread of work, drawn cases inside the ranges of the listed ones"""
    import random
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    sys.path.insert(0, os.path.join(root, "perf"))
    try:
        import operators as M
    finally:
        sys.path.pop(0)
    cases = M.listed()
    assert 4 <= len(cases) <= 12 and len({c["name"] for c in cases}) == len(cases)
    assert all(sum(c["op"] == op for c in cases) >= 2 for op in ("lce", "scan", "adamw"))
    work = [M.work(c)["flops"] for c in cases]
    assert max(work) >= 16 * min(work)
    r = random.Random(0)
    for _ in range(200):
        c = M.draw(r)
        w = M.work(c)
        assert "name" not in c and 0 < w["flops"] <= max(work) and w["bytes"] > 0

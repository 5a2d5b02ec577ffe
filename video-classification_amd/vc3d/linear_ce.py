"""Linear classifier and cross-entropy in one operator, for class counts whose logits are not worth keeping: the reference's
clf_haed and nn.CrossEntropyLoss (lib/models/model.py:24,38, lib/core/loss.py:10,25), which linear_apply + cross_entropy compute
with kept logits up to 1024 classes."""
import torch

from . import ops
from .capi import Vc3dError

_REDUCTION = {"none": 0, "mean": 1, "sum": 2}


class _EngineHeadFn(torch.autograd.Function):
    """linear_cross_entropy of a head whose weight and bias live in an engine's flat buffers: their gradients go there, as with
    autograd.linear_apply"""

    @staticmethod
    def forward(ctx, x, weight, bias, labels, engine):
        grad = any(ctx.needs_input_grad)
        ctx.keep = -1 if grad else 0
        try:
            loss, saved = ops.linear_ce_fwd(x, weight, labels, bias, keep_bytes=ctx.keep)
        except torch.OutOfMemoryError:
            ctx.keep = 0
            loss, saved = ops.linear_ce_fwd(x, weight, labels, bias, keep_bytes=0)
        if grad:
            ctx.save_for_backward(x, weight, labels, bias, saved)
            ctx.engine, ctx.params = engine, (weight, bias)
        return loss.view(())

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        x, weight, labels, bias, saved = ctx.saved_tensors
        want, eng = ctx.needs_input_grad, ctx.engine
        dx, dw, db = ops.linear_ce_bwd(x, weight, labels, bias, saved, dloss.contiguous().view(1), want=want[:3], keep_bytes=ctx.keep)
        wp, bp = ctx.params
        if eng.flat_grad is not None and id(wp) in eng.grad_views:
            eng._bind_grads()
            for p, g in ((wp, dw), (bp, db)):
                if g is not None:
                    eng.gview(p).add_(g)
            eng._ready(wp, *([bp] if bp is not None else []))
            dw = db = None
        return dx, dw, db, None, None


def linear_cross_entropy(x, weight, labels, bias=None, ignore_index=-100, reduction="mean", keep_bytes=-1):
    """F.cross_entropy(x @ weight.T + bias, labels) without the logits: x [..., D], weight [V][D], bias [V] or None, all fp32 or
    all bf16; labels int64 [...] on the GPU.  Logits, sums and the loss are fp32.  Rows whose label is ignore_index take no part
    (their x is not read and its gradient is 0); "mean" is over the others, and 0 where there is none (torch: NaN).  Any other
    label outside [0, V) gives a NaN.  reduction "none" returns labels' shape.  Differentiable in x, weight and bias; the
    gradients are of the inputs' type.  keep_bytes: whether the forward keeps the logits' gradient for the backward (N x V of the
    inputs' type; and, while there is room, the copy of a weight whose rows are no whole 16 bytes): 0 no, the backward computes the
    logits again; n: where it takes at most n bytes; -1: where that is quicker, takes at most 2 GB and there is memory for it.
    Never with reduction "none"."""
    if reduction not in _REDUCTION:
        raise Vc3dError("linear_cross_entropy: reduction 'none', 'mean' or 'sum', got %r" % (reduction,))
    return ops._tensors.linear_cross_entropy(x, weight, labels, bias, ignore_index, _REDUCTION[reduction], keep_bytes)


class HeadScores:
    """Class scores that are only wanted for their loss: the head's input and parameters, which a model in training hands to its
    criterion in the place of logits (config MODEL.FUSED_HEAD_LOSS).  scores() computes them after all."""

    def __init__(self, feat, weight, bias, engine=None):
        self.feat, self.weight, self.bias, self.engine = feat, weight, bias, engine

    def cross_entropy(self, y):
        """mean cross-entropy against y (int64 [N]), differentiable in the features and the head's parameters"""
        if self.engine is None:
            return linear_cross_entropy(self.feat, self.weight, y, self.bias)
        return _EngineHeadFn.apply(self.feat.contiguous(), self.weight, self.bias, y.contiguous(), self.engine)

    def scores(self):
        from .autograd import linear_apply
        return linear_apply(self.feat, self.weight, self.bias, self.engine)

"""Linear classifier and cross-entropy in one operator, for class counts whose logits are not worth keeping: the reference's
clf_haed and nn.CrossEntropyLoss (lib/models/model.py:24,38, lib/core/loss.py:10,25), which linear_apply + cross_entropy compute
with kept logits up to 1024 classes."""
import torch

from . import ops
from .capi import Vc3dError

_REDUCTION = {"none": 0, "mean": 1, "sum": 2}


class _LinearCEFn(torch.autograd.Function):
    """when ``engine`` is given, the gradients of weight and bias go to its flat buffer, as with autograd.linear_apply"""

    @staticmethod
    def forward(ctx, x, weight, labels, bias, ignore_index, reduction, engine, keep_bytes):
        d = ops._linear_ce_desc(x, weight, labels, bias, ignore_index, reduction, keep_bytes)
        loss, saved = ops._linear_ce_fwd(d, x, weight, labels, bias)
        if any(ctx.needs_input_grad):
            ctx.save_for_backward(x, weight, labels, bias, saved)
            ctx.desc, ctx.engine, ctx.params = d, engine, (weight, bias)
        return loss if reduction == 0 else loss.view(())

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        x, weight, labels, bias, saved = ctx.saved_tensors
        want, eng = ctx.needs_input_grad, ctx.engine
        dx, dw, db = ops._linear_ce_bwd(ctx.desc, x, weight, labels, bias, saved, dloss.contiguous(), (want[0], want[1], want[3]))
        wp, bp = ctx.params
        if eng is not None and eng.flat_grad is not None and id(wp) in eng.grad_views:
            eng._bind_grads()
            for p, g in ((wp, dw), (bp, db)):
                if g is not None:
                    eng.gview(p).add_(g)
            eng._ready(wp, *([bp] if bp is not None else []))
            dw = db = None
        return dx, dw, None, db, None, None, None, None


def _apply(x, weight, labels, bias, ignore_index, reduction, engine, keep_bytes):
    if not (torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or bias is not None and bias.requires_grad)):
        keep_bytes = 0  # no backward will come
    return _LinearCEFn.apply(x, weight, labels, bias, ignore_index, _REDUCTION[reduction], engine, keep_bytes)


def linear_cross_entropy(x, weight, labels, bias=None, ignore_index=-100, reduction="mean", keep_bytes=-1):
    """F.cross_entropy(x @ weight.T + bias, labels) without the logits: x [..., D], weight [V][D], bias [V] or None, all fp32 or
    all bf16; labels int64 [...] on the GPU.  Logits, sums and the loss are fp32.  Rows whose label is ignore_index take no part
    (their x is not read and its gradient is 0); "mean" is over the others, and 0 where there is none (torch: NaN).  Any other
    label outside [0, V) gives a NaN.  reduction "none" returns labels' shape.  Differentiable in x, weight and bias; the
    gradients are of the inputs' type.  keep_bytes: whether the forward keeps the logits' gradient for the
    backward (N x V of the inputs' type): 0 no, the backward computes the logits again; n: where it takes at most n bytes; -1: where
    that is quicker and takes at most 2 GB.  Never with reduction "none"."""
    if not torch.is_tensor(x) or not x.is_cuda:
        raise Vc3dError("linear_cross_entropy runs on the GPU only (no CPU fallback)")
    if reduction not in _REDUCTION:
        raise Vc3dError("linear_cross_entropy: reduction 'none', 'mean' or 'sum', got %r" % (reduction,))
    if x.dim() < 1 or x.shape[-1] == 0 or weight.dim() != 2 or tuple(labels.shape) != tuple(x.shape[:-1]):
        raise Vc3dError("linear_cross_entropy: x [..., D], weight [V][D] and labels [...] expected, got %s, %s, %s" %
                        (tuple(x.shape), tuple(weight.shape), tuple(labels.shape)))
    shape = labels.shape
    if x.dim() != 2:
        x, labels = x.reshape(-1, x.shape[-1]), labels.reshape(-1)
    loss = _apply(ops._rows(x), ops._rows(weight), labels.contiguous(), None if bias is None else bias.contiguous(),
                  int(ignore_index), reduction, None, int(keep_bytes))
    return loss.view(shape) if reduction == "none" else loss


class HeadScores:
    """Class scores that are only wanted for their loss: the head's input and parameters, which a model in training hands to its
    criterion in the place of logits (config MODEL.FUSED_HEAD_LOSS).  scores() computes them after all."""

    def __init__(self, feat, weight, bias, engine=None):
        self.feat, self.weight, self.bias, self.engine = feat, weight, bias, engine

    def cross_entropy(self, y):
        """mean cross-entropy against y (int64 [N]), differentiable in the features and the head's parameters"""
        return _apply(self.feat.contiguous(), self.weight, y.contiguous(), self.bias, -100, "mean", self.engine, -1)

    def scores(self):
        from .autograd import linear_apply
        return linear_apply(self.feat, self.weight, self.bias, self.engine)

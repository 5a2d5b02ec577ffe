"""Gated linear recurrence over time on the vc3d kernels: the sequence form of what lstm.py does step by step (reference
lib/models/lstm.py:16,25-27), with gates that do not read the state, so that all steps are computed at once.

    f_t = sigmoid(z_t)        h_t = f_t h_(t-1) + (1 - f_t) v_t        gates [B][T][2H] = (z | v)

The state is fp32; h and the gradient of gates are of gates' type (fp32 or bf16)."""
import torch

from . import ops
from .capi import Vc3dError
from .packed import PackedOperand


def gated_scan(gates, h0=None, lengths=None, reverse=False):
    """gates [B][T][2H] (fp32 or bf16; logits of the forget gate, then values; e.g. one GEMM's output), h0 [B][H] fp32 (zeros if
    None), lengths int32 or int64 [B] on the GPU (sequence b is its first lengths[b] steps; all T if None), reverse: from a
    sequence's last step to its first -> (h [B][T][H], last state [B][H] fp32).  h and the gradient of gates are 0 behind a
    sequence's end, whatever gates hold there; last is h0 where there is no step.  Differentiable in gates and h0."""
    return ops._tensors.gated_scan(gates, h0, lengths, reverse)


def gated_scan_step(gates, state):
    """one step of gated_scan for each of B sequences, for serving: gates [B][2H], state [B][H] fp32, which is updated in place
    -> h [B][H] of gates' type.  No gradient: refused where one is wanted (torch.no_grad() around it serves)."""
    return ops.gated_scan_step(gates, state)


class PackedGateWeight(PackedOperand):
    """bf16 operands of a gate projection's weight and bias, kept from call to call: [W | b0 b1 b2 0 ...], where the bias lies in 64
    more columns as the three bf16 numbers whose sum it is (8 bits each of its 24)"""

    def matrix(self, weight, bias=None):
        w = weight.detach().float().contiguous()
        return w if bias is None else ops.bias_columns(w, bias.detach().float().contiguous(), torch.float32)


class _GateProjectionFn(torch.autograd.Function):
    """x [N][Fin] W^T + b -> bf16 [N][2H] as a 1x1x1 conv over N positions, like lstm.py's gates; gradients fp32.  With a bias x gets
    64 more columns, ones and zeros: the bias is a part of the product, is added in its fp32 sums and rounded with them, once;
    and its gradient is a column of the weight's."""

    @staticmethod
    def forward(ctx, x, weight, bias, packed):
        N, fin = x.shape
        co = weight.shape[0]
        wf, wd = packed.get(weight, bias)
        x = x.detach().contiguous()
        xb = x.to(torch.bfloat16) if bias is None else ops.bias_columns(x)
        width = xb.shape[1]
        d = ops.conv_desc(N, width, 1, 1, 1, co, 1, 1, 0)
        ctx.save_for_backward(xb)
        ctx.d, ctx.wd, ctx.fin = d, wd, fin
        if N == 0:
            return torch.empty(0, co, dtype=torch.bfloat16, device=x.device)
        return ops.conv3d_fwd(d, xb.view(N, 1, 1, 1, width), wf).view(N, co)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dg):
        xb, = ctx.saved_tensors
        (N, width), co, fin, want = xb.shape, dg.shape[1], ctx.fin, ctx.needs_input_grad
        dg5 = dg.contiguous().view(N, 1, 1, 1, co)
        dx = dw = db = None
        if want[0]:
            dx = ops.conv3d_dgrad(ctx.d, dg5, ctx.wd).view(N, width)[:, :fin].float() if N > 0 else torch.empty(0, fin, device=dg.device)
        if want[1] or want[2]:
            both = torch.zeros(co, 1, 1, 1, width, dtype=torch.float32, device=dg.device)
            if N > 0:
                ops.conv3d_wgrad(ctx.d, xb.view(N, 1, 1, 1, width), dg5, both)
            both = both.view(co, width)
            dw = both[:, :fin].contiguous() if want[1] else None
            db = both[:, fin].contiguous() if want[2] else None
        return dx, dw, db, None


def gate_projection(x, weight, bias, packed):
    """gates [N][2H] in bf16 = x [N][Fin] W^T + b, from fp32 x, weight [2H][Fin] and bias [2H] (or None); Fin and 2H are multiples of
    64.  x and W are rounded to bf16, the bias is not; the sums are fp32 and round once, to the gates.  `packed`: a PackedGateWeight
    that keeps the bf16 operands from step to step."""
    if not x.is_cuda:
        raise Vc3dError("the vc3d gate projection runs on the GPU only (no CPU fallback)")
    if x.dim() != 2 or weight.dim() != 2 or x.shape[1] != weight.shape[1] or x.shape[1] % 64 or weight.shape[0] % 64:
        raise Vc3dError("gate projection: x [N][Fin] and weight [2H][Fin] with Fin and 2H multiples of 64 expected, got %s and %s" %
                        (tuple(x.shape), tuple(weight.shape)))
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise Vc3dError("gate projection: bias [%d] expected, got %s" % (weight.shape[0], tuple(bias.shape)))
    ops._same_device(x, weight=weight, bias=bias)
    with ops._on(x):  # (the conv's launches go to the current device's stream)
        return _GateProjectionFn.apply(x.float(), weight, bias, packed)

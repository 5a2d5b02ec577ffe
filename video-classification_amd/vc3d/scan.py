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
    -> h [B][H] of gates' type.  No gradient."""
    return ops.gated_scan_step(gates, state)


class PackedGateWeight(PackedOperand):
    """bf16 operands of a gate projection's weight, kept from call to call"""


class _GateProjectionFn(torch.autograd.Function):
    """x [N][Fin] W^T -> bf16 [N][2H] as a 1x1x1 conv over N positions, like lstm.py's gates; gradients fp32"""

    @staticmethod
    def forward(ctx, x, weight, packed):
        N, fin = x.shape
        co = weight.shape[0]
        wf, wd = packed.get(weight)
        xb = x.detach().to(torch.bfloat16).contiguous()
        d = ops.conv_desc(N, fin, 1, 1, 1, co, 1, 1, 0)
        ctx.save_for_backward(xb)
        ctx.d, ctx.wd = d, wd
        return ops.conv3d_fwd(d, xb.view(N, 1, 1, 1, fin), wf).view(N, co)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dg):
        xb, = ctx.saved_tensors
        (N, fin), co = xb.shape, dg.shape[1]
        dg5 = dg.contiguous().view(N, 1, 1, 1, co)
        dx = ops.conv3d_dgrad(ctx.d, dg5, ctx.wd).view(N, fin).float() if ctx.needs_input_grad[0] else None
        dw = torch.zeros(co, 1, 1, 1, fin, dtype=torch.float32, device=dg.device)
        ops.conv3d_wgrad(ctx.d, xb.view(N, 1, 1, 1, fin), dg5, dw)
        return dx, dw.view(co, fin), None


def gate_projection(x, weight, bias, packed):
    """gates [N][2H] in bf16 = x [N][Fin] W^T + b (the sum in fp32), from fp32 x, weight [2H][Fin] and bias [2H] (or None); Fin and 2H are multiples
    of 64.  `packed`: a PackedGateWeight that keeps the bf16 operands from step to step."""
    if not x.is_cuda:
        raise Vc3dError("the vc3d gate projection runs on the GPU only (no CPU fallback)")
    if x.dim() != 2 or weight.dim() != 2 or x.shape[1] != weight.shape[1] or x.shape[1] % 64 or weight.shape[0] % 64:
        raise Vc3dError("gate projection: x [N][Fin] and weight [2H][Fin] with Fin and 2H multiples of 64 expected, got %s and %s" %
                        (tuple(x.shape), tuple(weight.shape)))
    g = _GateProjectionFn.apply(x.float(), weight, packed)
    return g if bias is None else (g.float() + bias).to(g.dtype)

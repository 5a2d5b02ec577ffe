"""The recurrent head with a gated linear recurrence in the LSTM's place (config MODEL.RECURRENT_CELL = 'scan'; the reference's
cell is lib/models/lstm.py:12-30, whose interface this keeps: a state in the module, ``reset``, one step per call).

The gates come from the input alone, gates = x W^T + b, so a whole sequence of features is one matrix product and one scan
(``sequence``).  The product is the LSTM's: bf16 operands on the 1x1x1 conv kernels, bf16 gates; the state is fp32."""
import torch
import torch.nn as nn

import vc3d
from vc3d.scan import PackedGateWeight, gate_projection


class GatedScan(nn.Module):
    def __init__(self, in_dim, out_dim):
        super().__init__()
        self.gates = nn.Linear(in_dim, 2 * out_dim)  # the parameter holder: rows [0, out_dim) forget gate, the rest values
        self.out_dim = out_dim
        self.h = None
        self._packed = PackedGateWeight()

    def reset(self, batch_size):
        self.h = torch.zeros((batch_size, self.out_dim), device=self.gates.weight.device)

    def _gates(self, x):
        return gate_projection(x, self.gates.weight, self.gates.bias, self._packed)

    def forward(self, input):
        """one step: input [N][in_dim] -> h [N][out_dim]; the state that the next call sees is detached, as the LSTM's"""
        if self.h is None or self.h.shape[0] != input.shape[0] or self.h.device != input.device:
            self.reset(input.shape[0])
        gates = self._gates(input)
        if not torch.is_grad_enabled():
            # in place, on a copy: a state that a caller took out of the module stays what it was
            self.h = self.h.clone()
            vc3d.gated_scan_step(gates, self.h)
            return self.h
        _, h = vc3d.gated_scan(gates[:, None], self.h)
        self.h = h.detach()
        return h

    def sequence(self, input, lengths=None, h0=None):
        """all steps at once: input [N][T][in_dim], lengths [N] or None -> (h [N][T][out_dim] fp32, last state [N][out_dim]);
        the module's own state is neither read nor changed"""
        N, T, F = input.shape
        gates = self._gates(input.reshape(N * T, F)).view(N, T, 2 * self.out_dim)
        h, last = vc3d.gated_scan(gates, h0, lengths=lengths)
        return h.float(), last

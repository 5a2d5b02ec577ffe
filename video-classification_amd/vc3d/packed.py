"""bf16 operands of parameters that are kept in fp32, packed when a parameter has changed and used by every call until the next
change (the gate products of lstm.py and scan.py)."""
import weakref

import torch

from . import ops
from .capi import cur_stream


def _matrix_pack(matrix):
    """fp32 [Co][Ci] on the GPU -> its forward / weight-gradient operand and its data-gradient twin (a 1x1x1 conv's)"""
    co, ci = matrix.shape
    return ops.pack_weight(matrix.view(co, 1, 1, 1, ci).permute(0, 4, 1, 2, 3), want_dgrad=True)  # channels_last_3d storage


class PackedOperand:
    """The operands of `matrix(*weights)`.  What is kept belongs to these very tensors (not to others that came to lie at the same
    address: they are compared by identity, and their memory is held) in this very state (their version counters: a write through
    ``weight.data`` is not seen).  It may be used on any stream: one other than that which packed it waits for the packing, and the
    operands' memory is not given away before that stream is done with it.  A call that is captured into a graph packs for itself,
    into the graph's own memory: a replay then computes with what the weights hold when it runs, and neither reads nor
    fills what eager calls share."""

    def __init__(self):
        self.kept = None  # (weights, their key and memory, stream, event, operands): replaced as a whole

    def matrix(self, weight):
        return weight.detach().float().contiguous()

    def get(self, *weights):
        if torch.cuda.is_current_stream_capturing():
            return _matrix_pack(self.matrix(*weights))
        key = tuple(None if w is None else (w._version, w.data_ptr(), w.shape, w.stride(), w.dtype, w.device) for w in weights)
        stream, kept = cur_stream(), self.kept
        if kept is not None and kept[1] == key and all(w is None or r() is w for r, w in zip(kept[0], weights)):
            if stream != kept[3]:
                here = torch.cuda.current_stream()
                here.wait_event(kept[4])
                for t in kept[5]:
                    t.record_stream(here)
            return kept[5]
        operands = _matrix_pack(self.matrix(*weights))
        # (an event is made for a stream once: to destroy one for every change of weights took 20 us)
        same = kept is not None and kept[3] == stream and kept[1][0][-1] == key[0][-1]
        packed = kept[4] if same else torch.cuda.Event()
        packed.record()
        self.kept = (tuple(None if w is None else weakref.ref(w) for w in weights), key, tuple(None if w is None else w.detach() for w in weights),
                     stream, packed, operands)
        return operands

    def __reduce__(self):  # a copy of a module packs for itself
        return type(self), ()

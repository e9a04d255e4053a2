"""Gated linear recurrence along packed clouds (no counterpart in the reference): what lies beyond a
window of rows is carried in a state of one value per channel.

    log a_t = -softplus(decay) * sigmoid(gate_t);  h_t = a_t h_{t-1} + sqrt(1 - a_t^2) x_t
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor

from .. import csrc


class GatedScan(torch.autograd.Function):
    """(h, last) of gdl_gated_scan; differentiable w.r.t. x, gate, decay and h0."""

    @staticmethod
    def forward(ctx, x: Tensor, gate: Tensor, decay: Tensor, h0: Optional[Tensor], ptr: Tensor, reverse: bool):
        need = any(ctx.needs_input_grad[:4])
        h, last, states, held = csrc.gated_scan_cuda(x, gate, decay, ptr, h0, reverse, with_states=need)
        if need:
            ctx.save_for_backward(*held, states)
            ctx.reverse = reverse
            ctx.like = (decay.dtype, None if h0 is None else h0.dtype)
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    def backward(ctx, grad_h: Optional[Tensor], grad_last: Optional[Tensor]):
        csrc.once_only("gated_scan")
        x, gate, decay, ptr, states = ctx.saved_tensors
        dx, dgate, ddecay, dh0 = csrc.gated_scan_backward_cuda(x, gate, decay, ptr, states, grad_h, grad_last,
                                                               ctx.reverse, want_h0=ctx.needs_input_grad[3])
        return dx, dgate, ddecay.to(ctx.like[0]), dh0 if dh0 is None else dh0.to(ctx.like[1]), None, None


def gated_scan(x: Tensor, gate: Tensor, decay: Tensor, ptr: Tensor, *, h0: Optional[Tensor] = None,
               reverse: bool = False) -> Tuple[Tensor, Tensor]:
    """(h [N, C] of x's type, last [B, C] float32): the recurrence over x and gate [N, C] (float32 or
    bfloat16) within each cloud [ptr[b], ptr[b+1]), per channel, from h0 [B, C] (zeros if left out).

    decay [C] float32 sets each channel's shortest memory: a_t runs from exp(-softplus(decay)) (gate
    open) to 1 (gate shut: the state is kept). ``last`` is the state after the cloud's last row (h0 for
    an empty cloud): pass it as the next call's h0 to go on with a stream, one row or many at a time.
    ``reverse`` runs each cloud from its last row to its first. States are float32 throughout.
    Gradients w.r.t. x, gate, decay and h0; bit-reproducible."""
    if csrc.tracked(x, gate, decay, h0):
        return GatedScan.apply(x, gate, decay, h0, ptr, reverse)
    return csrc.gated_scan_cuda(x, gate, decay, ptr, h0, reverse, with_states=False)[:2]

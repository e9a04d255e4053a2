"""Attention along the order of packed clouds, with a sliding window, sinks and a learned bias by the
distance between the two points (no counterpart in the reference).

The rows of a cloud lie in an order that keeps neighbours near each other (a space-filling curve, a
sweep's scan order), so a window of rows is a neighbourhood. ``num_sinks`` first rows stay visible
beyond the window (register rows, or farthest-point samples put in front). The bias depends on the two
points' distance alone, so rotations and shifts of the cloud do not change it (they may change the order of
the rows, and with it the windows).
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch import Tensor

from .. import csrc


class WindowAttention(torch.autograd.Function):
    """out of gdl_window_attention; differentiable w.r.t. q, k, v and the bias table."""

    @staticmethod
    def forward(ctx, q: Tensor, k: Tensor, v: Tensor, bias: Optional[Tensor], pos_q: Optional[Tensor],
                pos_k: Optional[Tensor], meta, status: Optional[Tensor]):
        need = any(ctx.needs_input_grad[:4])
        out, lse, rest, args = csrc.window_attention_cuda(q, k, v, bias, *meta[:5], pos_q, pos_k, *meta[5:], with_lse=need,
                                                        status=status)
        if need:
            q, k, v, bias, ptr_q, ptr_k, pos_q, pos_k = args[0]
            ctx.save_for_backward(out, lse, rest, q, k, v, bias, ptr_q, ptr_k, pos_q, pos_k)
            ctx.meta, ctx.status = args[1], status
        return out

    @staticmethod
    def backward(ctx, grad_out: Tensor):
        csrc.once_only("window_attention")
        out, lse, rest, *held = ctx.saved_tensors
        dq, dk, dv, db = csrc.window_attention_backward_cuda(held, ctx.meta, out, lse, rest, grad_out,
                                                             want_bias=ctx.needs_input_grad[3], status=ctx.status)
        return dq, dk, dv, db, None, None, None, None


def window_attention(q: Tensor, k: Tensor, v: Tensor, ptr_q: Tensor, *, ptr_k: Optional[Tensor] = None,
                     window: Tuple[int, int] = (-1, -1), num_sinks: int = 0, scale: Optional[float] = None,
                     bias: Optional[Tensor] = None, pos_q: Optional[Tensor] = None, pos_k: Optional[Tensor] = None,
                     radius: float = 1.0, steps: int = 4, status: Optional[Tensor] = None) -> Tensor:
    """out [Nq, H, D]: attention of q [Nq, H, D] over k, v [Nk, Hk, D] within each cloud (H a multiple
    of Hk: heads that share keys and values), float32 or bfloat16, D <= 128.

    ptr_q, ptr_k  [B + 1] int64 bounds of the clouds' queries and keys (ptr_k: ptr_q if left out). The
                  queries of a cloud are its last rows: with fewer queries than keys they are the new
                  rows of a stream whose earlier keys are cached.
    window        (left, right): row i sees rows i - left .. i + right; -1 leaves a side open,
                  right = 0 is causal.
    num_sinks     the first rows of each cloud that stay visible to the left of the window.
    scale         of the products, 1 / sqrt(D) if left out.
    bias          [H, buckets] learned table (at most 64 buckets), with pos_q [Nq, 3], pos_k [Nk, 3]
                  (pos_k: pos_q if left out): bucket of t = 1 + distance^2 / radius^2 with `steps`
                  (1, 2, 4, 8 or 16) buckets to each doubling of t, the last one open. Positions are
                  constants (no gradient).

    status        int32 CUDA tensor of one element, zeroed by the caller: receives GDL_ERR_TIMEOUT (6) if a
                  bounded wait of a kernel gave up, forward or backward (its rows are then NaN).

    A row that sees no key gives 0, and so does one whose logits are all -inf (a bias may hold -inf); both take no
    part in a gradient. What a row does not see never reaches its result; a NaN or an infinity in q, or in a key that
    it sees, does. Logits are held in 32 bits: a row masked throughout by a large negative bias weighs its keys alike.
    Gradients w.r.t. q, k, v and bias (of first order); bit-reproducible."""
    if (pos_q is not None and pos_q.requires_grad) or (pos_k is not None and pos_k.requires_grad):
        raise csrc.nat.GdlError("window_attention: positions are constants of the bias; detach them")
    meta = (ptr_q, ptr_q if ptr_k is None else ptr_k, window, num_sinks,
            1.0 / math.sqrt(max(q.shape[-1], 1)) if scale is None else scale, radius, steps)
    pos_k = pos_q if pos_k is None else pos_k
    if csrc.tracked(q, k, v, bias, pos_q, pos_k):
        return WindowAttention.apply(q, k, v, bias, pos_q, pos_k, meta, status)
    return csrc.window_attention_cuda(q, k, v, bias, *meta[:5], pos_q, pos_k, *meta[5:], with_lse=False, status=status)[0]

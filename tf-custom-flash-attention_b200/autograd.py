"""Autograd binding: the gradient registration of the reference's Python layer.

Mirrors ``@tf.RegisterGradient("Sdpa")`` (mha.py:10-21): the backward of
``sdpa`` calls ``sdpa_grad`` with the forward's inputs, outputs and attrs;
seed and offset get no gradient, and the gradient reaching ``stats`` is
ignored (the reference drops it via ``*args``) unless the caller asks for
it with ``sdpa_with_stats(..., differentiable_stats=True)`` (an extension).
Gradients are not differentiable again (as the reference registers none for
``SdpaGrad``): doing so raises RuntimeError.
"""
from __future__ import annotations

import torch

from . import ops, rotary


class _FirstOrder(torch.autograd.Function):
    """compute() as a function of `inputs` that has no derivative."""

    @staticmethod
    def forward(ctx, compute, *inputs):
        return compute()

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("sdpa_b200 has no second derivatives: a gradient of an operator was differentiated again")


def _first_order(compute, *inputs):
    """compute(), the gradients an operator's kernel gives.  Its results carry no graph; where autograd builds one
    (create_graph=True) they get a node over all that they depend on, the saved inputs too, which refuses to be
    differentiated: without it the terms through them would be left out in silence."""
    return _FirstOrder.apply(compute, *inputs) if torch.is_grad_enabled() else compute()


class SdpaFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, seed, offset, dropout, scale, causal_mask, differentiable_stats=False):
        o, s = ops.sdpa(q, k, v, seed, offset, scale=scale, dropout=dropout, causal_mask=causal_mask)
        ctx.save_for_backward(q, k, v, o, s)
        ctx.attrs = (int(ops._scalar_u64(seed, "seed")), int(ops._scalar_u64(offset, "offset")), dropout, scale,
                     causal_mask)
        ctx.stats_grad = bool(differentiable_stats)
        if not ctx.stats_grad:
            ctx.mark_non_differentiable(s)
        return o, s

    @staticmethod
    def backward(ctx, d_o, d_stats):
        q, k, v, o, s = ctx.saved_tensors
        seed, offset, dropout, scale, causal = ctx.attrs
        if d_o is None:
            d_o = torch.zeros_like(o)
        d_stats = d_stats if ctx.stats_grad else None
        dq, dk, dv = _first_order(lambda: ops.sdpa_grad(q, k, v, o, s, d_o.contiguous(), seed, offset, dropout=dropout,
                                                        scale=scale, causal_mask=causal, d_stats=d_stats),
                                  q, k, v, d_o, d_stats)
        return dq, dk, dv, None, None, None, None, None, None


class SdpaBSHDFunction(torch.autograd.Function):
    """Same gradient registration over head-strided [B,S,H,D] tensors (ops.sdpa_bshd)."""

    @staticmethod
    def forward(ctx, q, k, v, seed, offset, dropout, scale, causal_mask):
        o, s = ops.sdpa_bshd(q, k, v, seed, offset, scale=scale, dropout=dropout, causal_mask=causal_mask)
        ctx.save_for_backward(q, k, v, o, s)
        ctx.attrs = (int(ops._scalar_u64(seed, "seed")), int(ops._scalar_u64(offset, "offset")), dropout, scale,
                     causal_mask)
        return o

    @staticmethod
    def backward(ctx, d_o):
        q, k, v, o, s = ctx.saved_tensors
        seed, offset, dropout, scale, causal = ctx.attrs
        dq, dk, dv = _first_order(lambda: ops.sdpa_grad_bshd(q, k, v, o, s, d_o.contiguous(), seed, offset,
                                                             dropout=dropout, scale=scale, causal_mask=causal),
                                  q, k, v, d_o)
        return dq, dk, dv, None, None, None, None, None


def sdpa_bshd(q, k, v, seed, offset, dropout: float = 0.0, scale: float = 1.0, causal_mask: bool = False):
    """Differentiable attention over [B,S,H,D] tensors (no head transposes); returns [B,S_q,H,D_v]."""
    return SdpaBSHDFunction.apply(q, k, v, seed, offset, dropout, scale, causal_mask)


def sdpa(q, k, v, seed, offset, dropout: float = 0.0, scale: float = 1.0, causal_mask: bool = False):
    """Differentiable attention, like mha.py:24-29 ``sdpa`` (returns the output only)."""
    o, _ = SdpaFunction.apply(q, k, v, seed, offset, dropout, scale, causal_mask)
    return o


def sdpa_with_stats(q, k, v, seed, offset, dropout: float = 0.0, scale: float = 1.0, causal_mask: bool = False,
                    differentiable_stats: bool = False):
    """Differentiable attention returning (o, stats) like test.py:14-17; with
    differentiable_stats=True a loss on stats also reaches q and k."""
    return SdpaFunction.apply(q, k, v, seed, offset, dropout, scale, causal_mask, differentiable_stats)


class QKNormRopeFunction(torch.autograd.Function):
    """Head norms and rotation of q and k (rotary.qk_norm_rope); table and positions get no gradient."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, table, q_positions, k_positions, eps, interleaved):
        out = rotary.qk_norm_rope(q, k, q_weight, k_weight, table, q_positions, k_positions, eps, interleaved)
        ctx.save_for_backward(q, k, q_weight, k_weight, table, q_positions, k_positions)
        ctx.attrs = (eps, interleaved)
        return out

    @staticmethod
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, table, q_positions, k_positions = ctx.saved_tensors
        grads = _first_order(lambda: rotary.qk_norm_rope_grad(q, k, dq_out, dk_out, q_weight, k_weight, table, q_positions,
                                                              k_positions, *ctx.attrs),
                             q, k, dq_out, dk_out, q_weight, k_weight)
        return (*grads, None, None, None, None, None)


def qk_norm_rope(q, k, q_weight=None, k_weight=None, table=None, q_positions=None, k_positions=None, eps: float = 1e-6,
                 interleaved: bool = False):
    """Differentiable ``rotary.qk_norm_rope``: gradients for q, k and the norm weights, first derivatives only
    (differentiating them again raises RuntimeError).

    A step captured into a CUDA graph needs leaves of which no eager autograd
    graph is alive (torch would join the capture with the stream of the old one
    and invalidate it)."""
    return QKNormRopeFunction.apply(q, k, q_weight, k_weight, table, q_positions, k_positions, eps, interleaved)

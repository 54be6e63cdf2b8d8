"""Query/key head norms with the position rotation, for training and evaluation.

``qk_norm_rope`` computes, for every head row x of q and k at position pos,

    y = R(pos) (x * rsqrt(mean(x^2) + eps) * weight)

in one pass: the norm is skipped without a weight, the rotation without a
table.  R turns the first ``rotary_dim`` features in pairs (i, i + rotary_dim/2),
or in neighbouring pairs (2i, 2i + 1) with ``interleaved=True``, by
pos * base^(-2i/rotary_dim); the other features pass through.  The arithmetic
is fp32, rounded once.  ``qk_norm_rope_grad`` is its gradient;
``autograd.qk_norm_rope`` binds the two.  No counterpart in the reference, whose
layer takes its queries and keys as they are (mha.py:103-129).
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .ops import _DTYPES, _FEATURE_MSG, InvalidArgumentError, _check


def rotary_table(max_positions: int, rotary_dim: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """cos | sin of position * base^(-2i/rotary_dim): float32 [max_positions, rotary_dim].

    The angles are taken in float64 (a float32 angle at position 10^5 is off by
    4e-3) and their cosines and sines rounded once."""
    if rotary_dim < 8 or rotary_dim % 8:
        raise InvalidArgumentError("rotary_dim must be a positive multiple of 8")
    if max_positions < 1:
        raise InvalidArgumentError("max_positions must be positive")
    dev = torch.device(device or "cuda")
    inv = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=dev) / rotary_dim)
    angle = torch.arange(max_positions, dtype=torch.float64, device=dev)[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], 1).float()


_CUDA_MSG = "sdpa_b200 runs on CUDA tensors only (no CPU kernel is registered)"


def _dtype_of(x: torch.Tensor) -> int:
    dt = _DTYPES.get(x.dtype)
    if dt is None:
        raise InvalidArgumentError(f"T must be half or float, got {x.dtype}")
    return dt


def _same(x: torch.Tensor, device, name: str):
    if x.device != device:
        if not x.is_cuda:
            raise InvalidArgumentError(_CUDA_MSG)
        raise InvalidArgumentError(f"{name} must be on {device} like the other inputs, got {x.device}")


def _launch(device, entry, *args):
    """Calls a C ABI entry on `device` with its current stream as the last argument."""
    index = device.index
    if index == torch.cuda.current_device():
        _check(entry(*args, torch._C._cuda_getCurrentRawStream(index)))
    else:
        with torch.cuda.device(index):
            _check(entry(*args, torch._C._cuda_getCurrentRawStream(index)))


def _rows(x: torch.Tensor, row: int, align: int):
    """x [..., H, D] as (tensor, elements between tokens), its last two axes (`row` elements) dense; copies only
    where they are not."""
    if not x.is_contiguous():
        H, D = x.shape[-2], x.shape[-1]
        try:
            y = x.view(-1, H, D)
        except RuntimeError:
            y = None
        if (y is not None and (D == 1 or y.stride(2) == 1) and (H == 1 or y.stride(1) == D) and y.data_ptr() % 16 == 0
                and (y.shape[0] == 1 or (y.stride(0) >= row and y.stride(0) % align == 0))):
            return y, (row if y.shape[0] == 1 else y.stride(0))
        x = x.contiguous()
    if x.data_ptr() % 16:
        x = x.clone()
    return x, row


def _check_features(D: int, what: str = "feature size"):
    if D > 128:
        raise InvalidArgumentError(_FEATURE_MSG)
    if D < 8 or D % 8:
        raise InvalidArgumentError(f"{what} must be a multiple of 8, got {D}")


def _weight(w, dtype, device, D: int):
    if w is None:
        return None
    if w.dim() != 1 or w.shape[0] != D:
        raise InvalidArgumentError(f"a norm weight must be [{D}], got {list(w.shape)}")
    if w.dtype != dtype and w.dtype != torch.float32:
        raise InvalidArgumentError("norm weights must have dtype T or float32")
    _same(w, device, "a norm weight")
    return w.contiguous()


def _weights(q_weight, k_weight, dtype, device, D: int):
    """(q weight, k weight, dtype code) of the norms."""
    q_weight, k_weight = _weight(q_weight, dtype, device, D), _weight(k_weight, dtype, device, D)
    if q_weight is None:
        return None, k_weight, _DTYPES[dtype if k_weight is None else k_weight.dtype]
    if k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise InvalidArgumentError("q_weight and k_weight must share a dtype")
    return q_weight, k_weight, _DTYPES[q_weight.dtype]


def _table(table, device, D: int):
    """(table, positions it holds, rotated features)."""
    if table is None:
        return None, 0, 0
    if table.dim() != 2 or table.dtype != torch.float32:
        raise InvalidArgumentError("table must be float32 [max_positions, rotary_dim]")
    positions, rot = table.shape
    if rot < 8 or rot % 8 or rot > D:
        raise InvalidArgumentError(f"rotary_dim must be a multiple of 8 no larger than the feature size, got {rot}")
    if positions < 1:
        raise InvalidArgumentError("table must hold at least one position")
    _same(table, device, "table")
    if not table.is_contiguous() or table.data_ptr() % 16:
        table = table.clone(memory_format=torch.contiguous_format)
    return table, positions, rot


def _positions(pos, lead, device, name: str):
    if pos is None:
        return None
    if pos.dtype not in (torch.int32, torch.int64):
        raise InvalidArgumentError(f"{name} must be int32 or int64")
    if pos.shape != lead:
        raise InvalidArgumentError(f"{name} must be {list(lead)}, got {list(pos.shape)}")
    _same(pos, device, name)
    if pos.dtype == torch.int64:  # (cut to 32 bits, a position past them could name a row of the table)
        pos = pos.clamp(-1, 0x7FFFFFFF).to(torch.int32)
    return pos.contiguous()


def _ptr(x):
    return None if x is None else x.data_ptr()


class _Call:
    """The checked arguments of one call, in the C ABI's terms."""

    __slots__ = ("dt", "device", "D", "q", "k", "qs", "ks", "q_lead", "k_lead", "q_tokens", "k_tokens", "H_q", "H_k", "align",
                 "qw", "kw", "rest", "qp", "kp")

    def __init__(self, q, k, q_weight, k_weight, table, q_positions, k_positions, eps, interleaved):
        qshape, kshape = q.shape, k.shape
        for shape, name in ((qshape, "q"), (kshape, "k")):
            if len(shape) < 3:
                raise InvalidArgumentError(f"{name} must be [..., S, H, D] but is rank {len(shape)}")
        self.D = D = qshape[-1]
        if kshape[-1] != D:
            raise InvalidArgumentError("K feature size mismatch")
        _check_features(D)
        self.dt = _dtype_of(q)
        if k.dtype != q.dtype:
            raise InvalidArgumentError("all floating-point inputs must share dtype T")
        if not q.is_cuda:
            raise InvalidArgumentError(_CUDA_MSG)
        self.device = device = q.device
        _same(k, device, "k")
        self.qw, self.kw, wdt = _weights(q_weight, k_weight, q.dtype, device, D)
        table, max_pos, rot = _table(table, device, D)
        # (the tensors are kept until the launch: a copy made here must outlive it)
        self.rest = (table, wdt, float(eps), None if table is None else table.data_ptr(), max_pos, rot, int(bool(interleaved)))
        self.q_lead, self.k_lead = qshape[:-2], kshape[:-2]
        if q_positions is not None and k_positions is None and self.q_lead == self.k_lead:
            k_positions = q_positions
        self.qp = _positions(q_positions, self.q_lead, device, "q_positions")
        self.kp = self.qp if k_positions is q_positions else _positions(k_positions, self.k_lead, device, "k_positions")
        self.H_q, self.H_k = qshape[-2], kshape[-2]
        self.q_tokens, self.k_tokens = math.prod(self.q_lead), math.prod(self.k_lead)
        self.align = 8 if self.dt == _lib.F16 else 4
        self.q, self.qs = _rows(q, self.H_q * D, self.align)
        self.k, self.ks = _rows(k, self.H_k * D, self.align)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight=None, k_weight=None, table=None, q_positions=None,
                 k_positions=None, eps: float = 1e-6, interleaved: bool = False):
    """(q_out, k_out): head norms and rotation of q [..., S, H_q, D] and k [..., S_k, H_k, D].

    ``q_weight`` / ``k_weight`` [D] (dtype T or float32) switch the norms on;
    ``table`` is ``rotary_table``'s.  ``q_positions`` [..., S] (int32 or int64) default
    to 0 .. S-1 along S; ``k_positions`` to q's where the two shapes agree, else
    to 0 .. S_k-1.  A position the table does not hold is clamped to its ends and
    raises bit 1 of ``device_status``.  Inputs may be strided along S (slices of
    a fused projection); outputs are contiguous."""
    c = _Call(q, k, q_weight, k_weight, table, q_positions, k_positions, eps, interleaved)
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    _launch(c.device, _lib.lib().sdpa_b200_qk_norm_rope, c.dt, c.q.data_ptr(), c.q_tokens, c.H_q, c.qs, _ptr(c.qp),
            c.q_lead[-1] or 1, c.k.data_ptr(), c.k_tokens, c.H_k, c.ks, _ptr(c.kp), c.k_lead[-1] or 1, c.D, _ptr(c.qw),
            _ptr(c.kw), *c.rest[1:], q_out.data_ptr(), k_out.data_ptr())
    return q_out, k_out


def qk_norm_rope_grad(q: torch.Tensor, k: torch.Tensor, dq_out: torch.Tensor, dk_out: torch.Tensor, q_weight=None,
                      k_weight=None, table=None, q_positions=None, k_positions=None, eps: float = 1e-6,
                      interleaved: bool = False):
    """(dq, dk, dq_weight, dk_weight) of ``qk_norm_rope`` from its inputs and its outputs' gradients.

    Weight gradients have the weights' dtype (None without a weight); they are
    summed in fp32 in a fixed order, so every run gives the same bits."""
    c = _Call(q, k, q_weight, k_weight, table, q_positions, k_positions, eps, interleaved)
    for x, ref, name in ((dq_out, q, "dq_out"), (dk_out, k, "dk_out")):
        if x.shape != ref.shape or x.dtype != ref.dtype:
            raise InvalidArgumentError(f"{name} must have the shape and dtype of its input")
        _same(x, c.device, name)
    gq, gqs = _rows(dq_out, c.H_q * c.D, c.align)
    gk, gks = _rows(dk_out, c.H_k * c.D, c.align)
    dq = torch.empty_like(q, memory_format=torch.contiguous_format)
    dk = torch.empty_like(k, memory_format=torch.contiguous_format)
    dqw = None if c.qw is None else torch.empty_like(c.qw)
    dkw = None if c.kw is None else torch.empty_like(c.kw)
    ws_bytes, ws = 0, None
    if dqw is not None or dkw is not None:
        ws_bytes = _lib.lib().sdpa_b200_qk_norm_rope_bwd_workspace_bytes(c.D)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=c.device)
    _launch(c.device, _lib.lib().sdpa_b200_qk_norm_rope_bwd, c.dt, c.q.data_ptr(), gq.data_ptr(), c.q_tokens, c.H_q, c.qs, gqs,
            _ptr(c.qp), c.q_lead[-1] or 1, c.k.data_ptr(), gk.data_ptr(), c.k_tokens, c.H_k, c.ks, gks, _ptr(c.kp),
            c.k_lead[-1] or 1, c.D, _ptr(c.qw), _ptr(c.kw), *c.rest[1:], dq.data_ptr(), dk.data_ptr(), _ptr(dqw), _ptr(dkw),
            _ptr(ws), ws_bytes)
    return dq, dk, dqw, dkw

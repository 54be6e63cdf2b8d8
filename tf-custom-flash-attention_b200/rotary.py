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


def _dtype_of(x: torch.Tensor) -> int:
    dt = _DTYPES.get(x.dtype)
    if dt is None:
        raise InvalidArgumentError(f"T must be half or float, got {x.dtype}")
    return dt


def _same(x: torch.Tensor, ref: torch.Tensor, name: str):
    if not x.is_cuda:
        raise InvalidArgumentError("sdpa_b200 runs on CUDA tensors only (no CPU kernel is registered)")
    if x.device != ref.device:
        raise InvalidArgumentError(f"{name} must be on {ref.device} like the other inputs, got {x.device}")


def _rows(x: torch.Tensor, align: int):
    """x [..., H, D] as (tensor, elements between tokens), its last two axes dense; copies only where they are not."""
    H, D = x.shape[-2], x.shape[-1]
    if not x.is_contiguous():
        try:
            y = x.view(-1, H, D)
        except RuntimeError:
            y = None
        if (y is not None and (D == 1 or y.stride(2) == 1) and (H == 1 or y.stride(1) == D) and y.data_ptr() % 16 == 0
                and (y.shape[0] == 1 or (y.stride(0) >= H * D and y.stride(0) % align == 0))):
            return y, (H * D if y.shape[0] == 1 else y.stride(0))
        x = x.contiguous()
    if x.data_ptr() % 16:
        x = x.clone()
    return x, H * D


def _check_heads(x: torch.Tensor, name: str, D: int):
    if x.dim() < 3:
        raise InvalidArgumentError(f"{name} must be [..., S, H, D] but is rank {x.dim()}")
    if x.shape[-1] != D:
        raise InvalidArgumentError("K feature size mismatch")


def _check_features(D: int, what: str = "feature size"):
    if D > 128:
        raise InvalidArgumentError(_FEATURE_MSG)
    if D < 8 or D % 8:
        raise InvalidArgumentError(f"{what} must be a multiple of 8, got {D}")


def _weights(q_weight, k_weight, q: torch.Tensor, D: int):
    """(q weight, k weight, dtype code) of the norms."""
    code = _DTYPES[q.dtype]
    given = [w for w in (q_weight, k_weight) if w is not None]
    for w in given:
        if w.dim() != 1 or w.shape[0] != D:
            raise InvalidArgumentError(f"a norm weight must be [{D}], got {list(w.shape)}")
        if w.dtype not in (q.dtype, torch.float32):
            raise InvalidArgumentError("norm weights must have dtype T or float32")
        _same(w, q, "a norm weight")
    if given:
        if given[0].dtype != given[-1].dtype:
            raise InvalidArgumentError("q_weight and k_weight must share a dtype")
        code = _DTYPES[given[0].dtype]
    return (None if q_weight is None else q_weight.contiguous(), None if k_weight is None else k_weight.contiguous(), code)


def _table(table, q: torch.Tensor, D: int):
    """(table, positions it holds, rotated features)."""
    if table is None:
        return None, 0, 0
    if table.dim() != 2 or table.dtype != torch.float32:
        raise InvalidArgumentError("table must be float32 [max_positions, rotary_dim]")
    rot = table.shape[1]
    if rot < 8 or rot % 8 or rot > D:
        raise InvalidArgumentError(f"rotary_dim must be a multiple of 8 no larger than the feature size, got {rot}")
    if table.shape[0] < 1:
        raise InvalidArgumentError("table must hold at least one position")
    _same(table, q, "table")
    if not table.is_contiguous() or table.data_ptr() % 16:
        table = table.clone(memory_format=torch.contiguous_format)
    return table, table.shape[0], rot


def _positions(pos, x: torch.Tensor, name: str):
    if pos is None:
        return None
    if pos.dtype.is_floating_point or pos.dtype == torch.bool:
        raise InvalidArgumentError(f"{name} must be integers")
    if tuple(pos.shape) != tuple(x.shape[:-2]):
        raise InvalidArgumentError(f"{name} must be {list(x.shape[:-2])}, got {list(pos.shape)}")
    _same(pos, x, name)
    return pos.to(torch.int32).contiguous()


def _ptr(x):
    return None if x is None else x.data_ptr()


def _prepare(q, k, q_weight, k_weight, table, q_positions, k_positions):
    D = q.shape[-1] if q.dim() else 0
    _check_heads(q, "q", D)
    _check_heads(k, "k", D)
    _check_features(D)
    dt = _dtype_of(q)
    if k.dtype != q.dtype:
        raise InvalidArgumentError("all floating-point inputs must share dtype T")
    _same(q, q, "q")
    _same(k, q, "k")
    qw, kw, wdt = _weights(q_weight, k_weight, q, D)
    table, max_pos, rot = _table(table, q, D)
    if q_positions is not None and k_positions is None and q.shape[:-2] == k.shape[:-2]:
        k_positions = q_positions
    qp = _positions(q_positions, q, "q_positions")
    kp = qp if k_positions is q_positions else _positions(k_positions, k, "k_positions")
    return D, dt, qw, kw, wdt, table, max_pos, rot, qp, kp


def _tokens(x: torch.Tensor) -> int:
    n = 1
    for s in x.shape[:-2]:
        n *= s
    return n


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight=None, k_weight=None, table=None, q_positions=None,
                 k_positions=None, eps: float = 1e-6, interleaved: bool = False):
    """(q_out, k_out): head norms and rotation of q [..., S, H_q, D] and k [..., S_k, H_k, D].

    ``q_weight`` / ``k_weight`` [D] (dtype T or float32) switch the norms on;
    ``table`` is ``rotary_table``'s.  ``q_positions`` [..., S] (integers) default
    to 0 .. S-1 along S; ``k_positions`` to q's where the two shapes agree, else
    to 0 .. S_k-1.  A position the table does not hold is clamped to its ends and
    raises bit 1 of ``device_status``.  Inputs may be strided along S (slices of
    a fused projection); outputs are contiguous."""
    D, dt, qw, kw, wdt, table, max_pos, rot, qp, kp = _prepare(q, k, q_weight, k_weight, table, q_positions, k_positions)
    align = 8 if dt == _lib.F16 else 4
    qx, qs = _rows(q, align)
    kx, ks = _rows(k, align)
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    with torch.cuda.device(q.device):
        st = torch.cuda.current_stream().cuda_stream
        rc = _lib.lib().sdpa_b200_qk_norm_rope(
            dt, qx.data_ptr(), _tokens(q), q.shape[-2], qs, _ptr(qp), max(q.shape[-3], 1), kx.data_ptr(), _tokens(k),
            k.shape[-2], ks, _ptr(kp), max(k.shape[-3], 1), D, _ptr(qw), _ptr(kw), wdt, float(eps), _ptr(table), max_pos,
            rot, int(bool(interleaved)), q_out.data_ptr(), k_out.data_ptr(), st)
    _check(rc)
    return q_out, k_out


def qk_norm_rope_grad(q: torch.Tensor, k: torch.Tensor, dq_out: torch.Tensor, dk_out: torch.Tensor, q_weight=None,
                      k_weight=None, table=None, q_positions=None, k_positions=None, eps: float = 1e-6,
                      interleaved: bool = False):
    """(dq, dk, dq_weight, dk_weight) of ``qk_norm_rope`` from its inputs and its outputs' gradients.

    Weight gradients have the weights' dtype (None without a weight); they are
    summed in fp32 in a fixed order, so every run gives the same bits."""
    D, dt, qw, kw, wdt, table, max_pos, rot, qp, kp = _prepare(q, k, q_weight, k_weight, table, q_positions, k_positions)
    for x, ref, name in ((dq_out, q, "dq_out"), (dk_out, k, "dk_out")):
        if x.shape != ref.shape or x.dtype != ref.dtype:
            raise InvalidArgumentError(f"{name} must have the shape and dtype of its input")
        _same(x, ref, name)
    align = 8 if dt == _lib.F16 else 4
    qx, qs = _rows(q, align)
    kx, ks = _rows(k, align)
    gq, gqs = _rows(dq_out, align)
    gk, gks = _rows(dk_out, align)
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    dqw = None if qw is None else torch.empty_like(qw)
    dkw = None if kw is None else torch.empty_like(kw)
    L = _lib.lib()
    ws_bytes, ws = 0, None
    if qw is not None or kw is not None:
        ws_bytes = L.sdpa_b200_qk_norm_rope_bwd_workspace_bytes(D)
        ws = torch.empty(ws_bytes // 4, dtype=torch.float32, device=q.device)
    with torch.cuda.device(q.device):
        st = torch.cuda.current_stream().cuda_stream
        rc = L.sdpa_b200_qk_norm_rope_bwd(
            dt, qx.data_ptr(), gq.data_ptr(), _tokens(q), q.shape[-2], qs, gqs, _ptr(qp), max(q.shape[-3], 1),
            kx.data_ptr(), gk.data_ptr(), _tokens(k), k.shape[-2], ks, gks, _ptr(kp), max(k.shape[-3], 1), D, _ptr(qw),
            _ptr(kw), wdt, float(eps), _ptr(table), max_pos, rot, int(bool(interleaved)), dq.data_ptr(), dk.data_ptr(),
            _ptr(dqw), _ptr(dkw), _ptr(ws), ws_bytes, st)
    _check(rc)
    return dq, dk, dqw, dkw

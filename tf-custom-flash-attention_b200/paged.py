"""Serving: the paged key/value cache, its write and the attention that reads it.

The cache is two pools, ``k_pages`` [pages, page_size, H_kv, D] and ``v_pages``
[pages, page_size, H_kv, D_v].  A call takes the new tokens of several
sequences one behind the other, [T, H, D], with three int32 device tensors:

    q_start    [N+1]   sequence n's new tokens are q_start[n] .. q_start[n+1]-1
    kv_len     [N]     tokens it has cached once its new ones are written
    page_table [N, M]  its key j lies at row j % page_size of page_table[n, j // page_size]

so new token i of sequence n is at position kv_len[n] - (q_start[n+1] -
q_start[n]) + i.  The kernels read these on the device, the host never does: a
captured graph replays with whatever they hold then.  Rows behind the last
sequence (T past q_start[N], the padding of a captured batch) are neither
written to the cache nor to the outputs.  Values outside their ranges reach no
memory and raise bit 1 of ``device_status``: a page id outside the pool reads
as zeros and is not written; a length past the table's capacity is clamped to
it by the attention, and a token whose position is past the table (or below
zero) is not written; starts are clamped to 0 .. T.  q_start ascends: a sequence
between two descending starts is empty to the attention, which leaves the whole call
out (its outputs stay as they were) where others then share tokens; which
tokens the write takes is not defined.

``paged_append`` writes new keys and values, with the head norms and the
position rotation of ``rotary.qk_norm_rope`` applied on the way (and to the
queries, in the same launch); ``paged_sdpa`` attends.  No counterparts in the
reference, which serves [B, S, D] tensors only.
"""
from __future__ import annotations

import torch

from . import _lib
from .ops import InvalidArgumentError
from .rotary import _CUDA_MSG, _check_features, _dtype_of, _launch, _ptr, _rows, _same, _table, _weights


def _check_batch(page_table, kv_len, q_start, device):
    """(N, M) of a batch's index tensors."""
    for x, name, dim in ((page_table, "page_table", 2), (kv_len, "kv_len", 1), (q_start, "q_start", 1)):
        if x.dtype != torch.int32 or x.dim() != dim or not x.is_contiguous():
            raise InvalidArgumentError(f"{name} must be a contiguous int32 tensor of rank {dim}")
        if x.device != device:
            _same(x, device, name)
    N, M = page_table.shape
    if kv_len.shape[0] != N or q_start.shape[0] != N + 1:
        raise InvalidArgumentError("page_table must be [N, M], kv_len [N] and q_start [N+1]")
    return N, M


def _check_pools(k_pages, v_pages, dtype, device):
    """(pages, page size, H_kv, D, D_v) of the pools."""
    for x, name in ((k_pages, "k_pages"), (v_pages, "v_pages")):
        if x.dim() != 4 or not x.is_contiguous():
            raise InvalidArgumentError(f"{name} must be a contiguous [pages, page_size, H_kv, D] tensor")
        if x.dtype != dtype:
            raise InvalidArgumentError("all floating-point inputs must share dtype T")
        if x.device != device:
            _same(x, device, name)
        if x.data_ptr() % 16:
            raise InvalidArgumentError(f"{name} must start at a multiple of 16 bytes")
    P, page, H_kv, D = k_pages.shape
    vP, vpage, vH, D_v = v_pages.shape
    if vP != P or vpage != page or vH != H_kv:
        raise InvalidArgumentError("k_pages and v_pages must have the same pages, page size and heads")
    if P < 1 or H_kv < 1:
        raise InvalidArgumentError("the pools must hold at least one page and one head")
    if page < 16 or page > 65536 or page & (page - 1):
        raise InvalidArgumentError(f"page_size must be a power of two from 16 to 65536, got {page}")
    _check_features(D)
    _check_features(D_v, "value feature size")
    return P, page, H_kv, D, D_v


def _check_tokens(x: torch.Tensor, name: str, T: int, D: int, H, dtype):
    if x.dim() != 3 or x.shape[0] != T or x.shape[2] != D or (H is not None and x.shape[1] != H):
        raise InvalidArgumentError(f"{name} must be [{T}, {'H' if H is None else H}, {D}], got {list(x.shape)}")
    if x.dtype != dtype:
        raise InvalidArgumentError("all floating-point inputs must share dtype T")


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                 kv_len: torch.Tensor, q_start: torch.Tensor, q=None, q_weight=None, k_weight=None, table=None,
                 eps: float = 1e-6, interleaved: bool = False):
    """Writes k [T, H_kv, D] and v [T, H_kv, D_v] at their positions in the pools.

    With ``k_weight`` the keys are normed, with ``table`` (``rotary_table``)
    rotated by their position, before they are written; ``q`` [T, H_q, D] gets
    the same (with ``q_weight``) and is returned, else None.  Rows of the result
    behind the last sequence are not written.  Positions that two sequences
    share (a page entered in both tables) must get the same rows from both, and
    k, v and q may lie in the pools only in rows that the call does not write."""
    dt = _dtype_of(k)
    if k.dim() != 3:
        raise InvalidArgumentError(f"k must be [T, H_kv, D] but is rank {k.dim()}")
    if not k.is_cuda:
        raise InvalidArgumentError(_CUDA_MSG)
    dtype, device, T = k.dtype, k.device, k.shape[0]
    P, page, H_kv, D, D_v = _check_pools(k_pages, v_pages, dtype, device)
    N, M = _check_batch(page_table, kv_len, q_start, device)
    _check_tokens(k, "k", T, D, H_kv, dtype)
    _check_tokens(v, "v", T, D_v, H_kv, dtype)
    _same(v, device, "v")
    if q is not None:
        _check_tokens(q, "q", T, D, None, dtype)
        _same(q, device, "q")
    elif q_weight is not None:
        raise InvalidArgumentError("q_weight without q")
    qw, kw, wdt = _weights(q_weight, k_weight, dtype, device, D)
    table, max_pos, rot = _table(table, device, D)
    align = 8 if dt == _lib.F16 else 4
    kx, ks = _rows(k, H_kv * D, align)
    vx, vs = _rows(v, H_kv * D_v, align)
    q_out, qx, qs, H_q = None, None, 0, 0
    if q is not None:
        H_q = q.shape[1]
        qx, qs = _rows(q, H_q * D, align)
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    _launch(device, _lib.lib().sdpa_b200_paged_append, dt, _ptr(qx), qs, kx.data_ptr(), ks, vx.data_ptr(), vs, T, H_q, H_kv, D,
            D_v, _ptr(qw), _ptr(kw), wdt, float(eps), _ptr(table), max_pos, rot, int(bool(interleaved)), _ptr(q_out),
            k_pages.data_ptr(), v_pages.data_ptr(), P, page, page_table.data_ptr(), M, kv_len.data_ptr(), q_start.data_ptr(), N)
    return q_out


def _span(x: torch.Tensor):
    """First byte and end of the stretch of memory that holds a tensor's elements (strides are not negative)."""
    at = x.data_ptr()
    if x.is_contiguous():
        return at, at + x.nbytes
    return at, at + (1 + sum((n - 1) * s for n, s in zip(x.shape, x.stride()))) * x.element_size()


def _meet(a, b) -> bool:
    return a[0] < b[1] and b[0] < a[1] and a[0] < a[1] and b[0] < b[1]


def _share_bytes(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the stretches of memory of two tensors meet."""
    return _meet(_span(a), _span(b))


_workspace_bytes: dict = {}  # of paged_sdpa, by what the query depends on


def paged_sdpa(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
               kv_len: torch.Tensor, q_start: torch.Tensor, scale: float = 1.0, causal_mask: bool = True, *, out=None):
    """Attention of new tokens q [T, H_q, D] over the cached keys of their sequences.

    Returns (output [T, H_q, D_v] T, stats [T, H_q] float32), stats as in
    ``sdpa``: max + ln(sum + 1e-6) of the scaled scores; no gradients.  H_q is a multiple of
    H_kv; query head h reads KV head h // (H_q / H_kv).  With ``causal_mask`` a
    token sees the keys up to its own position, else all kv_len of its sequence;
    one that sees none gets zeros and stats of -1e9.  ``out`` may pass
    (output, stats) to write into, memory apart from the inputs'; rows behind the last sequence keep what they
    held (and hold anything in a result allocated here).  A NaN or infinity
    cached behind a sequence's kv_len reaches nothing; one at a position that
    only later tokens of the same chunk see may reach the chunk's earlier rows.
    In float, products are taken of two parts of each value: an infinity gives
    NaN, finite values may have any size up to 2^128 (1 - 2^-12) as long as
    scores and sum_j exp(score_j - max) v_j stay in float's range."""
    dt = _dtype_of(q)
    if q.dim() != 3:
        raise InvalidArgumentError(f"q must be [T, H_q, D] but is rank {q.dim()}")
    if not q.is_cuda:
        raise InvalidArgumentError(_CUDA_MSG)
    dtype, device = q.dtype, q.device
    T, H_q, q_D = q.shape
    P, page, H_kv, D, D_v = _check_pools(k_pages, v_pages, dtype, device)
    N, M = _check_batch(page_table, kv_len, q_start, device)
    if q_D != D:
        raise InvalidArgumentError(f"q must be [{T}, H, {D}], got {list(q.shape)}")
    if H_q < 1 or H_q % H_kv:
        raise InvalidArgumentError("H_q must be a multiple of H_kv")
    if out is None:
        o = torch.empty_like(q, memory_format=torch.contiguous_format) if D_v == D else torch.empty(
            (T, H_q, D_v), dtype=dtype, device=device)
        stats = torch.empty((T, H_q), dtype=torch.float32, device=device)
    else:
        o, stats = out
        if tuple(o.shape) != (T, H_q, D_v) or o.dtype != dtype or not o.is_contiguous() or o.data_ptr() % 16:
            raise InvalidArgumentError("out[0] must be a contiguous [T, H_q, D_v] tensor of dtype T, 16-byte aligned")
        if tuple(stats.shape) != (T, H_q) or stats.dtype != torch.float32 or not stats.is_contiguous():
            raise InvalidArgumentError("out[1] must be a contiguous float32 [T, H_q] tensor")
        _same(o, device, "out[0]")
        _same(stats, device, "out[1]")
        # (other blocks still read what one has written over)
        at = (("q", _span(q)), ("k_pages", _span(k_pages)), ("v_pages", _span(v_pages)), ("page_table", _span(page_table)),
              ("kv_len", _span(kv_len)), ("q_start", _span(q_start)))
        to = _span(o), _span(stats)
        for i in (0, 1):
            for name, span in at:
                if _meet(to[i], span):
                    raise InvalidArgumentError(f"out[{i}] must not share memory with {name}")
        if _meet(*to):
            raise InvalidArgumentError("out[0] and out[1] must not share memory")
    if T == 0 or N == 0:
        return o, stats
    qx, qs = _rows(q, H_q * D, 8 if dt == _lib.F16 else 4)
    L = _lib.lib()
    key = (dt, T, N, H_q, H_kv, D, D_v, device.index)
    ws_bytes = _workspace_bytes.get(key)
    if ws_bytes is None:
        with torch.cuda.device(device):
            ws_bytes = L.sdpa_b200_paged_workspace_bytes(dt, T, N, H_q, H_kv, D, D_v)
        if len(_workspace_bytes) >= 4096:
            _workspace_bytes.clear()
        _workspace_bytes[key] = ws_bytes
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
    _launch(device, L.sdpa_b200_paged_sdpa, dt, qx.data_ptr(), qs, k_pages.data_ptr(), v_pages.data_ptr(), o.data_ptr(),
            stats.data_ptr(), T, H_q, H_kv, D, D_v, P, page, page_table.data_ptr(), M, kv_len.data_ptr(), q_start.data_ptr(), N,
            float(scale), int(bool(causal_mask)), ws.data_ptr(), ws_bytes)
    return o, stats


class PagedBatch:
    """The index tensors of one serving step (``PagedCache.batch``): page_table, kv_len, q_start, and its tokens.

    ``longest``: the largest kv_len of a sequence with new tokens, for checks on the host; None where only the device
    knows the lengths."""

    __slots__ = ("page_table", "kv_len", "q_start", "tokens", "longest")

    def __init__(self, page_table, kv_len, q_start, tokens: int, longest: int | None = None):
        self.page_table, self.kv_len, self.q_start, self.tokens = page_table, kv_len, q_start, tokens
        self.longest = longest


class PagedCache:
    """Pools of one attention layer and the page accounting of its sequences.

    ``batch([(sequence, new_tokens), ..])`` reserves room for the new tokens
    (sequence ids are any hashable; a new id starts an empty sequence) and
    returns the step's ``PagedBatch``; ``append`` and ``attend`` run on it;
    ``free`` gives a sequence's pages back.  Several layers with equal lengths can
    share one cache object's accounting by passing its batches to their own
    pools (``paged_append`` / ``paged_sdpa``)."""

    def __init__(self, pages: int, page_size: int, heads: int, head_dim: int, value_dim=None, dtype=torch.float16, device=None):
        dev = torch.device(device or "cuda")
        _dtype_of(torch.empty(0, dtype=dtype))  # fp16 or fp32
        self.k_pages = torch.zeros(pages, page_size, heads, head_dim, dtype=dtype, device=dev)
        self.v_pages = torch.zeros(pages, page_size, heads, head_dim if value_dim is None else value_dim, dtype=dtype, device=dev)
        _check_pools(self.k_pages, self.v_pages, dtype, self.k_pages.device)
        self.page_size = page_size
        self._free = list(range(pages - 1, -1, -1))
        self._pages: dict = {}   # sequence -> its pages in order
        self._length: dict = {}  # sequence -> cached tokens

    def length(self, sequence) -> int:
        """Tokens cached (or reserved) for a sequence; 0 for one that is not held."""
        return self._length.get(sequence, 0)

    def batch(self, new_tokens) -> PagedBatch:
        """Reserves `count` further tokens for each (sequence, count); nothing is reserved if the pages do not suffice."""
        new_tokens = [(s, int(c)) for s, c in new_tokens]
        seen = {s for s, _ in new_tokens}
        if len(seen) != len(new_tokens):
            raise InvalidArgumentError("a sequence may appear once in a batch")
        if any(c < 0 for _, c in new_tokens):
            raise InvalidArgumentError("token counts must not be negative")
        need = {s: -(-(self.length(s) + c) // self.page_size) - len(self._pages.get(s, ())) for s, c in new_tokens}
        if sum(need.values()) > len(self._free):
            raise InvalidArgumentError(f"the cache has {len(self._free)} free pages, the batch needs {sum(need.values())}")
        start, rows, lengths = [0], [], []
        for s, c in new_tokens:
            pages = self._pages.setdefault(s, [])
            pages.extend(self._free.pop() for _ in range(need[s]))
            self._length[s] = self.length(s) + c
            rows.append(pages)
            lengths.append(self._length[s])
            start.append(start[-1] + c)
        width = max([1, *map(len, rows)])
        index = torch.tensor([x for r in rows for x in (*r, *[-1] * (width - len(r)))] + lengths + start, dtype=torch.int32)
        index = index.to(self.k_pages.device)  # one copy for the three
        n = len(rows)
        table, kv_len, q_start = index.split([n * width, n, n + 1])
        return PagedBatch(table.view(n, width), kv_len, q_start, start[-1],
                          max((self._length[s] for s, c in new_tokens if c), default=0))

    def free(self, sequence):
        self._free.extend(reversed(self._pages.pop(sequence, [])))
        self._length.pop(sequence, None)

    def append(self, k, v, batch: PagedBatch, **kw):
        """``paged_append`` into this cache's pools."""
        return paged_append(k, v, self.k_pages, self.v_pages, batch.page_table, batch.kv_len, batch.q_start, **kw)

    def attend(self, q, batch: PagedBatch, **kw):
        """``paged_sdpa`` over this cache's pools."""
        return paged_sdpa(q, self.k_pages, self.v_pages, batch.page_table, batch.kv_len, batch.q_start, **kw)

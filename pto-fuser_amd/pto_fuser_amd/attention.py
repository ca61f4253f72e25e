"""Attention of a served model, for the attention layers that stand among recurrent ones.

* :func:`causal_attention` — a whole prompt, or several of different lengths packed into one buffer.
* :func:`attention_step` — one new token of each running sequence over a cache of keys and values in pages.
* :func:`assign_pages`, :func:`release_pages` — which pages of the cache new tokens take and which row each has, and back.
* :func:`store_kv` — keys and values into those rows.
* :func:`refuse_held` — marks the requests of a plan for which attention over its new tokens alone would be wrong.

No counterpart in the reference.  Forward only.  As in ``serving``: operands may be views whose innermost dimension is
contiguous, every operator raises ``ValueError`` before launching for what it does not support, works on the current stream of
the operands' device, and neither synchronises nor allocates anything but its outputs, scratch and operands that it has to copy.

A cache is two tensors [pages, page, G, D], views allowed; a page holds a power of two of rows from 16 to 65536, and a row of
the cache is named by page · page_size + offset.  ``tables`` [S, M] int32 holds the pages of S sequences, ``slots`` [B] int32
names each request's row of it as it names states elsewhere (no two the same; one outside the pool has no tokens; None: row b).
"""
from __future__ import annotations

import functools
import struct
from typing import NamedTuple, Optional

import torch

from . import _hip
from .ops import _dtype_code, _require
from .serving import _apart, _device_of, _dim, _exec, _pool, _ptr, _require_view, _size, _span

_ATTN = struct.Struct("@N6P8q7if")
_ATTN_STEP = struct.Struct("@N8PN10q9if")
_ASSIGN = struct.Struct("@N10P6i")
_RELEASE = struct.Struct("@N6P5i")
_REFUSE = struct.Struct("@N4P2q4i")
_STORE = struct.Struct("@N5P10q6i")
_ATTN_SIZE, _ATTN_STEP_SIZE, _ASSIGN_SIZE, _RELEASE_SIZE, _REFUSE_SIZE, _STORE_SIZE = (
    _size(s) for s in (_ATTN, _ATTN_STEP, _ASSIGN, _RELEASE, _REFUSE, _STORE))

HEAD_MAX = 256
ROW_MAX_STRIDE = 1 << 22
MAX_TOKENS = 1 << 30


def _heads(H: int, G: int, D: int) -> None:
    if H == 0 or G == 0 or H % G or not 0 < D <= HEAD_MAX or D % 8:
        raise ValueError(f"unsupported shape H={H} G={G} D={D} (H a multiple of G, D of 8 up to {HEAD_MAX})")


def _needed(t, name: str, shape, dtype, dev) -> None:
    if t is None:
        raise ValueError(f"{name} must be a tensor")
    _require(t, name, shape, dtype, dev)


def _scale(scale: Optional[float], D: int) -> float:
    scale = D ** -0.5 if scale is None else float(scale)
    if not 1e-30 < scale < 1e30:
        raise ValueError(f"scale must be positive and between 1e-30 and 1e30, got {scale}")
    return scale


def _page(page: int) -> None:
    if not 16 <= page <= 65536 or page & (page - 1):
        raise ValueError(f"a page holds a power of two of rows from 16 to 65536, got {page}")


def _vectors(t: torch.Tensor, strides) -> bool:
    """Whether rows with these strides, where ``t`` starts, are whole 16-byte vectors."""
    each = 16 // t.element_size()
    if t.data_ptr() % 16:
        return False
    for s in strides:
        if s % each:
            return False
    return True


def _strides(t: torch.Tensor):
    """Strides of all but the last dimension; 0 where there is nothing to step to, whatever the tensor says."""
    s, n = t.stride()[:-1], t.shape
    return s if 1 not in n else tuple([0 if m == 1 else x for x, m in zip(s, n)])


def _ends(t: torch.Tensor):
    """The address of a tensor's first byte and that after its last."""
    lo = t.data_ptr()
    return lo, lo + (t.numel() * t.element_size() if t.is_contiguous() else _span(t))


def _clear(name: str, t: torch.Tensor, **others) -> None:
    """``t``, which a call writes, overlaps neither itself nor ``others``: by their ends, and where those do not say, by
    :func:`serving._apart`."""
    if not t.is_contiguous():
        return _apart(name, t, **others)
    lo, hi = _ends(t)
    for u in others.values():
        if u is not None:
            at = u.data_ptr()
            if at < hi and (at >= lo or _ends(u)[1] > lo):
                return _apart(name, t, **others)


def _cache(k_cache, v_cache, dtype, dev):
    _dim(k_cache, "k_cache", 4, "[pages,page,G,D]")
    shape = k_cache.shape
    _page(shape[1])
    _require_view(k_cache, "k_cache", shape, dtype, dev)
    _require_view(v_cache, "v_cache", shape, dtype, dev)
    return shape


def _tables(tables, slots, B: int, dev):
    _dim(tables, "tables", 2, "[S,M]")
    shape = tables.shape
    _require(tables, "tables", shape, torch.int32, dev)
    if slots is not None or shape[0] != B:
        _pool(tables, slots, B, dev)
    return shape


def _rows(t: torch.Tensor):
    """``t`` as the kernels read it, copied where its rows are no whole vectors or lie too far apart, and its strides."""
    s = _strides(t)
    if s[0] <= ROW_MAX_STRIDE and _vectors(t, s):
        return t, s
    t = t.clone(memory_format=torch.contiguous_format)
    return t, _strides(t)


def causal_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, *,
                     lengths: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention over prompts packed in one buffer: o_i = Σ_{j≤i} softmax_j(scale · q_i·k_j) v_j within each prompt.

    q [N,H,D], k and v [N,G,D], float32 or bfloat16, D a multiple of 8 up to 256, query head h reading head h // (H // G) of
    keys and values; token and head strides are free (operands whose rows are not whole 16-byte vectors, or whose tokens lie
    more than 2^22 elements apart, are copied first).  ``cu_seqlens`` [B+1] int32, rising: prompt b has rows cu_seqlens[b] up
    to cu_seqlens[b+1], of which the first ``lengths[b]`` (int32; None: all) are live; a padded batch [B,T] has cu_seqlens of
    multiples of T.  Scores, maxima and sums are held in 32 bits; with bfloat16 operands the weights enter the product with v
    in bfloat16.  A value that is not finite reaches its own token and later ones of its prompt, and none before.

    Returns o [N,H,D] in q's type.  Rows of no live token are zero, or in a given ``out`` left as they were.  ``scale``
    (positive) is D^-1/2 by default."""
    dev = _device_of(q, "q")
    _dim(q, "q", 3, "[N,H,D]")
    _dim(k, "k", 3, "[N,G,D]")
    N, H, D = q.shape
    G, code, dtype = k.shape[1], _dtype_code(q.dtype), q.dtype
    _heads(H, G, D)
    if N > MAX_TOKENS:
        raise ValueError(f"q has {N} rows (up to {MAX_TOKENS})")
    _require_view(q, "q", (N, H, D), dtype, dev)
    _require_view(k, "k", (N, G, D), dtype, dev)
    _require_view(v, "v", (N, G, D), dtype, dev)
    _dim(cu_seqlens, "cu_seqlens", 1, "[B+1]")
    B = cu_seqlens.shape[0] - 1
    if B < 0:
        raise ValueError("cu_seqlens must have an entry more than there are prompts")
    _require(cu_seqlens, "cu_seqlens", (B + 1,), torch.int32, dev)
    if lengths is not None:
        _require(lengths, "lengths", (B,), torch.int32, dev)
    scale = _scale(scale, D)
    if out is None:
        o = torch.empty(N, H, D, device=dev, dtype=dtype)
    else:
        _require_view(out, "out", (N, H, D), dtype, dev)
        _clear("out", out, q=q, k=k, v=v, cu_seqlens=cu_seqlens, lengths=lengths)
        o = out
    q, sq = _rows(q)
    k, sk = _rows(k)
    v, sv = _rows(v)
    _exec("pf_attn_exec", dev, _ATTN, _ATTN_SIZE, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
          cu_seqlens.data_ptr(), _ptr(lengths), *sq, *sk, *sv, *_strides(o), N, B, H, G, D, code, int(out is None), scale)
    return o


@functools.lru_cache(maxsize=1024)
def _step_workspace(*sizes: int) -> int:
    return _hip.load().pf_attn_step_workspace_bytes(*sizes)


def attention_step(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, tables: torch.Tensor,
                   lengths: torch.Tensor, *, slots: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One new token of each of B sequences over its cache: o = Σ_j softmax_j(scale · q·k_j) v_j over its ``lengths[b]`` tokens,
    the new one (stored before) among them.

    q [B,H,D] float32 or bfloat16; k_cache, v_cache [pages,page,G,D] in its type, whole 16-byte vectors; D, H and G as in
    :func:`causal_attention`.  Sequence b's pages are ``tables[slots[b]]``; entries past its length are not read, and a page
    outside the cache holds no tokens.  lengths [B] int32, cut at M · page.  A sequence of no tokens gives zeros.  An infinity
    or NaN in v reaches its own column, as in the formula; what lies behind a sequence's tokens reaches nothing.  The keys of all
    sequences are shared out evenly over the chip, so the same sequence alone and in a batch may differ by rounding.
    Returns o [B,H,D] in q's type."""
    dev = _device_of(q, "q")
    _dim(q, "q", 3, "[B,H,D]")
    B, H, D = q.shape
    code, dtype = _dtype_code(q.dtype), q.dtype
    pages, page, G, Dk = _cache(k_cache, v_cache, dtype, dev)
    if Dk != D:
        raise ValueError(f"k_cache has heads of {Dk}, expected {D}")
    _heads(H, G, D)
    _require_view(q, "q", (B, H, D), dtype, dev)
    S, M = _tables(tables, slots, B, dev)
    _needed(lengths, "lengths", (B,), torch.int32, dev)
    if M * page > MAX_TOKENS:
        raise ValueError(f"tables hold {M} pages of {page} (up to {MAX_TOKENS} tokens)")
    sk, sv = _strides(k_cache), _strides(v_cache)
    for name, t, s in (("k_cache", k_cache, sk), ("v_cache", v_cache, sv)):
        if pages and (s[1] > ROW_MAX_STRIDE or not _vectors(t, s)):
            raise ValueError(f"{name} must be whole 16-byte vectors, its rows up to {ROW_MAX_STRIDE} elements apart")
    scale = _scale(scale, D)
    if out is None:
        o = torch.empty(B, H, D, device=dev, dtype=dtype)
    else:
        _require_view(out, "out", (B, H, D), dtype, dev)
        _clear("out", out, q=q, k_cache=k_cache, v_cache=v_cache, tables=tables, lengths=lengths, slots=slots)
        o = out
    q, sq = _rows(q)
    need = _step_workspace(B, H, G, D, M, page, code)
    ws = torch.empty(need, device=dev, dtype=torch.uint8) if need else None
    _exec("pf_attn_step_exec", dev, _ATTN_STEP, _ATTN_STEP_SIZE, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
          o.data_ptr(), tables.data_ptr(), lengths.data_ptr(), _ptr(slots), _ptr(ws), need, *sq, *_strides(o), *sk, *sv,
          B, S, H, G, D, M, pages, page, code, scale)
    return o


class PagePlan(NamedTuple):
    """Where the new tokens of a step or of arriving prompts go."""
    rows: torch.Tensor          # [capacity] int64: the cache row of each new token, -1 of none
    cu_seqlens: torch.Tensor    # [B+1] int32: the requests' new tokens among them
    lengths: torch.Tensor       # [B] int32: tokens of each request in the cache, the new ones among them
    taken: torch.Tensor         # [1] int32: pages taken from the pool


def _pool_state(tables, lengths, free, taken, slots, page_size: int, dev):
    _page(page_size)
    _dim(lengths, "lengths", 1, "[B]")
    B = lengths.shape[0]
    _require(lengths, "lengths", (B,), torch.int32, dev)
    S, M = _tables(tables, slots, B, dev)
    if M * page_size > MAX_TOKENS:
        raise ValueError(f"tables hold {M} pages of {page_size} (up to {MAX_TOKENS} tokens)")
    _dim(free, "free", 1, "[F]")
    _require(free, "free", free.shape, torch.int32, dev)
    _needed(taken, "taken", (1,), torch.int32, dev)
    return B, S, M, free.shape[0]


def assign_pages(tables: torch.Tensor, lengths: torch.Tensor, tokens: Optional[torch.Tensor], free: torch.Tensor,
                 taken: torch.Tensor, *, page_size: int, capacity: Optional[int] = None,
                 slots: Optional[torch.Tensor] = None) -> PagePlan:
    """Pages and cache rows for the new tokens of B requests, without the host knowing their lengths.

    ``lengths`` [B] int32: tokens of each request that the cache holds; ``tokens`` [B] int32: new ones of each (None: one
    each, a decoding step).  Pages are taken from ``free`` [F] int32 at ``taken`` [1] int32 on, for the requests in their
    order, and entered in ``tables`` (in place).  ``capacity`` (by default B, for a step): rows that the new tokens are
    packed into.

    A request is served whole or not at all: not where its slot is outside the pool, its tokens pass its table or the
    capacity, or its pages are more than the pool has left (after which no request that needs any is served).  Its rows are
    then -1, its length stays, and :func:`store_kv` skips it.  Returns a :class:`PagePlan`; lengths and taken are new tensors,
    which the caller passes on the next time."""
    dev = _device_of(tables, "tables")
    B, S, M, F = _pool_state(tables, lengths, free, taken, slots, page_size, dev)
    if tokens is not None:
        _require(tokens, "tokens", (B,), torch.int32, dev)
    if capacity is None:
        if tokens is not None:
            raise ValueError("capacity must be given with tokens")
        capacity = B
    if not 0 <= capacity <= MAX_TOKENS:
        raise ValueError(f"capacity must be 0 to {MAX_TOKENS}, got {capacity}")
    _clear("tables", tables, lengths=lengths, tokens=tokens, free=free, taken=taken, slots=slots)
    rows = torch.empty(capacity, device=dev, dtype=torch.int64)
    cu, after, taken_after = torch.empty(2 * B + 2, device=dev, dtype=torch.int32).split_with_sizes([B + 1, B, 1])
    _exec("pf_assign_exec", dev, _ASSIGN, _ASSIGN_SIZE, tables.data_ptr(), lengths.data_ptr(), _ptr(tokens), _ptr(slots),
          free.data_ptr(), taken.data_ptr(), rows.data_ptr(), cu.data_ptr(), after.data_ptr(), taken_after.data_ptr(),
          B, S, M, F, capacity, page_size)
    return PagePlan(rows, cu, after, taken_after)


def release_pages(tables: torch.Tensor, lengths: torch.Tensor, free: torch.Tensor, taken: torch.Tensor, *, page_size: int,
                  slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The pages of B requests that leave go back to ``free`` (in place), below ``taken``; returns taken afterwards [1].

    ``lengths`` [B] int32: tokens that each request holds, whose pages its table names; the caller sets them to 0.  A
    request is refused, and keeps its pages, where more would come back than were taken."""
    dev = _device_of(tables, "tables")
    B, S, M, F = _pool_state(tables, lengths, free, taken, slots, page_size, dev)
    _clear("free", free, tables=tables, lengths=lengths, taken=taken, slots=slots)
    after = torch.empty(1, device=dev, dtype=torch.int32)
    _exec("pf_release_exec", dev, _RELEASE, _RELEASE_SIZE, tables.data_ptr(), lengths.data_ptr(), _ptr(slots),
          free.data_ptr(), taken.data_ptr(), after.data_ptr(), B, S, M, F, page_size)
    return after


def _outside(at: int, size: int, other: int, other_size: int) -> bool:
    return other + other_size <= at or at + size <= other


def refuse_held(k: torch.Tensor, plan: PagePlan) -> None:
    """Makes attention over a plan's new tokens alone give NaN for requests that held tokens before it, which those tokens would
    have to see: their first key in k [N,G,D], N the plan's capacity, becomes NaN (in place; k is stored before).  Nothing on
    the host knows which those are."""
    dev = _device_of(k, "k")
    _dim(k, "k", 3, "[N,G,D]")
    N, G, D = k.shape
    code = _dtype_code(k.dtype)
    if not 0 < G <= 65536 or D == 0:
        raise ValueError(f"unsupported shape G={G} D={D} (G up to 65536)")
    _require_view(k, "k", (N, G, D), k.dtype, dev)
    rows, cu, lengths = plan.rows, plan.cu_seqlens, plan.lengths
    _dim(lengths, "lengths", 1, "[B]")
    B = lengths.shape[0]
    _needed(rows, "rows", (N,), torch.int64, dev)
    _needed(cu, "cu_seqlens", (B + 1,), torch.int32, dev)
    _needed(lengths, "lengths", (B,), torch.int32, dev)
    at, at_rows, at_cu, at_lengths, (st, sh) = k.data_ptr(), rows.data_ptr(), cu.data_ptr(), lengths.data_ptr(), k.stride()[:2]
    span = ((N - 1) * st + (G - 1) * sh + D) * k.element_size()
    # (by their ends where those say enough, as in store_kv: 4 us less of the host)
    if not (0 < D <= sh and (G - 1) * sh + D <= st and _outside(at, span, at_rows, 8 * N) and _outside(at, span, at_cu, 4 * B + 4)
            and _outside(at, span, at_lengths, 4 * B)):
        _apart("k", k, rows=rows, cu_seqlens=cu, lengths=lengths)
    _exec("pf_refuse_exec", dev, _REFUSE, _REFUSE_SIZE, at_cu, at_lengths, at_rows, at, st, sh, N, B, G, code)


def _caches_clear(k_cache, v_cache, held: int, others) -> bool:
    """Whether two caches of ``held`` bytes each, and the ranges of bytes ``others``, plainly lie apart: by their ends alone,
    which takes 2.7 us less of the host than :func:`serving._apart` through :func:`_clear`, of the 11 of a small call."""
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        return False
    first, last = sorted((k_cache.data_ptr(), v_cache.data_ptr()))
    if first + held > last:
        return False
    for lo, hi in others:
        if lo < last + held and hi > first and (lo < first + held or hi > last):
            return False
    return True


def store_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, rows: torch.Tensor) -> None:
    """Keys and values k, v [N,G,D] of N tokens into their rows of the cache [pages,page,G,D] (in place), all of one type.

    ``rows`` [N] int64, as :func:`assign_pages` gives them: one outside the cache (-1) is skipped, no two others are the same.
    float32 or bfloat16, D a multiple of 8; token and head strides of k and v are free."""
    dev = _device_of(k, "k")
    _dim(k, "k", 3, "[N,G,D]")
    N, G, D = k.shape
    code, dtype = _dtype_code(k.dtype), k.dtype
    if not 0 < G <= 65536 or not 0 < D <= 65536 or D % 8:
        raise ValueError(f"unsupported shape G={G} D={D} (D a multiple of 8; both up to 65536)")
    _require_view(k, "k", (N, G, D), dtype, dev)
    _require_view(v, "v", (N, G, D), dtype, dev)
    pages, page, Gc, Dc = _cache(k_cache, v_cache, dtype, dev)
    if (Gc, Dc) != (G, D):
        raise ValueError(f"k_cache has {Gc} heads of {Dc}, expected {G} of {D}")
    _needed(rows, "rows", (N,), torch.int64, dev)
    sk, sv, at_k, at_v, at_rows = k.stride(), v.stride(), k.data_ptr(), v.data_ptr(), rows.data_ptr()
    size = k.element_size()
    if not _caches_clear(k_cache, v_cache, k_cache.numel() * size,
                         ((at_k, at_k + ((N - 1) * sk[0] + (G - 1) * sk[1] + D) * size),
                          (at_v, at_v + ((N - 1) * sv[0] + (G - 1) * sv[1] + D) * size), (at_rows, at_rows + 8 * N))):
        _apart("k_cache", k_cache, k=k, v=v, v_cache=v_cache, rows=rows)
        _apart("v_cache", v_cache, k=k, v=v, rows=rows)
    _exec("pf_store_exec", dev, _STORE, _STORE_SIZE, at_k, at_v, k_cache.data_ptr(), v_cache.data_ptr(), at_rows, *sk[:2],
          *sv[:2], *k_cache.stride()[:3], *v_cache.stride()[:3], N, G, D, pages, page, code)

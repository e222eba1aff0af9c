"""Paged caches on the gfx950 library (``include/hz_paged.h``): keys and values of many rows of tokens (walkers
sampled site by site, requests) in a pool of pages, next to the token operators of
:mod:`hamiltonzero_amd.tokens`. The reference has no counterpart.

* :func:`paged_append` — new tokens' keys and values into their slots.
* :func:`paged_attention` — attention of new tokens over the slots of their rows; on request adds up the
  weights that each slot has had.
* :func:`paged_evict` — gives up the slots of least such weight and closes the cache over them, in place.

A cache is ``k_cache, v_cache [pages, page_size, Hk, D]`` (strided views are read and written in place: rows of D
contiguous elements, 16-byte aligned; a pool ``[pages, Hk, page_size, D]`` goes in transposed), with
``page_table [B, width]`` and ``lengths [B]``, int32 on the GPU and read there. Row b has the slots ``0 .. lengths[b] - 1``
(clamped to ``width * page_size``, its most), slot j in page ``page_table[b, j // page_size]`` at ``j % page_size``. Rows may
share pages that no call writes. An entry that is no page (negative, or not below ``pages``) hides its slots: the attention
does not see them, the append does not write them, the eviction does not move them (its results count them as slots like others, by
their scores). Slots from ``lengths[b]`` on are neither read nor written; those below must hold finite values.

Calls for inference: none has a gradient. Work goes to the current stream of the tensors' device; there is no CPU
fallback. What a call writes counts as changed in place.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch.autograd.graph import increment_version

from . import _native
from .tokens import MAX_HEAD_DIM, _DTYPES, _check, _check_first, _end, _fields, _float32, _holds_twice, _on, _overlap, _ptr, _stream, _strided, _wants_grad

Tensor = torch.Tensor


def _in_place(name: str, t: Tensor) -> tuple:
    """Address and strides of a cache that the kernels read and write where it is."""
    fields = _fields(t)
    if not t.is_contiguous() and (t.stride(3) != 1 or fields[1] % 8 or fields[2] % 8 or fields[3] % 8) or fields[0] % 16:
        raise ValueError(f"{name} must have contiguous heads and 16-byte aligned rows, got strides {t.stride()}")
    return fields


def _cache(k_cache: Tensor, v_cache: Tensor, page_table: Tensor, lengths: Tensor) -> Tuple[bytes, tuple]:
    """The library's structure of a checked cache, and ``(B, slots, Hk, D)``. The tables that it points to are the caller's: they
    stay as long as its arguments do."""
    _check_first("k_cache", k_cache, "[pages, page_size, Hk, D]")
    shape = k_cache.shape
    P, S, Hk, D = shape
    dev, dtype = k_cache.device, k_cache.dtype
    if D % 8 or D > MAX_HEAD_DIM:
        raise ValueError(f"head dimension must be a multiple of 8 up to {MAX_HEAD_DIM}, got {D}")
    _check("v_cache", v_cache, dev, dtype, shape)
    if not isinstance(page_table, Tensor) or page_table.dim() != 2 or page_table.numel() == 0:
        raise ValueError("page_table must be [B, width] with both axes at least 1 long")
    table_shape = page_table.shape
    B, width = table_shape
    _check("page_table", page_table, dev, torch.int32, table_shape)
    _check("lengths", lengths, dev, torch.int32, (B,))
    if not page_table.is_contiguous() or not lengths.is_contiguous():
        raise ValueError("page_table and lengths must be contiguous")
    args = _native.PAGED_CACHE.pack(*_in_place("k_cache", k_cache), *_in_place("v_cache", v_cache), page_table.data_ptr(),
                                    lengths.data_ptr(), B, P, S, width, Hk, D, _DTYPES[dtype])
    return args, (B, width * S, Hk, D)


def _range(t: Tensor) -> Tuple[int, int]:
    begin = t.data_ptr()
    return begin, begin + t.numel() * t.element_size() if t.is_contiguous() else _end(t)


def _touches(t: Tensor, others: Tuple[Tensor, ...]) -> bool:
    """Whether ``t`` shares memory with any of ``others``; ranges of addresses first, which mostly are apart."""
    t0, t1 = _range(t)
    for x in others:
        begin, end = _range(x)
        if t0 < end and begin < t1 and _overlap(t, x):
            return True
    return False


def _check_written(k_cache: Tensor, v_cache: Tensor, names: str, *others: Tensor) -> None:
    """The caches of a call that writes them: no element at two places, apart from each other and from ``others``, called ``names``."""
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if _holds_twice(t):
            raise ValueError(f"{name} must not hold one element at several places, got strides {t.stride()}")
    (k0, k1), (v0, v1) = _range(k_cache), _range(v_cache)
    if k0 < v1 and v0 < k1 and _overlap(k_cache, v_cache):
        raise ValueError("k_cache and v_cache must not overlap")
    for t in others:
        t0, t1 = _range(t)
        if (t0 < k1 and k0 < t1 and _overlap(t, k_cache)) or (t0 < v1 and v0 < t1 and _overlap(t, v_cache)):
            raise ValueError(f"{names} must not overlap the caches")


def _no_grad(*tensors: Optional[Tensor]) -> None:
    if _wants_grad(*tensors):
        raise ValueError("the paged operators have no gradients: call under torch.no_grad()")


def paged_append(k_cache: Tensor, v_cache: Tensor, k: Tensor, v: Tensor, page_table: Tensor, lengths: Tensor) -> None:
    """Writes the N new tokens ``k, v [B, N, Hk, D]`` of each row into its last slots: token i of row b into slot
    ``lengths[b] - N + i`` (``lengths`` count the new tokens already). Tokens of negative slots (the padded front of a prompt that is
    shorter than N) are left out; where a length is more than the table's slots, the row's last slots take the new
    tokens. ``k`` and ``v`` may be strided views; they must not overlap the caches, and no page may take two rows' new
    tokens at one slot."""
    args, (B, _, Hk, D) = _cache(k_cache, v_cache, page_table, lengths)
    _check_first("k", k, "[B, N, Hk, D]")
    N = k.shape[1]
    for name, t in (("k", k), ("v", v)):
        _check(name, t, k_cache.device, k_cache.dtype, (B, N, Hk, D))
    _check_written(k_cache, v_cache, "k and v", k, v)
    _no_grad(k_cache, v_cache, k, v)
    k, v = _strided(k), _strided(v)
    with _on(k_cache.device):
        _native.check(_native.lib().hz_paged_append(_stream(k_cache.device), args, _native.TOKEN_TENSOR.pack(*_fields(k)),
                                                    _native.TOKEN_TENSOR.pack(*_fields(v)), N))
    increment_version((k_cache, v_cache))


def paged_attention(
    q: Tensor,
    k_cache: Tensor,
    v_cache: Tensor,
    page_table: Tensor,
    lengths: Tensor,
    *,
    scale: Optional[float] = None,
    softcap: float = 0.0,
    slopes: Optional[Tensor] = None,
    scores: Optional[Tensor] = None,
    decay: float = 1.0,
    scores_out: Optional[Tensor] = None,
) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """Attention of the last tokens of each row, ``q [B, Nq, H, D]`` (one, or a few), over its slots: query i stands at position
    ``p = lengths[b] - Nq + i``, its key and value are in the cache already, and it sees the slots up to p. Scores as
    :func:`~hamiltonzero_amd.token_attention`'s with ``causal``: query head h uses key head ``h // (H // Hk)``, ``softcap``
    caps them, ``slopes`` (float32 ``[H]``) times the distance in slots is taken off. A query that sees no slot gets zeros.
    Returns ``out`` shaped as ``q``.

    With ``scores`` (float32 ``[B, Hk, width * page_size]``, the weights that each slot has had) returns ``(out,
    new_scores)``: ``decay * scores`` plus the sum of the weights that the queries and heads of the key head
    give the slot now, and 0 from ``lengths[b]`` on; in a new tensor or in ``scores_out``, which may be ``scores`` and must not overlap
    ``q`` or the caches. Its sums are float32, of weights that are not rounded. Such a call takes workspace for a score of every query, head and slot
    of the table, 4 bytes each, whatever the lengths: keep ``width`` near what the rows need.

    For a few queries: the slots are read once for up to 32 queries and heads of a key head (float32 heads above 64: 16), and again for every 32 more."""
    args, (B, slots, Hk, D) = _cache(k_cache, v_cache, page_table, lengths)
    dev = k_cache.device
    _check_first("q", q, "[B, Nq, H, D]")
    Nq, H = q.shape[1], q.shape[2]
    _check("q", q, dev, k_cache.dtype, (B, Nq, H, D))
    if H % Hk:
        raise ValueError(f"the query heads must be a multiple of the key heads, got {H} and {Hk}")
    if slopes is not None:
        _check("slopes", slopes, dev, torch.float32, (H,))
        slopes = slopes.contiguous()
    if scores is None:
        if scores_out is not None:
            raise ValueError("scores_out needs scores")
    else:
        _check("scores", scores, dev, torch.float32, (B, Hk, slots))
        if scores_out is not None and scores_out is not scores:
            _check("scores_out", scores_out, dev, torch.float32, (B, Hk, slots))
            if not scores_out.is_contiguous() or scores_out.data_ptr() % 16:
                raise ValueError("scores_out must be contiguous and 16-byte aligned")
            if _overlap(scores_out, scores) and (scores_out.data_ptr() != scores.data_ptr() or not scores.is_contiguous()):
                raise ValueError("scores_out must be scores or not overlap it")
    _no_grad(q, k_cache, v_cache, slopes, scores, scores_out)
    q = _strided(q)
    into = scores_out
    if scores is not None:
        if into is scores and (not scores.is_contiguous() or scores.data_ptr() % 16):
            raise ValueError("scores_out must be contiguous and 16-byte aligned")
        scores = scores.contiguous()
        if scores.data_ptr() % 16:
            scores = scores.clone()
        if into is None:
            into = torch.empty_like(scores)
        elif _touches(into, (q, k_cache, v_cache)):
            raise ValueError("scores_out must not overlap q or the caches")
    out = torch.empty((B, Nq, H, D), dtype=q.dtype, device=dev)
    args = args + _native.PAGED_ATTENTION_REST.pack(
        *_fields(q), out.data_ptr(), _ptr(slopes), _ptr(scores), _ptr(into), Nq, H,
        float(D) ** -0.5 if scale is None else _float32(scale), _float32(softcap), _float32(decay))
    lib = _native.lib()
    with _on(dev):
        size = lib.hz_paged_attention_workspace(args)
        work = torch.empty(size, dtype=torch.uint8, device=dev) if size > 0 else None
        _native.check(lib.hz_paged_attention(_stream(dev), args, _ptr(work), size))
    if scores is None:
        return out
    if scores_out is not None:
        increment_version((scores_out,))
    return out, into


def paged_evict(
    k_cache: Tensor,
    v_cache: Tensor,
    page_table: Tensor,
    lengths: Tensor,
    scores: Tensor,
    budget: int,
    *,
    sinks: int = 0,
    recent: int = 0,
) -> Tuple[Tensor, Tensor, Tensor]:
    """Cuts the rows longer than ``budget`` slots to it, for each key head by its own weights ``scores [B, Hk, width * page_size]``
    (float32, as :func:`paged_attention` adds them up; apart from the caches). Kept are the first ``sinks`` slots, the last ``recent`` ones, and
    of the others those of the largest scores (equal ones: the lowest slot first; a NaN is less than any number).

    The k-th kept slot at or behind the budget (ascending) moves to the k-th slot below it that was given up; what lies below the
    budget and is kept stays where it is. So a slot's number is no longer its token's position: call without ``slopes``
    afterwards, and let ``recent`` count tokens appended since the last eviction (rows cut at ``budget + recent`` slots or more).

    What is given up is not attended to again: results after it approximate those of the whole cache.

    Keys and values move in place. Returns ``(lengths, sources, scores)``, new tensors: ``min(lengths[b], budget)``; ``[B, Hk,
    min(budget, width * page_size)]`` int32, the slot whose token lies at s now, -1 from the new length on; and the scores
    at their new slots, 0 behind them. Rows that are cut must not share pages with other rows, and no row may have a page
    twice. Pages behind the budget are free afterwards."""
    args, (B, slots, Hk, D) = _cache(k_cache, v_cache, page_table, lengths)
    dev = k_cache.device
    _check("scores", scores, dev, torch.float32, (B, Hk, slots))
    for name, x in (("budget", budget), ("sinks", sinks), ("recent", recent)):
        if isinstance(x, bool) or not isinstance(x, int):
            raise TypeError(f"{name} must be an integer, got {type(x).__name__}")
    if not 1 <= budget < 1 << 30:
        raise ValueError(f"budget must be in [1, 2^30), got {budget}")
    if sinks < 0 or recent < 0 or sinks + recent > budget:
        raise ValueError(f"sinks and recent must not be negative and at most the budget together, got {sinks} and {recent} of {budget}")
    _no_grad(k_cache, v_cache, scores)
    scores = scores.contiguous()
    if scores.data_ptr() % 16:
        scores = scores.clone()
    _check_written(k_cache, v_cache, "scores", scores)
    new = torch.empty_like(scores)
    sources = torch.empty((B, Hk, min(budget, slots)), dtype=torch.int32, device=dev)
    new_lengths = torch.empty_like(lengths)
    args = args + _native.PAGED_EVICT_REST.pack(scores.data_ptr(), new.data_ptr(), sources.data_ptr(), new_lengths.data_ptr(),
                                                budget, sinks, recent)
    lib = _native.lib()
    with _on(dev):
        size = lib.hz_paged_evict_workspace(args)
        work = torch.empty(size, dtype=torch.uint8, device=dev) if size > 0 else None
        _native.check(lib.hz_paged_evict(_stream(dev), args, _ptr(work), size))
    increment_version((k_cache, v_cache))
    return new_lengths, sources, new


__all__ = ["paged_append", "paged_attention", "paged_evict"]

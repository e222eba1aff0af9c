"""float64 restatement of the paged operators (include/hz_paged.h), with bounds on what a kernel that rounds as documented may
be off by.

The rounding model is :mod:`oracle.token_oracle`'s. Joins of runs and of a run's waves multiply each sum by a power of two
whose exponent is a rounded difference (``2^-24`` of it, and of its value) and add it: 16 F covers them beside the sums
themselves. The weights that are added up are not rounded: P = 2^(s - largest) / sum is off by the score's and the sum's errors and by the
rounding of the difference; one below 2^-126, the least normal float32, is 0, which is off by less than that.
"""

from __future__ import annotations

import numpy as np

from .token_oracle import F, _sum_error


def rotation(x, freqs, positions, axes, interleaved, direction=1):
    """One of q or k ``[B, N, H, D]``; positions ``[B, N, A]``; a pair whose number is no axis stays."""
    nf, A = len(freqs), positions.shape[2]
    p = np.arange(nf)
    a, b = (2 * p, 2 * p + 1) if interleaved else (p, p + nf)
    known = (axes >= 0) & (axes < A)
    t = np.where(known, positions[:, :, np.where(known, axes, 0)].astype(np.float64) * freqs, 0)[:, :, None]
    cos, sin = np.cos(t), direction * np.sin(t)
    x = x.astype(np.float64)
    y = x.copy()
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    return y


def places(table, n, size, pages):
    """Page and place in it of the slots 0 .. n - 1 of one row, and which of them lie in a page."""
    j = np.arange(n)
    page = table[j // size]
    return page, j % size, (page >= 0) & (page < pages)


def length(n, table, size):
    return min(max(int(n), 0), len(table) * size)


def append(k_cache, v_cache, k, v, page_table, lengths):
    """In place."""
    P, S = k_cache.shape[:2]
    N = k.shape[1]
    for b in range(len(lengths)):
        n = length(lengths[b], page_table[b], S)
        page, at, known = places(page_table[b], n, S, P)
        for i in range(N):
            j = n - N + i
            if j >= 0 and known[j]:
                k_cache[page[j], at[j]] = k[b, i]
                v_cache[page[j], at[j]] = v[b, i]


def attention(q, k_cache, v_cache, page_table, lengths, *, scale, softcap=0.0, slopes=None, scores=None, decay=1.0, bf16=False, up=None):
    """``{"out", "t_out"[, "scores", "t_scores"]}``. ``up``: what a weight's rounding to the products' type may be off by."""
    q = q.astype(np.float64)
    B, Nq, H, D = q.shape
    P, S, Hk = k_cache.shape[:3]
    G = H // Hk
    u, rounded = (2.0**-8, 2.0**-8) if bf16 else (F, 2 * F)
    up = rounded if up is None else up
    slots = page_table.shape[1] * S
    r = {"out": np.zeros(q.shape), "t_out": np.zeros(q.shape)}
    had, t_had = np.zeros((B, Hk, slots)), np.zeros((B, Hk, slots))
    for b in range(B):
        n = length(lengths[b], page_table[b], S)
        page, at, known = places(page_table[b], n, S, P)
        pos = n - Nq + np.arange(Nq)
        seen = (np.arange(n)[None, :] <= pos[:, None]) & known[None, :]
        some = seen.any(1)
        dist = np.abs(pos[:, None] - np.arange(n)[None, :])
        page, at = np.where(known, page, 0), np.where(known, at, 0)
        for g in range(Hk):
            # slots of no page may hold anything
            kh = np.where(known[:, None], k_cache[page, at, g].astype(np.float64), 0)
            vh = np.where(known[:, None], v_cache[page, at, g].astype(np.float64), 0)
            for h in range(g * G, (g + 1) * G):
                if n == 0:
                    continue
                qh = q[b, :, h]
                x = scale * qh @ kh.T
                s = softcap * np.tanh(x / softcap) if softcap else x
                es = _sum_error(D) * abs(scale) * (np.abs(qh) @ np.abs(kh).T) + 4 * F * np.abs(s) + 16 * F * softcap
                if slopes is not None:
                    s = s - slopes[h] * dist
                    es = es + 4 * F * abs(slopes[h]) * dist
                s = np.where(seen, s, -np.inf)
                m = np.where(some, s.max(1, initial=-np.inf), 0)[:, None]
                w = np.exp(s - m)
                z = w.sum(1, keepdims=True)
                w = w / np.where(z == 0, 1, z)
                worst = 2 * np.where(seen, es, 0).max(1, initial=0)[:, None]
                rho = worst + _sum_error(n) + (8 + 16) * F
                r["out"][b, :, h] = w @ vh
                r["t_out"][b, :, h] = (rho + up) * (w @ np.abs(vh)) + (up + u) * np.abs(w @ vh)
                had[b, g, :n] += w.sum(0)
                apart = np.where(seen, m - np.where(seen, s, m), 0)
                t_had[b, g, :n] += (w * (worst + _sum_error(n) + 24 * F + 8 * F * (apart + 2))).sum(0)
            t_had[b, g, :n] += (Nq * G + 2) * F * had[b, g, :n] + Nq * G * 2.0**-126
    if scores is not None:
        for b in range(B):
            n = length(lengths[b], page_table[b], S)
            old = decay * scores[b, :, :n].astype(np.float64)
            r.setdefault("scores", np.zeros_like(had))[b, :, :n] = old + had[b, :, :n]
            r.setdefault("t_scores", np.zeros_like(had))[b, :, :n] = t_had[b, :, :n] + 2 * F * np.abs(old) + 2 * F * np.abs(had[b, :, :n])
    return r


def evict(k_cache, v_cache, page_table, lengths, scores, budget, sinks=0, recent=0):
    """The caches in place; ``(lengths, sources, scores)``."""
    P, S, Hk = k_cache.shape[:3]
    B, slots = len(lengths), page_table.shape[1] * S
    keep = min(budget, slots)
    new, sources, out = np.zeros(B, np.int32), np.full((B, Hk, keep), -1, np.int32), np.zeros_like(scores)
    for b in range(B):
        n = length(lengths[b], page_table[b], S)
        page, at, known = places(page_table[b], n, S, P)
        new[b] = min(n, budget)
        for h in range(Hk):
            if n <= budget:
                stay = list(range(n))
            else:
                free = range(sinks, n - recent)
                # the largest first, NaN as the least, of equal ones the lowest slot
                order = sorted(free, key=lambda s: (0, -float(scores[b, h, s]), s) if scores[b, h, s] == scores[b, h, s] else (1, 0.0, s))
                stay = sorted([*range(sinks), *order[:budget - sinks - recent], *range(n - recent, n)])
            source = {s: s for s in stay if s < budget}
            holes = sorted(set(range(min(n, budget))) - set(stay))
            source.update(zip(holes, (s for s in stay if s >= budget)))
            for s, a in source.items():
                sources[b, h, s] = a
                out[b, h, s] = scores[b, h, a]
                if a != s and known[a] and known[s]:
                    k_cache[page[s], at[s], h] = k_cache[page[a], at[a], h]
                    v_cache[page[s], at[s], h] = v_cache[page[a], at[a], h]
    return new, sources, out

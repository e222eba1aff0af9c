"""float64 restatement of the token operators (include/hz_token.h), with bounds on what a kernel that
rounds as documented may be off by.

Rounding model of :func:`attention`: a rounding to a type of significand eps is off by at most eps / 2
relative, ``u = 2^-24`` (float32) or ``2^-8`` (bfloat16); weights and score gradients go into their products
rounded to bfloat16 (``2^-8``) for bfloat16 tensors and in three parts (``2^-23``) for float32 ones; the rounded
weights are also what is summed, so with w' = w (1 + d), |d| <= up, the mean's error is at most up (sum of P |v| +
|out|), log of the sum's is at most up (1 + up), and so is the relative error of a P rebuilt from it; a sum of n
float32 terms in steps of sixteen, six products each, is off by at most ``(6 n / 16 + 16) 2^-24`` of the sum of
their magnitudes.
"""

from __future__ import annotations

import numpy as np

F = 2.0**-24


def _sum_error(n):
    return (6 * n / 16 + 16) * F


def qk_norm_rotary(x, w, freqs, positions, interleaved, eps, dy=None):
    """One of q or k: ``y``, and with ``dy`` also ``(dx, dw)``."""
    B, N, H, D = x.shape
    nf = 0 if freqs is None else len(freqs)
    p = np.arange(nf)
    a, b = (2 * p, 2 * p + 1) if interleaved else (p, p + nf)
    w = np.ones(D) if w is None else w.astype(np.float64)
    pos = np.broadcast_to(np.arange(N), (B, N)) if positions is None else positions
    t = pos.astype(np.float64)[:, :, None, None] * (np.zeros(0) if freqs is None else freqs)
    cos, sin = np.cos(t), np.sin(t)
    x = x.astype(np.float64)
    r = 1 / np.sqrt((x**2).mean(-1, keepdims=True) + eps)

    def turn(y, s):
        out = y.copy()
        out[..., a] = y[..., a] * cos - y[..., b] * s
        out[..., b] = y[..., b] * cos + y[..., a] * s
        return out

    y = turn(x * r * w, sin)
    if dy is None:
        return y
    g = turn(dy.astype(np.float64), -sin)
    n = x * r
    dw = (g * n).sum((0, 1, 2))
    g = g * w
    return y, r * (g - n * (g * n).mean(-1, keepdims=True)), dw


def visible(Nq, Nk, n, causal, prefix, documents):
    """[Nq, Nk] of one row with n keys."""
    p = n - Nq + np.arange(Nq)[:, None]
    j = np.arange(Nk)[None, :]
    seen = np.broadcast_to(j < n, (Nq, Nk)).copy()
    if causal:
        seen &= (j <= p) | (j < (0 if prefix is None else prefix))
    if documents is not None:
        mine = np.array([documents[x] if x >= 0 else -1 for x in p[:, 0]])[:, None]
        seen &= (mine >= 0) & (mine == documents[None, :])
    return seen


def attention(q, k, v, *, scale, softcap=0.0, slopes=None, causal=False, prefix=None, documents=None, kv_len=None,
              dout=None, bf16=False):
    """``{"out", "lse"[, "dq", "dk", "dv"]}`` and the bound of each under ``"t_" + name``."""
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    B, Nq, H, D = q.shape
    Nk, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    u, up = (2.0**-8, 2.0**-8) if bf16 else (F, 2 * F)
    r = {n: np.zeros(s) for n, s in (("out", q.shape), ("lse", q.shape[:3]), ("t_out", q.shape), ("t_lse", q.shape[:3]))}
    r["lse"][:] = -np.inf
    if dout is not None:
        dout = dout.astype(np.float64)
        for n, s in (("dq", q.shape), ("dk", k.shape), ("dv", v.shape)):
            r[n], r["t_" + n] = np.zeros(s), np.zeros(s)
    for b in range(B):
        n = Nk if kv_len is None else min(max(int(kv_len[b]), 0), Nk)
        docs = None if documents is None else documents[b]
        seen = visible(Nq, Nk, n, causal, None if prefix is None else prefix[b], docs)
        some = seen.any(1)
        used = seen.any(0)
        dist = np.abs(n - Nq + np.arange(Nq)[:, None] - np.arange(Nk)[None, :])
        for h in range(H):
            # rows that nothing uses may hold anything
            qh, kh = np.where(some[:, None], q[b, :, h], 0), np.where(used[:, None], k[b, :, h // G], 0)
            vh = np.where(used[:, None], v[b, :, h // G], 0)
            x = scale * qh @ kh.T
            t = np.tanh(x / softcap) if softcap else np.zeros_like(x)
            s = softcap * t if softcap else x
            es = _sum_error(D) * abs(scale) * (np.abs(qh) @ np.abs(kh).T) + 4 * F * np.abs(s) + 16 * F * softcap
            if slopes is not None:
                s = s - slopes[h] * dist
                es = es + 4 * F * abs(slopes[h]) * dist
            s = np.where(seen, s, -np.inf)
            m = np.where(some, s.max(1, initial=-np.inf), 0)[:, None]
            w = np.exp(s - m)
            z = w.sum(1, keepdims=True)
            w = w / np.where(z == 0, 1, z)
            lse = (m + np.log(np.where(z == 0, 1, z)))[:, 0]
            rho = (2 * np.where(seen, es, 0).max(1, initial=0) + _sum_error(Nk) + 8 * F)[:, None]
            out = w @ vh
            t_out = (rho + up) * (w @ np.abs(vh)) + (up + u) * np.abs(out)
            r["out"][b, :, h], r["t_out"][b, :, h] = out, t_out
            r["lse"][b, :, h] = np.where(some, lse, -np.inf)
            r["t_lse"][b, :, h] = up * (1 + up) + rho[:, 0] + 4 * F * (np.abs(lse) + 1)
            if dout is None:
                continue
            go = np.where(some[:, None], dout[b, :, h], 0)
            dp = go @ vh.T
            delta = (go * out).sum(1, keepdims=True)
            e_dp = _sum_error(D) * np.abs(go) @ np.abs(vh).T
            e_delta = (np.abs(go) * (t_out + D * F * np.abs(out))).sum(1, keepdims=True)
            rho2 = up * (1 + up) + 2 * rho + 8 * F * (np.abs(lse)[:, None] + 2)
            cap = 1 - t * t if softcap else np.ones_like(t)
            ds = w * (dp - delta) * cap
            e_ds = rho2 * np.abs(ds) + w * (e_dp + e_delta) * cap + w * np.abs(dp - delta) * 32 * F
            cn, cm = _sum_error(Nk), _sum_error(G * Nq)
            r["dq"][b, :, h] = scale * ds @ kh
            r["t_dq"][b, :, h] = abs(scale) * (e_ds + (up + cn) * np.abs(ds)) @ np.abs(kh)
            r["dk"][b, :, h // G] += scale * ds.T @ qh
            r["t_dk"][b, :, h // G] += abs(scale) * (e_ds + (up + cm) * np.abs(ds)).T @ np.abs(qh)
            r["dv"][b, :, h // G] += w.T @ go
            r["t_dv"][b, :, h // G] += (w * (rho2 + up + cm)).T @ np.abs(go)
    if dout is not None:
        for name in ("dq", "dk", "dv"):
            r["t_" + name] += u * np.abs(r[name])
    return r


def bucket_bias(table, buckets, q_positions, k_positions, de=None):
    """``e [B, Nq, Nk, H]``, or with ``de`` (same layout) ``(e, dtable, magnitudes)``: magnitudes is the sum of |de|."""
    R = len(buckets) // 2
    d = k_positions.astype(np.int64)[:, None, :] - q_positions.astype(np.int64)[:, :, None]
    m = buckets[np.clip(d, -R, R) + R]
    nb = table.shape[0]
    known = (m >= 0) & (m < nb)
    e = np.where(known[..., None], table.astype(np.float64)[np.where(known, m, 0)], 0)
    if de is None:
        return e
    grad, size = np.zeros(table.shape), np.zeros(table.shape)
    np.add.at(grad, m[known], de.astype(np.float64)[known])
    np.add.at(size, m[known], np.abs(de.astype(np.float64))[known])
    return e, grad, size

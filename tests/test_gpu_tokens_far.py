"""Scores far from zero: rows whose weights are known exactly whatever the scores' own roundings are (one key far
above the others, or every key the same), through every kernel family of the token attention, forward and reverse.

A float32 score of size S is off by a few 2^-24 S, so at 10^10 neighbouring scores are a thousand apart and a weight
rebuilt from a logarithm of their sum is 2^(some hundreds) or 0. What the inputs fix is checked: the dominant
key's weight is 1 and equal keys share theirs.
"""

import numpy as np
import pytest
import torch

import hamiltonzero_amd as hz

pytestmark = pytest.mark.gpu
F = 2.0**-24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
SCORES = [300.0, 1e4, 1e6, 1e10]


def _say(msg):
    print(f"[case] {msg}", flush=True)


def arr(t):
    return t.detach().double().cpu().numpy()


def normal(g, *shape, dtype, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def within(name, got, want, bound):
    got = arr(got)
    off = np.abs(got - want)
    worst = float(np.max(off / np.maximum(bound, 1e-300)))
    print(f"  {name}: {worst:.3f} of its bound", flush=True)
    assert (off <= bound).all(), (name, worst, np.argwhere(~(off <= bound))[:4].tolist())


def sum_error(n):
    return (6 * n / 16 + 16) * F


SHAPES = [  # B, Nq, Nk, H, Hk, D, options
    (2, 1, 300, 4, 1, 64, dict(causal=True)),  # the cache kernel, one block of columns
    (1, 5, 200, 8, 2, 128, dict(causal=True)),  # two blocks of columns
    (2, 40, 40, 2, 2, 32, dict()),
    (2, 150, 150, 4, 2, 64, dict(causal=True)),
    (1, 257, 257, 2, 1, 128, dict(documents=True)),
    (1, 200, 900, 1, 1, 16, dict(causal=True, slopes=True)),  # keys and queries shared out over workgroups
    (1, 300, 1500, 2, 1, 64, dict(causal=True, documents=True)),
    (2, 130, 130, 1, 1, 80, dict(cap=True)),
    (1, 130, 130, 2, 1, 24, dict(cap=True, slopes=True, causal=True)),
]


def build(case, S, dtype, seed):
    """q, k, v and options; every key but the first of each document is far below it in every query's score."""
    B, Nq, Nk, H, Hk, D, o = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v = (normal(g, *s, dtype=DT[dtype], std=0.25) for s in ((B, Nq, H, D), (B, Nk, Hk, D), (B, Nk, Hk, D)))
    v = v * 4
    q[..., 0], q[..., 1:] = 4.0, q[..., 1:] * 0.25
    k[..., 0] = 0.25
    kw = dict(scale=S / 4.0, causal=o.get("causal", False))
    tops = [0]
    if o.get("documents"):
        cut = Nk // 2
        kw["documents"] = torch.zeros(B, Nk, dtype=torch.int32, device="cuda")
        kw["documents"][:, cut:] = 1
        tops = [0, cut]
    for t in tops:
        k[:, t, :, 0] = 1.0
    if o.get("slopes"):
        kw["slopes"] = torch.full((H,), 0.01, device="cuda")
    if o.get("cap"):
        if dtype == "bf16" and S > 4096:
            pytest.skip("bfloat16 caps end at 8192")
        kw["softcap"] = 2.0 * S if dtype == "f32" else 8192.0
    return g, q, k, v, kw


def scores(q, k, kw):
    """float64, [B, H, Nq, Nk], hidden pairs -inf."""
    q, k = arr(q).transpose(0, 2, 1, 3), arr(k).transpose(0, 2, 1, 3)
    B, H, Nq, _ = q.shape
    Nk = k.shape[2]
    s = q @ np.repeat(k, H // k.shape[1], 1).transpose(0, 1, 3, 2) * kw["scale"]
    if "softcap" in kw:
        s = kw["softcap"] * np.tanh(s / kw["softcap"])
    p, j = Nk - Nq + np.arange(Nq)[:, None], np.arange(Nk)[None, :]
    if "slopes" in kw:
        s = s - arr(kw["slopes"])[:, None, None] * np.abs(p - j)
    if kw["causal"]:
        s = np.where(j <= p, s, -np.inf)
    if "documents" in kw:
        d = kw["documents"].cpu().numpy()
        at = d[:, Nk - Nq:] if Nq <= Nk else None
        s = np.where((at[:, :, None] == d[:, None, :])[:, None], s, -np.inf)
    return s


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("S", SCORES, ids=lambda s: f"{s:g}")
@pytest.mark.parametrize("case", SHAPES, ids=lambda c: "%d-%d-%d-%d-%d-%d-%s" % (*c[:6], "-".join(c[6])))
def test_one_key_far_above_the_others(case, S, dtype):
    B, Nq, Nk, H, Hk, D, _ = case
    _say(f"dominant {case} {S:g} {dtype}")
    g, q, k, v, kw = build(case, S, dtype, 50)
    s = scores(q, k, kw)
    top = s.argmax(-1)
    rest = np.sort(s, -1)[..., -2:]
    assert Nk == 1 or (rest[..., 1] - rest[..., 0]).min() > 120  # e^-120 is no float32: the weights are 1 and 0
    x = [t.requires_grad_() for t in (q, k, v)]
    out = hz.token_attention(*x, **kw)
    dout = normal(g, *out.shape, dtype=DT[dtype])
    dq, dk, dv = torch.autograd.grad(out, x, dout)
    G = H // Hk
    vn, gn = arr(v).transpose(0, 2, 1, 3), arr(dout).transpose(0, 2, 1, 3)
    want = np.take_along_axis(np.repeat(vn, G, 1), top[..., None], 2).transpose(0, 2, 1, 3)
    assert np.array_equal(arr(out), want)  # the dominant key's value itself
    sums, sizes = np.zeros((2, B, Hk, Nk, D))
    for b in range(B):
        for h in range(H):
            np.add.at(sums[b, h // G], top[b, h], gn[b, h])
            np.add.at(sizes[b, h // G], top[b, h], np.abs(gn[b, h]))
    u = F if dtype == "f32" else 2.0**-8
    turn = lambda y: y.transpose(0, 2, 1, 3)  # noqa: E731
    within("dv", dv, turn(sums), turn(sum_error(G * Nq) * sizes + u * np.abs(sums)))
    # score gradients are P (dP - rowsum(dout out)): two float32 sums of the same terms at the dominant key, 0 elsewhere
    each = 2 * sum_error(D) * (np.abs(gn) * np.abs(turn(want))).sum(-1) * (1 + 2 * u) * kw["scale"]  # [B, H, Nq]
    kn, qn = np.abs(arr(k)).transpose(0, 2, 1, 3), np.abs(arr(q)).transpose(0, 2, 1, 3)
    bound = each[..., None] * np.take_along_axis(np.repeat(kn, G, 1), top[..., None], 2)
    within("dq", dq, np.zeros(q.shape), turn(bound) + 1e-30)
    bound = np.zeros((B, Hk, Nk, D))
    for b in range(B):
        for h in range(H):
            np.add.at(bound[b, h // G], top[b, h], each[b, h][:, None] * qn[b, h])
    within("dk", dk, np.zeros(k.shape), turn(bound) + 1e-30)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("S", [-1e10, -1e4, *SCORES], ids=lambda s: f"{s:g}")
@pytest.mark.parametrize("B,Nq,Nk,H,Hk,D,causal", [(1, 3, 70, 4, 2, 64, True), (2, 140, 140, 2, 1, 32, True), (1, 130, 130, 2, 2, 128, False),
                                                   (1, 150, 1100, 1, 1, 64, True)])
def test_equal_keys_share_their_weight(B, Nq, Nk, H, Hk, D, causal, S, dtype):
    """Every key the same: a row that sees n keys gives each 1 / n, at any size of the score."""
    _say(f"equal {B} {Nq} {Nk} {H} {Hk} {D} {S:g} {dtype}")
    g = torch.Generator(device="cuda").manual_seed(51)
    dt = DT[dtype]
    q = normal(g, B, Nq, H, D, dtype=dt, std=0.25)
    q[..., 0] = 4.0
    k = normal(g, B, 1, Hk, D, dtype=dt, std=0.25).expand(B, Nk, Hk, D).clone()
    k[..., 0] = 1.0
    v = normal(g, B, Nk, Hk, D, dtype=dt)
    x = [t.requires_grad_() for t in (q, k, v)]
    out = hz.token_attention(*x, scale=S / 4, causal=causal)
    dout = normal(g, *out.shape, dtype=dt)
    dq, dk, dv = torch.autograd.grad(out, x, dout)
    p, j = Nk - Nq + np.arange(Nq)[:, None], np.arange(Nk)[None, :]
    seen = (j <= p) if causal else np.ones((Nq, Nk), bool)
    w = seen / seen.sum(1, keepdims=True)  # [Nq, Nk]
    G = H // Hk
    vn, gn = arr(v).transpose(0, 2, 1, 3), arr(dout).transpose(0, 2, 1, 3)
    vr = np.repeat(vn, G, 1)
    u, up = (F, 2 * F) if dtype == "f32" else (2.0**-8, 2.0**-8)
    # weights of equal scores are equal before their rounding: their sum, its inverse and the rounding to the products'
    # type are what they are off by; rebuilt ones also by five roundings of a logarithm of up to 32 (bfloat16: 256)
    rho = sum_error(Nk) + 16 * F
    drift = 5 * F * (32 if dtype == "f32" else 256)
    turn = lambda y: y.transpose(0, 2, 1, 3)  # noqa: E731
    within("out", out, turn(w @ vr), turn((rho + up) * (w @ np.abs(vr)) + (u + up) * np.abs(w @ vr)))
    heads = lambda y: y.reshape(B, Hk, G, Nk, D).sum(2)  # noqa: E731
    want, size = heads(w.T @ gn), heads(w.T @ np.abs(gn))
    within("dv", dv, turn(want), turn((rho + up * (1 + up) + up + drift + sum_error(G * Nq)) * size + u * np.abs(want)))
    assert torch.isfinite(dq).all() and torch.isfinite(dk).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("Nq", [4, 100])
def test_a_row_of_nan_stays_one(Nq, dtype):
    """A NaN in a query makes NaN of its output, its gradient and the gradient of the values it sees, and leaves
    the other rows' outputs and gradients of queries as they were."""
    _say(f"nan {Nq} {dtype}")
    g = torch.Generator(device="cuda").manual_seed(52)
    q, k, v = (normal(g, 1, n, 2, 32, dtype=DT[dtype]) for n in (Nq, 100, 100))
    dout = normal(g, 1, Nq, 2, 32, dtype=DT[dtype])

    def go(q):
        x = [t.clone().requires_grad_() for t in (q, k, v)]
        out = hz.token_attention(*x, causal=True)
        return (out.detach(), *torch.autograd.grad(out, x, dout))

    want = go(q)
    bad = q.clone()
    bad[0, 2, 1, 7] = float("nan")
    got = go(bad)
    for i in (0, 1):  # out, dq
        assert got[i][0, 2, 1].isnan().all()
        rest = torch.ones(Nq, 2, dtype=torch.bool, device="cuda")
        rest[2, 1] = False
        assert torch.equal(got[i][0][rest], want[i][0][rest])
    assert got[3][0, :100 - Nq + 3, 1].isnan().all()
    assert torch.equal(got[3][0, :, 0], want[3][0, :, 0])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("Nq", [3, 120])
def test_padding_may_hold_anything_beside_large_scores(Nq, dtype):
    _say(f"far padding {Nq} {dtype}")
    g = torch.Generator(device="cuda").manual_seed(53)
    B, Nk, H, Hk, D = 2, 150, 4, 2, 64
    q, k, v, dout = (normal(g, B, n, h, D, dtype=DT[dtype]) for n, h in ((Nq, H), (Nk, Hk), (Nk, Hk), (Nq, H)))
    docs = (torch.arange(Nk, device="cuda") > 70).int().repeat(B, 1)
    docs[:, 20:30], docs[0, 139:] = -1, -1
    n = torch.tensor([140, 150], dtype=torch.int32, device="cuda")

    def go(q, k, v, dout):
        x = [t.clone().requires_grad_() for t in (q, k, v)]
        out = hz.token_attention(*x, causal=True, documents=docs, kv_len=n, scale=1e4)
        return (out, *torch.autograd.grad(out, x, dout))

    want = go(q, k, v, dout)
    for bad in (float("nan"), float("-inf")):
        k2, v2, q2, d2 = (t.clone() for t in (k, v, q, dout))
        for t in (k2, v2):
            t[:, 20:30], t[0, 139:] = bad, bad
        for t in (q2, d2):
            t[0, -1:] = bad
        for a, b in zip(go(q2, k2, v2, d2), want):
            assert torch.isfinite(a).all() and torch.equal(a, b)

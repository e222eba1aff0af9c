"""GPU parity of the paged operators and of rotations by several axes with their float64 oracle, element by element within the
oracle's bounds (oracle/paged_oracle.py, oracle/token_oracle.py derive them), through the public entry points."""

import numpy as np
import pytest
import torch

import hamiltonzero_amd as hz
from oracle import paged_oracle as P
from oracle import token_oracle as O

pytestmark = pytest.mark.gpu
F = 2.0**-24
ANGLE = 2.0**-21  # the angle's rounding to float32 turns (2 pi 2^-25) and its sine's
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _say(msg):
    print(f"[case] {msg}", flush=True)


def arr(t):
    return t.detach().double().cpu().numpy()


def within(name, got, want, bound):
    """|got - want| <= bound for every element, no NaN; prints how near it comes."""
    got = arr(got)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    off = np.abs(got - want)
    bad = ~(off <= bound)
    worst = float(np.max(off / np.maximum(bound, 1e-300))) if off.size else 0.0
    print(f"  {name}: {worst:.3f} of its bound", flush=True)
    assert not bad.any(), (name, int(bad.sum()), worst, np.argwhere(bad)[:4].tolist())


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def ints(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32, device="cuda")


# --- rotations ------------------------------------------------------------------------------------

ROT = [  # B, N, H, Hk, D, freqs, axes, interleaved, positions
    (2, 5, 4, 2, 64, 32, 2, False, 1 << 10), (1, 1, 1, 1, 8, 4, 1, True, 1 << 30), (3, 7, 5, 1, 80, 40, 3, False, 1 << 30),
    (2, 33, 8, 8, 128, 64, 3, True, 1 << 20), (1, 9, 40, 3, 128, 32, 2, False, -(1 << 20)), (2, 4, 3, 3, 256, 128, 16, False, 1 << 30),
    (4, 3, 2, 1, 16, 8, 4, True, -7), (1, 2100, 2, 2, 24, 12, 2, True, 100), (1, 3, 70, 2, 32, 4, 2, False, 50), (2, 600, 3, 1, 80, 20, 2, True, 900),
    (300, 1, 2, 1, 16, 4, 2, False, 9), (1, 1, 200, 100, 8, 4, 2, False, 9), (2, 11, 1, 1, 48, 16, 3, False, 77),
]


@pytest.mark.parametrize("norm", [False, True], ids=["alone", "norm"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", ROT, ids=lambda c: "-".join(map(str, c)))
def test_rotation_by_axes(case, dtype, norm):
    B, N, H, Hk, D, nf, A, inter, far = case
    _say(f"rotation {case} {dtype} norm {norm}")
    g = gen(1)
    dt, u = DT[dtype], F if dtype == "f32" else 2.0**-8
    rows = normal(g, B, N, H + 2 * Hk, D, dtype=dt, std=2.0)
    q, k = (x.detach().requires_grad_() for x in (rows[:, :, :H], rows[:, :, H:H + Hk]))
    freqs = 100.0 ** (-torch.arange(nf, dtype=torch.float64, device="cuda") / nf)
    pos = torch.randint(min(0, far), abs(far), (B, N, A), generator=g, device="cuda").to(torch.int32)
    axes = torch.randint(0, A, (nf,), generator=g, device="cuda").to(torch.int32)
    axes[0] = A  # no axis: this pair stays
    if nf > 1:
        axes[1] = -1
    w = [(1 + 0.3 * torch.randn(D, generator=g, device="cuda")).requires_grad_() for _ in range(2)] if norm else []
    call = (lambda: hz.qk_norm_rotary(q, k, *w, freqs=freqs, positions=pos, axes=axes, interleaved=inter)) if norm else (
        lambda: hz.qk_rotary(q, k, freqs=freqs, positions=pos, axes=axes, interleaved=inter))
    out = call()
    cot = [normal(g, *o.shape, dtype=dt) for o in out]
    grads = torch.autograd.grad(out, (q, k, *w), cot)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(out, call()))
    a = (arr(freqs), pos.cpu().numpy(), axes.cpu().numpy(), inter)
    i = np.arange(nf)
    ia, ib = (2 * i, 2 * i + 1) if inter else (i, i + nf)

    def pair_size(x):  # |x_a| + |x_b| of each element's pair
        s = np.zeros_like(x)
        s[..., ia] = s[..., ib] = np.abs(x[..., ia]) + np.abs(x[..., ib])
        return s

    for n in range(2):
        x, dy = arr((q, k)[n]), arr(cot[n])
        if not norm:
            y, dx = P.rotation(x, *a), P.rotation(dy, *a, -1)
            within("y", out[n], y, u * np.abs(y) + (ANGLE + 4 * F) * pair_size(x))
            within("dx", grads[n], dx, u * np.abs(dx) + (ANGLE + 4 * F) * pair_size(dy))
            still = [e for e in range(D) if e not in {*ia[2:], *ib[2:]}]  # pairs 0 and 1 have no axis
            assert np.array_equal(arr(out[n])[..., still], x[..., still])
            # the same against differences of the oracle, which a linear map has exactly
            h = np.random.default_rng(5).standard_normal(x.shape)
            step = ((P.rotation(x + h, *a) - P.rotation(x, *a)) * dy).sum()
            assert abs((arr(grads[n]) * h).sum() - step) <= (np.abs(h) * (u * np.abs(dx) + (ANGLE + 4 * F) * pair_size(dy))).sum() + 1e-9 * abs(step)
            continue
        xw = arr(w[n])
        r = 1 / np.sqrt((x**2).mean(-1, keepdims=True) + 1e-6)
        y = P.rotation(x * r * xw, *a)
        size = np.abs(x * r * xw).max(-1, keepdims=True)
        within("y", out[n], y, u * np.abs(y) + (ANGLE + 16 * F) * 2 * size)
        gt = P.rotation(dy, *a, -1)
        m = x * r
        dw = (gt * m).sum((0, 1, 2))
        gw = gt * xw
        dx = r * (gw - m * (gw * m).mean(-1, keepdims=True))
        most = 1.5 * (np.abs(dy).max(-1, keepdims=True) * np.abs(xw).max())  # |turn(dy) w| <= sqrt 2 max max
        am = np.abs(m)
        within("dx", grads[n], dx, u * np.abs(dx) + (ANGLE + (16 + D) * F) * r * most * (1 + am * am.mean(-1, keepdims=True)) * 4)
        total = (1.5 * np.abs(dy).max(-1, keepdims=True) * am).sum((0, 1, 2))
        within("dw", grads[2 + n], dw, (ANGLE + 64 * F) * total + F * np.abs(dw))


def test_one_axis_is_what_the_norms_turn_by():
    """Axes of all zeros give the bits of the rotation without them, with the norms and alone."""
    g = gen(2)
    for dt in DT.values():
        q, k = normal(g, 2, 50, 4, 64, dtype=dt), normal(g, 2, 50, 2, 64, dtype=dt)
        freqs = torch.rand(16, generator=g, dtype=torch.float64, device="cuda")
        pos = torch.randint(0, 1 << 20, (2, 50), generator=g, device="cuda").to(torch.int32)
        axes = torch.zeros(16, dtype=torch.int32, device="cuda")
        for call in (hz.qk_norm_rotary, hz.qk_rotary):
            want = call(q, k, freqs=freqs, positions=pos)
            got = call(q, k, freqs=freqs, positions=pos[:, :, None], axes=axes)
            assert all(torch.equal(a, b) for a, b in zip(want, got))
        want = hz.qk_rotary(q, k, freqs=freqs)
        here = torch.arange(50, dtype=torch.int32, device="cuda").expand(2, 50)
        assert all(torch.equal(a, b) for a, b in zip(want, hz.qk_rotary(q, k, freqs=freqs, positions=here)))


def test_rotation_gradients_of_broadcasts_and_of_one_result():
    g = gen(3)
    freqs = torch.rand(8, generator=g, dtype=torch.float64, device="cuda")
    leaf = normal(g, 1, 1, 1, 16).requires_grad_()
    k = normal(g, 2, 7, 3, 16).requires_grad_()
    q, out_k = hz.qk_rotary(leaf.expand(2, 7, 5, 16), k, freqs=freqs)
    cot = normal(g, 2, 7, 5, 16)
    (got,) = torch.autograd.grad(q, leaf, cot, retain_graph=True)
    pos = np.broadcast_to(np.arange(7)[None, :, None], (2, 7, 1))
    want = P.rotation(arr(cot), arr(freqs), pos, np.zeros(8, int), False, -1)
    within("dq", got, want.sum((0, 1, 2), keepdims=True), (ANGLE + 70 * F) * np.abs(want).sum((0, 1, 2), keepdims=True) * 2)
    (gk,) = torch.autograd.grad(out_k[:, 3:], k, torch.ones(2, 4, 3, 16, device="cuda"))
    assert (gk[:, :3] == 0).all() and (gk[:, 3:] != 0).any()


# --- caches ---------------------------------------------------------------------------------------


def pool(g, pages, S, Hk, D, dt, layout="plain"):
    """Two caches [pages, S, Hk, D] of NaN: a pool of each, heads outside the slots, both in one buffer, or rows apart."""
    if layout == "heads":
        return [torch.full((pages, Hk, S, D), float("nan"), dtype=dt, device="cuda").transpose(1, 2) for _ in range(2)]
    if layout == "joint":
        both = torch.full((pages, S, 2, Hk, D), float("nan"), dtype=dt, device="cuda")
        return [both[:, :, 0], both[:, :, 1]]
    if layout == "apart":
        return [torch.full((pages, S + 2, Hk + 1, D + 8), float("nan"), dtype=dt, device="cuda")[:, 1:S + 1, :Hk, :D] for _ in range(2)]
    return [torch.full((pages, S, Hk, D), float("nan"), dtype=dt, device="cuda") for _ in range(2)]


def rows(g, B, slots, S, Hk, D, dt, lengths, layout="plain", shared=0, bad=False, std=1.0):
    """Caches whose rows' slots hold numbers and all else NaN, and their tables."""
    T = -(-slots // S)
    pages = B * T + 2
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(7))[:B * T].reshape(B, T).to(torch.int32)
    table[:, :shared] = table[:1, :shared]
    k, v = pool(g, pages, S, Hk, D, dt, layout)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), T * S)
        for t in range(-(-n // S)):
            m = min(S, n - t * S)
            for c in (k, v):
                c[int(table[b, t]), :m] = normal(g, m, Hk, D, dtype=dt, std=std)
    if bad:
        r = np.random.default_rng(8)
        for _ in range(max(1, B * T // 5)):
            table[r.integers(B), r.integers(T)] = int(r.choice([-1, pages, 2**31 - 1, -2**31]))
    return k, v, table.cuda(), ints(lengths)


ATTENTION = [  # B, Nq, H, Hk, D, S, lengths, options
    (1, 1, 1, 1, 8, 1, [1], dict()),
    (2, 1, 4, 2, 64, 16, [40, 1], dict(scores=True)),
    (3, 3, 8, 2, 128, 48, [700, 2, 0], dict(softcap=20.0, scores=True)),
    (3, 1, 6, 1, 80, 100, [333, 100, 99], dict(slopes=True, scores=True)),
    (1, 32, 1, 1, 16, 64, [100], dict(scores=True)),
    (1, 33, 1, 1, 32, 64, [40], dict(scores=True)),
    (2, 5, 40, 4, 128, 16, [130, 4], dict(softcap=5.0, scores=True)),
    (2, 7, 24, 3, 40, 3, [65, 66], dict(slopes=True)),
    (4, 1, 8, 8, 64, 16, [-5, 1000, 64, 63], dict(scores=True)),
    (70, 1, 2, 2, 32, 16, "ragged90", dict(scores=True, shared=1)),
    (300, 2, 8, 8, 16, 32, "ragged70", dict(scores=True)),
    (1100, 1, 2, 2, 16, 16, "ragged33", dict(scores=True, softcap=3.0)),
    (1, 1, 8, 2, 128, 64, [5000], dict(scores=True)),
    (2, 2, 2, 1, 64, 256, [9000, 300], dict(slopes=True, scores=True)),
    (67, 1, 1, 1, 8, 16, "one long", dict(scores=True)),
    (3, 2, 4, 2, 64, 16, [90, 33, 0], dict(layout="heads", scores=True)),
    (3, 1, 4, 2, 128, 16, [90, 33, 200], dict(layout="joint")),
    (3, 1, 4, 2, 32, 20, [90, 33, 59], dict(layout="apart", scores=True)),
    (2, 1, 4, 4, 80, 32, [90, 33], dict(layout="apart")),
    (4, 2, 4, 2, 64, 16, [200, 100, 37, 5], dict(bad=True, scores=True)),
    (4, 1, 4, 2, 128, 5, [200, 100, 37, 5], dict(bad=True, scores=True, softcap=9.0)),
    (2, 1, 128, 1, 16, 16, [77, 20], dict(scores=True)),
    (2, 1, 70, 1, 128, 16, [77, 20], dict(scores=True)),
    (70, 1, 2, 2, 32, 16, "ragged90", dict(scores=True, wide=1200)),
    (300, 2, 8, 8, 16, 32, "ragged70", dict(scores=True, wide=1100)),
    (260, 1, 8, 8, 32, 7, "one long", dict(scores=True)),
    (2, 1, 4, 4, 64, 16, [700, 1], dict(scores=True, wide=800)),
    (3, 2, 2, 2, 128, 16, [600, 90, 0], dict(scores=True, slopes=True, wide=800)),
    (2, 1, 4, 4, 40, 7, [700, 530], dict(scores=True, softcap=4.0)),
    (3, 2, 3, 3, 64, 9, [512, 511, 2], dict(scores=True, bad=True)),
    (2, 1, 128, 1, 48, 9, [77, 20], dict(scores=True, softcap=6.0)),
    (2, 20, 4, 2, 128, 9, [700, 20], dict(slopes=True, bad=True)),
]


def lengths_of(how, B):
    if not isinstance(how, str):
        return how
    r = np.random.default_rng(4)
    if how == "one long":
        n = r.integers(0, 5, B)
        n[B // 2] = 4000
        return n.tolist()
    return r.integers(0, int(how[6:]) + 1, B).tolist()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_attention(case, dtype):
    B, Nq, H, Hk, D, S, lengths, o = case
    _say(f"attention {case} {dtype}")
    g = gen(11)
    dt = DT[dtype]
    lengths = lengths_of(lengths, B)
    slots = max(max(lengths), 1, o.get("wide", 0)) + 5
    k, v, table, n = rows(g, B, slots, S, Hk, D, dt, lengths, o.get("layout", "plain"), o.get("shared", 0), o.get("bad", False))
    q = normal(g, B, Nq, H, D, dtype=dt, std=2.0)
    kw = dict(softcap=o.get("softcap", 0.0))
    if o.get("slopes"):
        kw["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device="cuda") / H).float()
    scores = None
    if o.get("scores"):
        scores = torch.rand(B, Hk, table.shape[1] * S, generator=g, device="cuda")
        kw["scores"], kw["decay"] = scores, 0.75
    got = hz.paged_attention(q, k, v, table, n, **kw)
    want = P.attention(arr(q), arr(k), arr(v), table.cpu().numpy(), lengths, scale=D**-0.5, softcap=kw["softcap"],
                       slopes=arr(kw["slopes"]) if o.get("slopes") else None, scores=None if scores is None else arr(scores),
                       decay=kw.get("decay", 1.0), bf16=dtype == "bf16")
    out = got[0] if scores is not None else got
    within("out", out, want["out"], want["t_out"])
    if scores is not None:
        within("scores", got[1], want["scores"], want["t_scores"])
        into = scores.clone()
        again, same = hz.paged_attention(q, k, v, table, n, **{**kw, "scores": into}, scores_out=into)
        assert same is into and torch.equal(into, got[1]) and torch.equal(again, out)
        fresh, first = hz.paged_attention(q, k, v, table, n, **{**kw, "scores": torch.zeros_like(scores)})
        assert torch.equal(fresh, out)
        # as much weight as there are queries that see a slot
        total = first.double().sum((1, 2)).cpu().numpy()
        sees = [(np.abs(arr(out[b])).sum(-1) > 0).sum() for b in range(B)]
        assert np.allclose(total, sees, rtol=1e-5)
        alone = hz.paged_attention(q, k, v, table, n, **{x: y for x, y in kw.items() if x not in ("scores", "decay")})
        assert torch.equal(alone, out)


def test_attention_is_the_contiguous_one():
    """Rows that lie one behind the other give what token_attention gives over the same cache, to the bounds of both."""
    g = gen(12)
    B, H, Hk, D, S, T = 3, 8, 2, 64, 16, 9
    for dtype, dt in DT.items():
        k, v = normal(g, B * T, S, Hk, D, dtype=dt), normal(g, B * T, S, Hk, D, dtype=dt)
        table = torch.arange(B * T, dtype=torch.int32, device="cuda").reshape(B, T)
        n = ints([144, 31, 7])
        q = normal(g, B, 3, H, D, dtype=dt)
        slopes = torch.rand(H, generator=g, device="cuda")
        got = hz.paged_attention(q, k, v, table, n, softcap=7.0, slopes=slopes, scale=0.4)
        want = hz.token_attention(q, k.reshape(B, -1, Hk, D), v.reshape(B, -1, Hk, D), softcap=7.0, slopes=slopes, scale=0.4, causal=True, kv_len=n)
        o = P.attention(arr(q), arr(k), arr(v), table.cpu().numpy(), [144, 31, 7], scale=0.4, softcap=7.0, slopes=arr(slopes), bf16=dtype == "bf16")
        within("paged", got, arr(want), 2 * o["t_out"])


def test_attention_weights_at_large_scores():
    """Scores far from zero: the base of a row is its largest score, so weights keep their precision where softmax is all but certain."""
    g = gen(13)
    for S in (16, 10):
        k, v, table, n = rows(g, 2, 300, S, 1, 64, torch.float32, [300, 17], std=4.0)
        q = normal(g, 2, 1, 2, 64, std=30.0)
        scores = torch.zeros(2, 1, table.shape[1] * S, device="cuda")
        out, new = hz.paged_attention(q, k, v, table, n, scores=scores)
        want = P.attention(arr(q), arr(k), arr(v), table.cpu().numpy(), [300, 17], scale=64**-0.5, scores=arr(scores))
        within("out", out, want["out"], want["t_out"])
        within("scores", new, want["scores"], want["t_scores"])


@pytest.mark.parametrize("heads", [2, 8], ids=["row", "rows"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("length", [90, 7000])
def test_attention_passes_nan_on(length, dtype, heads):
    """A NaN that a query attends to reaches its outputs and weights, wherever in a long row it lies, and nothing else."""
    _say(f"nan {length} {dtype} {heads}")
    g = gen(15)
    k, v, table, n = rows(g, 2, length, 16, 2, 64, DT[dtype], [length, length - 1])
    q = normal(g, 2, 1, heads, 64, dtype=DT[dtype])
    scores = torch.zeros(2, 2, table.shape[1] * 16, device="cuda")
    clean, weights = hz.paged_attention(q, k, v, table, n, scores=scores)
    G = heads // 2
    for first, last in ((0, 64), (length - 20, length - 4), (0, length)):
        bad = k.clone()
        for s in range(first, last):
            bad[int(table[0, s // 16]), s % 16, 1, 7] = float("nan")
        out, new = hz.paged_attention(q, bad, v, table, n, scores=scores)
        assert out[0, :, G:].isnan().all() and torch.equal(out[0, :, :G], clean[0, :, :G]) and torch.equal(out[1], clean[1])
        assert new[0, 1, :length].isnan().all() and torch.equal(new[0, 0], weights[0, 0]) and torch.equal(new[1], weights[1])
        bad = v.clone()
        for s in range(first, last):
            bad[int(table[0, s // 16]), s % 16, 1, 7] = float("nan")
        out, new = hz.paged_attention(q, k, bad, table, n, scores=scores)
        gone = torch.zeros_like(out, dtype=torch.bool)
        gone[0, :, G:, 7] = True
        assert torch.equal(out.isnan(), gone) and torch.equal(out[~gone], clean[~gone]) and torch.equal(new, weights)


def test_attention_behind_two_to_the_31():
    """Offsets of slots beyond 32 bits of elements: pages 2^31 elements apart."""
    g = gen(14)
    P_, S, Hk, D = 3, 16, 2, 32
    for dt, S in ((torch.bfloat16, 16), (torch.bfloat16, 9)):
        base = torch.empty(2**32 + 4096, dtype=dt, device="cuda")
        k = base.as_strided((P_, S, Hk, D), (2**31, Hk * D, D, 1))
        v = normal(g, P_, S, Hk, D, dtype=dt)
        table, n = ints([[2, 0, 1]]), ints([2 * S + 3])
        new_k, new_v = normal(g, 1, 2 * S + 3, Hk, D, dtype=dt), normal(g, 1, 2 * S + 3, Hk, D, dtype=dt)
        hz.paged_append(k, v, new_k, new_v, table, n)
        assert torch.equal(k[2], new_k[0, :S]) and torch.equal(k[0], new_k[0, S:2 * S]) and torch.equal(k[1, :3], new_k[0, 2 * S:])
        q = normal(g, 1, 1, 4, D, dtype=dt)
        scores = torch.rand(1, Hk, 3 * S, generator=g, device="cuda")
        out, had = hz.paged_attention(q, k, v, table, n, scores=scores)
        near = k.clone()
        assert all(torch.equal(a, b) for a, b in zip((out, had), hz.paged_attention(q, near, v, table, n, scores=scores)))
        near_v = v.clone()
        a, b = hz.paged_evict(near, near_v, table, n, scores, 7), hz.paged_evict(k, v, table, n, scores, 7)
        assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(near, k) and torch.equal(near_v, v)
        del base, k


# --- append ---------------------------------------------------------------------------------------

APPEND = [  # B, N, Hk, D, S, slots, lengths, layout, bad
    (1, 1, 1, 8, 1, 1, [1], "plain", False), (3, 1, 2, 64, 16, 40, [40, 1, 17], "plain", False), (3, 7, 2, 128, 16, 64, [64, 3, 0], "plain", False),
    (2, 33, 3, 80, 10, 35, [35, 33], "heads", False), (4, 5, 1, 24, 7, 50, [50, 20, 2, -4], "joint", False), (3, 9, 2, 32, 16, 48, [9, 48, 1000], "apart", False),
    (4, 6, 2, 32, 4, 40, [40, 33, 20, 6], "plain", True), (70, 3, 1, 16, 8, 24, "ragged24", "plain", False),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_append(case, dtype):
    B, N, Hk, D, S, slots, lengths, layout, bad = case
    _say(f"append {case} {dtype}")
    g = gen(21)
    dt = DT[dtype]
    lengths = lengths_of(lengths, B)
    k, v, table, n = rows(g, B, slots, S, Hk, D, dt, lengths, layout, 0, bad)
    proj = normal(g, B, N, 3 * Hk, D, dtype=dt)
    new_k, new_v = proj[:, :, Hk:2 * Hk], proj[:, :, 2 * Hk:]
    want_k, want_v = arr(k), arr(v)
    P.append(want_k, want_v, arr(new_k), arr(new_v), table.cpu().numpy(), lengths)
    versions = k._version, v._version
    assert hz.paged_append(k, v, new_k, new_v, table, n) is None
    np.testing.assert_array_equal(arr(k), want_k)
    np.testing.assert_array_equal(arr(v), want_v)
    assert k._version > versions[0] and v._version > versions[1]


# --- eviction -------------------------------------------------------------------------------------

EVICT = [  # B, Hk, D, S, lengths, budget, sinks, recent, scores, options
    (1, 1, 8, 1, [2], 1, 0, 0, "heavy", dict()),
    (3, 2, 64, 16, [200, 31, 30], 30, 0, 0, "heavy", dict()),
    (3, 2, 64, 16, [200, 130, 0], 100, 4, 20, "heavy", dict()),
    (2, 3, 32, 16, [250, 129], 128, 1, 127, "heavy", dict()),  # nothing is free
    (2, 3, 32, 16, [250, 129], 128, 0, 0, "zeros", dict()),
    (2, 2, 16, 10, [250, 251], 17, 2, 3, "few", dict()),
    (2, 2, 80, 100, [700, 333], 300, 4, 64, "few", dict()),
    (2, 2, 24, 16, [900, 1000], 999, 0, 0, "zeros", dict()),
    (2, 1, 16, 16, [1016, 500], 1, 0, 0, "heavy", dict()),
    (2, 1, 16, 16, [200, 190], 80, 2, 2, "odd", dict()),
    (2, 1, 16, 16, [800, 190], 80, 2, 2, "odd", dict()),
    (2, 1, 8, 64, [5000, 3000], 1000, 0, 100, "odd", dict()),
    (2, 2, 16, 64, [8100, 1500], 2000, 4, 100, "few", dict()),
    (2, 2, 16, 64, [8192, 2001], 2000, 0, 0, "zeros", dict()),
    (1, 2, 8, 64, [20000], 8192, 4, 1000, "heavy", dict()),
    (2, 1, 8, 256, [32768, 16385], 16384, 0, 0, "zeros", dict()),
    (1, 1, 8, 256, [32700], 32699, 0, 0, "few", dict()),
    (2, 1, 8, 256, [70001, 33000], 20000, 3, 500, "heavy", dict()),
    (1, 1, 8, 256, [70001], 40000, 0, 0, "zeros", dict()),
    (1, 1, 8, 256, [100000], 33000, 3, 50, "odd", dict()),
    (3, 2, 64, 16, [100, 31, 64], 30, 0, 0, "heavy", dict(layout="heads")),
    (3, 2, 64, 16, [100, 31, 64], 30, 0, 0, "heavy", dict(layout="joint")),
    (3, 2, 40, 20, [100, 31, 64], 30, 2, 5, "heavy", dict(layout="apart")),
    (3, 2, 64, 16, [100, 90, 64], 30, 0, 0, "heavy", dict(bad=True)),
    (2, 2, 16, 16, [2000, 1500], 700, 0, 0, "few", dict(bad=True)),
    (3, 2, 16, 16, [100, -2, 500], 600, 0, 0, "heavy", dict()),
    (70, 3, 16, 16, "ragged90", 40, 1, 8, "few", dict()),
    (2, 1, 128, 16, [300, 300], 100, 0, 0, "negative", dict()),
]


def weights(how, g, B, Hk, slots):
    x = torch.randn(B, Hk, slots, generator=g, device="cuda")
    if how == "heavy":
        return torch.exp(2 * x) * (torch.rand(B, Hk, slots, generator=g, device="cuda") < 0.9)
    if how == "zeros":
        return torch.zeros_like(x)
    if how == "few":
        return torch.randint(0, 4, (B, Hk, slots), generator=g, device="cuda").float()
    if how == "odd":
        odd = torch.tensor([float("nan"), float("inf"), -float("inf"), 0.0, -0.0, 1e-45, -1e-45, 3.4e38, 1.0], device="cuda")
        return odd[torch.randint(0, 9, (B, Hk, slots), generator=g, device="cuda")]
    return x


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", EVICT, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_evict(case, dtype):
    B, Hk, D, S, lengths, budget, sinks, recent, how, o = case
    _say(f"evict {case} {dtype}")
    g = gen(31)
    dt = DT[dtype]
    lengths = lengths_of(lengths, B)
    k, v, table, n = rows(g, B, max(max(lengths), 1), S, Hk, D, dt, lengths, o.get("layout", "plain"), 0, o.get("bad", False))
    scores = weights(how, g, B, Hk, table.shape[1] * S)
    kept = scores.clone()
    want_k, want_v = arr(k), arr(v)
    want = P.evict(want_k, want_v, table.cpu().numpy(), lengths, scores.cpu().numpy(), budget, sinks, recent)
    versions = k._version, v._version
    for turn in range(2):  # the same again: sources lie behind the budget and are still there
        got = hz.paged_evict(k, v, table, n, scores, budget, sinks=sinks, recent=recent)
        assert got[0].dtype == got[1].dtype == torch.int32
        np.testing.assert_array_equal(got[0].cpu().numpy(), want[0])
        np.testing.assert_array_equal(got[1].cpu().numpy(), want[1])
        np.testing.assert_array_equal(got[2].cpu().numpy().view(np.uint32), want[2].view(np.uint32))
        np.testing.assert_array_equal(arr(k), want_k)
        np.testing.assert_array_equal(arr(v), want_v)
        assert same_bits(scores, kept) and n.cpu().tolist() == list(lengths)
    assert k._version > versions[0] and v._version > versions[1]

"""Calls of the token operators for what they do besides their numbers: results written into a caller's tensors, operands
with tangents, gradients of broadcast and shared leaves, tables of different sizes at once; and the cache kernel's widest
form."""

import threading

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwd

import hamiltonzero_amd as hz
from oracle import token_oracle as O

pytestmark = pytest.mark.gpu
F = 2.0**-24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _say(msg):
    print(f"[case] {msg}", flush=True)


def arr(t):
    return t.detach().double().cpu().numpy()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


# --- results in a caller's tensors ------------------------------------------------------------------


def test_out_that_overlaps_is_refused():
    """Results shifted against an input or each other by a head or a token, and windows that hold an element twice."""
    H, Hk, D = 4, 2, 32
    rows = torch.zeros(2, 9, H + 2 * Hk, D, device="cuda")
    q, k = rows[:, :8, :H], rows[:, :8, H:H + Hk]
    a, b = torch.empty(2, 8, H, D, device="cuda"), torch.empty(2, 8, Hk, D, device="cuda")
    cache = torch.zeros(2, 12, Hk, D, device="cuda")
    both = torch.zeros(2, 12, H, D, device="cuda")
    window = torch.zeros(4096, device="cuda").as_strided((2, 8, H, D), (1024, 64, D, 1))  # tokens 64 apart, 128 long
    for out, text in (((rows[:, :8, 1:H + 1], b), "overlap"), ((rows[:, 1:, :H], b), "overlap"), ((a, rows[:, 1:, H:H + Hk]), "overlap"),
                      ((rows[:, :8, 2:H + 2], b), "overlap"), ((both[:, :8], both[:, 3:11, 2:]), "overlap"),
                      ((both[:, :8], both[:, :8, 2:]), "overlap"), ((a, rows[:, :8, H - 1:H - 1 + Hk]), "overlap"),
                      ((window, b), "several places")):
        with pytest.raises(ValueError, match=text):
            hz.qk_norm_rotary(q, k, out=out)
    with pytest.raises(ValueError, match="overlap"):
        hz.qk_norm_rotary(cache[:, :8].repeat(1, 1, 2, 1), cache[:, :8], out=(a, cache[:, 1:9]))


def test_out_beside_its_input_is_taken():
    """Slices of one buffer that share no element: heads beside heads, tokens beside tokens, the rows of a cache."""
    g = gen(60)
    B, N, H, Hk, D = 2, 6, 4, 2, 32
    rows = normal(g, B, N, 2 * (H + Hk), D)
    q, k = rows[:, :, :H], rows[:, :, H:H + Hk]
    want = hz.qk_norm_rotary(q, k)
    hz.qk_norm_rotary(q, k, out=(rows[:, :, H + Hk:2 * H + Hk], rows[:, :, 2 * H + Hk:]))
    assert torch.equal(rows[:, :, H + Hk:2 * H + Hk], want[0]) and torch.equal(rows[:, :, 2 * H + Hk:], want[1])
    cache = normal(g, B, 2 * N, H, D)
    q, k = cache[:, :N], cache[:, :N, :Hk].clone()
    want = hz.qk_norm_rotary(q, k)
    k_cache = torch.empty_like(cache[:, :, :Hk])
    hz.qk_norm_rotary(q, k, out=(cache[:, N:], k_cache[:, N:]))
    assert torch.equal(cache[:, N:], want[0]) and torch.equal(k_cache[:, N:], want[1])


def test_out_counts_as_a_change():
    """A tensor that a differentiable call saved is written by ``out=``: its backward says so, as after an in-place write."""
    g = gen(61)
    q, v = normal(g, 1, 4, 2, 32), normal(g, 1, 8, 2, 32)
    cache = normal(g, 1, 8, 2, 32)
    leaf = q.clone().requires_grad_()
    for part, row in ((slice(0, 1), 0), (slice(1, 2), 1)):
        out = hz.token_attention(leaf, cache, v, causal=True)
        x, into = torch.zeros(1, 4, 2, 32, device="cuda"), [torch.empty(1, 4, 2, 32, device="cuda"), cache[:, 4:]]
        versions = [t._version for t in into]
        with torch.no_grad():
            hz.qk_norm_rotary(x, x, out=tuple(into[::-1]) if row else tuple(into))
        assert all(t._version > n for t, n in zip(into, versions))
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out.sum(), leaf)
    with pytest.raises(ValueError, match="gradient"):  # a leaf of a graph is no place for results
        hz.qk_norm_rotary(x, x, out=(torch.empty_like(x).requires_grad_(), torch.empty_like(x)))


# --- forward mode, leaves that only inference has ----------------------------------------------------


def test_tangents_of_tables_are_refused():
    x = torch.zeros(2, 8, 4, 32, device="cuda")
    slopes, freqs = torch.ones(4, device="cuda"), torch.ones(16, dtype=torch.float64, device="cuda")
    with fwd.dual_level():
        s = fwd.make_dual(slopes, torch.ones_like(slopes))
        f = fwd.make_dual(freqs, torch.ones_like(freqs))
        with pytest.raises(NotImplementedError, match="forward mode"):
            hz.token_attention(x, x, x, slopes=s)
        with pytest.raises(NotImplementedError, match="forward mode"):
            hz.qk_norm_rotary(x, x, freqs=f)
        with pytest.raises(NotImplementedError, match="forward mode"), torch.no_grad():
            hz.token_attention(x, x, x, slopes=s)
        assert hz.token_attention(x, x, x, slopes=slopes).shape == x.shape
        out = torch.empty_like(x)
        with pytest.raises(NotImplementedError, match="forward mode"):
            hz.qk_norm_rotary(x, x, out=(fwd.make_dual(out, out), torch.empty_like(x)))


def test_parameters_serve_without_gradients():
    """Frequencies that are a parameter are refused where a gradient would be dropped, and taken where none is asked."""
    g = gen(62)
    q = normal(g, 1, 5, 2, 32)
    freqs = torch.rand(16, generator=g, dtype=torch.float64, device="cuda")
    leaf = freqs.clone().requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        hz.qk_norm_rotary(q, q, freqs=leaf)
    with torch.no_grad():
        got = hz.qk_norm_rotary(q, q, freqs=leaf)
    for a, b in zip(got, hz.qk_norm_rotary(q, q, freqs=freqs)):
        assert torch.equal(a, b)


# --- gradients of broadcast and shared leaves ----------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("N", [7, 70, 150])
def test_gradients_through_broadcasts(N, dtype):
    """Keys and values expanded over batch and heads, and a cotangent expanded over all but D: the same bits as for
    copies of them, which torch then adds up over the broadcast axes."""
    _say(f"broadcast {N} {dtype}")
    g = gen(63)
    dt, B, H, D = DT[dtype], 2, 4, 32
    q = normal(g, B, N, H, D, dtype=dt).requires_grad_()
    k = normal(g, 1, N, 2, D, dtype=dt).requires_grad_()
    v = normal(g, B, N, 1, D, dtype=dt).requires_grad_()
    cot = normal(g, 1, 1, 1, D, dtype=dt)
    out = hz.token_attention(q, k.expand(B, N, 2, D), v.expand(B, N, 2, D), causal=True)
    got = torch.autograd.grad(out, (q, k, v), cot.expand_as(out))
    full = [t.detach().expand(B, N, h, D).contiguous().requires_grad_() for t, h in ((q, H), (k, 2), (v, 2))]
    same = hz.token_attention(*full, causal=True)
    assert torch.equal(same, out)
    dq, dk, dv = torch.autograd.grad(same, full, cot.expand_as(out).contiguous())
    assert torch.equal(got[0], dq)
    u = F if dtype == "f32" else 2.0**-8
    for a, b, axis in ((got[1], dk, 0), (got[2], dv, 2)):  # two terms and one rounding
        want = b.double().sum(axis, keepdim=True)
        assert ((a.double() - want).abs() <= u * want.abs() + 2 * F * b.double().abs().sum(axis, keepdim=True)).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norm_gradients_through_broadcasts(dtype):
    g = gen(64)
    dt, B, N, H, D = DT[dtype], 3, 5, 4, 32
    q, k = normal(g, 1, N, 1, D, dtype=dt).requires_grad_(), normal(g, B, N, 2, D, dtype=dt).requires_grad_()
    freqs = torch.rand(16, generator=g, dtype=torch.float64, device="cuda")
    cot = normal(g, 1, 1, 1, D, dtype=dt)
    out = hz.qk_norm_rotary(q.expand(B, N, H, D), k, freqs=freqs)
    got = torch.autograd.grad(out, (q, k), [cot.expand_as(o) for o in out])
    full = [q.detach().expand(B, N, H, D).contiguous().requires_grad_(), k.detach().clone().requires_grad_()]
    same = hz.qk_norm_rotary(*full, freqs=freqs)
    for a, b in zip(same, out):
        assert torch.equal(a, b)
    dq, dk = torch.autograd.grad(same, full, [cot.expand_as(o).contiguous() for o in same])
    assert torch.equal(got[1], dk)
    want, size = dq.double().sum((0, 2), keepdim=True), dq.double().abs().sum((0, 2), keepdim=True)
    u = F if dtype == "f32" else 2.0**-8
    # torch sums the three batches and then the heads (or both at once), each result rounded to the type
    assert ((got[0].double() - want).abs() <= 2 * (u + 12 * F) * size).all()


# --- the cache kernel's widest form -----------------------------------------------------------------------

WIDE = [  # B, Nq, Nk, H, Hk, D, options: 17 to 32 rows of query and head share a key head
    (2, 5, 700, 8, 2, 128, dict(softcap=20.0, causal=True, kv_len=[700, 233])),
    (1, 1, 333, 32, 1, 128, dict(causal=True)),
    (2, 3, 200, 8, 1, 80, dict(causal=True, slopes=True)),
    (2, 17, 130, 1, 1, 64, dict(causal=True, documents=True)),
    (1, 3, 900, 7, 1, 64, dict(softcap=5.0, slopes=True, causal=True, documents=True)),
    (2, 6, 90, 4, 1, 40, dict(softcap=3.0, documents=True)),
    (1, 8, 41, 12, 3, 128, dict(causal=True, prefix=[30], slopes=True)),
    (3, 20, 20, 1, 1, 128, dict(causal=True, softcap=8.0, kv_len=[20, 0, 7])),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", WIDE, ids=lambda c: "%d-%d-%d-%d-%d-%d-%s" % (*c[:6], "-".join(c[6])))
def test_two_blocks_of_columns(case, dtype):
    B, Nq, Nk, H, Hk, D, o = case
    assert 16 < Nq * (H // Hk) <= 32
    _say(f"wide {case} {dtype}")
    g, dt = gen(65), DT[dtype]
    q, k, v = (normal(g, *s, dtype=dt, std=d).requires_grad_()
               for s, d in (((B, Nq, H, D), 2.0), ((B, Nk, Hk, D), 1.0), ((B, Nk, Hk, D), 1.0)))
    kw = {n: o[n] for n in ("softcap", "causal") if n in o}
    for n in ("kv_len", "prefix"):
        if n in o:
            kw[n] = torch.tensor(o[n], dtype=torch.int32, device="cuda")
    if "slopes" in o:
        kw["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device="cuda") / H).float()
    if "documents" in o:
        kw["documents"] = torch.randint(0, 3, (B, Nk), generator=torch.Generator().manual_seed(6)).sort(1).values.to(torch.int32).cuda()
        kw["documents"][:, -(Nq // 3):] = -1
    out = hz.token_attention(q, k, v, **kw)
    dout = normal(g, *out.shape, dtype=dt)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    with torch.no_grad():
        assert torch.equal(hz.token_attention(q, k, v, **kw), out)
    okw = {n: x.cpu().numpy() if isinstance(x, torch.Tensor) else x for n, x in kw.items()}
    want = O.attention(arr(q), arr(k), arr(v), scale=float(np.float32(D**-0.5)), dout=arr(dout), bf16=dtype == "bf16", **okw)
    for name, x in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        off = np.abs(arr(x) - want[name])
        print(f"  {name}: {float(np.max(off / np.maximum(want['t_' + name], 1e-300))):.3f} of its bound", flush=True)
        assert (off <= want["t_" + name]).all(), name


# --- tables of different sizes at once -----------------------------------------------------------------


def test_tables_of_different_sizes_in_two_threads():
    """A thread with the largest table beside one with the smallest: each call's memory is its own."""
    _say("two tables")
    pos = torch.arange(20, dtype=torch.int32, device="cuda")[None]
    sizes = [(512, 60, 4096), (2, 60, 1)]
    calls = []
    for nb, H, R in sizes:
        g = gen(nb)
        calls.append((normal(g, nb, H), torch.randint(0, nb, (2 * R + 1,), generator=g, device="cuda").to(torch.int32)))

    def one(table, plan, layout):
        t = table.clone().requires_grad_()
        e = hz.bucket_bias(t, plan, pos, pos, e_layout=layout)
        return e.detach(), torch.autograd.grad(e, t, torch.ones_like(e))[0]

    want = [[one(*c, layout) for layout in ("qhk", "qkh")] for c in calls]
    torch.cuda.synchronize()
    failed, start = [], threading.Barrier(2)

    def work(i):
        try:
            start.wait()
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(100):
                    for layout, w in zip(("qhk", "qkh"), want[i]):
                        for a, b in zip(one(*calls[i], layout), w):
                            assert torch.equal(a, b)
        except Exception as e:  # shown by the assertion below
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed[0]


# --- caches that fill the card -------------------------------------------------------------------------


def test_more_keys_than_a_reverse_pass_takes():
    """A thousand rows of 131072 keys (here the same ones): a forward alone has no grid of the keys' size."""
    _say("many long rows")
    g = gen(66)
    B, Nk, Hk, D = 1024, 131072, 2, 64
    k, v = (normal(g, 1, Nk, Hk, D, dtype=torch.bfloat16).expand(B, Nk, Hk, D) for _ in range(2))
    q = normal(g, B, 1, 4, D, dtype=torch.bfloat16)
    n = torch.full((B,), Nk, dtype=torch.int32, device="cuda")
    n[-1] = Nk - 77
    out = hz.token_attention(q, k, v, causal=True, kv_len=n)
    for b in (0, 517, B - 1):
        for h in range(4):
            keys, values = k[b, :n[b], h // 2].double(), v[b, :n[b], h // 2].double()
            w = torch.softmax(keys @ q[b, 0, h].double() * D**-0.5, 0)
            want, size = w @ values, w @ values.abs()
            assert ((out[b, 0, h].double() - want).abs() <= size * (2.0**-8 + 0.08 * 2**-8) + want.abs() * 2.0**-8).all()
    with pytest.raises(hz._native.HzError, match="grid limit"):
        hz.token_attention(q.clone().requires_grad_(), k, v)


def test_options_beyond_float32_are_refused():
    x = torch.zeros(1, 4, 2, 32, device="cuda")
    for call in (lambda: hz.token_attention(x, x, x, scale=1e39), lambda: hz.token_attention(x, x, x, softcap=1e300),
                 lambda: hz.qk_norm_rotary(x, x, eps=1e39)):
        with pytest.raises(hz._native.HzError):
            call()

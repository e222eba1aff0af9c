"""GPU parity of the token operators with their float64 oracle, element by element within the oracle's bounds
(oracle/token_oracle.py derives them), through the public entry points."""

import numpy as np
import pytest
import torch

import hamiltonzero_amd as hz
from hamiltonzero_amd import tokens
from oracle import token_oracle as O

pytestmark = pytest.mark.gpu
F = 2.0**-24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _say(msg):
    print(f"[case] {msg}", flush=True)


def arr(t):
    return t.detach().double().cpu().numpy()


def within(name, got, want, bound):
    """|got - want| <= bound for every element (infinities equal, no NaN); prints how near it comes."""
    got = arr(got)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]), name
    off = np.abs(np.where(inf, 0, got) - np.where(inf, 0, want))
    bad = ~(off <= bound)
    worst = float(np.max(off / np.maximum(bound, 1e-300))) if off.size else 0.0
    print(f"  {name}: {worst:.3f} of its bound", flush=True)
    assert not bad.any(), (name, int(bad.sum()), worst, np.argwhere(bad)[:4].tolist())


def normal(g, *shape, dtype, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# --- norms and rotation ---------------------------------------------------------------------------

NORM = [  # B, N, H, Hk, D, freqs, interleaved, positions
    (2, 5, 4, 2, 64, 32, False, "far"), (1, 1, 1, 1, 8, 4, True, None), (3, 7, 5, 1, 80, 20, False, "far"),
    (2, 33, 8, 8, 128, 64, True, None), (1, 9, 40, 3, 128, 32, False, "signed"), (2, 4, 3, 3, 256, 128, False, "far"),
    (4, 3, 2, 1, 16, 0, False, None), (1, 2100, 2, 2, 24, 8, True, "far"), (1, 3, 70, 2, 32, 16, False, None),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", NORM, ids=lambda c: "-".join(map(str, c)))
def test_norm_rotary(case, dtype):
    B, N, H, Hk, D, nf, inter, where = case
    _say(f"norm {case} {dtype}")
    g = gen(1)
    dt = DT[dtype]
    rows = normal(g, B, N, H + 2 * Hk, D, dtype=dt, std=2.0)
    q, k = (x.detach().requires_grad_() for x in (rows[:, :, :H], rows[:, :, H:H + Hk]))
    w = [(1 + 0.3 * torch.randn(D, generator=g, device="cuda")).requires_grad_() for _ in range(2)]
    freqs = None if nf == 0 else 10000.0 ** (-torch.arange(nf, dtype=torch.float64, device="cuda") / nf)
    pos = None
    if where is not None:
        lo, hi = (0, 1 << 30) if where == "far" else (-(1 << 20), 1 << 20)
        pos = torch.randint(lo, hi, (B, N), generator=g, device="cuda").to(torch.int32)
    out = hz.qk_norm_rotary(q, k, *w, freqs=freqs, positions=pos, interleaved=inter)
    cot = [normal(g, *o.shape, dtype=dt) for o in out]
    grads = torch.autograd.grad(out, (q, k, *w), cot)
    with torch.no_grad():
        again = hz.qk_norm_rotary(q, k, *w, freqs=freqs, positions=pos, interleaved=inter)
    u = F if dtype == "f32" else 2.0**-8
    angle_error = 2.0**-21  # the angle's rounding to float32 turns (2 pi 2^-25) and its sine's
    for i in range(2):
        x, dy = arr((q, k)[i]), arr(cot[i])
        y, dx, dw = O.qk_norm_rotary(x, arr(w[i]), None if freqs is None else arr(freqs), None if pos is None else pos.cpu().numpy(),
                                     inter, 1e-6, dy)
        r = 1 / np.sqrt((x**2).mean(-1, keepdims=True) + 1e-6)
        size = (np.abs(x * r * arr(w[i]))).max(-1, keepdims=True)
        within("y", out[i], y, u * np.abs(y) + (angle_error + 16 * F) * 2 * size)
        assert torch.equal(out[i], again[i])
        gw = 1.5 * (np.abs(dy).max(-1, keepdims=True) * np.abs(arr(w[i])).max())  # |turn(dy) w| <= sqrt 2 max max
        n = np.abs(x * r)
        within("dx", grads[i], dx, u * np.abs(dx) + (angle_error + (16 + D) * F) * r * gw * (1 + n * n.mean(-1, keepdims=True)) * 4)
        total = (1.5 * np.abs(dy).max(-1, keepdims=True) * n).sum((0, 1, 2))
        within("dw", grads[2 + i], dw, (angle_error + 64 * F) * total + F * np.abs(dw))


def test_norm_writes_into_a_cache_and_leaves_the_rest():
    g = gen(2)
    B, N, H, Hk, D = 2, 3, 4, 2, 32
    q, k = normal(g, B, N, H, D, dtype=torch.bfloat16), normal(g, B, N, Hk, D, dtype=torch.bfloat16)
    cache = torch.full((B, 10, Hk, D), 7.0, dtype=torch.bfloat16, device="cuda")
    freqs = torch.rand(16, dtype=torch.float64, device="cuda")
    want = hz.qk_norm_rotary(q, k, freqs=freqs)
    got_q = torch.empty_like(q)
    hz.qk_norm_rotary(q, k, freqs=freqs, out=(got_q, cache[:, 4:7]))
    assert torch.equal(got_q, want[0]) and torch.equal(cache[:, 4:7], want[1])
    assert (cache[:, :4] == 7).all() and (cache[:, 7:] == 7).all()


# --- attention ------------------------------------------------------------------------------------

ATTN = [  # B, Nq, Nk, H, Hk, D, options
    (1, 1, 1, 1, 1, 8, dict()),
    (2, 1, 40, 4, 2, 64, dict(causal=True)),
    (2, 3, 700, 8, 2, 128, dict(causal=True, kv_len="ragged", softcap=20.0)),
    (3, 1, 333, 6, 1, 80, dict(causal=True, kv_len="ragged", slopes=True)),
    (1, 32, 100, 1, 1, 16, dict(causal=True, prefix=True)),
    (1, 33, 33, 1, 1, 32, dict(causal=True)),
    (2, 130, 130, 4, 2, 128, dict(causal=True, softcap=5.0)),
    (2, 200, 200, 2, 2, 64, dict(causal=True, documents="padded", slopes=True)),
    (1, 257, 257, 3, 1, 40, dict(documents="shuffled", softcap=10.0)),
    (2, 150, 90, 2, 1, 64, dict()),
    (2, 150, 90, 2, 1, 32, dict(causal=True)),
    (2, 70, 300, 4, 4, 24, dict(causal=True, prefix=True, kv_len="short", slopes=True)),
    (1, 129, 385, 2, 1, 128, dict(causal=True, prefix=True, documents="padded")),
    (2, 64, 64, 2, 2, 128, dict(documents="none")),
    (2, 5, 64, 2, 2, 64, dict(documents="none", causal=True)),
    (2, 65, 129, 8, 1, 16, dict(causal=True, kv_len="zero", softcap=50.0)),
    (2, 4, 129, 8, 1, 16, dict(causal=True, kv_len="zero")),
]


def options(o, g, B, Nq, Nk, H):
    """The operator's keywords on the GPU and the oracle's."""
    kw = {k: v for k, v in o.items() if k in ("softcap", "causal")}
    if o.get("slopes"):
        kw["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device="cuda") / H).float()
    if o.get("prefix"):
        kw["prefix"] = torch.randint(0, Nk + 5, (B,), generator=g, device="cuda").to(torch.int32)
    how = o.get("documents")
    if how:
        if how == "none":
            d = torch.full((B, Nk), -3)
        elif how == "padded":
            d = torch.sort(torch.randint(0, 4, (B, Nk), generator=torch.Generator().manual_seed(3)), 1).values
            d[:, -(Nk // 6):] = -1
        else:
            d = torch.randint(-2, 3, (B, Nk), generator=torch.Generator().manual_seed(4))
        kw["documents"] = d.to(torch.int32).cuda()
    how = o.get("kv_len")
    if how:
        n = dict(ragged=[Nk, Nk // 3, Nk - 1], short=[Nq // 2, Nk + 50, 1], zero=[0, Nk, -4])[how][:B]
        kw["kv_len"] = torch.tensor(n, dtype=torch.int32, device="cuda")
    return kw, {k: v.cpu().numpy() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", ATTN, ids=lambda c: "%d-%d-%d-%d-%d-%d-%s" % (*c[:6], "-".join(f"{k}={v}" for k, v in c[6].items())))
def test_attention(case, dtype):
    B, Nq, Nk, H, Hk, D, o = case
    _say(f"attention {case} {dtype}")
    g = gen(5)
    dt = DT[dtype]
    q = normal(g, B, Nq, H, D, dtype=dt, std=2.0).requires_grad_()
    kv = normal(g, B, Nk, 2 * Hk, D, dtype=dt)
    k, v = kv[:, :, :Hk].detach().requires_grad_(), kv[:, :, Hk:].detach().requires_grad_()
    kw, okw = options(o, g, B, Nq, Nk, H)
    out = hz.token_attention(q, k, v, **kw)
    dout = normal(g, *out.shape, dtype=dt)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
    with torch.no_grad():
        assert torch.equal(hz.token_attention(q, k, v, **kw), out)
    want = O.attention(arr(q), arr(k), arr(v), scale=float(np.float32(D**-0.5)), dout=arr(dout), bf16=dtype == "bf16", **okw)
    opts = (kw.get("slopes"), kw.get("prefix"), kw.get("documents"), kw.get("kv_len"), D**-0.5, kw.get("softcap", 0.0),
            kw.get("causal", False))
    _, _, lse = tokens.token_attention_fwd(q.detach(), k.detach(), v.detach(), opts, True)
    within("lse", lse, want["lse"], want["t_lse"])
    for name, x in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        within(name, x, want[name], want["t_" + name])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("Nq", [2, 96])
def test_padding_may_hold_anything(Nq, dtype):
    """NaN and infinities in padding and behind kv_len change nothing, forward or backward."""
    _say(f"padding {Nq} {dtype}")
    g = gen(6)
    B, Nk, H, Hk, D = 2, 128, 4, 2, 64
    dt = DT[dtype]
    q, k, v = normal(g, B, Nq, H, D, dtype=dt), normal(g, B, Nk, Hk, D, dtype=dt), normal(g, B, Nk, Hk, D, dtype=dt)
    dout = normal(g, B, Nq, H, D, dtype=dt)
    kv_len = torch.tensor([100, 128], dtype=torch.int32, device="cuda")
    docs = torch.zeros(B, Nk, dtype=torch.int32, device="cuda")
    docs[0, 10:20] = -1
    docs[0, 98:100] = -5  # the last queries of row 0 are padding
    docs[1, 100:] = 1
    docs[1, 127:] = -1
    kw = dict(causal=True, documents=docs, kv_len=kv_len, softcap=8.0)

    def go(q, k, v, dout):
        x = [t.detach().clone().requires_grad_() for t in (q, k, v)]
        out = hz.token_attention(*x, **kw)
        return (out, *torch.autograd.grad(out, x, dout))

    want = go(q, k, v, dout)
    for bad in (float("nan"), float("inf")):
        k2, v2, q2, d2 = k.clone(), v.clone(), q.clone(), dout.clone()
        for t in (k2, v2):
            t[0, 10:20], t[0, 98:], t[1, 127] = bad, bad, bad
        for t in (q2, d2):
            t[0, -2:], t[1, -1] = bad, bad
        for a, b in zip(go(q2, k2, v2, d2), want):
            assert torch.isfinite(a).all() and torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_broadcasts_and_shared_inputs(dtype):
    g = gen(7)
    dt = DT[dtype]
    B, N, H, D = 2, 70, 4, 32
    base = normal(g, B, N, 3 * H, D + 8, dtype=dt)
    q = base[:, :, :H, :D]  # rows of D + 8
    k1, v1 = normal(g, 1, N, 2, D, dtype=dt), normal(g, B, N, 1, D, dtype=dt)
    want = hz.token_attention(q.contiguous(), k1.expand(B, N, 2, D).contiguous(), v1.expand(B, N, 2, D).contiguous(), causal=True)
    got = hz.token_attention(q, k1.expand(B, N, 2, D), v1.expand(B, N, 2, D), causal=True)
    assert torch.equal(got, want)
    odd = normal(g, B, N, H, D + 1, dtype=dt)[..., 1:]
    assert torch.equal(hz.token_attention(odd, odd, odd), hz.token_attention(*[odd.contiguous()] * 3))
    # one leaf as query, key and value, a broadcast one, and an expanded cotangent
    x = normal(g, B, N, H, D, dtype=dt).requires_grad_()
    y = k1.clone().requires_grad_()
    out = hz.token_attention(x, y.expand(B, N, 2, D), x[:, :, :2])
    dx, dy = torch.autograd.grad(out, (x, y), normal(g, 1, 1, 1, D, dtype=dt).expand_as(out))
    assert dx.shape == x.shape and dy.shape == y.shape and torch.isfinite(dx).all()


def test_long_cache_offsets():
    """A cache of more than 2^31 elements: the last row's tokens lie behind 32-bit offsets."""
    B, Nk, Hk, D = 3, 200003, 32, 128  # 2.46e9 elements, 4.9 GB a tensor
    g = gen(8)
    k = torch.empty(B, Nk, Hk, D, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    v = torch.empty(B, Nk, Hk, D, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    q = normal(g, B, 1, Hk, D, dtype=torch.bfloat16)
    n = torch.tensor([5, Nk - 7, Nk], dtype=torch.int32, device="cuda")
    out = hz.token_attention(q, k, v, causal=True, kv_len=n)
    few = hz.token_attention(q[2:], k[2:].clone(), v[2:].clone(), causal=True)
    s = (q[2].double() * k[2].double()[:, :, :]).sum(-1) * D**-0.5  # [Nk, Hk]
    want = (torch.softmax(s, 0)[:, :, None] * v[2].double()).sum(0)
    bound = (torch.softmax(s, 0)[:, :, None] * v[2].double().abs()).sum(0) * (2.0**-8 + 0.08 * 2**-8) + want.abs() * 2.0**-8
    assert ((few[0, 0].double() - want).abs() <= bound).all()
    assert ((out[2, 0].double() - want).abs() <= bound).all()
    del s, want, bound
    # many queries at the end of the last row
    q = normal(g, 1, 130, 1, D, dtype=torch.bfloat16)
    got = hz.token_attention(q, k[2:, :, 31:], v[2:, :, 31:], causal=True, documents=(torch.arange(Nk, device="cuda") >= Nk - 300).int()[None])
    want = hz.token_attention(q, k[2:, -300:, 31:].clone(), v[2:, -300:, 31:].clone(), causal=True)
    assert (got.float() - want.float()).abs().max() <= 2.0**-6 * want.float().abs().max()


# --- bias -----------------------------------------------------------------------------------------

BIAS = [  # B, Nq, Nk, H, buckets, R, positions
    (2, 33, 33, 4, 32, 128, "even"), (1, 1, 1, 1, 1, 0, "even"), (3, 17, 65, 12, 64, 16, "gaps"), (2, 64, 64, 8, 32, 128, "any"),
    (1, 100, 257, 16, 512, 512, "any"), (1, 9, 31, 256, 100, 40, "gaps"), (2, 5, 7, 3, 8, 4096, "extreme"), (1, 40, 130, 65, 200, 64, "any"),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout", ["qhk", "qkh"])
@pytest.mark.parametrize("case", BIAS, ids=lambda c: "-".join(map(str, c)))
def test_bucket_bias(case, layout, dtype):
    B, Nq, Nk, H, nb, R, where = case
    _say(f"bias {case} {layout} {dtype}")
    g = gen(9)
    table = torch.randn(nb, H, generator=g, device="cuda").requires_grad_()
    buckets = torch.randint(-1, nb + 1, (2 * R + 1,), generator=g, device="cuda").to(torch.int32)  # some are no row
    if where == "even":
        pos = [torch.arange(n, device="cuda").expand(B, n).to(torch.int32) for n in (Nq, Nk)]
    elif where == "gaps":
        pos = [torch.cumsum(torch.randint(1, 4, (B, n), generator=g, device="cuda"), 1).to(torch.int32) for n in (Nq, Nk)]
    elif where == "any":
        pos = [torch.randint(-R, R + 1, (B, n), generator=g, device="cuda").to(torch.int32) for n in (Nq, Nk)]
    else:
        pos = [torch.randint(-2**31, 2**31 - 1, (B, n), generator=g, device="cuda").to(torch.int32) for n in (Nq, Nk)]
    e = hz.bucket_bias(table, buckets, *pos, e_layout=layout, dtype=DT[dtype])
    de = normal(g, *e.shape, dtype=DT[dtype])
    (dt,) = torch.autograd.grad(e, (table,), de)
    (dt2,) = torch.autograd.grad(hz.bucket_bias(table, buckets, *pos, e_layout=layout, dtype=DT[dtype]), (table,), de)
    assert torch.equal(dt, dt2)
    turn = (lambda x: x) if layout == "qkh" else (lambda x: x.transpose(0, 1, 3, 2))
    want, grad, size = O.bucket_bias(arr(table), buckets.cpu().numpy(), *(x.cpu().numpy() for x in pos), turn(arr(de)))
    within("e", e, turn(want), (0 if dtype == "f32" else 2.0**-8) * np.abs(turn(want)))
    # a thread's column of n terms, then the columns and workgroups: below 2^-24 sqrt-free n' = 1024 terms here
    within("dtable", dt, grad, 1024 * F * size)


# --- refusals -------------------------------------------------------------------------------------


def test_entry_points_refuse():
    x = torch.zeros(2, 8, 4, 32, device="cuda")
    i = torch.zeros(2, 8, dtype=torch.int32, device="cuda")
    f = torch.zeros(8, dtype=torch.float64, device="cuda")
    bad = [
        (ValueError, lambda: hz.token_attention(x, x[:, :0], x[:, :0])),
        (ValueError, lambda: hz.token_attention(x, x, x[:, :4])),
        (ValueError, lambda: hz.token_attention(x, x[:, :, :3], x[:, :, :3])),
        (ValueError, lambda: hz.token_attention(x[..., :20], x[..., :20], x[..., :20])),
        (TypeError, lambda: hz.token_attention(x, x.bfloat16(), x)),
        (TypeError, lambda: hz.token_attention(x, x, x, documents=i.long())),
        (ValueError, lambda: hz.token_attention(x, x, x, documents=i[:1])),
        (ValueError, lambda: hz.token_attention(x, x, x, prefix=i[:, 0])),
        (ValueError, lambda: hz.token_attention(x, x, x, kv_len=i[:, 0].cpu())),
        (ValueError, lambda: hz.token_attention(x, x, x, slopes=torch.zeros(4, device="cuda", requires_grad=True))),
        (hz._native.HzError, lambda: hz.token_attention(x, x, x, softcap=-1.0)),
        (hz._native.HzError, lambda: hz.token_attention(x, x, x, scale=float("nan"))),
        (ValueError, lambda: hz.qk_norm_rotary(x, x, freqs=f[:6])),
        (TypeError, lambda: hz.qk_norm_rotary(x, x, freqs=f.float())),
        (TypeError, lambda: hz.qk_norm_rotary(x, x, torch.ones(32, device="cuda", dtype=torch.bfloat16))),
        (TypeError, lambda: hz.qk_norm_rotary(x, x, positions=i.long())),
        (ValueError, lambda: hz.qk_norm_rotary(x, x[:, :4])),
        (ValueError, lambda: hz.qk_norm_rotary(x, x, out=(x, x.clone().transpose(2, 3)))),
        (ValueError, lambda: hz.qk_norm_rotary(x.clone().requires_grad_(), x, out=(x, x))),
        (TypeError, lambda: hz.bucket_bias(f[:4].view(2, 2), i[0, :3], i, i)),
        (ValueError, lambda: hz.bucket_bias(x[0, 0], i[0, :4], i, i)),
        (ValueError, lambda: hz.bucket_bias(x[0, 0], i[0, :3], i, i[:1])),
        (ValueError, lambda: hz.bucket_bias(x[0, 0], i[0, :3], i, i, e_layout="compact")),
        (TypeError, lambda: hz.bucket_bias(x[0, 0], i[0, :3], i, i, dtype=torch.float16)),
    ]
    for n, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            raise AssertionError(f"case {n} was not refused")
    out = hz.token_attention(x.clone().requires_grad_(), x, x)
    (dx,) = torch.autograd.grad(out.sum(), [out.grad_fn.next_functions[0][0].variable], create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()

"""The token operators as a model uses them: together and with the attention that was there, on other streams, captured
into graphs, in calls that divide their work, and twice with the same bits."""

import numpy as np
import pytest
import torch

import hamiltonzero_amd as hz
from hamiltonzero_amd import kernels
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


def within(name, got, want, bound):
    got = arr(got)
    off = np.abs(got - want)
    worst = float(np.max(off / np.maximum(bound, 1e-300)))
    print(f"  {name}: {worst:.3f} of its bound, {off.max() / np.abs(want).max():.1e} of the largest value", flush=True)
    assert (off <= bound).all(), (name, worst, np.argwhere(~(off <= bound))[:4].tolist())


# --- calls that divide their work -------------------------------------------------------------------

DIVIDED = [  # B, Nq, Nk, H, Hk, D, options: few workgroups, so keys, queries and heads are shared out
    (1, 700, 700, 1, 1, 16, dict(causal=True)),
    (1, 513, 1500, 2, 1, 32, dict(causal=True, softcap=9.0)),
    (1, 300, 900, 4, 1, 64, dict(causal=True, slopes=True)),
    (1, 5000, 5000, 1, 1, 16, dict(causal=True, documents=7)),  # more than 64 tiles: the walk's second group
    (1, 4500, 4500, 2, 1, 8, dict(documents=3, softcap=4.0)),
    (1, 260, 9000, 1, 1, 16, dict(causal=True, documents=2)),
    (2, 640, 640, 3, 3, 24, dict(causal=True, documents=4, prefix=True)),
    (1, 1, 20000, 2, 1, 16, dict(causal=True)),
    (1, 6, 3000, 6, 1, 128, dict(causal=True, documents=2)),  # 36 rows: the kernel of many queries, divided
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", DIVIDED, ids=lambda c: "%d-%d-%d-%d-%d-%d-%s" % (*c[:6], "-".join(f"{k}={v}" for k, v in c[6].items())))
def test_divided_attention(case, dtype):
    B, Nq, Nk, H, Hk, D, o = case
    _say(f"divided {case} {dtype}")
    g = gen(11)
    dt = DT[dtype]
    q, k, v = (normal(g, *s, dtype=dt).requires_grad_() for s in ((B, Nq, H, D), (B, Nk, Hk, D), (B, Nk, Hk, D)))
    kw = {n: o[n] for n in ("causal", "softcap") if n in o}
    if "slopes" in o:
        kw["slopes"] = torch.full((H,), 0.01, device="cuda")
    if "documents" in o:
        cpu = torch.Generator().manual_seed(2)
        kw["documents"] = torch.sort(torch.randint(0, o["documents"], (B, Nk), generator=cpu), 1).values.to(torch.int32).cuda()
        kw["documents"][:, -min(7, Nq // 3):] = -1
    if "prefix" in o:
        kw["prefix"] = torch.tensor([100, 333], dtype=torch.int32, device="cuda")
    out = hz.token_attention(q, k, v, **kw)
    dout = normal(g, *out.shape, dtype=dt)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    again = hz.token_attention(q, k, v, **kw)
    assert torch.equal(out, again)
    for a, b in zip(grads, torch.autograd.grad(again, (q, k, v), dout)):
        assert torch.equal(a, b)  # no order of workgroups shows
    okw = {n: x.cpu().numpy() if isinstance(x, torch.Tensor) else x for n, x in kw.items()}
    want = O.attention(arr(q), arr(k), arr(v), scale=float(np.float32(D**-0.5)), dout=arr(dout), bf16=dtype == "bf16", **okw)
    for name, x in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        within(name, x, want[name], want["t_" + name])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,Nq,Nk,H,Hk,D,kw", [  # more than 512 blocks of queries: they begin the longest first
    (71, 40, 40, 8, 4, 16, dict()), (5, 300, 300, 48, 2, 8, dict(causal=True)), (9, 130, 700, 32, 8, 16, dict(causal=True, prefix=True)),
    (3, 700, 333, 32, 16, 8, dict(kv_len=True)), (2, 2000, 2100, 17, 1, 8, dict(causal=True, kv_len=True)),
], ids=lambda v: str(v) if not isinstance(v, dict) else "-".join(v) or "both")
def test_documents_of_many_blocks(B, Nq, Nk, H, Hk, D, kw, dtype):
    _say(f"many blocks {B} {Nq} {Nk} {H} {Hk} {D} {kw} {dtype}")
    g, cpu, dt = gen(18), torch.Generator().manual_seed(3), DT[dtype]
    q, k, v = (normal(g, *s, dtype=dt).requires_grad_() for s in ((B, Nq, H, D), (B, Nk, Hk, D), (B, Nk, Hk, D)))
    docs = torch.randint(0, 5, (B, Nk), generator=cpu).sort(1).values.to(torch.int32)
    docs[:, -3:] = -1
    docs[1] = torch.randint(-1, 4, (Nk,), generator=cpu).to(torch.int32)  # in no order
    kw = dict(kw, documents=docs.cuda())
    if "prefix" in kw:
        kw["prefix"] = torch.randint(0, Nk, (B,), generator=cpu).to(torch.int32).cuda()
    if "kv_len" in kw:
        kw["kv_len"] = torch.randint(0, Nk + 1, (B,), generator=cpu).to(torch.int32).cuda()
    out = hz.token_attention(q, k, v, **kw)
    dout = normal(g, *out.shape, dtype=dt)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    again = hz.token_attention(q, k, v, **kw)
    assert torch.equal(out, again)
    for a, b in zip(grads, torch.autograd.grad(again, (q, k, v), dout)):
        assert torch.equal(a, b)
    okw = {n: x.cpu().numpy() if isinstance(x, torch.Tensor) else x for n, x in kw.items()}
    rows = slice(0, 4)
    okw = {n: x[rows] if isinstance(x, np.ndarray) else x for n, x in okw.items()}
    want = O.attention(arr(q)[rows], arr(k)[rows], arr(v)[rows], scale=float(np.float32(D**-0.5)), dout=arr(dout)[rows], bf16=dtype == "bf16", **okw)
    for name, x in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        within(name, x[rows], want[name], want["t_" + name])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cap", [0.0, 50.0])
@pytest.mark.parametrize("N,D", [(24, 64), (200, 16), (333, 128)])
def test_errors_are_those_of_a_float32_computation(N, D, cap, dtype):
    """Root mean squares of the errors, next to those of the definition in float32 operations rounded to the type. A
    weight rounded to bfloat16 where it meets v or dout adds as much again as a result's rounding, sqrt(2) in all; the
    score gradients have two parts; so half again bounds every one. (float32: 1e-6 where there is next to no error.)"""
    g = gen(16)
    B, H, dt = 4, 4, DT[dtype]
    x = [normal(g, B, N, H, D, std=s, dtype=dt).requires_grad_() for s in (3.0, 1.0, 1.0)]
    cot = normal(g, B, N, H, D, dtype=dt)
    out = hz.token_attention(*x, causal=True, softcap=cap)
    got = [out, *torch.autograd.grad(out, x, cot)]

    def definition(float_, device):
        q, k, v = (t.detach().to(device, float_).transpose(1, 2).contiguous().requires_grad_() for t in x)
        y = (q @ k.transpose(-1, -2).contiguous()) * D**-0.5
        if cap:
            y = cap * torch.tanh(y / cap)
        y = y.masked_fill(torch.ones(N, N, dtype=torch.bool, device=device).triu(1), -torch.inf)
        o = y.softmax(-1) @ v
        res = [o, *torch.autograd.grad(o, (q, k, v), cot.to(device, float_).transpose(1, 2))]
        return [r.detach().transpose(1, 2) for r in res]

    for name, a, b, c in zip(("out", "dq", "dk", "dv"), got, definition(torch.float32, "cuda"), definition(torch.float64, "cpu")):
        size = c.norm()
        own = ((a.detach().double().cpu() - c).norm() / size).item()
        plain_ = ((b.to(dt).double().cpu() - c).norm() / size).item()
        print(f"  {name}: {own:.2e}, in float32 operations {plain_:.2e}", flush=True)
        assert own <= max(1.5 * plain_, 1e-6), name


def test_tables_anywhere():
    """Tables and positions that start in the middle of an allocation, one element past a 16-byte border."""
    s = inputs(21, torch.float32)
    for n in ("q", "k", "v", "dq", "dk", "pos", "n", "docs", "de"):
        s[n] = s[n][:1]
    want = everything(leaves(s))
    moved = dict(s)
    for n in ("w", "freqs", "slopes", "pos", "table", "n", "docs", "plan"):
        room = torch.empty(s[n].numel() + 1, dtype=s[n].dtype, device="cuda")
        moved[n] = room[1:].view(s[n].shape).copy_(s[n])
        assert moved[n].data_ptr() % 16 and moved[n].is_contiguous()
    for n in ("w", "table"):
        moved[n].requires_grad_()
    for n in ("q", "k", "v"):
        moved[n] = s[n].clone().requires_grad_()
    for a, b in zip(everything(moved), want):
        assert torch.equal(a, b)


def test_some_leaves_only_and_one_leaf_for_all():
    g = gen(17)
    x, k = normal(g, 2, 70, 4, 32), normal(g, 2, 70, 4, 32)
    three = [x.clone().requires_grad_() for _ in range(3)]
    out = hz.token_attention(*three, causal=True)
    want = torch.autograd.grad(out.sum(), three)
    one = x.clone().requires_grad_()
    same = hz.token_attention(one, one, one, causal=True)
    assert torch.equal(same, out)
    got, = torch.autograd.grad(same.sum(), one)  # the three are added in an order of torch's own
    assert (got - sum(want)).abs().max() <= 4 * F * sum(w.abs() for w in want).max()
    full = [x.clone().requires_grad_(), k.clone().requires_grad_(), x.clone().requires_grad_()]
    want = torch.autograd.grad(hz.token_attention(*full).square().sum(), full)
    for i in range(3):
        part = [t.detach().clone().requires_grad_(i == j) for j, t in enumerate(full)]
        got, = torch.autograd.grad(hz.token_attention(*part).square().sum(), part[i])
        assert torch.equal(got, want[i])


def test_more_refusals():
    x = torch.zeros(2, 8, 4, 32, device="cuda")
    y, room = torch.empty_like(x), torch.empty(1, 8, 4, 32, device="cuda").expand(2, 8, 4, 32)
    for out in ((x, y), (y, x), (y, y), (room, y)):
        with pytest.raises(ValueError, match="overlap|several places"):
            hz.qk_norm_rotary(x, x.clone(), out=out)
    import torch.autograd.forward_ad as fwd

    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: hz.token_attention(x, d, x), lambda: hz.qk_norm_rotary(d, x)):
            with pytest.raises(NotImplementedError, match="forward mode"):
                call()
        assert hz.token_attention(x, x, x).shape == x.shape
    with pytest.raises(RuntimeError):  # once differentiable
        q = x.clone().requires_grad_()
        a, = torch.autograd.grad(hz.token_attention(q, x, x).sum(), q, create_graph=True)
        torch.autograd.grad(a.sum(), q)


# --- together -------------------------------------------------------------------------------------


def model(x, w_in, w_q, w_k, freqs, positions, **kw):
    """One attention block up to its output projection: two query heads a key head."""
    B, N, _ = x.shape
    rows = (x @ w_in).view(B, N, 8, 32)
    q, k = hz.qk_norm_rotary(rows[:, :, :4], rows[:, :, 4:6], w_q, w_k, freqs=freqs, positions=positions)
    return hz.token_attention(q, k, rows[:, :, 6:], **kw)


def plain(x, w_in, w_q, w_k, freqs, documents, cap):
    """The same in float64 torch operations."""
    B, N, _ = x.shape
    rows = (x @ w_in).view(B, N, 8, 32)
    t = torch.arange(N, dtype=torch.float64)[:, None] * freqs
    c, s = t.cos()[:, None], t.sin()[:, None]

    def norm(y, w):
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w
        a, b = y[..., :16], y[..., 16:]
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    q, k, v = norm(rows[:, :, :4], w_q), norm(rows[:, :, 4:6], w_k), rows[:, :, 6:]
    k, v = k.repeat_interleave(2, 2), v.repeat_interleave(2, 2)
    y = cap * torch.tanh(torch.einsum("bihd,bjhd->bhij", q, k) * 32**-0.5 / cap)
    seen = torch.ones(N, N, dtype=torch.bool).tril() & (documents[:, :, None] == documents[:, None, :])
    return torch.einsum("bhij,bjhd->bihd", y.masked_fill(~seen[:, None], -torch.inf).softmax(-1), v)


def test_training_block_against_float64():
    """x through a projection, the norms with rotation and the attention, and back, in float32: the chain's relative
    error is the projection's 64-term sums and a few roundings an operator, far below 1e-5 of each result's size."""
    g = gen(12)
    B, N = 2, 150
    leaves = [normal(g, B, N, 64), normal(g, 64, 256, std=64**-0.5), 1 + 0.2 * normal(g, 32), 1 + 0.2 * normal(g, 32)]
    freqs = 100.0 ** (-torch.arange(16, dtype=torch.float64, device="cuda") / 16)
    docs = (torch.arange(N, device="cuda") > 60).int().expand(B, N).contiguous()
    pos = torch.arange(N, device="cuda", dtype=torch.int32).expand(B, N)
    x = [t.clone().requires_grad_() for t in leaves]
    out = model(*x, freqs, pos, causal=True, documents=docs, softcap=10.0)
    cot = normal(g, *out.shape)
    got = torch.autograd.grad(out, x, cot)
    y = [t.double().cpu().requires_grad_() for t in leaves]
    ref = plain(*y, freqs.cpu(), docs.cpu(), 10.0)
    want = torch.autograd.grad(ref, y, cot.double().cpu())
    for a, b in zip((out, *got), (ref, *want)):
        assert (a.detach().double().cpu() - b).abs().max() <= 1e-5 * b.abs().max()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_tokens_after_a_cache_match_the_whole_sequence(dtype):
    """A prompt of 70 tokens, then one token at a time with the keys written into a cache by the norm kernel."""
    g = gen(13)
    dt = DT[dtype]
    B, N, H, Hk, D, start = 3, 90, 8, 2, 64, 70
    q, k, v = normal(g, B, N, H, D, dtype=dt), normal(g, B, N, Hk, D, dtype=dt), normal(g, B, N, Hk, D, dtype=dt)
    freqs = 10000.0 ** (-torch.arange(32, dtype=torch.float64, device="cuda") / 32)
    pos = torch.arange(N, dtype=torch.int32, device="cuda").expand(B, N).contiguous()
    kw = dict(softcap=15.0, causal=True, slopes=torch.full((H,), 0.02, device="cuda"))
    qn, kn = hz.qk_norm_rotary(q, k, freqs=freqs, positions=pos)
    want = hz.token_attention(qn, kn, v, **kw).float()
    k_cache = torch.full((B, 128, Hk, D), float("nan"), dtype=dt, device="cuda")
    v_cache = k_cache.clone()
    v_cache[:, :start] = v[:, :start]
    q_row = torch.empty(B, start, H, D, dtype=dt, device="cuda")
    hz.qk_norm_rotary(q[:, :start], k[:, :start], freqs=freqs, positions=pos[:, :start], out=(q_row, k_cache[:, :start]))
    n = torch.full((B,), start, dtype=torch.int32, device="cuda")
    rows = [hz.token_attention(q_row, k_cache, v_cache, kv_len=n, **kw)]
    q_row = torch.empty(B, 1, H, D, dtype=dt, device="cuda")
    for i in range(start, N):
        v_cache[:, i] = v[:, i]
        hz.qk_norm_rotary(q[:, i:i + 1], k[:, i:i + 1], freqs=freqs, positions=pos[:, i:i + 1], out=(q_row, k_cache[:, i:i + 1]))
        n += 1
        rows.append(hz.token_attention(q_row, k_cache, v_cache, kv_len=n, **kw))
    got = torch.cat(rows, 1).float()
    # both sides within the operator's bound of the same exact values: twice it, as a share of the largest value
    bound = 2 * (2.0**-8 * 3 if dtype == "bf16" else 2e-5)
    assert (got - want).abs().max() <= bound * v.float().abs().max()


@pytest.mark.parametrize("layout", ["qhk", "qkh"])
def test_learned_bias_into_the_edge_attention(layout):
    """bucket_bias gives mhsea_ad its e and takes its gradient; float32 against float64."""
    g = gen(14)
    B, N, H, D = 3, 64, 8, 32
    q, k, v = (normal(g, B, N, H, D, std=0.5).requires_grad_() for _ in range(3))
    table = normal(g, 32, H).requires_grad_()
    plan = hz.relative_buckets(32, 16, device="cuda")
    pos = torch.cumsum(torch.randint(1, 3, (B, N), generator=g, device="cuda"), 1).to(torch.int32)
    mask = torch.ones(B, N, dtype=torch.bool, device="cuda")
    mask[1, 40:] = False
    e = hz.bucket_bias(table, plan, pos, pos, e_layout=layout)
    out, _ = hz.mhsea_ad(q, k, e, v, mask, scale=D**-0.5, e_layout=layout)
    cot = normal(g, *out.shape)
    got = torch.autograd.grad(out, (q, k, v, table), cot)
    x = [t.detach().double().cpu().requires_grad_() for t in (q, k, v, table)]
    d = (pos[:, None, :].long() - pos[:, :, None].long()).clamp(-16, 16).cpu() + 16
    bias = x[3][plan.long().cpu()[d]]  # [B, N, N, H]
    s = torch.einsum("bihd,bjhd->bhij", x[0], x[1]) * D**-0.5 + bias.permute(0, 3, 1, 2)
    m = mask.cpu()
    s = s.masked_fill(~m[:, None, None, :], -torch.inf)
    ref = torch.einsum("bhij,bjhd->bihd", s.softmax(-1), x[2]) * m[:, :, None, None]
    want = torch.autograd.grad(ref, x, cot.double().cpu())
    for a, b in zip((out, *got), (ref, *want)):
        assert (a.detach().double().cpu() - b).abs().max() <= 1e-5 * b.abs().max()  # the edge attention's own tolerance


def test_learned_bias_into_the_rectangular_attention():
    g = gen(15)
    B, Nq, Nk, H, D = 1, 40, 130, 4, 32
    q, k, v = normal(g, B, Nq, H, D), normal(g, B, Nk, H, D), normal(g, B, Nk, H, D)
    table, plan = normal(g, 32, H), hz.relative_buckets(32, 64, bidirectional=False, device="cuda")
    qp = torch.arange(Nk - Nq, Nk, dtype=torch.int32, device="cuda")[None]
    kp = torch.arange(Nk, dtype=torch.int32, device="cuda")[None]
    e = hz.bucket_bias(table, plan, qp, kp, e_layout="qkh")
    out = kernels.rect_attention_fwd(q, k, v, e, scale=D**-0.5)
    s = torch.einsum("bihd,bjhd->bhij", q.double(), k.double()) * D**-0.5
    s = s + O_bias(table, plan, qp, kp)
    want = torch.einsum("bhij,bjhd->bihd", s.softmax(-1), v.double())
    assert (out.double() - want).abs().max() <= 1e-5 * want.abs().max()


def O_bias(table, plan, qp, kp):
    e = O.bucket_bias(arr(table), plan.cpu().numpy(), qp.cpu().numpy(), kp.cpu().numpy())
    return torch.from_numpy(e).permute(0, 3, 1, 2).cuda()


# --- streams and graphs -----------------------------------------------------------------------------


def everything(s):
    """Every kernel of the operators once, forward and reverse: a list of results."""
    res = []
    q, k = hz.qk_norm_rotary(s["q"], s["k"], s["w"], s["w"], freqs=s["freqs"], positions=s["pos"])
    res += [q, k, *torch.autograd.grad((q, k), (s["q"], s["k"], s["w"]), (s["dq"], s["dk"]))]
    for kw in (dict(causal=True, softcap=5.0, documents=s["docs"]), dict(causal=True, slopes=s["slopes"])):
        out = hz.token_attention(s["q"], s["k"], s["v"], **kw)
        res += [out, *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dq"])]
    wide = s["q"].detach().repeat(1, 1, 70, 1)  # more than 512 blocks: documents put them in order
    out = hz.token_attention(wide, s["k"], s["v"], documents=s["docs"])
    res += [out, *torch.autograd.grad(out, (s["k"], s["v"]), wide)]
    res.append(hz.token_attention(s["q"].detach()[:, :2], s["k"].detach(), s["v"].detach(), causal=True, kv_len=s["n"]))
    for layout, de in (("qhk", s["de"]), ("qkh", s["de"].transpose(2, 3))):
        e = hz.bucket_bias(s["table"], s["plan"], s["pos"], s["pos"], e_layout=layout, dtype=s["q"].dtype)
        res += [e, *torch.autograd.grad(e, (s["table"],), de)]
    return res


def inputs(seed, dtype):
    g = gen(seed)
    B, N, H, Hk, D = 2, 200, 4, 2, 64
    s = dict(q=normal(g, B, N, H, D, dtype=dtype), k=normal(g, B, N, Hk, D, dtype=dtype), v=normal(g, B, N, Hk, D, dtype=dtype),
             dq=normal(g, B, N, H, D, dtype=dtype), dk=normal(g, B, N, Hk, D, dtype=dtype), w=1 + 0.1 * normal(g, D),
             freqs=torch.rand(32, generator=g, dtype=torch.float64, device="cuda"), slopes=0.1 * torch.rand(H, generator=g, device="cuda"),
             pos=torch.randint(0, 500, (B, N), generator=g, device="cuda").to(torch.int32), table=normal(g, 32, H),
             n=torch.randint(2, N + 1, (B,), generator=g, device="cuda").to(torch.int32), de=normal(g, B, N, H, N, dtype=dtype))
    s["docs"] = torch.sort(torch.randint(0, 3, (B, N), generator=g, device="cuda"), 1).values.to(torch.int32)
    s["docs"][:, -5:] = -1
    s["plan"] = hz.relative_buckets(32, 128, device="cuda")
    return s


def leaves(s):
    return {n: t.detach().clone().requires_grad_(n in ("q", "k", "v", "w", "table")) for n, t in s.items()}


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_side_streams(dtype):
    """The same bits from another stream than the tensors', and from two streams at once."""
    s = inputs(20, DT[dtype])
    want = everything(leaves(s))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append(everything(leaves(s)))
    torch.cuda.synchronize()
    for r in got:
        for a, b in zip(r, want):
            assert torch.equal(a, b)


def test_two_threads():
    """Each thread on a stream of its own, all operators several times: the bits of one thread alone."""
    import threading

    s = inputs(22, torch.bfloat16)
    want = everything(leaves(s))
    torch.cuda.synchronize()
    got, failed = [], []

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got.append(everything(leaves(s)))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # shown by the assertion below
            failed.append(e)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and len(got) == 10
    for r in got:
        for a, b in zip(r, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_captured_and_replayed(dtype):
    """Two captured graphs of all operators, replayed in turn with new inputs and eager work between."""
    _say(f"graphs {dtype}")
    graphs = []
    for seed in (30, 31):
        s = leaves(inputs(seed, DT[dtype]))  # leaves of this graph's own: no eager graph of theirs lives
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            everything(s)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = everything(s)
        graphs.append((graph, s, res))
    for round_ in range(3):
        for i, (graph, s, res) in enumerate(graphs):
            new = inputs(40 + 2 * round_ + i, DT[dtype])
            with torch.no_grad():
                for n in s:
                    s[n].copy_(new[n])
            graph.replay()
            eager = everything(leaves(new))
            torch.cuda.synchronize()
            for a, b in zip(res, eager):
                assert torch.equal(a, b), (round_, i)

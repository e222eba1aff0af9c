"""The token operators' work: query/key norms with rotation, masked and capped attention over tokens, and the
learned relative position bias, as cases that can be timed and compared.

A case is a dict of plain values. ``kind`` is the operator, ``pass`` is ``fwd`` (a call without gradients) or
``train`` (the call and the gradients of its inputs for a given cotangent). ``layout`` draws what belongs to the case
and not to its values: the lengths of a cache's rows, where documents and prefixes end.

``run`` computes the operators in elementary torch operations, or, with ``own``, by the package's calls.
"""

from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2}
EPS = 1e-6


def listed():
    return [
        # One decoded token of 64 sequences at far positions: the smallest norm-and-rotation call.
        dict(name="qk_token_bf16", kind="qk", **{"pass": "fwd"}, B=64, N=1, H=32, Hk=8, D=128, rot=128, interleaved=False,
             far=131072, dtype="bf16"),
        # A training step's queries and keys with shared key heads.
        dict(name="qk_train_bf16", kind="qk", **{"pass": "train"}, B=4, N=4096, H=32, Hk=8, D=128, rot=128,
             interleaved=False, far=0, dtype="bf16"),
        # Sites of a 15 x 15 lattice for many walkers, half of each head rotated, in float32.
        dict(name="qk_train_sites_f32", kind="qk", **{"pass": "train"}, B=256, N=225, H=8, Hk=8, D=64, rot=32,
             interleaved=True, far=0, dtype="f32"),
        # One token of a few short sequences: the smallest attention call.
        dict(name="attn_token_short_f32", kind="attn", **{"pass": "fwd"}, B=4, Nq=1, Nk=777, H=8, Hk=8, D=64, cap=0.0,
             slopes=True, causal=True, docs=0, prefix=False, cache=True, layout=1, dtype="f32"),
        # One token of each of 16 sequences with caches up to 32768 tokens long.
        dict(name="attn_token_long_bf16", kind="attn", **{"pass": "fwd"}, B=16, Nq=1, Nk=32768, H=32, Hk=8, D=128,
             cap=50.0, slopes=False, causal=True, docs=0, prefix=False, cache=True, layout=2, dtype="bf16"),
        # Two prompts with capped scores.
        dict(name="attn_prompt_bf16", kind="attn", **{"pass": "fwd"}, B=2, Nq=4096, Nk=4096, H=16, Hk=4, D=128, cap=30.0,
             slopes=False, causal=True, docs=0, prefix=False, cache=False, layout=3, dtype="bf16"),
        # A training step over one packed row of documents, its end padded.
        dict(name="attn_train_packed_bf16", kind="attn", **{"pass": "train"}, B=1, Nq=8192, Nk=8192, H=16, Hk=4, D=128,
             cap=50.0, slopes=False, causal=True, docs=4, prefix=False, cache=False, layout=4, dtype="bf16"),
        # Lattice sites as tokens behind a prefix that all of them see, with a distance bias, in float32.
        dict(name="attn_train_sites_f32", kind="attn", **{"pass": "train"}, B=64, Nq=225, Nk=225, H=8, Hk=8, D=32,
             cap=0.0, slopes=True, causal=True, docs=0, prefix=True, cache=False, layout=5, dtype="f32"),
        # Documents read in both directions, an odd length, capped, in float32.
        dict(name="attn_train_both_f32", kind="attn", **{"pass": "train"}, B=3, Nq=1021, Nk=1021, H=8, Hk=4, D=64,
             cap=20.0, slopes=True, causal=False, docs=3, prefix=False, cache=False, layout=6, dtype="f32"),
        # The smallest bias: a few short systems.
        dict(name="bias_small_f32", kind="bias", **{"pass": "fwd"}, B=4, Nq=33, Nk=33, H=4, nb=32, R=128, both=True,
             e_layout="qhk", dtype="f32"),
        # The bias of 1024 walkers of 64 sites, and its table's gradient.
        dict(name="bias_train_sites_f32", kind="bias", **{"pass": "train"}, B=1024, Nq=64, Nk=64, H=8, nb=32, R=128,
             both=True, e_layout="qhk", dtype="f32"),
        # Long rows with the heads innermost, an odd length, in bfloat16.
        dict(name="bias_train_rows_bf16", kind="bias", **{"pass": "train"}, B=2, Nq=1777, Nk=2048, H=16, nb=64, R=512,
             both=False, e_layout="qkh", dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    kind = rng.choice(["qk", "attn", "attn", "attn", "bias"])
    dtype = rng.choice(["f32", "bf16"])
    if kind == "qk":
        train = rng.random() < 0.6
        D = rng.choice([16, 32, 64, 80, 128])
        Hk = rng.choice([1, 2, 4, 8])
        H = Hk * rng.choice([1, 2, 4])
        N = _log(rng, 1, 4096)
        B = _log(rng, 1, max(1, min(64, 16384 // N)))
        return dict(kind="qk", **{"pass": "train" if train else "fwd"}, B=B, N=N, H=H, Hk=Hk, D=D,
                    rot=rng.choice([D, D // 2]), interleaved=rng.random() < 0.5, far=rng.choice([0, 131072]), dtype=dtype)
    if kind == "bias":
        train = rng.random() < 0.6
        H = rng.choice([1, 4, 8, 12, 16])
        Nk = _log(rng, 1, 2048)
        Nq = Nk if rng.random() < 0.6 else _log(rng, 1, 1777)
        B = _log(rng, 1, max(1, min(1024, (1 << 22) // (Nq * Nk))))
        return dict(kind="bias", **{"pass": "train" if train else "fwd"}, B=B, Nq=Nq, Nk=Nk, H=H,
                    nb=rng.choice([8, 32, 64]), R=rng.choice([16, 128, 512]), both=rng.random() < 0.5,
                    e_layout=rng.choice(["qhk", "qkh"]), dtype=dtype)
    D = rng.choice([16, 32, 64, 80, 128])
    Hk = rng.choice([1, 2, 4, 8])
    H = Hk * rng.choice([1, 2, 4])
    cap = rng.choice([0.0, 0.0, 20.0, 50.0])
    slopes = rng.random() < 0.4
    layout = rng.randrange(1 << 20)
    if rng.random() < 0.35:  # tokens after a cache, one or a few
        Nk = _log(rng, 1, 32768)
        B = _log(rng, 1, min(32, (1 << 18) // Nk))
        return dict(kind="attn", **{"pass": "fwd"}, B=B, Nq=rng.choice([1, 1, 1, 2, 5]), Nk=Nk, H=H, Hk=Hk, D=D, cap=cap,
                    slopes=slopes, causal=True, docs=0, prefix=False, cache=True, layout=layout, dtype=dtype)
    H = min(H, Hk * max(1, 2048 // (Hk * D)))
    N = _log(rng, 2, 2800 if dtype == "bf16" else 1024)
    B = _log(rng, 1, max(1, min(64, (1 << 22 if dtype == "bf16" else 1 << 20) // (N * N))))
    causal = rng.random() < 0.7
    return dict(kind="attn", **{"pass": rng.choice(["fwd", "train"])}, B=B, Nq=N, Nk=N, H=H, Hk=Hk, D=D, cap=cap,
                slopes=slopes, causal=causal, docs=rng.choice([0, 0, 1, 4]), prefix=causal and rng.random() < 0.4,
                cache=False, layout=layout, dtype=dtype)


# --- what belongs to a case and not to its values -------------------------------------------------------------------

def _kv_len(case):
    """Tokens in each row of a cache; rows are ragged."""
    if not case["cache"]:
        return None
    r = random.Random(case["layout"])
    least = min(case["Nq"], case["Nk"])
    return [r.randint(max(least, case["Nk"] // 4), case["Nk"]) for _ in range(case["B"])]


def _documents(case):
    """Documents of each packed row as (number, begin, end); behind the last one the row is padding."""
    if not case["docs"]:
        return None
    r = random.Random(case["layout"] + 1)
    rows = []
    for _ in range(case["B"]):
        end = case["Nk"] - r.randint(0, case["Nk"] // 8)
        cuts = sorted(r.randint(0, end) for _ in range(case["docs"] - 1))
        edges = [0, *cuts, end]
        rows.append([(n, a, b) for n, (a, b) in enumerate(zip(edges, edges[1:])) if b > a])
    return rows


def _prefix(case):
    if not case["prefix"]:
        return None
    r = random.Random(case["layout"] + 2)
    return [r.randint(0, case["Nk"] // 2) for _ in range(case["B"])]


def _pairs(case):
    """Visible pairs of query and key in all rows, for one head."""
    kv_len, docs, prefix = _kv_len(case), _documents(case), _prefix(case)

    def seen(begin, end, pre, first):  # queries first .. end - 1 against keys begin .. end - 1
        n = end - first
        if not case["causal"]:
            return n * (end - begin)
        pre = min(max(pre, begin), end)
        total = 0
        if first < pre:
            total += (min(pre, end) - first) * (pre - begin)
            first = min(pre, end)
        n = end - first
        return total + n * (first - begin) + n * (n + 1) // 2

    total = 0
    for b in range(case["B"]):
        n = kv_len[b] if kv_len else case["Nk"]
        pre = prefix[b] if prefix else 0
        spans = [(a, e) for _, a, e in docs[b]] if docs else [(0, n)]
        for a, e in spans:
            total += seen(a, e, pre, max(a, n - case["Nq"]))
    return total


def work(case):
    w = BYTES[case["dtype"]]
    train = case["pass"] == "train"
    if case["kind"] == "qk":
        n = case["B"] * case["N"] * (case["H"] + case["Hk"]) * case["D"]
        return {"bytes": n * w * (5 if train else 2), "flops": n * (20 if train else 7)}
    if case["kind"] == "bias":
        n = case["B"] * case["Nq"] * case["Nk"] * case["H"]
        return {"bytes": n * w * (2 if train else 1), "flops": n if train else 0}
    B, Nq, H, Hk, D = case["B"], case["Nq"], case["H"], case["Hk"], case["D"]
    keys = sum(_kv_len(case)) if case["cache"] else B * case["Nk"]
    qo, kv = B * Nq * H * D * w, 2 * keys * Hk * D * w
    flops = _pairs(case) * H * D * 4
    # a training pass reads q, k, v and the cotangent, and writes the output and the three gradients
    return {"bytes": 2 * qo + kv + (2 * qo + kv if train else 0), "flops": flops * (3.5 if train else 1)}


# --- inputs ---------------------------------------------------------------------------------------------------------

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _buckets(nb, R, both):
    """Bucket of each distance -R .. R: exact near ones, then ever wider ones; with ``both`` half of them for each sign."""
    half = nb // 2 if both else nb
    exact_ = half // 2
    out = []
    for d in range(-R, R + 1):
        n, base = (abs(d), half if d > 0 else 0) if both else (max(-d, 0), 0)
        if n >= exact_:
            n = exact_ + int(math.log(n / exact_) / math.log(max(R, exact_ + 1) / exact_) * (half - exact_))
        out.append(base + min(n, half - 1))
    return out


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = SimpleNamespace(case=case)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=DEVICE) * std).to(dt)

    train = case["pass"] == "train"
    if case["kind"] == "qk":
        B, N, H, Hk, D = (case[n] for n in ("B", "N", "H", "Hk", "D"))
        # both are slices of one projection's output, as a model holds them
        rows = normal(B, N, H + 2 * Hk, D)
        s.q, s.k = rows[:, :, :H], rows[:, :, H:H + Hk]
        s.wq = 1 + 0.2 * torch.randn(D, generator=g, device=DEVICE)
        s.wk = 1 + 0.2 * torch.randn(D, generator=g, device=DEVICE)
        half = case["rot"] // 2
        s.freqs = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEVICE) / half)
        first = torch.randint(0, case["far"] + 1, (B, 1), generator=g, device=DEVICE)
        s.positions = (first + torch.arange(N, device=DEVICE)).to(torch.int32)
        if train:
            s.q, s.k = s.q.detach().requires_grad_(), s.k.detach().requires_grad_()
            s.wq.requires_grad_(), s.wk.requires_grad_()
            s.dq, s.dk = normal(B, N, H, D), normal(B, N, Hk, D)
        return s
    if case["kind"] == "bias":
        B, Nq, Nk, H = (case[n] for n in ("B", "Nq", "Nk", "H"))
        s.table = torch.randn(case["nb"], H, generator=g, device=DEVICE)
        s.buckets = _ints(_buckets(case["nb"], case["R"], case["both"]))
        # sites in ascending order with gaps, another choice for each row
        s.kpos = torch.cumsum(torch.randint(1, 3, (B, Nk), generator=g, device=DEVICE), 1).to(torch.int32)
        s.qpos = s.kpos if Nq == Nk else torch.cumsum(torch.randint(1, 3, (B, Nq), generator=g, device=DEVICE), 1).to(torch.int32)
        if train:
            s.table.requires_grad_()
            s.de = normal(*((B, Nq, H, Nk) if case["e_layout"] == "qhk" else (B, Nq, Nk, H)))
        return s
    B, Nq, Nk, H, Hk, D = (case[n] for n in ("B", "Nq", "Nk", "H", "Hk", "D"))
    s.q, s.k, s.v = normal(B, Nq, H, D, std=3.0), normal(B, Nk, Hk, D), normal(B, Nk, Hk, D)
    s.slopes = None
    if case["slopes"]:
        s.slopes = 2.0 ** (-8.0 * torch.arange(1, H + 1, dtype=torch.float32, device=DEVICE) / H)
    kv_len, docs, prefix = _kv_len(case), _documents(case), _prefix(case)
    s.kv_len = None if kv_len is None else _ints(kv_len)
    s.prefix = None if prefix is None else _ints(prefix)
    s.documents = None
    if docs is not None:
        rows = [[-1] * Nk for _ in range(B)]
        for row, spans in zip(rows, docs):
            for n, a, b in spans:
                row[a:b] = [n] * (b - a)
        s.documents = _ints(rows)
    if train:
        s.q.requires_grad_(), s.k.requires_grad_(), s.v.requires_grad_()
        s.dout = normal(B, Nq, H, D)
    return s


# --- one pass -------------------------------------------------------------------------------------------------------

def run(s):
    c = s.case
    train = c["pass"] == "train"
    if not own:
        with torch.no_grad():
            return {"qk": _plain_qk, "attn": _plain_attn, "bias": _plain_bias}[c["kind"]](s, train)
    import hamiltonzero_amd as hz

    if c["kind"] == "qk":
        q, k = hz.qk_norm_rotary(s.q, s.k, s.wq, s.wk, freqs=s.freqs, positions=s.positions,
                                 interleaved=c["interleaved"], eps=EPS)
        return (q, k, *torch.autograd.grad((q, k), (s.q, s.k, s.wq, s.wk), (s.dq, s.dk))) if train else (q, k)
    if c["kind"] == "bias":
        e = hz.bucket_bias(s.table, s.buckets, s.qpos, s.kpos, e_layout=c["e_layout"], dtype=DTYPES[c["dtype"]])
        return (e, *torch.autograd.grad(e, (s.table,), s.de)) if train else (e,)
    out = hz.token_attention(s.q, s.k, s.v, softcap=c["cap"], slopes=s.slopes, causal=c["causal"], prefix=s.prefix,
                             documents=s.documents, kv_len=s.kv_len)
    return (out, *torch.autograd.grad(out, (s.q, s.k, s.v), s.dout)) if train else (out,)


def _turn(x, cos, sin, interleaved):
    """Rotates the pairs of the first 2 * half elements of each head."""
    half = cos.shape[-1]
    r, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :half], r[..., half:])
    a, b = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((r, rest), -1)


def _plain_qk(s, train):
    c = s.case
    t = s.positions.double()[:, :, None, None] * s.freqs
    cos, sin = t.cos().float(), t.sin().float()
    outs, grads, wgrads = [], [], []
    for x, w, dy in ((s.q, s.wq, s.dq if train else None), (s.k, s.wk, s.dk if train else None)):
        x = x.float()
        r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        n = x * r
        outs.append(_turn(n * w, cos, sin, c["interleaved"]).to(s.q.dtype))
        if train:
            d = _turn(dy.float(), cos, -sin, c["interleaved"])
            wgrads.append((d * n).double().sum((0, 1, 2)).float())
            d = d * w
            grads.append((r * (d - n * (d * n).mean(-1, keepdim=True))).to(s.q.dtype))
    return (*outs, *grads, *wgrads)


def _plain_attn(s, train):
    c = s.case
    B, Nq, Nk, H, Hk, D = (c[n] for n in ("B", "Nq", "Nk", "H", "Hk", "D"))
    G = H // Hk
    scale = D ** -0.5
    heads = lambda x: x.float().transpose(1, 2)  # noqa: E731  [B, heads, N, D]
    q = heads(s.q).reshape(B, Hk, G * Nq, D)
    k, v = heads(s.k), heads(s.v)
    x = (q @ k.transpose(-1, -2)).reshape(B, H, Nq, Nk) * scale
    t = torch.tanh(x / c["cap"]) if c["cap"] else None
    y = c["cap"] * t if c["cap"] else x
    j = torch.arange(Nk, device=DEVICE)
    n = torch.full((B,), Nk, device=DEVICE) if s.kv_len is None else s.kv_len.long()
    p = n[:, None] - Nq + torch.arange(Nq, device=DEVICE)  # [B, Nq]
    if s.slopes is not None:
        y = y - s.slopes[None, :, None, None] * (p[:, None, :, None] - j).abs()
    seen = (j < n[:, None])[:, None, :].expand(B, Nq, Nk)
    if c["causal"]:
        near = j <= p[:, :, None]
        if s.prefix is not None:
            near = near | (j < s.prefix[:, None])[:, None, :]
        seen = seen & near
    if s.documents is not None:
        d = s.documents
        dq = torch.where(p >= 0, d.gather(1, p.clamp(min=0)), -1)
        seen = seen & (dq[:, :, None] == d[:, None, :]) & (dq[:, :, None] >= 0)
    seen = seen[:, None]
    y = torch.where(seen, y, -math.inf)
    m = y.amax(-1, keepdim=True)
    w = torch.exp(y - torch.where(m == -math.inf, 0.0, m))
    z = w.sum(-1, keepdim=True)
    w = w / torch.where(z == 0, 1.0, z)
    packed = lambda x: x.reshape(B, Hk, G * Nq, -1)  # noqa: E731
    flat = lambda x, n_: x.reshape(B, n_, -1, D).transpose(1, 2).contiguous()  # noqa: E731
    o = packed(w) @ v
    out = flat(o, H).to(s.q.dtype)
    if not train:
        return (out,)
    do = heads(s.dout).reshape(B, Hk, G * Nq, D)
    dv = packed(w).transpose(-1, -2) @ do
    dw = (do @ v.transpose(-1, -2)).reshape(B, H, Nq, Nk)
    dy = w * (dw - (do * o).sum(-1).reshape(B, H, Nq, 1))
    if c["cap"]:
        dy = dy * (1 - t * t)
    dy = packed(dy * scale)
    dq, dk = dy @ k, dy.transpose(-1, -2) @ q
    return (out, *(flat(x, n_).to(s.q.dtype) for x, n_ in ((dq, H), (dk, Hk), (dv, Hk))))


def _plain_bias(s, train):
    c = s.case
    R = c["R"]
    d = s.kpos[:, None, :].long() - s.qpos[:, :, None].long()
    idx = s.buckets.long()[d.clamp(-R, R) + R]  # [B, Nq, Nk]
    e = s.table[idx].to(DTYPES[c["dtype"]])  # [B, Nq, Nk, H]
    if c["e_layout"] == "qhk":
        e = e.transpose(2, 3).contiguous()
    if not train:
        return (e,)
    de = s.de.transpose(2, 3) if c["e_layout"] == "qhk" else s.de
    # one row of pairs at a time by a product with its buckets, the rows' sums in 64 bits
    of = (idx[:, :, None, :] == torch.arange(c["nb"], device=DEVICE)[:, None]).float()
    return (e, (of @ de.float()).double().sum((0, 1)).float())


# --- the same in 64 bits, from the definitions ----------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"qk": _exact_qk, "attn": _exact_attn, "bias": _exact_bias}[case["kind"]](s, case["pass"] == "train")


def _exact_qk(s, train):
    c = s.case
    half = s.freqs.numel()
    at = torch.arange(half, device=DEVICE)
    ia, ib = (2 * at, 2 * at + 1) if c["interleaved"] else (at, at + half)
    angle = torch.outer(s.positions.reshape(-1).double(), s.freqs).reshape(*s.positions.shape, 1, half)
    z = torch.polar(torch.ones_like(angle), angle)  # a rotation is a product of complex numbers
    outs, xs, ws = [], [], []
    for x, w in ((s.q, s.wq), (s.k, s.wk)):
        x, w = x.detach().double().requires_grad_(train), w.detach().double().requires_grad_(train)
        xs.append(x), ws.append(w)
        y = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / c["D"] + EPS) * w
        turned = torch.complex(y[..., ia], y[..., ib]) * z
        outs.append(y.index_copy(-1, ia, turned.real).index_copy(-1, ib, turned.imag))
    if not train:
        return tuple(outs)
    grads = torch.autograd.grad(outs, (*xs, *ws), (s.dq.double(), s.dk.double()))
    return (*(o.detach() for o in outs), *grads)


def _exact_attn(s, train):
    c = s.case
    B, Nq, Nk, H, Hk, D = (c[n] for n in ("B", "Nq", "Nk", "H", "Hk", "D"))
    if B * H * Nq * Nk * D * (4 if train else 1) > 1 << 40:
        return None
    q, k, v = (x.detach().double().requires_grad_(train) for x in (s.q, s.k, s.v))
    out = torch.empty_like(q)
    grads = [torch.zeros_like(x) for x in (q, k, v)]
    for b in range(B):
        n = Nk if s.kv_len is None else int(s.kv_len[b])
        at = torch.arange(n - Nq, n, device=DEVICE)[:, None]
        key = torch.arange(Nk, device=DEVICE)[None, :]
        hidden = (key >= n).expand(Nq, Nk).clone()
        if c["causal"]:
            hidden |= (key > at) & (key >= (0 if s.prefix is None else int(s.prefix[b])))
        if s.documents is not None:
            number = torch.cat((s.documents[b], s.documents.new_full((1,), -1)))
            mine = number[torch.where(at < 0, Nk, at)]
            hidden |= (mine != s.documents[b][None, :]) | (mine < 0)
        some = ~hidden.all(1, keepdim=True)
        for h in range(H):
            i = h // (H // Hk)
            with torch.set_grad_enabled(train):
                y = q[b, :, h] @ k[b, :, i].T / math.sqrt(D)
                if c["cap"]:
                    y = torch.tanh(y / c["cap"]) * c["cap"]
                if s.slopes is not None:
                    y = y - float(s.slopes[h]) * (at - key).abs()
                # a row that sees nothing is computed over all keys and then left out
                y = y.masked_fill(hidden & some, -math.inf)
                o = torch.softmax(y, -1).masked_fill(~some, 0.0) @ v[b, :, i]
            out[b, :, h].detach().copy_(o.detach())
            if train:
                for total, part in zip(grads, torch.autograd.grad(o, (q, k, v), s.dout[b, :, h].double())):
                    total += part
    return (out.detach(), *grads) if train else (out.detach(),)


def _exact_bias(s, train):
    c = s.case
    B, Nq, Nk, H = (c[n] for n in ("B", "Nq", "Nk", "H"))
    far = (len(s.buckets) - 1) // 2
    e = torch.empty(B, Nq, Nk, H, dtype=torch.float64, device=DEVICE)
    number = torch.empty(B, Nq, Nk, dtype=torch.int64, device=DEVICE)
    for i in range(Nq):
        distance = torch.minimum(torch.maximum(s.kpos.long() - s.qpos[:, i:i + 1].long(), torch.tensor(-far, device=DEVICE)),
                                 torch.tensor(far, device=DEVICE))
        number[:, i] = s.buckets.long().take(distance + far)
    for h in range(H):
        e[..., h] = s.table.detach()[:, h].double().take(number)
    heads_inside = c["e_layout"] == "qkh"
    e = e if heads_inside else e.permute(0, 1, 3, 2).contiguous()
    if not train:
        return (e,)
    de = (s.de if heads_inside else s.de.permute(0, 1, 3, 2)).double()
    rows = [de[number == m].sum(0) for m in range(c["nb"])]
    return (e, torch.stack(rows))

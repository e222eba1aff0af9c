"""The paged operators' work: rotation of queries and keys by positions of several axes, new tokens appended to a
paged cache, attention of new tokens over it with the weights that each slot has had, and eviction by those weights, as
cases that can be timed and compared.

A case is a dict of plain values. ``kind`` is the operator, ``pass`` is ``fwd`` or ``train`` (the call and the gradients
of its inputs for a given cotangent; the rotations only). ``layout`` draws what belongs to the case and not to its values:
the tokens in each row of a cache. A cache is a pool of pages of ``S`` slots; a row's pages lie anywhere in it.

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
SPARE = 3  # pages of the pool that no row has


def listed():
    return [
        # The next site of 64 walkers on a cubic lattice: the smallest rotation.
        dict(name="rotary_token_bf16", kind="rotary", **{"pass": "fwd"}, B=64, N=1, H=32, Hk=8, D=128, rot=128, A=3,
             norm=False, interleaved=False, mixed=False, dtype="bf16"),
        # A training step over tokens of 8 layers of 30 x 34 sites, the axes' frequencies one after the other.
        dict(name="rotary_train_layers_bf16", kind="rotary", **{"pass": "train"}, B=2, N=8160, H=32, Hk=8, D=128, rot=128,
             A=3, norm=False, interleaved=False, mixed=False, dtype="bf16"),
        # Sites of a 15 x 15 lattice by row and column for many walkers, behind the norms, in float32.
        dict(name="rotary_train_sites_f32", kind="rotary", **{"pass": "train"}, B=256, N=225, H=8, Hk=8, D=64, rot=64,
             A=2, norm=True, interleaved=True, mixed=True, dtype="f32"),
        # One new token of each of 64 rows goes into its page.
        dict(name="append_token_bf16", kind="append", **{"pass": "fwd"}, B=64, N=1, Nk=256, S=16, Hk=8, D=128, layout=1,
             dtype="bf16"),
        # Eight prompts of an odd length, some of them shorter and padded in front.
        dict(name="append_prompt_f32", kind="append", **{"pass": "fwd"}, B=8, N=2047, Nk=4096, S=64, Hk=8, D=128, layout=2,
             dtype="f32"),
        # One token of a few short rows: the smallest attention call.
        dict(name="paged_token_short_f32", kind="attn", **{"pass": "fwd"}, B=4, Nq=1, Nk=777, S=16, H=8, Hk=8, D=64,
             cap=0.0, slopes=True, scores=False, shared=0, layout=3, dtype="f32"),
        # The next site of 512 walkers that share their first pages, in float32.
        dict(name="paged_walkers_f32", kind="attn", **{"pass": "fwd"}, B=512, Nq=1, Nk=225, S=16, H=8, Hk=8, D=64,
             cap=0.0, slopes=False, scores=True, shared=2, layout=4, dtype="f32"),
        # One token of each of 16 rows of up to 32768 tokens.
        dict(name="paged_token_long_bf16", kind="attn", **{"pass": "fwd"}, B=16, Nq=1, Nk=32768, S=64, H=32, Hk=8, D=128,
             cap=50.0, slopes=False, scores=False, shared=0, layout=5, dtype="bf16"),
        # Three proposed tokens of one very long row, with the weights of all slots, in pages of an odd size.
        dict(name="paged_few_long_bf16", kind="attn", **{"pass": "fwd"}, B=1, Nq=3, Nk=131072, S=48, H=32, Hk=4, D=128,
             cap=0.0, slopes=False, scores=True, shared=0, layout=6, dtype="bf16"),
        # Ragged rows halved, single slots as pages: the smallest eviction.
        dict(name="evict_short_f32", kind="evict", **{"pass": "fwd"}, B=4, Nk=777, S=1, Hk=8, D=64, budget=300, sinks=4,
             recent=64, layout=7, dtype="f32"),
        # 256 walkers' caches of sites cut to 128 slots.
        dict(name="evict_walkers_f32", kind="evict", **{"pass": "fwd"}, B=256, Nk=225, S=16, Hk=8, D=64, budget=128,
             sinks=1, recent=32, layout=8, dtype="f32"),
        # 16 rows of up to 32768 tokens cut to 8192.
        dict(name="evict_long_bf16", kind="evict", **{"pass": "fwd"}, B=16, Nk=32768, S=64, Hk=8, D=128, budget=8192,
             sinks=4, recent=1024, layout=9, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "attn", "attn", "attn", "evict"])
    dtype = rng.choice(["f32", "bf16"])
    layout = rng.randrange(1 << 20)
    D = rng.choice([16, 32, 64, 80, 128])
    Hk = rng.choice([1, 2, 4, 8])
    if kind == "rotary":
        H = Hk * rng.choice([1, 2, 4])
        N = _log(rng, 1, 8160)
        B = _log(rng, 1, max(1, min(256, 16384 // N)))
        return dict(kind="rotary", **{"pass": rng.choice(["fwd", "train"])}, B=B, N=N, H=H, Hk=Hk, D=D,
                    rot=rng.choice([D, D // 2]), A=rng.choice([1, 2, 2, 3, 3, 4]), norm=rng.random() < 0.5,
                    interleaved=rng.random() < 0.5, mixed=rng.random() < 0.5, dtype=dtype)
    S = rng.choice([1, 16, 16, 48, 64, 64, 100, 256])
    if kind == "append":
        N = _log(rng, 1, 2047)
        B = _log(rng, 1, max(1, min(256, 16384 // N)))
        return dict(kind="append", **{"pass": "fwd"}, B=B, N=N, Nk=N + _log(rng, 1, 2048), S=S, Hk=Hk, D=D, layout=layout,
                    dtype=dtype)
    Nk = _log(rng, 1, 32768)
    if kind == "evict":
        B = _log(rng, 1, min(256, max(1, (1 << 18) // Nk)))
        budget = _log(rng, 1, Nk)
        sinks = rng.choice([0, 1, 4])
        recent = rng.choice([0, budget // 8, budget // 2])
        if sinks + recent > budget:
            sinks = recent = 0
        return dict(kind="evict", **{"pass": "fwd"}, B=B, Nk=Nk, S=S, Hk=Hk, D=D, budget=budget, sinks=sinks, recent=recent,
                    layout=layout, dtype=dtype)
    B = _log(rng, 1, min(512, (1 << 18) // Nk))
    return dict(kind="attn", **{"pass": "fwd"}, B=B, Nq=rng.choice([1, 1, 1, 2, 5]), Nk=Nk, S=S,
                H=Hk * rng.choice([1, 2, 4, 8]), Hk=Hk, D=D, cap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                slopes=rng.random() < 0.3, scores=rng.random() < 0.5, shared=rng.choice([0, 0, 2]), layout=layout,
                dtype=dtype)


# --- what belongs to a case and not to its values -------------------------------------------------------------------

def _lengths(case):
    """Tokens in each row, new ones included; rows are ragged, and of three or more one may be empty."""
    r = random.Random(case["layout"])
    Nk = case["Nk"]
    n = [r.randint((Nk + 3) // 4, Nk) for _ in range(case["B"])]
    if case["kind"] == "append":  # some prompts are shorter than the call's N tokens
        n = [r.randint((case["N"] + 1) // 2, case["N"]) if r.random() < 0.3 else max(x, case["N"]) for x in n]
    elif case["B"] >= 3 and r.random() < 0.25:
        n[r.randrange(case["B"])] = r.randint(0, 1)
    return n


def _width(case):
    return -(-case["Nk"] // case["S"])


def work(case):
    w = BYTES[case["dtype"]]
    if case["kind"] == "rotary":
        n = case["B"] * case["N"] * (case["H"] + case["Hk"]) * case["D"]
        train = case["pass"] == "train"
        passes = (5 if case["norm"] else 4) if train else 2
        return {"bytes": n * w * passes, "flops": n * (7 if case["norm"] else 3) * (3 if train and case["norm"] else 2 if train else 1)}
    token = 2 * case["Hk"] * case["D"] * w  # a token's key and value
    if case["kind"] == "append":
        return {"bytes": 2 * token * sum(min(x, case["N"]) for x in _lengths(case)), "flops": 0}
    if case["kind"] == "evict":
        moved = values = 0.0
        m, fixed = case["budget"], case["sinks"] + case["recent"]
        for n in _lengths(case):
            values += n + min(n, m)
            if n > m:
                late = min(case["recent"], n - m)  # recent tokens behind the budget, and of the others there those that stay
                moved += late + (n - m - late) * (m - fixed) / max(n - fixed, 1)
        cap = case["B"] * _width(case) * case["S"]
        return {"bytes": 2 * token * moved + 4 * case["Hk"] * (values + cap), "flops": 0}
    Nq, H, D = case["Nq"], case["H"], case["D"]
    lengths = _lengths(case)
    pairs = sum(max(0, n - Nq + 1 + i) for n in lengths for i in range(Nq)) * H
    read = sum(lengths)
    if case["shared"]:  # pages that several rows have are read once
        first = case["shared"] * case["S"]
        read -= sum(min(n, first) for n in lengths) - min(max(lengths), first)
    scores = 8 * case["Hk"] * sum(lengths) if case["scores"] else 0
    return {"bytes": 2 * case["B"] * Nq * H * D * w + token * read + scores, "flops": 4 * D * pairs}


# --- inputs ---------------------------------------------------------------------------------------------------------

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = SimpleNamespace(case=case)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=dt) * std

    B, Hk, D = case["B"], case["Hk"], case["D"]
    if case["kind"] == "rotary":
        N, H, A, half = case["N"], case["H"], case["A"], case["rot"] // 2
        # both are slices of one projection's output, as a model holds them
        rows = normal(B, N, H + 2 * Hk, D)
        s.q, s.k = rows[:, :, :H], rows[:, :, H:H + Hk]
        s.freqs = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEVICE) / half)
        # each frequency's axis: in turn, or a run of frequencies for each
        s.axes = (torch.arange(half, device=DEVICE) % A if case["mixed"] else torch.arange(half, device=DEVICE) * A // half).to(torch.int32)
        # tokens in the order of a box, the last axis fastest, behind a text of some length
        side = max(1, math.ceil(N ** (1 / A)))
        i = torch.arange(N, device=DEVICE)
        box = torch.stack([i // side ** (A - 1 - a) % side if a else i // side ** (A - 1) for a in range(A)], -1)
        s.positions = (box + torch.randint(0, 4096, (B, 1, 1), generator=g, device=DEVICE)).to(torch.int32)
        s.wq = s.wk = None
        if case["norm"]:
            s.wq = 1 + 0.2 * torch.randn(D, generator=g, device=DEVICE)
            s.wk = 1 + 0.2 * torch.randn(D, generator=g, device=DEVICE)
        if case["pass"] == "train":
            s.leaves = [x.detach().requires_grad_() for x in (s.q, s.k, s.wq, s.wk) if x is not None]
            s.q, s.k = s.leaves[:2]
            if case["norm"]:
                s.wq, s.wk = s.leaves[2:]
            s.cot = (normal(B, N, H, D), normal(B, N, Hk, D))
        return s
    S, T = case["S"], _width(case)
    pages = B * T + SPARE
    s.k_cache, s.v_cache = normal(pages, S, Hk, D), normal(pages, S, Hk, D)
    s.page_table = torch.randperm(pages, generator=g, device=DEVICE)[:B * T].reshape(B, T).to(torch.int32)
    s.lengths = _ints(_lengths(case))
    if case["kind"] == "append":
        rows = normal(B, case["N"], 3 * Hk, D)
        s.k, s.v = rows[:, :, Hk:2 * Hk], rows[:, :, 2 * Hk:]
        return s
    # weights that slots have had: few have most of them, and some none at all
    had = torch.exp(2 * torch.randn(B, Hk, T * S, generator=g, device=DEVICE))
    had *= torch.rand(B, Hk, T * S, generator=g, device=DEVICE) < 0.9
    s.scores = had * (torch.arange(T * S, device=DEVICE) < s.lengths[:, None, None])
    if case["kind"] == "evict":
        return s
    s.page_table[:, :case["shared"]] = s.page_table[:1, :case["shared"]]
    s.q = normal(B, case["Nq"], case["H"], D, std=3.0)
    s.slopes = None
    if case["slopes"]:
        s.slopes = 2.0 ** (-8.0 * torch.arange(1, case["H"] + 1, dtype=torch.float32, device=DEVICE) / case["H"])
    return s


# --- one pass -------------------------------------------------------------------------------------------------------

def run(s):
    c = s.case
    if not own:
        with torch.no_grad():
            return {"rotary": _plain_rotary, "append": _plain_append, "attn": _plain_attn, "evict": _plain_evict}[c["kind"]](s)
    import hamiltonzero_amd as hz

    if c["kind"] == "rotary":
        if c["norm"]:
            out = hz.qk_norm_rotary(s.q, s.k, s.wq, s.wk, freqs=s.freqs, positions=s.positions, axes=s.axes,
                                    interleaved=c["interleaved"], eps=EPS)
        else:
            out = hz.qk_rotary(s.q, s.k, freqs=s.freqs, positions=s.positions, axes=s.axes, interleaved=c["interleaved"])
        return (*out, *torch.autograd.grad(out, s.leaves, s.cot)) if c["pass"] == "train" else out
    if c["kind"] == "append":
        hz.paged_append(s.k_cache, s.v_cache, s.k, s.v, s.page_table, s.lengths)
        return s.k_cache, s.v_cache
    if c["kind"] == "evict":
        lengths, sources, scores = hz.paged_evict(s.k_cache, s.v_cache, s.page_table, s.lengths, s.scores, c["budget"],
                                                  sinks=c["sinks"], recent=c["recent"])
        return s.k_cache, s.v_cache, lengths, sources, scores
    options = dict(softcap=c["cap"], slopes=s.slopes)
    if c["scores"]:
        return hz.paged_attention(s.q, s.k_cache, s.v_cache, s.page_table, s.lengths, scores=s.scores, decay=0.98, **options)
    return (hz.paged_attention(s.q, s.k_cache, s.v_cache, s.page_table, s.lengths, **options),)


def _turn(x, cos, sin, interleaved):
    """Rotates the pairs of the first 2 * half elements of each head."""
    half = cos.shape[-1]
    r, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :half], r[..., half:])
    a, b = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((r, rest), -1)


def _plain_rotary(s):
    c = s.case
    train = c["pass"] == "train"
    t = (s.positions[:, :, s.axes.long()].double() * s.freqs)[:, :, None]
    cos, sin = t.cos().float(), t.sin().float()

    def one(x, w, dy):
        x = x.float()
        if not c["norm"]:
            y = _turn(x, cos, sin, c["interleaved"])
            return y, _turn(dy.float(), cos, -sin, c["interleaved"]) if train else None, None
        r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        n = x * r
        y = _turn(n * w, cos, sin, c["interleaved"])
        if not train:
            return y, None, None
        d = _turn(dy.float(), cos, -sin, c["interleaved"])
        dw = (d * n).double().sum((0, 1, 2)).float()
        d = d * w
        return y, r * (d - n * (d * n).mean(-1, keepdim=True)), dw

    dq, dk = s.cot if train else (None, None)
    (q, gq, gwq), (k, gk, gwk) = one(s.q, s.wq, dq), one(s.k, s.wk, dk)
    out = [x.to(s.q.dtype) for x in ((q, k, gq, gk) if train else (q, k))]
    return (*out, gwq, gwk) if train and c["norm"] else tuple(out)


def _plain_append(s):
    c = s.case
    slot = s.lengths.long()[:, None] - c["N"] + torch.arange(c["N"], device=DEVICE)
    row, i = torch.nonzero(slot >= 0, as_tuple=True)
    slot = slot[row, i]
    page = s.page_table.long()[row, slot // c["S"]]
    s.k_cache[page, slot % c["S"]] = s.k[row, i]
    s.v_cache[page, slot % c["S"]] = s.v[row, i]
    return s.k_cache, s.v_cache


def _plain_attn(s):
    c = s.case
    B, Nq, H, Hk, D = (c[n] for n in ("B", "Nq", "H", "Hk", "D"))
    G = H // Hk
    rows = lambda cache: cache[s.page_table.long()].float().reshape(B, -1, Hk, D).transpose(1, 2)  # noqa: E731
    k = rows(s.k_cache)
    n = k.shape[2]
    q = s.q.float().reshape(B, Nq, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Nq, D)
    x = (q @ k.transpose(-1, -2)).reshape(B, Hk, G, Nq, n) * D ** -0.5
    del k
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    j = torch.arange(n, device=DEVICE)
    p = s.lengths.long()[:, None] - Nq + torch.arange(Nq, device=DEVICE)  # [B, Nq]
    if s.slopes is not None:
        x = x - s.slopes.reshape(Hk, G, 1, 1) * (p[:, None, None, :, None] - j).abs()
    x = torch.where((j <= p[:, :, None])[:, None, None], x, -math.inf)
    m = x.amax(-1, keepdim=True)
    w = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    z = w.sum(-1, keepdim=True)
    w = w / torch.where(z == 0, 1.0, z)
    v = rows(s.v_cache)
    v = torch.where((j < s.lengths[:, None])[:, None, :, None], v, 0.0)
    out = (w.reshape(B, Hk, G * Nq, n) @ v).reshape(B, Hk, G, Nq, D).permute(0, 3, 1, 2, 4).reshape(B, Nq, H, D).to(s.q.dtype)
    if not c["scores"]:
        return (out,)
    new = 0.98 * s.scores + w.sum((2, 3))
    return out, torch.where(j < s.lengths[:, None, None], new, 0.0)


def _plain_evict(s):
    c = s.case
    m = c["budget"]
    B, Hk, cap = s.scores.shape
    n = s.lengths.long()[:, None, None]
    j = torch.arange(cap, device=DEVICE)
    inside = j < n
    fixed = inside & ((j < c["sinks"]) | (j >= n - c["recent"]))
    # the largest first, the lowest slot first among equals
    rank = torch.where(fixed, math.inf, torch.where(inside, s.scores, -math.inf))
    order = rank.argsort(dim=-1, descending=True, stable=True)
    place = torch.empty_like(order).scatter_(-1, order, j.expand(B, Hk, cap))
    stays = inside & (place < m)
    hole, late = (j < m) & inside & ~stays, (j >= m) & stays
    # the k-th late survivor goes into the k-th hole, where its row is longer than the budget
    holes, lates = torch.nonzero(hole), torch.nonzero(late)
    src = torch.where(stays & (j < m), j, -1)
    src[holes[:, 0], holes[:, 1], holes[:, 2]] = lates[:, 2]
    b, h, to, at = holes[:, 0], holes[:, 1], holes[:, 2], lates[:, 2]
    page = lambda slot: s.page_table.long()[b, slot // c["S"]]  # noqa: E731
    for cache in (s.k_cache, s.v_cache):
        cache[page(to), to % c["S"], h] = cache[page(at), at % c["S"], h]
    scores = torch.where(src >= 0, s.scores.gather(-1, src.clamp(min=0)), 0.0)
    return s.k_cache, s.v_cache, s.lengths.clamp(max=m), src[..., :min(m, cap)].to(torch.int32), scores


# --- the same in 64 bits, from the definitions ----------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "append": _exact_append, "attn": _exact_attn, "evict": _exact_evict}[case["kind"]](s)


def _exact_rotary(s):
    c = s.case
    train = c["pass"] == "train"
    half = s.freqs.numel()
    at = torch.arange(half, device=DEVICE)
    ia, ib = (2 * at, 2 * at + 1) if c["interleaved"] else (at, at + half)
    angle = torch.zeros(c["B"], c["N"], 1, half, dtype=torch.float64, device=DEVICE)
    for a in range(c["A"]):
        angle += torch.where(s.axes == a, s.freqs * s.positions[:, :, a, None].double(), 0.0)[:, :, None]
    z = torch.polar(torch.ones_like(angle), angle)  # a rotation is a product of complex numbers
    leaves, outs = [], []
    for x, w in ((s.q, s.wq), (s.k, s.wk)):
        y = x = x.detach().double().requires_grad_(train)
        leaves.append(x)
        if c["norm"]:
            w = w.detach().double().requires_grad_(train)
            leaves.append(w)
            y = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / c["D"] + EPS) * w
        turned = torch.complex(y[..., ia], y[..., ib]) * z
        outs.append(y.index_copy(-1, ia, turned.real).index_copy(-1, ib, turned.imag))
    if not train:
        return tuple(outs)
    grads = torch.autograd.grad(outs, leaves, [x.double() for x in s.cot])
    return (*(o.detach() for o in outs), *grads[::2], *grads[1::2]) if c["norm"] else (*(o.detach() for o in outs), *grads)


def _exact_append(s):
    c = s.case
    caches = s.k_cache.double(), s.v_cache.double()
    table, lengths = s.page_table.tolist(), s.lengths.tolist()
    for b, n in enumerate(lengths):
        first, t = n - c["N"], max(0, n - c["N"])
        while t < n:  # a page's tokens at a time
            end = min(n, (t // c["S"] + 1) * c["S"])
            for cache, new in zip(caches, (s.k, s.v)):
                cache[table[b][t // c["S"]], t % c["S"]:t % c["S"] + end - t] = new[b, t - first:end - first].double()
            t = end
    return caches


def _exact_attn(s):
    c = s.case
    Nq, H, Hk, D, S = (c[n] for n in ("Nq", "H", "Hk", "D", "S"))
    G = H // Hk
    out = torch.zeros(c["B"], Nq, H, D, dtype=torch.float64, device=DEVICE)
    had = torch.zeros(s.scores.shape, dtype=torch.float64, device=DEVICE)
    at = torch.arange(Nq, device=DEVICE)
    for b, n in enumerate(s.lengths.tolist()):
        if n == 0:
            continue
        pages = s.page_table[b, :-(-n // S)].long()
        k, v = (cache[pages].flatten(0, 1)[:n].double() for cache in (s.k_cache, s.v_cache))
        j = torch.arange(n, device=DEVICE)
        away = (n - Nq + at)[:, None] - j  # how far a query is behind a key
        some = (away >= 0).any(1, keepdim=True)
        for h in range(Hk):
            y = torch.einsum("igd,nd->gin", s.q[b, :, h * G:(h + 1) * G].double(), k[:, h]) / math.sqrt(D)
            if c["cap"]:
                y = torch.tanh(y / c["cap"]) * c["cap"]
            if s.slopes is not None:
                y = y - s.slopes[h * G:(h + 1) * G, None, None].double() * away.abs()
            # a row that sees nothing is computed over all keys and then left out
            w = torch.softmax(y.masked_fill((away < 0) & some, -math.inf), -1).masked_fill(~some, 0.0)
            out[b, :, h * G:(h + 1) * G] = torch.einsum("gin,nd->igd", w, v[:, h])
            had[b, h, :n] = s.scores[b, h, :n].double() * 0.98 + w.sum((0, 1))
    return (out, had) if c["scores"] else (out,)


def _exact_evict(s):
    c = s.case
    m, S = c["budget"], c["S"]
    caches = s.k_cache.double(), s.v_cache.double()
    had = torch.zeros(s.scores.shape, dtype=torch.float64)
    old = s.scores.double().cpu()
    for b, n in enumerate(s.lengths.tolist()):
        pages = s.page_table[b].long()
        for h in range(c["Hk"]):
            if n <= m:
                had[b, h, :n] = old[b, h, :n]
                continue
            free = old[b, h, c["sinks"]:n - c["recent"]]
            # sorted from the last slot on, ascending: of equal ones the lowest slot comes last and stays
            by_weight = free.numel() - 1 - free.flip(0).sort(stable=True).indices
            keep = torch.zeros(n, dtype=torch.bool)
            keep[:c["sinks"]] = True
            keep[n - c["recent"]:] = True
            keep[c["sinks"] + by_weight[free.numel() - (m - c["sinks"] - c["recent"]):]] = True
            late = m + torch.nonzero(keep[m:])[:, 0]
            to = torch.nonzero(~keep[:m])[:, 0]
            had[b, h, :m] = torch.where(keep[:m], old[b, h, :m], 0.0)
            had[b, h, to] = old[b, h, late]
            late, to = late.to(DEVICE), to.to(DEVICE)
            for cache in caches:
                cache[pages[to // S], to % S, h] = cache[pages[late // S], late % S, h]
    return (*caches, None, None, had.to(DEVICE))

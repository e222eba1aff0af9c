"""The weights of paged attention. Those that it adds up are a softmax's at any size of the scores: those of a query sum to one, to float32's
roundings, and one number that all of them share (a logarithm of the sum, rounded at the size of the scores) would show. Those that meet the values
are rounded to 2^-16 and less: an output is rounded once. The same call gives the same bits."""

import numpy as np
import pytest
import torch

import hamiltonzero_amd as hz
from oracle import paged_oracle as P
from oracle.token_oracle import F, _sum_error

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def arr(t):
    return t.detach().double().cpu().numpy()


# Heads with one query each, so that a head's weights are one softmax; wide tables are divided, others not; B 600 has a wave a row.
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1.0, 100.0, 3000.0])
@pytest.mark.parametrize("B,n,S,T", [(2, 300, 16, 20), (2, 300, 10, 30), (2, 2500, 16, 160), (2, 2500, 10, 260), (1, 60, 4, 500), (300, 70, 16, 5)],
                         ids=lambda x: str(x))
def test_weights_of_a_query_sum_to_one(B, n, S, T, size, dtype):
    print(f"[case] weights {B} {n} {S} {T} {size} {dtype}", flush=True)
    H, D = 8, 64
    g = torch.Generator(device="cuda").manual_seed(51)
    # keys near one another: scores of about size, with a spread of a few around it
    base = torch.randn(D, generator=g, device="cuda")
    q = base.expand(B, 1, H, D) + 0.1 * torch.randn(B, 1, H, D, generator=g, device="cuda")
    k = size * base / 8 + 0.3 * torch.randn(B * T, S, H, D, generator=g, device="cuda")
    q, k = q.to(DT[dtype]).contiguous(), k.to(DT[dtype])
    v = torch.randn(B * T, S, H, D, generator=g, device="cuda").to(DT[dtype])
    table = torch.randperm(B * T, generator=torch.Generator().manual_seed(5)).reshape(B, T).to(torch.int32)
    lengths = [n - b % 7 for b in range(B)]
    scores = torch.zeros(B, H, T * S, device="cuda")
    _, new = hz.paged_attention(q, k, v, table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), scores=scores)
    w = arr(new)
    # Each weight: the difference to the largest score and the power of two (8 F of their size, 2 F each and rounded up), the reciprocal of the
    # sum and the product; the sum itself as the outputs'; joins 24 F. What an exponential's error at a distance d weighs is w d.
    with np.errstate(divide="ignore"):
        far = np.where(w > 0, -np.log(np.where(w > 0, w, 1)), 0)
    bound = _sum_error(n) + 24 * F + 8 * F * ((w * far).sum(2) + 2)
    off = np.abs(w.sum(2) - 1)
    print(f"  sums: {(off / bound).max():.3f} of their bound", flush=True)
    assert (off <= bound).all(), (off.max(), bound.min())
    assert w.max() <= 1


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("slots", [70, 3000])
def test_equal_scores_of_any_size_weigh_the_same(slots, dtype):
    """Equal keys: each weight is 1 / n, whatever the score (difference to the largest 0, its power of two 1, sums of ones exact)."""
    D, S, H = 32, 16, 4
    T = -(-slots // S)
    for size in (0.0, 3.0, 1e4, -1e6, 1e12):
        q = torch.full((1, 1, H, D), 1.0, device="cuda", dtype=DT[dtype])
        k = torch.full((T, S, H, D), size / D, device="cuda", dtype=DT[dtype])
        n = torch.tensor([slots], dtype=torch.int32, device="cuda")
        table = torch.arange(T, dtype=torch.int32, device="cuda")[None]
        _, new = hz.paged_attention(q, k, k.clone(), table, n, scale=1.0, scores=torch.zeros(1, H, T * S, device="cuda"))
        # the reciprocal's rounding and the product's
        assert (np.abs(arr(new)[:, :, :slots] * slots - 1) <= 4 * F).all(), (size, arr(new)[0, 0, 0] * slots - 1)
        assert (new[:, :, slots:] == 0).all()


def test_weights_against_the_oracle_at_large_scores():
    """Element by element; the oracle's bound has no term that grows with the largest score beside the products' own."""
    for S, n in ((16, [300, 17]), (10, [2300, 1])):
        g = torch.Generator(device="cuda").manual_seed(52)
        T = -(-max(n) // S) + 40
        k = torch.randn(2 * T, S, 2, 64, generator=g, device="cuda") * 4
        v = torch.randn(2 * T, S, 2, 64, generator=g, device="cuda")
        table = torch.arange(2 * T, dtype=torch.int32).reshape(2, T)
        q = torch.randn(2, 2, 6, 64, generator=g, device="cuda") * 30
        scores = torch.zeros(2, 2, T * S, device="cuda")
        _, new = hz.paged_attention(q, k, v, table.cuda(), torch.tensor(n, dtype=torch.int32, device="cuda"), scores=scores)
        want = P.attention(arr(q), arr(k), arr(v), table.numpy(), n, scale=64**-0.5, scores=arr(scores))
        assert (np.abs(arr(new) - want["scores"]) <= want["t_scores"]).all()


@pytest.mark.parametrize("o", [dict(), dict(softcap=20.0), dict(slopes=True)], ids=["plain", "cap", "slopes"])
@pytest.mark.parametrize("B,Nq,H,Hk,D,S,n", [(2, 1, 8, 2, 64, 16, 300), (3, 3, 16, 2, 128, 48, 4000), (1, 5, 8, 1, 32, 10, 2000), (2, 1, 4, 4, 80, 100, 90), (1, 50, 2, 2, 16, 16, 700)],
                         ids=lambda x: str(x))
def test_bfloat16_outputs_are_rounded_once(B, Nq, H, Hk, D, S, n, o):
    """bfloat16's own half step of the result, and 2^-16 (one for a weight's upper part and the rest of it, rounded) of the weights."""
    print(f"[case] once {B} {Nq} {H} {Hk} {D} {S} {n} {o}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(53)
    T = -(-n // S)
    k, v = (torch.randn(B * T, S, Hk, D, generator=g, device="cuda").bfloat16() for _ in range(2))
    q = (torch.randn(B, Nq, H, D, generator=g, device="cuda") * 2).bfloat16()
    table = torch.randperm(B * T, generator=torch.Generator().manual_seed(6)).reshape(B, T).to(torch.int32)
    lengths = [n - 3 * b for b in range(B)]
    kw = dict(o)
    if o.get("slopes"):
        kw["slopes"] = torch.rand(H, generator=g, device="cuda") * 0.1
    out = hz.paged_attention(q, k, v, table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), **kw)
    if o.get("slopes"):
        kw["slopes"] = arr(kw["slopes"])
    want = P.attention(arr(q), arr(k), arr(v), table.numpy(), lengths, scale=D**-0.5, bf16=True, up=2.0**-16, **kw)
    off = np.abs(arr(out) - want["out"])
    print(f"  out: {(off / np.maximum(want['t_out'], 1e-300)).max():.3f} of its bound", flush=True)
    assert (off <= want["t_out"]).all(), ((off > want["t_out"]).mean(), (off / np.maximum(want["t_out"], 1e-300)).max())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,Nq,H,Hk,D,S,n", [(4, 1, 32, 8, 128, 64, 9000), (1, 3, 32, 4, 128, 48, 30000), (70, 2, 8, 8, 64, 10, 1500), (300, 1, 8, 8, 64, 16, 200)],
                         ids=lambda x: str(x))
def test_the_same_call_gives_the_same_bits(B, Nq, H, Hk, D, S, n, dtype):
    """Again, and again with other calls between them that use the same memory for their workspaces."""
    print(f"[case] again {B} {Nq} {H} {Hk} {D} {S} {n} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(54)
    T = -(-n // S)
    k, v = (torch.randn(B * T, S, Hk, D, generator=g, device="cuda").to(DT[dtype]) for _ in range(2))
    q = torch.randn(B, Nq, H, D, generator=g, device="cuda").to(DT[dtype])
    table = torch.randperm(B * T, generator=g, device="cuda").reshape(B, T).to(torch.int32)
    lengths = torch.randint(n // 3, n + 1, (B,), generator=g, device="cuda").to(torch.int32)
    scores = torch.rand(B, Hk, T * S, generator=g, device="cuda")
    first = hz.paged_attention(q, k, v, table, lengths, scores=scores)
    for turn in range(4):
        if turn % 2:
            hz.paged_attention(-q, v, k, table, lengths // 2, scores=scores)
        again = hz.paged_attention(q, k, v, table, lengths, scores=scores)
        assert all(torch.equal(a, b) for a, b in zip(first, again)), turn

"""GPU parity of paged attention where 5 to 64 rows are divided into runs: every wave then works the division out for itself, a row a lane, and
all of its lanes' rows count. Element by element within the oracle's bounds."""

import numpy as np
import pytest
import torch

import hamiltonzero_amd as hz
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def arr(t):
    return t.detach().double().cpu().numpy()


def within(name, got, want, bound):
    off = np.abs(arr(got) - want)
    worst = float(np.max(off / np.maximum(bound, 1e-300)))
    print(f"  {name}: {worst:.3f} of its bound", flush=True)
    assert (off <= bound).all(), (name, worst, np.argwhere(~(off <= bound))[:4].tolist())


def ragged(B, last):
    """Lengths of every kind, the longest in the lanes that a few active ones would not reach; some rows empty or of one slot."""
    r = np.random.default_rng(B)
    n = r.integers(0, 2600, B)
    n[::5] = r.integers(0, 2, len(n[::5]))
    n[B - 1] = last
    return n.tolist()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("Nq,H,Hk", [(1, 1, 1), (1, 2, 1), (2, 2, 2), (1, 16, 2), (3, 4, 1)], ids=lambda x: str(x))
@pytest.mark.parametrize("B", [5, 9, 17, 33, 64])
def test_rows_divided_by_every_wave(B, Nq, H, Hk, dtype):
    print(f"[case] divided {B} {Nq} {H} {Hk} {dtype}", flush=True)
    D, S, slots = 32, 48 if B % 2 else 10, 2900
    T = -(-slots // S)
    g = torch.Generator(device="cuda").manual_seed(41)
    normal = lambda *shape, std=1.0: (torch.randn(*shape, generator=g, device="cuda") * std).to(DT[dtype])  # noqa: E731
    k, v = normal(B * T, S, Hk, D), normal(B * T, S, Hk, D)
    table = torch.randperm(B * T, generator=torch.Generator().manual_seed(B)).reshape(B, T).to(torch.int32)
    lengths = ragged(B, 2600)
    n, q = torch.tensor(lengths, dtype=torch.int32, device="cuda"), normal(B, Nq, H, D, std=2.0)
    scores = torch.rand(B, Hk, T * S, generator=g, device="cuda")
    want = P.attention(arr(q), arr(k), arr(v), table.numpy(), lengths, scale=D**-0.5, scores=arr(scores), decay=0.75, bf16=dtype == "bf16")
    table = table.cuda()
    out, new = hz.paged_attention(q, k, v, table, n, scores=scores, decay=0.75)
    within("out", out, want["out"], want["t_out"])
    within("scores", new, want["scores"], want["t_scores"])
    assert torch.equal(hz.paged_attention(q, k, v, table, n), out)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("how", ["groups", "every second", "all", "last rows", "padding"])
@pytest.mark.parametrize("S", [64, 48, 10, 1])
def test_shared_pages_in_pools_of_any_size(S, how, dtype):
    """Whichever pages rows share, and however large the pool: the bits that rows with pages of their own give."""
    print(f"[case] shared {S} {how} {dtype}", flush=True)
    B, H, Hk, D, slots = 9, 4, 2, 64, 2000
    T = -(-slots // S)
    g = torch.Generator(device="cuda").manual_seed(42)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda").to(DT[dtype])  # noqa: E731
    pages = 3 * T + 5  # fewer than all tables have
    k, v = normal(pages, S, Hk, D), normal(pages, S, Hk, D)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(S)).to(torch.int32)
    own = [order[i * T:(i + 1) * T] for i in range(3)]
    first = {"groups": [0, 0, 0, 1, 1, 1, 2, 2, 2], "every second": [0, 1, 2] * 3, "all": [0] * 9, "last rows": [0, 1, 2, 0, 1, 2, 0, 0, 0], "padding": [0, 1, 2] * 3}[how]
    table = torch.stack([own[i] for i in first])
    lengths = [2000, 1999, 1000, 1700, 1, 1500, 0, 1300, 1800]
    if how == "padding":  # behind the lengths: no page, the same one for all, numbers out of range
        for b, n in enumerate(lengths):
            table[b, -(-n // S):] = [-1, 0, 2**31 - 1][b % 3]
    q, n = normal(B, 1, H, D), torch.tensor(lengths, dtype=torch.int32, device="cuda")
    scores = torch.rand(B, Hk, T * S, generator=g, device="cuda")
    got = hz.paged_attention(q, k, v, table.cuda(), n, scores=scores)
    at = table.long().clamp(0, pages - 1).flatten().cuda()
    apart = torch.arange(B * T, dtype=torch.int32, device="cuda").reshape(B, T)
    want = hz.paged_attention(q, k[at].contiguous(), v[at].contiguous(), apart, n, scores=scores)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(hz.paged_attention(q, k, v, table.cuda(), n), got[0])

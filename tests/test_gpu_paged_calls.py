"""Calls of the paged operators for what they do besides their numbers: refusals of the entry points, other streams and threads,
captured graphs whose rows grow, what is left alone; and all of them together, a cache that is filled, read and cut token by token."""

import threading

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwd

import hamiltonzero_amd as hz
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu
F = 2.0**-24
ANGLE = 2.0**-21
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def arr(t):
    return t.detach().double().cpu().numpy()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def ints(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def filled(g, B=3, T=4, S=16, Hk=2, D=32, dtype=torch.float32, lengths=(40, 17, 64)):
    k, v = normal(g, B * T, S, Hk, D, dtype=dtype), normal(g, B * T, S, Hk, D, dtype=dtype)
    table = torch.randperm(B * T, generator=g, device="cuda").reshape(B, T).to(torch.int32)
    return k, v, table, ints(lengths)


# --- refusals ---------------------------------------------------------------------------------------


def test_entry_points_refuse():
    g = gen(1)
    k, v, table, n = filled(g)
    q, new = normal(g, 3, 1, 4, 32), normal(g, 3, 2, 2, 32)
    scores = torch.zeros(3, 2, 64, device="cuda")
    attend = lambda **o: hz.paged_attention(**{**dict(q=q, k_cache=k, v_cache=v, page_table=table, lengths=n), **o})  # noqa: E731
    append = lambda **o: hz.paged_append(**{**dict(k_cache=k, v_cache=v, k=new, v=new, page_table=table, lengths=n), **o})  # noqa: E731
    evict = lambda **o: hz.paged_evict(**{**dict(k_cache=k, v_cache=v, page_table=table, lengths=n, scores=scores, budget=8), **o})  # noqa: E731
    shared = [  # of all three: caches and tables
        (dict(k_cache=k.half()), TypeError, "float32 or bfloat16"), (dict(v_cache=v.bfloat16()), TypeError, "v_cache.dtype"),
        (dict(v_cache=v[:3]), ValueError, "v_cache must have shape"), (dict(v_cache=v.cpu()), ValueError, "v_cache is on"),
        (dict(k_cache=k[:0], v_cache=v[:0]), ValueError, "at least 1 long"), (dict(k_cache=k[0], v_cache=v[0]), ValueError, "pages, page_size"),
        (dict(k_cache=k[..., :20], v_cache=v[..., :20]), ValueError, "multiple of 8"),
        (dict(k_cache=k.transpose(2, 3), v_cache=v.transpose(2, 3)), ValueError, "head dimension|contiguous heads|shape"),
        (dict(page_table=table.long()), TypeError, "page_table.dtype"), (dict(page_table=table[0]), ValueError, r"\[B, width\]"),
        (dict(page_table=table[:, :0]), ValueError, "at least 1 long"), (dict(page_table=table.T), ValueError, "lengths must have shape"),
        (dict(page_table=table[:, ::2]), ValueError, "contiguous"), (dict(page_table=table.cpu()), ValueError, "page_table is on"),
        (dict(lengths=n.float()), TypeError, "lengths.dtype"), (dict(lengths=n[:2]), ValueError, "lengths must have shape"),
        (dict(lengths=[1, 2, 3]), TypeError, "lengths must be a tensor"), (dict(lengths=ints([1, 2, 3, 4, 5, 6])[::2]), ValueError, "contiguous"),
    ]
    for call in (attend, append, evict):
        for over, error, text in shared:
            with pytest.raises(error, match=text):
                call(**over)
        flat = torch.zeros(4 + 12 * 16 * 64, device="cuda")[4:].reshape(12, 16, 2, 32)[:, :, :, :]  # 16 bytes on: taken
        call(k_cache=flat)
        odd = torch.zeros(2 + 12 * 16 * 64, device="cuda")[2:].reshape(12, 16, 2, 32)
        with pytest.raises(ValueError, match="16-byte aligned"):
            call(k_cache=odd)
        steps = torch.zeros(12, 16, 2, 33, device="cuda")[..., :32]
        with pytest.raises(ValueError, match="16-byte aligned"):
            call(k_cache=steps)
    for over, error, text in (
        (dict(q=q[:2]), ValueError, "q must have shape"), (dict(q=q.bfloat16()), TypeError, "q.dtype"), (dict(q=normal(g, 3, 1, 3, 32)), ValueError, "multiple of the key heads"),
        (dict(q=q[:, :0]), ValueError, "at least 1 long"), (dict(slopes=torch.ones(3, device="cuda")), ValueError, "slopes must have shape"),
        (dict(scores=scores[:, :, :60]), ValueError, "scores must have shape"), (dict(scores=scores.double()), TypeError, "scores.dtype"),
        (dict(scores_out=scores), ValueError, "scores_out needs scores"), (dict(scores=scores, scores_out=scores[:, :1]), ValueError, "scores_out must have shape"),
        (dict(scores=scores, scores_out=torch.zeros(3, 2, 128, device="cuda")[:, :, ::2]), ValueError, "contiguous"),
    ):
        with pytest.raises(error, match=text):
            attend(**over)
    twice = torch.zeros(3 * 2 * 64 + 4, device="cuda")
    with pytest.raises(ValueError, match="not overlap"):
        attend(scores=twice[4:].reshape(3, 2, 64), scores_out=twice[:-4].reshape(3, 2, 64))
    with pytest.raises(hz.tokens._native.HzError, match="scale"):
        attend(scale=float("nan"))
    with pytest.raises(hz.tokens._native.HzError, match="softcap"):
        attend(softcap=-1.0)
    with pytest.raises(hz.tokens._native.HzError, match="decay"):
        attend(scores=scores, decay=1e39)
    for over, error, text in (
        (dict(k=new[:2]), ValueError, "k must have shape"), (dict(v=new[:, :1]), ValueError, "v must have shape"), (dict(k=new.bfloat16()), TypeError, "k.dtype"),
        (dict(k=new[:, :0], v=new[:, :0]), ValueError, "at least 1 long"),
        (dict(k=k[:6].reshape(3, 32, 2, 32)[:, :2]), ValueError, "must not overlap the caches"),
        (dict(v_cache=k), ValueError, "must not overlap"), (dict(k_cache=k[:1].expand(12, 16, 2, 32)), ValueError, "several places"),
    ):
        with pytest.raises(error, match=text):
            append(**over)
    for over, error, text in (
        (dict(budget=0), ValueError, "budget"), (dict(budget=1 << 30), ValueError, "budget"), (dict(budget=8.0), TypeError, "budget"), (dict(budget=True), TypeError, "budget"),
        (dict(sinks=-1), ValueError, "negative"), (dict(sinks=5, recent=4), ValueError, "budget together"), (dict(recent=None), TypeError, "recent"),
        (dict(scores=scores[:, :1]), ValueError, "scores must have shape"), (dict(v_cache=k), ValueError, "must not overlap"),
        (dict(v_cache=v[:1].expand(12, 16, 2, 32)), ValueError, "several places"),
    ):
        with pytest.raises(error, match=text):
            evict(**over)
    torch.cuda.synchronize()


def test_no_gradients_and_no_tangents():
    g = gen(2)
    k, v, table, n = filled(g)
    q, scores = normal(g, 3, 1, 4, 32), torch.zeros(3, 2, 64, device="cuda")
    leaf = q.clone().requires_grad_()
    with pytest.raises(ValueError, match="no gradients"):
        hz.paged_attention(leaf, k, v, table, n)
    with pytest.raises(ValueError, match="no gradients"):
        hz.paged_attention(q, k.clone().requires_grad_(), v, table, n)
    with pytest.raises(ValueError, match="no gradients"):
        hz.paged_append(k, v, leaf[:, :, :2], q[:, :, :2], table, n)
    with pytest.raises(ValueError, match="no gradients"):
        hz.paged_evict(k, v, table, n, scores.requires_grad_(), 8)
    with torch.no_grad():
        want = hz.paged_attention(q, k, v, table, n)
        assert torch.equal(hz.paged_attention(leaf, k, v, table, n), want)
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="forward mode"):
            hz.paged_attention(fwd.make_dual(q, q), k, v, table, n)
        with pytest.raises(NotImplementedError, match="forward mode"):
            hz.qk_rotary(fwd.make_dual(q, q), q, freqs=torch.ones(16, dtype=torch.float64, device="cuda"))
    with torch.inference_mode():
        k2, v2 = k.clone(), v.clone()
        assert torch.equal(hz.paged_attention(q, k2, v2, table, n), want)
        hz.paged_append(k2, v2, q[:, :, :2], q[:, :, 2:], table, n)
        hz.paged_evict(k2, v2, table, n, scores.detach(), 8)
        out = torch.empty_like(q), torch.empty_like(q)
        hz.qk_rotary(q, q, freqs=torch.ones(16, dtype=torch.float64, device="cuda"), out=out)


def test_rotation_refuses():
    x = torch.zeros(2, 3, 4, 32, device="cuda")
    freqs = torch.ones(16, dtype=torch.float64, device="cuda")
    pos, axes = torch.zeros(2, 3, 2, dtype=torch.int32, device="cuda"), torch.zeros(16, dtype=torch.int32, device="cuda")
    for call in (hz.qk_rotary, hz.qk_norm_rotary):
        good = dict(freqs=freqs, positions=pos, axes=axes)
        call(x, x, **good)
        for over, error, text in (
            (dict(positions=None), ValueError, "axes needs"), (dict(positions=pos[:, :, 0]), ValueError, "n_axes"), (dict(positions=pos.long()), TypeError, "positions.dtype"),
            (dict(positions=pos[:, :2]), ValueError, "positions must have shape"), (dict(positions=pos.expand(2, 3, 2).repeat(1, 1, 9)), ValueError, "n_axes"),
            (dict(positions=pos[:, :, :0]), ValueError, "n_axes"), (dict(axes=axes[:8]), ValueError, "axes must have shape"), (dict(axes=axes.long()), TypeError, "axes.dtype"),
            (dict(axes=None), ValueError, "positions must have shape"), (dict(freqs=freqs[:6]), ValueError, "multiple of 4"), (dict(freqs=freqs.float()), TypeError, "freqs.dtype"),
            (dict(freqs=freqs.repeat(2)), ValueError, "D / 2"), (dict(freqs=freqs.clone().requires_grad_()), ValueError, "detach"),
            (dict(out=(x, torch.empty_like(x))), ValueError, "overlap"),
        ):
            with pytest.raises(error, match=text):
                call(x, x, **{**good, **over})
    with pytest.raises(ValueError, match="no_grad"):
        hz.qk_rotary(x.clone().requires_grad_(), x, freqs=freqs, out=(torch.empty_like(x), torch.empty_like(x)))


# --- streams, threads, graphs -------------------------------------------------------------------------


def test_other_streams_and_threads():
    g = gen(3)
    cases = []
    for i, (lengths, S) in enumerate((((40, 17, 64), 16), ((30, 1, 28), 7), ((64, 64, 64), 16))):
        k, v, table, n = filled(g, S=S, lengths=lengths, dtype=torch.bfloat16 if i else torch.float32)
        q = normal(g, 3, 2, 8, 32, dtype=k.dtype)
        scores = torch.rand(3, 2, 4 * S, generator=g, device="cuda")
        want = hz.paged_attention(q, k, v, table, n, scores=scores)
        kk, vv = k.clone(), v.clone()
        cut = hz.paged_evict(kk, vv, table, n, scores, 9, sinks=1)
        cases.append((k, v, table, n, q, scores, want, kk, vv, cut))
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            k, v, table, n, q, scores, want, kk, vv, cut = cases[i]
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream), torch.no_grad():
                for _ in range(20):
                    got = hz.paged_attention(q, k, v, table, n, scores=scores)
                    k2, v2 = k.clone(), v.clone()
                    again = hz.paged_evict(k2, v2, table, n, scores, 9, sinks=1)
            stream.synchronize()
            same = [*zip(got, want), *zip(again, cut), (k2, kk), (v2, vv)]
            assert all(torch.equal(a, b) for a, b in same)
        except BaseException as e:  # noqa: BLE001
            failed.append((i, e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed, failed


def decode_step(s):
    """One token of every row: rotate, append, attend, add up the weights."""
    q, k = hz.qk_rotary(s["q"], s["k"], freqs=s["freqs"], positions=s["pos"], axes=s["axes"])
    hz.paged_append(s["kc"], s["vc"], k, s["v"], s["table"], s["n"])
    return hz.paged_attention(q, s["kc"], s["vc"], s["table"], s["n"], scores=s["scores"], decay=0.9, scores_out=s["scores"])[0]


def new_state(g, dt, B, T, S, H, Hk, D):
    kc, vc = normal(g, B * T, S, Hk, D, dtype=dt), normal(g, B * T, S, Hk, D, dtype=dt)
    table = torch.randperm(B * T, generator=g, device="cuda").reshape(B, T).to(torch.int32)
    s = dict(kc=kc, vc=vc, table=table, n=torch.zeros(B, dtype=torch.int32, device="cuda"), scores=torch.zeros(B, Hk, T * S, device="cuda"),
             freqs=10.0 ** (-torch.arange(D // 2, dtype=torch.float64, device="cuda") / 8), axes=(torch.arange(D // 2, device="cuda") % 2).to(torch.int32))
    s.update(q=torch.empty(B, 1, H, D, dtype=dt, device="cuda"), k=torch.empty(B, 1, Hk, D, dtype=dt, device="cuda"),
             v=torch.empty(B, 1, Hk, D, dtype=dt, device="cuda"), pos=torch.zeros(B, 1, 2, dtype=torch.int32, device="cuda"))
    return s


def feed(s, g, i, side=5):
    for name in ("q", "k", "v"):
        s[name].copy_(torch.randn(s[name].shape, generator=g, device="cuda"))
    s["pos"][:, :, 0], s["pos"][:, :, 1] = i // side, i % side


@pytest.mark.parametrize("B,T", [(3, 7), (70, 7), (3, 30), (70, 30)])
def test_captured_steps_follow_rows_that_grow(B, T):
    """Two graphs of the same step with a pool of their own, replayed in turn with eager steps between; rows grow through the replays, so the
    division of the rows changes under the captured launches. Every step against an eager twin."""
    dims = dict(B=B, T=T, S=48, H=4, Hk=2, D=64)
    eager, graphed = (new_state(gen(4), torch.bfloat16, **dims) for _ in range(2))
    warm = torch.cuda.Stream()
    with torch.cuda.stream(warm), torch.no_grad():
        graphed["n"].fill_(1)
        decode_step(graphed)
    warm.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.graph(graph):
            outs.append(decode_step(graphed))
        graphs.append(graph)
    fresh = new_state(gen(4), torch.bfloat16, **dims)  # what the captures wrote, back to the start
    for name in ("kc", "vc", "scores", "n"):
        graphed[name].copy_(fresh[name])
    a, b = gen(5), gen(5)
    for i in range(40):
        feed(eager, a, i), feed(graphed, b, i)
        jump = 1 if i % 5 else 37 if T == 7 else 200  # many slots at once: what they hold is the pool's numbers
        for s in (eager, graphed):
            s["n"].add_(jump).clamp_(max=T * 48)
        with torch.no_grad():
            want = decode_step(eager)
        if i % 7 == 3:
            with torch.no_grad():
                got = decode_step(graphed)
        else:
            graphs[i % 2].replay()
            got = outs[i % 2]
        torch.cuda.synchronize()
        assert torch.equal(got, want), i
        for name in ("kc", "vc", "scores"):
            assert torch.equal(eager[name], graphed[name]), (i, name)


def test_captured_rotation_and_its_gradient():
    g = gen(6)
    freqs = torch.rand(16, generator=g, dtype=torch.float64, device="cuda")
    pos, axes = torch.zeros(2, 9, 3, dtype=torch.int32, device="cuda"), (torch.arange(16, device="cuda") % 3).to(torch.int32)
    q, k = normal(g, 2, 9, 4, 64).requires_grad_(), normal(g, 2, 9, 2, 64).requires_grad_()
    cot = normal(g, 2, 9, 4, 64), normal(g, 2, 9, 2, 64)

    def step():
        out = hz.qk_rotary(q, k, freqs=freqs, positions=pos, axes=axes)
        return (*out, *torch.autograd.grad(out, (q, k), cot))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for turn in range(4):
        pos.copy_(torch.randint(0, 500, pos.shape, generator=g, device="cuda"))
        with torch.no_grad():
            q.copy_(normal(g, *q.shape))
        graph.replay()
        held = [t.clone() for t in got]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), turn


def test_captured_eviction():
    g = gen(7)
    for S, T in ((16, 8), (64, 40)):  # one launch; two, with a workspace
        k, v = normal(g, 3 * T, S, 2, 32), normal(g, 3 * T, S, 2, 32)
        table = torch.randperm(3 * T, generator=g, device="cuda").reshape(3, T).to(torch.int32)
        n, scores = ints([S * T, 5, S * T // 2]), torch.zeros(3, 2, S * T, device="cuda")
        hz.paged_evict(k.clone(), v.clone(), table, n, scores, 40)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = hz.paged_evict(k, v, table, n, scores, 40, sinks=1, recent=4)
        for turn in range(4):
            k.copy_(normal(g, *k.shape)), v.copy_(normal(g, *v.shape))
            scores.copy_(torch.rand(scores.shape, generator=g, device="cuda"))
            n.copy_(torch.randint(0, S * T + 1, (3,), generator=g, device="cuda"))
            k2, v2 = k.clone(), v.clone()
            graph.replay()
            want = hz.paged_evict(k2, v2, table, n, scores, 40, sinks=1, recent=4)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(k, k2) and torch.equal(v, v2), turn


# --- what is left alone -------------------------------------------------------------------------------


def test_results_do_not_depend_on_what_lies_around():
    """Rows beside, more table behind, other pages and slots behind the lengths: the same bits."""
    g = gen(8)
    k, v, table, n = filled(g, B=3, T=6, lengths=(40, 17, 90))
    q = normal(g, 3, 2, 4, 32)
    want = hz.paged_attention(q, k, v, table, n)
    one = hz.paged_attention(q[1:2], k, v, table[1:2], n[1:2])
    assert torch.equal(one, want[1:2])
    wide = torch.cat([table, torch.full((3, 5), -7, dtype=torch.int32, device="cuda")], 1)
    assert torch.equal(hz.paged_attention(q, k, v, wide, n)[:2], want[:2])
    used = torch.zeros(18, 16, dtype=torch.bool, device="cuda")
    for b, m in enumerate((40, 17, 90)):
        for j in range(m):
            used[table[b, j // 16], j % 16] = True
    for c in (k, v):
        c[~used] = float("nan")
    assert torch.equal(hz.paged_attention(q, k, v, table, n), want)
    strided = torch.zeros(3, 2, 9, 32, device="cuda")[:, :, 2:6]
    strided.copy_(q)
    assert torch.equal(hz.paged_attention(strided, k, v, table, n), want)
    odd = torch.zeros(3 * 2 * 4 * 32 + 1, device="cuda")[1:].reshape(3, 2, 4, 32).copy_(q)  # not 16-byte aligned: copied
    assert torch.equal(hz.paged_attention(odd, k, v, table, n), want)
    scores = torch.rand(3 * 2 * 96 + 1, generator=g, device="cuda")[1:].reshape(3, 2, 96)
    a = hz.paged_attention(q, k, v, table, n, scores=scores)[1]
    assert torch.equal(a, hz.paged_attention(q, k, v, table, n, scores=scores.clone())[1])


def test_rows_may_share_pages_that_are_read():
    g = gen(9)
    for dt in DT.values():
        k, v = normal(g, 9, 16, 2, 64, dtype=dt), normal(g, 9, 16, 2, 64, dtype=dt)
        table = ints([[0, 1, 2], [0, 1, 3], [0, 1, 2], [4, 4, 4]])
        n, q = ints([40, 45, 40, 48]), normal(g, 4, 1, 4, 64, dtype=dt)
        q[2] = q[0]
        got = hz.paged_attention(q, k, v, table, n)
        assert torch.equal(got[0], got[2])
        apart = torch.arange(12, dtype=torch.int32, device="cuda").reshape(4, 3)
        own_k, own_v = k[table.long().flatten()].contiguous(), v[table.long().flatten()].contiguous()
        assert torch.equal(hz.paged_attention(q, own_k, own_v, apart, n), got)


# --- all of them together -----------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_tokens_one_by_one_with_evictions(dtype):
    """Sites of a 5 x 9 lattice, row after row, for walkers that begin at different times; the cache is cut to 16 slots whenever a row has 24.
    Against the same in 64 bits on the operators' own rounded keys and selections, within the bounds."""
    dt, u = DT[dtype], F if dtype == "f32" else 2.0**-8
    B, T, S, H, Hk, D = 4, 3, 8, 4, 2, 32
    g = gen(10)
    s = new_state(g, dt, B, T, S, H, Hk, D)
    kc, vc, had = arr(s["kc"]), arr(s["vc"]), np.zeros((B, Hk, T * S))
    t_had = np.zeros_like(had)
    table, n = s["table"].cpu().numpy(), np.zeros(B, int)
    for i in range(45):
        feed(s, g, i)
        begun = np.array([1, 1, i >= 3, i >= 20])
        n = n + begun
        s["n"].copy_(ints(n))
        with torch.no_grad():
            out = decode_step(s)
            q, k = hz.qk_rotary(s["q"], s["k"], freqs=s["freqs"], positions=s["pos"], axes=s["axes"])
        a = arr(s["freqs"]), s["pos"].cpu().numpy(), s["axes"].cpu().numpy(), False
        for got, x in ((q, arr(s["q"])), (k, arr(s["k"]))):
            y = P.rotation(x, *a)
            size = np.abs(x) + np.abs(np.roll(x, D // 2, -1))
            assert (np.abs(arr(got) - y) <= u * np.abs(y) + (ANGLE + 4 * F) * size).all(), i
        P.append(kc, vc, arr(k), arr(s["v"]), table, n)
        assert np.array_equal(arr(s["kc"]), kc) and np.array_equal(arr(s["vc"]), vc), i
        want = P.attention(arr(q), kc, vc, table, n, scale=D**-0.5, scores=had, decay=0.9, bf16=dtype == "bf16")
        assert (np.abs(arr(out) - want["out"]) <= want["t_out"]).all(), i
        t_had = 0.9 * t_had * (np.arange(T * S) < n[:, None, None]) + want["t_scores"]
        had = want["scores"]
        assert (np.abs(arr(s["scores"]) - had) <= t_had).all(), i
        if (n >= 24).any():
            before = s["scores"].clone()
            lengths, sources, new = hz.paged_evict(s["kc"], s["vc"], s["table"], s["n"], before, 16, sinks=1, recent=8)
            ref = P.evict(kc, vc, table, n, before.cpu().numpy(), 16, sinks=1, recent=8)
            for got, x in zip((lengths, sources, new), ref):
                assert np.array_equal(got.cpu().numpy(), x), i
            assert np.array_equal(arr(s["kc"]), kc) and np.array_equal(arr(s["vc"]), vc), i
            n = ref[0].astype(int)
            s["scores"].copy_(new)
            move = np.where(ref[1] >= 0, ref[1], 0)
            inside = np.pad(ref[1] >= 0, ((0, 0), (0, 0), (0, T * S - 16)))
            pick = lambda x: np.where(inside, np.pad(np.take_along_axis(x, move, 2), ((0, 0), (0, 0), (0, T * S - 16))), 0)  # noqa: E731
            had, t_had = pick(had), pick(t_had)
    assert (n[:3] < 24).all() and n[3] > 16

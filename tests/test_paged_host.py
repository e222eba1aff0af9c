"""Paged operators without a GPU: the oracle against brute force and differences, and the refusals of the C ABI and of the Python
entry points (all before any GPU work)."""

import numpy as np
import pytest
import torch

import hamiltonzero_amd as hz
from hamiltonzero_amd import _native
from oracle import paged_oracle as P
from oracle import token_oracle as O

A = 0x10000  # a fake address: every call below fails its checks and never reads it


@pytest.fixture(scope="module")
def lib():
    if not _native.LIB_PATH.exists():
        pytest.skip("libhz_mhsea.so not built (run python -m hamiltonzero_amd.build)")
    return _native.lib()


# --- the oracle ------------------------------------------------------------------------------------


def test_oracle_attention_is_the_contiguous_one():
    rng = np.random.default_rng(1)
    B, Nq, H, Hk, D, S, T = 3, 2, 4, 2, 8, 5, 4
    q = rng.standard_normal((B, Nq, H, D))
    kc, vc = rng.standard_normal((2, 20, S, Hk, D))
    table = rng.permutation(20)[:B * T].reshape(B, T)
    lengths = np.array([20, 1, 13])
    slopes = np.array([0.5, 0.25, 0.125, 0.0625])
    got = P.attention(q, kc, vc, table, lengths, scale=0.3, softcap=4.0, slopes=slopes, scores=np.zeros((B, Hk, S * T)))
    k, v = kc[table].reshape(B, -1, Hk, D), vc[table].reshape(B, -1, Hk, D)
    want = O.attention(q, k, v, scale=0.3, softcap=4.0, slopes=slopes, causal=True, kv_len=lengths)
    np.testing.assert_allclose(got["out"], want["out"], rtol=1e-12, atol=1e-14)
    sums = got["scores"].sum(2)  # each query that sees a slot gives its heads' weights
    np.testing.assert_allclose(sums, (np.minimum(lengths, Nq) * (H // Hk))[:, None] * np.ones((1, Hk)), rtol=1e-12)


def test_oracle_rotation_turns_back_and_is_its_transpose():
    rng = np.random.default_rng(2)
    x, g = rng.standard_normal((2, 2, 5, 3, 16))
    freqs, axes = rng.random(8), np.array([0, 1, 2, 3, 0, 1, -1, 7])
    pos = rng.integers(-50, 50, (2, 5, 4))
    for inter in (False, True):
        y = P.rotation(x, freqs, pos, axes, inter)
        np.testing.assert_allclose(P.rotation(y, freqs, pos, axes, inter, -1), x, rtol=1e-12, atol=1e-14)
        np.testing.assert_allclose((y * g).sum(), (x * P.rotation(g, freqs, pos, axes, inter, -1)).sum(), rtol=1e-12)
        one = P.rotation(x, freqs, pos[:, :, :1], np.zeros(8, int), inter)
        want = x.copy()  # one axis is the rotation of the norms' oracle, whose input of a unit mean square is not scaled
        r = np.sqrt((x**2).mean(-1, keepdims=True))
        want = O.qk_norm_rotary(x, None, freqs, pos[:, :, 0], inter, 0.0) * r
        np.testing.assert_allclose(one, want, rtol=1e-12, atol=1e-13)


def test_oracle_eviction_keeps_the_largest_and_moves_few():
    rng = np.random.default_rng(3)
    B, Hk, D, S, T = 2, 3, 4, 4, 8
    kc, vc = rng.standard_normal((2, B * T, S, Hk, D))
    table = rng.permutation(B * T).reshape(B, T)
    lengths = np.array([31, 9])
    scores = rng.integers(0, 6, (B, Hk, S * T)).astype(np.float32)
    k0 = kc.copy()
    new, src, out = P.evict(kc, vc, table, lengths, scores, 10, sinks=2, recent=3)
    assert new.tolist() == [10, 9]
    for h in range(Hk):
        kept = sorted(src[0, h])
        assert len(set(kept)) == 10 and set(kept) >= {0, 1, 28, 29, 30}
        rest = set(range(2, 28)) - set(kept)
        assert min(scores[0, h, [s for s in kept if 2 <= s < 28]]) >= max(scores[0, h, list(rest)])
        assert all(src[0, h, s] == s or src[0, h, s] >= 10 for s in range(10))
        for s in range(10):
            a = src[0, h, s]
            assert np.array_equal(kc[table[0, s // S], s % S, h], k0[table[0, a // S], a % S, h])
        assert src[1, h].tolist() == [*range(9), -1] and np.array_equal(out[1, h, :9], scores[1, h, :9])
    assert np.array_equal(kc[table[1]], k0[table[1]])


# --- refusals --------------------------------------------------------------------------------------

TENSOR = dict(data=A, batch=2 * 16 * 32, token=2 * 32, head=32)
CACHE = dict(k=TENSOR, v=TENSOR, page_table=A, lengths=A, B=3, pages=7, page_size=16, table_width=4, Hk=2, D=32, dtype=0)
ATTN = dict(q=TENSOR, out=A, slopes=None, scores=None, scores_out=None, Nq=1, H=4, scale=0.2, softcap=0.0, decay=1.0)
EVICT = dict(scores=A, scores_out=2 * A, sources=A, lengths_out=2 * A, budget=10, sinks=1, recent=2)


def flat(d):
    return [y for x in d.values() for y in ([z or 0 for z in x.values()] if isinstance(x, dict) else [x or 0])]


def changed(base, over):
    out = {k: dict(v) if isinstance(v, dict) else v for k, v in base.items()}
    for k, v in over.items():
        if k in out:
            if isinstance(v, dict):
                out[k].update(v)
            else:
                out[k] = v
    return out


def cache(over=()):
    return _native.PAGED_CACHE.pack(*flat(changed(CACHE, dict(over))))


E, N, L = _native.HZ_EINVAL, _native.HZ_ENULL, _native.HZ_EALIGN
CACHE_BAD = [
    (dict(dtype=3), E, "dtype"), (dict(B=0), E, ">= 1"), (dict(pages=0), E, ">= 1"), (dict(page_size=0), E, ">= 1"),
    (dict(table_width=0), E, ">= 1"), (dict(Hk=0), E, ">= 1"), (dict(D=0), E, "head dimension"), (dict(D=20), E, "head dimension"),
    (dict(D=136), E, "head dimension"), (dict(pages=1 << 30), E, "2\\^30"), (dict(page_size=1 << 16, table_width=1 << 14), E, "2\\^30"),
    (dict(page_size=1 << 40), E, "2\\^30"), (dict(B=1 << 23, Hk=2), E, "grid"), (dict(B=1 << 62), E, "grid"),
    (dict(k=dict(data=None)), N, "k_cache"), (dict(v=dict(data=A + 8)), L, "v_cache"), (dict(k=dict(token=4)), E, "multiples of 8"),
    (dict(v=dict(batch=-8)), E, "not negative"), (dict(page_table=None), N, "page_table"), (dict(lengths=None), N, "lengths"),
    (dict(page_table=A + 2), L, "page_table"), (dict(lengths=A + 1), L, "lengths"),
]


def refused(rc, code, text, lib):
    import re

    assert rc == code, (rc, lib.hz_last_error())
    assert re.search(text, lib.hz_last_error().decode()), lib.hz_last_error()


@pytest.mark.parametrize("over,code,text", CACHE_BAD)
def test_abi_refuses_caches(lib, over, code, text):
    t = _native.TOKEN_TENSOR.pack(*flat(dict(t=TENSOR)))
    refused(lib.hz_paged_append(None, cache(over), t, t, 1), code, text, lib)
    a = cache(over) + _native.PAGED_ATTENTION_REST.pack(*flat(ATTN))
    refused(lib.hz_paged_attention(None, a, A, 1 << 40), code, text, lib)
    e = cache(over) + _native.PAGED_EVICT_REST.pack(*flat(EVICT))
    refused(lib.hz_paged_evict(None, e, A, 1 << 40), code, text, lib)


@pytest.mark.parametrize("over,code,text", [
    (dict(Nq=0), E, ">= 1"), (dict(H=0), E, ">= 1"), (dict(H=3), E, "multiple of Hk"), (dict(Nq=1 << 22), E, "grid"), (dict(H=1 << 40), E, "grid"),
    (dict(scale=float("nan")), E, "scale"), (dict(scale=float("inf")), E, "scale"), (dict(softcap=-1.0), E, "softcap"),
    (dict(softcap=float("inf")), E, "softcap"), (dict(decay=float("nan")), E, "decay"), (dict(decay=float("inf")), E, "decay"),
    (dict(q=dict(data=None)), N, "q must"), (dict(q=dict(head=12)), E, "q: strides"), (dict(out=None), N, "out"), (dict(out=A + 4), L, "out"),
    (dict(slopes=A + 2), L, "slopes"), (dict(scores=A), N, "scores_out"), (dict(scores_out=A + 4), L, "scores_out"),
    (dict(scores=A + 8, scores_out=A), L, "scores"),
])
def test_abi_refuses_attention(lib, over, code, text):
    a = cache() + _native.PAGED_ATTENTION_REST.pack(*flat(changed(ATTN, over)))
    refused(lib.hz_paged_attention(None, a, A, 1 << 40), code, text, lib)


def test_abi_refuses_caps_of_bfloat16_and_short_workspaces(lib):
    a = cache(dict(dtype=1)) + _native.PAGED_ATTENTION_REST.pack(*flat(changed(ATTN, dict(softcap=8193.0))))
    refused(lib.hz_paged_attention(None, a, A, 1 << 40), E, "softcap", lib)
    assert lib.hz_paged_attention_workspace(cache() + _native.PAGED_ATTENTION_REST.pack(*flat(ATTN))) == 0  # short rows need none
    a = cache(dict(page_size=512)) + _native.PAGED_ATTENTION_REST.pack(*flat(ATTN))
    size = lib.hz_paged_attention_workspace(a)
    assert size > 0
    refused(lib.hz_paged_attention(None, a, A, size - 1), E, "workspace", lib)
    refused(lib.hz_paged_attention(None, a, None, size), N, "workspace", lib)
    refused(lib.hz_paged_attention(None, a, A + 8, size), L, "workspace", lib)
    e = cache(dict(page_size=512)) + _native.PAGED_EVICT_REST.pack(*flat(EVICT))
    size = lib.hz_paged_evict_workspace(e)
    assert size > 0
    refused(lib.hz_paged_evict(None, e, A, size - 1), E, "workspace", lib)
    assert lib.hz_paged_evict_workspace(cache() + _native.PAGED_EVICT_REST.pack(*flat(EVICT))) == 0  # short rows need none
    for bad in (cache(dict(D=4)),):
        assert lib.hz_paged_attention_workspace(bad + _native.PAGED_ATTENTION_REST.pack(*flat(ATTN))) == -1
        assert lib.hz_paged_evict_workspace(bad + _native.PAGED_EVICT_REST.pack(*flat(EVICT))) == -1
    assert lib.hz_paged_attention(None, None, A, 1) == N and lib.hz_paged_evict(None, None, A, 1) == N
    assert lib.hz_paged_append(None, None, None, None, 1) == N
    assert lib.hz_paged_attention_workspace(None) == -1 and lib.hz_paged_evict_workspace(None) == -1


@pytest.mark.parametrize("over,code,text", [
    (dict(budget=0), E, "budget"), (dict(budget=1 << 30), E, "budget"), (dict(sinks=-1), E, "sinks"), (dict(recent=-1), E, "recent"),
    (dict(sinks=6, recent=5), E, "budget together"), (dict(sinks=1 << 62, recent=1 << 62), E, "together"), (dict(scores=None), N, "scores"),
    (dict(scores_out=None), N, "scores_out"), (dict(sources=None), N, "sources"), (dict(lengths_out=None), N, "lengths_out"),
    (dict(scores=A + 4), L, "scores"), (dict(sources=A + 2), L, "sources"), (dict(scores_out=A), E, "must not be the inputs"),
    (dict(lengths_out=A), E, "must not be the inputs"),
])
def test_abi_refuses_eviction(lib, over, code, text):
    e = cache() + _native.PAGED_EVICT_REST.pack(*flat(changed(EVICT, over)))
    refused(lib.hz_paged_evict(None, e, A, 1 << 40), code, text, lib)


def test_abi_refuses_evictions_of_more_threads_than_a_launch_has(lib):
    """The moves of one row, 32 of 256 threads: 2^32 threads at 2^29 - 31 of them."""
    long = dict(D=128, B=1, Hk=1, page_size=1, table_width=(1 << 30) - 1)
    for budget, most in (((1 << 29) - 1, False), ((1 << 29) - 31, False), ((1 << 29) - 32, True), ((1 << 29) + 40, True)):
        e = cache(long) + _native.PAGED_EVICT_REST.pack(*flat(changed(EVICT, dict(budget=budget))))
        if most:  # taken: only the workspace is too small
            assert lib.hz_paged_evict_workspace(e) > 1 << 31
            refused(lib.hz_paged_evict(None, e, A, 1), E, "workspace", lib)
        else:
            assert lib.hz_paged_evict_workspace(e) == -1
            refused(lib.hz_paged_evict(None, e, A, 1 << 40), E, "grid", lib)


def test_abi_refuses_appends(lib):
    t = _native.TOKEN_TENSOR.pack(*flat(dict(t=TENSOR)))
    for n, text in ((0, "N must"), (1 << 30, "N must"), (1 << 29, "grid")):
        refused(lib.hz_paged_append(None, cache(), t, t, n), E, text, lib)
    bad = _native.TOKEN_TENSOR.pack(*flat(changed(dict(t=TENSOR), dict(t=dict(data=None)))))
    refused(lib.hz_paged_append(None, cache(), bad, t, 1), N, "k must", lib)
    refused(lib.hz_paged_append(None, cache(), t, bad, 1), N, "v must", lib)
    assert lib.hz_paged_append(None, cache(), None, t, 1) == N


@pytest.mark.parametrize("over,n", [(dict(D=128, B=1 << 20, Hk=16), 1 << 4), (dict(D=128, B=1, Hk=1), 1 << 28), (dict(D=128, B=1, Hk=1), 1 << 27),
                                    (dict(D=128, dtype=1, B=4, Hk=4), 1 << 24), (dict(D=8, dtype=1, B=4, Hk=2), 1 << 29)], ids=str)
def test_abi_refuses_appends_of_more_threads_than_a_launch_has(lib, over, n):
    """A thread for each 16 bytes of a head: 2^32 and more."""
    t = _native.TOKEN_TENSOR.pack(*flat(dict(t=dict(TENSOR, batch=0, token=0, head=0))))
    refused(lib.hz_paged_append(None, cache(over), t, t, n), E, "grid", lib)


ROTARY = dict(q=TENSOR, k=TENSOR, q_out=TENSOR, k_out=TENSOR, w_q=None, w_k=None, freqs=A, positions=A, B=2, N=3, H=4, Hk=2, D=32,
              n_freqs=16, eps=1e-6, interleaved=0, dtype=0, axes=A, n_axes=2, norm=0)


@pytest.mark.parametrize("over,code,text", [
    (dict(n_axes=0), E, "n_axes"), (dict(n_axes=17), E, "n_axes"), (dict(norm=2), E, "norm"), (dict(positions=None), N, "positions"),
    (dict(axes=A + 2), L, "axes"), (dict(n_freqs=20), E, "n_freqs"), (dict(n_freqs=6), E, "n_freqs"), (dict(freqs=None), N, "freqs"),
    (dict(D=264), E, "head dimension"), (dict(q=dict(data=None)), N, "q must"), (dict(k_out=dict(head=4)), E, "strides"),
    (dict(B=0), E, ">= 1"), (dict(norm=1, eps=-1.0), E, "eps"),
])
def test_abi_refuses_rotations(lib, over, code, text):
    p = _native.QK_ROTARY.pack(*flat(changed(ROTARY, over)))
    refused(lib.hz_qk_rotary_fwd(None, p), code, text, lib)
    if "q" not in over:  # the reverse mode of a rotation alone does not read q
        refused(lib.hz_qk_rotary_bwd(None, p, A, A, None, None, None, 0), code, text, lib)


def test_abi_refuses_rotations_backward(lib):
    p = _native.QK_ROTARY.pack(*flat(ROTARY))
    refused(lib.hz_qk_rotary_bwd(None, p, None, A, None, None, None, 0), N, "dq", lib)
    refused(lib.hz_qk_rotary_bwd(None, p, A, A, A, None, None, 0), E, "norms", lib)
    norm = _native.QK_ROTARY.pack(*flat(changed(ROTARY, dict(norm=1))))
    size = lib.hz_qk_rotary_workspace(2, 3, 32, 1)
    assert size > 0 and lib.hz_qk_rotary_workspace(2, 3, 32, 0) == 0 and lib.hz_qk_rotary_workspace(0, 3, 32, 1) == -1
    refused(lib.hz_qk_rotary_bwd(None, norm, A, A, None, None, A, size - 1), E, "workspace", lib)
    refused(lib.hz_qk_rotary_bwd(None, None, A, A, None, None, None, 0), N, "p must", lib)
    assert lib.hz_qk_rotary_fwd(None, None) == N


def test_python_refuses_cpu_tensors():
    k = torch.zeros(4, 16, 2, 32)
    table, n, q = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros(1, 1, 4, 32)
    for call in (lambda: hz.paged_attention(q, k, k.clone(), table, n), lambda: hz.paged_append(k, k.clone(), q, q, table, n),
                 lambda: hz.paged_evict(k, k.clone(), table, n, torch.zeros(1, 2, 64), 4), lambda: hz.qk_rotary(q, q, freqs=torch.ones(16, dtype=torch.float64))):
        with pytest.raises(ValueError, match="GPU tensors"):
            call()
    with pytest.raises(TypeError, match="must be a tensor"):
        hz.paged_attention(q, [k], k, table, n)
    with pytest.raises(TypeError, match="freqs"):
        hz.qk_rotary(q, q, freqs=None)

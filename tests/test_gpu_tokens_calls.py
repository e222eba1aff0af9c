"""Calls of the token operators for what they do besides their numbers: results written into a caller's tensors, operands
with tangents, gradients of broadcast and shared leaves, tables of different sizes at once; and the cache kernel's widest
form."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

import hamiltonzero_amd as hz

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

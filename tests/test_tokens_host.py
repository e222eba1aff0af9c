"""Token operators without a GPU: the plan of buckets, the oracle's gradients against differences, and the
refusals of the C ABI and of the Python entry points (all before any GPU work)."""

import math

import numpy as np
import pytest
import torch

import hamiltonzero_amd as hz
from hamiltonzero_amd import _native, tokens
from oracle import token_oracle as O

A = 0x10000  # a fake address: every call below fails its checks and never reads it


@pytest.fixture(scope="module")
def lib():
    if not _native.LIB_PATH.exists():
        pytest.skip("libhz_mhsea.so not built (run python -m hamiltonzero_amd.build)")
    return _native.lib()


# --- buckets ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("n,R,both", [(32, 128, True), (32, 128, False), (64, 512, False), (2, 16, True), (1, 5, False),
                                      (2, 0, True), (8, 3, True), (16, 4, True), (512, 4096, True), (512, 300, False)])
def test_buckets_follow_the_formula(n, R, both):
    got = hz.relative_buckets(n, R, bidirectional=both).tolist()
    assert len(got) == 2 * R + 1 and got[R] == 0 and all(0 <= x < n for x in got)
    half = n // 2 if both else n
    near = half // 2
    for d in range(-R, R + 1):
        m, base = (abs(d), half if d > 0 else 0) if both else (max(-d, 0), 0)
        if m < near:
            want = m
        elif near and R > near:
            x = math.log(m / near) / math.log(R / near) * (half - near)
            if abs(x - round(x)) < 1e-9:  # on a border: the exact one counts (the next test)
                continue
            want = min(near + int(x), half - 1)
        else:
            want = min(near, half - 1)
        assert got[d + R] == base + want, d


def test_buckets_at_exact_borders():
    # half = 16, near = 8, R = 128: border t lies at 8 * 16^(t / 8), a whole number for t = 2, 4, 6
    got = hz.relative_buckets(32, 128).tolist()
    side = [got[128 - d] for d in range(129)]
    for t, d in ((2, 16), (4, 32), (6, 64)):
        assert side[d] == 8 + t and side[d - 1] == 8 + t - 1
    assert side[128] == 15


def test_buckets_refuse():
    for args in ((0, 16), (513, 16), (3, 16), (32, -1), (32, 4097)):
        with pytest.raises(ValueError):
            hz.relative_buckets(*args)


# --- the oracle against differences ------------------------------------------------------------------


def _difference(f, x, d, h=1e-5):
    return (f(x + h * d) - f(x - h * d)) / (2 * h)


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_norm_gradients(interleaved):
    rng = np.random.default_rng(1)
    x, w, dy, d = rng.normal(size=(2, 3, 2, 16)), rng.normal(size=16), rng.normal(size=(2, 3, 2, 16)), rng.normal(size=(2, 3, 2, 16))
    freqs, pos = rng.uniform(0.1, 1, 4), rng.integers(0, 50, (2, 3))
    _, dx, dw = O.qk_norm_rotary(x, w, freqs, pos, interleaved, 1e-6, dy)
    f = lambda x_: (O.qk_norm_rotary(x_, w, freqs, pos, interleaved, 1e-6) * dy).sum()  # noqa: E731
    assert abs(_difference(f, x, d) - (dx * d).sum()) < 1e-7
    dd = rng.normal(size=16)
    f = lambda w_: (O.qk_norm_rotary(x, w_, freqs, pos, interleaved, 1e-6) * dy).sum()  # noqa: E731
    assert abs(_difference(f, w, dd) - (dw * dd).sum()) < 1e-7


@pytest.mark.parametrize("kw", [dict(), dict(softcap=2.0, causal=True), dict(slopes=True, causal=True, prefix=[3, 0]),
                                dict(documents=True, softcap=3.0), dict(kv_len=[5, 0], causal=True)])
def test_oracle_attention_gradients(kw):
    rng = np.random.default_rng(2)
    B, Nq, Nk, H, Hk, D = 2, 6, 7, 4, 2, 8
    kw = dict(kw)
    if kw.pop("slopes", False):
        kw["slopes"] = rng.uniform(0, 0.5, H)
    if kw.pop("documents", False):
        kw["documents"] = np.array([[0, 0, 1, 1, 1, -1, -1], [-1, 2, 2, 0, 0, 0, 2]])
    x = [rng.normal(size=s) for s in ((B, Nq, H, D), (B, Nk, Hk, D), (B, Nk, Hk, D))]
    dout = rng.normal(size=(B, Nq, H, D))
    r = O.attention(*x, scale=0.7, dout=dout, **kw)
    for i, name in enumerate(("dq", "dk", "dv")):
        d = rng.normal(size=x[i].shape)

        def f(y):
            z = list(x)
            z[i] = y
            return (O.attention(*z, scale=0.7, **kw)["out"] * dout).sum()

        assert abs(_difference(f, x[i], d) - (r[name] * d).sum()) < 1e-6, name


# --- refusals of the C ABI ----------------------------------------------------------------------------


def _norm(**over):
    f = dict(q=(A, 8192, 512, 64), k=(A, 8192, 512, 64), qo=(A, 8192, 512, 64), ko=(A, 8192, 512, 64), w_q=A, w_k=A, freqs=A,
             positions=A, B=2, N=16, H=8, Hk=8, D=64, n_freqs=32, eps=1e-6, interleaved=0, dtype=0)
    f.update(over)
    flat = [x for v in f.values() for x in (v if isinstance(v, tuple) else (v,))]
    return _native.QK_NORM_ROTARY.pack(*flat)


def _attn(**over):
    f = dict(q=(A, 8192, 512, 64), k=(A, 8192, 512, 64), v=(A, 8192, 512, 64), out=A, out_low=0, lse=A, slopes=0, prefix=0, documents=0,
             kv_len=0, B=2, Nq=16, Nk=16, H=8, Hk=8, D=64, scale=0.125, softcap=0.0, causal=1, dtype=0)
    f.update(over)
    flat = [x for v in f.values() for x in (v if isinstance(v, tuple) else (v,))]
    return _native.TOKEN_ATTENTION.pack(*flat)


E = _native


@pytest.mark.parametrize("over,code,needle", [
    (dict(D=60), E.HZ_EINVAL, "head dimension"), (dict(D=264), E.HZ_EINVAL, "head dimension"), (dict(D=0), E.HZ_EINVAL, "head dimension"),
    (dict(n_freqs=6), E.HZ_EINVAL, "n_freqs"), (dict(n_freqs=36), E.HZ_EINVAL, "n_freqs"), (dict(n_freqs=-4), E.HZ_EINVAL, "n_freqs"),
    (dict(B=0), E.HZ_EINVAL, "B, N, H and Hk"), (dict(N=0), E.HZ_EINVAL, "B, N, H and Hk"), (dict(Hk=0), E.HZ_EINVAL, "B, N, H and Hk"),
    (dict(N=1 << 31), E.HZ_EINVAL, "supported size"), (dict(dtype=2), E.HZ_EINVAL, "dtype"),
    (dict(eps=float("nan")), E.HZ_EINVAL, "eps"), (dict(eps=-1.0), E.HZ_EINVAL, "eps"), (dict(freqs=0), E.HZ_ENULL, "freqs"),
    (dict(freqs=A + 4), E.HZ_EALIGN, "freqs"), (dict(w_k=A + 2), E.HZ_EALIGN, "w_k"), (dict(q=(0, 0, 0, 0)), E.HZ_ENULL, "q must"),
    (dict(k=(A + 8, 0, 0, 0)), E.HZ_EALIGN, "k must"), (dict(qo=(A, 4, 0, 0)), E.HZ_EINVAL, "q_out: strides"),
    (dict(ko=(A, -8, 0, 0)), E.HZ_EINVAL, "k_out: strides"),
])
def test_norm_refuses(lib, over, code, needle):
    assert lib.hz_qk_norm_rotary_fwd(None, _norm(**over)) == code
    assert needle in lib.hz_last_error().decode()
    assert lib.hz_qk_norm_rotary_bwd(None, _norm(**over), A, A, A, A, A, 1 << 40) == code


def test_norm_backward_refuses(lib):
    need = lib.hz_qk_norm_rotary_workspace(2, 16, 64)
    assert need > 0 and lib.hz_qk_norm_rotary_workspace(0, 16, 64) == -1
    assert lib.hz_qk_norm_rotary_bwd(None, _norm(), A, A, A, A, A, need - 1) == E.HZ_EINVAL
    assert "workspace" in lib.hz_last_error().decode()
    assert lib.hz_qk_norm_rotary_bwd(None, _norm(), A, A, A, A, None, need) == E.HZ_ENULL
    assert lib.hz_qk_norm_rotary_bwd(None, _norm(), A, None, A, A, A, need) == E.HZ_ENULL
    assert lib.hz_qk_norm_rotary_bwd(None, _norm(), A + 8, A, A, A, A, need) == E.HZ_EALIGN
    assert lib.hz_qk_norm_rotary_fwd(None, None) == E.HZ_ENULL


@pytest.mark.parametrize("over,code,needle", [
    (dict(D=60), E.HZ_EINVAL, "head dimension"), (dict(D=136), E.HZ_EINVAL, "head dimension"),
    (dict(H=6, Hk=4), E.HZ_EINVAL, "multiple of Hk"), (dict(Nq=0), E.HZ_EINVAL, ">= 1"), (dict(Nk=0), E.HZ_EINVAL, ">= 1"),
    (dict(Nk=1 << 30), E.HZ_EINVAL, "2^30"), (dict(B=1 << 21), E.HZ_EINVAL, "grid limit"), (dict(dtype=-1), E.HZ_EINVAL, "dtype"),
    (dict(scale=float("inf")), E.HZ_EINVAL, "scale"), (dict(softcap=-1.0), E.HZ_EINVAL, "softcap"),
    (dict(softcap=float("nan")), E.HZ_EINVAL, "softcap"), (dict(softcap=1e-37, scale=1.0), E.HZ_EINVAL, "softcap"),
    (dict(softcap=8193.0, dtype=1), E.HZ_EINVAL, "softcap"), (dict(scale=1e31), E.HZ_EINVAL, "scale"), (dict(causal=2), E.HZ_EINVAL, "causal"),
    (dict(causal=0, prefix=A), E.HZ_EINVAL, "prefix needs causal"), (dict(prefix=A + 2), E.HZ_EALIGN, "prefix"),
    (dict(documents=A + 1), E.HZ_EALIGN, "documents"), (dict(kv_len=A + 1), E.HZ_EALIGN, "kv_len"),
    (dict(slopes=A + 2), E.HZ_EALIGN, "slopes"), (dict(lse=A + 2), E.HZ_EALIGN, "lse"), (dict(out=0), E.HZ_ENULL, "out"),
    (dict(out=A + 4), E.HZ_EALIGN, "out"), (dict(out_low=A + 8), E.HZ_EALIGN, "out_low"), (dict(v=(0, 0, 0, 0)), E.HZ_ENULL, "v must"),
    (dict(k=(A, 0, 12, 0)), E.HZ_EINVAL, "k: strides"), (dict(q=(A + 4, 0, 0, 0)), E.HZ_EALIGN, "q must"),
])
def test_attention_refuses(lib, over, code, needle):
    assert lib.hz_token_attention_fwd(None, _attn(**over), A, 1 << 40) == code
    assert needle in lib.hz_last_error().decode()
    d = _native.TOKEN_TENSOR.pack(A, 8192, 512, 64)
    assert lib.hz_token_attention_bwd(None, _attn(**over), d, A, A, A, A, 1 << 40) == code


def test_attention_workspaces_and_backward_refuse(lib):
    d = _native.TOKEN_TENSOR.pack(A, 8192, 512, 64)
    need = lib.hz_token_attention_fwd_workspace(_attn(Nq=1))
    assert need > 0 and lib.hz_token_attention_fwd_workspace(_attn(D=60)) == -1
    assert lib.hz_token_attention_fwd(None, _attn(Nq=1), A, need - 1) == E.HZ_EINVAL
    assert lib.hz_token_attention_fwd(None, _attn(Nq=1), None, need) == E.HZ_ENULL
    assert lib.hz_token_attention_fwd(None, None, A, need) == E.HZ_ENULL
    need = lib.hz_token_attention_bwd_workspace(_attn())
    assert need > 0 and lib.hz_token_attention_bwd_workspace(_attn(Nk=0)) == -1
    for args, code in (((_attn(lse=0), d, A, A, A, A, need), E.HZ_ENULL), ((_attn(), None, A, A, A, A, need), E.HZ_ENULL),
                       ((_attn(), _native.TOKEN_TENSOR.pack(A, 1, 0, 0), A, A, A, A, need), E.HZ_EINVAL),
                       ((_attn(), d, A, None, A, A, need), E.HZ_ENULL), ((_attn(), d, A, A, A + 8, A, need), E.HZ_EALIGN),
                       ((_attn(), d, A, A, A, A, need - 1), E.HZ_EINVAL), ((_attn(), d, A, A, A, None, need), E.HZ_ENULL)):
        assert lib.hz_token_attention_bwd(None, *args) == code


@pytest.mark.parametrize("over,code,needle", [
    (dict(B=0), E.HZ_EINVAL, ">= 1"), (dict(H=0), E.HZ_EINVAL, "H must"), (dict(H=257), E.HZ_EINVAL, "H must"),
    (dict(nb=0), E.HZ_EINVAL, "n_buckets"), (dict(nb=513), E.HZ_EINVAL, "n_buckets"), (dict(R=-1), E.HZ_EINVAL, "R must"),
    (dict(R=4097), E.HZ_EINVAL, "R must"), (dict(nb=512, H=65), E.HZ_EINVAL, "table of"), (dict(dtype=3), E.HZ_EINVAL, "dtype"),
    (dict(flags=1), E.HZ_EINVAL, "flag"), (dict(B=1 << 29, Nq=1 << 29, Nk=1 << 29), E.HZ_EINVAL, "tensor size"),
    (dict(buckets=None), E.HZ_ENULL, "buckets"), (dict(qpos=A + 2), E.HZ_EALIGN, "q_positions"), (dict(x=None), E.HZ_ENULL, "must"),
    (dict(x=A + 4), E.HZ_EALIGN, "aligned"),
])
def test_bias_refuses(lib, over, code, needle):
    f = dict(table=A, buckets=A, qpos=A, kpos=A, x=A, B=2, Nq=8, Nk=8, H=4, nb=32, R=16, dtype=0, flags=0)
    f.update(over)
    assert lib.hz_bucket_bias_fwd(None, *f.values()) == code
    assert needle in lib.hz_last_error().decode()
    sizes = [f[n] for n in ("B", "Nq", "Nk", "H", "nb", "R", "dtype", "flags")]
    assert lib.hz_bucket_bias_bwd(None, f["x"], f["buckets"], f["qpos"], f["kpos"], A, A, 1 << 40, *sizes) == code
    need = lib.hz_bucket_bias_workspace(2, 8, 8, 4, 32, 0, 0)
    assert lib.hz_bucket_bias_bwd(None, A, A, A, A, A, A, need - 1, 2, 8, 8, 4, 32, 16, 0, 0) == E.HZ_EINVAL


def test_host_tensors_are_refused():
    x = torch.zeros(1, 2, 2, 16)
    with pytest.raises(ValueError, match="GPU"):
        hz.token_attention(x, x, x)
    with pytest.raises(ValueError, match="GPU"):
        hz.qk_norm_rotary(x, x)
    with pytest.raises(ValueError, match="GPU"):
        hz.bucket_bias(torch.zeros(4, 2), torch.zeros(3, dtype=torch.int32), x, x)
    with pytest.raises(TypeError):
        hz.token_attention(x.double(), x, x)


def test_strided_views_are_taken_in_place():
    base = torch.zeros(3, 5, 12, 16)
    assert tokens._strided(base[:, :, 4:8]) is not None
    view = base[:, :, 4:8]
    assert tokens._strided(view) is view and tokens._fields(view)[1:] == (960, 192, 16)
    odd = torch.zeros(3, 5, 4, 17)[..., :16]
    assert tokens._strided(odd) is not odd and tokens._strided(odd).is_contiguous()
    off = torch.zeros(3 * 5 * 4 * 16 + 1)[1:].view(3, 5, 4, 16)
    assert tokens._strided(off).data_ptr() % 16 == 0
    wide = torch.zeros(1, 1, 2, 16).expand(3, 5, 2, 16)
    assert tokens._strided(wide) is wide and tokens._fields(wide)[1:] == (0, 0, 16)
    turned = torch.zeros(3, 16, 4, 5).transpose(1, 3)
    assert tokens._strided(turned).is_contiguous()

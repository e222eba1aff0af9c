"""Sizes that the token attention's C entry takes and refuses, by its workspace calls and checks (nothing is enqueued)."""

import math
import struct

import pytest

from hamiltonzero_amd import _native, tokens

A = 0x10000  # a fake address: never read


@pytest.fixture(scope="module")
def lib():
    if not _native.LIB_PATH.exists():
        pytest.skip("libhz_mhsea.so not built (run python -m hamiltonzero_amd.build)")
    return _native.lib()


def attn(B, Nq, Nk, H, Hk, D, lse=0, documents=0):
    rows = (A, Nk * Hk * D, Hk * D, D)
    return _native.TOKEN_ATTENTION.pack(A, Nq * H * D, H * D, D, *rows, *rows, A, 0, lse, 0, 0, documents, 0, B, Nq, Nk, H, Hk, D,
                                        0.125, 0.0, 1, _native.HZ_DTYPE_BF16)


@pytest.mark.parametrize("B,Nq,Nk,H,Hk,D", [(256, 1, 131072, 32, 8, 128), (32, 1, 1 << 20, 8, 8, 64), (4, 200, (1 << 30) - 1, 8, 8, 8),
                                            (1 << 20, 1, 700, 1, 1, 16)])
def test_long_caches(lib, B, Nq, Nk, H, Hk, D):
    """A forward takes any cache; only what a reverse pass divides its keys into is limited."""
    assert lib.hz_token_attention_fwd_workspace(attn(B, Nq, Nk, H, Hk, D)) >= 0
    assert lib.hz_token_attention_fwd_workspace(attn(B, Nq, Nk, H, Hk, D, lse=A)) == -1
    assert lib.hz_token_attention_bwd_workspace(attn(B, Nq, Nk, H, Hk, D, lse=A)) == -1
    assert "grid limit" in lib.hz_last_error().decode()
    d = _native.TOKEN_TENSOR.pack(A, 8, 8, 8)
    assert lib.hz_token_attention_fwd(None, attn(B, Nq, Nk, H, Hk, D, lse=A), A, 1 << 60) == _native.HZ_EINVAL
    assert lib.hz_token_attention_bwd(None, attn(B, Nq, Nk, H, Hk, D, lse=A), d, A, A, A, A, 1 << 60) == _native.HZ_EINVAL


def test_documents_of_too_many_tokens(lib):
    assert lib.hz_token_attention_fwd_workspace(attn(256, 200, 1 << 24, 1, 1, 8, documents=A)) == -1
    assert "documents" in lib.hz_last_error().decode()
    assert lib.hz_token_attention_fwd(None, attn(256, 1, 1 << 24, 1, 1, 8, documents=A), A, 1 << 60) == _native.HZ_EINVAL
    assert lib.hz_token_attention_fwd_workspace(attn(128, 200, 1 << 24, 1, 1, 8, documents=A)) > 0


@pytest.mark.parametrize("x", [0.0, 1.5, -3.4028234663852886e38, 3.402823567e38, 1e39, -1e300, math.inf, -math.inf, math.nan])
def test_options_beyond_float32(x):
    """They reach the library, whose checks name them, as infinities: no error of the packing comes first."""
    got, = struct.unpack("f", struct.pack("f", tokens._float32(x)))
    assert (math.isnan(got) and math.isnan(x)) or got == x or (math.isinf(got) and got * x > 0 and abs(x) > 3.4028234e38)

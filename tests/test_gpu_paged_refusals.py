"""Memory that a paged call may not write: scores in the caches or in the queries."""

import pytest
import torch

import hamiltonzero_amd as hz

pytestmark = pytest.mark.gpu


def buffers():
    """Caches [12, 16, 2, 32] and queries of one float32 buffer, with 3 * 2 * 64 scores in each of them and behind, 16-byte aligned."""
    n = 12 * 16 * 2 * 32
    base = torch.randn(2 * n + 3 * 4 * 32 + 4 + 384, device="cuda")
    k, v = base[:n].reshape(12, 16, 2, 32), base[n:2 * n].reshape(12, 16, 2, 32)
    q = base[2 * n:2 * n + 384].reshape(3, 1, 4, 32)
    table = torch.arange(12, dtype=torch.int32, device="cuda").reshape(3, 4)
    lengths = torch.tensor([40, 17, 64], dtype=torch.int32, device="cuda")
    scores_at = lambda i: base[i:i + 384].reshape(3, 2, 64)  # noqa: E731
    return base, n, k, v, q, table, lengths, scores_at


def test_scores_out_in_what_is_read_is_refused():
    base, n, k, v, q, table, lengths, scores_at = buffers()
    scores = torch.rand(3, 2, 64, device="cuda")
    kept = base.clone()
    for i in (0, n - 384, n - 4, n, 2 * n - 384, 2 * n - 4, 2 * n, 2 * n + 380):
        with pytest.raises(ValueError, match="scores_out must not overlap q or the caches"):
            hz.paged_attention(q, k, v, table, lengths, scores=scores, scores_out=scores_at(i))
        assert torch.equal(base, kept)
    out, new = hz.paged_attention(q, k, v, table, lengths, scores=scores)
    again, into = hz.paged_attention(q, k, v, table, lengths, scores=scores, scores_out=scores_at(2 * n + 384))  # next to the queries
    assert torch.equal(out, again) and torch.equal(into, new) and torch.equal(base[:2 * n + 384], kept[:2 * n + 384])
    # between the rows of caches that are views, where no cache has an element
    wide = torch.randn(12, 16, 2, 64, device="cuda")
    a, b = wide[..., :32], torch.randn(12, 16, 2, 32, device="cuda")
    with pytest.raises(ValueError, match="scores_out must not overlap"):
        hz.paged_attention(q, a, b, table, lengths, scores=scores, scores_out=wide.view(-1)[:384].reshape(3, 2, 64))
    # a query that is copied is read from its copy
    odd = torch.randn(3, 1, 4, 33, device="cuda")[..., :32]
    assert hz.paged_attention(odd, k, v, table, lengths, scores=scores, scores_out=scores.clone())[0].shape == q.shape


def test_eviction_by_scores_in_the_caches_is_refused():
    base, n, k, v, q, table, lengths, scores_at = buffers()
    kept = base.clone()
    for i in (0, n - 384, n - 4, n, 2 * n - 4):
        with pytest.raises(ValueError, match="scores must not overlap the caches"):
            hz.paged_evict(k, v, table, lengths, scores_at(i), 8)
        assert torch.equal(base, kept)
    hz.paged_evict(k, v, table, lengths, scores_at(2 * n), 8)  # behind them
    # a view that is copied is read from its copy
    hz.paged_evict(k, v, table, lengths, base[:768].reshape(3, 2, 128)[:, :, ::2], 8)
    with pytest.raises(ValueError, match="k and v must not overlap the caches"):
        hz.paged_append(k, v, k[:6].reshape(3, 32, 2, 32)[:, :2], q.reshape(3, 2, 2, 32), table, lengths)
    with pytest.raises(ValueError, match="k_cache and v_cache must not overlap"):
        hz.paged_append(k, k, q.reshape(3, 2, 2, 32), q.reshape(3, 2, 2, 32), table, lengths)

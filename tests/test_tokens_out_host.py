"""Whether strided tensors share memory, as the operators that write into a caller's tensors decide it, against a count of every
element's place."""

import random

import pytest
import torch

from hamiltonzero_amd import tokens


def places(t):
    """The address of every element."""
    at = torch.zeros((), dtype=torch.int64)
    for n, s in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(n) * s
    return (t.data_ptr() + at.reshape(-1) * t.element_size()).tolist()


def share(a, b):
    size = lambda t: {x + i for x in places(t) for i in range(t.element_size())}  # noqa: E731
    return bool(size(a) & size(b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_random_windows(dtype):
    rng = random.Random(1)
    base = torch.zeros(4000, dtype=dtype)
    found = [0, 0, 0, 0]
    for _ in range(1500):
        pair = []
        for _ in range(2):
            shape = [rng.choice([1, 1, 2, 3, 5]) for _ in range(3)] + [8]
            strides = [rng.choice([0, 8, 16, 24, 40, 64, 80, 8 * rng.randint(0, 12)]) for _ in range(3)] + [1]
            pair.append(base.as_strided(shape, strides, 8 * rng.randint(0, 30) + rng.choice([0, 0, 0, 3])))
        a, b = pair
        want = share(a, b)
        assert tokens._overlap(a, b) == want and tokens._overlap(b, a) == want, (a.shape, a.stride(), b.shape, b.stride())
        twice = len(set(places(a))) < a.numel()
        assert tokens._holds_twice(a) == twice, (a.shape, a.stride())
        found[2 * want + twice] += 1
    assert min(found) > 20, found  # of each kind some


def test_views_of_one_buffer():
    rows = torch.zeros(2, 9, 8, 32)
    q, k = rows[:, :8, :4], rows[:, :8, 4:6]
    for a, b, want in ((q, k, False), (q, rows[:, :8, 1:5], True), (q, rows[:, 1:, :4], True), (k, rows[:, 1:, 4:6], True),
                       (k, rows[:, :8, 6:], False), (q, rows[:, 8:, :4], False), (q, rows[:, :8, :4, 16:], True),
                       (rows[..., :16], rows[..., 16:], False), (q, torch.zeros_like(q), False), (q, q, True)):
        assert tokens._overlap(a, b) == want and tokens._overlap(b, a) == want
    cache = torch.zeros(3, 2, 1000, 16).transpose(1, 2)  # heads outside tokens
    assert not tokens._overlap(cache[:, 5:6], cache[:, 6:7]) and tokens._overlap(cache[:, 5:7], cache[:, 6:8])
    assert not tokens._holds_twice(cache) and tokens._holds_twice(cache[:1].expand(3, -1, -1, -1))
    assert tokens._holds_twice(torch.zeros(4096).as_strided((2, 8, 4, 32), (1024, 64, 32, 1)))


def test_large_views_are_decided_at_once():
    """Nothing grows with the number of elements."""
    x = torch.empty(4, 1 << 14, 8, 16, dtype=torch.bfloat16)
    assert not tokens._overlap(x[:, : 1 << 13], x[:, 1 << 13:]) and not tokens._overlap(x[:, :, :4], x[:, :, 4:])
    assert tokens._overlap(x[:, : (1 << 13) + 1], x[:, 1 << 13:]) and not tokens._holds_twice(x[:, ::2])


def test_results_against_inputs_and_each_other():
    rows, other = torch.zeros(2, 9, 8, 32), torch.zeros(2, 8, 4, 32)
    q, k = rows[:, :8, :4], rows[:, :8, 4:6]
    a, b = other, torch.zeros(2, 8, 2, 32)
    assert not tokens._meet((a, b), (q, k)) and not tokens._meet((a, rows[:, :8, 6:]), (q, k)) and not tokens._meet((a, b), (q, q))
    for out in ((q, b), (a, k), (rows[:, 1:, :4], b), (a, rows[:, 1:, 5:7]), (rows[:, :8, 4:], b), (a, a[:, :, 1:3]), (a, a)):
        assert tokens._meet(out, (q, k)) and tokens._meet(out[::-1], (q, k))

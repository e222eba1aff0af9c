"""Rotations of many tokens of few heads: a workgroup takes up to sixteen tokens at a time, which lie in several rows of the batch where rows are
short. Element by element within the bounds of one rounding and of the angle's."""

import numpy as np
import pytest
import torch

import hamiltonzero_amd as hz
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu
F = 2.0**-24
ANGLE = 2.0**-21  # the angle's rounding to float32 turns (2 pi 2^-25) and its sine's
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def arr(t):
    return t.detach().double().cpu().numpy()


def within(name, got, want, bound):
    off = np.abs(arr(got) - want)
    assert (off <= bound).all(), (name, float((off / np.maximum(bound, 1e-300)).max()), np.argwhere(~(off <= bound))[:4].tolist())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("B,N,H,Hk,D,nf,A", [(7001, 3, 1, 1, 16, 8, 2), (20011, 1, 2, 1, 8, 4, 3), (5, 4099, 3, 2, 32, 12, 2), (2, 8200, 6, 4, 64, 32, 3), (1, 17000, 7, 4, 24, 8, 1),
                                              (3001, 5, 12, 8, 48, 24, 2)], ids=lambda x: str(x))
def test_many_tokens(B, N, H, Hk, D, nf, A, inter, dtype):
    print(f"[case] many {B} {N} {H} {Hk} {D} {nf} {A} {inter} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(61)
    dt, u = DT[dtype], F if dtype == "f32" else 2.0**-8
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda").to(dt)  # noqa: E731
    rows = normal(B, N, H + 2 * Hk, D)
    q, k = (x.detach().requires_grad_() for x in (rows[:, :, :H], rows[:, :, H:H + Hk]))
    freqs = 100.0 ** (-torch.arange(nf, dtype=torch.float64, device="cuda") / nf)
    pos = torch.randint(-500, 5000, (B, N, A), generator=g, device="cuda").to(torch.int32)
    axes = (torch.arange(nf, device="cuda") % A).to(torch.int32)
    a = (arr(freqs), pos.cpu().numpy(), axes.cpu().numpy(), inter)
    i = np.arange(nf)
    ia, ib = (2 * i, 2 * i + 1) if inter else (i, i + nf)

    def pair_size(x):
        s = np.zeros_like(x)
        s[..., ia] = s[..., ib] = np.abs(x[..., ia]) + np.abs(x[..., ib])
        return s

    out = hz.qk_rotary(q, k, freqs=freqs, positions=pos, axes=axes, interleaved=inter)
    cot = [normal(*o.shape) for o in out]
    grads = torch.autograd.grad(out, (q, k), cot)
    w = torch.rand(D, generator=g, device="cuda") + 0.5
    normed = hz.qk_norm_rotary(q.detach(), k.detach(), w, w, freqs=freqs, positions=pos, axes=axes, interleaved=inter)
    for n in range(2):
        x, dy = arr((q, k)[n]), arr(cot[n])
        y, dx = P.rotation(x, *a), P.rotation(dy, *a, -1)
        within("y", out[n], y, u * np.abs(y) + (ANGLE + 4 * F) * pair_size(x))
        within("dx", grads[n], dx, u * np.abs(dx) + (ANGLE + 4 * F) * pair_size(dy))
        m = x / np.sqrt((x**2).mean(-1, keepdims=True) + 1e-6) * arr(w)
        y = P.rotation(m, *a)
        within("norm", normed[n], y, u * np.abs(y) + (ANGLE + 16 * F) * 2 * np.abs(m).max(-1, keepdims=True))

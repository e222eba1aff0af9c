"""Token operators on the gfx950 library (``include/hz_token.h``): what an autoregressive
wavefunction over the same sites, or a model of token sequences, needs next to the MHSEA kernels.
The reference has no counterpart.

* :func:`qk_norm_rotary` — RMS norms of queries and keys for each head, and the rotation by position (of one axis or
  several) in the same pass; :func:`qk_rotary` — the rotation alone.
* :func:`token_attention` — attention with shared key heads, tanh-capped scores, a distance bias and
  causal, prefix, document and length masks; single tokens over a cache.
* :func:`bucket_bias` — a learned relative position bias by buckets, in the bias layouts of
  :mod:`hamiltonzero_amd.kernels` and of the rectangular attention; :func:`relative_buckets` makes
  its plan.

All are differentiable in reverse mode (once) through ``torch.autograd``, not in forward mode; a call that
needs no gradient enqueues the forward alone. Tensors are float32 or bfloat16 GPU tensors on one device; work goes to
the current stream of that device. There is no CPU fallback. Query, key and value tensors (and their
cotangents) may be strided views whose last axis is contiguous (slices of one projection, a cache's
rows); others are copied first. Every axis must be at least 1 long.
"""

from __future__ import annotations

import contextlib
import math
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version
from torch.autograd.function import once_differentiable

from . import _native

Tensor = torch.Tensor

_DTYPES = {torch.float32: _native.HZ_DTYPE_F32, torch.bfloat16: _native.HZ_DTYPE_BF16}
MAX_HEAD_DIM = 128
MAX_ROTARY_HEAD_DIM = 256
MAX_AXES = 16
MAX_BUCKETS = 512
MAX_BUCKET_RANGE = 4096


def _on(device: torch.device):
    """The launches need ``device`` as the current one."""
    if device.index == torch.cuda.current_device():
        return _HERE
    return torch.cuda.device(device)


_HERE = contextlib.nullcontext()


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _float32(x: float) -> float:
    """``x`` as the library's structures hold it: infinite beyond float32's range, which it refuses."""
    x = float(x)
    return x if not abs(x) > 3.4028234663852886e38 else math.copysign(math.inf, x)


def _ptr(t: Optional[Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _strided(t: Tensor) -> Tensor:
    """``t`` if the kernels can read it in place (contiguous heads, 16-byte rows), else a copy."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t
        st = t.stride()
        if st[-1] == 1 and all(s % 8 == 0 or n == 1 for s, n in zip(st[:-1], t.shape)):
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _fields(t: Tensor) -> tuple:
    """Address and strides of batch, token and head axes; an axis of one element has none."""
    (n0, n1, n2, _), (s0, s1, s2, _) = t.shape, t.stride()
    return t.data_ptr(), 0 if n0 == 1 else s0, 0 if n1 == 1 else s1, 0 if n2 == 1 else s2


def _reaches(d: int, terms: list) -> bool:
    """Whether ``d`` is a sum of ``c * step`` with ``low <= c <= high`` for each ``(step, low, high)`` of ``terms`` (positive
    steps in descending order). Steps that enclose each other, as a view's do, leave a choice or two each."""
    if not terms:
        return d == 0
    step, low, high = terms[0]
    rest = terms[1:]
    first = max(low, -((sum(s * h for s, _, h in rest) - d) // step))
    last = min(high, (d - sum(s * l for s, l, _ in rest)) // step)
    return any(_reaches(d - c * step, rest) for c in range(first, last + 1))


def _steps(t: Tensor) -> list:
    """``(bytes, count)`` of each axis of ``t`` that moves, with its elements' bytes as one more."""
    size = t.element_size()
    return [(s * size, n) for s, n in zip(t.stride(), t.shape) if n > 1 and s] + [(1, size)]


def _end(t: Tensor) -> int:
    """The address behind the last element of a strided [B, N, H, D] tensor."""
    (n0, n1, n2, n3), (s0, s1, s2, s3) = t.shape, t.stride()
    return t.data_ptr() + ((n0 - 1) * s0 + (n1 - 1) * s1 + (n2 - 1) * s2 + (n3 - 1) * s3 + 1) * t.element_size()


def _overlap(a: Tensor, b: Tensor) -> bool:
    """Whether two strided tensors share a byte. (Views of one buffer may lie between each other's rows and share none.)"""
    d = b.data_ptr() - a.data_ptr()
    low, high = {}, {}
    for s, n in _steps(a):
        high[s] = high.get(s, 0) + n - 1
    for s, n in _steps(b):
        low[s] = low.get(s, 0) + 1 - n
    return _reaches(d, [(s, low.get(s, 0), high.get(s, 0)) for s in sorted({*low, *high}, reverse=True)])


def _holds_twice(t: Tensor) -> bool:
    """Whether two elements of a strided tensor lie at one place."""
    if t.is_contiguous():
        return False
    far, nested = 0, True
    for s, n in sorted(zip(t.stride(), t.shape)):
        if n > 1:
            nested = nested and s > far
            far += s * (n - 1)
    if nested or any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
        return not nested
    # the same sum of steps from indices that first differ at some axis
    steps = sorted(_steps(t), reverse=True)
    return any(_reaches(0, [(s, 1, n - 1), *((s2, 1 - n2, n2 - 1) for s2, n2 in steps[i + 1:])]) for i, (s, n) in enumerate(steps) if n > 1)


def _meet(out: Tuple[Tensor, Tensor], inputs: Tuple[Tensor, Tensor]) -> bool:
    """Whether the results share memory with each other or with an input; ranges of addresses first, which mostly are apart."""
    all_ = [(t, t.data_ptr(), _end(t)) for t in (*out, *inputs)]
    return any(begin < last and first < end and _overlap(t, x)
               for i, (t, begin, end) in enumerate(all_[:2]) for x, first, last in (all_[1:] if i == 0 else all_[2:]))


def _like(t: Tensor) -> Tensor:
    """A new contiguous tensor like ``t``, whose own strides may be a view's."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _check(name: str, t: Tensor, device: torch.device, dtype: torch.dtype, shape: tuple) -> None:
    if not isinstance(t, Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype != dtype:
        raise TypeError(f"{name}.dtype must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}: every tensor operand must be on {device}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")


def _check_first(name: str, t: Tensor, layout: str) -> None:
    if not isinstance(t, Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name}.dtype must be float32 or bfloat16, got {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} is on {t.device}: the token operators need GPU tensors")
    if t.dim() != 4 or t.numel() == 0:
        raise ValueError(f"{name} must be {layout} with every axis at least 1 long, got {tuple(t.shape)}")


def _wants_grad(*tensors: Optional[Tensor]) -> bool:
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("the token operators have no forward mode")
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# --- norms and rotation ---------------------------------------------------------------------------


def _rotary_args(q, k, q_out, k_out, w_q, w_k, rot, eps) -> bytes:
    """An ``hz_qk_norm_rotary``'s fields, those of an ``hz_qk_rotary`` where there are axes or no norms. ``q`` and ``k`` may be None in the
    reverse mode of a rotation alone; the shapes are then the cotangents'."""
    freqs, positions, axes, n_axes, interleaved, norm = rot
    B, N, H, D = q_out.shape
    none = (0, 0, 0, 0)
    one = _native.QK_NORM_ROTARY if norm and n_axes is None else _native.QK_ROTARY
    args = (*(none if q is None else _fields(q)), *(none if k is None else _fields(k)), *_fields(q_out), *_fields(k_out), _ptr(w_q),
            _ptr(w_k), _ptr(freqs), _ptr(positions), B, N, H, k_out.shape[2], D, 0 if freqs is None else freqs.shape[0], eps,
            interleaved, _DTYPES[q_out.dtype])
    return one.pack(*args) if one is _native.QK_NORM_ROTARY else one.pack(*args, _ptr(axes), n_axes or 1, norm)


def _rotary_fwd(q, k, w_q, w_k, rot, eps, out=None):
    q, k = _strided(q), _strided(k)
    q_out, k_out = out or (_like(q), _like(k))
    args = _rotary_args(q, k, q_out, k_out, w_q, w_k, rot, eps)
    lib = _native.lib()
    call = lib.hz_qk_norm_rotary_fwd if len(args) == _native.QK_NORM_ROTARY.size else lib.hz_qk_rotary_fwd
    with _on(q.device):
        _native.check(call(_stream(q.device), args))
    return q_out, k_out


class _QKNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, w_q, w_k, freqs, positions, axes, options):
        n_axes, interleaved, eps = options
        ctx.save_for_backward(q, k, w_q, w_k, freqs, positions, axes)
        ctx.options = options
        return _rotary_fwd(q, k, w_q, w_k, (freqs, positions, axes, n_axes, interleaved, True), eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, w_q, w_k, freqs, positions, axes = ctx.saved_tensors
        n_axes, interleaved, eps = ctx.options
        q, k, gq, gk = _strided(q), _strided(k), _strided(gq), _strided(gk)
        dev, D = q.device, q.shape[-1]
        dq, dk = _like(q), _like(k)
        dw_q = torch.empty(D, dtype=torch.float32, device=dev) if ctx.needs_input_grad[2] else None
        dw_k = torch.empty(D, dtype=torch.float32, device=dev) if ctx.needs_input_grad[3] else None
        args = _rotary_args(q, k, gq, gk, w_q, w_k, (freqs, positions, axes, n_axes, interleaved, True), eps)
        lib = _native.lib()
        call = lib.hz_qk_norm_rotary_bwd if len(args) == _native.QK_NORM_ROTARY.size else lib.hz_qk_rotary_bwd
        size = lib.hz_qk_norm_rotary_workspace(q.shape[0], q.shape[1], D)
        work = torch.empty(size, dtype=torch.uint8, device=dev)
        with _on(dev):
            _native.check(call(_stream(dev), args, _ptr(dq), _ptr(dk), _ptr(dw_q), _ptr(dw_k), _ptr(work), size))
        return dq, dk, dw_q, dw_k, None, None, None, None


class _QKRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, freqs, positions, axes, options):
        n_axes, interleaved = options
        ctx.save_for_backward(freqs, positions, axes)
        ctx.options = options
        return _rotary_fwd(q, k, None, None, (freqs, positions, axes, n_axes, interleaved, False), 0.0)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        n_axes, interleaved = ctx.options
        gq, gk = _strided(gq), _strided(gk)
        dev = gq.device
        dq, dk = _like(gq), _like(gk)
        args = _rotary_args(None, None, gq, gk, None, None, (*ctx.saved_tensors, n_axes, interleaved, False), 0.0)
        with _on(dev):
            _native.check(_native.lib().hz_qk_rotary_bwd(_stream(dev), args, _ptr(dq), _ptr(dk), 0, 0, 0, 0))
        return dq, dk, None, None, None, None


def _check_rotary(q, k, freqs, positions, axes):
    """Checks the operands that both rotations have; ``freqs, positions, axes, n_axes`` as the kernels take them (``n_axes`` None: positions
    of one axis)."""
    _check_first("q", q, "[B, N, H, D]")
    _check_first("k", k, "[B, N, Hk, D]")
    B, N, H, D = q.shape
    dev = q.device
    _check("k", k, dev, q.dtype, (B, N, k.shape[2], D))
    if D % 8 or D > MAX_ROTARY_HEAD_DIM:
        raise ValueError(f"head dimension must be a multiple of 8 up to {MAX_ROTARY_HEAD_DIM}, got {D}")
    if freqs is not None:
        if freqs.dim() != 1 or freqs.shape[0] % 4 or not 0 < 2 * freqs.shape[0] <= D:
            raise ValueError(f"freqs must hold a multiple of 4 frequencies, at most D / 2 = {D // 2}, got {tuple(freqs.shape)}")
        _check("freqs", freqs, dev, torch.float64, (freqs.shape[0],))
        if freqs.requires_grad and torch.is_grad_enabled():
            raise ValueError("freqs has no gradient here: detach it")
        freqs = freqs.contiguous()
    n_axes = None
    if axes is not None:
        if freqs is None or positions is None:
            raise ValueError("axes needs freqs and positions")
        if not isinstance(positions, Tensor) or positions.dim() != 3 or not 1 <= positions.shape[2] <= MAX_AXES:
            raise ValueError(f"positions must be [B, N, n_axes] with 1 to {MAX_AXES} axes where axes is given")
        n_axes = positions.shape[2]
        _check("axes", axes, dev, torch.int32, (freqs.shape[0],))
        axes = axes.contiguous()
    if positions is not None:
        _check("positions", positions, dev, torch.int32, (B, N) if n_axes is None else (B, N, n_axes))
        positions = positions.contiguous()
    return freqs, positions, axes, n_axes


def _check_rotary_out(out, q, k):
    for name, t, like in (("out[0]", out[0], q), ("out[1]", out[1], k)):
        _check(name, t, q.device, q.dtype, tuple(like.shape))
        if _strided(t) is not t:
            raise ValueError(f"{name} must have contiguous heads and 16-byte aligned rows, got strides {t.stride()}")
        if _holds_twice(t):
            raise ValueError(f"{name} must not hold one element at several places, got strides {t.stride()}")
    if _meet(out, (q, k)):
        raise ValueError("out must not overlap the inputs, nor one result the other")


def qk_norm_rotary(
    q: Tensor,
    k: Tensor,
    w_q: Optional[Tensor] = None,
    w_k: Optional[Tensor] = None,
    *,
    freqs: Optional[Tensor] = None,
    positions: Optional[Tensor] = None,
    axes: Optional[Tensor] = None,
    interleaved: bool = False,
    eps: float = 1e-6,
    out: Optional[Tuple[Tensor, Tensor]] = None,
) -> Tuple[Tensor, Tensor]:
    """RMS-normalises each head of ``q [B, N, H, D]`` and ``k [B, N, Hk, D]`` (``x / sqrt(mean(x^2) +
    eps)``, times ``w_q`` / ``w_k`` ``[D]`` float32 when given) and rotates its first ``2 * len(freqs)``
    elements by the angles ``positions * freqs``.

    ``freqs`` float64, in radians a position (None: no rotation), its length a multiple of 4;
    ``positions [B, N]`` int32 (None: 0 .. N - 1). A pair is elements ``p`` and ``p + len(freqs)``, or ``2 p``
    and ``2 p + 1`` with ``interleaved``. Angles are formed in float64 and reduced to a turn there, so that far positions are as exact as near ones.
    D is a multiple of 8 up to 256.

    With ``axes`` (int32, as long as ``freqs``) positions have several axes, ``positions [B, N, n_axes]`` (row and column of a
    lattice site, layer, time; up to 16), and pair p turns by ``positions[..., axes[p]] * freqs[p]``; a pair whose number is no axis
    stays as it is.

    Returns the two results, new tensors or ``out``: strided views of the same shapes that do not overlap
    the inputs or each other (a cache's rows, say), for calls that need no gradient. What is written there counts as
    changed in place: the backward of an earlier call that saved it raises."""
    freqs, positions, axes, n_axes = _check_rotary(q, k, freqs, positions, axes)
    D, dev = q.shape[3], q.device
    for name, w in (("w_q", w_q), ("w_k", w_k)):
        if w is not None:
            _check(name, w, dev, torch.float32, (D,))
    cw_q, cw_k = (None if w is None else w.contiguous() for w in (w_q, w_k))
    if out is not None:
        _check_rotary_out(out, q, k)
    if _wants_grad(q, k, w_q, w_k, freqs, *(out or ())):
        if out is not None:
            raise ValueError("out= holds results without gradients: call under torch.no_grad()")
        return _QKNormRotary.apply(q, k, cw_q, cw_k, freqs, positions, axes, (n_axes, bool(interleaved), _float32(eps)))
    res = _rotary_fwd(q, k, cw_q, cw_k, (freqs, positions, axes, n_axes, bool(interleaved), True), _float32(eps), out)
    if out is not None:
        increment_version(res)  # as after an in-place write: a graph that saved what is overwritten says so
    return res


def qk_rotary(
    q: Tensor,
    k: Tensor,
    *,
    freqs: Tensor,
    positions: Optional[Tensor] = None,
    axes: Optional[Tensor] = None,
    interleaved: bool = False,
    out: Optional[Tuple[Tensor, Tensor]] = None,
) -> Tuple[Tensor, Tensor]:
    """The rotation of :func:`qk_norm_rotary` without its norms: the first ``2 * len(freqs)`` elements of each head of ``q [B, N,
    H, D]`` and ``k [B, N, Hk, D]`` by the angles ``positions * freqs``, or with ``axes`` by ``positions[..., axes[p]] *
    freqs[p]``. Arguments, ``out`` and errors as there. (Its gradient is the rotation back: no input is kept for it.)"""
    if not isinstance(freqs, Tensor):
        raise TypeError(f"freqs must be a tensor, got {type(freqs).__name__}")
    freqs, positions, axes, n_axes = _check_rotary(q, k, freqs, positions, axes)
    if out is not None:
        _check_rotary_out(out, q, k)
    if _wants_grad(q, k, freqs, *(out or ())):
        if out is not None:
            raise ValueError("out= holds results without gradients: call under torch.no_grad()")
        return _QKRotary.apply(q, k, freqs, positions, axes, (n_axes, bool(interleaved)))
    res = _rotary_fwd(q, k, None, None, (freqs, positions, axes, n_axes, bool(interleaved), False), 0.0, out)
    if out is not None:
        increment_version(res)
    return res


# --- attention ------------------------------------------------------------------------------------


def _attention_args(q, k, v, out, out_low, lse, opts) -> bytes:
    slopes, prefix, documents, kv_len, scale, softcap, causal = opts
    B, Nq, H, D = q.shape
    return _native.TOKEN_ATTENTION.pack(
        *_fields(q), *_fields(k), *_fields(v), out.data_ptr(), _ptr(out_low), _ptr(lse), _ptr(slopes), _ptr(prefix),
        _ptr(documents), _ptr(kv_len), B, Nq, k.shape[1], H, k.shape[2], D, scale, softcap, causal, _DTYPES[q.dtype])


def token_attention_fwd(q: Tensor, k: Tensor, v: Tensor, opts: tuple,
                        for_backward: bool) -> Tuple[Tensor, Optional[Tensor], Optional[Tensor]]:
    """The forward call with checked operands: ``(out, out_low, lse)``, the last two what the reverse pass
    needs besides (``out_low``, what the rounding of ``out`` left out, for bfloat16 only)."""
    q, k, v = _strided(q), _strided(k), _strided(v)
    dev = q.device
    out = _like(q)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=dev) if for_backward else None
    out_low = torch.empty_like(out) if for_backward and q.dtype == torch.bfloat16 else None
    args = _attention_args(q, k, v, out, out_low, lse, opts)
    lib = _native.lib()
    with _on(dev):
        size = lib.hz_token_attention_fwd_workspace(args)
        work = torch.empty(size, dtype=torch.uint8, device=dev) if size > 0 else None
        _native.check(lib.hz_token_attention_fwd(_stream(dev), args, _ptr(work), size))
    return out, out_low, lse


class _TokenAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, opts):
        out, out_low, lse = token_attention_fwd(q, k, v, opts, True)
        ctx.save_for_backward(q, k, v, out, out_low, lse, *opts[:4])
        ctx.options = opts[4:]
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, out_low, lse, *tables = ctx.saved_tensors
        q, k, v, dout = _strided(q), _strided(k), _strided(v), _strided(dout)
        dev = q.device
        dq, dk, dv = _like(q), _like(k), _like(v)
        args = _attention_args(q, k, v, out, out_low, lse, (*tables, *ctx.options))
        lib = _native.lib()
        with _on(dev):
            size = lib.hz_token_attention_bwd_workspace(args)
            work = torch.empty(size, dtype=torch.uint8, device=dev)
            _native.check(lib.hz_token_attention_bwd(_stream(dev), args, _native.TOKEN_TENSOR.pack(*_fields(dout)),
                                                     _ptr(dq), _ptr(dk), _ptr(dv), _ptr(work), size))
        return dq, dk, dv, None


def token_attention(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    *,
    scale: Optional[float] = None,
    softcap: float = 0.0,
    slopes: Optional[Tensor] = None,
    causal: bool = False,
    prefix: Optional[Tensor] = None,
    documents: Optional[Tensor] = None,
    kv_len: Optional[Tensor] = None,
) -> Tensor:
    """Attention of ``q [B, Nq, H, D]`` over ``k, v [B, Nk, Hk, D]``; query head h uses key head
    ``h // (H // Hk)``. Returns ``out`` shaped as ``q``.

    Row b holds ``kv_len[b]`` keys (int32 ``[B]``; None: Nk), and its queries are the last tokens:
    query i stands at position ``p = kv_len[b] - Nq + i``. With ``scale`` (None: ``D ** -0.5``)::

        s_ij = softcap * tanh(scale q_i.k_j / softcap) - slopes[h] |p_i - j|

    without the cap where ``softcap`` is 0 and without the distance bias where ``slopes`` (float32 ``[H]``,
    no gradient) is None. Key j is seen if ``j < kv_len[b]``, and with ``causal`` if ``j <= p_i`` or
    ``j < prefix[b]`` (int32 ``[B]``), and with ``documents`` (int32 ``[B, Nk]``, negative: padding) if it and
    position p_i are of the same document. A query that sees nothing gets zeros and no gradient;
    keys behind ``kv_len`` and padding are never used, whatever they hold. D is a multiple of 8 up to 128,
    ``softcap`` at most 8192 for bfloat16.

    For single tokens ``k`` and ``v`` are the caches (strided views are read in place) and the new token's
    key and value are already in them."""
    _check_first("q", q, "[B, Nq, H, D]")
    _check_first("k", k, "[B, Nk, Hk, D]")
    B, Nq, H, D = q.shape
    Nk, Hk = k.shape[1], k.shape[2]
    dev = q.device
    if D % 8 or D > MAX_HEAD_DIM:
        raise ValueError(f"head dimension must be a multiple of 8 up to {MAX_HEAD_DIM}, got {D}")
    _check("k", k, dev, q.dtype, (B, Nk, Hk, D))
    _check("v", v, dev, q.dtype, (B, Nk, Hk, D))
    if H % Hk:
        raise ValueError(f"the query heads must be a multiple of the key heads, got {H} and {Hk}")
    if slopes is not None:
        _check("slopes", slopes, dev, torch.float32, (H,))
        if slopes.requires_grad and torch.is_grad_enabled():
            raise ValueError("slopes has no gradient here: detach it")
        slopes = slopes.contiguous()
    if prefix is not None:
        if not causal:
            raise ValueError("prefix needs causal=True")
        _check("prefix", prefix, dev, torch.int32, (B,))
        prefix = prefix.contiguous()
    if documents is not None:
        _check("documents", documents, dev, torch.int32, (B, Nk))
        documents = documents.contiguous()
    if kv_len is not None:
        _check("kv_len", kv_len, dev, torch.int32, (B,))
        kv_len = kv_len.contiguous()
    opts = (slopes, prefix, documents, kv_len, float(D) ** -0.5 if scale is None else _float32(scale), _float32(softcap),
            bool(causal))
    if _wants_grad(q, k, v, slopes):
        return _TokenAttention.apply(q, k, v, opts)
    return token_attention_fwd(q, k, v, opts, False)[0]


# --- relative position bias -----------------------------------------------------------------------


def relative_buckets(n_buckets: int, max_distance: int, *, bidirectional: bool = True, device=None) -> Tensor:
    """Bucket of each distance ``-max_distance .. max_distance`` (key position minus query position) as int32
    ``[2 max_distance + 1]``: with n buckets for a direction, the distances below n // 2 have one each and the
    others share the rest, evenly in their logarithm, up to ``max_distance``; distances beyond it are
    clamped to it. ``bidirectional`` gives half of the buckets to keys behind the query; otherwise those
    share the bucket of distance 0. The borders are exact (integer powers are compared, not logarithms)."""
    if not 1 <= n_buckets <= MAX_BUCKETS or (bidirectional and n_buckets % 2):
        raise ValueError(f"n_buckets must be in [1, {MAX_BUCKETS}], and even for two directions, got {n_buckets}")
    if not 0 <= max_distance <= MAX_BUCKET_RANGE:
        raise ValueError(f"max_distance must be in [0, {MAX_BUCKET_RANGE}], got {max_distance}")
    n = n_buckets // 2 if bidirectional else n_buckets
    near = n // 2
    span = n - near
    if near and max_distance > near:
        # the first distance of wide bucket t: d^span near^t >= max_distance^t near^span
        borders, d = [], near
        for t in range(1, span):
            while d**span * near**t < max_distance**t * near**span:
                d += 1
            borders.append(d)
    else:
        borders = []
    side, t = [], 0
    for d in range(max_distance + 1):
        while t < len(borders) and d >= borders[t]:
            t += 1
        side.append(d if d < near else min(near + t, n - 1))
    behind = [n + x for x in side] if bidirectional else [side[0]] * len(side)
    return torch.tensor(side[:0:-1] + side[:1] + behind[1:], dtype=torch.int32, device=device)


def _bias_call(table, e, buckets, q_positions, k_positions, qkh, R, nb, H, backward):
    B, Nq = q_positions.shape
    sizes = (B, Nq, k_positions.shape[1], H, nb, R, _DTYPES[e.dtype], _native.HZ_FLAG_E_QKH if qkh else 0)
    dev = e.device
    lib = _native.lib()
    with _on(dev):
        if not backward:
            _native.check(lib.hz_bucket_bias_fwd(_stream(dev), _ptr(table), _ptr(buckets), _ptr(q_positions),
                                                 _ptr(k_positions), _ptr(e), *sizes))
            return
        size = lib.hz_bucket_bias_workspace(*sizes[:5], *sizes[6:])
        work = torch.empty(size, dtype=torch.uint8, device=dev)
        _native.check(lib.hz_bucket_bias_bwd(_stream(dev), _ptr(e), _ptr(buckets), _ptr(q_positions), _ptr(k_positions),
                                             _ptr(table), _ptr(work), size, *sizes))


def _bias_fwd(table, buckets, q_positions, k_positions, qkh, dtype):
    (B, Nq), Nk, (nb, H) = q_positions.shape, k_positions.shape[1], table.shape
    e = torch.empty((B, Nq, Nk, H) if qkh else (B, Nq, H, Nk), dtype=dtype, device=table.device)
    _bias_call(table, e, buckets, q_positions, k_positions, qkh, buckets.shape[0] // 2, nb, H, False)
    return e


class _BucketBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, buckets, q_positions, k_positions, qkh, dtype):
        ctx.save_for_backward(buckets, q_positions, k_positions)
        ctx.options = (qkh, tuple(table.shape))
        return _bias_fwd(table, buckets, q_positions, k_positions, qkh, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, de):
        buckets, q_positions, k_positions = ctx.saved_tensors
        qkh, (nb, H) = ctx.options
        de = de.contiguous()
        if de.data_ptr() % 16:
            de = de.clone()
        dtable = torch.empty((nb, H), dtype=torch.float32, device=de.device)
        _bias_call(dtable, de, buckets, q_positions, k_positions, qkh, buckets.shape[0] // 2, nb, H, True)
        return dtable, None, None, None, None, None


def bucket_bias(
    table: Tensor,
    buckets: Tensor,
    q_positions: Tensor,
    k_positions: Tensor,
    *,
    e_layout: str = "qhk",
    dtype: torch.dtype = torch.float32,
) -> Tensor:
    """Learned relative position bias: ``table[buckets[R + clamp(k - q, -R, R)], h]`` for every query
    position ``q_positions [B, Nq]`` and key position ``k_positions [B, Nk]`` (int32), ``table [n_buckets,
    H]`` float32 and ``buckets [2 R + 1]`` int32 (:func:`relative_buckets`; a number that is no row of the
    table gives a zero bias). Returns ``e`` in ``dtype`` as ``[B, Nq, H, Nk]`` (``"qhk"``, what ``mhsea_ad``
    takes as ``e``) or ``[B, Nq, Nk, H]`` (``"qkh"``, also the rectangular attention's bias). The gradient
    goes to ``table``."""
    if not isinstance(table, Tensor) or not table.is_cuda:
        raise ValueError("bucket_bias needs GPU tensors")
    if table.dim() != 2 or not 1 <= table.shape[0] <= MAX_BUCKETS or not 1 <= table.shape[1] <= 256:
        raise ValueError(f"table must be [n_buckets, H] with at most {MAX_BUCKETS} buckets and 256 heads, got {tuple(table.shape)}")
    if e_layout not in ("qhk", "qkh"):
        raise ValueError(f"e_layout must be 'qhk' or 'qkh', got {e_layout!r}")
    if dtype not in _DTYPES:
        raise TypeError(f"dtype must be float32 or bfloat16, got {dtype}")
    dev = table.device
    _check("table", table, dev, torch.float32, tuple(table.shape))
    for name, t in (("q_positions", q_positions), ("k_positions", k_positions)):
        if not isinstance(t, Tensor) or t.dim() != 2 or 0 in t.shape:
            raise ValueError(f"{name} must be [B, N] with both axes at least 1 long")
    B = q_positions.shape[0]
    _check("q_positions", q_positions, dev, torch.int32, tuple(q_positions.shape))
    _check("k_positions", k_positions, dev, torch.int32, (B, k_positions.shape[1]))
    if not isinstance(buckets, Tensor) or buckets.dim() != 1 or buckets.shape[0] % 2 != 1 or buckets.shape[0] > 2 * MAX_BUCKET_RANGE + 1:
        raise ValueError(f"buckets must be [2 R + 1] with R at most {MAX_BUCKET_RANGE}")
    _check("buckets", buckets, dev, torch.int32, tuple(buckets.shape))
    args = (table.contiguous(), buckets.contiguous(), q_positions.contiguous(), k_positions.contiguous(),
            e_layout == "qkh", dtype)
    if _wants_grad(table):
        return _BucketBias.apply(*args)
    return _bias_fwd(*args)


__all__ = ["bucket_bias", "qk_norm_rotary", "qk_rotary", "relative_buckets", "token_attention"]

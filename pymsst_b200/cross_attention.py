"""Attention over states of another length, and rotary positions with several axes.

:func:`cross_attention` is :class:`~pymsst_b200.fused.AttentionFn` for
queries and keys of different lengths: padded key batches, key / value heads
shared by groups of query heads, dropout on the probabilities from
counter-based bits (:mod:`pymsst_b200.dropout`), any number of queries down
to one.  :func:`rotary_axes` is the rotary embedding for tokens that carry
several positions (frame, band, channel).
"""
from __future__ import annotations

import ctypes
from typing import Sequence

import torch
from torch.autograd.function import once_differentiable

from . import _native as nat
from .dropout import check_key, drop_threshold, needs_function, on_device

MAX_HEAD_DIM = 256


def _plane_empty(b, h, n, d, dtype, device) -> torch.Tensor:
    """[b, h, n, d] view of a new [b, n, h, d] plane."""
    return torch.empty_strided((b, h, n, d), (n * h * d, d, h * d, 1), dtype=dtype, device=device)


def _copy_plane(t: torch.Tensor) -> torch.Tensor:
    """A copy of t [b, h, n, d], always a new one, as a view of a [b, n, h, d] plane."""
    return t.transpose(1, 2).clone(memory_format=torch.contiguous_format).transpose(1, 2)


def _plane(t: torch.Tensor) -> torch.Tensor:
    """t itself when the kernels read it in place, else a copy in a [b, n, h, d] plane.  They need contiguous head
    elements and, for the tensor cores (16-bit types, head dims in multiples of 8), 16-byte aligned rows at positive
    strides; the stride of a dimension of one does not count."""
    b, h, n, d = t.shape
    sb, sh, sn, sd = t.stride()
    ok = sd == 1 or d == 1
    if ok and t.element_size() == 2 and d % 8 == 0:
        ok = (t.data_ptr() % 16 == 0 and (b < 2 or (sb > 0 and sb % 8 == 0)) and (h < 2 or (sh > 0 and sh % 8 == 0))
              and (n < 2 or (sn > 0 and sn % 8 == 0)))
    return t if ok else _copy_plane(t)


_I64x12, _I64x24 = ctypes.c_int64 * 12, ctypes.c_int64 * 24


def _strides(*planes: torch.Tensor):
    out: list[int] = []
    for t in planes:
        sb, sh, sn, _ = t.stride()
        out += (sb, sn, sh)
    return (_I64x12 if len(out) == 12 else _I64x24)(*out)


# ------------------------------------------------------------------- attention
def _attention_forward(q, k, v, lengths, scale, threshold, key, site):
    b, hq, nq, d = q.shape
    hk, nk = k.shape[1], k.shape[2]
    device = q.device
    o = _plane_empty(b, hq, nq, d, q.dtype, device)
    code = nat.dtype_code(q.dtype)
    lib = nat.library()
    lse = torch.empty(lib.pmb_cross_attention_lse_size(b, hq, nq), dtype=torch.float32, device=device)
    ws_bytes = lib.pmb_cross_attention_forward_workspace_size(b, hq, hk, nq, nk, d, code)
    ws = nat.workspace(ws_bytes, device) if ws_bytes else None
    with on_device(device):
        nat.call(
            "pmb_cross_attention_forward", q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(),
            nat.ptr(lengths), b, hq, hk, nq, nk, d, _strides(q, k, v, o), scale, threshold, nat.ptr(key), site, code,
            nat.ptr(ws), ws_bytes, nat.stream_handle(device),
        )
    return o, lse


class CrossAttentionFn(torch.autograd.Function):
    """dropout(softmax(scale q k^T)) v over each batch item's keys; saves q, k, v, o and the fp32 row sums, no
    probabilities and no mask."""

    @staticmethod
    def forward(ctx, q, k, v, lengths, scale, threshold, key, site):
        o, lse = _attention_forward(q, k, v, lengths, scale, threshold, key, site)
        ctx.meta = (scale, threshold, site)
        ctx.save_for_backward(q, k, v, o, lse, lengths, key)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, o, lse, lengths, key = ctx.saved_tensors
        scale, threshold, site = ctx.meta
        b, hq, nq, d = q.shape
        hk, nk = k.shape[1], k.shape[2]
        device = q.device
        grad = _plane(grad)
        dq = _plane_empty(b, hq, nq, d, q.dtype, device)
        dk, dv = (_plane_empty(b, hk, nk, d, q.dtype, device) for _ in range(2))
        code = nat.dtype_code(q.dtype)
        ws_bytes = int(nat.library().pmb_cross_attention_backward_workspace_size(b, hq, hk, nq, nk, d, code))
        ws = nat.workspace(ws_bytes, device)
        with on_device(device):
            nat.call(
                "pmb_cross_attention_backward", q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                grad.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), nat.ptr(lengths), b, hq,
                hk, nq, nk, d, _strides(q, k, v, o, grad, dq, dk, dv), scale, threshold, nat.ptr(key), site, code,
                ws.data_ptr(), ws_bytes, nat.stream_handle(device),
            )
        return dq, dk, dv, None, None, None, None, None


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, key_lengths: torch.Tensor | None = None,
                    scale: float | None = None, dropout_p: float = 0.0, key: torch.Tensor | None = None,
                    site: int = 0) -> torch.Tensor:
    """dropout(softmax(scale q k^T)) v for q [b, heads, nq, d] and k, v [b, kv_heads, nk, d] (any strides), heads a
    multiple of kv_heads (query head h reads key / value head h // (heads // kv_heads)), d up to 256; ``scale``
    defaults to d ** -0.5.  fp32, bf16 and fp16.  Returns [b, heads, nq, d], a view of a [b, nq, heads, d] plane.

    ``key_lengths`` (int32 or int64 [b], values clamped to [0, nk]): each batch item's keys are its first ones; what
    lies behind them is never used and gets a zero gradient.  Rows without keys, or with scores of -infinity alone, give
    zeros and no gradient; NaN in a row's live scores makes the row NaN.  ``dropout_p`` needs a ``key`` of :class:`~pymsst_b200.dropout.DropoutGenerator`; ``site`` as in :func:`~pymsst_b200.dropout.dropout`.
    Forward and backward are deterministic."""
    name = "cross_attention"
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
        raise ValueError(f"{name}: q, k, v must be [b, heads, n, d] with k and v alike, got {tuple(q.shape)}, "
                         f"{tuple(k.shape)} and {tuple(v.shape)}")
    b, hq, _, d = q.shape
    if k.shape[0] != b or k.shape[3] != d or k.shape[1] == 0 or hq % k.shape[1]:
        raise ValueError(f"{name}: q {tuple(q.shape)} and k {tuple(k.shape)} do not fit (same batch and head dim, "
                         "heads a multiple of the key / value heads)")
    nk = k.shape[2]
    if not 0 < d <= MAX_HEAD_DIM:
        raise ValueError(f"{name}: head dim must be in [1, {MAX_HEAD_DIM}], got {d}")
    if not q.dtype == k.dtype == v.dtype:
        raise TypeError(f"{name}: q, k, v must have one type, got {q.dtype}, {k.dtype} and {v.dtype}")
    nat.dtype_code(q.dtype)
    if key_lengths is not None:
        if key_lengths.shape != (b,) or key_lengths.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{name}: key_lengths must be int32 or int64 [{b}], got {key_lengths.dtype} "
                             f"{tuple(key_lengths.shape)}")
    threshold = drop_threshold(dropout_p)
    check_key(key, threshold, site, q.device, name)
    nat.require_cuda(q, k, v, key_lengths, name=name)
    if key_lengths is not None:
        if key_lengths.dtype == torch.int64:
            key_lengths = key_lengths.clamp(0, nk).to(torch.int32)
        key_lengths = key_lengths.contiguous()
    scale = float(d) ** -0.5 if scale is None else float(scale)
    q, k, v = _plane(q), _plane(k), _plane(v)
    if needs_function(q, k, v):
        return CrossAttentionFn.apply(q, k, v, key_lengths, scale, threshold, key, site)
    return _attention_forward(q, k, v, key_lengths, scale, threshold, key, site)[0]


# ---------------------------------------------------------------------- rotary
_POSITION_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
MAX_AXES = 4


def _pair_view(t: torch.Tensor) -> torch.Tensor:
    """t itself when pairs of head elements can be read whole, else a copy in a [b, n, h, d] plane."""
    strides = [s for s, size in zip(t.stride()[:3], t.shape[:3]) if size > 1]
    if t.stride(-1) != 1 or any(s % 2 for s in strides) or t.data_ptr() % (2 * t.element_size()):
        t = _copy_plane(t)
    return t


def _rotary_strides(*views: torch.Tensor):
    out: list[int] = []
    for t in views:
        b, h, n, _ = t.shape
        sb, sh, sn, _ = t.stride()
        out += (sb if b > 1 else 0, sn if n > 1 else 0, sh if h > 1 else 0)
    return nat.i64_array(out)


def _rotary(t, positions, freqs, sections, inverse):
    t = _pair_view(t)
    b, h, n, d = t.shape
    device = t.device
    y = _plane_empty(b, h, n, d, t.dtype, device)
    axes = len(sections)
    with on_device(device):
        nat.call(
            "pmb_rotary_axes", t.data_ptr(), positions.data_ptr(), freqs.data_ptr(), y.data_ptr(), b, n, h, d,
            _rotary_strides(t, y), n * axes if positions.dim() == 3 else 0, _POSITION_TYPES[positions.dtype], axes,
            nat.i64_array(sections), inverse, nat.dtype_code(t.dtype), nat.stream_handle(device),
        )
    return y


class RotaryAxesFn(torch.autograd.Function):
    """Rotation by the tokens' angles; saves positions and frequencies, the backward rotates back."""

    @staticmethod
    def forward(ctx, t, positions, freqs, sections):
        ctx.sections = sections
        ctx.save_for_backward(positions, freqs)
        return _rotary(t, positions, freqs, sections, 0)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        positions, freqs = ctx.saved_tensors
        return _rotary(grad, positions, freqs, ctx.sections, 1), None, None, None


def rotary_axes(t: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, sections: Sequence[int]) -> torch.Tensor:
    """Rotary embedding of t [b, heads, n, d] (any strides, d even) whose tokens have one position per axis:
    ``positions`` [b, n, axes] or, shared by the batch, [n, axes] (int32, int64 or float32).  ``sections`` gives the
    pairs of each axis in order (1 to 4 axes), ``freqs`` (fp32, their sum) the frequency of every pair:
    (t[2p], t[2p + 1]) turns by position * freq, interleaved pairs as in the rest of the package; pairs behind the
    sections are left alone.  Angles are formed in fp64, so far positions keep their accuracy.  fp32, bf16 and fp16.
    Returns [b, heads, n, d], a view of a [b, n, heads, d] plane.  Query and key heads of one token grid are rotated
    in one call by giving them as one tensor.  Positions and frequencies get no gradient."""
    name = "rotary_axes"
    if t.dim() != 4 or t.shape[-1] % 2 or t.shape[-1] == 0:
        raise ValueError(f"{name}: t must be [b, heads, n, d] with an even d, got {tuple(t.shape)}")
    nat.dtype_code(t.dtype)
    b, _, n, d = t.shape
    sections = tuple(int(s) for s in sections)
    axes = len(sections)
    if not 1 <= axes <= MAX_AXES or min(sections) <= 0 or sum(sections) > d // 2:
        raise ValueError(f"{name}: 1 to {MAX_AXES} positive sections of at most {d // 2} pairs together, got "
                         f"{sections}")
    if tuple(positions.shape) not in ((b, n, axes), (n, axes)) or positions.dtype not in _POSITION_TYPES:
        raise ValueError(f"{name}: positions must be int32, int64 or float32 [{b}, {n}, {axes}] or [{n}, {axes}], got "
                         f"{positions.dtype} {tuple(positions.shape)}")
    if freqs.dtype != torch.float32 or tuple(freqs.shape) != (sum(sections),):
        raise ValueError(f"{name}: freqs must be float32 [{sum(sections)}], got {freqs.dtype} {tuple(freqs.shape)}")
    if torch.is_grad_enabled() and (freqs.requires_grad or positions.requires_grad):
        raise ValueError(f"{name}: positions and freqs get no gradient; detach them")
    nat.require_cuda(t, positions, freqs, name=name)
    positions, freqs = positions.contiguous(), freqs.contiguous()
    if needs_function(t, positions, freqs):
        return RotaryAxesFn.apply(t, positions, freqs, sections)
    return _rotary(t, positions, freqs, sections, 0)

"""Dropout from counter-based random bits, on the sm_100a kernels.

A mask is a pure function of a key (seed, step), a site number and the
element's index, so none is stored: the backward and a recomputed forward
(activation checkpointing) draw the same mask from the same key, inside a
captured CUDA graph too.  :class:`DropoutGenerator` hands out one key per
forward; sites tell apart the places of a model that share it.

The bits are Philox4x32 with seven rounds, 16 per element; the layout is
given in ``include/pymsst_b200.h``.  A probability is met to 2^-17: elements
whose bits are below ``round(65536 p)`` are dropped and the others scaled by
the exact inverse of the resulting keep probability.

Role in the model: nn.Dropout and nn.GELU + nn.Dropout of pymss-core's
Attention and FeedForward, which the reference trains unchanged
(src/pymsst/training/module.py:221-224).
"""
from __future__ import annotations

import contextlib

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native as nat

_NO_GUARD = contextlib.nullcontext()
_MAX_SITE = 2**32

# Generator states whose addresses captured graphs hold: every replay reads and writes them, so they must not go back
# to the allocator when the generator does.
_captured_states: list[torch.Tensor] = []


def on_device(device: torch.device):
    """Context in which launches go to ``device`` (nothing to do when it is the current one)."""
    return _NO_GUARD if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def needs_function(*tensors: torch.Tensor | None) -> bool:
    """Whether a call has to go through its autograd Function: an input needs a gradient, or carries a forward-mode
    tangent, which the Function refuses (the kernel alone would leave it out)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    if getattr(forward_ad, "_current_level", 0) < 0:  # no dual level is open (1.5 us less than asking every tensor)
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def drop_threshold(p: float) -> int:
    """round(65536 p): the 16-bit numbers below it drop their element."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must be in [0, 1], got {p}")
    return int(round(p * 65536))


def check_key(key, threshold: int, site: int, device: torch.device, name: str) -> None:
    """Raise unless (key, site) can drive a dropout of this threshold on ``device``."""
    if not 0 <= site < _MAX_SITE:
        raise ValueError(f"{name}: site must be in [0, 2^32), got {site}")
    if threshold == 0:
        return
    if key is None:
        raise ValueError(f"{name}: a dropout probability above 0 needs a key (DropoutGenerator.next_key())")
    if key.dtype != torch.int64 or key.numel() != 2 or not key.is_contiguous():
        raise ValueError(f"{name}: key must be two contiguous int64 (seed, step), got {key.dtype} {tuple(key.shape)}")
    if key.device != device:
        raise ValueError(f"{name}: key is on {key.device}, the tensors on {device}")


class DropoutGenerator:
    """Source of dropout keys: ``state`` holds (seed, step) on the device, :meth:`next_key` returns a copy of it and
    moves the step on, in one kernel.  Captured into a CUDA graph, every replay draws new masks; the steps go on
    where the last replay or eager call left them.  The graph keeps to the generator it was captured with, whose
    state then stays allocated for good: a model that is given another one has to be captured again (Trainer does)."""

    def __init__(self, seed: int = 0, device: torch.device | str | None = None):
        if device is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.state = torch.tensor([_as_int64(seed), 0], dtype=torch.int64, device=device)

    def next_key(self) -> torch.Tensor:
        """int64 [2] (seed, step) for one forward."""
        device = nat.require_cuda(self.state, name="DropoutGenerator")
        key = torch.empty_like(self.state)
        with on_device(device):
            if torch.cuda.is_current_stream_capturing() and not any(t is self.state for t in _captured_states):
                _captured_states.append(self.state)
            nat.call("pmb_dropout_next_key", self.state.data_ptr(), key.data_ptr(), nat.stream_handle(device))
        torch.autograd.graph.increment_version(self.state)  # a backward that saved the state itself now raises
        return key

    def manual_seed(self, seed: int, step: int = 0) -> None:
        """Set seed and step in place (a captured graph reads the same state)."""
        self.state.copy_(torch.tensor([_as_int64(seed), _as_int64(step)], dtype=torch.int64))

    def state_dict(self) -> dict:
        seed, step = self.state.tolist()
        return {"seed": seed, "step": step}

    def load_state_dict(self, state: dict) -> None:
        self.manual_seed(state["seed"], state["step"])


def _as_int64(value: int) -> int:
    value = int(value) & (2**64 - 1)
    return value - 2**64 if value >= 2**63 else value


def _dropout(x, residual, threshold, key, site):
    device = x.device
    x = x.contiguous()
    y = torch.empty_like(x)
    if residual is not None:
        residual = residual.contiguous()
    with on_device(device):
        nat.call("pmb_dropout", x.data_ptr(), nat.ptr(residual), y.data_ptr(), x.numel(), threshold, nat.ptr(key),
                 site, nat.dtype_code(x.dtype), nat.stream_handle(device))
    return y


class DropoutFn(torch.autograd.Function):
    """residual + drop(x), or drop(x); saves the key alone."""

    @staticmethod
    def forward(ctx, x, residual, threshold, key, site):
        ctx.threshold, ctx.site = threshold, site
        ctx.save_for_backward(key)
        return _dropout(x, residual, threshold, key, site)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (key,) = ctx.saved_tensors
        gx = None
        if ctx.needs_input_grad[0]:
            gx = _dropout(grad, None, ctx.threshold, key, ctx.site)
        return gx, grad if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x: torch.Tensor, p: float, key: torch.Tensor | None = None, site: int = 0,
            residual: torch.Tensor | None = None) -> torch.Tensor:
    """``residual + drop(x)``, or ``drop(x)``: each element is zeroed with probability ``p`` and scaled by the inverse
    of the keep probability otherwise.  ``residual`` has x's shape and type.  fp32, bf16 and fp16; one rounding.
    Elements are numbered in row-major order of x's shape, whatever its strides.  The key must not be changed in
    place before the backward (:meth:`DropoutGenerator.next_key` returns a new one each time)."""
    threshold = drop_threshold(p)
    check_key(key, threshold, site, x.device, "dropout")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"dropout: residual must be {tuple(x.shape)} {x.dtype}, got {tuple(residual.shape)} "
                         f"{residual.dtype}")
    nat.require_cuda(x, residual, name="dropout")
    nat.dtype_code(x.dtype)
    if needs_function(x, residual):
        return DropoutFn.apply(x, residual, threshold, key, site)
    return _dropout(x, residual, threshold, key, site)


def _gelu_dropout(x, threshold, key, site):
    device = x.device
    y = torch.empty_like(x)
    with on_device(device):
        nat.call("pmb_gelu_dropout_forward", x.data_ptr(), y.data_ptr(), x.numel(), threshold, nat.ptr(key), site,
                 nat.dtype_code(x.dtype), nat.stream_handle(device))
    return y


class GeluDropoutFn(torch.autograd.Function):
    """drop(gelu(x)); saves x and the key."""

    @staticmethod
    def forward(ctx, x, threshold, key, site):
        x = x.contiguous()
        ctx.threshold, ctx.site = threshold, site
        ctx.save_for_backward(x, key)
        return _gelu_dropout(x, threshold, key, site)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, key = ctx.saved_tensors
        grad = grad.contiguous()
        gx = torch.empty_like(x)
        device = x.device
        with on_device(device):
            nat.call("pmb_gelu_dropout_backward", grad.data_ptr(), x.data_ptr(), gx.data_ptr(), x.numel(),
                     ctx.threshold, nat.ptr(key), ctx.site, nat.dtype_code(x.dtype), nat.stream_handle(device))
        return gx, None, None, None


def gelu_dropout(x: torch.Tensor, p: float, key: torch.Tensor | None = None, site: int = 0) -> torch.Tensor:
    """``drop(gelu(x))`` (the exact erf form), the feed-forward's activation with its dropout in one pass each way.
    fp32, bf16 and fp16; see :func:`dropout` for the key."""
    threshold = drop_threshold(p)
    check_key(key, threshold, site, x.device, "gelu_dropout")
    nat.require_cuda(x, name="gelu_dropout")
    nat.dtype_code(x.dtype)
    if needs_function(x):
        return GeluDropoutFn.apply(x, threshold, key, site)
    return _gelu_dropout(x.contiguous(), threshold, key, site)

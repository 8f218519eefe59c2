"""Dropout from a counter-based generator on the sm_100a kernels.

``dropout(x, p, rng, residual)`` is ``residual + keep * x / (1 - p)``.  Whether element
i (in row-major order) is kept is a function of the seed, the offset and i alone, so
the mask is never stored: the backward pass makes it again.  The same numbers give the
same mask on every call, device and launch shape.

``rng`` holds (seed, offset): an int64 tensor on x's device, which a training step
captured in a CUDA graph advances on the device (``rng[1] += 1``), or two Python
integers.  The backward pass uses the values that the forward read, whatever has become
of the tensor since.  For Monte Carlo dropout at inference call it as in training.

``layer`` is added to the seed, so the layers of a model take masks of their own from one
``rng``.  Layer i + 1 under seed s therefore has the mask of layer i under seed s + 1:
seeds that are to be independent (ranks of a data-parallel job, samples of Monte Carlo
dropout) have to lie further apart than the layers do, as ``base + rank * 2**32`` does, or
to differ in the offset.

The rate is ``round(65536 p) / 65536``: one 16-bit random word decides about an
element, and the scale is made from that rate.
"""

from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable
from torch.library import custom_op

from . import _native as nat
from .norm import DTYPES

_NS = "mednext_accel_b200"
_LOW63, _BIT63 = (1 << 63) - 1, 1 << 63


def _signed(v: int) -> int:
    """v modulo 2^64 as a signed 64-bit integer."""
    return (v & _LOW63) - (v & _BIT63)


def _launch(x: Tensor, residual: Tensor | None, rng: Tensor | None, seed: int, offset: int, drop: int,
            used: Tensor | None) -> Tensor:
    y = torch.empty_like(x)
    nat.launch("mednext_dropout", x, x.data_ptr(), nat.ptr(residual), y.data_ptr(), nat.ptr(rng),
               seed & (_LOW63 | _BIT63), offset & (_LOW63 | _BIT63), nat.ptr(used), x.numel(), drop,
               nat.dtype_code(x.dtype))
    return y


@custom_op(f"{_NS}::dropout_forward", mutates_args=())
def dropout_forward(x: Tensor, residual: Tensor | None, rng: Tensor | None, seed: int, offset: int,
                    drop: int) -> tuple[Tensor, Tensor]:
    """(y, the [seed, offset] that was used) of a contiguous x."""
    nat.require_device(x)
    used = torch.empty(2, dtype=torch.int64, device=x.device)
    return _launch(x, residual, rng, seed, offset, drop, used), used


@dropout_forward.register_fake
def _(x, residual, rng, seed, offset, drop):
    return torch.empty_like(x), x.new_empty(2, dtype=torch.int64)


@custom_op(f"{_NS}::dropout_backward", mutates_args=())
def dropout_backward(dy: Tensor, used: Tensor, drop: int) -> Tensor:
    nat.require_device(dy)
    return _launch(dy, None, used, 0, 0, drop, None)


@dropout_backward.register_fake
def _(dy, used, drop):
    return torch.empty_like(dy)


def _setup(ctx, inputs, output):
    ctx.save_for_backward(output[1])
    ctx.drop = inputs[5]
    ctx.mark_non_differentiable(output[1])
    ctx.set_materialize_grads(False)


def _op_backward(ctx, dy, _dused):
    if dy is None:
        return None, None, None, None, None, None
    need = ctx.needs_input_grad
    dx = dropout_backward(dy.contiguous(), ctx.saved_tensors[0], ctx.drop) if need[0] else None
    return dx, dy if need[1] else None, None, None, None, None


dropout_forward.register_autograd(_op_backward, setup_context=_setup)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, rng, seed, offset, drop):
        used = torch.empty(2, dtype=torch.int64, device=x.device) if rng is not None else None
        y = _launch(x, residual, rng, seed, offset, drop, used)
        ctx.save_for_backward(used)
        ctx.state = (seed, offset, drop)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need = ctx.needs_input_grad
        dx = None
        if need[0]:
            used = ctx.saved_tensors[0]
            seed, offset, drop = ctx.state
            if used is not None:
                seed = offset = 0  # used holds the sums already
            dx = _launch(dy.contiguous(), None, used, seed, offset, drop, None)
        return dx, dy if need[1] else None, None, None, None, None


def dropout(x: Tensor, p: float, rng: Tensor | tuple[int, int], residual: Tensor | None = None,
            layer: int = 0) -> Tensor:
    """Drop elements of ``x`` with probability ``p``, scale the others by 1 / (1 - p), and add
    ``residual``; see the module's notes for ``rng`` and ``layer``.

    x: float32, bfloat16 or float16 on an sm_100 device; residual: x's shape and type.
    A dropped element contributes 0 whatever x holds there.  The result is contiguous;
    tensors that are not are copied first.  Differentiable once in x and residual."""
    if not x.is_cuda:
        raise ValueError("dropout requires CUDA tensors")
    if x.dtype not in DTYPES:
        raise ValueError("dropout requires a float16, bfloat16 or float32 input")
    if not 0.0 <= p <= 1.0:
        raise ValueError("dropout requires a probability between 0 and 1")
    state = None
    if isinstance(rng, Tensor):
        if (rng.dtype != torch.int64 or rng.ndim != 1 or rng.shape[0] != 2 or rng.get_device() != x.get_device()
                or not rng.is_contiguous()):
            raise ValueError("dropout requires rng as a contiguous int64 tensor [seed, offset] on the input's device")
        state, seed, offset = rng, layer, 0
    else:
        if not (isinstance(rng, (tuple, list)) and len(rng) == 2 and all(isinstance(v, int) for v in rng)):
            raise ValueError("dropout requires rng as an int64 tensor or two integers (seed, offset)")
        seed, offset = rng[0] + layer, rng[1]
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device:
            raise ValueError("dropout requires a residual of the input's shape, type and device")
        if not residual.is_contiguous():
            residual = residual.contiguous()
    nat.require_device(x)
    drop = round(p * 65536)
    if not x.is_contiguous():
        x = x.contiguous()
    seed, offset = _signed(seed), _signed(offset)
    if torch.compiler.is_compiling():
        return dropout_forward(x, residual, state, seed, offset, drop)[0]
    if (x.requires_grad or (residual is not None and residual.requires_grad)) and torch.is_grad_enabled():
        return _Dropout.apply(x, residual, state, seed, offset, drop)
    return _launch(x, residual, state, seed, offset, drop, None)

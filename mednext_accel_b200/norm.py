"""Layer norm over one axis on the sm_100a kernels, with its backward pass.

``layer_norm(x, weight, bias, eps, dim)`` normalises every token's ``x.shape[dim]``
values.  ``dim=-1`` is ``F.layer_norm`` over the last axis; ``dim=1`` on an
[N, C, *spatial] tensor normalises the channels of each voxel where they lie, with no
transposed copy.  :class:`LayerNorm3d` is the layer for NCDHW features.

Statistics and sums are fp32 for every input type, each output is rounded once, and
the results (the weight and bias gradients among them) are the same bits from call to
call.  Like GroupNorm's statistics here, each token's mean and reciprocal deviation are
kept for the backward pass (8 bytes a token).

Calls outside ``torch.compile`` go straight to the library, through an autograd
function where a gradient is wanted; inside it they are the ops
``mednext_accel_b200::layer_norm_forward`` / ``layer_norm_backward``.  The direct
route keeps a small call short: a ``custom_op`` call that records a gradient costs
about 18 us on the host, the autograd function's 6 us.
"""

from __future__ import annotations

import math
from functools import lru_cache

import torch
from torch import Tensor, nn
from torch.autograd.function import once_differentiable
from torch.library import custom_op

from . import _native as nat

_NS = "mednext_accel_b200"
CHANNELS_MOST = 16384  # of the channels-first kernels
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def dense_order(x: Tensor) -> list[int] | None:
    """The order of the axes in which ``x`` is contiguous memory, or None.

    A channels-last volume or a transposed matrix is dense in another order than its
    own; the operators here then run on that order instead of on a copy."""
    order = sorted(range(x.ndim), key=lambda i: x.stride(i), reverse=True)
    return order if x.permute(order).is_contiguous() else None


def in_dense_order(x: Tensor, dim: int) -> tuple[Tensor, int, list[int] | None]:
    """(contiguous tensor of x's values, where ``dim`` went, the inverse permutation
    or None): a view where x is dense in some order of its axes, else a copy."""
    if x.is_contiguous():
        return x, dim, None
    order = dense_order(x)
    if order is None:
        return x.contiguous(), dim, None
    inverse = [order.index(i) for i in range(x.ndim)]
    return x.permute(order), inverse[dim], inverse


def axis_sizes(x: Tensor, dim: int) -> tuple[int, int, int]:
    """A contiguous x's shape as (outer, size of dim, inner)."""
    c, inner = x.shape[dim], x.stride(dim)
    if c < 2 or x.numel() == 0:  # the stride of such an axis may be anything
        return math.prod(x.shape[:dim]), c, math.prod(x.shape[dim + 1:])
    return x.numel() // (c * inner), c, inner


def _param_code(x: Tensor, weight: Tensor | None, bias: Tensor | None) -> int:
    p = weight if weight is not None else bias
    return nat.dtype_code(p.dtype) if p is not None else 0


def _forward(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float, dim: int,
             want_stats: bool) -> tuple[Tensor, Tensor | None]:
    outer, c, inner = axis_sizes(x, dim)
    y = torch.empty_like(x)
    stats = x.new_empty((outer * inner, 2), dtype=torch.float32) if want_stats else None
    nat.launch("mednext_ln_fwd", x, x.data_ptr(), nat.ptr(weight), nat.ptr(bias), y.data_ptr(), nat.ptr(stats),
               outer, c, inner, eps, nat.dtype_code(x.dtype), _param_code(x, weight, bias))
    return y, stats


@lru_cache(maxsize=1024)
def _workspace_size(outer: int, c: int, inner: int, code: int) -> int:
    return nat.load().mednext_ln_bwd_workspace_size(outer, c, inner, code)


def _backward(dy: Tensor, x: Tensor, stats: Tensor, weight: Tensor | None, bias: Tensor | None, dim: int,
              want_params: bool) -> tuple[Tensor, Tensor | None, Tensor | None]:
    outer, c, inner = axis_sizes(x, dim)
    code = nat.dtype_code(x.dtype)
    dx = torch.empty_like(x)
    dw = torch.empty_like(weight) if want_params and weight is not None else None
    db = torch.empty_like(bias) if want_params and bias is not None else None
    ws, nbytes = None, 0
    if dw is not None or db is not None:
        nbytes = _workspace_size(outer, c, inner, code)
        ws = stats.new_empty(nbytes // 4) if nbytes else None  # floats
    nat.launch("mednext_ln_bwd", x, dy.data_ptr(), x.data_ptr(), stats.data_ptr(), nat.ptr(weight), dx.data_ptr(),
               nat.ptr(dw), nat.ptr(db), nat.ptr(ws), nbytes, outer, c, inner, code, _param_code(x, weight, bias))
    return dx, dw, db


@custom_op(f"{_NS}::layer_norm_forward", mutates_args=())
def layer_norm_forward(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float,
                       dim: int) -> tuple[Tensor, Tensor]:
    """(y, stats [tokens, 2] fp32) of a contiguous x."""
    nat.require_device(x)
    return _forward(x, weight, bias, eps, dim, True)


@layer_norm_forward.register_fake
def _(x, weight, bias, eps, dim):
    return torch.empty_like(x), x.new_empty((x.numel() // x.shape[dim], 2), dtype=torch.float32)


@custom_op(f"{_NS}::layer_norm_backward", mutates_args=())
def layer_norm_backward(dy: Tensor, x: Tensor, stats: Tensor, weight: Tensor | None, bias: Tensor | None,
                        dim: int) -> tuple[Tensor, Tensor, Tensor]:
    """(dx, dweight, dbias); the gradient of an absent parameter is empty."""
    nat.require_device(x)
    dx, dw, db = _backward(dy, x, stats, weight, bias, dim, True)
    return dx, x.new_empty(0) if dw is None else dw, x.new_empty(0) if db is None else db


@layer_norm_backward.register_fake
def _(dy, x, stats, weight, bias, dim):
    return (torch.empty_like(x), x.new_empty(0) if weight is None else torch.empty_like(weight),
            x.new_empty(0) if bias is None else torch.empty_like(bias))


def _setup(ctx, inputs, output):
    x, weight, bias, _eps, dim = inputs
    ctx.save_for_backward(x, output[1], weight, bias)
    ctx.dim = dim
    ctx.mark_non_differentiable(output[1])
    ctx.set_materialize_grads(False)


def _op_backward(ctx, dy, _dstats):
    if dy is None:
        return None, None, None, None, None
    x, stats, weight, bias = ctx.saved_tensors
    dx, dw, db = layer_norm_backward(dy.contiguous(), x, stats, weight, bias, ctx.dim)
    need = ctx.needs_input_grad
    return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None, None, None)


layer_norm_forward.register_autograd(_op_backward, setup_context=_setup)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, dim):
        y, stats = _forward(x, weight, bias, eps, dim, True)
        ctx.save_for_backward(x, stats, weight, bias)
        ctx.dim = dim
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, stats, weight, bias = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = _backward(dy.contiguous(), x, stats, weight, bias, ctx.dim, need[1] or need[2])
        return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None, None, None)


def layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, eps: float = 1e-6,
               dim: int = -1) -> Tensor:
    """Layer norm of ``x`` over ``dim``: (x - mean) / sqrt(var + eps) * weight + bias.

    x: float32, bfloat16 or float16 on an sm_100 device, in any strides (a tensor that is
    dense in another order of its axes, as channels-last, keeps that order); weight and
    bias: [x.shape[dim]], float32 or x's type, or None.  Differentiable once in x,
    weight and bias.  The computation runs in x's type, not autocast's."""
    if not x.is_cuda:
        raise ValueError("layer_norm requires CUDA tensors")
    dtype, ndim, index = x.dtype, x.ndim, x.get_device()
    if dtype not in DTYPES:
        raise ValueError("layer_norm requires a float16, bfloat16 or float32 input")
    if not -ndim <= dim < ndim:
        raise ValueError(f"layer_norm: dim {dim} is out of range for a tensor of {ndim} dimensions")
    if dim < 0:
        dim += ndim
    size = x.shape[dim]
    if size == 0:
        raise ValueError("layer_norm requires a nonempty normalised dimension")
    grad = x.requires_grad
    if weight is not None:
        weight = _check_param("weight", weight, size, dtype, index)
        grad = grad or weight.requires_grad
    if bias is not None:
        bias = _check_param("bias", bias, size, dtype, index)
        grad = grad or bias.requires_grad
        if weight is not None and weight.dtype != bias.dtype:
            raise ValueError("layer_norm requires weight and bias of one type")
    if not 0.0 < eps < math.inf:
        raise ValueError("layer_norm requires eps to be finite and positive")
    nat.require_device(x)
    inverse = None
    if not x.is_contiguous():
        x, dim, inverse = in_dense_order(x, dim)
    if size > CHANNELS_MOST and x.stride(dim) > 1:  # past the channels-first kernels: as rows, by copies
        y = layer_norm(x.movedim(dim, -1).contiguous(), weight, bias, eps).movedim(-1, dim).contiguous()
        return y if inverse is None else y.permute(inverse)
    if torch.compiler.is_compiling():
        y = layer_norm_forward(x, weight, bias, float(eps), dim)[0]
    elif grad and torch.is_grad_enabled():
        y = _LayerNorm.apply(x, weight, bias, float(eps), dim)
    else:
        y = _forward(x, weight, bias, float(eps), dim, False)[0]
    return y if inverse is None else y.permute(inverse)


def _check_param(name: str, p: Tensor, size: int, dtype: torch.dtype, index: int) -> Tensor:
    if not p.is_cuda or p.get_device() != index:
        raise ValueError(f"layer_norm requires {name} on the input's device")
    if p.ndim != 1 or p.shape[0] != size:
        raise ValueError(f"layer_norm requires {name} with shape ({size},)")
    if p.dtype != torch.float32 and p.dtype != dtype:
        raise ValueError(f"layer_norm requires a float32 {name}, or one of the input's type")
    return p if p.is_contiguous() else p.contiguous()


class LayerNorm3d(nn.Module):
    """Layer norm over the channels of [N, C, D, H, W] (or [N, C, *spatial]) features."""

    def __init__(self, channels: int, eps: float = 1e-6, bias: bool = True) -> None:
        super().__init__()
        if channels <= 0:
            raise ValueError("channels must be positive")
        if not (math.isfinite(eps) and eps > 0):
            raise ValueError("eps must be finite and positive")
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(channels))
        self.bias = nn.Parameter(torch.zeros(channels)) if bias else None

    def forward(self, x: Tensor) -> Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps, dim=1)

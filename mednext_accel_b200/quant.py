"""Products in 8-bit integers for serving: one scale per token, one per output channel.

``quantize_int8(w)`` lays the rows of a weight matrix out once; ``int8_linear(x, q,
scale, bias, dim)`` quantises the activations token by token on the way and
multiplies.  ``dim=1`` on [N, K, *spatial] is a 1x1x1 convolution, which
:class:`Int8Pointwise3d` serves in place of an ``nn.Conv3d``.

The integer sums are exact; scales, their products and the bias are fp32 with one
rounding to x's type.  Inference only: there is no gradient.
"""

from __future__ import annotations

from functools import lru_cache

import torch
from torch import Tensor, nn
from torch.library import custom_op

from . import _native as nat
from .norm import DTYPES, axis_sizes, in_dense_order

_NS = "mednext_accel_b200"
MAX_K = 131072  # 127 * 127 * K stays inside a signed 32-bit sum


def _check_input(what: str, x: Tensor, dim: int) -> int:
    if not x.is_cuda:
        raise ValueError(f"{what} requires CUDA tensors")
    if x.dtype not in DTYPES:
        raise ValueError(f"{what} requires a float16, bfloat16 or float32 input")
    ndim = x.ndim
    if not -ndim <= dim < ndim:
        raise ValueError(f"{what}: dim {dim} is out of range for a tensor of {ndim} dimensions")
    if not 0 < x.shape[dim] <= MAX_K:
        raise ValueError(f"{what} requires 1 to {MAX_K} values per token")
    return dim if dim >= 0 else dim + ndim


def quantize_int8(x: Tensor, dim: int = -1) -> tuple[Tensor, Tensor]:
    """x's tokens along ``dim`` as 8-bit rows, and their scales.

    Returns (q [tokens, K] int8, scale [tokens] float32) with the tokens in row-major
    order of x's other axes: q = rint(x 127 / m), scale = m / 127, m = max |x| (at
    least 127 * 2^-126).  q's rows start 16 bytes apart at a multiple of 16, as
    :func:`int8_linear` takes weights."""
    dim = _check_input("quantize_int8", x, dim)
    nat.require_device(x)
    x = x.detach().contiguous()
    outer, k, inner = axis_sizes(x, dim)
    pitch = (k + 15) // 16 * 16
    q = torch.empty((outer * inner, pitch), dtype=torch.int8, device=x.device)
    scale = torch.empty((outer * inner,), dtype=torch.float32, device=x.device)
    nat.launch("mednext_int8_quantize", x, x.data_ptr(), q.data_ptr(), scale.data_ptr(), outer, k, inner, pitch,
               nat.dtype_code(x.dtype))
    return q[:, :k], scale


@lru_cache(maxsize=1024)
def _workspace_size(outer: int, k: int, inner: int, n: int, code: int) -> int:
    return nat.load().mednext_int8_linear_workspace_size(outer, k, inner, n, code)


def _launch(x: Tensor, weight: Tensor, scale: Tensor, bias: Tensor | None, dim: int) -> Tensor:
    outer, k, inner = axis_sizes(x, dim)
    n, code = weight.shape[0], nat.dtype_code(x.dtype)
    pitch, at = weight.stride(0), weight.data_ptr()
    if pitch % 16 or at % 16 or pitch < k or weight.stride(1) != 1:
        pitch = (k + 15) // 16 * 16
        held = weight.new_empty((n, pitch))
        held[:, :k] = weight
        weight, at = held, held.data_ptr()
    y = x.new_empty((*x.shape[:dim], n, *x.shape[dim + 1:]))
    nbytes = _workspace_size(outer, k, inner, n, code)
    ws = weight.new_empty(nbytes) if nbytes else None  # bytes, like the weight
    nat.launch("mednext_int8_linear", x, x.data_ptr(), at, scale.data_ptr(),
               None if bias is None else bias.data_ptr(), y.data_ptr(), None if ws is None else ws.data_ptr(), nbytes,
               outer, k, inner, n, pitch, code)
    return y


@custom_op(f"{_NS}::int8_linear", mutates_args=())
def int8_linear_op(x: Tensor, weight: Tensor, scale: Tensor, bias: Tensor | None, dim: int) -> Tensor:
    """The product of a contiguous x."""
    nat.require_device(x)
    return _launch(x, weight, scale, bias, dim)


@int8_linear_op.register_fake
def _(x, weight, scale, bias, dim):
    return x.new_empty((*x.shape[:dim], weight.shape[0], *x.shape[dim + 1:]))


def int8_linear(x: Tensor, weight: Tensor, scale: Tensor, bias: Tensor | None = None, dim: int = -1) -> Tensor:
    """x quantised token by token, times an 8-bit weight: x's shape with N along ``dim``.

    x: float32, bfloat16 or float16 on an sm_100 device, any strides, K values along
    ``dim``; weight: [N, K] int8 and scale: [N] float32 as :func:`quantize_int8` gives
    them for a float weight's rows (rows whose start is not a multiple of 16 bytes are
    copied on every call); bias: [N] float32 or None."""
    dim = _check_input("int8_linear", x, dim)
    if ((x.requires_grad or scale.requires_grad or (bias is not None and bias.requires_grad))
            and torch.is_grad_enabled()):
        raise ValueError("int8_linear has no gradient: call it under torch.no_grad(), on detached tensors")
    k = x.shape[dim]
    if weight.dtype != torch.int8 or weight.ndim != 2 or weight.shape[1] != k or weight.shape[0] == 0:
        raise ValueError(f"int8_linear requires an int8 weight with shape (N, {k})")
    n = weight.shape[0]
    if scale.dtype != torch.float32 or scale.shape != (n,):
        raise ValueError(f"int8_linear requires a float32 scale with shape ({n},)")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (n,)):
        raise ValueError(f"int8_linear requires a float32 bias with shape ({n},)")
    index = x.get_device()  # -1 for a CPU tensor
    if weight.get_device() != index or scale.get_device() != index or (bias is not None and bias.get_device() != index):
        raise ValueError("int8_linear requires all tensors on the same CUDA device")
    nat.require_device(x)
    if not scale.is_contiguous():
        scale = scale.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    inverse = None
    if not x.is_contiguous():
        x, dim, inverse = in_dense_order(x, dim)
    y = int8_linear_op(x, weight, scale, bias, dim) if torch.compiler.is_compiling() else _launch(
        x, weight, scale, bias, dim)
    return y if inverse is None else y.permute(inverse)


class Int8Pointwise3d(nn.Module):
    """An ``nn.Conv3d`` with a 1x1x1 kernel, served in 8-bit integers.

    Its 8-bit rows, float32 scales and float32 bias keep their types and values when the
    module, or a model that holds it, is cast (``.half()``, ``.to(dtype)``): the products
    take x in any of its types and these as they are."""

    def __init__(self, conv: nn.Conv3d) -> None:
        super().__init__()
        transposed = getattr(conv, "transposed", False)  # its weight would be [in, out]
        if (transposed or conv.groups != 1 or set(conv.kernel_size) != {1} or set(conv.stride) != {1}
                or (conv.padding not in ("same", "valid") and set(conv.padding) != {0})):
            raise ValueError("Int8Pointwise3d requires a dense 1x1x1 convolution of stride 1 without padding, not transposed")
        q, scale = quantize_int8(conv.weight.reshape(conv.out_channels, conv.in_channels))
        # the padded rows are the buffer: a slice's row pitch would not survive a state dict
        self.in_channels = conv.in_channels
        pitch = q.stride(0)
        self.register_buffer("weight", q.as_strided((conv.out_channels, pitch), (pitch, 1)))
        self.register_buffer("scale", scale)
        self.register_buffer("bias", None if conv.bias is None else conv.bias.detach().float().clone())

    def _apply(self, fn, recurse=True):
        held = dict(self._buffers)
        super()._apply(fn, recurse)
        for name, t in held.items():
            now = self._buffers[name]
            if t is not None and now.dtype != t.dtype:
                self._buffers[name] = t.to(now.device)
        return self

    def forward(self, x: Tensor) -> Tensor:
        return int8_linear(x, self.weight[:, : self.in_channels], self.scale, self.bias, dim=1)

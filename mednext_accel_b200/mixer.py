"""A channel mixer on the sm_100a operators: the expansion branch of a block over the channels
of each voxel, with layer norm in front and dropout behind it.

    y = x + dropout(project(gelu(expand(layer_norm(x)))))

Training runs the layer norm, the tensor-core pointwise products of the block (16-bit
contiguous features; others take torch's convolutions), torch's GELU and the counter-based
dropout, whose residual add is the branch's; :meth:`ChannelMixer3d.int8` gives the serving
form, whose two products run in 8-bit integers.  No reference
counterpart: the reference's blocks normalise each channel over the volume and have no
dropout.
"""

from __future__ import annotations

import copy

import torch
from torch import Tensor, nn
from torch.nn import functional as F

from .drop import dropout
from .norm import LayerNorm3d
from .pointwise import pointwise_conv3d
from .quant import Int8Pointwise3d


def _pointwise(x: Tensor, conv: nn.Conv3d) -> Tensor:
    if x.is_cuda and x.dtype in (torch.bfloat16, torch.float16) and x.is_contiguous():
        bias = None if conv.bias is None else conv.bias.to(x.dtype)
        return pointwise_conv3d(x, conv.weight.to(x.dtype), bias)
    return F.conv3d(x, conv.weight.to(x.dtype), None if conv.bias is None else conv.bias.to(x.dtype))


class ChannelMixer3d(nn.Module):
    """``forward(x, rng)``: x [N, C, D, H, W] in float32, bfloat16 or float16, ``rng`` the
    [seed, offset] tensor of :func:`dropout`, needed while training with ``p > 0``.  ``layer``
    tells the mixers of one model apart in their masks; seeds of independent models lie further
    apart than their layers.

    The branch runs in x's type and the result has it.  Under autocast the convolutions of
    float32 or non-contiguous features, which are torch's, run in autocast's type."""

    def __init__(self, channels: int, expansion_ratio: int, p: float = 0.0, layer: int = 0) -> None:
        super().__init__()
        if channels <= 0 or expansion_ratio <= 0:
            raise ValueError("channels and expansion_ratio must be positive")
        if not 0.0 <= p <= 1.0:
            raise ValueError("p must be a probability")
        self.p = p
        self.layer = layer
        self.norm = LayerNorm3d(channels)
        self.expand = nn.Conv3d(channels, channels * expansion_ratio, kernel_size=1)
        self.project = nn.Conv3d(channels * expansion_ratio, channels, kernel_size=1)

    def forward(self, x: Tensor, rng: Tensor | tuple[int, int] | None = None) -> Tensor:
        y = _pointwise(F.gelu(_pointwise(self.norm(x), self.expand)), self.project).to(x.dtype)
        if not self.training or self.p == 0.0:
            return x + y
        if rng is None:
            raise ValueError("ChannelMixer3d requires rng while training with dropout")
        return dropout(y, self.p, rng, residual=x, layer=self.layer)

    def int8(self) -> Int8ChannelMixer3d:
        """The serving form of the mixer as it is now: its weights are quantised, its norm is
        copied, and neither form follows what becomes of the other."""
        return Int8ChannelMixer3d(self)


class Int8ChannelMixer3d(nn.Module):
    """:class:`ChannelMixer3d` for inference, its products in 8-bit integers."""

    def __init__(self, mixer: ChannelMixer3d) -> None:
        super().__init__()
        self.norm = copy.deepcopy(mixer.norm).requires_grad_(False)
        self.expand = Int8Pointwise3d(mixer.expand)
        self.project = Int8Pointwise3d(mixer.project)

    @torch.no_grad()
    def forward(self, x: Tensor) -> Tensor:
        return x + self.project(F.gelu(self.expand(self.norm(x))))

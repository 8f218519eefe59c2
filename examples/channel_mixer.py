"""Train a small stack of channel mixers in one CUDA graph, then serve it in 8-bit integers.

    python examples/channel_mixer.py [--steps N] [--size S]

Voxels of a synthetic volume are classified from 32 features each.  The training step
(layer norm, tensor-core pointwise products, dropout from a counter-based generator,
cross-entropy, AdamW) is captured once and replayed; the generator's offset advances on the
device, so every replay drops other elements.  The trained mixers are then quantised and
their predictions compared with the 16-bit ones.
"""

from __future__ import annotations

import argparse
import copy
import sys
from pathlib import Path

import torch
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import mednext_accel_b200 as mx  # noqa: E402


class MixerNet(nn.Module):
    def __init__(self, channels: int = 32, classes: int = 3, depth: int = 2, p: float = 0.1) -> None:
        super().__init__()
        self.mixers = nn.ModuleList(mx.ChannelMixer3d(channels, 2, p, layer=i) for i in range(depth))
        self.head = nn.Conv3d(channels, classes, kernel_size=1)

    def forward(self, x: torch.Tensor, rng: torch.Tensor | None = None) -> torch.Tensor:
        for mixer in self.mixers:
            x = mixer(x) if isinstance(mixer, mx.Int8ChannelMixer3d) else mixer(x, rng)
        return torch.nn.functional.conv3d(x, self.head.weight.to(x.dtype), self.head.bias.to(x.dtype))

    def int8(self) -> MixerNet:
        served = MixerNet(depth=0)
        served.head = copy.deepcopy(self.head).requires_grad_(False)
        served.mixers = nn.ModuleList(mixer.int8() for mixer in self.mixers)
        return served.eval()


def synthetic(size: int, device: str = "cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """Features [1, 32, S, S, S] (bf16) and the class that a fixed random map gives them."""
    gen = torch.Generator(device=device).manual_seed(0)
    x = torch.randn((1, 32, size, size, size), generator=gen, device=device)
    mix = torch.randn((3, 32), generator=gen, device=device)
    target = torch.einsum("kc,ncdhw->nkdhw", mix, x.abs() - 0.8).argmax(1)
    return x.to(torch.bfloat16), target


def train(net: MixerNet, x: torch.Tensor, target: torch.Tensor, steps: int) -> list[float]:
    net.train()
    opt = torch.optim.AdamW(net.parameters(), lr=1e-2, capturable=True)
    rng = torch.tensor([1234, 0], device=x.device)  # seed, offset

    def step() -> torch.Tensor:
        opt.zero_grad(set_to_none=True)
        loss = mx.cross_entropy(net(x, rng), target)
        loss.backward()
        opt.step()
        rng[1] += 1
        return loss.detach()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        losses = [float(step()) for _ in range(3)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            loss = step()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(steps):
        graph.replay()
        losses.append(float(loss))
    return losses


@torch.no_grad()
def compare(net: MixerNet, x: torch.Tensor, target: torch.Tensor) -> tuple[float, float, float]:
    """(accuracy in 16 bits, accuracy in 8, share of voxels whose class agrees)."""
    net.eval()
    full, low = net(x).argmax(1), net.int8()(x).argmax(1)
    mean = lambda t: float(t.float().mean())  # noqa: E731
    return mean(full == target), mean(low == target), mean(full == low)


def main(argv: list[str] | None = None) -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--size", type=int, default=32)
    args = ap.parse_args(argv)
    torch.manual_seed(0)
    net = MixerNet().cuda()
    x, target = synthetic(args.size)
    losses = train(net, x, target, args.steps)
    full, low, same = compare(net, x, target)
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f}; accuracy bf16 {full:.3f}, int8 {low:.3f}; same class {same:.4f}")
    return 0


if __name__ == "__main__":
    sys.exit(main())

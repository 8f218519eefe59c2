"""The layer norm, dropout and 8-bit products together: the channel mixer against the same
computation in 64 bits, and the example that trains and serves it."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch
from torch.nn import functional as F

import mednext_accel_b200 as mx
from mednext_accel_b200 import _native as nat

from philox import dropout_words

pytestmark = pytest.mark.gpu


def reference(mixer, x, keep, p):
    """Forward in 64 bits; keep: the mask, None at inference."""
    w = {k: v.detach().double().requires_grad_() for k, v in mixer.named_parameters()}
    xd = x.detach().double().requires_grad_()
    y = F.layer_norm(xd.movedim(1, -1), (x.shape[1],), w["norm.weight"], w["norm.bias"], mixer.norm.eps).movedim(-1, 1)
    y = F.conv3d(F.gelu(F.conv3d(y, w["expand.weight"], w["expand.bias"])), w["project.weight"], w["project.bias"])
    if keep is not None:
        t = round(p * 65536)
        y = torch.where(keep, y * (65536 / (65536 - t)), 0.0)
    return xd + y, xd, w


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("dtype,tol", [(torch.bfloat16, 2e-2), (torch.float16, 4e-3), (torch.float32, 1e-5)])
@pytest.mark.parametrize("shape", [(1, 16, 8, 8, 16), (2, 24, 5, 6, 8)])
def test_training_matches_64_bits(shape, dtype, tol):
    """Each of the branch's tensors (norm, expand, GELU, project) is rounded once to its
    16-bit type, 2^-8 or 2^-11 each: relative L2 within 2e-2 as the block tests hold, a
    sixth of it for float16; float32 is torch's fp32 convolutions."""
    torch.manual_seed(0)
    mixer = mx.ChannelMixer3d(shape[1], 2, p=0.25, layer=3).cuda().train()
    x = torch.randn(shape, device="cuda").to(dtype)
    dy = torch.randn(shape, device="cuda").to(dtype)
    rng = torch.tensor([40, 2], device="cuda")
    xg = x.clone().requires_grad_()
    old = torch.backends.cudnn.allow_tf32
    torch.backends.cudnn.allow_tf32 = False
    try:
        y = mixer(xg, rng)
        grads = torch.autograd.grad(y, [xg, *mixer.parameters()], dy)
    finally:
        torch.backends.cudnn.allow_tf32 = old
    keep = torch.from_numpy(dropout_words(43, 2, 0, x.numel()) >= round(0.25 * 65536)).cuda().view(shape)
    want, xd, w = reference(mixer, x, keep, 0.25)
    want_grads = torch.autograd.grad(want, [xd, *w.values()], dy.double())
    assert rel(y, want) <= tol
    for (name, _), got, ref in zip([("x", None), *mixer.named_parameters()], grads, want_grads, strict=True):
        assert rel(got, ref) <= tol, name
    assert nat.device_error() == 0


def test_serving_form_is_near_the_trained_one():
    """Two products with factors within 1/254 of their token's or channel's largest value."""
    torch.manual_seed(1)
    mixer = mx.ChannelMixer3d(32, 4, p=0.1).cuda().eval()
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.randn((1, 32, 8, 12, 16), device="cuda").to(dtype)
        served = mixer.int8().eval()
        with torch.no_grad():
            branch = mixer(x).float() - x.float()
            low = served(x).float() - x.float()
        assert served(x).dtype == dtype
        assert rel(low, branch) <= 0.03


def test_dropout_needs_its_numbers():
    mixer = mx.ChannelMixer3d(8, 2, p=0.5).cuda().train()
    x = torch.randn((1, 8, 4, 4, 4), device="cuda")
    with pytest.raises(ValueError, match="rng"):
        mixer(x)
    mixer.eval()
    assert mixer(x).shape == x.shape
    with pytest.raises(ValueError, match="probability"):
        mx.ChannelMixer3d(8, 2, p=1.5)


def test_example_trains_and_serves():
    path = Path(__file__).resolve().parents[1] / "examples" / "channel_mixer.py"
    spec = importlib.util.spec_from_file_location("channel_mixer_example", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    torch.manual_seed(0)
    net = example.MixerNet().cuda()
    x, target = example.synthetic(16)
    losses = example.train(net, x, target, 40)
    assert losses[-1] < 0.8 * losses[0]
    full, low, same = example.compare(net, x, target)
    assert full > 0.5 and same > 0.95 and abs(full - low) < 0.03


def step(module, x, lr=0.1):
    """One optimiser step that moves every parameter."""
    opt = torch.optim.SGD(module.parameters(), lr=lr)
    y = module(x)
    (y.float() * torch.linspace(-1, 1, y.numel(), device=y.device).view_as(y)).sum().backward()
    before = [p.detach().clone() for p in module.parameters()]
    opt.step()
    assert all(not torch.equal(p, q) for p, q in zip(before, module.parameters(), strict=True))


def test_served_mixer_does_not_follow_the_trained_one():
    torch.manual_seed(2)
    mixer = mx.ChannelMixer3d(16, 2).cuda()
    x = torch.randn((1, 16, 4, 6, 8), device="cuda").to(torch.bfloat16)
    served = mixer.int8()
    want = served(x)
    step(mixer, x)
    assert torch.equal(served(x), want)
    assert not torch.equal(mixer.int8()(x), want)


def test_trained_mixer_does_not_follow_the_served_one():
    mixer = mx.ChannelMixer3d(16, 2).cuda()
    x = torch.randn((1, 16, 4, 6, 8), device="cuda")
    step(mixer, x)  # parameters with gradients
    grads = [p.grad for p in mixer.parameters()]
    served = mixer.int8()
    assert not any(p.requires_grad or p.grad is not None for p in served.parameters())
    served.bfloat16()
    assert all(p.requires_grad and p.dtype == torch.float32 for p in mixer.parameters())
    assert all(p.grad is g for p, g in zip(mixer.parameters(), grads, strict=True))


def test_served_example_does_not_follow_the_trained_one():
    path = Path(__file__).resolve().parents[1] / "examples" / "channel_mixer.py"
    spec = importlib.util.spec_from_file_location("channel_mixer_example", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    net = example.MixerNet(p=0.0).cuda()
    x, _ = example.synthetic(8)
    served = net.int8()
    with torch.no_grad():
        want = served(x)
    step(net, x)
    with torch.no_grad():
        assert torch.equal(served(x), want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_served_mixer_can_be_cast(dtype):
    """The norm's parameters are rounded to the new type, up to 2^-8 each: rows within 2e-2 as above."""
    mixer = mx.ChannelMixer3d(32, 2).cuda()
    with torch.no_grad():
        mixer.norm.weight.uniform_(0.5, 1.5)
    x = torch.randn((1, 32, 4, 6, 8), device="cuda").to(dtype)
    served = mixer.int8()
    want = served(x).float() - x.float()
    served.to(dtype)
    assert served.norm.weight.dtype == dtype
    assert rel(served(x).float() - x.float(), want) <= 2e-2


def test_training_under_autocast_matches_64_bits():
    """float32 features under bfloat16 autocast: the products in bfloat16, tolerances as for it above; what
    dropout leaves out is exact."""
    torch.manual_seed(0)
    shape = (2, 24, 5, 6, 8)
    mixer = mx.ChannelMixer3d(shape[1], 2, p=0.25, layer=3).cuda().train()
    x, dy = (torch.randn(shape, device="cuda") for _ in range(2))
    xg = x.clone().requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = mixer(xg, torch.tensor([40, 2], device="cuda"))
    assert y.dtype == torch.float32
    grads = torch.autograd.grad(y, [xg, *mixer.parameters()], dy)
    keep = torch.from_numpy(dropout_words(43, 2, 0, x.numel()) >= round(0.25 * 65536)).cuda().view(shape)
    assert torch.equal(y[~keep], x[~keep])
    want, xd, w = reference(mixer, x, keep, 0.25)
    want_grads = torch.autograd.grad(want, [xd, *w.values()], dy.double())
    assert rel(y, want) <= 2e-2
    for (name, _), got, ref in zip([("x", None), *mixer.named_parameters()], grads, want_grads, strict=True):
        assert got.dtype == torch.float32 and rel(got, ref) <= 2e-2, name
    assert nat.device_error() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cast", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("memory_format", [torch.contiguous_format, torch.channels_last_3d])
def test_features_keep_their_type_under_autocast(dtype, cast, memory_format):
    torch.manual_seed(0)
    mixer = mx.ChannelMixer3d(16, 2, p=0.5).cuda()
    served = mixer.int8()
    x = torch.randn((2, 16, 4, 6, 8), device="cuda").to(dtype).contiguous(memory_format=memory_format)
    want, _, _ = reference(mixer, x, None, 0.5)
    with torch.autocast("cuda", dtype=cast):
        mixer.train()
        y = mixer(x, (1, 2))
        mixer.eval()
        z, low = mixer(x), served(x)
    assert y.dtype == z.dtype == low.dtype == dtype
    assert rel(z, want) <= 2e-2 and rel(low, want) <= 3e-2
    y.float().sum().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in mixer.parameters())

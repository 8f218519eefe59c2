"""Dropout on the sm_100a kernels.  Which elements are dropped is compared exactly with
Philox4x32-10 in numpy (itself pinned to its published answers in test_operators_host.py);
the values are one fp32 product, and one sum with a residual, rounded once: the same
bits as torch's own elementwise operations in fp32."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import mednext_accel_b200 as mx
from mednext_accel_b200 import _native as nat

from philox import dropout_words

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def kept(n, p, seed, offset, begin=0):
    return torch.from_numpy(dropout_words(seed, offset, begin, n) >= round(p * 65536)).cuda()


def want(x, keep, p, residual=None):
    t = round(p * 65536)
    scale = 0.0 if t == 65536 else 65536.0 / (65536 - t)
    y = torch.where(keep.view(x.shape), x.float() * scale, 0.0)
    return (y if residual is None else residual.float() + y).to(x.dtype)


def data(n, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(n, generator=gen, device="cuda").to(dtype) for _ in range(3)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 15, 16, 255, 2048, 2049, 100003, 1 << 20])
def test_mask_and_values(n, dtype):
    x, r, dy = data(n, dtype, n)
    for p, seed, offset in ((0.1, 1, 0), (0.5, 2**63 - 1, 2**40 + 3), (0.3, -5, 7)):
        keep = kept(n, p, seed, offset)
        for rng in ((seed, offset), torch.tensor([seed, offset], device="cuda")):
            assert torch.equal(mx.dropout(x, p, rng), want(x, keep, p))
            assert torch.equal(mx.dropout(x, p, rng, residual=r), want(x, keep, p, r))
            xg, rg = x.clone().requires_grad_(), r.clone().requires_grad_()
            y = mx.dropout(xg, p, rng, residual=rg)
            assert torch.equal(y, want(x, keep, p, r))
            dx, dr = torch.autograd.grad(y, (xg, rg), dy)
            assert torch.equal(dx, want(dy, keep, p)) and torch.equal(dr, dy)
    assert nat.device_error() == 0


def test_the_same_for_every_type_and_layer_adds_to_the_seed():
    x = torch.ones(5000, device="cuda")
    y = mx.dropout(x, 0.4, (11, 3), layer=2)
    assert torch.equal(y, mx.dropout(x, 0.4, (13, 3)))
    assert torch.equal(y, mx.dropout(x, 0.4, torch.tensor([11, 3], device="cuda"), layer=2))
    for dtype in DTYPES:
        assert torch.equal(y != 0, mx.dropout(x.to(dtype), 0.4, (13, 3)) != 0)
    assert torch.equal(mx.dropout(x, 0.4, (2**63 - 1, 0), layer=1), mx.dropout(x, 0.4, (-(2**63), 0)))
    assert torch.equal(mx.dropout(x, 0.4, torch.tensor([2**63 - 1, 0], device="cuda"), layer=1),
                       mx.dropout(x, 0.4, (-(2**63), 0)))
    assert not torch.equal(y, mx.dropout(x, 0.4, (13, 4))) and not torch.equal(y, mx.dropout(x, 0.4, (14, 3)))


def test_rate_of_a_large_mask():
    """The number kept of n = 2^22 is binomial: within 5 standard deviations."""
    n = 1 << 22
    for p in (0.02, 0.25, 0.5, 0.9):
        rate = round(p * 65536) / 65536
        count = int((mx.dropout(torch.ones(n, device="cuda"), p, (99, 1)) != 0).sum())
        assert abs(count - n * (1 - rate)) <= 5 * (n * rate * (1 - rate)) ** 0.5


@pytest.mark.parametrize("dtype", DTYPES)
def test_ends_of_the_rate(dtype):
    x, r, dy = data(1003, dtype)
    assert torch.equal(mx.dropout(x, 0.0, (1, 1)), x)
    assert torch.equal(mx.dropout(x, 1e-9, (1, 1), residual=r), (x.float() + r.float()).to(dtype))
    x[5], x[6] = float("inf"), float("nan")
    assert torch.equal(mx.dropout(x, 1.0, (1, 1)), torch.zeros_like(x))
    assert torch.equal(mx.dropout(x, 1.0, (1, 1), residual=r), r)
    xg = x.requires_grad_()
    dy[7] = float("inf")
    assert not torch.autograd.grad(mx.dropout(xg, 1.0, (1, 1)), xg, dy)[0].any()


def test_dropped_infinities_and_nan_leave_nothing():
    n, p = 4096, 0.5
    keep = kept(n, p, 3, 4)
    x = torch.where(keep, torch.ones(n, device="cuda"), float("nan")).to(torch.bfloat16)
    x[~keep.roll(1) & ~keep] = float("inf")
    assert torch.equal(mx.dropout(x, p, (3, 4)), torch.where(keep, 2.0, 0.0).to(torch.bfloat16))
    some = ~kept(n, p, 5, 6)
    y = mx.dropout(torch.where(some, 1.0, float("nan")), p, (5, 6))
    assert torch.equal(y.isnan(), ~some)  # a kept NaN stays


def test_strides_and_alignment():
    x, r, _ = data(64 * 48, torch.bfloat16)
    x, r = x.view(64, 48), r.view(64, 48)
    keep = kept(x.numel(), 0.3, 8, 9).view(48, 64)
    got = mx.dropout(x.t(), 0.3, (8, 9), residual=r.t())  # by row-major order of the tensor, not of memory
    assert got.is_contiguous() and torch.equal(got, want(x.t(), keep, 0.3, r.t()))
    for dtype in DTYPES:
        n = 10007
        flat = [torch.randn(n + 8, device="cuda").to(dtype) for _ in range(2)]
        for a, b in ((1, 0), (0, 1), (3, 2), (4, 4)):
            x, r = flat[0][a: a + n], flat[1][b: b + n]
            keep = kept(n, 0.3, 8, 9)
            assert torch.equal(mx.dropout(x, 0.3, (8, 9)), want(x, keep, 0.3))
            assert torch.equal(mx.dropout(x, 0.3, (8, 9), residual=r), want(x, keep, 0.3, r))
    x = torch.randn((1, 5), device="cuda").expand(4, 5)
    assert torch.equal(mx.dropout(x, 0.5, (1, 2)), want(x, kept(20, 0.5, 1, 2), 0.5))
    # in place, through the C entry point
    x = torch.randn(1000, device="cuda")
    ref = mx.dropout(x, 0.5, (1, 2))
    nat.launch("mednext_dropout", x, x.data_ptr(), None, x.data_ptr(), None, 1, 2, None, 1000, 32768, 0)
    assert torch.equal(x, ref)


def test_elements_past_32_bits():
    n = 2**31 + 1003
    x = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    y = mx.dropout(x, 0.5, (21, 22))
    for begin in (0, 2**31 - 500, n - 700):
        assert torch.equal(y[begin: begin + 700], want(x[:700], kept(700, 0.5, 21, 22, begin), 0.5))


def test_empty():
    x = torch.empty((0, 3), device="cuda", requires_grad=True)
    y = mx.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64, device="cuda"))
    assert y.shape == (0, 3) and torch.autograd.grad(y, x, torch.empty_like(y))[0].shape == (0, 3)


def test_backward_uses_the_numbers_that_forward_read():
    rng = torch.tensor([5, 0], device="cuda")
    x = torch.ones(3000, device="cuda", requires_grad=True)
    y = mx.dropout(x, 0.5, rng)
    rng[1] += 1  # the next step's numbers, before this step's backward
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(dx, y.detach())
    assert not torch.equal(mx.dropout(x.detach(), 0.5, rng), y.detach())


def test_captured_step_advances_on_the_device():
    rng = torch.tensor([5, 0], device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x = torch.ones(3000, device="cuda", requires_grad=True)
        torch.autograd.grad(mx.dropout(x, 0.5, rng), x, torch.ones(3000, device="cuda"))
        dy = torch.ones(3000, device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            y = mx.dropout(x, 0.5, rng)
            rng[1] += 1
            (dx,) = torch.autograd.grad(y, x, dy)
    torch.cuda.current_stream().wait_stream(s)
    for step in range(3):
        g.replay()
        torch.cuda.synchronize()
        ref = want(dy, kept(3000, 0.5, 5, step), 0.5)
        assert torch.equal(y.detach(), ref) and torch.equal(dx, ref)


def test_gradient_against_differences():
    """The map is linear: a difference with any step gives the gradient to fp32 rounding of
    the 200 values' sum (64 * 2^-24 of the sum of magnitudes, over the step 1)."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    x, d, dy = (torch.randn(200, generator=gen, device="cuda") for _ in range(3))
    xg = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(mx.dropout(xg, 0.3, (1, 2)), xg, dy)
    loss = lambda t: (mx.dropout(t, 0.3, (1, 2)).double() * dy.double()).sum()  # noqa: E731
    slope = (loss(x + d) - loss(x - d)) / 2
    bound = 64 * 2.0**-24 * ((x.abs() + d.abs()) * dy.abs()).double().sum() * 2
    assert abs(slope - (dx.double() * d.double()).sum()) <= bound


def test_inside_compile():
    x, r, dy = data(3000, torch.bfloat16)
    rng = torch.tensor([5, 6], device="cuda")
    xg, rg = x.clone().requires_grad_(), r.clone().requires_grad_()
    y = torch.compile(lambda a, b: mx.dropout(a, 0.25, rng, residual=b), backend="aot_eager", fullgraph=True)(xg, rg)
    keep = kept(3000, 0.25, 5, 6)
    assert torch.equal(y, want(x, keep, 0.25, r))
    dx, dr = torch.autograd.grad(y, (xg, rg), dy)
    assert torch.equal(dx, want(dy, keep, 0.25)) and torch.equal(dr, dy)


def test_refusals():
    x = torch.zeros(8, device="cuda")
    rng = torch.zeros(2, dtype=torch.int64, device="cuda")
    for args, kw, text in (
        ((x.double(), 0.5, rng), {}, "float16, bfloat16 or float32"),
        ((x, 1.5, rng), {}, "probability"),
        ((x, float("nan"), rng), {}, "probability"),
        ((x, 0.5, rng.cpu()), {}, "rng"),
        ((x, 0.5, rng.int()), {}, "rng"),
        ((x, 0.5, torch.zeros(4, dtype=torch.int64, device="cuda")[::2]), {}, "rng"),
        ((x, 0.5, (1, 2.5)), {}, "integers"),
        ((x, 0.5, None), {}, "integers"),
        ((x, 0.5, rng), {"residual": x[:4]}, "residual"),
        ((x, 0.5, rng), {"residual": x.half()}, "residual"),
    ):
        with pytest.raises(ValueError, match=text):
            mx.dropout(*args, **kw)


def test_words_match_numpy_layout():
    """Word order inside a group: element i % 8 is the low, then the high half of each output."""
    w = dropout_words(7, 9, 0, 16)
    for t in np.unique(w)[::3]:
        p = float(t) / 65536
        got = mx.dropout(torch.ones(16, device="cuda"), p, (7, 9)) != 0
        assert got.cpu().tolist() == (w >= t).tolist()


def test_spaced_seeds_give_every_layer_a_mask_of_its_own():
    """`layer` is added to the seed: seeds further apart than the layers, as the function's notes ask, share no mask."""
    x = torch.ones(4096, device="cuda")
    masks = [mx.dropout(x, 0.5, (7 + rank * 2**32, 0), layer=layer) != 0 for rank in range(4) for layer in range(4)]
    assert len({tuple(m.cpu().tolist()) for m in masks}) == 16


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_masks_with_residual_and_gradients(dtype):
    """Enough elements for several groups per thread in every type, the last CTA's ragged; the whole mask exactly."""
    n, p = 10_000_005, 0.1
    x, r, dy = data(n, dtype)
    keep = kept(n, p, 31, 2**33 + 5)
    xg, rg = x.clone().requires_grad_(), r.clone().requires_grad_()
    y = mx.dropout(xg, p, torch.tensor([30, 2**33 + 5], device="cuda"), residual=rg, layer=1)
    assert torch.equal(y, want(x, keep, p, r))
    dx, dr = torch.autograd.grad(y, (xg, rg), dy)
    assert torch.equal(dx, want(dy, keep, p)) and torch.equal(dr, dy)
    assert torch.equal(mx.dropout(x, p, (31, 2**33 + 5)), want(x, keep, p))
    assert nat.device_error() == 0

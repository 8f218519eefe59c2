"""Layer norm on the sm_100a kernels against the formula in 64 bits.

Tolerances, elementwise, with u the unit roundoff of the output's type and e = 64 * 2^-24
(fp32 arithmetic with sums of a few hundred terms per thread; the sums' errors grow
like the square root of their length, 64 bounds that and the formula's own few roundings).
k = max|x| r is a token's condition: an error of 2^-24 max|x| in its mean moves xh by k 2^-24.

  y:  u |y|  + e (|w| (|xh| + k) + |b|)
  dx: u |dx| + e r (|g| + mean|g| + |xh| mean|g xh| + k |mean(g xh)| + |xh| k mean|g|)
  dw: u |dw| + e sum |dy| (|xh| + k);  db: u |db| + e sum |dy|
"""

from __future__ import annotations

import pytest
import torch

import mednext_accel_b200 as mx
from mednext_accel_b200 import _native as nat

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 2.0**-149, torch.bfloat16: 2.0**-133, torch.float16: 2.0**-24}  # least subnormals
E = 64 * 2.0**-24
EPS = 1e-6


def reference(x, w, b, dy, dim, eps=EPS):
    """{name: (value, tolerance without the output's own rounding)} in 64 bits."""
    x, dy = x.double().movedim(dim, -1), dy.double().movedim(dim, -1)
    c = x.shape[-1]
    one = torch.ones(c, device=x.device, dtype=torch.float64)
    w = one if w is None else w.double()
    b = 0 * one if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    r = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = (x - mean) * r
    k = x.abs().amax(-1, keepdim=True) * r
    g = dy * w
    mg, mgx = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    ag, agx = g.abs().mean(-1, keepdim=True), (g * xh).abs().mean(-1, keepdim=True)
    flat = lambda t: t.reshape(-1, c).sum(0)  # noqa: E731
    back = lambda t: t.movedim(-1, dim)  # noqa: E731
    return {
        "y": (back(xh * w + b), back(E * (w.abs() * (xh.abs() + k) + b.abs()))),
        "dx": (back(r * (g - mg - xh * mgx)),
               back(E * r * (g.abs() + ag + xh.abs() * agx + k * mgx.abs() + xh.abs() * k * ag))),
        "dw": (flat(dy * xh), E * flat(dy.abs() * (xh.abs() + k))),
        "db": (flat(dy), E * flat(dy.abs())),
    }


def assert_near(got, want, tol, what):
    assert got.shape == want.shape, what
    u = U[got.dtype]
    err = (got.double() - want).abs()
    bound = u * want.abs() + tol * (1 + u) + TINY[got.dtype]
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {float((err / bound).max()):.3g} of its bound"


def inputs(shape, dim, dtype, seed=0, pdt=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c = shape[dim]
    rnd = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    x = (rnd(*shape) * 1.5 + 0.5).to(dtype)
    return x, (1 + 0.3 * rnd(c)).to(pdt), (0.2 * rnd(c)).to(pdt), rnd(*shape).to(dtype)


def check(x, w, b, dy, dim, eps=EPS):
    xg = x.detach().requires_grad_()
    params = [p.detach().requires_grad_() if p is not None else None for p in (w, b)]
    y = mx.layer_norm(xg, *params, eps=eps, dim=dim)
    leaves = [xg] + [p for p in params if p is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        inference = mx.layer_norm(x, w, b, eps=eps, dim=dim)
    assert torch.equal(inference, y)
    assert y.stride() == x.stride() or not x.is_contiguous()
    want = reference(x, w, b, dy, dim, eps)
    assert_near(y.detach(), *want["y"], "y")
    assert_near(grads[0], *want["dx"], "dx")
    names = [n for n, p in (("dw", w), ("db", b)) if p is not None]
    for name, g in zip(names, grads[1:], strict=True):
        assert_near(g, *want[name], name)
    assert nat.device_error() == 0
    return y, grads


WIDTHS = [1, 2, 7, 8, 24, 31, 32, 33, 64, 96, 100, 129, 255, 256, 264, 512, 777, 1000, 1024, 1536, 2047, 2048, 4096,
          5000, 8192, 8200, 16384, 20001, 40000]


@pytest.mark.parametrize("c", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rows_of_every_width(c, dtype):
    for rows in (1, 3, 37):
        check(*inputs((rows, c), 1, dtype, seed=c + rows), -1)


@pytest.mark.parametrize("rows", [1, 2, 5, 148, 1000, 4099, 70001])
@pytest.mark.parametrize("c", [24, 33, 256, 520])
def test_many_rows(rows, c):
    check(*inputs((rows, c), 1, torch.bfloat16, seed=rows), -1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [
    (1, 1, 2), (1, 3, 1), (2, 8, 7), (1, 16, 64), (3, 31, 33), (2, 32, 128), (1, 33, 130), (2, 64, 6, 5, 4),
    (1, 96, 9, 11, 13), (2, 128, 8, 8, 8), (1, 200, 17, 2), (1, 256, 1000), (2, 512, 8, 8, 8), (1, 513, 72), (1, 1000, 50),
    (2, 1024, 66), (1, 1100, 64), (1, 2500, 35),
])
def test_channels_first(shape, dtype):
    check(*inputs(shape, 1, dtype, seed=sum(shape)), 1)


@pytest.mark.parametrize("v", [40 * 40 * 40, 33 * 35 * 37])
@pytest.mark.parametrize("c", [32, 48, 160])
def test_channels_first_many_voxels(c, v):
    check(*inputs((2, c, v), 1, torch.bfloat16, seed=c), 1)


@pytest.mark.parametrize("dim", [0, 1, 2, 3, -2])
def test_any_axis(dim):
    check(*inputs((6, 10, 12, 8), dim, torch.float32), dim)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("parts", ["none", "weight", "bias"])
def test_absent_parameters(parts, dtype):
    x, w, b, dy = inputs((50, 72), 1, dtype)
    check(x, w if parts == "weight" else None, b if parts == "bias" else None, dy, -1)
    x, w, b, dy = inputs((2, 40, 90), 1, dtype)
    check(x, w if parts == "weight" else None, b if parts == "bias" else None, dy, 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_parameters_of_the_inputs_type(dtype):
    for shape, dim in (((100, 256), 1), ((2, 48, 200), 1), ((30, 5003), 1)):
        check(*inputs(shape, dim, dtype, pdt=dtype), dim)


def test_strides_orders_and_alignment():
    x, w, b, dy = inputs((2, 24, 6, 5, 8), 1, torch.bfloat16)
    cl = x.to(memory_format=torch.channels_last_3d)
    y, grads = check(cl, w, b, dy, 1)  # dense in another order: kept
    assert y.stride() == cl.stride() and grads[0].stride() == cl.stride()
    x, w, b, dy = inputs((40, 64), 1, torch.float32)
    check(x.t().contiguous().t(), w, b, dy, 1)  # a transposed matrix
    wide = torch.randn((40, 100), device="cuda")
    check(wide[:, 10:74], w, b, dy, 1)  # gaps between rows
    check(wide[::2, 10:74], w, b, dy[::2], 1)
    check(x, w, b, torch.ones((), device="cuda").expand(40, 64), 1)  # a broadcast gradient
    for shape, dim in (((41, 64), 1), ((1, 24, 96), 1)):
        x, w, b, dy = inputs(shape, dim, torch.bfloat16)
        flat = torch.empty(x.numel() + 9, dtype=x.dtype, device="cuda")
        for shift in (1, 4):
            moved = flat[shift: shift + x.numel()].view(shape)  # not 16-byte aligned
            moved.copy_(x)
            y, _ = check(moved, w, b, dy, dim)
            assert torch.allclose(y.float(), mx.layer_norm(x, w, b, eps=EPS, dim=dim).float(), rtol=2**-7, atol=1e-6)
        c = w.numel()
        held = torch.empty(c + 3, device="cuda")
        held[1: c + 1] = w
        check(x, held[1: c + 1], b, dy, dim)
        check(x, w.repeat_interleave(2)[::2], b, dy, dim)


def test_a_mean_far_above_the_spread():
    x, w, b, dy = inputs((64, 512), 1, torch.float32)
    check(x + 3000.0, w, b, dy, -1)
    x, w, b, dy = inputs((1, 64, 640), 1, torch.float32)
    check(x + 3000.0, w, b, dy, 1)


def test_constant_and_huge_rows():
    x, w, b, dy = inputs((8, 96), 1, torch.float32)
    x[0] = 0.0
    x[1] = 7.0
    x[2] *= 1e15
    check(x, w, b, dy, -1, eps=1e-5)
    xt = x.t().reshape(1, 96, 8).contiguous()
    check(xt, w, b, dy.t().reshape(1, 96, 8).contiguous(), 1, eps=1e-5)


@pytest.mark.parametrize("shape,dim", [((9, 256), 1), ((9, 260), 1), ((9, 9000), 1), ((1, 40, 72), 1), ((1, 40, 71), 1)])
def test_a_token_with_nan_or_infinity_touches_no_other(shape, dim):
    x, w, b, dy = inputs(shape, dim, torch.float32)
    clean = mx.layer_norm(x, w, b, dim=dim)
    bad = x.clone()
    tokens = bad.numel() // shape[dim]
    view = bad.movedim(dim, -1)
    for i, value in ((2, float("nan")), (5, float("inf"))):
        view[tuple(j.item() for j in torch.unravel_index(torch.tensor(i), view.shape[:-1]))][3] = value
    xg = bad.requires_grad_()
    y = mx.layer_norm(xg, w, b, dim=dim)
    (dx,) = torch.autograd.grad(y, xg, dy)
    rows = lambda t: t.detach().movedim(dim, -1).reshape(tokens, -1)  # noqa: E731
    keep = [i for i in range(tokens) if i not in (2, 5)]
    assert torch.equal(rows(y)[keep], rows(clean)[keep])
    assert rows(y)[[2, 5]].isnan().all()
    assert rows(dx)[keep].isfinite().all() and rows(dx)[[2, 5]].isnan().all()


def test_no_tokens():
    for shape, dim in (((0, 40), 1), ((2, 40, 0), 1), ((0, 40, 3, 3, 3), 1)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        w = torch.ones(40, device="cuda", requires_grad=True)
        b = torch.ones(40, device="cuda", requires_grad=True)
        y = mx.layer_norm(x, w, b, dim=dim)
        assert y.shape == shape
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
        assert dx.shape == shape and not dw.any() and not db.any()


@pytest.mark.parametrize("shape,dim", [((5, 48), 1), ((1, 12, 20), 1), ((3, 9001), 1)])
def test_gradients_against_differences(shape, dim):
    """Central differences of the kernel's own forward, h = 2^-6: the loss is a sum of n
    fp32 values (error about 2^-24 |dy||y|, divided by 2 h) and the third-order term is
    about h^2 / 6 of the first, so 2e-3 of |grad||direction| holds both."""
    x, w, b, dy = inputs(shape, dim, torch.float32, seed=3)
    gen = torch.Generator(device="cuda").manual_seed(4)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(mx.layer_norm(*leaves, eps=1e-3, dim=dim), leaves, dy)
    for i in range(3):
        d = torch.randn(leaves[i].shape, generator=gen, device="cuda")
        h = 2.0**-6

        def loss(sign, i=i, d=d, h=h):
            moved = [t.detach() + sign * h * d if j == i else t.detach() for j, t in enumerate(leaves)]
            return (mx.layer_norm(*moved, eps=1e-3, dim=dim).double() * dy.double()).sum()

        slope = (loss(1) - loss(-1)) / (2 * h)
        want = (grads[i].double() * d.double()).sum()
        assert abs(slope - want) <= 2e-3 * grads[i].double().norm() * d.double().norm()


def test_results_are_bitwise_reproducible_on_any_stream():
    for shape, dim in (((30000, 96), 1), ((2, 64, 30000), 1), ((500, 6000), 1)):
        x, w, b, dy = inputs(shape, dim, torch.bfloat16)
        first = check_free(x, w, b, dy, dim)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = check_free(x, w, b, dy, dim)
        torch.cuda.current_stream().wait_stream(side)
        for p, q in zip(first, again, strict=True):
            assert torch.equal(p, q)


def check_free(x, w, b, dy, dim):
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = mx.layer_norm(*leaves, dim=dim)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


def test_only_the_wanted_gradients():
    x, w, b, dy = inputs((20, 64), 1, torch.float32)
    want = check_free(x, w, b, dy, 1)
    xg = x.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(mx.layer_norm(xg, w, b), xg, dy)[0], want[1])
    wg = w.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(mx.layer_norm(x, wg, b), wg, dy)[0], want[2])


def test_graph_capture_follows_its_inputs():
    x, w, b, dy = inputs((2, 32, 500), 1, torch.bfloat16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)]
        torch.autograd.grad(mx.layer_norm(*leaves, dim=1), leaves, dy)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            y = mx.layer_norm(*leaves, dim=1)
            grads = torch.autograd.grad(y, leaves, dy)
    torch.cuda.current_stream().wait_stream(s)
    x2 = inputs((2, 32, 500), 1, torch.bfloat16, seed=9)[0]
    with torch.no_grad():
        leaves[0].copy_(x2)
    g.replay()
    torch.cuda.synchronize()
    want = check_free(x2, w, b, dy, 1)
    for got, ref in zip((y, *grads), want, strict=True):
        assert torch.equal(got, ref)


def test_inside_compile():
    x, w, b, dy = inputs((2, 32, 100), 1, torch.bfloat16)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    fn = torch.compile(lambda *t: mx.layer_norm(*t, dim=1), backend="aot_eager", fullgraph=True)
    y = fn(*leaves)
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    for p, q in zip(got, check_free(x, w, b, dy, 1), strict=True):
        assert torch.equal(p, q) or torch.allclose(p.float(), q.float(), rtol=2**-7, atol=1e-5)


def test_layer():
    layer = mx.LayerNorm3d(24).cuda()
    x = torch.randn((1, 24, 4, 5, 6), device="cuda", requires_grad=True)
    y = layer(x)
    want = torch.nn.functional.layer_norm(x.movedim(1, -1), (24,), layer.weight, layer.bias, 1e-6).movedim(-1, 1)
    assert torch.allclose(y, want, rtol=1e-5, atol=1e-5)
    y.sum().backward()
    assert layer.weight.grad.shape == (24,) and layer.bias.grad.shape == (24,)


def test_refusals():
    x = torch.zeros((4, 8), device="cuda")
    w = torch.ones(8, device="cuda")
    for args, kw, text in (
        ((x.double(),), {}, "float16, bfloat16 or float32"),
        ((x,), {"dim": 2}, "out of range"),
        ((x, w[:7]), {}, "shape"),
        ((x, w.half()), {}, "float32 weight"),
        ((x, w, w.cpu()), {}, "device"),
        ((x.half(), w, w.half()), {}, "one type"),
        ((x,), {"eps": 0.0}, "eps"),
        ((x,), {"eps": float("nan")}, "eps"),
        ((torch.zeros((4, 0), device="cuda"),), {}, "nonempty"),
    ):
        with pytest.raises(ValueError, match=text):
            mx.layer_norm(*args, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 600, 2048), (2, 1000, 777), (1, 1025, 256), (1, 4096, 40), (1, 16384, 9), (1, 16385, 3)])
def test_channels_first_wide(shape, dtype):
    """More channels than a tile's warps hold at once, and than the channels-first form has."""
    x, w, b, dy = inputs(shape, 1, dtype, seed=sum(shape))
    check(x, w, b, dy, 1)
    if shape[1] > 16384:
        check(x.transpose(1, 2).contiguous().transpose(1, 2), w, b, dy, 1)
        y = x.permute(1, 2, 0).contiguous().permute(2, 0, 1)
        check(y, w, b, dy, 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,c", [(9001, 1), (20011, 3), (30001, 31), (12007, 97), (7777, 333), (5003, 777), (4001, 2047)])
def test_many_odd_rows_at_any_element(rows, c, dtype):
    """Blocks of rows that start and end off every boundary, each tensor at its own element: the bits of aligned copies,
    and within bounds of the 64-bit result."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x = (torch.randn((rows, c), generator=gen, device="cuda") * 2 + 0.5).to(dtype)
    dy = torch.randn((rows, c), generator=gen, device="cuda").to(dtype)
    w = torch.randn(c, generator=gen, device="cuda")
    b = torch.randn(c, generator=gen, device="cuda")

    def at(t, off):
        held = torch.full((t.numel() + 16,), 7.0, dtype=t.dtype, device="cuda")
        view = held[off:off + t.numel()].view(t.shape)
        view.copy_(t)
        return view

    results = []
    for ox, od in ((0, 0), (1, 6), (5, 3)):
        xs = at(x, ox).requires_grad_()
        ws, bs = w.clone().requires_grad_(), b.clone().requires_grad_()
        y = mx.layer_norm(xs, ws, bs)
        results.append((y, *torch.autograd.grad(y, (xs, ws, bs), at(dy, od))))
    for other in results[1:]:
        assert all(torch.equal(p, q) for p, q in zip(results[0], other))
    x64 = x.double()
    mean = x64.mean(1, keepdim=True)
    rstd = (x64.var(1, unbiased=False, keepdim=True) + 1e-6).rsqrt()
    xh = (x64 - mean) * rstd
    want = xh * w.double() + b.double()
    u = 2.0**-8 if dtype == torch.bfloat16 else 2.0**-11
    size = want.abs() + xh.abs() * w.double().abs() + b.double().abs() + 1e-3
    assert ((results[0][0].double() - want).abs() <= u * want.abs() + 2.0**-16 * size).all()
    g = dy.double() * w.double()
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    size = rstd * (g.abs() + g.abs().mean(1, keepdim=True) + xh.abs() * (g * xh).abs().mean(1, keepdim=True))
    assert ((results[0][1].double() - dx).abs() <= u * dx.abs() + 2.0**-16 * size + 1e-7).all()
    for got, terms in ((results[0][2], dy.double() * xh), (results[0][3], dy.double())):
        assert ((got.double() - terms.sum(0)).abs() <= 2.0**-16 * terms.abs().sum(0) + 1e-6).all()
    assert nat.device_error() == 0


@pytest.mark.parametrize("shape,dim", [((3000, 256), 1), ((1, 32, 20000), 1), ((40, 9000), 1)])
def test_the_fold_reads_the_partials_of_its_own_call(shape, dim):
    """Calls in a row take the same workspace, and each fold starts while its partials are written: every call gives
    the bits of a call on its own."""
    x, w, b, dy = inputs(shape, dim, torch.bfloat16)
    gradients = [dy, dy.neg(), dy * 3, dy.flip(0).contiguous()]
    want = []
    for g in gradients:
        want.append(check_free(x, w, b, g, dim)[2:])
        torch.cuda.synchronize()
    results = [check_free(x, w, b, gradients[i % 4], dim)[2:] for i in range(60)]  # queued, not waited for
    for i, got in enumerate(results):
        assert all(torch.equal(p, q) for p, q in zip(got, want[i % 4], strict=True)), i


@pytest.mark.parametrize("rows,c,dtype", [
    (60001, 24, torch.float32), (40009, 97, torch.float32), (30011, 100, torch.float32), (20011, 522, torch.float32),
    (9001, 1000, torch.float32), (4001, 2047, torch.float32), (4003, 4096, torch.float32), (2003, 5000, torch.float32),
    (40009, 98, torch.bfloat16), (30011, 250, torch.float16), (20011, 522, torch.bfloat16), (20011, 522, torch.float16),
    (4001, 4094, torch.bfloat16), (9001, 1000, torch.float16), (2003, 4095, torch.bfloat16), (2003, 3001, torch.float32),
])
def test_many_rows_of_each_word_and_type(rows, c, dtype):
    """Several rows in flight per group (from 12 CTAs' worth of rows on each SM) for every word that rows can be
    read in: 16 bytes, 4 bytes of 16-bit data, single elements."""
    check(*inputs((rows, c), 1, dtype, seed=rows + c), -1)

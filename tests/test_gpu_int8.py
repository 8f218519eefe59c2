"""8-bit products on the sm_100a kernels.

Quantised rows and scales are compared exactly with the same fp32 formula in torch
operations.  Products are compared with the exact integer sum in 64 bits: what remains is
the rounding of the sum to fp32, two products and a sum, each 2^-24, and the output's
own rounding u:  |err| <= u |y| + 4 * 2^-24 (|sum s_t s_j| + |b|).
"""

from __future__ import annotations

import pytest
import torch

import mednext_accel_b200 as mx
from mednext_accel_b200 import _native as nat

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
LEAST = 127 * 2.0**-126


def quantized(x, dim):
    """(q [tokens, K], scale [tokens]) by the formula, in fp32 torch operations.  Both
    quotients are of two tensors: torch makes a reciprocal and a product, two roundings,
    of a quotient with a number."""
    x = x.float().movedim(dim, -1).reshape(-1, x.shape[dim])
    m = x.abs().amax(1, keepdim=True).clamp_min(LEAST)
    top = torch.full_like(m, 127.0)
    return (x * torch.div(top, m)).round(), torch.div(m, top)[:, 0]


def product(x, w, s, b, dim):
    """(value, magnitude) in 64 bits from the quantised rows."""
    q, qs = quantized(x, dim)
    acc = (q.double() @ w.double().t()) * qs.double()[:, None] * s.double()
    bias = torch.zeros_like(s) if b is None else b
    shape = (*x.movedim(dim, -1).shape[:-1], w.shape[0])
    back = lambda t: t.reshape(shape).movedim(-1, dim)  # noqa: E731
    return back(acc + bias.double()), back(acc.abs() + bias.double().abs())


def check(x, w, s, b, dim):
    y = mx.int8_linear(x, w, s, b, dim=dim)
    want, size = product(x, w, s, b, dim)
    assert y.shape == want.shape and y.dtype == x.dtype
    err = (y.double() - want).abs()
    bound = U[x.dtype] * want.abs() + 4 * 2.0**-24 * size * (1 + U[x.dtype]) + (2.0**-24 if x.dtype == torch.float16 else 1e-38)
    bad = ~(err <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / bound).max()):.3g} of its bound"
    assert nat.device_error() == 0
    return y


def weights(n, k, seed=0, pad=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    pitch = (k + 15) // 16 * 16 + pad
    held = torch.randint(-127, 128, (n, pitch), generator=gen, device="cuda").to(torch.int8)  # used past k too: not to be read
    return held[:, :k], torch.rand(n, generator=gen, device="cuda") * 1e-2 + 1e-4, torch.randn(n, generator=gen, device="cuda")


def activations(shape, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * 2).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape,dim", [
    ((1, 1), 1), ((3, 7), 1), ((5, 16), 1), ((9, 33), 1), ((64, 256), 1), ((3, 1000), 1), ((2, 4096), 1), ((2, 20000), 1),
    ((1, 32, 64), 1), ((2, 5, 7), 1), ((1, 96, 131), 1), ((2, 64, 4, 6, 8), 1), ((1, 513, 40), 1), ((1, 2048, 33), 1),
    ((4, 6, 5), 0), ((1, 40, 1001), 1), ((3, 128, 640), 1),
])
def test_quantized_rows_are_the_formulas(shape, dim, dtype):
    x = activations(shape, dtype, sum(shape))
    x.select(dim, 0).mul_(30)
    q, s = mx.quantize_int8(x, dim)
    wq, ws = quantized(x, dim)
    assert q.stride(0) % 16 == 0 and torch.equal(q.float(), wq) and torch.equal(s, ws)
    whole = q.as_strided((q.shape[0], q.stride(0)), (q.stride(0), 1))
    assert not whole[:, q.shape[1]:].any()


def test_quantize_zeros_small_and_not_finite():
    x = torch.zeros((6, 40), device="cuda")
    x[1] = 1e-40  # subnormal
    x[2, 3] = float("inf")
    x[3, 4] = float("nan")
    x[4] = torch.linspace(-3e38, 3e38, 40, device="cuda")  # its step overflows: not finite either
    x[5, 0] = -2.0
    for t, dim in ((x, 1), (x.t().reshape(1, 40, 6).contiguous(), 1)):
        q, s = mx.quantize_int8(t, dim)
        good = [0, 1, 5]
        wq, ws = quantized(x, 1)
        assert torch.equal(q[good].float(), wq[good]) and torch.equal(s[good], ws[good])
        assert not q[[0, 2, 3, 4]].any() and s[2].isinf() and s[3].isnan() and not s[4].isfinite()
        w, ws, b = weights(20, 40)
        y = mx.int8_linear(t, w, ws, b, dim=dim)
        y = y if t is x else y[0].t()
        assert y[[2, 3, 4]].isnan().all() and y[good].isfinite().all() and torch.equal(y[0], b)


def test_quantize_up_to_the_largest_number():
    x = torch.linspace(-1.0, 1.0, 40, device="cuda") * 3.4e38
    q, s = mx.quantize_int8(x)
    wq, ws = quantized(x, 0)
    assert x.isfinite().all() and torch.equal(q.float(), wq) and torch.equal(s, ws)
    assert q[0, 0] == -127 and q[0, -1] == 127


SIZES = [(1, 1, 1), (1, 16, 16), (1, 512, 2048), (2, 100, 77), (4, 4096, 40), (7, 33, 130), (8, 2048, 512), (9, 64, 64),
         (16, 256, 300), (17, 1000, 31), (33, 48, 1000), (64, 128, 128), (127, 129, 127), (128, 32, 64), (129, 200, 257),
         (300, 512, 256), (500, 777, 333), (1000, 96, 96), (2049, 64, 128), (3, 20000, 65), (700, 2064, 520)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("t,k,n", SIZES)
def test_rows(t, k, n, dtype):
    w, s, b = weights(n, k, seed=t)
    check(activations((t, k), dtype, seed=k), w, s, b, -1)
    check(activations((t, k), dtype, seed=k), w, s, None, -1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("outer,k,v,n", [
    (1, 32, 4096, 64), (2, 32, 1000, 64), (1, 64, 999, 32), (3, 96, 17 * 19, 48), (1, 2048, 512, 512), (2, 512, 64, 2048),
    (1, 256, 343, 1024), (2, 31, 33, 5), (5, 128, 128, 128), (1, 1, 300, 1), (4, 40, 2, 24), (1, 300, 1, 200), (2, 1024, 130, 130),
    (40, 16, 8, 16), (1, 160, 2000, 320), (1, 700, 1100, 90),
])
def test_channels_first(outer, k, v, n, dtype):
    w, s, b = weights(n, k, seed=v)
    check(activations((outer, k, v), dtype, seed=n), w, s, b, 1)


def test_extremes_of_the_sum():
    """Every product at its largest magnitude: K = 131072 reaches 127 * 127 * K < 2^31."""
    for k in (131072, 4096):
        x = torch.ones((3, k), device="cuda")
        x[1] = -1.0
        w = torch.full((5, k), 127, dtype=torch.int8, device="cuda")
        w[2] = -128  # a weight of -128 stays inside at K <= 131072 too
        w[3] = -127
        s = torch.full((5,), 1e-4, device="cuda")
        check(x, w, s, None, -1)


def test_strides_orders_and_weights_that_need_a_copy():
    x = activations((2, 48, 6, 5, 8), torch.bfloat16)
    w, s, b = weights(40, 48)
    y = check(x.to(memory_format=torch.channels_last_3d), w, s, b, 1)
    assert y.is_contiguous(memory_format=torch.channels_last_3d)
    check(activations((96, 64), torch.float32).t().contiguous().t()[:, :48], w, s, b, -1)
    flat = activations((50 * 48 + 3,), torch.bfloat16)
    check(flat[1: 1 + 50 * 48].view(50, 48), w, s, b, -1)
    check(flat[1: 1 + 50 * 48].view(1, 48, 50), w, s, b, 1)
    check(flat[:48], w, s, b, 0)
    check(activations((2, 3, 48), torch.float16), *weights(40, 48, pad=32), -1)
    x = activations((30, 37), torch.bfloat16)
    w, s, b = weights(21, 37)
    want = check(x, w, s, b, -1)
    assert torch.equal(check(x, w.contiguous(), s, b, -1), want)  # rows of 37 bytes
    assert torch.equal(check(x, w.t().contiguous().t(), s, b, -1), want)
    assert torch.equal(check(x, w, s.repeat_interleave(2)[::2], b.repeat_interleave(2)[::2], -1), want)


def test_quantized_weights_round_trip():
    gen = torch.Generator(device="cuda").manual_seed(0)
    w = torch.randn((70, 90), generator=gen, device="cuda")
    q, s = mx.quantize_int8(w)
    x = activations((40, 90), torch.float32)
    check(x, q, s, None, -1)
    err = (mx.int8_linear(x, q, s) - x @ w.t()).norm() / (x @ w.t()).norm()
    assert err < 0.02  # each factor is within 1/254 of its token's or channel's largest value


def test_reproducible_and_on_another_stream():
    x = activations((1, 64, 30000), torch.bfloat16)
    w, s, b = weights(96, 64)
    first = check(x, w, s, b, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [mx.int8_linear(x, w, s, b, dim=1) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(first, y) for y in again)


def test_graph_capture_follows_its_inputs():
    x = activations((5, 200), torch.bfloat16)
    big = activations((1, 64, 700), torch.bfloat16)
    w, s, b = weights(300, 200)
    w2, s2, b2 = weights(80, 64)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        mx.int8_linear(x, w, s, b), mx.int8_linear(big, w2, s2, b2, dim=1)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            y, z = mx.int8_linear(x, w, s, b), mx.int8_linear(big, w2, s2, b2, dim=1)
    torch.cuda.current_stream().wait_stream(st)
    x.copy_(activations((5, 200), torch.bfloat16, seed=5))
    big.copy_(activations((1, 64, 700), torch.bfloat16, seed=6))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, mx.int8_linear(x, w, s, b)) and torch.equal(z, mx.int8_linear(big, w2, s2, b2, dim=1))


def test_empty():
    w, s, b = weights(6, 10)
    assert mx.int8_linear(torch.empty((0, 10), device="cuda"), w, s, b).shape == (0, 6)
    assert mx.int8_linear(torch.empty((2, 10, 0), device="cuda"), w, s, b, dim=1).shape == (2, 6, 0)
    q, qs = mx.quantize_int8(torch.empty((0, 10), device="cuda"))
    assert q.shape == (0, 10) and qs.shape == (0,)


def test_inside_compile():
    x = activations((2, 32, 100), torch.bfloat16)
    w, s, b = weights(48, 32)
    y = torch.compile(lambda t: mx.int8_linear(t, w, s, b, dim=1), backend="aot_eager", fullgraph=True)(x)
    assert torch.equal(y, mx.int8_linear(x, w, s, b, dim=1))


def test_convolution_in_8_bits():
    torch.manual_seed(0)
    conv = torch.nn.Conv3d(40, 72, 1).cuda()
    layer = mx.Int8Pointwise3d(conv)
    x = torch.randn((2, 40, 5, 6, 7), device="cuda")
    with torch.no_grad():
        want, got = conv(x), layer(x)
    assert (got - want).norm() / want.norm() < 0.02
    other = mx.Int8Pointwise3d(torch.nn.Conv3d(40, 72, 1).cuda())
    other.load_state_dict(layer.state_dict())
    with torch.no_grad():
        assert torch.equal(other(x), got)
    with pytest.raises(ValueError, match="1x1x1"):
        mx.Int8Pointwise3d(torch.nn.Conv3d(4, 4, 3).cuda())


def test_refusals():
    w, s, b = weights(8, 16)
    x = torch.zeros((4, 16), device="cuda")
    for args, kw, text in (
        ((x.double(), w, s, b), {}, "float16, bfloat16 or float32"),
        ((x[:, :8], w, s, b), {}, "int8 weight"),
        ((x, w.int(), s, b), {}, "int8 weight"),
        ((x, w, s[:4], b), {}, "scale"),
        ((x, w, s.half(), b), {}, "scale"),
        ((x, w, s, b.half()), {}, "bias"),
        ((x, w.cpu(), s, b), {}, "device"),
        ((x, w, s, b), {"dim": 2}, "out of range"),
        ((x.clone().requires_grad_(), w, s, b), {}, "no gradient"),
    ):
        with pytest.raises(ValueError, match=text):
            mx.int8_linear(*args, **kw)
    with pytest.raises(ValueError, match="131072"):
        mx.quantize_int8(torch.zeros((1, 131073), device="cuda"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,k,n", [(2500, 300, 2056), (2305, 1024, 2304), (5000, 256, 1000), (1030, 2000, 4104)])
def test_large_rows(t, k, n, dtype):
    """Enough tiles for pairs of SMs; ragged last tiles in every direction."""
    w, s, b = weights(n, k, seed=t)
    check(activations((t, k), dtype, seed=k), w, s, b, -1)


@pytest.mark.parametrize("outer,k,v,n", [(3, 300, 1000, 1800), (1, 512, 4096, 1300), (20, 260, 264, 1100), (2, 1000, 2568, 900)])
def test_large_channels_first(outer, k, v, n):
    w, s, b = weights(n, k, seed=v)
    check(activations((outer, k, v), torch.bfloat16, seed=n), w, s, b, 1)


# A few hundred tokens and a long K share K over a cluster of SMs: whole and ragged slices, SMs
# without a slice, K past what a slice's registers hold, ragged tiles of tokens and channels.
CLUSTERED = [(9, 769, 1), (31, 896, 128), (33, 1024, 5), (100, 1921, 130), (64, 2048, 512), (512, 2048, 512), (17, 2049, 257),
             (70, 2500, 384), (64, 4096, 1024), (200, 4100, 100), (16, 8200, 127), (40, 16384, 136), (24, 16400, 64),
             (130, 2031, 77), (32, 2176, 129)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("t,k,n", CLUSTERED)
def test_long_rows(t, k, n, dtype):
    w, s, b = weights(n, k, seed=t)
    check(activations((t, k), dtype, seed=k), w, s, b, -1)
    check(activations((t, k), dtype, seed=k), w, s, None, -1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("outer,k,v,n", [
    (1, 2048, 512, 512), (1, 1024, 343, 256), (2, 1000, 64, 300), (3, 2048, 27, 130), (1, 4096, 125, 64), (1, 900, 10, 1),
    (4, 1025, 33, 129), (1, 16384, 34, 40), (1, 2300, 216, 512), (7, 1024, 30, 128), (1, 8192, 9, 257), (1, 769, 32, 128),
])
def test_deep_volumes(outer, k, v, n, dtype):
    w, s, b = weights(n, k, seed=v)
    check(activations((outer, k, v), dtype, seed=n), w, s, b, 1)
    check(activations((outer, k, v), dtype, seed=n), w, s, None, 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_long_tokens_off_their_alignment(dtype):
    """x at any element, in rows and channels first: the bits of an aligned copy."""
    w, s, b = weights(200, 2048, seed=3)
    for shape, dim in (((65, 2048), 1), ((2, 2048, 30), 1)):
        x = activations(shape, dtype, seed=4)
        held = torch.empty(x.numel() + 3, dtype=dtype, device="cuda")
        moved = held[3:].view(shape)
        moved.copy_(x)
        assert moved.data_ptr() % 16 and torch.equal(mx.int8_linear(moved, w, s, b, dim=dim), mx.int8_linear(x, w, s, b, dim=dim))
    assert nat.device_error() == 0


def test_long_tokens_that_are_zero_or_not_finite():
    w, s, b = weights(150, 2048, seed=5)
    for shape, dim in (((40, 2048), 1), ((1, 2048, 40), 1)):
        x = activations(shape, torch.bfloat16, seed=6)
        tokens = x if shape[0] == 40 else x[0].t()  # views
        tokens[3] = 0
        tokens[11, 2047] = float("inf")
        tokens[20, 0] = float("nan")
        tokens[39, 700] = -float("inf")
        y = mx.int8_linear(x, w, s, b, dim=dim)
        rows = y if shape[0] == 40 else y[0].t()
        bad = torch.tensor([11, 20, 39], device="cuda")
        good = torch.ones(40, dtype=torch.bool, device="cuda")
        good[bad] = False
        assert rows[bad].isnan().all() and rows[good].isfinite().all()
        assert torch.equal(rows[3], b.to(torch.bfloat16))
    assert nat.device_error() == 0


def test_long_tokens_are_the_same_bits_in_any_company():
    """A token's result does not depend on the other tokens of the call: integer sums have no order, and
    the forms for few, some and many tokens round alike."""
    w, s, b = weights(300, 2048, seed=7)
    x = activations((5000, 2048), torch.bfloat16, seed=8)
    y = mx.int8_linear(x, w, s, b)
    for start, count in ((0, 5), (5, 64), (69, 300), (4000, 33)):
        assert torch.equal(mx.int8_linear(x[start:start + count], w, s, b), y[start:start + count])
    v = x[:300].t().contiguous()[None]
    assert torch.equal(mx.int8_linear(v, w, s, b, dim=1)[0].t(), y[:300])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = [mx.int8_linear(x[:64], w, s, b) for _ in range(20)]
    stream.synchronize()
    assert all(torch.equal(a, y[:64]) for a in again)
    assert nat.device_error() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("outer,k,v,n", [
    (1, 192, 12000, 64), (2, 100, 8192, 100), (1, 256, 9480, 256), (1, 128, 10000, 512), (3, 65, 3208, 129), (1, 40, 20000, 300),
    (1, 250, 9608, 200), (40, 97, 264, 31), (1, 129, 30008, 384), (200, 70, 8, 16), (2, 160, 24 * 1000, 1),
])
def test_many_voxels_of_medium_width(outer, k, v, n, dtype):
    w, s, b = weights(n, k, seed=v, pad=16)
    check(activations((outer, k, v), dtype, seed=n), w, s, b, 1)
    check(activations((outer, k, v), dtype, seed=n), w, s, None, 1)


def test_voxels_of_medium_width_zero_or_not_finite_and_the_same_bits():
    w, s, b = weights(96, 192, seed=9)
    x = activations((1, 192, 20000), torch.float16, seed=10)
    x[0, :, 5] = 0
    x[0, 191, 77] = float("inf")
    x[0, 0, 19999] = float("nan")
    y = mx.int8_linear(x, w, s, b, dim=1)
    bad = torch.tensor([77, 19999], device="cuda")
    good = torch.ones(20000, dtype=torch.bool, device="cuda")
    good[bad] = False
    assert y[0][:, bad].isnan().all() and y[0][:, good].isfinite().all() and torch.equal(y[0, :, 5], b.half())
    assert torch.equal(mx.int8_linear(x[0].t().contiguous(), w, s, b)[good], y[0].t()[good])  # the rows' form
    for _ in range(20):
        assert torch.equal(mx.int8_linear(x, w, s, b, dim=1)[0][:, good], y[0][:, good])
    assert nat.device_error() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,k,off", [(9473, 777, 0), (12001, 33, 1), (20000, 1023, 3), (9999, 1301, 5), (9500, 2047, 1), (9480, 2049, 0), (9472, 5, 7), (10007, 96, 5), (30000, 1, 0)])
def test_many_odd_rows_are_quantised_alike(t, k, off, dtype):
    """Rows off every boundary, in blocks: the formula's bytes."""
    x = activations((t, k), dtype, seed=k)
    held = torch.empty(x.numel() + 8, dtype=dtype, device="cuda")
    view = held[off:off + x.numel()].view(t, k)
    view.copy_(x)
    view[17] = 0
    view[t - 1, k - 1] = float("inf")
    q, s = mx.quantize_int8(view)
    wq, ws = quantized(view, 1)
    assert torch.equal(q[:-1].float(), wq[:-1]) and torch.equal(s[:-1], ws[:-1])
    assert not q[-1].any() and s[-1].isinf()
    assert nat.device_error() == 0


@pytest.mark.parametrize("cast", [
    lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.double(), lambda m: m.to(torch.float16), lambda m: m.type(torch.half),
    lambda m: m.to("cpu", torch.bfloat16).cuda(),
])
def test_a_cast_module_keeps_its_numbers(cast):
    """The 8-bit rows, their fp32 scales and the fp32 bias are what the products take, whatever the model is cast to."""
    torch.manual_seed(0)
    model = torch.nn.Sequential(mx.Int8Pointwise3d(torch.nn.Conv3d(24, 40, 1).cuda()))
    x = activations((1, 24, 4, 5, 6), torch.float16)
    want = model(x)
    held = {name: t.clone() for name, t in model.state_dict().items()}
    model = cast(model)
    for name, t in model.state_dict().items():
        assert t.is_cuda and t.dtype == held[name].dtype and torch.equal(t, held[name]), name
    assert torch.equal(model(x), want)
    without = cast(mx.Int8Pointwise3d(torch.nn.Conv3d(24, 40, 1, bias=False).cuda()))
    assert without.bias is None and without(x).shape == want.shape


UNSTAGED = [((2, 64, 33 * 35 * 37), 100, 1), ((1, 64, 33 * 35 * 37), 512, 1), ((1, 32, 33 * 35 * 37), 64, 1),
            ((1, 512, 33 * 35 * 37), 128, 1), ((100003, 64), 77, -1), ((70001, 130), 301, -1)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape,n,dim", UNSTAGED)
def test_many_tiles_off_16_byte_rows(shape, n, dim, dtype):
    """Odd patches and odd widths: several tiles on each SM, so that accumulators are used again (two
    of 256 columns, four of up to 128), and a ragged last tile of tokens and of channels."""
    k = shape[dim]
    w, s, b = weights(n, k, seed=n)
    x = activations(shape, dtype, seed=k)
    y = check(x, w, s, b, dim)
    first = x[:1] if dim == 1 else x[:37]  # the bits do not depend on the company
    assert torch.equal(mx.int8_linear(first, w, s, b, dim=dim), y[: first.shape[0]])

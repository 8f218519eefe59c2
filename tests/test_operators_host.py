"""What the layer norm, dropout and 8-bit product operators do without a GPU: refusals of
the C entry points and of the Python functions, workspace sizes, and the generator's
published answers."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import mednext_accel_b200 as mx
from mednext_accel_b200 import _native as nat

from philox import dropout_words, philox4x32_10

FAKE = 1 << 20  # never dereferenced: validation fails first


@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_generator_gives_its_published_answers(counter, key, want):
    assert tuple(int(v[0]) for v in philox4x32_10(counter, key)) == want


def test_words_do_not_depend_on_where_a_range_begins():
    whole = dropout_words(3, 4, 0, 100)
    for begin in (1, 8, 13, 99):
        assert np.array_equal(dropout_words(3, 4, begin, 100 - begin), whole[begin:])


def test_layer_norm_refusals():
    lib = nat.load()
    ok = (FAKE, None, None, FAKE, None, 4, 8, 1, 1e-6, 1, 0, None)

    def fwd(**kw):
        names = ("x", "w", "b", "y", "stats", "outer", "c", "inner", "eps", "dtype", "pdt", "stream")
        return lib.mednext_ln_fwd(*(kw.get(n, v) for n, v in zip(names, ok, strict=True)))

    assert fwd(x=None) == nat.ERR_NULL_POINTER
    assert fwd(y=None) == nat.ERR_NULL_POINTER
    assert fwd(c=0) == nat.ERR_BAD_SHAPE
    assert fwd(outer=-1) == nat.ERR_BAD_SHAPE
    assert fwd(outer=1 << 39, inner=1 << 39) == nat.ERR_BAD_SHAPE
    assert fwd(outer=1 << 39, c=1 << 20) == nat.ERR_BAD_SHAPE
    assert fwd(dtype=3) == nat.ERR_BAD_DTYPE
    assert fwd(pdt=2) == nat.ERR_BAD_DTYPE
    assert fwd(eps=0.0) == nat.ERR_BAD_VALUE
    assert fwd(eps=float("inf")) == nat.ERR_BAD_VALUE
    assert fwd(x=FAKE + 1) == nat.ERR_ALIGNMENT
    assert fwd(w=FAKE + 2) == nat.ERR_ALIGNMENT
    assert fwd(stats=FAKE + 4) == nat.ERR_ALIGNMENT
    assert fwd(outer=0, x=None, y=None) == nat.OK  # nothing to do
    need = lib.mednext_ln_bwd_workspace_size(4, 8, 1, 1)
    assert need > 0 and lib.mednext_ln_bwd_workspace_size(4, 0, 1, 1) == 0
    bwd = lambda ws, nbytes, stats=FAKE: lib.mednext_ln_bwd(  # noqa: E731
        FAKE, FAKE, stats, None, FAKE, FAKE, FAKE, ws, nbytes, 4, 8, 1, 1, 0, None)
    assert bwd(FAKE, need - 1) == nat.ERR_WORKSPACE
    assert bwd(None, need) == nat.ERR_WORKSPACE
    assert bwd(FAKE, need, None) == nat.ERR_NULL_POINTER


def test_dropout_refusals():
    lib = nat.load()
    call = lambda x=FAKE, y=FAKE, rng=None, n=8, drop=100, dtype=1: lib.mednext_dropout(  # noqa: E731
        x, None, y, rng, 0, 0, None, n, drop, dtype, None)
    assert call(x=None) == nat.ERR_NULL_POINTER
    assert call(n=-1) == nat.ERR_BAD_SHAPE
    assert call(drop=65537) == nat.ERR_BAD_VALUE
    assert call(drop=-1) == nat.ERR_BAD_VALUE
    assert call(dtype=3) == nat.ERR_BAD_DTYPE
    assert call(x=FAKE + 1) == nat.ERR_ALIGNMENT
    assert call(rng=FAKE + 4) == nat.ERR_ALIGNMENT
    assert call(n=0, x=None, y=None) == nat.OK


def test_int8_refusals():
    lib = nat.load()
    need = lib.mednext_int8_linear_workspace_size(100, 40, 1, 24, 1)
    assert need >= 100 * 48 + 400
    names = ("x", "w", "s", "b", "y", "ws", "bytes", "outer", "k", "inner", "n", "pitch", "dtype", "stream")
    ok = (FAKE, FAKE, FAKE, None, FAKE, FAKE, need, 100, 40, 1, 24, 48, 1, None)

    def call(**kw):
        return lib.mednext_int8_linear(*(kw.get(n, v) for n, v in zip(names, ok, strict=True)))

    for name in ("x", "w", "s", "y"):
        assert call(**{name: None}) == nat.ERR_NULL_POINTER
    assert call(k=131073, pitch=131088) == nat.ERR_BAD_SHAPE
    assert call(n=0) == nat.ERR_BAD_SHAPE
    assert call(pitch=40) == nat.ERR_BAD_SHAPE
    assert call(pitch=32) == nat.ERR_BAD_SHAPE
    assert call(outer=1 << 20, inner=1 << 20) == nat.ERR_BAD_SHAPE
    assert call(dtype=3) == nat.ERR_BAD_DTYPE
    assert call(w=FAKE + 8) == nat.ERR_ALIGNMENT
    assert call(ws=None) == nat.ERR_WORKSPACE
    assert call(bytes=need - 1) == nat.ERR_WORKSPACE
    assert call(outer=0, x=None) == nat.OK
    quantize = lambda pitch=48, q=FAKE: lib.mednext_int8_quantize(FAKE, q, FAKE, 4, 40, 1, pitch, 1, None)  # noqa: E731
    assert quantize(pitch=32) == nat.ERR_BAD_SHAPE
    assert quantize(pitch=44) == nat.ERR_BAD_SHAPE
    assert quantize(q=FAKE + 8) == nat.ERR_ALIGNMENT
    assert quantize(q=None) == nat.ERR_NULL_POINTER


def test_tensors_on_the_cpu_are_refused():
    x = torch.zeros((4, 8))
    with pytest.raises(ValueError, match="CUDA"):
        mx.layer_norm(x)
    with pytest.raises(ValueError, match="CUDA"):
        mx.dropout(x, 0.5, (1, 2))
    with pytest.raises(ValueError, match="CUDA"):
        mx.int8_linear(x, torch.zeros((4, 8), dtype=torch.int8), torch.ones(4))
    with pytest.raises(ValueError, match="CUDA"):
        mx.quantize_int8(x)
    with pytest.raises(ValueError, match="positive"):
        mx.LayerNorm3d(0)


def test_8_bit_convolutions_refuse_transposed_weights():
    """A transposed convolution's weight is [in, out]: its rows are not the output channels."""
    for cin, cout in ((8, 8), (4, 12)):
        with pytest.raises(ValueError, match="1x1x1"):
            mx.Int8Pointwise3d(torch.nn.ConvTranspose3d(cin, cout, 1))
    head = mx.mednext_small(in_channels=1, out_channels=3, kernel_size=3)
    heads = [m for m in head.modules() if getattr(m, "transposed", False) and set(m.kernel_size) == {1}]
    assert heads
    for m in heads:
        with pytest.raises(ValueError, match="1x1x1"):
            mx.Int8Pointwise3d(m)


@pytest.mark.parametrize("padding", ["same", "valid", 0, (0, 0, 0)])
def test_8_bit_convolutions_take_every_way_to_say_no_padding(padding):
    with pytest.raises(ValueError, match="CUDA"):  # nothing but the device is refused
        mx.Int8Pointwise3d(torch.nn.Conv3d(4, 8, 1, padding=padding))
    with pytest.raises(ValueError, match="1x1x1"):
        mx.Int8Pointwise3d(torch.nn.Conv3d(4, 8, 1, padding=1))

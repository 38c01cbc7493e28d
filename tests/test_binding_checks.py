"""What the Python binding refuses and accepts before a call reaches the library, without a device (a context
handle of None: the library's own refusal is "null context")."""

import ctypes

import numpy as np
import pytest

from helpers import amd


@pytest.fixture
def ctx():
    c = amd().Context.__new__(amd().Context)
    c.h = None
    return c


def weight():
    return amd().weight(amd().W_F8, 32, 64, 0x10000, scale=0x10000)


def reaches(call):
    with pytest.raises(amd().AnimaError, match="null context"):
        call()


@pytest.mark.parametrize("W", [None, 5, b"x", "LinearDesc", "pointer"])
def test_weights_by_type(ctx, W):
    """Anything but a Weight in a weight's place is refused, also another ctypes object."""
    W = {"LinearDesc": amd().LinearDesc(), "pointer": ctypes.pointer(weight())}.get(W, W) if isinstance(W, str) else W
    good = weight()
    reaches(lambda: ctx.linear(good, 1, 0x10000, x=0x10000))
    reaches(lambda: ctx.linear_glu(good, good, 1, x=0x10000, out=0x10000))
    for call in (lambda: ctx.linear(W, 1, 0x10000, x=0x10000), lambda: ctx.linear_glu(W, good, 1, x=0x10000, out=0x10000),
                 lambda: ctx.linear_glu(good, W, 1, x=0x10000, out=0x10000)):
        with pytest.raises(TypeError):
            call()


@pytest.mark.parametrize("flag", [True, False, 1, 0, np.bool_(True), np.bool_(False), np.int32(1)])
def test_flags(ctx, flag):
    """Truth values of any kind, numpy's among them."""
    reaches(lambda: ctx.linear(weight(), 1, 0x10000, x=0x10000, x_rotated=flag, out_bf16=flag))
    reaches(lambda: ctx.residual_norm(1, 64, 0x10000, y=0x10000, y_bf16=flag, h=0x10000))
    reaches(lambda: ctx.quant_rows_f8(0x10000, 1, 64, 0x10000, 0x10000, bf16=flag))


def test_released_buffers(ctx):
    """A released buffer is a null pointer, which the library refuses."""
    b = amd().DeviceBuffer.__new__(amd().DeviceBuffer)
    b.ptr = None
    reaches(lambda: ctx.linear(weight(), 1, b, x=b))
    reaches(lambda: ctx.linear_glu(weight(), weight(), 1, x=b, out=b))
    reaches(lambda: ctx.residual_norm(1, 64, b, h=b))


@pytest.mark.parametrize("name,cls", [("anima_linear", "LinearDesc"), ("anima_linear_glu", "GluDesc"),
                                      ("anima_residual_norm", "ResNormDesc")])
def test_entry_points_take_their_descriptor(name, cls):
    """The loaded library's functions take their own descriptor, by value or by reference, and no other struct."""
    f, m = getattr(amd().lib(), name), amd()
    d = getattr(m, cls)()
    assert f(None, d) == f(None, ctypes.byref(d)) == f(None, None) == -1
    for other in (m.Weight(), b"bytes", 7):
        with pytest.raises(ctypes.ArgumentError):
            f(None, other)

"""GPU parity: gelu and its slope far to the left, where they are small, relative to themselves.

Both go through the epilogue of an empty product: z is the bias, exact in bf16; the slope's products with ones are read from dbias,
a sum over one row. Tolerances: the exponent v = z^2 / 2 is off by a half-ulp of each of two products and of a constant, 3 |v| 2^-24 in
all, which is the relative error of exp; the function beside it, exp and the reciprocal of the hardware and the products are within
2^-20 together. In the slope P(z) + z p(z), p the density, the two terms are within that of themselves, so it is within that of
the sum of their magnitudes.
"""
import numpy as np
import pytest
from scipy.special import ndtr

import ffn_reference as ref
from dotcompute_amd import hip

pytestmark = pytest.mark.gpu


def points():
    z = ref.to_bf16(np.concatenate([-np.geomspace(1e-3, 12.8, 800), np.geomspace(1e-3, 12.8, 200)]))
    return z, ref.from_bf16(z).astype(np.float64)


def relative(z):
    return 3 * 2.0 ** -24 * z * z / 2 + 2.0 ** -20


def empty(ctx, e, rows):
    return hip.DeviceArray(ctx, e.ptr, 0, np.dtype(np.uint16), (rows, 0))


def test_gelu(ctx):
    bits, z = points()
    b, e, y = ctx.to_device(bits), ctx.empty(8, np.uint16), ctx.empty((1, z.size), np.float32)
    ctx.linear(hip.Linear.of(empty(ctx, e, 1), empty(ctx, e, z.size), y, bias=b, activation="gelu"))
    ctx.synchronize()
    want = z * ndtr(z)
    off = np.abs(y.to_host()[0] - want) / np.abs(want)
    assert np.all(off <= relative(z)), (z[np.argmax(off / relative(z))], np.max(off))
    for a in (b, e, y):
        ctx.free(a)


def test_slope_of_gelu(ctx):
    bits, z = points()
    ones, pre, db = ctx.to_device(ref.to_bf16(np.ones((1, z.size)))), ctx.to_device(bits.reshape(1, -1)), ctx.empty(z.size, np.float32)
    e = ctx.empty(8, np.uint16)
    ctx.linear_backward(hip.LinearGrad.of(ones, empty(ctx, e, 1), empty(ctx, e, z.size), pre=pre, dbias=db, activation="gelu"))
    ctx.synchronize()
    density = np.exp(-0.5 * z * z) / np.sqrt(2 * np.pi)
    off = np.abs(db.to_host() - (ndtr(z) + z * density))
    bound = relative(z) * (ndtr(z) + np.abs(z) * density)
    assert np.all(off <= bound), (z[np.argmax(off / bound)], np.max(off / bound))
    for a in (ones, pre, db, e):
        ctx.free(a)

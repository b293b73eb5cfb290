"""GPU parity: RMS norm with the residual's addition, its gradients, and rows in 8 bits, against float64.

Tolerances, from the arithmetic: a float32 sum of n squares in lanes and a tree is within (n / 64 + 12) half-ulps, its
root halves that, and a handful of roundings follow: 4e-6 of a value for the rows here (at most 66,000 long, 1032 terms a
lane in 16 waves: 65 in a row). Results in bf16 add half a step of 8 bits, in e4m3 half a step of 4 bits or of the smallest
value. The weight's gradient adds up to 1024 / 16 parts and 3 rows each after one another: 1e-5 of the sum of magnitudes.
"""
import numpy as np
import pytest

import ffn_reference as ref
from dotcompute_amd import hip

pytestmark = pytest.mark.gpu
F32 = 4e-6
EPS = 1e-6


class Matrix:
    """A row-major matrix inside a device buffer: `shift` elements in, `pad` more columns a row; every other element of the
    buffer keeps the pattern it was made with."""

    def __init__(self, ctx, host, dtype, shift=0, pad=0):
        rows, cols = host.shape
        self.ctx, self.shift, self.shape, self.stride = ctx, shift, host.shape, cols + pad
        self.host = np.full(shift + rows * self.stride + 8, 77, dtype)
        self.view(self.host)[:] = host
        self.base = ctx.to_device(self.host)
        self.a = hip.DeviceArray(ctx, self.base.ptr + shift * np.dtype(dtype).itemsize, host.nbytes, np.dtype(dtype), host.shape)

    def view(self, flat):
        rows, cols = self.shape
        return flat[self.shift:self.shift + rows * self.stride].reshape(rows, self.stride)[:, :cols]

    def read(self):
        """The matrix, after a look at what surrounds it."""
        now = self.base.to_host()
        out = self.view(now).copy()
        self.view(now)[:] = self.view(self.host)
        assert np.array_equal(now, self.host), "written outside the matrix"
        return out


def values(rng, shape, dtype, scale=1.0, shift=0.0):
    x = (rng.normal(size=shape) * scale + shift).astype(np.float32)
    return ref.to_bf16(x) if dtype == "bf16" else x


def wide(x):
    return (ref.from_bf16(x) if x.dtype == np.uint16 else x).astype(np.float64)


def close(got, want, dtype, what, extra=0.0):
    bound = np.abs(want) * (F32 + (ref.BF16 * (1 + F32) if dtype == "bf16" else 0.0)) + extra + 1e-37
    off = np.abs(wide(got) - want)
    assert np.all(off <= bound), f"{what}: {np.max(off / bound):.3g} of the bound"


# Rows by shape of the kernel: a wave a row (many short rows), 4 and 16 waves a row, rows read again; odd lengths among them.
SHAPES = [(1, 1), (1, 64), (3, 7), (5, 2050), (2, 4096), (7, 3333), (2, 8191), (3, 16384), (2, 30001), (1, 65536), (2, 66001),
          (2049, 100), (2048, 513), (2050, 2047), (2051, 4096)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_rms_norm(ctx, rows, cols, dtype):
    rng = np.random.default_rng(rows * 7 + cols)
    np_t = np.uint16 if dtype == "bf16" else np.float32
    odd = cols % 2  # odd rows lie one element into their buffers, further apart than they are long
    x = Matrix(ctx, values(rng, (rows, cols), dtype), np_t, odd, 3 * odd)
    r = Matrix(ctx, values(rng, (rows, cols), dtype), np_t, odd, odd)
    w = Matrix(ctx, values(rng, (1, cols), dtype, 0.1, 1.0), np_t, odd)
    h = Matrix(ctx, np.zeros((rows, cols), np_t), np_t, 0, odd)
    y = Matrix(ctx, np.zeros((rows, cols), np_t), np_t, odd, 5 * odd)
    w1 = hip.DeviceArray(ctx, w.a.ptr, w.a.nbytes, w.a.dtype, (cols,))
    ctx.rms_norm(hip.RmsNorm.of(x.a, w1, y.a, residual=r.a, sum=h.a, eps=EPS, x_stride=x.stride, residual_stride=r.stride,
                                sum_stride=h.stride, y_stride=y.stride))
    ctx.synchronize()
    h64, y64 = ref.rms_norm(wide(x.view(x.host)), wide(w.view(w.host))[0], EPS, wide(r.view(r.host)))
    close(h.read(), h64, dtype, "sum")
    close(y.read(), y64, dtype, "y")
    for m in (x, r, w):
        m.read()
    # the same without a residual, in 8 bits
    q, scales = Matrix(ctx, np.zeros((rows, cols), np.uint8), np.uint8, odd, 3 * odd), ctx.empty(rows, np.float32)
    ctx.rms_norm(hip.RmsNorm.of(x.a, w1, q.a, scales=scales, eps=EPS, x_stride=x.stride, y_stride=q.stride))
    ctx.synchronize()
    check_fp8(q.read(), scales.to_host(), ref.rms_norm(wide(x.view(x.host)), wide(w.view(w.host))[0], EPS)[1])
    for a in (x.base, r.base, w.base, h.base, y.base, q.base, scales):
        ctx.free(a)


def check_fp8(q, scales, y64):
    top = np.max(np.abs(y64), axis=1)
    assert np.all(np.abs(scales - top / ref.TOP) <= 2 * F32 * top / ref.TOP + 1e-44)
    got = ref.from_fp8(q).astype(np.float64) * scales[:, None]
    bound = np.maximum(np.abs(y64) * ref.FP8, (ref.LEAST / 2) * scales[:, None].astype(np.float64)) * (1 + 1e-4) + 1e-44
    off = np.abs(got - y64)
    assert np.all(off <= bound), np.max(off / bound)


# Rows that one wave holds, with one chunk a lane and with two, and the first that it does not; rows that leave waves without one.
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(5, 256), (6, 257), (7, 511), (9, 512), (3, 513), (1030, 1001), (2, 1024), (5, 1025)])
def test_rms_norm_of_a_wave_a_row(ctx, rows, cols, dtype):
    test_rms_norm(ctx, rows, cols, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 1000), (4, 70001), (2100, 129)])
def test_quantize(ctx, rows, cols, dtype):
    rng = np.random.default_rng(cols)
    x = values(rng, (rows, cols), dtype, 5.0)
    dx, q, s = ctx.to_device(x), ctx.empty((rows, cols), np.uint8), ctx.empty(rows, np.float32)
    ctx.quantize_fp8(dx, q, s)
    ctx.synchronize()
    want, ws = ref.rows_fp8(wide(x).astype(np.float32))
    assert np.array_equal(s.to_host(), ws) and np.array_equal(q.to_host(), want)  # a division and a product: the same bits
    for a in (dx, q, s):
        ctx.free(a)


def test_sum_and_y_in_place(ctx):
    """sum over the residual, y over x: as a block that keeps one buffer for its running sum calls it."""
    rng = np.random.default_rng(5)
    for rows, cols in ((3, 4096), (2, 66001), (2049, 300)):
        x, r, w = (values(rng, s, "bf16") for s in ((rows, cols), (rows, cols), (cols,)))
        dx, dr, dw = ctx.to_device(x), ctx.to_device(r), ctx.to_device(w)
        ctx.rms_norm(hip.RmsNorm.of(dx, dw, dx, residual=dr, sum=dr, eps=EPS))
        ctx.synchronize()
        h64, y64 = ref.rms_norm(wide(x), wide(w), EPS, wide(r))
        close(dr.to_host(), h64, "bf16", "sum")
        close(dx.to_host(), y64, "bf16", "y")
        for a in (dx, dr, dw):
            ctx.free(a)


def test_rows_of_zeros_infinities_and_nan(ctx):
    cols = 300
    x = np.random.default_rng(6).normal(size=(6, cols)).astype(np.float32)
    x[1] = 0.0
    x[2, 17] = np.inf
    x[3, 299] = np.nan
    x[4] *= 1e-30  # (their squares vanish: eps alone is left)
    w = np.ones(cols, np.float32)
    dx, dw, y = ctx.to_device(x), ctx.to_device(w), ctx.empty((6, cols), np.float32)
    q, s = ctx.empty((6, cols), np.uint8), ctx.empty(6, np.float32)
    ctx.rms_norm(hip.RmsNorm.of(dx, dw, y, eps=EPS))
    ctx.rms_norm(hip.RmsNorm.of(dx, dw, q, scales=s, eps=EPS))
    ctx.synchronize()
    got, codes, scales = y.to_host(), q.to_host(), s.to_host()
    good = [0, 1, 4, 5]
    _, y64 = ref.rms_norm(x[good].astype(np.float64), w.astype(np.float64), EPS)
    close(got[good], y64, "f32", "y")
    check_fp8(codes[good], scales[good], y64)
    assert np.all(got[1] == 0) and np.all(codes[1] == 0) and scales[1] == 0
    # an infinity over an infinite root is no number, the row's other values over it are zero; a NaN reaches its row
    assert np.isnan(got[2, 17]) and np.all(np.delete(got[2], 17) == 0) and np.all(np.isnan(got[3]))
    assert np.isnan(scales[2]) and np.isnan(scales[3])
    # no eps and nothing in the row: 0 / 0, as the formula says
    ctx.rms_norm(hip.RmsNorm.of(dx, dw, y, eps=0.0))
    ctx.synchronize()
    assert np.all(np.isnan(y.to_host()[1])) and np.all(np.isfinite(y.to_host()[0]))
    for a in (dx, dw, y, q, s):
        ctx.free(a)


GRAD_SHAPES = [(1, 1), (1, 300), (4, 7), (1500, 512), (1031, 2050), (9, 4096), (5, 8192), (3, 20001), (2, 32768), (3, 40001)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", GRAD_SHAPES)
def test_rms_norm_backward(ctx, rows, cols, dtype):
    rng = np.random.default_rng(rows + cols)
    np_t = np.uint16 if dtype == "bf16" else np.float32
    odd = cols % 2
    dy, h, dh = (Matrix(ctx, values(rng, (rows, cols), dtype), np_t, odd, p * odd) for p in (1, 2, 3))
    w = values(rng, (cols,), dtype, 0.1, 1.0)
    dx, dw, dwt = Matrix(ctx, np.zeros((rows, cols), np_t), np_t, odd, odd), ctx.to_device(w), ctx.empty(cols, np.float32)
    args = dict(dy=dy.a, h=h.a, weight=dw, eps=EPS, dy_stride=dy.stride, h_stride=h.stride)
    ctx.rms_norm_backward(hip.RmsNormGrad.of(dh=dh.a, dx=dx.a, dweight=dwt, dh_stride=dh.stride, dx_stride=dx.stride, **args))
    ctx.synchronize()
    hv, dv, wv = wide(h.view(h.host)), wide(dy.view(dy.host)), wide(w)
    x64, w64 = ref.rms_norm_grad(dv, hv, wv, EPS, wide(dh.view(dh.host)))
    s = 1.0 / np.sqrt(np.mean(hv * hv, axis=1, keepdims=True) + EPS)
    g = np.abs(dv * wv)
    terms = s * (g + np.abs(hv) * s * np.mean(g * np.abs(hv) * s, axis=1, keepdims=True)) + np.abs(wide(dh.view(dh.host)))
    close(dx.read(), x64, dtype, "dx", F32 * terms)
    first = dwt.to_host()
    assert np.all(np.abs(first - w64) <= 1e-5 * np.sum(np.abs(dv * hv * s), axis=0) + 1e-37)
    # each gradient alone, without dh: the weight's are the same bits
    ctx.rms_norm_backward(hip.RmsNormGrad.of(dweight=dwt, **args))
    ctx.rms_norm_backward(hip.RmsNormGrad.of(dx=dx.a, dx_stride=dx.stride, **args))
    ctx.synchronize()
    assert np.array_equal(dwt.to_host(), first)
    close(dx.read(), ref.rms_norm_grad(dv, hv, wv, EPS)[0], dtype, "dx alone", F32 * terms)
    for a in (dy.base, h.base, dh.base, dx.base, dw, dwt):
        ctx.free(a)


# Widths on both sides of those where a row's gradient takes another form (float32 2048, 8192, 16384; bf16 8192, 16384), with
# rows enough for workgroups that walk over several.
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(600, 2052), (300, 4097), (530, 8192), (300, 8197), (520, 16381), (270, 16384), (260, 16385)])
def test_rms_norm_backward_of_wide_rows(ctx, rows, cols, dtype):
    test_rms_norm_backward(ctx, rows, cols, dtype)


def test_nothing_to_do(ctx):
    """No rows: nothing is written but the empty sum; no columns: nothing at all."""
    f = ctx.to_device(np.full(4, 7.0, np.float32))
    e = ctx.empty(1, np.float32)
    none = hip.DeviceArray(ctx, e.ptr, 0, np.dtype(np.float32), (0, 4))
    ctx.rms_norm(hip.RmsNorm.of(none, f, none))
    ctx.rms_norm_backward(hip.RmsNormGrad.of(dy=none, h=none, weight=f, dx=none, dweight=f))
    ctx.synchronize()
    assert np.all(f.to_host() == 0)
    ctx.free(f)
    ctx.free(e)

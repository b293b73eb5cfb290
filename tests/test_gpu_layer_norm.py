"""GPU parity: layer norm with the residual's addition, its gradients, and rows in 8 bits with block scales, against float64.

Tolerances, from the arithmetic. A float32 sum of n terms in lanes and a tree is within (n / 1024 + 20) half-steps of the sum of their magnitudes, which is
4e-6 of it for the rows here (at most 66,000 long: 65 terms in a row). The mean is held in two parts, so it is that close in terms of the
deviations, as is the root of their squares: u = (h - mean) s is within 8e-6 (|u| + 1), the 1 being the mean of |u| at most. h itself is a float32
sum, half a step of its magnitude off the exact one, times s. Results in bf16 add half a step of 8 bits, in e4m3 half a step of 4 bits or of the
smallest value. The weights' gradients add up to 1024 / 16 parts and 3 rows each after one another: 1e-5 of the sum of magnitudes.
"""
import numpy as np
import pytest

import ffn_reference as ref
import gated_reference as gated
from dotcompute_amd import hip
from test_gpu_rms_norm import Matrix, values, wide

pytestmark = pytest.mark.gpu
F32 = 8e-6
HALF = 2.0 ** -24
EPS = 1e-5


def within(got, want, bound, what):
    off = np.abs(wide(got) - want)
    assert np.all(off <= bound), f"{what}: {np.max(off / bound):.3g} of the bound"


def unit(h):
    d = h - np.mean(h, axis=1, keepdims=True)
    s = 1.0 / np.sqrt(np.mean(d * d, axis=1, keepdims=True) + EPS)
    return d * s, s


def y_bound(h, w, b, y, dtype):
    u, s = unit(h)
    bound = np.abs(w) * (F32 * (np.abs(u) + 1) + HALF * np.abs(h) * s) + 2 * HALF * (np.abs(y) + (0 if b is None else np.abs(b)))
    return bound + (ref.BF16 * (1 + F32) * np.abs(y) if dtype == "bf16" else 0.0) + 1e-37


def check_blocks(q, scales, y, bound):
    """Codes with block scales, each within half a step of y's own error bound; the scales are y's own but where y's error may cross a border."""
    top = np.max(gated._blocked(np.abs(y)), axis=2)
    off = np.max(gated._blocked(np.broadcast_to(bound, y.shape)), axis=2)
    low, high = gated.scale_of(np.maximum(top - off, 0)).T, gated.scale_of(top + off).T
    assert np.all((scales >= low) & (scales <= high))
    step = np.repeat(gated.scale_value(scales).T, gated.BLOCK, axis=1)[:, :y.shape[1]]
    got = gated.values(q, scales)
    limit = np.maximum(np.abs(y) * ref.FP8, step * ref.LEAST / 2) * (1 + 1e-4) + bound
    assert np.all(np.abs(got - y) <= limit), np.max(np.abs(got - y) / limit)


# Rows by shape of the kernel: a wave a row (many short rows), 4 and 16 waves a row, rows read again; odd lengths among them.
SHAPES = [(1, 1), (1, 64), (3, 7), (5, 2050), (2, 4096), (7, 3333), (2, 8191), (3, 16384), (2, 30001), (1, 65536), (2, 66001),
          (2049, 100), (2048, 513), (2050, 2047), (2051, 4096), (5, 256), (6, 257), (9, 512), (1030, 1001), (2, 1024), (5, 1025),
          (300, 6001), (270, 12001), (260, 16384), (256, 4100), (257, 4100)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_layer_norm(ctx, rows, cols, dtype, mean=0.5):
    rng = np.random.default_rng(rows * 7 + cols)
    np_t = np.uint16 if dtype == "bf16" else np.float32
    odd = cols % 2  # odd rows lie one element into their buffers, further apart than they are long
    x = Matrix(ctx, values(rng, (rows, cols), dtype, 1.0, mean), np_t, odd, 3 * odd)
    r = Matrix(ctx, values(rng, (rows, cols), dtype), np_t, odd, odd)
    w, b = (values(rng, (cols,), dtype, 0.1, shift) for shift in (1.0, 0.0))
    dw, db = ctx.to_device(w), ctx.to_device(b)
    h = Matrix(ctx, np.zeros((rows, cols), np_t), np_t, 0, odd)
    y = Matrix(ctx, np.zeros((rows, cols), np_t), np_t, odd, 5 * odd)
    ctx.layer_norm(hip.LayerNorm.of(x.a, dw, db, y.a, residual=r.a, sum=h.a, eps=EPS, x_stride=x.stride, residual_stride=r.stride,
                                    sum_stride=h.stride, y_stride=y.stride))
    ctx.synchronize()
    x64, w64, b64 = wide(x.view(x.host)), wide(w), wide(b)
    h64, y64 = gated.layer_norm(x64, w64, b64, EPS, wide(r.view(r.host)))
    within(h.read(), h64, np.abs(h64) * (HALF + (ref.BF16 * (1 + F32) if dtype == "bf16" else 0)) + 1e-37, "sum")
    within(y.read(), y64, y_bound(h64, w64, b64, y64, dtype), "y")
    for m in (x, r):
        m.read()
    # the same without a residual, in 8 bits with a scale a row, and with block scales
    _, y64 = gated.layer_norm(x64, w64, b64, EPS)
    bound = y_bound(x64, w64, b64, y64, "f32")
    q, scales = Matrix(ctx, np.zeros((rows, cols), np.uint8), np.uint8, odd, 3 * odd), ctx.empty(rows, np.float32)
    ctx.layer_norm(hip.LayerNorm.of(x.a, dw, db, q.a, scales=scales, eps=EPS, x_stride=x.stride, y_stride=q.stride))
    block = Matrix(ctx, np.zeros((gated.blocks(cols), rows), np.uint8), np.uint8, 3 * odd, 5 * odd)
    q2 = Matrix(ctx, np.zeros((rows, cols), np.uint8), np.uint8, odd, odd)
    ctx.layer_norm(hip.LayerNorm.of(x.a, dw, db, q2.a, scales=block.a, eps=EPS, x_stride=x.stride, y_stride=q2.stride,
                                    scales_stride=block.stride))
    ctx.synchronize()
    codes, s = q.read(), scales.to_host()
    top = np.max(np.abs(y64), axis=1)
    assert np.all(np.abs(s - top / ref.TOP) <= np.max(bound, axis=1) / ref.TOP + 4 * HALF * top / ref.TOP + 1e-44)
    limit = np.maximum(np.abs(y64) * ref.FP8, s[:, None].astype(np.float64) * ref.LEAST / 2) * (1 + 1e-4) + bound + 1e-44
    assert np.all(np.abs(ref.from_fp8(codes).astype(np.float64) * s[:, None] - y64) <= limit)
    check_blocks(q2.read(), block.read(), y64, bound)
    for a in (x.base, r.base, dw, db, h.base, y.base, q.base, q2.base, scales, block.base):
        ctx.free(a)


@pytest.mark.parametrize("rows,cols", [(3, 100), (4, 4096), (2, 12000), (1, 66001)])
def test_layer_norm_of_values_far_from_zero(ctx, rows, cols):
    """A mean of 300 deviations: the variance keeps its digits."""
    test_layer_norm(ctx, rows, cols, "f32", 300.0)


def test_layer_norm_without_bias_and_in_place(ctx):
    """sum over the residual, y over x: as a block that keeps one buffer for its running sum calls it."""
    rng = np.random.default_rng(5)
    for rows, cols in ((3, 4096), (2, 66001), (2049, 300)):
        x, r, w = (values(rng, s, "bf16") for s in ((rows, cols), (rows, cols), (cols,)))
        dx, dr, dw = ctx.to_device(x), ctx.to_device(r), ctx.to_device(w)
        ctx.layer_norm(hip.LayerNorm.of(dx, dw, None, dx, residual=dr, sum=dr, eps=EPS))
        ctx.synchronize()
        h64, y64 = gated.layer_norm(wide(x), wide(w), None, EPS, wide(r))
        within(dr.to_host(), h64, np.abs(h64) * (HALF + ref.BF16 * (1 + F32)) + 1e-37, "sum")
        within(dx.to_host(), y64, y_bound(h64, wide(w), None, y64, "bf16"), "y")
        for a in (dx, dr, dw):
            ctx.free(a)


def test_layer_norm_of_flat_rows_infinities_and_nan(ctx):
    cols = 300
    x = np.random.default_rng(6).normal(size=(7, cols)).astype(np.float32)
    x[1] = 0.0
    x[2, 17] = np.inf
    x[3, 299] = np.nan
    x[4] *= 1e-30  # (their squares vanish: eps alone is left)
    x[5] = 3.0  # no deviation
    w, b = np.ones(cols, np.float32), np.full(cols, 0.25, np.float32)
    dx, dw, db, y = ctx.to_device(x), ctx.to_device(w), ctx.to_device(b), ctx.empty((7, cols), np.float32)
    q, s, k = ctx.empty((7, cols), np.uint8), ctx.empty(7, np.float32), ctx.empty((3, 7), np.uint8)
    ctx.layer_norm(hip.LayerNorm.of(dx, dw, db, y, eps=EPS))
    ctx.layer_norm(hip.LayerNorm.of(dx, dw, db, q, scales=s, eps=EPS))
    ctx.synchronize()
    got, codes, scales = y.to_host(), q.to_host(), s.to_host()
    good = [0, 1, 4, 5, 6]
    h64 = x[good].astype(np.float64)
    _, y64 = gated.layer_norm(h64, w.astype(np.float64), b.astype(np.float64), EPS)
    within(got[good], y64, y_bound(h64, w, b, y64, "f32"), "y")
    assert np.all(got[1] == 0.25) and np.all(got[5] == 0.25)
    # an infinity or a NaN reaches its row through the mean, and no other
    assert np.all(np.isnan(got[2:4])) and np.all(np.isnan(scales[2:4])) and np.all(np.isfinite(scales[good]))
    ctx.layer_norm(hip.LayerNorm.of(dx, dw, db, q, scales=k, eps=EPS))
    ctx.synchronize()
    codes, scales = q.to_host(), k.to_host()
    assert np.all(scales[:, 2:4] == 255) and np.all(scales[:, good] < 255)
    check_blocks(codes[good], scales[:, good], y64, y_bound(h64, w, b, y64, "f32"))
    # no eps and no deviation: 0 / 0, as the formula says
    ctx.layer_norm(hip.LayerNorm.of(dx, dw, db, y, eps=0.0))
    ctx.synchronize()
    assert np.all(np.isnan(y.to_host()[5])) and np.all(np.isfinite(y.to_host()[0]))
    for a in (dx, dw, db, y, q, s, k):
        ctx.free(a)


GRAD_SHAPES = [(1, 1), (1, 300), (4, 7), (1500, 512), (1031, 2050), (9, 4096), (5, 8192), (3, 20001), (2, 32768), (3, 40001), (600, 2052),
               (300, 4097), (530, 8192), (300, 8197), (520, 16381), (270, 16384), (260, 16385), (1027, 1030), (4099, 130), (257, 513), (700, 1601),
               (515, 2816), (1300, 3000), (9000, 8)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", GRAD_SHAPES)
def test_layer_norm_backward(ctx, rows, cols, dtype):
    rng = np.random.default_rng(rows + cols)
    np_t = np.uint16 if dtype == "bf16" else np.float32
    odd = cols % 2
    dy, dh = (Matrix(ctx, values(rng, (rows, cols), dtype), np_t, odd, p * odd) for p in (1, 3))
    h = Matrix(ctx, values(rng, (rows, cols), dtype, 1.0, 2.0), np_t, odd, 2 * odd)
    w = values(rng, (cols,), dtype, 0.1, 1.0)
    dx, dw = Matrix(ctx, np.zeros((rows, cols), np_t), np_t, odd, odd), ctx.to_device(w)
    dwt, dbt = ctx.empty(cols, np.float32), ctx.empty(cols, np.float32)
    args = dict(dy=dy.a, h=h.a, weight=dw, eps=EPS, dy_stride=dy.stride, h_stride=h.stride)
    ctx.layer_norm_backward(hip.LayerNormGrad.of(dh=dh.a, dx=dx.a, dweight=dwt, dbias=dbt, dh_stride=dh.stride, dx_stride=dx.stride, **args))
    ctx.synchronize()
    hv, dv, wv = wide(h.view(h.host)), wide(dy.view(dy.host)), wide(w)
    dh64 = wide(dh.view(dh.host))
    x64, w64, b64 = gated.layer_norm_grad(dv, hv, wv, EPS, dh64)
    u, s = unit(hv)
    g = np.abs(dv * wv)
    terms = s * (g + np.mean(g, axis=1, keepdims=True) + (np.abs(u) + 1) * np.mean(g * (np.abs(u) + 1), axis=1, keepdims=True))
    half = ref.BF16 * (1 + F32) if dtype == "bf16" else 0.0

    def bound(x, rest):
        return F32 * terms + np.abs(x) * half + 2 * HALF * (np.abs(x) + rest) + 1e-37

    within(dx.read(), x64, bound(x64, np.abs(dh64)), "dx")
    first = dwt.to_host(), dbt.to_host()
    assert np.all(np.abs(first[0] - w64) <= 1e-5 * np.sum(np.abs(dv) * (np.abs(u) + 1), axis=0) + 1e-37)
    assert np.all(np.abs(first[1] - b64) <= 1e-5 * np.sum(np.abs(dv), axis=0) + 1e-37)
    # each gradient alone, without dh: the weights' are the same bits
    dwt.copy_from(np.zeros(cols, np.float32))
    dbt.copy_from(np.zeros(cols, np.float32))
    ctx.layer_norm_backward(hip.LayerNormGrad.of(dweight=dwt, **args))
    ctx.layer_norm_backward(hip.LayerNormGrad.of(dbias=dbt, **args))
    ctx.layer_norm_backward(hip.LayerNormGrad.of(dx=dx.a, dx_stride=dx.stride, **args))
    ctx.synchronize()
    assert np.array_equal(dwt.to_host(), first[0]) and np.array_equal(dbt.to_host(), first[1])
    x64 = gated.layer_norm_grad(dv, hv, wv, EPS)[0]
    within(dx.read(), x64, bound(x64, 0.0), "dx alone")
    for a in (dy.base, h.base, dh.base, dx.base, dw, dwt, dbt):
        ctx.free(a)


def test_layer_norm_backward_against_differences(ctx):
    """The gradients are those of sum(y dy), by central differences in float64 of the reference, whose step's error is 1e-8 here."""
    rng = np.random.default_rng(11)
    h, dy, w, b = rng.normal(size=(2, 9)) + 1, rng.normal(size=(2, 9)), rng.normal(size=9), rng.normal(size=9)
    h, dy, w, b = (a.astype(np.float32) for a in (h, dy, w, b))
    arrays = [ctx.to_device(a) for a in (dy, h, w)] + [ctx.empty((2, 9), np.float32), ctx.empty(9, np.float32), ctx.empty(9, np.float32)]
    ctx.layer_norm_backward(hip.LayerNormGrad.of(*arrays, eps=EPS))
    ctx.synchronize()

    def loss(h_, w_, b_):
        return np.sum(gated.layer_norm(h_, w_, b_, EPS)[1] * dy)

    at = [a.astype(np.float64) for a in (h, w, b)]
    for i, got in enumerate(a.to_host() for a in arrays[3:]):
        for where in np.ndindex(got.shape):
            both = []
            for step in (1e-5, -1e-5):
                moved = [a.copy() for a in at]
                moved[i][where] += step
                both.append(loss(*moved))
            assert abs(got[where] - (both[0] - both[1]) / 2e-5) <= 1e-4, (i, where)
    for a in arrays:
        ctx.free(a)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 1000), (4, 70001), (2100, 129), (17, 512), (16, 513), (33, 4096), (5, 255)])
def test_quantize_blocks(ctx, rows, cols, dtype):
    """Powers of two and one rounding: the same bits. Rows of their own magnitudes, blocks at and next to the borders of a scale."""
    rng = np.random.default_rng(cols)
    x = rng.normal(size=(rows, cols)) * np.exp(rng.normal(size=(rows, 1)) * 3)
    x[:, ::131] = 0.0
    x[0, 0] = 448.0 * 2.0 ** 3  # exactly on a border
    if cols > 128:
        x[0, 128:256] = 0.0
        x[0, 200 % cols] = 450.0  # the next float of bf16 over one
    x = x.astype(np.float32) if dtype == "f32" else ref.to_bf16(x)
    odd = cols % 2
    m = Matrix(ctx, x, x.dtype, odd, 3 * odd)
    q = Matrix(ctx, np.zeros((rows, cols), np.uint8), np.uint8, odd, odd)
    s = Matrix(ctx, np.zeros((gated.blocks(cols), rows), np.uint8), np.uint8, odd, 5 * odd)
    ctx.quantize_fp8_blocks(m.a, q.a, s.a, x_stride=m.stride, q_stride=q.stride, scales_stride=s.stride)
    ctx.synchronize()
    want, ws = gated.rows_fp8(wide(x))
    assert np.array_equal(s.read(), ws) and np.array_equal(q.read(), want)
    for a in (m.base, q.base, s.base):
        ctx.free(a)


def test_quantize_blocks_of_the_ends(ctx):
    """Blocks of zeros, of the smallest and the largest floats; infinities and NaN make their block NaN and no other."""
    tiny, top = np.float32(1e-45), np.finfo(np.float32).max
    x = np.zeros((6, 300), np.float32)
    x[1, 3], x[1, 150], x[1, 290] = tiny, 2.0 ** -119, 1.75 * 2.0 ** -119
    x[2, 3], x[2, 150], x[2, 299] = top, -top, 1.0
    x[3, 127], x[4, 128], x[5, 299] = np.inf, np.nan, -np.inf
    x[5, :128] = np.linspace(-448, 448, 128, dtype=np.float32)
    dx, q, s = ctx.to_device(x), ctx.empty((6, 300), np.uint8), ctx.empty((3, 6), np.uint8)
    ctx.quantize_fp8_blocks(dx, q, s)
    ctx.synchronize()
    want, ws = gated.rows_fp8(x)
    codes, scales = q.to_host(), s.to_host()
    assert np.array_equal(scales, ws)
    assert ws[:, 0].max() == 0 and list(ws[:, 2])[:2] == [247, 247] and ws[0, 3] == ws[1, 4] == ws[2, 5] == 255
    fine = np.repeat(ws.T != 255, 128, axis=1)[:, :300]
    assert np.array_equal(codes[fine], want[fine]) and np.all(np.isnan(ref.from_fp8(codes[~fine])))
    for a in (dx, q, s):
        ctx.free(a)


def test_nothing_to_do(ctx):
    """No rows: nothing is written but the empty sums; no columns: nothing but the scales of rows."""
    f, g = ctx.to_device(np.full(4, 7.0, np.float32)), ctx.to_device(np.full(4, 7.0, np.float32))
    e = ctx.empty(1, np.float32)
    none = hip.DeviceArray(ctx, e.ptr, 0, np.dtype(np.float32), (0, 4))
    ctx.layer_norm(hip.LayerNorm.of(none, f, f, none))
    ctx.layer_norm_backward(hip.LayerNormGrad.of(dy=none, h=none, weight=f, dx=none, dweight=f, dbias=g))
    codes = hip.DeviceArray(ctx, e.ptr, 0, np.dtype(np.uint8), (0, 4))
    ctx.quantize_fp8_blocks(none, codes, hip.DeviceArray(ctx, e.ptr, 0, np.dtype(np.uint8), (1, 0)))
    ctx.synchronize()
    assert np.all(f.to_host() == 0) and np.all(g.to_host() == 0)
    flat = hip.DeviceArray(ctx, e.ptr, 0, np.dtype(np.float32), (4, 0))
    nothing = hip.DeviceArray(ctx, e.ptr, 0, np.dtype(np.float32), (0,))
    f.copy_from(np.full(4, 7.0, np.float32))
    ctx.layer_norm(hip.LayerNorm.of(flat, nothing, None, hip.DeviceArray(ctx, e.ptr, 0, np.dtype(np.uint8), (4, 0)), scales=f))
    ctx.layer_norm(hip.LayerNorm.of(flat, nothing, None, hip.DeviceArray(ctx, e.ptr, 0, np.dtype(np.uint8), (4, 0)),
                                    scales=hip.DeviceArray(ctx, e.ptr, 0, np.dtype(np.uint8), (0, 4))))
    ctx.synchronize()
    assert np.all(f.to_host() == 0)
    for a in (e, f, g):
        ctx.free(a)

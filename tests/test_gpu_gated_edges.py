"""GPU parity at the edges of what the gated block's operators document: rows of equal large values, gradients over their own operands, single rows whose
stride says nothing, tall and wide gradients' kernels.

Tolerances: of rows of a value v the formula leaves the bias alone. What a lane holds is the row's distance from a mean whose sum has been rounded ten times at
most (forty, where a thread adds twenty terms before that), so within that many half steps of v, and that distance is known to 8e-6 of itself; times
s = 1 / sqrt(eps) at most. Sums of squares in 8 bits lose at most 2^-13 of the largest for each of 64 terms, 2^-7 of themselves. The others as in the
operators' own tests.
"""
import numpy as np
import pytest

import ffn_reference as ref
import gated_reference as gated
from dotcompute_amd import hip
from test_gpu_layer_norm import EPS, F32, HALF, unit, within, y_bound
from test_gpu_layer_norm import test_layer_norm as layer_norm
from test_gpu_rms_norm import values, wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [7, 100, 300, 1025, 5000, 12001, 20001])
def test_rows_of_one_large_value(ctx, cols):
    """No variance but rounding's, which is not below zero: finite at an eps far below a step of the values' squares."""
    eps, rows = 1e-12, np.float32([[1e6], [3e6], [7e6 / 3], [-1e5 / 3]])
    x = np.repeat(rows, cols, axis=1)
    rng = np.random.default_rng(cols)
    dy = rng.normal(size=x.shape).astype(np.float32)
    w, b = np.ones(cols, np.float32), np.full(cols, 0.25, np.float32)
    dx, dw, db, ddy, y, d = (ctx.to_device(a) for a in (x, w, b, dy, np.zeros_like(x), np.zeros_like(x)))
    dwt, dbt = ctx.empty(cols, np.float32), ctx.empty(cols, np.float32)
    ctx.layer_norm(hip.LayerNorm.of(dx, dw, db, y, eps=eps))
    ctx.layer_norm_backward(hip.LayerNormGrad.of(ddy, dx, dw, d, dwt, dbt, eps=eps))
    ctx.synchronize()
    off = (10 if cols <= 16384 else 40) * HALF * np.abs(rows.astype(np.float64)) * F32 / np.sqrt(eps)
    assert np.all(np.abs(y.to_host() - 0.25) <= off + 2 * HALF)
    assert np.all(np.isfinite(d.to_host())) and np.all(np.isfinite(dwt.to_host()))
    assert np.all(np.abs(dbt.to_host() - np.sum(dy.astype(np.float64), axis=0)) <= 1e-6 * np.sum(np.abs(dy), axis=0))
    for a in (dx, dw, db, ddy, y, d, dwt, dbt):
        ctx.free(a)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(3, 7), (700, 1027), (300, 5001), (520, 16381), (5, 12001), (3, 40001)])
def test_gradients_over_their_operands(ctx, rows, cols, dtype):
    """dx over dy, and over dh: the bits of dx in a buffer of its own."""
    rng = np.random.default_rng(rows + cols)
    dy, dh = (values(rng, (rows, cols), dtype) for _ in range(2))
    h, w = values(rng, (rows, cols), dtype, 1.0, 2.0), values(rng, (cols,), dtype, 0.1, 1.0)
    a = [ctx.to_device(v) for v in (dy, h, w)]
    d, dx = ctx.to_device(dh), ctx.to_device(np.zeros_like(dy))
    sums = [ctx.empty(cols, np.float32) for _ in range(4)]
    ctx.layer_norm_backward(hip.LayerNormGrad.of(*a, dx, sums[0], sums[1], dh=d, eps=EPS))
    ctx.layer_norm_backward(hip.LayerNormGrad.of(*a, d, sums[2], sums[3], dh=d, eps=EPS))
    ctx.synchronize()
    want = dx.to_host()
    assert np.array_equal(d.to_host(), want)
    assert all(np.array_equal(sums[i].to_host(), sums[i + 2].to_host()) for i in range(2))
    d.copy_from(dh)
    ctx.layer_norm_backward(hip.LayerNormGrad.of(*a, a[0], sums[2], sums[3], dh=d, eps=EPS))
    ctx.synchronize()
    assert np.array_equal(a[0].to_host(), want)
    assert all(np.array_equal(sums[i].to_host(), sums[i + 2].to_host()) for i in range(2))
    x64 = gated.layer_norm_grad(wide(dy), wide(h), wide(w), EPS, wide(dh))[0]
    u, s = unit(wide(h))
    g = np.abs(wide(dy) * wide(w))
    terms = s * (g + np.mean(g, axis=1, keepdims=True) + (np.abs(u) + 1) * np.mean(g * (np.abs(u) + 1), axis=1, keepdims=True))
    half = ref.BF16 * (1 + F32) if dtype == "bf16" else 0.0
    within(want, x64, F32 * terms + np.abs(x64) * half + 2 * HALF * (np.abs(x64) + np.abs(wide(dh))) + 1e-37, "dx")
    for v in (*a, d, dx, *sums):
        ctx.free(v)


@pytest.mark.parametrize("cols", [100, 2050, 12001, 40001])
@pytest.mark.parametrize("stride", [0, -7, 1 << 60])
def test_single_rows_have_no_stride(ctx, cols, stride):
    rng = np.random.default_rng(cols)
    x, w = values(rng, (1, cols), "bf16"), values(rng, (cols,), "bf16", 0.1, 1.0)
    dx, dw, y, q = ctx.to_device(x), ctx.to_device(w), ctx.empty((1, cols), np.uint16), ctx.empty((1, cols), np.uint8)
    codes, sums = ctx.empty((gated.blocks(cols), 1), np.uint8), ctx.empty(cols, np.float32)

    def call(run, args, *names):
        for name in names:
            setattr(args, name, stride)
        run(args)
        ctx.synchronize()

    call(ctx.layer_norm, hip.LayerNorm.of(dx, dw, None, y, sum=dx, eps=EPS), "x_stride", "sum_stride", "y_stride")
    _, y64 = gated.layer_norm(wide(x), wide(w), None, EPS)
    within(y.to_host(), y64, y_bound(wide(x), wide(w), None, y64, "bf16"), "y")
    call(ctx.layer_norm_backward, hip.LayerNormGrad.of(y, dx, dw, y, sums, None, dh=y, eps=EPS), "dy_stride", "h_stride", "dh_stride", "dx_stride")
    assert np.all(np.isfinite(wide(y.to_host())))
    ctx.quantize_fp8_blocks(dx, q, codes)
    ctx.synchronize()
    want, scales = gated.rows_fp8(wide(x))
    assert np.array_equal(q.to_host(), want) and np.array_equal(codes.to_host(), scales)
    # a row of x, and a weight of one row; one block of columns has no row after its first
    out = ctx.empty((1, 1), np.float32)
    call(ctx.linear_blocks, hip.LinearBlocks.of(q, q, codes, codes, out), "x_stride", "w_stride", "y_stride",
         *(("x_scales_stride", "w_scales_stride") if cols <= 128 else ()))
    z = float(np.sum(gated.values(want, scales) ** 2))
    assert abs(out.to_host()[0, 0] - z) <= 2.0 ** -6 * z
    call(ctx.gated_linear, hip.GatedLinear.of(q, q, q, out, activation="none", x_scales=codes, gate_scales=codes, up_scales=codes), "x_stride",
         "w_gate_stride", "w_up_stride", "y_stride")
    assert abs(out.to_host()[0, 0] - z * z) <= 2.0 ** -5 * z * z
    for a in (dx, dw, y, q, codes, sums, out):
        ctx.free(a)


@pytest.mark.parametrize("rows,cols", [(1, 8193), (300, 8193), (257, 9000), (3, 12289), (2, 16383), (2, 16385)])
def test_layer_norm_of_long_rows(ctx, rows, cols):
    """Rows on both sides of what a workgroup holds in two and in four pieces to a lane."""
    layer_norm(ctx, rows, cols, "f32")
    layer_norm(ctx, rows, 2 * cols, "bf16")

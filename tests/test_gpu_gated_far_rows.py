"""The gated block's operators where offsets pass 32 bits, and over more rows than a grid has workgroups for.

Rows that lie gigabytes apart go through the same kernels as the same rows close together, so the results are the same bits.
"""
import numpy as np
import pytest

import ffn_reference as ref
import gated_reference as gated
from dotcompute_amd import hip
from test_gpu_far_rows import bf16, both
from test_gpu_layer_norm import EPS, within, y_bound

pytestmark = [pytest.mark.gpu, pytest.mark.slow]


@pytest.mark.parametrize("cols", [520, 40001])
def test_layer_norm_of_far_rows(ctx, cols):
    rng = np.random.default_rng(1)
    w, b = ctx.to_device(bf16(rng, cols)), ctx.to_device(bf16(rng, cols))
    dw, db = ctx.empty(cols, np.float32), ctx.empty(cols, np.float32)
    blank = np.zeros((5, cols), np.uint16)
    mats = {"x": bf16(rng, 5, cols), "residual": bf16(rng, 5, cols), "sum": blank, "y": blank}
    both(ctx, mats, lambda a, s: ctx.layer_norm(hip.LayerNorm.of(weight=w, bias=b, **a, **s)), ("sum", "y"), (1 << 30) + 8)
    codes = {"x": mats["x"], "y": np.zeros((5, cols), np.uint8), "scales": np.zeros((gated.blocks(cols), 5), np.uint8)}
    stride = (1 << 32) + 8 if cols == 520 else 1 << 25  # (313 rows of scales)
    both(ctx, codes, lambda a, s: ctx.layer_norm(hip.LayerNorm.of(weight=w, bias=b, **a, **s)), ("y", "scales"), stride)
    mats = {"dy": bf16(rng, 5, cols), "h": bf16(rng, 5, cols), "dx": blank}
    both(ctx, mats, lambda a, s: ctx.layer_norm_backward(hip.LayerNormGrad.of(weight=w, dweight=dw, dbias=db, **a, **s)), ("dx",), (1 << 30) + 8)
    for a in (w, b, dw, db):
        ctx.free(a)


def test_quantize_blocks_of_far_rows(ctx):
    rng = np.random.default_rng(2)
    mats = {"x": bf16(rng, 19, 520), "q": np.zeros((19, 520), np.uint8), "scales": np.zeros((5, 19), np.uint8)}
    both(ctx, mats, lambda a, s: ctx.quantize_fp8_blocks(**a, **s), ("q", "scales"), (1 << 30) + 8)


@pytest.mark.parametrize("m", [6, 200])
def test_gated_of_far_rows(ctx, m):
    """Operands' rows far apart are copied; results and block scales are written and read where they lie."""
    rng = np.random.default_rng(m)
    stride = (1 << 32) // m // 8 * 8 + 8
    mats = {"x": bf16(rng, m, 136), "w_gate": bf16(rng, 9, 136), "w_up": bf16(rng, 9, 136), "y": np.zeros((m, 9), np.uint16),
            "pre_gate": np.zeros((m, 9), np.uint16), "pre_up": np.zeros((m, 9), np.uint16)}
    y, g, u = both(ctx, mats, lambda a, s: ctx.gated_linear(hip.GatedLinear.of(**a, **s)), ("y", "pre_gate", "pre_up"), stride)
    assert np.any(y)
    back = {"dy": bf16(rng, m, 9), "x": mats["x"], "w_gate": mats["w_gate"], "w_up": mats["w_up"], "pre_gate": g, "pre_up": u,
            "dx": np.zeros((m, 136), np.uint16), "dw_gate": np.zeros((9, 136), np.uint16), "dw_up": np.zeros((9, 136), np.uint16)}
    both(ctx, back, lambda a, s: ctx.gated_linear_backward(hip.GatedLinearGrad.of(**a, **s)), ("dx", "dw_gate", "dw_up"), stride // 2 // 8 * 8)
    (xq, xs), (wq, ws) = (gated.rows_fp8(rng.normal(size=(rows, 1000))) for rows in (m, 72))
    x, w, y = ctx.to_device(xq), ctx.to_device(wq), ctx.empty((m, 72), np.float32)

    def run(a, s):
        ctx.linear_blocks(hip.LinearBlocks.of(x, w, a["x_scales"], a["w_scales"], y, **s))
        ctx.synchronize()
        results.append(y.to_host())
        ctx.gated_linear(hip.GatedLinear.of(x, w, w, y, x_scales=a["x_scales"], gate_scales=a["w_scales"], up_scales=a["w_scales"],
                                            x_scales_stride=s["x_scales_stride"], gate_scales_stride=s["w_scales_stride"],
                                            up_scales_stride=s["w_scales_stride"]))
        ctx.synchronize()
        results.append(y.to_host())

    results = []
    both(ctx, {"x_scales": xs, "w_scales": ws}, run, (), (1 << 32) + 8)
    assert np.array_equal(results[0], results[2]) and np.array_equal(results[1], results[3]) and np.any(results[1])
    for a in (x, w, y):
        ctx.free(a)


def test_layer_norm_of_more_rows_than_workgroups(ctx):
    rows, cols = (1 << 22) + 7, 8
    rng = np.random.default_rng(5)
    x, w, b = rng.normal(size=(rows, cols)).astype(np.float32), rng.normal(size=cols).astype(np.float32), rng.normal(size=cols).astype(np.float32)
    dx, dw, db, y = ctx.to_device(x), ctx.to_device(w), ctx.to_device(b), ctx.empty((rows, cols), np.float32)
    q, s = ctx.empty((rows, cols), np.uint8), ctx.empty((1, rows), np.uint8)
    ctx.layer_norm(hip.LayerNorm.of(dx, dw, db, y, eps=EPS))
    ctx.quantize_fp8_blocks(dx, q, s)
    ctx.synchronize()
    x64, w64, b64 = (a.astype(np.float64) for a in (x, w, b))
    y64 = gated.layer_norm(x64, w64, b64, EPS)[1]
    within(y.to_host(), y64, y_bound(x64, w64, b64, y64, "f32"), "y")
    assert np.array_equal(s.to_host()[0], gated.scale_of(np.max(np.abs(x64), axis=1)))
    assert np.array_equal(q.to_host()[-1000:], gated.rows_fp8(x64[-1000:])[0])
    for a in (dx, dw, db, y, q, s):
        ctx.free(a)


def test_gated_gradients_over_many_rows(ctx):
    """dx and the biases' gradients alone, over more rows than the weights' sums may have: whole numbers, whose sums are exact."""
    m, n, k = (1 << 23) + 9, 8, 24
    rng = np.random.default_rng(1)
    dy, g, u = (rng.integers(-1, 2, size=(m, n), dtype=np.int8) for _ in range(3))
    wg, wu = (rng.integers(-6, 7, size=(n, k), dtype=np.int8) for _ in range(2))
    on = [ctx.to_device(ref.to_bf16(a)) for a in (dy, wg, wu, g, u)]
    x, dx, dbs = ctx.empty((m, k), np.uint16), ctx.empty((m, k), np.uint16), [ctx.empty(n, np.float32) for _ in range(2)]
    ctx.gated_linear_backward(hip.GatedLinearGrad.of(on[0], x, *on[1:], dx=dx, dbias_gate=dbs[0], dbias_up=dbs[1], activation="relu"))
    ctx.synchronize()
    dg, du = dy * u * (g > 0), dy * np.maximum(g, 0)
    assert np.array_equal(dbs[0].to_host(), dg.sum(axis=0, dtype=np.int64)) and np.array_equal(dbs[1].to_host(), du.sum(axis=0, dtype=np.int64))
    got = dx.to_host()
    for at in range(0, m, 1 << 20):
        part = slice(at, at + (1 << 20))
        want = dg[part].astype(np.float32) @ wg.astype(np.float32) + du[part].astype(np.float32) @ wu.astype(np.float32)
        assert np.array_equal(ref.from_bf16(got[part]), want), at
    for a in on + [x, dx] + dbs:
        ctx.free(a)

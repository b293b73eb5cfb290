"""GPU parity: layer norm of rows whose first elements lie far from the rest, in each part of a row that a wave holds: what a value near the mean is taken
from is then no sample of the others. Against float64.

Tolerance, of u = (h - mean) s, from the arithmetic, in half-steps e = 2^-24. A wave's sum of d^2, d = h - k, takes up to 16 additions in a lane and six
between lanes, whose roundings, as independent ones, leave it 0.8 e of itself off (the last steps, which one value goes through, count most), and so the sum
of d. With C chunks to a lane sum(n (k - mean)^2) is at most C times the row's squares, C = 4 over 16 waves: their join is 2 C / sqrt(16) e = 2 e off and 1 e
for its own additions, s half of that; the mean 2 e of a deviation, as sum(d) is off by 0.8 e of (1 + sqrt(C)) deviations, over 1 to 16 waves. s is
the hardware's root to 2 e, u has two roundings. All in all 3 e of |u| + 1 in one standard deviation of its random part; 10 e of it is allowed, three of them, and
over that a result's own rounding. (Of the mean of the first 16 elements as k the root alone would be off by 64 / 4 of what it is here.)
The gradient by h has two means of g and g u, whose sums are off as the above: 20 e of its terms' magnitudes.
"""
import numpy as np
import pytest

import ffn_reference as ref
import gated_reference as gated
from dotcompute_amd import hip
from test_gpu_layer_norm import EPS, HALF, unit, within
from test_gpu_rms_norm import wide

pytestmark = pytest.mark.gpu


def uneven(rng, rows, cols, dtype, waves, ahead, apart):
    """Normal values; in each of `waves` parts' first elements, `ahead` of them, `apart` deviations away."""
    elems = 8 if dtype == "bf16" else 4
    x = rng.normal(size=(rows, cols))
    for w in range(waves):
        x[:, w * 64 * elems:w * 64 * elems + ahead * elems] += apart * rng.choice([-1, 1], size=(rows, 1))
    return ref.to_bf16(x) if dtype == "bf16" else x.astype(np.float32)


# By the lanes' chunks and the waves to a row (bf16 1024: two chunks and one wave; 16384: two over 16; float32 300 rows: two over 8; 16384: four over 16).
ROWS = [("bf16", 64, 512, 1), ("bf16", 64, 1024, 1), ("bf16", 64, 4096, 8), ("bf16", 40, 16384, 16), ("f32", 64, 256, 1), ("f32", 64, 4096, 16),
        ("f32", 300, 4096, 8), ("f32", 40, 8192, 16), ("f32", 40, 16384, 16), ("f32", 64, 250, 1), ("f32", 40, 16301, 16)]


@pytest.mark.parametrize("ahead", [4, 64], ids=["quad", "chunk"])
@pytest.mark.parametrize("dtype,rows,cols,waves", ROWS)
def test_layer_norm(ctx, dtype, rows, cols, waves, ahead):
    for apart in (3.0, 50.0, 3000.0):
        rng = np.random.default_rng(cols + ahead)
        x = uneven(rng, rows, cols, dtype, waves, ahead, apart)
        w = np.ones(cols, np.float32) if dtype == "f32" else ref.to_bf16(np.ones(cols))
        dx, dw, y = ctx.to_device(x), ctx.to_device(w), ctx.empty((rows, cols), x.dtype)
        ctx.layer_norm(hip.LayerNorm.of(dx, dw, None, y, eps=EPS))
        ctx.synchronize()
        u, _ = unit(wide(x))
        within(y.to_host(), u, 10 * HALF * (np.abs(u) + 1) + (ref.BF16 * (1 + 20 * HALF) * np.abs(u) if dtype == "bf16" else 0.0), ("y", apart))
        for a in (dx, dw, y):
            ctx.free(a)


GRAD_ROWS = [("bf16", 512, 1), ("bf16", 4096, 8), ("bf16", 8192, 16), ("bf16", 16384, 16), ("f32", 256, 1), ("f32", 4096, 16), ("f32", 8192, 16),
             ("f32", 16384, 16), ("f32", 16301, 16)]


@pytest.mark.parametrize("ahead", [4, 64], ids=["quad", "chunk"])
@pytest.mark.parametrize("dtype,cols,waves", GRAD_ROWS)
def test_layer_norm_backward(ctx, dtype, cols, waves, ahead):
    """A row at a time, with gradients of one or minus one: dweight is then u, in float32 whatever the operands' type."""
    for seed in range(24):
        rng = np.random.default_rng(1000 * seed + cols + ahead)
        h = uneven(rng, 1, cols, dtype, waves, ahead, (3.0, 50.0, 3000.0)[seed % 3])
        to = ref.to_bf16 if dtype == "bf16" else (lambda v: v.astype(np.float32))
        dy, w = to(rng.choice([-1.0, 1.0], size=(1, cols))), to(np.ones(cols))
        ddy, dh, dw, dx = ctx.to_device(dy), ctx.to_device(h), ctx.to_device(w), ctx.empty((1, cols), h.dtype)
        dweight, dbias = ctx.empty(cols, np.float32), ctx.empty(cols, np.float32)
        ctx.layer_norm_backward(hip.LayerNormGrad.of(ddy, dh, dw, dx, dweight, dbias, eps=EPS))
        ctx.synchronize()
        u, s = unit(wide(h))
        x64, w64, b64 = gated.layer_norm_grad(wide(dy), wide(h), wide(w), EPS)
        within(dweight.to_host(), w64, 10 * HALF * (np.abs(u[0]) + 1), "dweight")
        assert np.array_equal(dbias.to_host(), b64)
        terms = s * (1 + 1 + (np.abs(u) + 1) * np.mean(np.abs(u) + 1, axis=1, keepdims=True))
        within(dx.to_host(), x64, 20 * HALF * terms + (ref.BF16 * (1 + 20 * HALF) * np.abs(x64) if dtype == "bf16" else 0.0), "dx")
        for a in (ddy, dh, dw, dx, dweight, dbias):
            ctx.free(a)


@pytest.mark.parametrize("dtype,cols", [("f32", 4), ("f32", 64), ("f32", 256), ("bf16", 8), ("bf16", 128), ("bf16", 512)])
def test_rows_of_one_value_near_the_largest(ctx, dtype, cols):
    """Rows that one wave holds, of lanes that are a power of two: every sum on the way to the value's mean is exact, and a float as long as a lane's is, so
    that nothing is left of the row but the bias."""
    to = ref.to_bf16 if dtype == "bf16" else (lambda v: v.astype(np.float32))
    rng = np.random.default_rng(cols)
    h = to(np.repeat(np.array([[1e37], [-3e37], [4e37], [1e-37], [7e5]]), cols, axis=1))
    w, b, dy = to(rng.normal(size=cols)), to(rng.normal(size=cols)), to(rng.normal(size=h.shape))
    dh, dw, db, ddy, y, dx = (ctx.to_device(a) for a in (h, w, b, dy, np.zeros_like(h), np.zeros_like(h)))
    dweight = ctx.empty(cols, np.float32)
    ctx.layer_norm(hip.LayerNorm.of(dh, dw, db, y, eps=EPS))
    ctx.layer_norm_backward(hip.LayerNormGrad.of(ddy, dh, dw, dx, dweight, eps=EPS))
    ctx.synchronize()
    assert np.array_equal(y.to_host(), np.broadcast_to(b, h.shape)) and np.all(dweight.to_host() == 0)
    g, s = wide(dy) * wide(w), EPS ** -0.5
    want = s * (g - np.mean(g, axis=1, keepdims=True))
    terms = s * (np.abs(g) + np.mean(np.abs(g), axis=1, keepdims=True))
    within(dx.to_host(), want, 20 * HALF * terms + (ref.BF16 * (1 + 20 * HALF) * np.abs(want) if dtype == "bf16" else 0.0), "dx")
    for a in (dh, dw, db, ddy, y, dx, dweight):
        ctx.free(a)

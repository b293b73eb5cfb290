"""GPU parity: rows in 8 bits with scales, where rows lie apart, hold next to nothing, or are empty."""
import numpy as np
import pytest

import ffn_reference as ref
from dotcompute_amd import hip
from test_gpu_rms_norm import Matrix, values, wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(3, 7), (5, 1001), (9, 4096)])
def test_rows_that_lie_apart(ctx, rows, cols, dtype):
    """The same bits as the definition in float32 (a division and a product), and nothing else is written."""
    np_t = np.uint16 if dtype == "bf16" else np.float32
    x = values(np.random.default_rng(cols), (rows, cols), dtype, 5.0)
    a, q = Matrix(ctx, x, np_t, 1, 3), Matrix(ctx, np.zeros((rows, cols), np.uint8), np.uint8, 3, 5)
    s = ctx.empty(rows, np.float32)
    ctx.quantize_fp8(a.a, q.a, s, x_stride=a.stride, q_stride=q.stride)
    ctx.synchronize()
    want, scales = ref.rows_fp8(wide(x).astype(np.float32))
    assert np.array_equal(q.read(), want) and np.array_equal(s.to_host(), scales)
    a.read()
    for m in (a.base, q.base, s):
        ctx.free(m)


# Maxima on both sides of 448 2^-128 = 1.3e-36, below which their reciprocals are no floats, and the smallest floats.
TINY = [1e-30, 2e-36, 1.3e-36, 1e-36, 1e-37, 2e-38, 1e-40, 1e-44, 0.0]


def check_codes(q, s, want):
    """Codes stand for the values to half a step of 4 bits or of the smallest code; a scale of at least 2^-128 has 21 bits (where it is one
    of the smaller floats), and a product that is one itself is off by half the smallest float."""
    scale = s[:, None].astype(np.float64)
    off = np.abs(ref.from_fp8(q) * scale - want)
    assert np.all(off <= np.maximum(np.abs(want) * ref.FP8, ref.LEAST / 2 * scale) * (1 + 2.0 ** -18) + 2.0 ** -149), off.max(axis=1)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cols", [40, 1000, 5000])
def test_rows_of_next_to_nothing(ctx, cols, dtype):
    unit = np.random.default_rng(cols).uniform(-1, 1, size=(len(TINY), cols)).astype(np.float32)
    unit[:, 3] = 1.0
    x = unit * np.float32(TINY)[:, None]
    x = ref.to_bf16(x) if dtype == "bf16" else x
    dx, q, s = ctx.to_device(x), ctx.empty(x.shape, np.uint8), ctx.empty(len(TINY), np.float32)
    ctx.quantize_fp8(dx, q, s)
    ctx.synchronize()
    check_codes(q.to_host(), s.to_host(), wide(x))
    assert s.to_host()[-1] == 0 and np.all(ref.from_fp8(q.to_host()[-1]) == 0)  # (zeros of either sign)
    for a in (dx, q, s):
        ctx.free(a)


@pytest.mark.parametrize("cols", [200, 70001])
def test_norms_of_next_to_nothing(ctx, cols):
    """A weight that takes a norm's results there: what float32 makes of h w / rms(h), in 8 bits."""
    rng = np.random.default_rng(cols)
    h, w = rng.normal(size=(2, cols)).astype(np.float32), (1e-37 * rng.uniform(0.5, 1, size=cols)).astype(np.float32)
    dh, dw, q, s = ctx.to_device(h), ctx.to_device(w), ctx.empty(h.shape, np.uint8), ctx.empty(2, np.float32)
    ctx.rms_norm(hip.RmsNorm.of(dh, dw, q, scales=s))
    ctx.synchronize()
    want = ref.rms_norm(wide(h), wide(w), 1e-6)[1]
    # (the norm's own error, 4e-6 of a value, may move a code's rounding by that)
    scale = s.to_host()[:, None].astype(np.float64)
    off = np.abs(ref.from_fp8(q.to_host()) * scale - want)
    assert np.all(off <= np.maximum(np.abs(want) * ref.FP8, ref.LEAST / 2 * scale) * (1 + 2.0 ** -16) + 2.0 ** -149)
    for a in (dh, dw, q, s):
        ctx.free(a)


def test_rows_of_nothing(ctx):
    """Their scales are those of zeros, so that a product over them is its bias."""
    m, n = 5, 12
    e, bias = ctx.empty(8, np.uint16), ctx.to_device(ref.to_bf16(np.arange(n)))
    s, y = [ctx.to_device(np.full(r, np.nan, np.float32)) for r in (m, n)], ctx.empty((m, n), np.float32)

    def part(dtype, *shape):
        return hip.DeviceArray(ctx, e.ptr, 0, np.dtype(dtype), shape)

    ctx.rms_norm(hip.RmsNorm.of(part(np.uint16, m, 0), part(np.uint16, 0), part(np.uint8, m, 0), scales=s[0]))
    ctx.quantize_fp8(part(np.uint16, n, 0), part(np.uint8, n, 0), s[1])
    ctx.linear(hip.Linear.of(part(np.uint8, m, 0), part(np.uint8, n, 0), y, bias=bias, x_scales=s[0], w_scales=s[1]))
    ctx.synchronize()
    assert np.all(s[0].to_host() == 0) and np.all(s[1].to_host() == 0)
    assert np.array_equal(y.to_host(), np.tile(np.arange(n, dtype=np.float32), (m, 1)))
    for a in (e, bias, y, *s):
        ctx.free(a)

"""GPU parity: matrix products with bias, activation and residual in their epilogue, and their gradients, against float64.

Tolerances, from the arithmetic: products of bf16 values are exact in float32. An instruction of the matrix
cores adds at least 16 of them and may cut what it adds at an ulp of the largest, so a sum over k of terms of magnitude S in
all is within (k / 16 + 8) ulps of S: (k / 16 + 8) 2^-23 S. The 8-bit instructions add 64 or 128 products that they first cut at
2^-13 of the largest among those of a lane's part (measured with pairs of powers of two), which each product may lose once
more: 2^-13 of the largest |x| times the largest |w| in each 64 of k, 64 times. Whatever is a sum of small whole numbers they
add exactly, which is tested bit for bit. No activation's slope passes 1.13 (gelu's); the activations
themselves are within 4e-6 of max(1, |z|); results in bf16 add half a step of 8 bits. The gradients' operand dz is rounded to bf16
before the products: half a step of 8 bits of each term.
"""
import numpy as np
import pytest

import ffn_reference as ref
from dotcompute_amd import hip
from test_gpu_rms_norm import Matrix

pytestmark = pytest.mark.gpu
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def bf16(rng, shape, scale=1.0):
    return ref.to_bf16(rng.normal(size=shape) * scale)


def wide(b):
    return ref.from_bf16(b).astype(np.float64)


def sum_bound(k, magnitude):
    return (k / 16 + 8) * 2.0 ** -23 * magnitude


def cut_bound(x, w):
    """What the 8-bit instructions may cut off a product at a time."""
    k = x.shape[1]
    x, w = (np.pad(np.abs(a), ((0, 0), (0, -k % 64))).reshape(a.shape[0], -1, 64).max(axis=2, initial=0.0) for a in (x, w))
    return 64 * 2.0 ** -13 * (x @ w.T)


def within(got, want, bound, what):
    off = np.abs(got - want)
    assert np.all(off <= bound), f"{what}: {np.max(off / bound):.3g} of the bound"


def run_linear(ctx, m, n, k, dtype="bf16", activation="none", y="bf16", bias=True, residual=False, pre=False, odd=0, in_place=False,
               seed=0):
    rng = np.random.default_rng(seed + 3 * m + 5 * n + 7 * k)
    size = np.uint8 if dtype == "fp8" else np.uint16
    a = {}
    if dtype == "fp8":
        (xq, xs), (wq, ws) = (ref.rows_fp8(rng.normal(size=(r, k)).astype(np.float32)) for r in (m, n))
        x64, w64 = ref.from_fp8(xq) * xs[:, None].astype(np.float64), ref.from_fp8(wq) * ws[:, None].astype(np.float64)
        a["x_scales"], a["w_scales"] = ctx.to_device(xs), ctx.to_device(ws)
    else:
        xq, wq = bf16(rng, (m, k)), bf16(rng, (n, k), max(k, 1) ** -0.5)
        x64, w64 = wide(xq), wide(wq)
    mats = {"x": Matrix(ctx, xq, size, odd, odd), "w": Matrix(ctx, wq, size, 3 * odd, 5 * odd),
            "y": Matrix(ctx, np.zeros((m, n), np.uint16 if y == "bf16" else np.float32), np.uint16 if y == "bf16" else np.float32, odd,
                        7 * odd)}
    b64 = r64 = None
    if bias:
        b = bf16(rng, n)
        b64, a["bias"] = wide(b), ctx.to_device(b)
    if residual:
        r = bf16(rng, (m, n))
        r64 = wide(r)
        mats["residual"] = mats["y"] if in_place else Matrix(ctx, r, np.uint16, 0, odd)
        if in_place:
            mats["y"].base.copy_from(np.concatenate([r.reshape(-1), np.full(8, 77, np.uint16)]))
    if pre:
        mats["pre"] = Matrix(ctx, np.zeros((m, n), np.uint16), np.uint16, odd, 3 * odd)
    ctx.linear(hip.Linear.of(activation=activation, **{name: q.a for name, q in mats.items()}, **a,
                             **{name + "_stride": q.stride for name, q in mats.items()}))
    ctx.synchronize()
    z64, y64 = ref.linear(x64, w64, b64, activation, r64)
    magnitude = np.abs(x64) @ np.abs(w64).T + (0 if b64 is None else np.abs(b64))
    z_off = sum_bound(k, magnitude) + (cut_bound(x64, w64) if dtype == "fp8" else 0.0)
    half = ref.BF16 * (1 + 2.0 ** -8)
    if pre:
        within(wide(mats["pre"].read()), z64, z_off + half * np.abs(z64) + 1e-37, "pre")
    got = mats["y"].read()
    got = wide(got) if y == "bf16" else got.astype(np.float64)
    off = 1.13 * z_off + 4e-6 * (np.maximum(1.0, np.abs(z64)) + np.abs(y64)) + (half * np.abs(y64) if y == "bf16" else 0.0)
    within(got, y64, off, "y")
    for q in {id(q.base): q.base for q in mats.values()}.values():
        ctx.free(q)
    for q in a.values():
        ctx.free(q)
    return got


# Few rows (one instruction's worth and more), the tile kernels from one tile to hundreds, one step along k to many, with a
# ragged last tile or step.
SHAPES = [(1, 1, 1), (1, 64, 64), (1, 1000, 777), (7, 48, 4096), (16, 512, 130), (17, 33, 8), (32, 4096, 1024), (33, 70, 40),
          (64, 64, 64), (100, 200, 300), (128, 256, 64), (130, 1030, 520), (257, 129, 1000), (300, 300, 4104), (777, 1111, 333),
          (1024, 2048, 192)]


@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_shapes(ctx, m, n, k, dtype):
    run_linear(ctx, m, n, k, dtype, "silu", pre=True, residual=True)


@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("m,n,k", SHAPES + [(2048, 4096, 256), (512, 512, 4096), (1537, 1025, 1023)])
def test_linear_of_whole_numbers_is_exact(ctx, m, n, k, dtype):
    """Values -6..6 and scales that are powers of two: every sum is a whole number below 2^24, in any order."""
    rng = np.random.default_rng(m + n + k)
    x, w = (rng.integers(-6, 7, size=(r, k)).astype(np.float32) for r in (m, n))
    code = ref.to_fp8 if dtype == "fp8" else ref.to_bf16
    a = [ctx.to_device(code(x)), ctx.to_device(code(w)), ctx.empty((m, n), np.float32)]
    xs, ws = (np.exp2(rng.integers(-3, 4, size=r)).astype(np.float32) for r in (m, n))
    scales = [ctx.to_device(xs), ctx.to_device(ws)] if dtype == "fp8" else [None, None]
    ctx.linear(hip.Linear.of(*a, x_scales=scales[0], w_scales=scales[1]))
    ctx.synchronize()
    want = x @ w.T  # (exact in float32 for the same reason)
    if dtype == "fp8":
        want = want * xs[:, None] * ws
    assert np.array_equal(a[2].to_host(), want)
    for q in a + scales:
        if q is not None:
            ctx.free(q)


@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("m,n,k", [(3, 50, 100), (31, 20, 33), (90, 140, 210), (300, 260, 513)])
def test_linear_strides_and_alignments(ctx, m, n, k, dtype):
    """Rows one element into their buffers, and further apart than they are long; nothing else is written."""
    run_linear(ctx, m, n, k, dtype, "gelu", pre=True, residual=True, odd=1)
    run_linear(ctx, m, n, k, dtype, "gelu", y="f32", odd=1)


@pytest.mark.parametrize("activation", ACTS)
@pytest.mark.parametrize("m", [5, 200])
def test_linear_activations(ctx, activation, m):
    for y in ("bf16", "f32"):
        run_linear(ctx, m, 96, 128, "bf16", activation, y, pre=True)
        run_linear(ctx, m, 96, 128, "fp8", activation, y, residual=True, bias=False)


@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("m,n,k", [(100, 300, 9000), (300, 300, 8000), (520, 512, 20000), (101, 301, 9001), (1100, 300, 6000)])
def test_linear_of_long_sums(ctx, m, n, k, dtype):
    """Few tiles with long sums, which workgroups share: the epilogue is the adding kernel's."""
    run_linear(ctx, m, n, k, dtype, "silu", residual=True, pre=True)
    run_linear(ctx, m, n, k, dtype, "none", "f32", bias=False, residual=True, odd=1)


@pytest.mark.slow
@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("m,n,k", [(2048, 4096, 256), (4352, 4096, 136), (2000, 3000, 1000), (1537, 2049, 1023), (512, 512, 4096),
                                   (64, 8192, 2048)])
def test_linear_larger(ctx, m, n, k, dtype):
    """Each tile size, with one to four groups of waves along k."""
    run_linear(ctx, m, n, k, dtype, "gelu_tanh", pre=True)


def test_linear_of_nothing(ctx):
    """k = 0: bias, activation and residual alone; no rows or no outputs: nothing."""
    for m, n in ((3, 40), (70, 70)):
        run_linear(ctx, m, n, 0, activation="silu", residual=True, pre=True)
    e = ctx.empty(8, np.uint16)

    def part(*shape):
        return hip.DeviceArray(ctx, e.ptr, 0, np.dtype(np.uint16), shape)

    ctx.linear(hip.Linear.of(part(0, 4), part(2, 4), part(0, 2)))
    ctx.linear(hip.Linear.of(part(2, 4), part(0, 4), part(2, 0)))
    ctx.synchronize()
    ctx.free(e)


def test_linear_over_its_residual(ctx):
    for m, n, k in ((2, 80, 64), (100, 130, 70)):
        run_linear(ctx, m, n, k, activation="relu", residual=True, in_place=True)


def test_linear_keeps_nonfinite_values_to_their_rows(ctx):
    for m in (4, 70):
        rng = np.random.default_rng(m)
        x, w = bf16(rng, (m, 40)), bf16(rng, (48, 40))
        x[1, 3], x[2, 39] = ref.to_bf16(np.nan), ref.to_bf16(np.inf)
        dx, dw, y = ctx.to_device(x), ctx.to_device(w), ctx.empty((m, 48), np.float32)
        ctx.linear(hip.Linear.of(dx, dw, y))
        ctx.synchronize()
        got = y.to_host()
        assert np.all(np.isnan(got[1])) and np.all(np.isinf(got[2]) | np.isnan(got[2]))
        assert np.all(np.isfinite(np.delete(got, [1, 2], axis=0)))
        for a in (dx, dw, y):
            ctx.free(a)


def test_activations_of_the_ends(ctx):
    """Large and infinite z, through the bias of an empty product: the limits, no NaN but 0 times an infinity."""
    z = np.array([0.0, -0.0, 1e-30, 20.0, -20.0, 100.0, -100.0, 1e4, -1e4, 3e38, -3e38, np.inf], np.float32)
    b = ref.to_bf16(z)
    z = wide(b)
    db, e, y = ctx.to_device(b), ctx.empty(8, np.uint16), ctx.empty((2, z.size), np.float32)
    x = hip.DeviceArray(ctx, e.ptr, 0, np.dtype(np.uint16), (2, 0))
    w = hip.DeviceArray(ctx, e.ptr, 0, np.dtype(np.uint16), (z.size, 0))
    for name in ACTS:
        ctx.linear(hip.Linear.of(x, w, y, bias=db, activation=name))
        ctx.synchronize()
        got = y.to_host()
        want = np.where(z > 0, z, 0.0) if name != "none" else z
        small = np.abs(z) < 50
        with np.errstate(all="ignore"):
            want = np.where(small, ref.act(name, z), want)
        assert np.allclose(got[0], want, rtol=1e-5, atol=1e-5) and np.array_equal(got[0], got[1]), name
    for a in (db, e, y):
        ctx.free(a)


def run_backward(ctx, m, n, k, activation, odd=0, dx=True, dw=True, dbias=True, seed=0):
    rng = np.random.default_rng(seed + m + 3 * n + 5 * k)
    dy, x, w, pre = bf16(rng, (m, n)), bf16(rng, (m, k)), bf16(rng, (n, k)), bf16(rng, (m, n))
    mats = {"dy": Matrix(ctx, dy, np.uint16, odd, odd), "x": Matrix(ctx, x, np.uint16, odd, 3 * odd),
            "w": Matrix(ctx, w, np.uint16, 3 * odd, odd)}
    if activation != "none":
        mats["pre"] = Matrix(ctx, pre, np.uint16, odd, 5 * odd)
    if dx:
        mats["dx"] = Matrix(ctx, np.zeros((m, k), np.uint16), np.uint16, odd, odd)
    if dw:
        mats["dw"] = Matrix(ctx, np.zeros((n, k), np.uint16), np.uint16, odd, odd)
    db = ctx.to_device(np.full(n, 5.0, np.float32))
    ctx.linear_backward(hip.LinearGrad.of(activation=activation, dbias=db if dbias else None, **{a: q.a for a, q in mats.items()},
                                          **{a + "_stride": q.stride for a, q in mats.items()}))
    ctx.synchronize()
    y64, z64 = wide(dy), wide(pre)
    dz = y64 * ref.act_slope(activation, z64)
    dz_off = np.abs(y64) * 4e-6 * np.maximum(1.0, np.abs(z64))  # the slope's error
    x64, w64, b64 = ref.linear_grad(y64, wide(x), wide(w), z64, activation)
    half = ref.BF16 * (1 + 2.0 ** -8)
    exact = activation in ("none", "relu")
    rough = np.abs(dz) * (0.0 if exact else half) + dz_off
    got = {a: wide(mats[a].read()) for a in ("dx", "dw") if a in mats}
    if dx:
        s = np.abs(dz) @ np.abs(wide(w))
        within(got["dx"], x64, sum_bound(n, s) + rough @ np.abs(wide(w)) + half * np.abs(x64) + 1e-37, "dx")
    if dw:
        s = np.abs(dz).T @ np.abs(wide(x))
        within(got["dw"], w64, sum_bound(m, s) + rough.T @ np.abs(wide(x)) + half * np.abs(w64) + 1e-37, "dw")
    if dbias:  # 64 rows a part, parts in 16 chains
        s = np.abs(dz).sum(axis=0)
        within(db.to_host(), b64, (m / 1024 + 64) * 2.0 ** -24 * s + dz_off.sum(axis=0) + 1e-37, "dbias")
    else:
        assert np.all(db.to_host() == 5.0)
    for q in mats.values():
        q.read() if q not in (mats.get("dx"), mats.get("dw")) else None
        ctx.free(q.base)
    ctx.free(db)
    return got


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 64, 200), (5, 7, 9), (64, 64, 64), (70, 130, 50), (128, 256, 512), (257, 300, 129),
                                   (1000, 72, 333), (520, 1040, 264)])
@pytest.mark.parametrize("activation", ["none", "gelu"])
def test_linear_backward_shapes(ctx, m, n, k, activation):
    run_backward(ctx, m, n, k, activation)
    run_backward(ctx, m, n, k, activation, odd=1)


@pytest.mark.parametrize("activation", ACTS)
def test_linear_backward_activations(ctx, activation):
    run_backward(ctx, 96, 200, 64, activation)


@pytest.mark.slow
@pytest.mark.parametrize("m,n,k", [(2000, 3000, 1000), (2048, 2048, 520), (4100, 260, 136)])
def test_linear_backward_larger(ctx, m, n, k):
    run_backward(ctx, m, n, k, "silu")


@pytest.mark.parametrize("m,n,k", [(16, 2048, 520), (64, 2000, 136), (2000, 300, 264), (1, 3000, 200), (2500, 1, 90), (3000, 144, 700),
                                   (45, 5001, 553), (1717, 104, 1368), (491, 3000, 1500), (4500, 200, 72)])
def test_linear_backward_of_unlike_sums(ctx, m, n, k):
    """Sums over few rows beside sums over many outputs, and the other way round: one launch, in parts of their own."""
    run_backward(ctx, m, n, k, "silu")


@pytest.mark.parametrize("activation", ["none", "silu"])
def test_linear_backward_in_parts(ctx, activation):
    """Each gradient alone is the same bits as all of them together."""
    full = run_backward(ctx, 100, 136, 72, activation)
    assert np.array_equal(run_backward(ctx, 100, 136, 72, activation, dw=False, dbias=False)["dx"], full["dx"])
    assert np.array_equal(run_backward(ctx, 100, 136, 72, activation, dx=False, dbias=False)["dw"], full["dw"])
    run_backward(ctx, 100, 136, 72, activation, dx=False, dw=False)


@pytest.mark.parametrize("stride", [-8, 0, 3, 1 << 40])
def test_the_stride_of_a_single_row_says_nothing(ctx, stride):
    rng = np.random.default_rng(5)
    x, w, dy = bf16(rng, (1, 136)), bf16(rng, (72, 136)), bf16(rng, (1, 72))
    a = {name: ctx.to_device(v) for name, v in dict(x=x, w=w, dy=dy).items()}
    y, dx, dw = ctx.empty((1, 72), np.uint16), ctx.empty((1, 136), np.uint16), ctx.empty((72, 136), np.uint16)
    got = []
    for one in ({}, {"stride": stride}):
        s = {name + "_stride": v for name in ("x", "y", "dy", "dx") for v in one.values()}
        ctx.linear(hip.Linear.of(a["x"], a["w"], y, **{k: v for k, v in s.items() if k in ("x_stride", "y_stride")}))
        ctx.linear_backward(hip.LinearGrad.of(a["dy"], a["x"], a["w"], dx=dx, dw=dw, **{k: v for k, v in s.items() if k != "y_stride"}))
        # one output: w is the single row
        w1 = hip.DeviceArray(ctx, a["w"].ptr, 272, np.dtype(np.uint16), (1, 136))
        dw1, dy1, dx1 = ctx.empty((1, 136), np.uint16), ctx.to_device(dy.reshape(72, 1)), ctx.empty((72, 136), np.uint16)
        ctx.linear_backward(hip.LinearGrad.of(dy1, a["w"], w1, dx=dx1, dw=dw1, **{k + "_stride": v for k in ("w", "dw") for v in one.values()}))
        ctx.synchronize()
        got.append([t.to_host() for t in (y, dx, dw, dw1, dx1)])
    assert all(np.array_equal(p, q) for p, q in zip(*got))
    within(wide(got[0][4]), wide(dy).T @ wide(w[:1]), 2.0 ** -8 * np.abs(wide(dy).T @ wide(w[:1])), "dx of one output")


def test_linear_backward_of_nothing(ctx):
    """No rows: dw and dbias are empty sums; no outputs: dx is."""
    e, w, db = ctx.empty(8, np.uint16), ctx.to_device(np.full((9, 5), 7, np.uint16)), ctx.to_device(np.full(9, 7.0, np.float32))
    dw = ctx.to_device(np.full((9, 5), 7, np.uint16))

    def part(*shape):
        return hip.DeviceArray(ctx, e.ptr, 0, np.dtype(np.uint16), shape)

    ctx.linear_backward(hip.LinearGrad.of(dy=part(0, 9), x=part(0, 5), w=w, dx=part(0, 5), dw=dw, dbias=db))
    ctx.synchronize()
    assert np.all(dw.to_host() == 0) and np.all(db.to_host() == 0)
    x, dx = ctx.to_device(np.full((40, 5), 7, np.uint16)), ctx.to_device(np.full((40, 5), 7, np.uint16))
    ctx.linear_backward(hip.LinearGrad.of(dy=part(40, 0), x=x, w=part(0, 5), dx=dx, dw=part(0, 5)))
    ctx.synchronize()
    assert np.all(dx.to_host() == 0)
    for a in (e, w, db, dw, x, dx):
        ctx.free(a)


def test_calls_leave_nothing_behind(ctx):
    """Calls of a block in the order of a training step, over and over, give the same bits: no state is left between them."""
    first = None
    for _ in range(3):
        got = run_backward(ctx, 200, 264, 136, "gelu", seed=9), run_linear(ctx, 200, 264, 136, activation="gelu", seed=9)
        flat = np.concatenate([got[0]["dx"].ravel(), got[0]["dw"].ravel(), got[1].ravel()])
        assert first is None or np.array_equal(first, flat)
        first = flat

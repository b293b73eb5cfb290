"""GPU parity: both projections of a gated block with their gate, their gradients, and products of 8-bit values with block scales, against float64.

Tolerances, from the arithmetic, as tests/test_gpu_linear.py's: a sum over k of terms of magnitude S in all is within (k / 16 + 8) 2^-23 S, and in 8 bits
each 64 products lose at most 64 times 2^-13 of the largest; block scales are powers of two and change neither. With g and u off by at most
eg and eu, and act(g) by another 4e-6 max(1, |g|) and 1.13 eg (no activation's slope passes 1.13): act(g) u is within
|act(g)| eu + (|u| + eu) (1.13 eg + 4e-6 max(1, |g|)) and the product's rounding. Results in bf16 add half a step of 8 bits.
The gradients' operands are rounded to bf16 before the products: half a step of 8 bits of each term.
"""
import numpy as np
import pytest

import ffn_reference as ref
import gated_reference as gated
from dotcompute_amd import hip
from test_gpu_linear import ACTS, bf16, cut_bound, sum_bound, wide, within
from test_gpu_rms_norm import Matrix

pytestmark = pytest.mark.gpu
HALF = ref.BF16 * (1 + 2.0 ** -8)


class Operand:
    """Rows of normal values in bf16 or e4m3, in a buffer of their own, with their scales; `values`: what they stand for."""

    def __init__(self, ctx, rng, rows, k, dtype, scale, odd, pad):
        x = rng.normal(size=(rows, k)) * scale
        self.scales = self.stride = None
        if dtype == "fp8":
            q, s = ref.rows_fp8(x.astype(np.float32))
            self.values, self.scales = ref.from_fp8(q) * s[:, None].astype(np.float64), ctx.to_device(s)
        elif dtype == "blocks":
            q, s = gated.rows_fp8(x * np.exp(rng.normal(size=(rows, 1))))
            self.values = gated.values(q, s)
            self.block = Matrix(ctx, s, np.uint8, 3 * odd, 5 * odd)
            self.scales, self.stride = self.block.a, self.block.stride
        else:
            q = ref.to_bf16(x)
            self.values = wide(q)
        self.m = Matrix(ctx, q, q.dtype, odd, pad)

    def free(self, ctx):
        ctx.free(self.m.base)
        if self.scales is not None:
            ctx.free(self.block.base if self.stride else self.scales)


def arguments(names, operands):
    """Arrays, scales and strides by their names in a call."""
    a = {}
    for (name, scales), o in zip(names, operands):
        a[name], a[name + "_stride"] = o.m.a, o.m.stride
        if o.scales is not None:
            a[scales] = o.scales
            if o.stride:
                a[scales + "_stride"] = o.stride
    return a


def z_bound(x, w, b, z, dtype):
    k = x.shape[1]
    off = sum_bound(k, np.abs(x) @ np.abs(w).T + (0 if b is None else np.abs(b)))
    return off + (cut_bound(x, w) if dtype != "bf16" else 0.0)


def run_gated(ctx, m, n, k, dtype="bf16", activation="silu", y="bf16", bias=True, pre=False, odd=0, seed=0):
    rng = np.random.default_rng(seed + 3 * m + 5 * n + 7 * k)
    x = Operand(ctx, rng, m, k, dtype, 1.0, odd, odd)
    ws = [Operand(ctx, rng, n, k, dtype, max(k, 1) ** -0.5, p * odd, q * odd) for p, q in ((3, 5), (1, 9))]
    a = arguments((("x", "x_scales"), ("w_gate", "gate_scales"), ("w_up", "up_scales")), [x] + ws)
    bs = [bf16(rng, n) for _ in range(2)] if bias else [None, None]
    for name, b in zip(("bias_gate", "bias_up"), bs):
        a[name] = None if b is None else ctx.to_device(b)
    np_y = np.uint16 if y == "bf16" else np.float32
    out = Matrix(ctx, np.zeros((m, n), np_y), np_y, odd, 7 * odd)
    kept = [Matrix(ctx, np.zeros((m, n), np.uint16), np.uint16, p * odd, q * odd) for p, q in ((1, 3), (0, 1))] if pre else []
    for name, q in zip(("pre_gate", "pre_up"), kept):
        a[name], a[name + "_stride"] = q.a, q.stride
    ctx.gated_linear(hip.GatedLinear.of(y=out.a, y_stride=out.stride, activation=activation, **a))
    ctx.synchronize()
    b64 = [None if b is None else wide(b) for b in bs]
    g, u, y64 = gated.gated(x.values, ws[0].values, ws[1].values, *b64, activation)
    eg, eu = (z_bound(x.values, w.values, b, z, dtype) for w, b, z in zip(ws, b64, (g, u)))
    for what, q, z, e in zip(("pre_gate", "pre_up"), kept, (g, u), (eg, eu)):
        within(wide(q.read()), z, e + HALF * np.abs(z) + 1e-37, what)
    got = out.read()
    got = wide(got) if y == "bf16" else got.astype(np.float64)
    off = np.abs(ref.act(activation, g)) * eu + (np.abs(u) + eu) * (1.13 * eg + 4e-6 * np.maximum(1.0, np.abs(g))) + 2.0 ** -23 * np.abs(y64)
    within(got, y64, off + (HALF * np.abs(y64) if y == "bf16" else 0.0) + 1e-37, "y")
    for o in [x] + ws:
        o.free(ctx)
    for q in kept + [out]:
        ctx.free(q.base)
    for name in ("bias_gate", "bias_up"):
        if a[name] is not None:
            ctx.free(a[name])
    return got


SHAPES = [(1, 1, 1), (1, 64, 64), (1, 1000, 777), (7, 48, 4096), (16, 512, 130), (17, 33, 8), (32, 4096, 1024), (33, 70, 40), (64, 64, 64),
          (100, 200, 300), (128, 256, 64), (130, 1030, 520), (257, 129, 1000), (300, 300, 4104), (777, 1111, 333), (1024, 2048, 192)]
TYPES = ["bf16", "fp8", "blocks"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gated_shapes(ctx, m, n, k, dtype):
    run_gated(ctx, m, n, k, dtype, "silu", pre=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(3, 50, 100), (31, 20, 33), (90, 140, 210), (300, 260, 513)])
def test_gated_strides_and_alignments(ctx, m, n, k, dtype):
    """Rows one element into their buffers, and further apart than they are long; nothing else is written."""
    run_gated(ctx, m, n, k, dtype, "gelu", pre=True, odd=1)
    run_gated(ctx, m, n, k, dtype, "gelu", "f32", bias=False, odd=1)


@pytest.mark.parametrize("activation", ACTS)
@pytest.mark.parametrize("m", [5, 200])
def test_gated_activations(ctx, activation, m):
    for y in ("bf16", "f32"):
        run_gated(ctx, m, 96, 128, "bf16", activation, y, pre=True)
        run_gated(ctx, m, 96, 128, "blocks", activation, y)


@pytest.mark.parametrize("k", [0, 5])
@pytest.mark.parametrize("dtype", TYPES)
def test_gated_of_next_to_nothing(ctx, k, dtype):
    """k = 0: the biases alone; no rows or no outputs: nothing."""
    for m, n in ((1, 1), (3, 41), (70, 70)):
        run_gated(ctx, m, n, k, dtype, pre=True)
        run_gated(ctx, m, n, k, dtype, y="f32", bias=False)
    e = ctx.empty(8, np.uint16)

    def part(*shape):
        return hip.DeviceArray(ctx, e.ptr, 0, np.dtype(np.uint16), shape)

    ctx.gated_linear(hip.GatedLinear.of(part(0, 4), part(2, 4), part(2, 4), part(0, 2)))
    ctx.gated_linear(hip.GatedLinear.of(part(2, 4), part(0, 4), part(0, 4), part(2, 0)))
    ctx.synchronize()
    ctx.free(e)


def test_gated_keeps_nonfinite_values_to_their_rows_and_columns(ctx):
    for m in (4, 70):
        rng = np.random.default_rng(m)
        x, wg, wu = bf16(rng, (m, 40)), bf16(rng, (48, 40)), bf16(rng, (48, 40))
        x[1, 3], x[2, 39] = ref.to_bf16(np.nan), ref.to_bf16(np.inf)
        wg[5, 7], wu[9, 0] = ref.to_bf16(np.nan), ref.to_bf16(np.nan)
        arrays = [ctx.to_device(a) for a in (x, wg, wu)] + [ctx.empty((m, 48), np.float32)]
        ctx.gated_linear(hip.GatedLinear.of(*arrays))
        ctx.synchronize()
        got = arrays[3].to_host()
        assert np.all(np.isnan(got[1])) and not np.any(np.isfinite(got[2][np.abs(got[2]) > 0])) and np.all(np.isnan(got[:, [5, 9]]))
        assert np.all(np.isfinite(np.delete(np.delete(got, [1, 2], axis=0), [5, 9], axis=1)))
        for a in arrays:
            ctx.free(a)


# ---- gradients -----------------------------------------------------------------------------------
def run_gated_backward(ctx, m, n, k, activation="silu", odd=0, outputs=("dx", "dw_gate", "dw_up", "dbias_gate", "dbias_up"), seed=0):
    rng = np.random.default_rng(seed + m + 3 * n + 5 * k)
    host = {"dy": bf16(rng, (m, n)), "x": bf16(rng, (m, k)), "w_gate": bf16(rng, (n, k)), "w_up": bf16(rng, (n, k)),
            "pre_gate": bf16(rng, (m, n)), "pre_up": bf16(rng, (m, n))}
    pads = {"dy": (1, 1), "x": (1, 3), "w_gate": (3, 1), "w_up": (1, 7), "pre_gate": (1, 5), "pre_up": (0, 1)}
    mats = {name: Matrix(ctx, v, np.uint16, pads[name][0] * odd, pads[name][1] * odd) for name, v in host.items()}
    shapes = {"dx": (m, k), "dw_gate": (n, k), "dw_up": (n, k)}
    results = {name: Matrix(ctx, np.zeros(shapes[name], np.uint16), np.uint16, odd, odd) for name in shapes if name in outputs}
    sums = {name: ctx.to_device(np.full(n, 5.0, np.float32)) for name in ("dbias_gate", "dbias_up")}
    every = {**mats, **results}
    ctx.gated_linear_backward(hip.GatedLinearGrad.of(activation=activation, **{name: q.a for name, q in every.items()},
                                                     **{name + "_stride": q.stride for name, q in every.items()},
                                                     **{name: a for name, a in sums.items() if name in outputs}))
    ctx.synchronize()
    v = {name: wide(a) for name, a in host.items()}
    dy, g, u, x = v["dy"], v["pre_gate"], v["pre_up"], v["x"]
    want = dict(zip(("dx", "dw_gate", "dw_up", "dbias_gate", "dbias_up"), gated.gated_grad(dy, x, v["w_gate"], v["w_up"], g, u, activation)))
    dz = {"gate": dy * u * ref.act_slope(activation, g), "up": dy * ref.act(activation, g)}
    # float32: the product of dy and u, its with the slope, or the activation's error
    off = {"gate": np.abs(dy * u) * 4e-6 * np.maximum(1.0, np.abs(g)) + 2.0 ** -22 * np.abs(dz["gate"]),
           "up": np.abs(dy) * 4e-6 * np.maximum(1.0, np.abs(g)) + 2.0 ** -23 * np.abs(dz["up"])}
    rough = {f: np.abs(dz[f]) * HALF + off[f] for f in dz}
    got = {name: wide(q.read()) for name, q in results.items()}
    if "dx" in got:
        wg, wu = np.abs(v["w_gate"]), np.abs(v["w_up"])
        s = np.abs(dz["gate"]) @ wg + np.abs(dz["up"]) @ wu
        bound = sum_bound(2 * n, s) + rough["gate"] @ wg + rough["up"] @ wu + HALF * np.abs(want["dx"]) + 1e-37
        within(got["dx"], want["dx"], bound, "dx")
    for f in ("gate", "up"):
        if "dw_" + f in got:
            w64 = want["dw_" + f]
            bound = sum_bound(m, np.abs(dz[f]).T @ np.abs(x)) + rough[f].T @ np.abs(x) + HALF * np.abs(w64) + 1e-37
            within(got["dw_" + f], w64, bound, "dw_" + f)
        db = sums["dbias_" + f].to_host()
        if "dbias_" + f in outputs:  # 64 rows a part, parts in 16 chains
            bound = (m / 1024 + 64) * 2.0 ** -24 * np.abs(dz[f]).sum(axis=0) + off[f].sum(axis=0) + 1e-37
            within(db, want["dbias_" + f], bound, "dbias_" + f)
            got["dbias_" + f] = db
        else:
            assert np.all(db == 5.0)
    for name, q in every.items():
        if name in mats:
            q.read()
        ctx.free(q.base)
    for a in sums.values():
        ctx.free(a)
    return got


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 64, 200), (5, 7, 9), (64, 64, 64), (70, 130, 50), (128, 256, 512), (257, 300, 129),
                                   (1000, 72, 333), (520, 1040, 264)])
@pytest.mark.parametrize("activation", ["none", "gelu"])
def test_gated_backward_shapes(ctx, m, n, k, activation):
    run_gated_backward(ctx, m, n, k, activation)
    run_gated_backward(ctx, m, n, k, activation, odd=1)


@pytest.mark.parametrize("activation", ACTS)
def test_gated_backward_activations(ctx, activation):
    run_gated_backward(ctx, 96, 200, 64, activation)


@pytest.mark.parametrize("m", [50, 100])
def test_gated_backward_in_parts(ctx, m):
    """Each gradient alone is the same bits as all of them together."""
    full = run_gated_backward(ctx, m, 136, 72)
    names = list(full)
    for outputs in [(name,) for name in names] + [("dw_gate", "dw_up"), ("dx", "dw_up"), ("dbias_gate", "dbias_up"), ("dw_up", "dbias_gate")]:
        got = run_gated_backward(ctx, m, 136, 72, outputs=outputs)
        assert set(got) == set(outputs) and all(np.array_equal(got[name], full[name]) for name in outputs)


def test_gated_backward_of_nothing(ctx):
    """No rows: the weights' and biases' gradients are empty sums; no outputs: dx is."""
    e, w = ctx.empty(8, np.uint16), ctx.to_device(np.full((9, 5), 7, np.uint16))
    dws = [ctx.to_device(np.full((9, 5), 7, np.uint16)) for _ in range(2)]
    dbs = [ctx.to_device(np.full(9, 7.0, np.float32)) for _ in range(2)]

    def part(*shape):
        return hip.DeviceArray(ctx, e.ptr, 0, np.dtype(np.uint16), shape)

    ctx.gated_linear_backward(hip.GatedLinearGrad.of(part(0, 9), part(0, 5), w, w, part(0, 9), part(0, 9), part(0, 5), *dws, *dbs))
    ctx.synchronize()
    assert all(np.all(a.to_host() == 0) for a in dws + dbs)
    x, dx = ctx.to_device(np.full((40, 5), 7, np.uint16)), ctx.to_device(np.full((40, 5), 7, np.uint16))
    ctx.gated_linear_backward(hip.GatedLinearGrad.of(part(40, 0), x, part(0, 5), part(0, 5), part(40, 0), part(40, 0), dx))
    ctx.synchronize()
    assert np.all(dx.to_host() == 0)
    for a in [e, w, x, dx] + dws + dbs:
        ctx.free(a)


def test_gated_backward_against_differences(ctx):
    """The gradients are those of sum(y dy), by central differences in float64 of the reference, whose step's error is 1e-8 here; bf16 as above."""
    rng = np.random.default_rng(3)
    m, n, k = 3, 4, 5
    host = [bf16(rng, s) for s in ((m, n), (m, k), (n, k), (n, k))]
    dy, x, wg, wu = (wide(a) for a in host)
    g, u, _ = gated.gated(x, wg, wu)
    g, u = ref.to_bf16(g), ref.to_bf16(u)
    arrays = [ctx.to_device(a) for a in host + [g, u]]
    outs = [ctx.empty(s, np.uint16) for s in ((m, k), (n, k), (n, k))] + [ctx.empty(n, np.float32) for _ in range(2)]
    ctx.gated_linear_backward(hip.GatedLinearGrad.of(*arrays, *outs))
    ctx.synchronize()
    at = [x, wg, wu, np.zeros(n), np.zeros(n)]
    # g and u were rounded to bf16, and dz is: each term is off by at most 2^-8 of itself for its u or act, 3 2^-8 through the slope, and 2^-8 for dz
    term = np.abs(dy) * (np.abs(u.astype(np.float64) * 0 + wide(u)) + np.abs(wide(g)) + 1)
    sizes = [term @ (np.abs(wg) + np.abs(wu)), term.T @ np.abs(x), term.T @ np.abs(x), term.sum(axis=0), term.sum(axis=0)]
    for i, (out, size) in enumerate(zip(outs, sizes)):
        got = out.to_host()
        got = wide(got) if got.dtype == np.uint16 else got
        for where in np.ndindex(got.shape):
            both = []
            for step in (1e-5, -1e-5):
                moved = [a.copy() for a in at]
                moved[i][where] += step
                both.append(np.sum(gated.gated(*moved)[2] * dy))
            want = (both[0] - both[1]) / 2e-5
            assert abs(got[where] - want) <= 6 / 256 * size[where] + abs(want) / 256, (i, where)
    for a in arrays + outs:
        ctx.free(a)


# ---- block scales ----------------------------------------------------------------------------------
def run_blocks(ctx, m, n, k, activation="none", y="bf16", bias=True, residual=False, odd=0, in_place=False):
    rng = np.random.default_rng(3 * m + 5 * n + 7 * k)
    x, w = Operand(ctx, rng, m, k, "blocks", 1.0, odd, odd), Operand(ctx, rng, n, k, "blocks", max(k, 1) ** -0.5, 3 * odd, 5 * odd)
    a = arguments((("x", "x_scales"), ("w", "w_scales")), [x, w])
    np_y = np.uint16 if y == "bf16" else np.float32
    out = Matrix(ctx, np.zeros((m, n), np_y), np_y, odd, 7 * odd)
    b64 = r64 = r = None
    if bias:
        b = bf16(rng, n)
        b64, a["bias"] = wide(b), ctx.to_device(b)
    if residual:
        host = bf16(rng, (m, n))
        r64 = wide(host)
        r = out if in_place else Matrix(ctx, host, np.uint16, 0, odd)
        if in_place:
            out.base.copy_from(np.concatenate([host.reshape(-1), np.full(8, 77, np.uint16)]))
        a["residual"], a["residual_stride"] = r.a, r.stride
    ctx.linear_blocks(hip.LinearBlocks.of(y=out.a, y_stride=out.stride, activation=activation, **a))
    ctx.synchronize()
    z64, y64 = ref.linear(x.values, w.values, b64, activation, r64)
    off = 1.13 * z_bound(x.values, w.values, b64, z64, "blocks") + 4e-6 * (np.maximum(1.0, np.abs(z64)) + np.abs(y64))
    got = out.read()
    got = wide(got) if y == "bf16" else got.astype(np.float64)
    within(got, y64, off + (HALF * np.abs(y64) if y == "bf16" else 0.0) + 1e-37, "y")
    for o in (x, w):
        o.free(ctx)
    for q in {id(q): q for q in (out, r) if q is not None}.values():
        ctx.free(q.base)
    if bias:
        ctx.free(a["bias"])


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_blocks_shapes(ctx, m, n, k):
    run_blocks(ctx, m, n, k, "silu", residual=True)
    run_blocks(ctx, m, n, k, "gelu", "f32", bias=False)


@pytest.mark.parametrize("m,n,k", [(3, 50, 100), (31, 20, 33), (90, 140, 210), (300, 260, 513), (4, 40, 0), (70, 70, 0)])
def test_linear_blocks_strides_and_alignments(ctx, m, n, k):
    run_blocks(ctx, m, n, k, "gelu_tanh", residual=True, odd=1)
    run_blocks(ctx, m, n, k, "relu", "f32", odd=1)
    run_blocks(ctx, m, n, k, "none", residual=True, in_place=True)


def whole_numbers(ctx, rng, rows, k):
    """Values -6..6 times 1/2, 1 or 2 by block, as codes with block scales; and themselves."""
    v = rng.integers(-6, 7, size=(rows, k)).astype(np.float64)
    s = rng.integers(126, 129, size=(gated.blocks(k), rows)).astype(np.uint8)
    q = ref.to_fp8(v)
    return q, s, gated.values(q, s)


@pytest.mark.parametrize("m,n,k", SHAPES + [(2048, 4096, 256), (512, 512, 4096), (1537, 1025, 1023)])
def test_block_scales_of_whole_numbers_are_exact(ctx, m, n, k):
    """Every sum is a whole number of quarters below 2^22, in any order: each scale reaches its row and its block of k and no other."""
    rng = np.random.default_rng(m + n + k)
    (xq, xs, x), (wq, ws, w), (uq, us, u) = (whole_numbers(ctx, rng, r, k) for r in (m, n, n))
    dev = {name: ctx.to_device(a) for name, a in dict(x=xq, w=wq, u=uq, xs=xs, ws=ws, us=us).items()}
    y = ctx.empty((m, n), np.float32)
    ctx.linear_blocks(hip.LinearBlocks.of(dev["x"], dev["w"], dev["xs"], dev["ws"], y))
    ctx.synchronize()
    assert np.array_equal(y.to_host(), x @ w.T)
    # a gated layer's two projections: a bias of one and a weight of zeros make one of the factors 1
    one, none = ctx.to_device(np.full(n, 0x3F80, np.uint16)), ctx.to_device(np.zeros((n, k), np.uint8))
    for gate, up, biases, want in ((dev["u"], none, dict(bias_up=one), x @ u.T), (none, dev["u"], dict(bias_gate=one), x @ u.T)):
        ctx.gated_linear(hip.GatedLinear.of(dev["x"], gate, up, y, x_scales=dev["xs"], gate_scales=dev["us"], up_scales=dev["us"],
                                            activation="none", **biases))
        ctx.synchronize()
        assert np.array_equal(y.to_host(), want)
    for a in list(dev.values()) + [y, one, none]:
        ctx.free(a)


@pytest.mark.parametrize("m", [5, 40, 300])
def test_block_scales_of_the_ends(ctx, m):
    """A NaN scale reaches its row, or its column; the largest and the smallest that leave a float keep their values; others stay the same bits."""
    rng = np.random.default_rng(m)
    n, k = 200, 400
    (xq, xs, _), (wq, ws, _) = (whole_numbers(ctx, rng, r, k) for r in (m, n))
    results = []
    for bad in (False, True):
        xs, ws = xs.copy(), ws.copy()
        if bad:
            xs[1, 2], ws[3, 7], ws[0, n - 1] = 255, 255, 255
            xs[:, 0], xs[:, m - 1] = 127 + 100, 127 - 100
        arrays = [ctx.to_device(a) for a in (xq, wq, xs, ws)] + [ctx.empty((m, n), np.float32)]
        ctx.linear_blocks(hip.LinearBlocks.of(*arrays))
        ctx.synchronize()
        results.append(arrays[4].to_host())
        for a in arrays:
            ctx.free(a)
    good, got = results
    assert np.all(np.isnan(got[2])) and np.all(np.isnan(got[:, [7, n - 1]]))
    rows, cols = np.setdiff1d(np.arange(m), [0, 2, m - 1]), np.setdiff1d(np.arange(n), [7, n - 1])
    assert np.array_equal(got[np.ix_(rows, cols)], good[np.ix_(rows, cols)])
    for row, scale in ((0, 2.0 ** 100), (m - 1, 2.0 ** -100)):
        flat = gated.values(xq[row:row + 1], np.full((gated.blocks(k), 1), 127, np.uint8)) @ gated.values(wq, ws).T
        assert np.array_equal(got[row, cols], (flat[0] * scale)[cols])


def test_calls_leave_nothing_behind(ctx):
    """Calls of a block in the order of a training step, over and over, give the same bits: no state is left between them."""
    first = None
    for _ in range(3):
        got = [run_gated(ctx, 200, 264, 136, dtype, seed=9) for dtype in TYPES]
        back = run_gated_backward(ctx, 200, 264, 136, seed=9)
        flat = np.concatenate([a.ravel() for a in got + list(back.values())])
        assert first is None or np.array_equal(first, flat)
        first = flat

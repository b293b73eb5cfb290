"""GPU parity: every kernel of the linear layers, at shapes that it takes (tests/linear_kernels.py), against float64; with the residual in place,
with values that are no numbers, and with each activation. Tolerances are those of tests/test_gpu_linear.py."""
import numpy as np
import pytest

import ffn_reference as ref
from dotcompute_amd import hip
from linear_kernels import FORWARD, LARGE, PAIRS, SINGLES
from test_gpu_linear import ACTS, bf16, run_backward, run_linear

pytestmark = pytest.mark.gpu

forward = pytest.mark.parametrize("kernel,m,n,k,dtype", FORWARD, ids=lambda v: str(v))


@forward
def test_forward(ctx, kernel, m, n, k, dtype):
    run_linear(ctx, m, n, k, dtype, "silu", pre=True, residual=True)
    run_linear(ctx, m, n, k, dtype, "gelu", "f32", bias=False)


@forward
def test_over_the_residual(ctx, kernel, m, n, k, dtype):
    run_linear(ctx, m, n, k, dtype, "relu", residual=True, in_place=True)


@pytest.mark.slow
@pytest.mark.parametrize("kernel,m,n,k,dtype", LARGE, ids=lambda v: str(v))
def test_forward_large(ctx, kernel, m, n, k, dtype):
    run_linear(ctx, m, n, k, dtype, "silu", pre=True, residual=True, in_place=True)


@forward
def test_whole_numbers_are_exact(ctx, kernel, m, n, k, dtype):
    """Values -6..6: every sum is a whole number below 2^24, in any order."""
    rng = np.random.default_rng(m + n + k)
    x, w = (rng.integers(-6, 7, size=(r, k)).astype(np.float32) for r in (m, n))
    code, ones = (ref.to_fp8 if dtype == "fp8" else ref.to_bf16), [None, None]
    if dtype == "fp8":
        ones = [ctx.to_device(np.ones(r, np.float32)) for r in (m, n)]
    a = [ctx.to_device(code(x)), ctx.to_device(code(w)), ctx.empty((m, n), np.float32)]
    ctx.linear(hip.Linear.of(*a, x_scales=ones[0], w_scales=ones[1]))
    ctx.synchronize()
    assert np.array_equal(a[2].to_host(), x @ w.T)
    for q in a + [s for s in ones if s is not None]:
        ctx.free(q)


@forward
def test_no_numbers_stay_in_their_rows_and_columns(ctx, kernel, m, n, k, dtype):
    """A NaN in x reaches its row, one in w its column, an infinity in x (8 bits: in a scale) its row; the rest are the same bits as without."""
    rng = np.random.default_rng(m + k)
    to = (lambda v: ref.to_fp8(v)) if dtype == "fp8" else ref.to_bf16
    x, w = to(rng.normal(size=(m, k))), to(rng.normal(size=(n, k)))
    nan = np.uint8(0x7F) if dtype == "fp8" else np.uint16(0x7FC0)
    row, far, col = m // 2, m - 1, n - 1
    got = []
    for bad in (False, True):
        xs, ws = np.ones(m, np.float32), np.ones(n, np.float32)
        if bad:
            x[row, k - 1] = w[col, 0] = nan
            if dtype == "fp8":
                xs[far] = np.inf
            else:
                x[far, k // 2] = ref.to_bf16(np.inf)
        a = [ctx.to_device(x), ctx.to_device(w), ctx.empty((m, n), np.float32)]
        s = [ctx.to_device(xs), ctx.to_device(ws)] if dtype == "fp8" else [None, None]
        ctx.linear(hip.Linear.of(*a, x_scales=s[0], w_scales=s[1]))
        ctx.synchronize()
        got.append(a[2].to_host())
        for q in a + [q for q in s if q is not None]:
            ctx.free(q)
    clean, dirty = got
    assert np.all(np.isnan(dirty[row])) and np.all(np.isnan(dirty[:, col])) and not np.any(np.isfinite(dirty[far]))
    rest = np.ones((m, n), bool)
    rest[[row, far]] = False
    rest[:, col] = False
    assert np.all(np.isfinite(clean)) and np.array_equal(clean[rest], dirty[rest])


@pytest.mark.parametrize("activation", ACTS)
@pytest.mark.parametrize("kernel,m,n,k,dtype", [c for c in FORWARD if c[0] in ("64", "64/split", "128x2")], ids=lambda v: str(v))
def test_activations(ctx, activation, kernel, m, n, k, dtype):
    for y in ("bf16", "f32"):
        run_linear(ctx, m, n, k, dtype, activation, y, pre=True, residual=True)


@pytest.mark.parametrize("kernel,m,n,k", PAIRS, ids=lambda v: str(v))
def test_both_gradients(ctx, kernel, m, n, k):
    run_backward(ctx, m, n, k, "silu")


@pytest.mark.parametrize("kernel,rows,sums,cols", SINGLES, ids=lambda v: str(v))
def test_one_gradient(ctx, kernel, rows, sums, cols):
    """dx of a layer, and dw of one with as many rows as that has outputs: the same kernel."""
    run_backward(ctx, rows, sums, cols, "gelu", dw=False)
    run_backward(ctx, sums, rows, cols, "gelu", dx=False, dbias=False)


@pytest.mark.parametrize("kernel,m,n,k", [c for c in PAIRS if c[0] in ("64x2", "128", "128/a/b", "256", "256/a")], ids=lambda v: str(v))
def test_gradients_of_no_numbers(ctx, kernel, m, n, k):
    """A NaN in dy reaches its row of dx, of dw and its dbias; one in x a column of dw, one in w a column of dx. The rest are the same bits."""
    rng = np.random.default_rng(m + n + k)
    dy, x, w, pre = bf16(rng, (m, n)), bf16(rng, (m, k)), bf16(rng, (n, k)), bf16(rng, (m, n))
    i, j, cx, cw = m - 1, n - 1, k - 1, k // 2
    got = []
    for bad in (False, True):
        if bad:
            dy[i, j] = x[0, cx] = w[0, cw] = 0x7FC0
        on = [ctx.to_device(a) for a in (dy, x, w, pre)]
        out = [ctx.empty((m, k), np.uint16), ctx.empty((n, k), np.uint16), ctx.empty(n, np.float32)]
        ctx.linear_backward(hip.LinearGrad.of(*on, dx=out[0], dw=out[1], dbias=out[2], activation="silu"))
        ctx.synchronize()
        got.append([ref.from_bf16(out[0].to_host()), ref.from_bf16(out[1].to_host()), out[2].to_host()])
        for a in on + out:
            ctx.free(a)
    for clean, dirty, row, col in ((got[0][0], got[1][0], i, cw), (got[0][1], got[1][1], j, cx)):
        assert np.all(np.isnan(dirty[row])) and np.all(np.isnan(dirty[:, col]))
        rest = np.ones(clean.shape, bool)
        rest[row], rest[:, col] = False, False
        assert np.all(np.isfinite(clean)) and np.array_equal(clean[rest], dirty[rest])
    assert np.isnan(got[1][2][j]) and np.array_equal(np.delete(got[0][2], j), np.delete(got[1][2], j))

"""GPU parity: gradients over more rows than a sum along them may have, dx and dbias alone.

Whole numbers, so that every sum is exact in float32 (dbias adds at most 2^23 + 9 values of -1, 0 and 1 in any order).
"""
import numpy as np
import pytest

import ffn_reference as ref
from dotcompute_amd import hip

pytestmark = [pytest.mark.gpu, pytest.mark.slow]


@pytest.mark.parametrize("activation", ["none", "relu"])
def test_gradients_over_many_rows(ctx, activation):
    m, n, k = (1 << 23) + 9, 8, 24
    rng = np.random.default_rng(1)
    dy, w = rng.integers(-1, 2, size=(m, n), dtype=np.int8), rng.integers(-6, 7, size=(n, k), dtype=np.int8)
    pre = rng.integers(-1, 2, size=(m, n), dtype=np.int8)
    on = [ctx.to_device(ref.to_bf16(a)) for a in (dy, w, pre)]
    x, dx, db = ctx.empty((m, k), np.uint16), ctx.empty((m, k), np.uint16), ctx.empty(n, np.float32)
    ctx.linear_backward(hip.LinearGrad.of(on[0], x, on[1], pre=on[2] if activation == "relu" else None, dx=dx, dbias=db,
                                          activation=activation))
    ctx.synchronize()
    dz = dy * (pre > 0) if activation == "relu" else dy
    assert np.array_equal(db.to_host(), dz.sum(axis=0, dtype=np.int64))
    got = dx.to_host()
    for at in range(0, m, 1 << 20):
        rows = slice(at, at + (1 << 20))
        assert np.array_equal(ref.from_bf16(got[rows]), dz[rows].astype(np.float32) @ w.astype(np.float32)), at
    for a in on + [x, dx, db]:
        ctx.free(a)

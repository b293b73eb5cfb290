"""A gated layer over the most rows that it may have, and more results than 32 bits count: with k = 0, whose results are the biases' alone, act(bg) bu."""
import numpy as np
import pytest

import ffn_reference as ref
from dotcompute_amd import hip

pytestmark = [pytest.mark.gpu, pytest.mark.slow]
U16 = np.dtype(np.uint16)


def test_biases_alone_over_the_most_rows(ctx):
    """2^30 - 1 rows of nine results, two lanes' work each: 2^31 of them. Products of whole numbers below 2^8 are bf16 values."""
    m, n = (1 << 30) - 1, 9
    bg, bu = np.arange(1, 10, dtype=np.float32), np.arange(3, 12, dtype=np.float32)
    biases = [ctx.to_device(ref.to_bf16(b)) for b in (bg, bu)]
    y = ctx.empty((m, n), np.uint16)
    x, w = (hip.DeviceArray(ctx, biases[0].ptr, 0, U16, (rows, 0)) for rows in (m, n))

    def rows(first, count):
        return hip.DeviceArray(ctx, y.ptr + 2 * n * first, 2 * n * count, U16, (count, n))

    places = [0, 1 << 24, (1 << 28) - 1000, (1 << 29) - 1000, (1 << 30) * 3 // 4, m - 4096]
    places += [int(v) for v in np.random.default_rng(1).integers(0, m - 4096, size=40)]
    for at in places:
        rows(at, 4096).copy_from(np.zeros((4096, n), np.uint16))
    ctx.gated_linear(hip.GatedLinear.of(x, w, w, y, *biases, activation="relu"))
    ctx.synchronize()
    want = np.broadcast_to(ref.to_bf16(bg * bu), (4096, n))
    for at in places:
        assert np.array_equal(rows(at, 4096).to_host(), want), at
    for a in biases + [y]:
        ctx.free(a)

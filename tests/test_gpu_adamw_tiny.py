"""GPU parity: 8-bit AdamW states that have faded to the smallest floats, as those of values whose gradients stay zero do."""
import numpy as np
import pytest

import ffn_reference as ref
from dotcompute_amd import hip

pytestmark = pytest.mark.gpu


def test_states_that_fade(ctx):
    """A block each for maxima of m from 1e-35 down; gradients of zero, so m is 0.9 of what it was: to half a step of 4 bits or of the
    smallest code, the rounding of small scales (21 bits) and products (float32's smallest value) beside it."""
    tops = np.float32([1e-35, 2e-36, 1.4e-36, 1.2e-36, 1e-37, 1e-38])
    n = tops.size * ref.BLOCK
    rng = np.random.default_rng(1)
    codes = ref.to_fp8(rng.uniform(-448, 448, size=n))
    codes[::ref.BLOCK] = ref.to_fp8(448.0)
    scales = np.maximum(tops / np.float32(448), np.float32(2.0 ** -128))
    host = dict(param=np.zeros(n, np.float32), grad=np.zeros(n, np.float32), m=codes, v=np.full(n, 0x38, np.uint8), m_scales=scales,
                v_scales=np.ones(tops.size, np.float32))
    on = {name: ctx.to_device(a) for name, a in host.items()}
    ctx.adamw_step(hip.AdamW.of(lr=1e-3, step=5, weight_decay=0.0), hip.AdamWTensors.of([on]))
    ctx.synchronize()
    want = 0.9 * ref.from_fp8(codes).astype(np.float64) * np.repeat(scales.astype(np.float64), ref.BLOCK)
    scale = np.repeat(on["m_scales"].to_host().astype(np.float64), ref.BLOCK)
    off = np.abs(ref.from_fp8(on["m"].to_host()) * scale - want)
    bound = np.maximum(np.abs(want) * ref.FP8, ref.LEAST / 2 * scale) * (1 + 2.0 ** -16) + 2.0 ** -148
    assert np.all(off <= bound), (off / bound).reshape(-1, ref.BLOCK).max(axis=1)
    for a in on.values():
        ctx.free(a)

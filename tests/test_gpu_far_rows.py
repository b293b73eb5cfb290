"""The feed-forward operators where offsets pass 32 bits: rows that lie gigabytes apart, and a tensor of more than 2^31 elements.

The same rows close together go through the same kernels, so the results are the same bits.
"""
import numpy as np
import pytest

import ffn_reference as ref
from dotcompute_amd import hip

pytestmark = [pytest.mark.gpu, pytest.mark.slow]


class Far:
    """A matrix whose rows lie `stride` elements apart in one allocation."""

    def __init__(self, ctx, host, stride):
        self.ctx, self.host, self.stride = ctx, host, stride
        self.base = ctx.empty((host.shape[0] - 1) * stride + host.shape[1], host.dtype)
        self.a = hip.DeviceArray(ctx, self.base.ptr, self.base.nbytes, host.dtype, host.shape)
        for r in range(host.shape[0]):
            self.row(r).copy_from(host[r])

    def row(self, r):
        size, cols = self.host.dtype.itemsize, self.host.shape[1]
        return hip.DeviceArray(self.ctx, self.base.ptr + r * self.stride * size, cols * size, self.host.dtype, (cols,))

    def read(self):
        return np.stack([self.row(r).to_host() for r in range(self.host.shape[0])])

    def free(self):
        self.ctx.free(self.base)


def both(ctx, matrices, run, outputs, stride):
    """What run() leaves in `outputs`, with dense matrices and with far ones."""
    got = []
    for s in (None, stride):
        m = {name: Far(ctx, h, h.shape[1] if s is None else s) for name, h in matrices.items()}
        run({name: q.a for name, q in m.items()}, {name + "_stride": q.stride for name, q in m.items()})
        ctx.synchronize()
        got.append([m[name].read() for name in outputs])
        for q in m.values():
            q.free()
    for near, far in zip(*got):
        assert np.array_equal(near, far)
    return got[0]


def bf16(rng, *shape):
    return ref.to_bf16(rng.normal(size=shape))


def test_norm_of_far_rows(ctx):
    rng = np.random.default_rng(1)
    w = ctx.to_device(bf16(rng, 520))
    dw = ctx.empty(520, np.float32)
    blank = np.zeros((5, 520), np.uint16)
    mats = {"x": bf16(rng, 5, 520), "residual": bf16(rng, 5, 520), "sum": blank, "y": blank}
    both(ctx, mats, lambda a, s: ctx.rms_norm(hip.RmsNorm.of(weight=w, **a, **s)), ("sum", "y"), (1 << 30) + 8)
    mats = {"dy": bf16(rng, 5, 520), "h": bf16(rng, 5, 520), "dx": blank}
    both(ctx, mats, lambda a, s: ctx.rms_norm_backward(hip.RmsNormGrad.of(weight=w, dweight=dw, **a, **s)), ("dx",), (1 << 30) + 8)
    ctx.free(w), ctx.free(dw)


@pytest.mark.parametrize("m", [20, 300])
def test_linear_to_far_rows(ctx, m):
    """Results, residual and pre far apart (operands' rows are at most 2^23 elements long, and copied where they lie further)."""
    rng = np.random.default_rng(m)
    x, w = ctx.to_device(bf16(rng, m, 136)), ctx.to_device(bf16(rng, 72, 136))
    blank = np.zeros((m, 72), np.uint16)
    stride = (1 << 33) // m // 8 * 8
    y, _ = both(ctx, {"y": blank, "pre": blank, "residual": bf16(rng, m, 72)},
                lambda a, s: ctx.linear(hip.Linear.of(x, w, activation="silu", **a, **s)), ("y", "pre"), stride)
    assert np.any(y)
    ctx.free(x), ctx.free(w)


def test_linear_of_far_rows(ctx):
    rng = np.random.default_rng(3)
    mats = {"x": bf16(rng, 6, 136), "w": bf16(rng, 7, 136), "y": np.zeros((6, 7), np.uint16)}
    both(ctx, mats, lambda a, s: ctx.linear(hip.Linear.of(**a, **s)), ("y",), (1 << 30) + 8)
    mats = {"dy": bf16(rng, 6, 24), "pre": bf16(rng, 6, 24), "x": bf16(rng, 6, 136), "w": bf16(rng, 24, 136),
            "dx": np.zeros((6, 136), np.uint16), "dw": np.zeros((24, 136), np.uint16)}
    both(ctx, mats, lambda a, s: ctx.linear_backward(hip.LinearGrad.of(activation="gelu", **a, **s)), ("dx", "dw"), (1 << 28) + 8)


def test_adamw_past_31_bits(ctx):
    """The last elements of a tensor of 2^31 + 1000, in 8-bit states, step as a tensor of their own does."""
    n, tail = (1 << 31) + 1000, 1000 + 256 * 4
    rng = np.random.default_rng(4)
    parts = {"param": np.float32, "grad": np.uint16, "m": np.uint8, "v": np.uint8, "m_scales": np.float32, "v_scales": np.float32,
             "copy": np.uint16}
    full = {name: ctx.empty(-(-n // 256) if name.endswith("scales") else n, t) for name, t in parts.items()}
    for a in full.values():
        hip.check(hip.load().dc_hip_memset_async(ctx.handle, a.ptr, 0, a.nbytes), "memset")
    small, ends = {}, {}
    for name, a in full.items():
        size = -(-tail // 256) if name.endswith("scales") else tail
        host = {"param": rng.normal(size=size).astype(np.float32), "grad": bf16(rng, size)}.get(name, np.zeros(size, parts[name]))
        small[name] = ctx.to_device(host)
        item = np.dtype(parts[name]).itemsize
        ends[name] = hip.DeviceArray(ctx, a.ptr + (a.size - size) * item, size * item, np.dtype(parts[name]), (size,)).copy_from(host)
    for step in (1, 2):
        for tensors in (full, small):
            ctx.adamw_step(hip.AdamW.of(lr=1e-2, step=step), hip.AdamWTensors.of([tensors]))
    ctx.synchronize()
    for name, a in small.items():
        assert np.array_equal(ends[name].to_host(), a.to_host()), name
        assert np.any(a.to_host())
    for a in list(full.values()) + list(small.values()):
        ctx.free(a)

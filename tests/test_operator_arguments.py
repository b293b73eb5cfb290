"""CPU: what the binding looks at before an operator's call, since a kernel is handed addresses alone."""
import types

import numpy as np
import pytest

from dotcompute_amd import hip

P = 4096  # an address that nobody reads
BF16, F32, CODE = np.dtype(np.uint16), np.dtype(np.float32), np.dtype(np.uint8)


def context(*sizes):
    """A context with allocations of those many bytes, far from each other."""
    ctx = types.SimpleNamespace(handle=None)
    ctx._arrays = [hip.DeviceArray(ctx, P + (i << 20), size, CODE, (size,)) for i, size in enumerate(sizes)]
    return ctx


def rows(ctx, which, at, shape, dtype=BF16):
    """A matrix whose rows start `at` elements into an allocation."""
    return hip.DeviceArray(ctx, ctx._arrays[which].ptr + at * dtype.itemsize, int(np.prod(shape)) * dtype.itemsize, dtype, shape)


def test_rows_end_within_their_allocation():
    """Three rows of 8, 10 apart, 2 elements in, take 30 elements."""
    for size, fits in ((60, True), (59, False), (1 << 16, True), (48, False)):
        ctx = context(size, 48, 1 << 16)
        x, w, y = rows(ctx, 0, 2, (3, 8)), rows(ctx, 2, 0, (3, 8)), rows(ctx, 2, 0, (3, 3))
        if fits:
            assert hip.Linear.of(x, w, y, x_stride=10).x_stride == 10
        else:
            with pytest.raises(ValueError, match="x_stride"):
                hip.Linear.of(x, w, y, x_stride=10)
    ctx = context(60, 48, 1 << 16)
    x, w = rows(ctx, 0, 2, (3, 8)), rows(ctx, 2, 0, (8,))
    assert hip.RmsNorm.of(x, w, x, x_stride=10, y_stride=10).y_stride == 10
    for bad in (dict(y_stride=11), dict(x_stride=11)):
        with pytest.raises(ValueError, match="stride"):
            hip.RmsNorm.of(x, w, x, **bad)
    # a single row's stride says nothing; memory of others is taken at its word
    one = rows(ctx, 0, 2, (1, 8))
    assert hip.RmsNorm.of(one, w, one, x_stride=1 << 40).x_stride == 1 << 40
    other = hip.DeviceArray(ctx, P + (9 << 20), 48, BF16, (3, 8))
    assert hip.RmsNorm.of(other, w, other, x_stride=100, y_stride=100).x_stride == 100


def array(shape, dtype):
    return hip.DeviceArray(None, P, int(np.prod(shape)) * dtype.itemsize, dtype, shape)


@pytest.mark.parametrize("name", ["m_scales", "v_scales"])
@pytest.mark.parametrize("dtype", [BF16, CODE], ids=["u16", "u8"])
def test_scales_of_adamw_states_are_float32(name, dtype):
    """The kernel reads and writes four bytes of each: fewer would be another array's."""
    part = dict(param=array((300,), F32), grad=array((300,), BF16), m=array((300,), CODE), v=array((300,), CODE),
                m_scales=array((2,), F32), v_scales=array((2,), F32))
    assert hip.AdamWTensors.of([part]).state_dtype == hip.DTYPE_FP8
    with pytest.raises(ValueError, match="types"):
        hip.AdamWTensors.of([{**part, name: array((2,), dtype)}])


@pytest.mark.parametrize("kind", [int, np.int64, np.int32])
def test_sizes_of_large_arrays(kind):
    """Elements are counted in whole numbers, whatever the shape's are."""
    a = hip.DeviceArray(None, P, 1 << 33, CODE, (kind(1 << 17), kind(1 << 16)))
    assert a.size == 1 << 33 and type(a.size) is int


def test_a_step_leaves_its_argument_block_alone():
    """One block of numbers serves tensors of either states, in any order and from any thread."""
    ctx = types.SimpleNamespace(handle=None)
    args = hip.AdamW.of(lr=1e-3)
    before = bytes(args)
    with pytest.raises(hip.HipError):  # (no context)
        hip.Context.adamw_step(ctx, args, hip.AdamWTensors((hip.AdamWTensor * 0)(), hip.DTYPE_FP8, []))
    assert bytes(args) == before


def test_rows_to_8_bits_take_strides():
    ctx = context(60, 48, 1 << 16)
    x, q, s = rows(ctx, 0, 2, (3, 8)), rows(ctx, 1, 0, (3, 8), CODE), rows(ctx, 2, 0, (3,), F32)
    for bad in (dict(x_stride=11), dict(q_stride=21)):
        with pytest.raises(ValueError, match="stride"):
            hip.Context.quantize_fp8(ctx, x, q, s, **bad)
    for status, strides in ((hip.DC_ERR_DIMENSION, dict(x_stride=7)), (hip.DC_ERR_DIMENSION, dict(q_stride=7)),
                            (hip.DC_ERR_INVALID_ARGUMENT, dict(x_stride=10, q_stride=20)), (hip.DC_ERR_INVALID_ARGUMENT, {})):
        with pytest.raises(hip.HipError) as e:  # (the last two: no context)
            hip.Context.quantize_fp8(ctx, x, q, s, **strides)
        assert e.value.status == status


def test_sums_along_many_rows_are_refused_where_they_are_asked_for():
    """m beyond 2^23 is too long for dw's sums, and nothing to the other gradients (which get as far as the missing context)."""
    n = (1 << 23) + 1
    args = dict(m=n, n=8, k=8, dy=P, x=P, w=P, dy_stride=8, x_stride=8, w_stride=8, dx_stride=8, dw_stride=8)
    for outputs, status in ((dict(dw=P), hip.DC_ERR_UNSUPPORTED), (dict(dx=P, dw=P), hip.DC_ERR_UNSUPPORTED),
                            (dict(dx=P), hip.DC_ERR_INVALID_ARGUMENT), (dict(dbias=P), hip.DC_ERR_INVALID_ARGUMENT)):
        assert hip.load().dc_hip_linear_backward(None, hip.LinearGrad(**args, **outputs)) == status

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

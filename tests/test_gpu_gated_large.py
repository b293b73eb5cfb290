"""GPU parity: the gated block's operators on operands of just over 96 MiB, which their kernels load as not to be kept by the caches: each such kernel, by
the tests and tolerances of smaller ones."""
import pytest

from test_gpu_gated import run_gated, run_gated_backward
from test_gpu_layer_norm import test_layer_norm as layer_norm
from test_gpu_layer_norm import test_layer_norm_backward as layer_norm_backward
from test_gpu_layer_norm import test_quantize_blocks as quantize_blocks

pytestmark = pytest.mark.gpu
LARGE = 96 << 20


@pytest.mark.parametrize("rows,cols,dtype", [(6200, 2051, "bf16"), (21000, 601, "bf16"), (1060, 12001, "bf16"), (3100, 2051, "f32"), (420, 15217, "f32"), (8300, 4100, "bf16")])
def test_layer_norm(ctx, rows, cols, dtype):
    assert rows * cols * (8 if dtype == "bf16" else 16) > LARGE
    layer_norm(ctx, rows, cols, dtype)  # (the last shape in 8 bits too)


@pytest.mark.parametrize("rows,cols,dtype", [(6200, 2051, "bf16"), (1060, 12001, "bf16"), (3100, 2051, "f32"), (1250, 5101, "f32"), (621, 10241, "f32")])
def test_layer_norm_backward(ctx, rows, cols, dtype):
    assert rows * cols * (8 if dtype == "bf16" else 16) > LARGE
    layer_norm_backward(ctx, rows, cols, dtype)


@pytest.mark.parametrize("rows,cols,dtype", [(8301, 4101, "bf16"), (5001, 4100, "f32")])
def test_quantize_blocks(ctx, rows, cols, dtype):
    assert rows * cols * (3 if dtype == "bf16" else 5) > LARGE
    quantize_blocks(ctx, rows, cols, dtype)


@pytest.mark.parametrize("m,n,k,dtype", [(1, 6200, 4104, "bf16"), (13, 6200, 4104, "bf16"), (40, 6200, 4104, "bf16"), (3, 12400, 4112, "fp8"), (3, 12400, 4112, "blocks")])
def test_gated(ctx, m, n, k, dtype):
    assert 2 * n * k * (2 if dtype == "bf16" else 1) > LARGE
    run_gated(ctx, m, n, k, dtype, "silu", pre=True)


def test_gated_backward(ctx):
    assert 2600 * 2803 * 14 > LARGE
    run_gated_backward(ctx, 2600, 2803, 72, "silu")

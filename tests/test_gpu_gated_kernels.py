"""GPU parity: every kernel of the gated layers and of the products with block scales, at shapes that it takes (tests/gated_kernels.py and
tests/linear_kernels.py), against float64. Tolerances are those of tests/test_gpu_gated.py."""
import pytest

from gated_kernels import BLOCKS, FORWARD, GRADIENTS
from linear_kernels import FORWARD as LINEAR
from test_gpu_gated import run_blocks, run_gated, run_gated_backward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kernel,m,n,k,dtype", FORWARD, ids=lambda v: str(v))
def test_forward(ctx, kernel, m, n, k, dtype):
    run_gated(ctx, m, n, k, dtype, "silu", pre=True)


@pytest.mark.parametrize("kernel,m,n,k,dtype", [c for c in FORWARD if c[1] * c[2] * c[3] < 3e8], ids=lambda v: str(v))
def test_forward_in_float32(ctx, kernel, m, n, k, dtype):
    run_gated(ctx, m, n, k, dtype, "gelu", "f32", bias=False, odd=1)


@pytest.mark.parametrize("kernel,m,n,k", GRADIENTS, ids=lambda v: str(v))
def test_gradients(ctx, kernel, m, n, k):
    run_gated_backward(ctx, m, n, k, "silu")


@pytest.mark.parametrize("kernel,m,n,k", [c[:4] for c in LINEAR if c[4] == "fp8" and c[0] != "any"], ids=lambda v: str(v))
def test_blocks(ctx, kernel, m, n, k):
    run_blocks(ctx, m, n, k, "silu", residual=True)
    run_blocks(ctx, m, n, k, "relu", bias=False, residual=True, in_place=True)


@pytest.mark.parametrize("m,n,k", BLOCKS)
def test_blocks_of_few_rows(ctx, m, n, k):
    run_blocks(ctx, m, n, k, "silu", residual=True, odd=1)
    run_blocks(ctx, m, n, k, "none", "f32")

"""GPU parity: every kernel of a gated layer's gradients asked for by themselves, at shapes that it takes (tests/gated_single_kernels.py), against float64.
Tolerances are those of tests/test_gpu_gated.py."""
import pytest

from gated_single_kernels import SINGLES
from test_gpu_gated import run_gated_backward

pytestmark = pytest.mark.gpu
OUTPUTS = {"dx": [("dx",)], "dw": [("dw_gate",), ("dw_up", "dbias_up")], "dws": [("dw_gate", "dw_up", "dbias_gate", "dbias_up")]}


@pytest.mark.parametrize("which,kernel,m,n,k", SINGLES, ids=lambda v: str(v))
def test_single_gradients(ctx, which, kernel, m, n, k):
    for i, outputs in enumerate(OUTPUTS[which]):
        run_gated_backward(ctx, m, n, k, "silu", odd=i, outputs=outputs)


@pytest.mark.parametrize("which,kernel,m,n,k", [c for c in SINGLES if c[2] * c[3] * c[4] < 1e9], ids=lambda v: str(v))
def test_single_gradients_of_rows_at_any_place(ctx, which, kernel, m, n, k):
    """Operands that are copied, and results one element into their buffers."""
    run_gated_backward(ctx, m, n, k, "gelu", odd=1, outputs=OUTPUTS[which][0])

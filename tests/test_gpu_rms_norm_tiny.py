"""GPU parity: the gradient of an RMS norm without eps over rows that are nearly zero."""
import numpy as np
import pytest

import ffn_reference as ref
from dotcompute_amd import hip
from test_gpu_rms_norm import F32, close, values, wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cols", [300, 4096, 40001])
def test_gradient_of_nearly_nothing(ctx, cols, dtype):
    """h of 3e-20: s is 3e19 and its square no float, the gradients are. The squares of h are among the smallest floats, each off
    by at most 2^-150, 8e-7 of their mean: s by half that and s^3 by 1.5 times, beside the usual 4e-6."""
    rng = np.random.default_rng(cols)
    rows = 5
    h, dy, w = values(rng, (rows, cols), dtype, 3e-20), values(rng, (rows, cols), dtype), values(rng, (cols,), dtype, 0.1, 1.0)
    on = [ctx.to_device(a) for a in (dy, h, w)]
    dx, dw = ctx.empty((rows, cols), h.dtype), ctx.empty(cols, np.float32)
    ctx.rms_norm_backward(hip.RmsNormGrad.of(*on, dx=dx, dweight=dw, eps=0.0))
    ctx.synchronize()
    hv, dv, wv = wide(h), wide(dy), wide(w)
    x64, w64 = ref.rms_norm_grad(dv, hv, wv, 0.0)
    s = 1.0 / np.sqrt(np.mean(hv * hv, axis=1, keepdims=True))
    g = np.abs(dv * wv)
    terms = s * (g + np.abs(hv) * s * np.mean(g * np.abs(hv) * s, axis=1, keepdims=True))
    close(dx.to_host(), x64, dtype, "dx", (F32 + 1.2e-6) * terms)
    assert np.all(np.abs(dw.to_host() - w64) <= 1e-5 * np.sum(np.abs(dv * hv * s), axis=0))
    for a in on + [dx, dw]:
        ctx.free(a)

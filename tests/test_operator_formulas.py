"""CPU: the float64 gradients of tests/ffn_reference.py against central differences of its forward formulas, its
element types against known codes, and the shapes the argument blocks of the binding accept."""
import ctypes as C
import subprocess

import numpy as np
import pytest

import ffn_reference as ref
from dotcompute_amd import hip

ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def difference(f, x, step=1e-6):
    """df/dx of a scalar function by central differences, element by element."""
    g = np.empty_like(x)
    for i in np.ndindex(x.shape):
        old = x[i]
        x[i] = old + step
        up = f()
        x[i] = old - step
        down = f()
        x[i] = old
        g[i] = (up - down) / (2 * step)
    return g


# Central differences of step d are off by d^2 times a third derivative (here of order 1) and by 2^-53 / d of the
# function's value (of order 10): 1e-12 and 1e-9, so 1e-7 holds with room.
TOL = 1e-7


def test_rms_norm_gradient_is_the_difference():
    rng = np.random.default_rng(1)
    h, w, dy, dh = rng.normal(size=(3, 7)), rng.normal(size=7), rng.normal(size=(3, 7)), rng.normal(size=(3, 7))
    dx, dw = ref.rms_norm_grad(dy, h, w, 1e-3, dh)

    def f():
        return np.sum(ref.rms_norm(h, w, 1e-3)[1] * dy) + np.sum(h * dh)

    assert np.max(np.abs(difference(f, h) - dx)) < TOL
    assert np.max(np.abs(difference(f, w) - dw)) < TOL


@pytest.mark.parametrize("name", ACTS)
def test_linear_gradient_is_the_difference(name):
    rng = np.random.default_rng(2)
    x, w, b, dy = rng.normal(size=(4, 5)), rng.normal(size=(3, 5)), rng.normal(size=3), rng.normal(size=(4, 3))
    z, _ = ref.linear(x, w, b, name)
    assert np.min(np.abs(z)) > 1e-4  # (away from relu's corner)
    dx, dw, db = ref.linear_grad(dy, x, w, z, name)

    def f():
        return np.sum(ref.linear(x, w, b, name)[1] * dy)

    assert np.max(np.abs(difference(f, x) - dx)) < TOL
    assert np.max(np.abs(difference(f, w) - dw)) < TOL
    assert np.max(np.abs(difference(f, b) - db)) < TOL


def test_fp8_values():
    v = ref.FP8_VALUES
    assert v[0x01] == 2.0 ** -9 and v[0x08] == 2.0 ** -6 and v[0x38] == 1.0 and v[0x7E] == 448.0 and v[0xB8] == -1.0
    assert np.isnan(v[0x7F]) and np.isnan(v[0xFF])
    keep = ~np.isnan(v)
    assert np.array_equal(ref.to_fp8(v[keep]), np.arange(256, dtype=np.uint8)[keep])
    assert list(ref.to_fp8([1.0625, 1.1875, 1e9, -1e9])) == [0x38, 0x3A, 0x7E, 0xFE]  # ties to even, and the ends


LAYOUTS = {
    "dc_rms_norm": (hip.RmsNorm, 112), "dc_rms_norm_grad": (hip.RmsNormGrad, 104), "dc_linear": (hip.Linear, 144),
    "dc_linear_grad": (hip.LinearGrad, 136), "dc_adamw": (hip.AdamW, 64), "dc_adamw_tensor": (hip.AdamWTensor, 72),
}


def test_argument_blocks_are_laid_out_as_the_header_says(tmp_path):
    """Every field of the binding's structures lies where a C compiler puts the header's."""
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "dotcompute_hip.h"', "int main(void) {"]
    for name, (mirror, _) in LAYOUTS.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        for f, _ in mirror._fields_:
            lines.append(f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));')
    (tmp_path / "probe.c").write_text("\n".join(lines + ["return 0; }"]))
    include = hip.HEADER.rsplit("/", 1)[0]
    subprocess.run(["gcc", "-std=c11", "-I", include, str(tmp_path / "probe.c"), "-o", str(tmp_path / "probe")], check=True)
    out = subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True, check=True).stdout
    got = dict(line.split() for line in out.splitlines())
    for name, (mirror, size) in LAYOUTS.items():
        assert int(got[name]) == C.sizeof(mirror) == size, name
        for f, _ in mirror._fields_:
            assert int(got[f"{name}.{f}"]) == getattr(mirror, f).offset, (name, f)


# ---- refusals: no device is needed, arguments are looked at first --------------------------------------
BAD, UNSUPPORTED, ALIGN, DIM = (hip.DC_ERR_INVALID_ARGUMENT, hip.DC_ERR_UNSUPPORTED, hip.DC_ERR_MISALIGNED,
                                hip.DC_ERR_DIMENSION)
P = 4096  # an address that nobody reads


def norm(**change):
    a = dict(rows=2, cols=8, dtype=hip.DTYPE_BF16, y_dtype=hip.DTYPE_BF16, eps=1e-6, x=P, weight=P, y=P, x_stride=8, y_stride=8)
    return hip.RmsNorm(**{**a, **change})


@pytest.mark.parametrize("change,status", [
    (dict(rows=-1), BAD), (dict(cols=-1), BAD), (dict(cols=1 << 30, x_stride=1 << 30, y_stride=1 << 30), UNSUPPORTED),
    (dict(dtype=hip.DTYPE_FP8), BAD), (dict(dtype=9), BAD), (dict(y_dtype=hip.DTYPE_F32), BAD), (dict(reserved=1), BAD),
    (dict(eps=-1.0), BAD), (dict(eps=float("nan")), BAD), (dict(x=None), BAD), (dict(weight=None), BAD), (dict(y=None), BAD),
    (dict(scales=P), BAD), (dict(y_dtype=hip.DTYPE_FP8), BAD), (dict(x_stride=7), DIM), (dict(y_stride=0), DIM),
    (dict(residual=P, residual_stride=7), DIM), (dict(sum=P, sum_stride=7), DIM), (dict(x=P + 1), ALIGN),
    (dict(weight=P + 1), ALIGN), (dict(dtype=hip.DTYPE_F32, y_dtype=hip.DTYPE_F32, x=P + 2), ALIGN),
    (dict(y_dtype=hip.DTYPE_FP8, scales=P + 2), ALIGN), (dict(), BAD)])  # (the last: no context)
def test_rms_norm_refusals(change, status):
    assert hip.load().dc_hip_rms_norm(None, norm(**change)) == status


def norm_grad(**change):
    a = dict(rows=2, cols=8, dtype=hip.DTYPE_F32, eps=1e-6, dy=P, h=P, weight=P, dx=P, dweight=P, dy_stride=8, h_stride=8,
             dx_stride=8)
    return hip.RmsNormGrad(**{**a, **change})


@pytest.mark.parametrize("change,status", [
    (dict(rows=-1), BAD), (dict(cols=1 << 30), UNSUPPORTED), (dict(dtype=hip.DTYPE_FP8), BAD), (dict(eps=-1.0), BAD),
    (dict(dy=None), BAD), (dict(h=None), BAD), (dict(weight=None), BAD), (dict(h_stride=7), DIM), (dict(dx_stride=7), DIM),
    (dict(dh=P, dh_stride=7), DIM), (dict(dweight=P + 2), ALIGN), (dict(dy=P + 2), ALIGN), (dict(), BAD)])
def test_rms_norm_backward_refusals(change, status):
    assert hip.load().dc_hip_rms_norm_backward(None, norm_grad(**change)) == status


def linear(**change):
    a = dict(m=2, n=8, k=8, dtype=hip.DTYPE_BF16, y_dtype=hip.DTYPE_BF16, x=P, w=P, y=P, x_stride=8, w_stride=8, y_stride=8)
    return hip.Linear(**{**a, **change})


@pytest.mark.parametrize("change,status", [
    (dict(m=-1), BAD), (dict(n=-1), BAD), (dict(k=-1), BAD), (dict(m=1 << 31), BAD), (dict(n=(1 << 23) + 1), UNSUPPORTED),
    (dict(k=(1 << 23) + 1), UNSUPPORTED), (dict(activation=5), BAD), (dict(activation=-1), BAD), (dict(dtype=hip.DTYPE_F32), BAD),
    (dict(y_dtype=hip.DTYPE_FP8), BAD), (dict(reserved=1), BAD), (dict(x_scales=P), BAD), (dict(dtype=hip.DTYPE_FP8), BAD),
    (dict(dtype=hip.DTYPE_FP8, x_scales=P), BAD), (dict(x=None), BAD), (dict(w=None), BAD), (dict(y=None), BAD),
    (dict(x_stride=7), DIM), (dict(w_stride=7), DIM), (dict(y_stride=7), DIM), (dict(residual=P, residual_stride=7), DIM),
    (dict(pre=P, pre_stride=7), DIM), (dict(x=P + 1), ALIGN), (dict(bias=P + 1), ALIGN),
    (dict(y_dtype=hip.DTYPE_F32, y=P + 2), ALIGN), (dict(dtype=hip.DTYPE_FP8, x_scales=P + 1, w_scales=P), ALIGN), (dict(), BAD)])
def test_linear_refusals(change, status):
    assert hip.load().dc_hip_linear(None, linear(**change)) == status


def linear_grad(**change):
    a = dict(m=2, n=8, k=8, activation=1, dy=P, x=P, w=P, pre=P, dx=P, dw=P, dbias=P, dy_stride=8, x_stride=8, w_stride=8,
             pre_stride=8, dx_stride=8, dw_stride=8)
    return hip.LinearGrad(**{**a, **change})


@pytest.mark.parametrize("change,status", [
    (dict(m=-1), BAD), (dict(m=(1 << 23) + 1), UNSUPPORTED), (dict(k=(1 << 23) + 1), UNSUPPORTED), (dict(activation=7), BAD),
    (dict(reserved=3), BAD), (dict(dy=None), BAD), (dict(pre=None), BAD), (dict(x=None), BAD), (dict(w=None), BAD),
    (dict(dy_stride=7), DIM), (dict(pre_stride=7), DIM), (dict(x_stride=7), DIM), (dict(w_stride=7), DIM), (dict(dx_stride=7), DIM),
    (dict(dw_stride=7), DIM), (dict(dbias=P + 2), ALIGN), (dict(dw=P + 1), ALIGN), (dict(), BAD)])
def test_linear_backward_refusals(change, status):
    assert hip.load().dc_hip_linear_backward(None, linear_grad(**change)) == status


def test_quantize_refusals():
    def f(x=P, dtype=0, xs=8, q=P, qs=8, s=P, rows=2, cols=8):
        return hip.load().dc_hip_quantize_fp8(None, x, dtype, xs, q, qs, s, rows, cols)

    assert f(rows=-1) == BAD and f(dtype=2) == BAD and f(x=None) == BAD and f(q=None) == BAD and f(s=None) == BAD
    assert f(xs=7) == DIM and f(qs=7) == DIM and f(x=P + 2) == ALIGN and f(s=P + 1) == ALIGN and f() == BAD
    assert f(cols=1 << 30) == UNSUPPORTED


def adamw(tensor=None, count=1, null=False, **change):
    a = hip.AdamW.of(lr=1e-3)
    for name, v in change.items():
        setattr(a, name, v)
    t = hip.AdamWTensor(**{**dict(param=P, grad=P, m=P, v=P, n=4), **(tensor or {})})
    return hip.load().dc_hip_adamw_step(None, a, None if null else t, count)


@pytest.mark.parametrize("status,change", [
    (BAD, dict(count=-1)), (BAD, dict(null=True)), (BAD, dict(state_dtype=1)), (BAD, dict(reserved=1)), (BAD, dict(step=0)),
    (BAD, dict(beta1=1.0)), (BAD, dict(beta1=-0.1)), (BAD, dict(beta2=1.0)), (BAD, dict(beta2=float("nan"))), (BAD, dict(eps=-1.0)),
    (BAD, dict(lr=float("inf"))), (BAD, dict(weight_decay=float("nan"))), (BAD, dict(grad_scale=float("inf"))),
    (BAD, dict(tensor=dict(n=-1))), (BAD, dict(tensor=dict(param=None))), (BAD, dict(tensor=dict(grad=None))),
    (BAD, dict(tensor=dict(m=None))), (BAD, dict(tensor=dict(v=None))), (BAD, dict(tensor=dict(grad_dtype=2))),
    (BAD, dict(tensor=dict(reserved=1))), (BAD, dict(tensor=dict(m_scales=P))), (BAD, dict(state_dtype=2)),
    (ALIGN, dict(tensor=dict(param=P + 2))), (ALIGN, dict(tensor=dict(grad=P + 2))), (ALIGN, dict(tensor=dict(m=P + 1))),
    (ALIGN, dict(tensor=dict(copy=P + 1))), (ALIGN, dict(tensor=dict(grad=P + 1, grad_dtype=1))), (BAD, dict())])
def test_adamw_refusals(status, change):
    assert adamw(**change) == status


def test_null_argument_blocks():
    L = hip.load()
    for f in (L.dc_hip_rms_norm, L.dc_hip_rms_norm_backward, L.dc_hip_linear, L.dc_hip_linear_backward):
        assert f(None, None) == BAD
    assert L.dc_hip_adamw_step(None, None, None, 0) == BAD


def array(shape, dtype):
    return hip.DeviceArray(None, P, int(np.prod(shape)) * np.dtype(dtype).itemsize, np.dtype(dtype), shape)


def test_the_binding_refuses_arrays_that_do_not_fit():
    b, f, q = np.uint16, np.float32, np.uint8
    x, w, y = array((2, 8), b), array((3, 8), b), array((2, 3), b)
    assert hip.Linear.of(x, w, y, activation="silu").x_stride == 8
    for bad in (dict(w=array((3, 9), b)), dict(y=array((3, 2), b)), dict(bias=array((2,), b)), dict(bias=array((3,), f)),
                dict(w=array((3, 8), q)), dict(residual=array((2, 8), b)), dict(z_stride=3), dict(x=array((8,), b))):
        with pytest.raises(ValueError):
            hip.Linear.of(**{**dict(x=x, w=w, y=y), **bad})
    with pytest.raises(KeyError):
        hip.Linear.of(x, w, y, activation="swish")
    with pytest.raises(ValueError):
        hip.RmsNorm.of(x, array((7,), b), x)
    with pytest.raises(ValueError):
        hip.RmsNormGrad.of(dy=x, h=x, weight=array((8,), b), dweight=array((8,), b))
    with pytest.raises(ValueError):
        hip.LinearGrad.of(dy=y, x=x, w=w, dbias=array((3,), b))
    part = dict(param=array((4,), f), grad=array((4,), b), m=array((4,), f), v=array((4,), f))
    assert hip.AdamWTensors.of([part]).items[0].grad_dtype == hip.DTYPE_BF16
    for bad in (dict(m=array((5,), f)), dict(m=array((4,), q)), dict(param=array((4,), b)), dict(grad=array((4,), q)),
                dict(copy=array((4,), f)), dict(other=array((4,), f))):
        with pytest.raises(ValueError):
            hip.AdamWTensors.of([{**part, **bad}])
    eight = dict(param=array((4,), f), grad=array((4,), b), m=array((4,), q), v=array((4,), q), m_scales=array((1,), f),
                 v_scales=array((1,), f))
    assert hip.AdamWTensors.of([eight]).state_dtype == hip.DTYPE_FP8
    with pytest.raises(ValueError):
        hip.AdamWTensors.of([part, eight])

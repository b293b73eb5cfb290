"""CPU: what the gated block's operators and the block scales' refuse, in the library (with no context: calls whose arguments are fine get as far as that)
and in the binding, since a kernel is handed addresses alone."""
import ctypes as C
import os
import subprocess

import pytest

from dotcompute_amd import hip
from test_operator_arguments import BF16, CODE, F32, context, rows

P = 4096  # an address that nobody reads
INVALID, UNSUPPORTED, MISALIGNED, DIMENSION = hip.DC_ERR_INVALID_ARGUMENT, hip.DC_ERR_UNSUPPORTED, hip.DC_ERR_MISALIGNED, hip.DC_ERR_DIMENSION


def status(name, cls, base, **change):
    return getattr(hip.load(), name)(None, cls(**{**base, **change}))


NORM = dict(rows=3, cols=300, dtype=hip.DTYPE_BF16, y_dtype=hip.DTYPE_BF16, eps=1e-5, x=P, weight=P, bias=P, y=P, x_stride=300, y_stride=300)
CODES = dict(y_dtype=hip.DTYPE_FP8, scales=P)


@pytest.mark.parametrize("change,want", [
    ({}, INVALID),  # (no context)
    (dict(rows=-1), INVALID), (dict(cols=-1), INVALID), (dict(cols=(1 << 25) + 1), UNSUPPORTED), (dict(dtype=hip.DTYPE_FP8), INVALID),
    (dict(y_dtype=hip.DTYPE_F32), INVALID), (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID), (dict(x=None), INVALID),
    (dict(weight=None), INVALID), (dict(y=None), INVALID), (dict(x=P + 1), MISALIGNED), (dict(bias=P + 1), MISALIGNED), (dict(x_stride=299), DIMENSION),
    (dict(y_stride=299), DIMENSION), (dict(residual=P, residual_stride=10), DIMENSION), (dict(sum=P, sum_stride=10), DIMENSION),
    (dict(scales=P), INVALID), (dict(scale_block=128), INVALID), (dict(y_dtype=hip.DTYPE_FP8), INVALID), (dict(**CODES, scale_block=64), INVALID),
    (dict(y_dtype=hip.DTYPE_FP8, scales=P + 2), MISALIGNED), (dict(**CODES, scale_block=128, scales_stride=2), DIMENSION),
])
def test_layer_norm_refuses(change, want):
    assert status("dc_hip_layer_norm", hip.LayerNorm, NORM, **change) == want


NORM_GRAD = dict(rows=3, cols=300, dtype=hip.DTYPE_F32, eps=1e-5, dy=P, h=P, weight=P, dx=P, dweight=P, dbias=P, dy_stride=300, h_stride=300,
                 dx_stride=300)


@pytest.mark.parametrize("change,want", [
    (dict(rows=-1), INVALID), (dict(cols=(1 << 25) + 1), UNSUPPORTED), (dict(dtype=hip.DTYPE_FP8), INVALID), (dict(eps=-1.0), INVALID),
    (dict(dy=None), INVALID), (dict(h=None), INVALID), (dict(weight=None), INVALID), (dict(dy=P + 2), MISALIGNED), (dict(dbias=P + 1), MISALIGNED),
    (dict(dweight=P + 2), MISALIGNED), (dict(dy_stride=299), DIMENSION), (dict(h_stride=0), DIMENSION), (dict(dx_stride=5), DIMENSION),
    (dict(dh=P, dh_stride=1), DIMENSION),
])
def test_layer_norm_backward_refuses(change, want):
    assert status("dc_hip_layer_norm_backward", hip.LayerNormGrad, NORM_GRAD, **change) == want


@pytest.mark.parametrize("change,want", [
    ({}, INVALID), (dict(rows=-1), INVALID), (dict(cols=(1 << 25) + 1), UNSUPPORTED), (dict(dtype=hip.DTYPE_FP8), INVALID), (dict(x=None), INVALID),
    (dict(q=None), INVALID), (dict(scales=None), INVALID), (dict(x=P + 1), MISALIGNED), (dict(x_stride=299), DIMENSION), (dict(q_stride=299), DIMENSION),
    (dict(scales_stride=2), DIMENSION),
])
def test_quantize_blocks_refuses(change, want):
    a = dict(x=P, dtype=hip.DTYPE_BF16, x_stride=300, q=P, q_stride=300, scales=P, scales_stride=3, rows=3, cols=300)
    a.update(change)
    assert hip.load().dc_hip_quantize_fp8_blocks(None, *a.values()) == want


BLOCKS = dict(m=3, n=5, k=300, y_dtype=hip.DTYPE_BF16, x=P, w=P, x_scales=P, w_scales=P, y=P, x_stride=300, w_stride=300, x_scales_stride=3,
              w_scales_stride=5, y_stride=5)


@pytest.mark.parametrize("change,want", [
    ({}, INVALID), (dict(m=-1), INVALID), (dict(m=1 << 30), INVALID), (dict(n=(1 << 23) + 1), UNSUPPORTED), (dict(k=(1 << 23) + 1), UNSUPPORTED),
    (dict(activation=5), INVALID), (dict(y_dtype=hip.DTYPE_FP8), INVALID), (dict(x=None), INVALID), (dict(w=None), INVALID), (dict(x_scales=None), INVALID),
    (dict(w_scales=None), INVALID), (dict(y=None), INVALID), (dict(y=P + 1), MISALIGNED), (dict(bias=P + 1), MISALIGNED), (dict(x_stride=299), DIMENSION),
    (dict(w_stride=299), DIMENSION), (dict(x_scales_stride=2), DIMENSION), (dict(w_scales_stride=4), DIMENSION), (dict(y_stride=4), DIMENSION),
    (dict(residual=P, residual_stride=4), DIMENSION),
])
def test_linear_blocks_refuses(change, want):
    assert status("dc_hip_linear_blocks", hip.LinearBlocks, BLOCKS, **change) == want


GATED = dict(m=3, n=5, k=300, dtype=hip.DTYPE_BF16, y_dtype=hip.DTYPE_BF16, activation=4, x=P, w_gate=P, w_up=P, y=P, x_stride=300, w_gate_stride=300,
             w_up_stride=300, y_stride=5)
ROWS = dict(dtype=hip.DTYPE_FP8, x_scales=P, gate_scales=P, up_scales=P)
BY_BLOCKS = dict(**ROWS, scale_block=128, x_scales_stride=3, gate_scales_stride=5, up_scales_stride=5)


@pytest.mark.parametrize("change,want", [
    ({}, INVALID), (dict(m=-1), INVALID), (dict(n=(1 << 22) + 1), UNSUPPORTED), (dict(k=(1 << 23) + 1), UNSUPPORTED), (dict(activation=-1), INVALID),
    (dict(dtype=hip.DTYPE_F32), INVALID), (dict(y_dtype=hip.DTYPE_FP8), INVALID), (dict(x=None), INVALID), (dict(w_gate=None), INVALID),
    (dict(w_up=None), INVALID), (dict(y=None), INVALID), (dict(x=P + 1), MISALIGNED), (dict(bias_up=P + 1), MISALIGNED), (dict(pre_up=P + 1), MISALIGNED),
    (dict(x_stride=299), DIMENSION), (dict(w_up_stride=299), DIMENSION), (dict(pre_gate=P, pre_gate_stride=4), DIMENSION), (dict(y_stride=4), DIMENSION),
    (dict(x_scales=P), INVALID), (dict(scale_block=128), INVALID), (dict(dtype=hip.DTYPE_FP8), INVALID), ({**ROWS, "up_scales": None}, INVALID),
    ({**ROWS, "scale_block": 32}, INVALID), ({**ROWS, "gate_scales": P + 2}, MISALIGNED), ({**BY_BLOCKS, "up_scales": None}, INVALID),
    ({**BY_BLOCKS, "up_scales_stride": 4}, DIMENSION), ({**BY_BLOCKS, "x_scales_stride": 2}, DIMENSION),
])
def test_gated_linear_refuses(change, want):
    assert status("dc_hip_gated_linear", hip.GatedLinear, GATED, **change) == want


GATED_GRAD = dict(m=3, n=5, k=300, activation=4, dy=P, x=P, w_gate=P, w_up=P, pre_gate=P, pre_up=P, dx=P, dw_gate=P, dw_up=P, dbias_gate=P, dbias_up=P,
                  dy_stride=5, x_stride=300, w_gate_stride=300, w_up_stride=300, pre_gate_stride=5, pre_up_stride=5, dx_stride=300,
                  dw_gate_stride=300, dw_up_stride=300)


@pytest.mark.parametrize("change,want", [
    ({}, INVALID), (dict(m=-1), INVALID), (dict(n=(1 << 22) + 1), UNSUPPORTED), (dict(k=(1 << 23) + 1), UNSUPPORTED), (dict(reserved=1), INVALID),
    (dict(m=(1 << 23) + 1), UNSUPPORTED), (dict(m=(1 << 23) + 1, dw_gate=None), UNSUPPORTED), (dict(activation=5), INVALID), (dict(dy=None), INVALID),
    (dict(pre_gate=None), INVALID), (dict(pre_up=None), INVALID), (dict(x=None), INVALID), (dict(w_gate=None), INVALID), (dict(w_up=None), INVALID),
    (dict(dy=P + 1), MISALIGNED), (dict(dbias_gate=P + 2), MISALIGNED), (dict(dx=P + 1), MISALIGNED), (dict(dy_stride=4), DIMENSION),
    (dict(pre_up_stride=4), DIMENSION), (dict(w_up_stride=1), DIMENSION), (dict(dw_gate_stride=299), DIMENSION), (dict(dx_stride=299), DIMENSION),
])
def test_gated_linear_backward_refuses(change, want):
    assert status("dc_hip_gated_linear_backward", hip.GatedLinearGrad, GATED_GRAD, **change) == want


def test_operands_that_nothing_asked_for_may_be_left_out():
    """(They get as far as the missing context, which is INVALID too: what is looked at before it would say something else.)"""
    only_bias = dict(dx=None, dw_gate=None, dw_up=None, x_stride=0, w_gate_stride=0, w_up_stride=0, m=(1 << 23) + 1)
    assert status("dc_hip_gated_linear_backward", hip.GatedLinearGrad, GATED_GRAD, **only_bias) == INVALID
    assert status("dc_hip_layer_norm", hip.LayerNorm, NORM, bias=None) == INVALID


def test_the_binding_looks_at_shapes_types_and_strides():
    ctx = context(1 << 16, 1 << 16)

    def m(shape, dtype=BF16, at=0):
        return rows(ctx, 1, at, shape, dtype)

    x, w, y = m((3, 300)), m((300,)), m((3, 300), CODE)
    assert hip.LayerNorm.of(x, w, None, y, scales=m((3, 3), CODE)).scale_block == 128
    assert hip.LayerNorm.of(x, w, w, y, scales=m((3,), F32)).scale_block == 0
    for bad in (dict(scales=m((2, 3), CODE)), dict(scales=m((3, 3), F32)), dict(scales=m((3,), CODE)), dict(residual=m((3, 299))),
                dict(scales=m((3, 3), CODE), scales_stride=1 << 16), dict(scales=m((3,), F32), scales_stride=3)):
        with pytest.raises(ValueError):
            hip.LayerNorm.of(x, w, None, y, **bad)
    with pytest.raises(ValueError, match="bias"):
        hip.LayerNorm.of(x, w, m((300,), F32), x)
    with pytest.raises(ValueError, match="dbias"):
        hip.LayerNormGrad.of(x, x, w, dbias=m((300,)))
    q, s = m((5, 300), CODE), m((3, 5), CODE)
    assert hip.LinearBlocks.of(y, q, m((3, 3), CODE), s, m((3, 5))).w_scales_stride == 5
    for bad in ((y, q, m((3, 3), CODE), m((5, 3), CODE), m((3, 5))), (y, x, m((3, 3), CODE), s, m((3, 5))), (x, q, m((3, 3), CODE), s, m((3, 5)))):
        with pytest.raises(ValueError):
            hip.LinearBlocks.of(*bad)
    wg, out = m((5, 300)), m((3, 5))
    assert hip.GatedLinear.of(x, wg, wg, out).scale_block == 0
    codes = dict(x_scales=m((3, 3), CODE), gate_scales=s, up_scales=s)
    assert hip.GatedLinear.of(y, q, q, out, **codes).scale_block == 128
    for bad in (dict(bias_gate=m((4,))), dict(pre_up=m((3, 4))), dict(w_up_stride=1 << 16)):
        with pytest.raises(ValueError):
            hip.GatedLinear.of(x, wg, wg, out, **bad)
    with pytest.raises(ValueError, match="up_scales"):
        hip.GatedLinear.of(y, q, q, out, **{**codes, "up_scales": m((5,), F32)})
    with pytest.raises(ValueError, match="w_up"):
        hip.GatedLinear.of(x, wg, m((4, 300)), out)
    with pytest.raises(ValueError, match="dbias_up"):
        hip.GatedLinearGrad.of(out, x, wg, wg, out, out, dbias_up=m((5,)))
    with pytest.raises(ValueError, match="pre_gate"):
        hip.GatedLinearGrad.of(out, x, wg, wg, m((3, 4)), out)
    for bad in (dict(scales_stride=1 << 16), dict(x_stride=1 << 16)):
        with pytest.raises(ValueError, match="stride"):
            hip.Context.quantize_fp8_blocks(ctx, x, y, m((3, 3), CODE), **bad)
    with pytest.raises(ValueError, match="scales"):
        hip.Context.quantize_fp8_blocks(ctx, x, y, m((2, 3), CODE))


def test_struct_sizes_match_the_header(tmp_path):
    """The binding's structures have the header's layout: every field's place."""
    names = {"dc_layer_norm": hip.LayerNorm, "dc_layer_norm_grad": hip.LayerNormGrad, "dc_linear_blocks": hip.LinearBlocks,
             "dc_gated_linear": hip.GatedLinear, "dc_gated_linear_grad": hip.GatedLinearGrad}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "dotcompute_hip.h"', "int main(void) {"]
    for struct, cls in names.items():
        lines.append(f'printf("%zu\\n", sizeof({struct}));')
        lines += [f'printf("%zu\\n", offsetof({struct}, {f[0]}));' for f in cls._fields_]
    (tmp_path / "probe.c").write_text("\n".join(lines + ["return 0; }"]))
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(root, "include"), str(tmp_path / "probe.c"), "-o", str(tmp_path / "probe")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for cls in names.values():
        want += [C.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_]
    assert got == want

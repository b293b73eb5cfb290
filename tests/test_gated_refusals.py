"""CPU: that what the gated block's operators refuse as invalid is looked at, each check by itself. With no context a call whose arguments are fine is
refused as invalid too, so each of these calls has a second fault, which is looked at later and has a code of its own: without the check that a case is
for, that code would come back. (The cases whose codes are others are in tests/test_gated_arguments.py.)"""
import pytest

from dotcompute_amd import hip
from test_gated_arguments import BLOCKS, BY_BLOCKS, CODES, GATED, GATED_GRAD, NORM, NORM_GRAD, P, ROWS, status

INVALID, UNSUPPORTED, MISALIGNED, DIMENSION = hip.DC_ERR_INVALID_ARGUMENT, hip.DC_ERR_UNSUPPORTED, hip.DC_ERR_MISALIGNED, hip.DC_ERR_DIMENSION

# The second faults, and the codes that they have by themselves.
SUM = dict(sum=P, sum_stride=10), DIMENSION
TOO_WIDE = dict(cols=(1 << 25) + 1), UNSUPPORTED
PARTS = dict(dbias=P + 1), MISALIGNED
SHORT_SCALES = dict(scales_stride=2), DIMENSION
WIDE_N = dict(n=(1 << 23) + 1), UNSUPPORTED
SHORT_RESIDUAL = dict(residual=P, residual_stride=4), DIMENSION
SHORT_Y = dict(y_stride=4), DIMENSION
SHORT_PRE = dict(pre_up=P, pre_up_stride=4), DIMENSION
SUMS = dict(dbias_up=P + 2), MISALIGNED


def check(call, base, faults, second):
    """The faults beside the second one are INVALID; the second one alone says that it is looked at, and what without the check would come back."""
    change, code = second
    assert call({**base, **change}) == code
    assert call({**base, **change, **faults}) == INVALID


def calls(name, cls):
    return lambda arguments: status(name, cls, arguments)


@pytest.mark.parametrize("faults,second", [
    (dict(rows=-1), TOO_WIDE), (dict(rows=-7, dtype=hip.DTYPE_F32, y_dtype=hip.DTYPE_F32), TOO_WIDE),
    (dict(dtype=hip.DTYPE_FP8, y_dtype=hip.DTYPE_FP8, scales=P), SUM), (dict(dtype=9, y_dtype=9), SUM), (dict(y_dtype=hip.DTYPE_F32), SUM),
    (dict(y_dtype=7), SUM), (dict(scale_block=128), SUM), (dict(**CODES, scale_block=64), SUM), (dict(**CODES, scale_block=-128), SUM),
    (dict(eps=-1.0), SUM), (dict(eps=float("nan")), SUM), (dict(scales=P), SUM), (dict(y_dtype=hip.DTYPE_FP8), SUM),
    (dict(y_dtype=hip.DTYPE_FP8, scale_block=128), SUM), (dict(x=None), SUM), (dict(weight=None), SUM), (dict(y=None), SUM),
])
def test_layer_norm(faults, second):
    check(calls("dc_hip_layer_norm", hip.LayerNorm), NORM, faults, second)


@pytest.mark.parametrize("faults", [dict(cols=-1), dict(cols=-1, rows=0)])
def test_layer_norm_of_fewer_than_no_columns(faults):
    """(Next to what is looked at with no columns as well: the alignment of a row's scale.)"""
    check(calls("dc_hip_layer_norm", hip.LayerNorm), {**NORM, "y_dtype": hip.DTYPE_FP8}, faults, (dict(scales=P + 2), MISALIGNED))


@pytest.mark.parametrize("faults", [
    dict(rows=-1), dict(cols=-1), dict(dtype=hip.DTYPE_FP8), dict(dtype=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(dy=None), dict(h=None),
    dict(weight=None),
])
def test_layer_norm_backward(faults):
    check(calls("dc_hip_layer_norm_backward", hip.LayerNormGrad), NORM_GRAD, faults, PARTS)


@pytest.mark.parametrize("faults,second", [
    (dict(rows=-1), TOO_WIDE), (dict(dtype=hip.DTYPE_FP8), SHORT_SCALES), (dict(dtype=3), SHORT_SCALES), (dict(x=None), SHORT_SCALES),
    (dict(q=None), SHORT_SCALES), (dict(scales=None), SHORT_SCALES),
])
def test_quantize_blocks(faults, second):
    base = dict(x=P, dtype=hip.DTYPE_BF16, x_stride=300, q=P, q_stride=300, scales=P, scales_stride=3, rows=3, cols=300)
    check(lambda arguments: hip.load().dc_hip_quantize_fp8_blocks(None, *arguments.values()), base, faults, second)


@pytest.mark.parametrize("faults,second", [
    (dict(m=-1), WIDE_N), (dict(m=1 << 30), WIDE_N), (dict(k=-1), WIDE_N), (dict(activation=5), WIDE_N), (dict(activation=-1), WIDE_N),
    (dict(n=-1), (dict(k=(1 << 23) + 1), UNSUPPORTED)), (dict(y_dtype=hip.DTYPE_FP8), SHORT_RESIDUAL), (dict(y_dtype=-1), SHORT_RESIDUAL),
    (dict(x=None), SHORT_RESIDUAL), (dict(w=None), SHORT_RESIDUAL), (dict(x_scales=None), SHORT_RESIDUAL), (dict(w_scales=None), SHORT_RESIDUAL),
    (dict(y=None), SHORT_RESIDUAL),
])
def test_linear_blocks(faults, second):
    check(calls("dc_hip_linear_blocks", hip.LinearBlocks), BLOCKS, faults, second)


@pytest.mark.parametrize("faults,second", [
    (dict(m=-1), WIDE_N), (dict(m=1 << 30), WIDE_N), (dict(k=-1), WIDE_N), (dict(activation=-1), WIDE_N), (dict(activation=5), WIDE_N),
    (dict(n=-1), (dict(k=(1 << 23) + 1), UNSUPPORTED)), (dict(dtype=hip.DTYPE_F32), SHORT_Y), (dict(dtype=5), SHORT_Y),
    (dict(y_dtype=hip.DTYPE_FP8), SHORT_Y), (dict(y_dtype=-1), SHORT_Y), (dict(x=None), SHORT_Y), (dict(w_gate=None), SHORT_Y), (dict(w_up=None), SHORT_Y),
    (dict(y=None), SHORT_PRE), (dict(x_scales=P), SHORT_Y), (dict(gate_scales=P), SHORT_Y), (dict(up_scales=P), SHORT_Y), (dict(scale_block=128), SHORT_Y),
    (dict(dtype=hip.DTYPE_FP8), SHORT_Y), ({**ROWS, "x_scales": None}, SHORT_Y), ({**ROWS, "gate_scales": None}, SHORT_Y),
    ({**ROWS, "up_scales": None}, SHORT_Y), ({**ROWS, "scale_block": 32}, SHORT_Y), ({**BY_BLOCKS, "x_scales": None}, SHORT_Y),
    ({**BY_BLOCKS, "gate_scales": None}, SHORT_Y), ({**BY_BLOCKS, "up_scales": None}, SHORT_Y), ({**ROWS, "x_scales": None, "k": 0}, SHORT_Y),
])
def test_gated_linear(faults, second):
    check(calls("dc_hip_gated_linear", hip.GatedLinear), GATED, faults, second)


@pytest.mark.parametrize("faults,second", [
    (dict(m=-1), SUMS), (dict(m=1 << 30), SUMS), (dict(n=-1), SUMS), (dict(k=-1), SUMS), (dict(activation=5), SUMS), (dict(activation=-1), SUMS),
    (dict(reserved=1), SUMS), (dict(dy=None), SUMS), (dict(pre_gate=None), SUMS), (dict(pre_up=None), SUMS), (dict(x=None), SUMS), (dict(w_gate=None), SUMS),
    (dict(w_up=None), SUMS), (dict(x=None, dw_gate=None), SUMS), (dict(x=None, dw_up=None), SUMS),
])
def test_gated_linear_backward(faults, second):
    check(calls("dc_hip_gated_linear_backward", hip.GatedLinearGrad), GATED_GRAD, faults, second)


@pytest.mark.parametrize("change", [
    dict(dx=None, dw_gate=None, dw_up=None, x=None, w_gate=None, w_up=None), dict(dx=None, w_gate=None, w_up=None), dict(dw_gate=None, dw_up=None, x=None),
])
def test_operands_that_nothing_asked_for_are_not_looked_at(change):
    """(What is looked at past them says so.)"""
    assert status("dc_hip_gated_linear_backward", hip.GatedLinearGrad, GATED_GRAD, **change, dbias_up=P + 2) == MISALIGNED

"""CPU: the float64 gradients of tests/gated_reference.py against central differences of its forward formulas, its block scales against their definition, and
what the cases of perf/more_operators.py compute against it."""
import importlib.util
import os
import random

import numpy as np
import pytest

import ffn_reference as ref
import gated_reference as gated
from test_operator_formulas import ACTS, TOL, difference

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_layer_norm_gradients_are_the_differences():
    rng = np.random.default_rng(1)
    h, w, b, dy, dh = (rng.normal(size=s) for s in ((3, 7), 7, 7, (3, 7), (3, 7)))

    def f():
        return np.sum(gated.layer_norm(h, w, b, 1e-3)[1] * dy) + np.sum(h * dh)

    for got, x in zip(gated.layer_norm_grad(dy, h, w, 1e-3, dh), (h, w, b)):
        assert np.allclose(got, difference(f, x), atol=TOL, rtol=TOL)


@pytest.mark.parametrize("activation", ACTS)
def test_gated_gradients_are_the_differences(activation):
    rng = np.random.default_rng(2)
    x, wg, wu, bg, bu, dy = (rng.normal(size=s) for s in ((3, 4), (5, 4), (5, 4), 5, 5, (3, 5)))

    def f():
        return np.sum(gated.gated(x, wg, wu, bg, bu, activation)[2] * dy)

    g, u, _ = gated.gated(x, wg, wu, bg, bu, activation)
    for got, at in zip(gated.gated_grad(dy, x, wg, wu, g, u, activation), (x, wg, wu, bg, bu)):
        assert np.allclose(got, difference(f, at), atol=TOL, rtol=TOL)


def test_block_scales_are_the_least_powers_of_two():
    top = np.concatenate([448.0 * 2.0 ** np.arange(-140, 100), np.nextafter(np.float32(448.0), np.float32(1e9)) * 2.0 ** np.arange(-100, 100),
                          np.abs(np.random.default_rng(3).normal(size=1000)), [0.0, 1e-45, 3.4e38]])
    s = gated.scale_of(top)
    value = gated.scale_value(s)
    assert np.all(top <= 448.0 * value) and np.all((s == 0) | (top > 224.0 * value))
    assert list(gated.scale_of(np.array([np.inf, np.nan]))) == [255, 255]
    q, scales = gated.rows_fp8(np.array([[0.0] * 200 + [-448.0, 3.0] + [1.0] * 100]))
    assert scales.shape == (3, 1) and list(scales[:, 0]) == [0, 127, 119] and np.array_equal(gated.values(q, scales)[0, 200:202], [-448.0, 3.0])


@pytest.fixture(scope="module")
def cases():
    torch = pytest.importorskip("torch")
    spec = importlib.util.spec_from_file_location("more_operators", os.path.join(ROOT, "perf", "more_operators.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.DEV = "cpu"
    return module, torch


def test_the_plain_forms_and_the_exact_ones_agree(cases):
    """Relative in the 2-norm: a rounding to bf16 is within 2^-8, to e4m3 2^-4; float32 sums of a few hundred terms within 1e-5."""
    module, torch = cases
    rng = random.Random(5)
    kinds = set()
    for _ in range(40):
        case = module.draw(rng)
        kinds.add(case["kind"])
        for name in ("rows", "cols", "m", "n", "k"):
            if name in case:
                case[name] = min(case[name], 20 + case[name] % 300)
        state = module.State(case, module._inputs(case, 7))
        if case["kind"] == "layer_norm":
            state.t["y"] = None
        got, want = module._plain(state), module.exact(case, 7)
        assert set(got) == set(want)
        for name, v in got.items():
            if want[name] is None:
                continue
            bound = {torch.bfloat16: ref.BF16, torch.float8_e4m3fn: ref.FP8}.get(v.dtype, 1e-5)
            off = torch.linalg.vector_norm(v.float().double() - want[name]) / torch.linalg.vector_norm(want[name])
            assert off <= bound, (case, name)
    assert len(kinds) == 6


def test_the_cases_block_scales_are_the_reference_s(cases):
    module, torch = cases
    x = np.random.default_rng(6).normal(size=(5, 300)).astype(np.float32)
    x[2] *= 1e-37
    x[3, 128:256] = 0.0
    q, scales = module._blocks_fp8(torch.from_numpy(x))
    want, ws = gated.rows_fp8(x)
    assert np.array_equal(scales.numpy(), ws) and np.array_equal(q.view(torch.uint8).numpy(), want)

"""The example's gated form: a step's errors and gradients against float64, what it serves in bf16 and in 8 bits, its operators run together on two
contexts.

Tolerances, relative in the 2-norm: every value that is kept in bf16 is off by at most 2^-8 of itself. The error adds up those of n1 (which both factors of a
carry), a, branch, s, n2 and its own rounding, 7 at most; a gradient adds the ones of the backward chain (e, dn2, ds, da, dz, dn1, its own) and of the
saved values, 16 at most; no operand here is amplified by more than 2: 2 * 7 * 2^-8 of the results before the target is taken off, and 2 * 16 * 2^-8
of a gradient. In 8 bits each operand of a product is within 2^-4 of its values, n1 counting twice: 9 * 2^-4.
"""
import numpy as np
import pytest

import ffn_reference as ref
import gated_reference as gated
from dotcompute_amd import hip
from dotcompute_amd.examples import feed_forward as ff
from test_gpu_feed_forward import apart, wide

pytestmark = pytest.mark.gpu


def block64(p, x):
    _, n1 = gated.layer_norm(x, p["norm1"], p["shift1"], 1e-5)
    g, u, a = gated.gated(n1, p["wg"], p["wu"], p["bg"], p["bu"], "silu")
    s = x + a @ p["w2"].T + p["b2"]
    _, n2 = gated.layer_norm(s, p["norm2"], p["shift2"], 1e-5)
    return n1, g, u, a, s, n2, n2 @ p["head"].T


def parameters(model):
    return {name: wide(c.to_host()) for name, c in model.copy.items()}


@pytest.mark.parametrize("rows,width,hidden,outputs", [(1, 32, 48, 16), (100, 96, 160, 40), (257, 130, 66, 34)])
def test_step_matches_float64(ctx, rows, width, hidden, outputs):
    model = ff.Model(ctx, width, hidden, outputs, gated=True)
    x, target = ff.data(rows, width, outputs)
    p = parameters(model)
    trainer = ff.Trainer(model, x, target)
    for call, args in trainer.forward + trainer.backward:
        call(args)
    x64 = wide(x)
    n1, g, u, a, s, n2, y = block64(p, x64)
    error = wide(trainer.error.to_host())
    assert apart(error, y - wide(target), y) <= 2 * 7 / 256
    e = error  # the gradients of the error that the device saw
    grad = {"head": e.T @ n2}
    ds, grad["norm2"], grad["shift2"] = gated.layer_norm_grad(e @ p["head"], s, p["norm2"], 1e-5)
    da, grad["w2"], grad["b2"] = ds @ p["w2"], ds.T @ a, ds.sum(axis=0)
    dn1, grad["wg"], grad["wu"], grad["bg"], grad["bu"] = gated.gated_grad(da, n1, p["wg"], p["wu"], g, u, "silu")
    _, grad["norm1"], grad["shift1"] = gated.layer_norm_grad(dn1, x64, p["norm1"], 1e-5)
    for name, want in grad.items():
        got = model.grad[name].to_host()
        got = wide(got) if got.dtype == np.uint16 else got
        assert apart(got, want) <= 2 * 16 / 256, name
    before = {name: c.to_host() for name, c in model.copy.items()}
    model.step(1e-2, rows)
    for name, c in model.copy.items():
        assert np.any(c.to_host() != before[name]), name


@pytest.mark.parametrize("rows", [1, 3, 32, 200])
def test_serving(ctx, rows):
    model = ff.Model(ctx, 200, 264, 32, gated=True)
    x, _ = ff.data(rows, 200, 32)
    y = block64(parameters(model), wide(x))[-1]
    assert apart(ff.Server(model, rows, fp8=False)(x), y) <= 2 * 7 / 256
    assert apart(ff.Server(model, rows)(x), y) <= 9 / 16


def test_steps_on_two_contexts_at_once(ctx):
    """Every context has a stream and workspaces of its own: steps enqueued by turns on two of them give the bits of steps on one."""
    x, target = ff.data(300, 72, 24)
    with hip.Context(0) as other:
        def model_on(c):
            m = ff.Model(c, 72, 144, 24, gated=True)
            return m, ff.Trainer(m, x, target)

        def state(m, t):
            return [a.to_host() for a in m.copy.values()] + [t.error.to_host()]

        alone = model_on(ctx)
        for _ in range(5):
            alone[1].run(1e-2)
        pair = model_on(ctx), model_on(other)
        for _ in range(5):
            for _, trainer in pair:
                trainer.run(1e-2)
        for m, t in pair:
            for one, two in zip(state(*alone), state(m, t)):
                assert np.array_equal(one, two)
        del pair, alone

"""The example that trains a feed-forward block and serves it: one step against float64, a loss that falls, 8 bits beside bf16.

Tolerances, relative in the 2-norm: every value that is kept in bf16 is off by at most 2^-8 of itself. The error adds up those
of n1, a, branch, s, n2 and its own rounding, 6 at most; a gradient adds the ones of the backward chain (e, dn2, ds, da, dz, dn1,
its own) and of the saved values, 14 at most; they enter a product as they are, no operand here being amplified by more than
2: 2 * 6 * 2^-8 of the results before the target is taken off, and 2 * 14 * 2^-8 of a gradient. In 8 bits three products' two operands each are within
2^-4 of their values: 6 * 2^-4.
"""
import numpy as np
import pytest

import ffn_reference as ref
from dotcompute_amd import hip
from dotcompute_amd.examples import feed_forward as ff

pytestmark = pytest.mark.gpu


def wide(b):
    return ref.from_bf16(b).astype(np.float64)


def apart(got, want, scale=None):
    return np.linalg.norm(got - want) / np.linalg.norm(want if scale is None else scale)


def block64(p, x):
    _, n1 = ref.rms_norm(x, p["norm1"], 1e-6)
    z, a = ref.linear(n1, p["w1"], p["b1"], "silu")
    s = x + a @ p["w2"].T + p["b2"]
    _, n2 = ref.rms_norm(s, p["norm2"], 1e-6)
    return n1, z, a, s, n2, n2 @ p["head"].T


@pytest.mark.parametrize("rows,width,hidden,outputs", [(1, 32, 48, 16), (100, 96, 160, 40), (257, 130, 66, 34)])
def test_step_matches_float64(ctx, rows, width, hidden, outputs):
    model = ff.Model(ctx, width, hidden, outputs)
    x, target = ff.data(rows, width, outputs)
    p = {name: wide(c.to_host()) for name, c in model.copy.items()}
    trainer = ff.Trainer(model, x, target)
    for call, args in trainer.forward + trainer.backward:
        call(args)
    x64 = wide(x)
    n1, z, a, s, n2, y = block64(p, x64)
    e = y - wide(target)
    error = wide(trainer.error.to_host())
    assert apart(error, e, y) <= 2 * 6 / 256
    e = error  # the gradients of the error that the device saw
    g = {"head": e.T @ n2}
    ds, g["norm2"] = ref.rms_norm_grad(e @ p["head"], s, p["norm2"], 1e-6)
    da, g["w2"], g["b2"] = ds @ p["w2"], ds.T @ a, ds.sum(axis=0)
    dz = da * ref.act_slope("silu", z)
    dn1, g["w1"], g["b1"] = dz @ p["w1"], dz.T @ n1, dz.sum(axis=0)
    _, g["norm1"] = ref.rms_norm_grad(dn1, x64, p["norm1"], 1e-6)
    for name, want in g.items():
        got = model.grad[name].to_host()
        got = wide(got) if got.dtype == np.uint16 else got
        assert apart(got, want) <= 2 * 14 / 256, name
    before = {name: c.to_host() for name, c in model.copy.items()}
    model.step(1e-2, rows)
    for name, c in model.copy.items():
        assert np.any(c.to_host() != before[name]), name


def test_training_and_serving(ctx):
    model = ff.Model(ctx, 64, 256, 32)
    x, target = ff.data(512, 64, 32)
    trainer = ff.Trainer(model, x, target)
    trainer.run(3e-3)
    first = trainer.loss()
    for _ in range(200):
        trainer.run(3e-3)
    assert trainer.loss() < first / 10
    for rows in (1, 3, 32):
        wide_rows, coded = ff.Server(model, rows, fp8=False)(x[:rows]), ff.Server(model, rows)(x[:rows])
        p = {name: wide(c.to_host()) for name, c in model.copy.items()}
        y = block64(p, wide(x[:rows]))[-1]
        assert apart(wide_rows, y) <= 2 * 6 / 256
        assert apart(coded, y) <= 6 / 16


def test_a_step_on_another_context(ctx):
    """Every context has a stream and workspaces of its own: the same steps on a second one give the same bits."""
    x, target = ff.data(300, 72, 24)
    results = []
    with hip.Context(0) as other:
        for c in (ctx, other):
            model = ff.Model(c, 72, 144, 24)
            trainer = ff.Trainer(model, x, target)
            for _ in range(5):
                trainer.run(1e-2)
            results.append([a.to_host() for a in model.copy.values()] + [trainer.error.to_host()])
        for one, two in zip(*results):
            assert np.array_equal(one, two)
        del model, trainer

"""GPU parity: the AdamW step over many tensors, states in 32 bits and in 8, against float64.

Tolerances, from the arithmetic: m, v and param are each a few float32 operations on values of the step: 6 half-ulps
(4e-7) of the magnitudes added. In 8 bits a state is read back within half a step of what it is (4 bits, or the smallest
value of its block), and those above zero are never held as zero.
"""
import numpy as np
import pytest

import ffn_reference as ref
from dotcompute_amd import hip

pytestmark = pytest.mark.gpu
F32 = 4e-7
HYPER = dict(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1)


def tensor(rng, n, grad="f32", eight=False, copy=True, first=False):
    """(host arrays, float64 m and v): one tensor of a step, its arrays as the kernels take them."""
    p = rng.normal(size=n).astype(np.float32) * np.float32(0.02)
    g = rng.normal(size=n).astype(np.float32) * np.float32(1e-2)
    m = np.zeros(n, np.float32) if first else rng.normal(size=n).astype(np.float32) * np.float32(1e-3)
    root = np.zeros(n, np.float32) if first else np.abs(rng.normal(size=n).astype(np.float32) * np.float32(1e-2))
    h = dict(param=p, grad=ref.to_bf16(g) if grad == "bf16" else g)
    if eight:
        (h["m"], h["m_scales"]), (h["v"], h["v_scales"]) = blocks(m), blocks(root)
    else:
        h["m"], h["v"] = m, root * root
    if copy:
        h["copy"] = np.full(n, 0x7777, np.uint16)
    return h


def blocks(x):
    b = np.zeros((-(-x.size // ref.BLOCK), ref.BLOCK), np.float32)
    b.reshape(-1)[:x.size] = x
    q, s = ref.rows_fp8(b)
    return q.reshape(-1)[:x.size].copy(), s


def unblock(q, s):
    return ref.from_fp8(q).astype(np.float64) * np.repeat(s.astype(np.float64), ref.BLOCK)[:q.size]


def wide(h, eight):
    g = ref.from_bf16(h["grad"]) if h["grad"].dtype == np.uint16 else h["grad"]
    m, v = (unblock(h["m"], h["m_scales"]), unblock(h["v"], h["v_scales"]) ** 2) if eight else (h["m"], h["v"])
    return [np.asarray(a, np.float64) for a in (h["param"], g, m, v)]


def step(ctx, hosts, shift=0, **hyper):
    """One step over device copies of the host arrays, `shift` elements into their buffers; what it left there."""
    keep, parts = [], []
    for h in hosts:
        part = {}
        for name, a in h.items():
            at = 0 if name.endswith("scales") else shift
            base = ctx.to_device(np.concatenate([np.zeros(at, a.dtype), a, np.full(4, 99, a.dtype)]))
            keep.append((base, at))
            part[name] = hip.DeviceArray(ctx, base.ptr + at * a.itemsize, a.nbytes, a.dtype, a.shape)
        parts.append(part)
    ctx.adamw_step(hip.AdamW.of(**hyper), hip.AdamWTensors.of(parts))
    ctx.synchronize()
    out, k = [], 0
    for h in hosts:
        got = {}
        for name, a in h.items():
            base, at = keep[k]
            k += 1
            flat = base.to_host()
            assert np.all(flat[at + a.size:] == np.array(99, a.dtype)) and np.all(flat[:at] == 0), name
            got[name] = flat[at:at + a.size]
            ctx.free(base)
        out.append(got)
    return out


def check(got, h, eight, **hyper):
    p, g, m, v = wide(h, eight)
    gs = g * hyper.get("grad_scale", 1.0)
    want_p, want_m, want_v = ref.adamw(p, g, m, v, **hyper)
    mag_m = np.abs(hyper["beta1"] * m) + np.abs((1 - hyper["beta1"]) * gs)
    move = hyper["lr"] / (1 - hyper["beta1"] ** hyper["step"]) * mag_m / (
        np.sqrt(want_v / (1 - hyper["beta2"] ** hyper["step"])) + hyper["eps"])
    assert np.all(np.abs(got["param"] - want_p) <= F32 * (np.abs(p) + 2 * move))
    if "copy" in h:
        assert np.array_equal(got["copy"], ref.to_bf16(got["param"]))
    assert np.array_equal(got["grad"], h["grad"])
    if not eight:
        assert np.all(np.abs(got["m"] - want_m) <= F32 * mag_m + 1e-44)
        assert np.all(np.abs(got["v"] - want_v) <= F32 * want_v + 1e-44)
        return
    for name, want in (("m", want_m), ("v", np.sqrt(want_v))):
        s = got[name + "_scales"].astype(np.float64)
        top = np.zeros(s.size * ref.BLOCK)
        top[:want.size] = np.abs(want)
        top = top.reshape(-1, ref.BLOCK).max(axis=1)
        slack = 2 * F32 * (np.abs(want) + mag_m if name == "m" else want)
        reach = np.zeros(s.size * ref.BLOCK)
        reach[:want.size] = slack
        assert np.all(np.abs(s - top / ref.TOP) <= (reach.reshape(-1, ref.BLOCK).max(axis=1) + F32 * top) / ref.TOP + 1e-44)
        each = np.repeat(s, ref.BLOCK)[:want.size]
        # (a root below half of the smallest value is held as the smallest: up to a whole one away)
        least = ref.LEAST if name == "v" else ref.LEAST / 2
        bound = np.maximum(np.abs(want) * ref.FP8, least * each) * (1 + 1e-4) + slack + 1e-44
        assert np.all(np.abs(unblock(got[name], got[name + "_scales"]) - want) <= bound), name
    assert np.all((ref.from_fp8(got["v"]) > 0) == (want_v > 0))


SIZES = [1, 3, 4, 255, 256, 257, 1024, 4095, 4096, 4097, 10_007]


@pytest.mark.parametrize("eight", [False, True], ids=["f32", "fp8"])
@pytest.mark.parametrize("grad", ["f32", "bf16"])
@pytest.mark.parametrize("shift", [0, 1])
def test_sizes(ctx, eight, grad, shift):
    rng = np.random.default_rng(3)
    hosts = [tensor(rng, n, grad, eight, copy=n % 2 == 0) for n in SIZES]
    hyper = dict(HYPER, step=7, grad_scale=0.25)
    for h, got in zip(hosts, step(ctx, hosts, shift, **hyper)):
        check(got, h, eight, **hyper)


@pytest.mark.parametrize("eight", [False, True], ids=["f32", "fp8"])
def test_many_tensors_of_either_gradient(ctx, eight):
    """More tensors than a launch takes, none of them empty but one, gradients of both types; the first step."""
    rng = np.random.default_rng(4)
    hosts = [tensor(rng, 1 + (i * 37) % 600, "bf16" if i % 3 else "f32", eight, first=True) for i in range(130)]
    hosts.insert(50, tensor(rng, 0, "f32", eight))
    hyper = dict(HYPER, step=1)
    for h, got in zip(hosts, step(ctx, hosts, **hyper)):
        if h["param"].size:
            check(got, h, eight, **hyper)


def test_ten_steps_follow_the_formula(ctx):
    """32-bit states over ten steps: errors of a step add up, at most ten of them."""
    rng = np.random.default_rng(5)
    h = tensor(rng, 5000, first=True)
    p, g, m, v = wide(h, False)
    for t in range(1, 11):
        h["grad"] = (rng.normal(size=5000) * 1e-2).astype(np.float32)
        p, m, v = ref.adamw(p, h["grad"].astype(np.float64), m, v, step=t, **HYPER)
        h = step(ctx, [h], step=t, **HYPER)[0]
    # a step moves a value by at most lr / (1 - beta1): ten times six half-ulps of that and of the value
    assert np.all(np.abs(h["param"] - p) <= 10 * F32 * (np.abs(p) + 10 * HYPER["lr"]))
    assert np.all(np.abs(h["m"] - m) <= 10 * F32 * 0.05) and np.all(np.abs(h["v"] - v) <= 10 * F32 * 0.05 ** 2)


def test_gradients_of_zero_and_no_number(ctx):
    """8 bits: a block without any gradient yet stays zero and finite; one with a NaN reads back as NaN, others do not."""
    n = 4 * ref.BLOCK
    h = tensor(np.random.default_rng(6), n, "f32", True, first=True)
    h["grad"][:ref.BLOCK] = 0.0
    h["grad"][ref.BLOCK + 5] = np.nan
    h["grad"][2 * ref.BLOCK + 9] = np.inf
    old = h["param"].copy()
    got = step(ctx, [h], step=1, **HYPER)[0]
    assert np.all(got["m"][:256] == 0) and np.all(got["v"][:256] == 0) and got["m_scales"][0] == 0 and got["v_scales"][0] == 0
    assert np.allclose(got["param"][:256], old[:256] * (1 - 1e-4), rtol=1e-6, atol=0)
    assert np.isnan(got["m_scales"][1]) and np.isnan(got["v_scales"][1]) and np.isnan(got["param"][256 + 5])
    assert np.all(np.isfinite(np.delete(got["param"], [256 + 5, 512 + 9])))
    assert np.isinf(got["m_scales"][2]) and np.all(np.isfinite(got["m_scales"][3:])) and np.all(ref.from_fp8(got["v"][768:]) > 0)


def test_the_same_bits_each_time(ctx):
    h = [tensor(np.random.default_rng(7), n, "bf16", True) for n in (10_007, 300)]
    a, b = step(ctx, h, step=3, **HYPER), step(ctx, h, step=3, **HYPER)
    assert all(np.array_equal(x[k], y[k]) for x, y in zip(a, b) for k in x)


def test_no_tensors(ctx):
    ctx.adamw_step(hip.AdamW.of(**HYPER), hip.AdamWTensors.of([]))
    ctx.synchronize()

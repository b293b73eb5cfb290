"""Operators of a feed-forward block: what a program calls to train one and to serve tokens through it.

Each case is one pass through an operator on inputs resident on the GPU. ``listed()`` gives the fixed cases,
``draw()`` more of the same ranges, ``prepare()`` the inputs of one case, ``run()`` one pass, in plain torch or
(``own``) through the public ctypes binding (``dotcompute_amd.hip``), ``exact()`` the same result in 64 bits.

Kinds of cases:
  norm             h = x + residual, y = h / rms(h) * weight; y in x's type, or in 8 bits (e4m3) with a scale a row
  norm_backward    the gradients of y by x (added to the one that reaches h directly) and by the weight
  linear           y = act(x w^T + bias) + residual, w a row per output; x and w in bfloat16, or in 8 bits with a
                   scale a row; with z = x w^T + bias kept for the backward pass where the case says so
  linear_backward  the gradients of y by x, w and bias (bfloat16, sums in 32 bits)
  adamw            one AdamW step over all tensors of a stack of blocks, states in 32 bits, or in 8 bits with a scale
                   for every 256 elements (the second moment by its root)
"""
import math

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6
TOP = 448.0  # the largest e4m3 value
LOWEST = 2.0 ** -9  # the smallest one above zero
BIG = 3.4028234663852886e38  # the largest float32 value: what 448 / 0 counts as
BLOCK = 256  # elements of an 8-bit state that share a scale
ADAMW = {"lr": 1e-4, "beta1": 0.9, "beta2": 0.95, "eps": 1e-8, "weight_decay": 0.1, "step": 100}


def listed():
    return [
        # eight sequences, one new token each, on their way into an 8-bit product. Latency.
        {"name": "norm_fp8_tokens", "kind": "norm", "dtype": "bf16", "out": "fp8", "rows": 8, "cols": 4096},
        # a training batch's worth of tokens
        {"name": "norm_batch", "kind": "norm", "dtype": "bf16", "out": "same", "rows": 16384, "cols": 4096},
        # its gradient, over rows and a width that no tile divides
        {"name": "norm_backward_odd", "kind": "norm_backward", "dtype": "bf16", "rows": 8191, "cols": 2050},
        # one token through a layer with everything in the epilogue. Bound by reading the weights.
        {"name": "linear_token", "kind": "linear", "dtype": "bf16", "act": "silu", "pre": False, "residual": True,
         "m": 1, "n": 4096, "k": 4096},
        # a ragged handful of tokens through 8-bit weights
        {"name": "linear_fp8_tokens", "kind": "linear", "dtype": "fp8", "act": "none", "pre": False, "residual": True,
         "m": 17, "n": 8192, "k": 4096},
        # a training pass, every side odd
        {"name": "linear_odd", "kind": "linear", "dtype": "bf16", "act": "gelu", "pre": True, "residual": False,
         "m": 1537, "n": 2049, "k": 1023},
        # the largest one
        {"name": "linear_8192", "kind": "linear", "dtype": "bf16", "act": "gelu_tanh", "pre": True, "residual": False,
         "m": 8192, "n": 8192, "k": 8192},
        # a long prompt through 8-bit weights
        {"name": "linear_fp8_prompt", "kind": "linear", "dtype": "fp8", "act": "relu", "pre": False, "residual": False,
         "m": 4096, "n": 8192, "k": 4096},
        # gradients of a layer whose sides are multiples of 8 only
        {"name": "linear_backward_2000", "kind": "linear_backward", "act": "gelu", "m": 2000, "n": 3000, "k": 1000},
        # gradients of a wide layer over a long batch
        {"name": "linear_backward_8192", "kind": "linear_backward", "act": "silu", "m": 8192, "n": 8192, "k": 2048},
        # the step of a small model: thirty tensors, most of them small. Launches.
        {"name": "adamw_small", "kind": "adamw", "states": "f32", "layers": 6, "width": 100},
        # the step of a large one with 8-bit states
        {"name": "adamw_8bit", "kind": "adamw", "states": "fp8", "layers": 4, "width": 2048},
    ]


def _log_size(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Widths of real layers: multiples of a tile, of 8, or odd."""
    step = rng.choice([1, 8, 64, 64, 256])
    return max(lo, _log_size(rng, lo, hi) // step * step)


def draw(rng):
    kind = rng.choice(["norm", "norm_backward", "linear", "linear", "linear_backward", "adamw"])
    if kind in ("norm", "norm_backward"):
        cols = _width(rng, 64, 16384)
        case = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f32"]), "cols": cols,
                "rows": _log_size(rng, 1, min(16384, (1 << 26) // cols))}
        if kind == "norm":
            case["out"] = rng.choice(["same", "fp8"])
        return case
    if kind == "adamw":
        width = _width(rng, 32, 2048)
        layers = rng.randint(1, max(1, min(8, (1 << 27) // (8 * width * width))))
        return {"kind": kind, "states": rng.choice(["f32", "fp8"]), "layers": layers, "width": width}
    act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    m, n, k = _log_size(rng, 1, 8192), _width(rng, 64, 8192), _width(rng, 64, 8192)
    if kind == "linear":
        return {"kind": kind, "dtype": rng.choice(["bf16", "fp8"]), "act": act, "pre": rng.random() < 0.3,
                "residual": rng.random() < 0.5, "m": m, "n": n, "k": k}
    if m * n * k > 8192 * 8192 * 2048:
        k = max(64, 8192 * 8192 * 2048 // (m * n))
    return {"kind": kind, "act": act, "m": m, "n": n, "k": k}


# ---- inputs --------------------------------------------------------------------------------------

_T = {"bf16": torch.bfloat16, "f32": torch.float32, "fp8": torch.float8_e4m3fn}


def _sizes(case):
    """The tensors of a stack of blocks: a norm's weight, two matrices and their biases in each."""
    d = case["width"]
    return [n for _ in range(case["layers"]) for n in (d, 4 * d * d, 4 * d, 4 * d * d, d)]


def _padded(n):
    return (n + BLOCK - 1) // BLOCK * BLOCK


def _rows_fp8(t):
    """Rows in 8 bits: (e4m3 values, the scale of each row)."""
    top = t.abs().amax(1)
    return (t * (TOP / top)[:, None]).clamp_(-TOP, TOP).to(_T["fp8"]), top / TOP


def _inputs(case, seed):
    """The case's input tensors by name, from the seed alone."""
    gen, kind = torch.Generator(device=DEV).manual_seed(int(seed)), case["kind"]

    def randn(*shape, dtype="bf16", scale=1.0, shift=0.0):
        t = torch.randn(*shape, device=DEV, generator=gen)
        if scale != 1.0 or shift != 0.0:
            t.mul_(scale).add_(shift)
        return t if dtype == "f32" else t.to(_T[dtype])

    if kind in ("norm", "norm_backward"):
        rows, cols, dt = case["rows"], case["cols"], case["dtype"]
        t = {"x": randn(rows, cols, dtype=dt), "weight": randn(cols, dtype=dt, scale=0.1, shift=1.0),
             "residual": randn(rows, cols, dtype=dt)}
        if kind == "norm_backward":
            t["dy"] = randn(rows, cols, dtype=dt)
        return t
    if kind == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        t = {"bias": randn(n, scale=0.1)}
        if case["dtype"] == "fp8":
            t["x"], t["x_scales"] = _rows_fp8(randn(m, k, dtype="f32"))
            t["w"], t["w_scales"] = _rows_fp8(randn(n, k, dtype="f32", scale=k ** -0.5))
        else:
            t["x"], t["w"] = randn(m, k), randn(n, k, scale=k ** -0.5)
        if case["residual"]:
            t["residual"] = randn(m, n)
        return t
    if kind == "linear_backward":
        m, n, k = case["m"], case["n"], case["k"]
        return {"dy": randn(m, n), "x": randn(m, k), "w": randn(n, k, scale=k ** -0.5), "pre": randn(m, n)}
    total = sum(_padded(n) for n in _sizes(case))
    used = torch.zeros(total, device=DEV)
    at = 0
    for n in _sizes(case):
        used[at:at + n] = 1.0
        at += _padded(n)
    t = {"param": randn(total, dtype="f32", scale=0.02).mul_(used),
         "grad": randn(total, dtype="f32", scale=1e-3).mul_(used).to(torch.bfloat16)}
    m = randn(total, dtype="f32", scale=3e-4).mul_(used)
    root = randn(total, dtype="f32", scale=2e-4, shift=1e-3).abs_().mul_(used)
    if case["states"] == "fp8":
        t["m"], t["m_scales"] = _blocks_fp8(m, 0.0)
        t["v"], t["v_scales"] = _blocks_fp8(root, LOWEST)
    else:
        t["m"], t["v"] = m, root.square_()
    return t


# ---- the plain forms -----------------------------------------------------------------------------


def _blocks_fp8(t, least):
    """8-bit states: e4m3 values and a scale for every BLOCK of them; `least`: what small ones are held as."""
    blocks = t.view(-1, BLOCK)
    top = blocks.abs().amax(1)
    codes = (blocks * (TOP / top).clamp(max=BIG)[:, None]).clamp(-TOP, TOP)
    if least:
        codes = torch.where(blocks > 0, codes.clamp(min=least), codes)
    return codes.to(_T["fp8"]).view(-1), top / TOP


def _act(name, z):
    if name == "relu":
        return z.clamp(min=0.0)
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_slope(name, z):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * math.sqrt(0.5 / math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    return torch.ones_like(z)


def _plain(s):
    case, t = s.case, s.t
    kind = case["kind"]
    if kind == "norm":
        h = t["x"].float() + t["residual"].float()
        y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * t["weight"].float()
        if case["out"] == "same":
            return {"sum": h.to(t["x"].dtype), "y": y.to(t["x"].dtype)}
        top = y.abs().amax(1)
        q = (y * (TOP / top).clamp(max=BIG)[:, None]).clamp(-TOP, TOP).to(_T["fp8"])
        return {"sum": h.to(t["x"].dtype), "y": q, "scales": top / TOP}
    if kind == "norm_backward":
        h, dy = t["x"].float(), t["dy"].float()
        rstd = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
        unit, g = h * rstd, dy * t["weight"].float()
        dx = rstd * (g - unit * (g * unit).mean(1, keepdim=True)) + t["residual"].float()
        return {"dx": dx.to(t["x"].dtype), "dweight": (dy * unit).sum(0)}
    if kind == "linear":
        z = t["x"].float() @ t["w"].float().t()
        if case["dtype"] == "fp8":
            z = z * t["x_scales"][:, None] * t["w_scales"][None, :]
        z = z + t["bias"].float()
        y = _act(case["act"], z)
        if case["residual"]:
            y = y + t["residual"].float()
        out = {"y": y.to(torch.bfloat16)}
        if case["pre"]:
            out["pre"] = z.to(torch.bfloat16)
        return out
    if kind == "linear_backward":
        dz = t["dy"].float()
        if case["act"] != "none":
            dz = dz * _act_slope(case["act"], t["pre"].float())
        return {"dx": (dz @ t["w"].float()).to(torch.bfloat16), "dw": (dz.t() @ t["x"].float()).to(torch.bfloat16),
                "dbias": dz.sum(0)}
    a, g = ADAMW, t["grad"].float()
    m, v = t["m"], t["v"]
    if case["states"] == "fp8":
        m = (m.float().view(-1, BLOCK) * t["m_scales"][:, None]).view(-1)
        v = (v.float().view(-1, BLOCK) * t["v_scales"][:, None]).square().view(-1)
    m = a["beta1"] * m + (1.0 - a["beta1"]) * g
    v = a["beta2"] * v + (1.0 - a["beta2"]) * (g * g)
    root = torch.sqrt(v)
    rate = a["lr"] / (1.0 - a["beta1"] ** a["step"])
    p = t["param"] * (1.0 - a["lr"] * a["weight_decay"]) - \
        rate * m / (root * (1.0 / math.sqrt(1.0 - a["beta2"] ** a["step"])) + a["eps"])
    if case["states"] == "fp8":
        m, m_scales = _blocks_fp8(m, 0.0)
        v, v_scales = _blocks_fp8(root, LOWEST)
        t["m_scales"].copy_(m_scales)
        t["v_scales"].copy_(v_scales)
    t["param"].copy_(p)
    t["copy"].copy_(p)
    t["m"].copy_(m)
    t["v"].copy_(v)
    return {name: t[name] for name in _ADAMW_OUT if name in t}


_ADAMW_OUT = ("param", "copy", "m", "v", "m_scales", "v_scales")


# ---- a program's state ---------------------------------------------------------------------------


class State:
    """A case, its tensors by name and, for the framework's calls, their arguments."""

    def __init__(self, case, tensors):
        self.case, self.t, self.args, self.tensors = case, tensors, None, None


_ctx = None


def context():
    """The program's one context, made on first use."""
    global _ctx
    if _ctx is None:
        from dotcompute_amd import hip

        _ctx = hip.Context(0)
    return _ctx


def _array(t):
    """The binding's view of a tensor's memory (the state keeps the tensor)."""
    import numpy as np

    from dotcompute_amd import hip

    dt = np.dtype({torch.float32: np.float32, torch.bfloat16: np.uint16, _T["fp8"]: np.uint8}[t.dtype])
    return hip.DeviceArray(context(), t.data_ptr(), t.numel() * dt.itemsize, dt, tuple(t.shape))


def _arguments(s):
    """What the framework's calls take: the tensors of the state by their places in the operator."""
    from dotcompute_amd import hip

    case, kind = s.case, s.case["kind"]
    a = {name: _array(t) for name, t in s.t.items()}
    if kind == "norm":
        s.args = hip.RmsNorm.of(eps=EPS, **a)
    elif kind == "norm_backward":
        s.args = hip.RmsNormGrad.of(eps=EPS, dy=a["dy"], h=a["x"], weight=a["weight"], dh=a["residual"], dx=a["dx"],
                                    dweight=a["dweight"])
    elif kind == "linear":
        s.args = hip.Linear.of(activation=case["act"], **a)
    elif kind == "linear_backward":
        s.args = hip.LinearGrad.of(activation=case["act"], **a)
    else:
        s.args = hip.AdamW.of(**ADAMW)
        parts, at = [], 0
        for n in _sizes(case):
            part = {name: _array(t[at // BLOCK:(at + _padded(n)) // BLOCK] if name.endswith("scales") else t[at:at + n])
                    for name, t in s.t.items()}
            parts.append(part)
            at += _padded(n)
        s.tensors = hip.AdamWTensors.of(parts)


def prepare(case, seed):
    kind, t = case["kind"], _inputs(case, seed)

    def empty(*shape, dtype):
        return torch.zeros(*shape, device=DEV, dtype=_T[dtype])

    # the outputs' buffers, as a program keeps them
    if kind == "norm":
        rows, cols, dt = case["rows"], case["cols"], case["dtype"]
        t["sum"], t["y"] = empty(rows, cols, dtype=dt), empty(rows, cols, dtype=dt if case["out"] == "same" else "fp8")
        if case["out"] == "fp8":
            t["scales"] = empty(rows, dtype="f32")
    elif kind == "norm_backward":
        t["dx"], t["dweight"] = torch.zeros_like(t["x"]), empty(case["cols"], dtype="f32")
    elif kind == "linear":
        t["y"] = empty(case["m"], case["n"], dtype="bf16")
        if case["pre"]:
            t["pre"] = torch.zeros_like(t["y"])
    elif kind == "linear_backward":
        t["dx"], t["dw"] = torch.zeros_like(t["x"]), torch.zeros_like(t["w"])
        t["dbias"] = empty(case["n"], dtype="f32")
    else:
        t["copy"] = empty(t["param"].numel(), dtype="bf16")
    s = State(case, t)
    if own:
        _arguments(s)
    torch.cuda.synchronize()  # the inputs are made on torch's stream, a context has its own
    return s


def run(s):
    if not own:
        return _plain(s)
    ctx, t, kind = context(), s.t, s.case["kind"]
    if kind == "norm":
        ctx.rms_norm(s.args)
        return {name: t[name] for name in ("sum", "y", "scales") if name in t}
    if kind == "norm_backward":
        ctx.rms_norm_backward(s.args)
        return {"dx": t["dx"], "dweight": t["dweight"]}
    if kind == "linear":
        ctx.linear(s.args)
        return {name: t[name] for name in ("y", "pre") if name in t}
    if kind == "linear_backward":
        ctx.linear_backward(s.args)
        return {"dx": t["dx"], "dw": t["dw"], "dbias": t["dbias"]}
    ctx.adamw_step(s.args, s.tensors)
    return {name: t[name] for name in _ADAMW_OUT if name in t}


def work(case):
    """Bytes and operations that no implementation can do without: each input read and each output
    written once."""
    kind = case["kind"]
    if kind in ("norm", "norm_backward"):
        rows, cols, size = case["rows"], case["cols"], 2 if case["dtype"] == "bf16" else 4
        if kind == "norm":
            out = rows * (cols + 4) if case["out"] == "fp8" else rows * cols * size
            return {"bytes": 3 * rows * cols * size + cols * size + out, "flops": 5 * rows * cols}
        return {"bytes": 4 * rows * cols * size + cols * (size + 4), "flops": 12 * rows * cols}
    if kind == "adamw":
        n = sum(_sizes(case))
        return {"bytes": n * 28 if case["states"] == "f32" else n * 16 + n / BLOCK * 16, "flops": 15 * n}
    m, n, k = case["m"], case["n"], case["k"]
    if kind == "linear_backward":
        return {"bytes": 2 * (2 * m * n + 2 * m * k + 2 * n * k) + 4 * n, "flops": 4 * m * n * k}
    size = 1 if case["dtype"] == "fp8" else 2
    return {"bytes": size * (m + n) * k + (4 * (m + n) if size == 1 else 0) + 2 * n +
            2 * m * n * (1 + case["pre"] + case["residual"]), "flops": 2 * m * n * k}


# ---- the same results in 64 bits, from the operators' definitions -----------------------------------


def _erf_part(z):
    return torch.special.ndtr(z)  # the normal distribution's function: gelu(z) = z P(z)


def exact(case, seed):
    kind, t = case["kind"], _inputs(case, seed)
    d = {name: v.double() if v.dtype != _T["fp8"] else v.float().double() for name, v in t.items()}
    if kind == "norm":
        h = d["x"] + d["residual"]
        y = d["weight"] * h / torch.sqrt(torch.linalg.vector_norm(h, dim=1, keepdim=True) ** 2 / case["cols"] + EPS)
        if case["out"] == "same":
            return {"sum": h, "y": y}
        scales = y.abs().max(dim=1).values / TOP
        return {"sum": h, "y": y / scales[:, None], "scales": scales}
    if kind == "norm_backward":
        h, dy, n = d["x"], d["dy"], case["cols"]
        ms = torch.linalg.vector_norm(h, dim=1, keepdim=True) ** 2 / n + EPS
        g = dy * d["weight"]
        along = (g * h).sum(1, keepdim=True) / (n * ms)
        return {"dx": (g - h * along) / torch.sqrt(ms) + d["residual"], "dweight": (dy * h / torch.sqrt(ms)).sum(0)}
    if kind == "linear":
        x, w = d["x"], d["w"]
        if case["dtype"] == "fp8":
            x, w = x * d["x_scales"][:, None], w * d["w_scales"][:, None]
        z = torch.addmm(d["bias"], x, w.t())
        y = {"none": lambda: z, "relu": lambda: torch.where(z > 0, z, torch.zeros_like(z)), "gelu": lambda: z * _erf_part(z),
             "gelu_tanh": lambda: z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)),
             "silu": lambda: z * torch.sigmoid(z)}[case["act"]]()
        out = {"y": y + d["residual"] if case["residual"] else y}
        if case["pre"]:
            out["pre"] = z
        return out
    if kind == "linear_backward":
        z = d["pre"]
        if case["act"] == "none":
            slope = torch.ones_like(z)
        elif case["act"] == "relu":
            slope = torch.where(z > 0, 1.0, 0.0)
        elif case["act"] == "gelu":
            slope = _erf_part(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        else:  # z s(u(z)): s + z s (1 - s) u'
            c = math.sqrt(2 / math.pi)
            u, du = (z, 1.0) if case["act"] == "silu" else (2 * c * (z + 0.044715 * z ** 3), 2 * c * (1 + 0.134145 * z * z))
            sig = torch.sigmoid(u)
            slope = sig + z * sig * (1 - sig) * du
        dz = d["dy"] * slope
        return {"dx": torch.mm(dz, d["w"]), "dw": torch.mm(dz.t(), d["x"]), "dbias": dz.sum(0)}
    a, g, eight = ADAMW, d["grad"], case["states"] == "fp8"
    m, v = d["m"], d["v"]
    if eight:
        m = m * torch.repeat_interleave(d["m_scales"], BLOCK)
        v = (v * torch.repeat_interleave(d["v_scales"], BLOCK)) ** 2
    m = m + (1 - a["beta1"]) * (g - m)
    v = v + (1 - a["beta2"]) * (g * g - v)
    hat_m, hat_v = m / (1 - a["beta1"] ** a["step"]), v / (1 - a["beta2"] ** a["step"])
    p = d["param"] - a["lr"] * (hat_m / (torch.sqrt(hat_v) + a["eps"]) + a["weight_decay"] * d["param"])
    out = {"param": p, "copy": p, "m": m, "v": v}
    if eight:
        for name, state in (("m", m), ("v", torch.sqrt(v))):
            top = state.abs().view(-1, BLOCK).max(dim=1).values / TOP
            out[name + "_scales"] = top
            unit = torch.where(top > 0, top, torch.ones_like(top))
            out[name] = state / torch.repeat_interleave(unit, BLOCK)
    return out

"""Operators of a gated feed-forward block: layer norm, both projections with their gate, 8-bit products with a scale for each
block of 128.

Each case is one pass through an operator on inputs resident on the GPU. ``listed()`` gives the fixed cases, ``draw()`` more of the
same ranges, ``prepare()`` the inputs of one case, ``run()`` one pass, in plain torch or (``own``) through the public ctypes
binding (``dotcompute_amd.hip``), ``exact()`` the same result in 64 bits.

Kinds of cases:
  layer_norm           h = x + residual, y = (h - mean) / deviation * weight + bias; y in x's type, or in 8 bits (e4m3) with a scale a row
  layer_norm_backward  the gradients of y by x (added to the one that reaches h directly), by the weight and by the bias
  gated                y = act(x wg^T + bg) (x wu^T + bu); bfloat16, or 8 bits with a scale a row ("fp8") or for every 128 of a row
                       ("blocks"); with both projections' results kept for the backward pass where the case says so
  gated_backward       the gradients of y by x, both weights and both biases (bfloat16, sums in 32 bits)
  linear_blocks        y = act(x w^T + bias) + residual of 8-bit values with a scale for every 128 of a row, for both operands
  quantize_blocks      rows in 8 bits with such scales: powers of two, held as their exponents (e8m0: 2^(byte - 127))
"""
import math

import torch

own = False

DEV = "cuda:0"
EPS = 1e-5
TOP = 448.0  # the largest e4m3 value
BLOCK = 128  # elements of a row that share a scale


def listed():
    return [
        # eight sequences, one new token each, on their way into an 8-bit product. Latency.
        {"name": "layer_norm_fp8_tokens", "kind": "layer_norm", "dtype": "bf16", "out": "fp8", "rows": 8, "cols": 4096},
        # a training batch's worth of tokens
        {"name": "layer_norm_batch", "kind": "layer_norm", "dtype": "bf16", "out": "same", "rows": 16384, "cols": 4096},
        # its gradient, over rows and a width that no tile divides
        {"name": "layer_norm_backward_odd", "kind": "layer_norm_backward", "dtype": "bf16", "rows": 8191, "cols": 2050},
        # a small batch in float32
        {"name": "layer_norm_backward_f32", "kind": "layer_norm_backward", "dtype": "f32", "rows": 500, "cols": 1024},
        # one token through both projections. Bound by reading the weights.
        {"name": "gated_token", "kind": "gated", "dtype": "bf16", "act": "silu", "pre": False, "m": 1, "n": 8192, "k": 4096},
        # a training pass
        {"name": "gated_batch", "kind": "gated", "dtype": "bf16", "act": "silu", "pre": True, "m": 4096, "n": 8192, "k": 4096},
        # gradients of a small block whose sides are multiples of 8 only
        {"name": "gated_backward_2000", "kind": "gated_backward", "act": "gelu_tanh", "m": 2000, "n": 2504, "k": 1000},
        # gradients of a wide block over a long batch: the largest one
        {"name": "gated_backward_8192", "kind": "gated_backward", "act": "silu", "m": 8192, "n": 8192, "k": 2048},
        # a ragged handful of tokens through 8-bit weights
        {"name": "linear_blocks_tokens", "kind": "linear_blocks", "act": "none", "residual": True, "m": 17, "n": 8192, "k": 4096},
        # a long prompt through them
        {"name": "linear_blocks_prompt", "kind": "linear_blocks", "act": "none", "residual": True, "m": 4096, "n": 4096, "k": 8192},
        # what those tokens' product takes. Latency.
        {"name": "quantize_blocks_tokens", "kind": "quantize_blocks", "dtype": "bf16", "rows": 17, "cols": 4096},
        # a prompt's activations, or a weight, over sides that no block divides
        {"name": "quantize_blocks_odd", "kind": "quantize_blocks", "dtype": "bf16", "rows": 8191, "cols": 8190},
    ]


def _log_size(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Widths of real layers: multiples of a tile, of 8, or odd."""
    step = rng.choice([1, 8, 64, 64, 256])
    return max(lo, _log_size(rng, lo, hi) // step * step)


def draw(rng):
    kind = rng.choice(["layer_norm", "layer_norm_backward", "gated", "gated", "gated_backward", "linear_blocks", "quantize_blocks"])
    if kind in ("layer_norm", "layer_norm_backward", "quantize_blocks"):
        cols = _width(rng, 64, 16384)
        case = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f32"]), "cols": cols,
                "rows": _log_size(rng, 1, min(16384, (1 << 26) // cols))}
        if kind == "layer_norm":
            case["out"] = rng.choice(["same", "fp8"])
        return case
    act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu", "silu"])
    m, n, k = _log_size(rng, 1, 8192), _width(rng, 64, 8192), _width(rng, 64, 8192)
    if kind == "gated":
        if m * n * k > 8192 * 8192 * 4096:
            k = max(64, 8192 * 8192 * 4096 // (m * n))
        return {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "fp8", "blocks"]), "act": act, "pre": rng.random() < 0.4,
                "m": m, "n": n, "k": k}
    if kind == "linear_blocks":
        return {"kind": kind, "act": act, "residual": rng.random() < 0.5, "m": m, "n": n, "k": k}
    if m * n * k > 8192 * 8192 * 2048:
        k = max(64, 8192 * 8192 * 2048 // (m * n))
    return {"kind": kind, "act": act, "m": m, "n": n, "k": k}


# ---- inputs --------------------------------------------------------------------------------------

_T = {"bf16": torch.bfloat16, "f32": torch.float32, "fp8": torch.float8_e4m3fn}


def _rows_fp8(t):
    """Rows in 8 bits: (e4m3 values, the scale of each row)."""
    top = t.abs().amax(1)
    return (t * (TOP / top)[:, None]).clamp_(-TOP, TOP).to(_T["fp8"]), top / TOP


def _blocks_of(t):
    """[rows][blocks][BLOCK], the last block filled up with zeros."""
    rows, cols = t.shape
    return torch.nn.functional.pad(t, (0, -cols % BLOCK)).view(rows, -1, BLOCK)


def _blocks_fp8(t):
    """Rows in 8 bits with a scale for every BLOCK of a row, the least power of two that takes its largest value to 448 or below:
    (e4m3 values, the scales' exponents plus 127 as [blocks][rows])."""
    b = _blocks_of(t)
    top = b.abs().amax(2)
    fraction, exponent = torch.frexp(top)  # top = fraction 2^exponent, fraction in [1/2, 1)
    e = torch.where(top > 0, exponent - 9 + (fraction > 0.875).int(), torch.full_like(exponent, -127)).clamp(min=-127)
    q = torch.ldexp(b, -e[:, :, None]).to(_T["fp8"])
    return q.view(t.shape[0], -1)[:, :t.shape[1]].contiguous(), (e + 127).to(torch.uint8).t().contiguous()


def _inputs(case, seed):
    """The case's input tensors by name, from the seed alone."""
    gen, kind = torch.Generator(device=DEV).manual_seed(int(seed)), case["kind"]

    def randn(*shape, dtype="bf16", scale=1.0, shift=0.0):
        t = torch.randn(*shape, device=DEV, generator=gen)
        if scale != 1.0 or shift != 0.0:
            t.mul_(scale).add_(shift)
        return t if dtype == "f32" else t.to(_T[dtype])

    if kind in ("layer_norm", "layer_norm_backward"):
        rows, cols, dt = case["rows"], case["cols"], case["dtype"]
        t = {"x": randn(rows, cols, dtype=dt, shift=0.5), "weight": randn(cols, dtype=dt, scale=0.1, shift=1.0),
             "residual": randn(rows, cols, dtype=dt)}
        if kind == "layer_norm":
            t["bias"] = randn(cols, dtype=dt, scale=0.1)
        else:
            t["dy"] = randn(rows, cols, dtype=dt)
        return t
    if kind == "quantize_blocks":
        t = randn(case["rows"], case["cols"], dtype="f32")
        return {"x": t.mul_(torch.exp(randn(case["rows"], 1, dtype="f32"))).to(_T[case["dtype"]])}
    m, n, k = case["m"], case["n"], case["k"]
    if kind == "gated_backward":
        return {"dy": randn(m, n), "x": randn(m, k), "w_gate": randn(n, k, scale=k ** -0.5), "w_up": randn(n, k, scale=k ** -0.5),
                "pre_gate": randn(m, n), "pre_up": randn(m, n)}
    weights = {"w": "w_scales"} if kind == "linear_blocks" else {"w_gate": "gate_scales", "w_up": "up_scales"}
    t = {name.replace("w", "bias", 1): randn(n, scale=0.1) for name in weights}
    dtype = "blocks" if kind == "linear_blocks" else case["dtype"]
    code = {"fp8": _rows_fp8, "blocks": _blocks_fp8}.get(dtype)
    if code:
        t["x"], t["x_scales"] = code(randn(m, k, dtype="f32"))
        for name, scales in weights.items():
            t[name], t[scales] = code(randn(n, k, dtype="f32", scale=k ** -0.5))
    else:
        t["x"] = randn(m, k)
        for name in weights:
            t[name] = randn(n, k, scale=k ** -0.5)
    if case.get("residual"):
        t["residual"] = randn(m, n)
    return t


# ---- the plain forms -----------------------------------------------------------------------------


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


def _wide(q, scales, dtype):
    """The values that codes (or bfloat16 values) stand for, in 32 bits."""
    v = q.float()
    if dtype == "fp8":
        return v * scales[:, None]
    if dtype == "blocks":
        s = torch.exp2(scales.float() - 127.0).t()  # [rows][blocks]
        return (_blocks_of(v) * s[:, :, None]).view(q.shape[0], -1)[:, :q.shape[1]]
    return v


def _plain(s):
    case, t = s.case, s.t
    kind, bf16 = case["kind"], torch.bfloat16
    if kind == "layer_norm":
        h = t["x"].float() + t["residual"].float()
        d = h - h.mean(1, keepdim=True)
        y = d * torch.rsqrt((d * d).mean(1, keepdim=True) + EPS) * t["weight"].float() + t["bias"].float()
        if case["out"] == "same":
            return {"sum": h.to(t["x"].dtype), "y": y.to(t["x"].dtype)}
        top = y.abs().amax(1)
        return {"sum": h.to(t["x"].dtype), "y": (y * (TOP / top)[:, None]).clamp(-TOP, TOP).to(_T["fp8"]), "scales": top / TOP}
    if kind == "layer_norm_backward":
        h, dy = t["x"].float(), t["dy"].float()
        d = h - h.mean(1, keepdim=True)
        rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)
        unit, g = d * rstd, dy * t["weight"].float()
        dx = rstd * (g - g.mean(1, keepdim=True) - unit * (g * unit).mean(1, keepdim=True)) + t["residual"].float()
        return {"dx": dx.to(t["x"].dtype), "dweight": (dy * unit).sum(0), "dbias": dy.sum(0)}
    if kind == "quantize_blocks":
        q, scales = _blocks_fp8(t["x"].float())
        return {"q": q, "scales": scales}
    if kind == "gated":
        x = _wide(t["x"], t.get("x_scales"), case["dtype"])
        g = x @ _wide(t["w_gate"], t.get("gate_scales"), case["dtype"]).t() + t["bias_gate"].float()
        u = x @ _wide(t["w_up"], t.get("up_scales"), case["dtype"]).t() + t["bias_up"].float()
        out = {"y": (_act(case["act"], g) * u).to(bf16)}
        if case["pre"]:
            out["pre_gate"], out["pre_up"] = g.to(bf16), u.to(bf16)
        return out
    if kind == "gated_backward":
        dy, x, g, u = t["dy"].float(), t["x"].float(), t["pre_gate"].float(), t["pre_up"].float()
        dg, du = dy * u * _act_slope(case["act"], g), dy * _act(case["act"], g)
        return {"dx": (dg @ t["w_gate"].float() + du @ t["w_up"].float()).to(bf16), "dw_gate": (dg.t() @ x).to(bf16),
                "dw_up": (du.t() @ x).to(bf16), "dbias_gate": dg.sum(0), "dbias_up": du.sum(0)}
    z = _wide(t["x"], t["x_scales"], "blocks") @ _wide(t["w"], t["w_scales"], "blocks").t() + t["bias"].float()
    y = _act(case["act"], z)
    return {"y": (y + t["residual"].float() if case["residual"] else y).to(bf16)}


# ---- a program's state ---------------------------------------------------------------------------


class State:
    """A case, its tensors by name and, for the framework's calls, their arguments."""

    def __init__(self, case, tensors):
        self.case, self.t, self.args = case, tensors, None


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

    dt = np.dtype({torch.float32: np.float32, torch.bfloat16: np.uint16, _T["fp8"]: np.uint8, torch.uint8: np.uint8}[t.dtype])
    return hip.DeviceArray(context(), t.data_ptr(), t.numel() * dt.itemsize, dt, tuple(t.shape))


def _arguments(s):
    """What the framework's calls take: the tensors of the state by their places in the operator."""
    from dotcompute_amd import hip

    case, kind = s.case, s.case["kind"]
    a = {name: _array(t) for name, t in s.t.items()}
    if kind == "layer_norm":
        s.args = hip.LayerNorm.of(eps=EPS, **a)
    elif kind == "layer_norm_backward":
        s.args = hip.LayerNormGrad.of(eps=EPS, dy=a["dy"], h=a["x"], weight=a["weight"], dh=a["residual"], dx=a["dx"],
                                      dweight=a["dweight"], dbias=a["dbias"])
    elif kind == "gated":
        s.args = hip.GatedLinear.of(activation=case["act"], **a)
    elif kind == "gated_backward":
        s.args = hip.GatedLinearGrad.of(activation=case["act"], **a)
    elif kind == "linear_blocks":
        s.args = hip.LinearBlocks.of(activation=case["act"], **a)
    else:
        s.args = a


def prepare(case, seed):
    kind, t = case["kind"], _inputs(case, seed)

    def empty(*shape, dtype):
        return torch.zeros(*shape, device=DEV, dtype=_T[dtype])

    # the outputs' buffers, as a program keeps them
    if kind == "layer_norm":
        rows, cols, dt = case["rows"], case["cols"], case["dtype"]
        t["sum"], t["y"] = empty(rows, cols, dtype=dt), empty(rows, cols, dtype=dt if case["out"] == "same" else "fp8")
        if case["out"] == "fp8":
            t["scales"] = empty(rows, dtype="f32")
    elif kind == "layer_norm_backward":
        t["dx"] = torch.zeros_like(t["x"])
        t["dweight"], t["dbias"] = empty(case["cols"], dtype="f32"), empty(case["cols"], dtype="f32")
    elif kind == "quantize_blocks":
        t["q"] = empty(case["rows"], case["cols"], dtype="fp8")
        t["scales"] = torch.zeros((case["cols"] + BLOCK - 1) // BLOCK, case["rows"], device=DEV, dtype=torch.uint8)
    elif kind == "gated_backward":
        for name in ("x", "w_gate", "w_up"):
            t["d" + name] = torch.zeros_like(t[name])
        t["dbias_gate"], t["dbias_up"] = empty(case["n"], dtype="f32"), empty(case["n"], dtype="f32")
    else:
        t["y"] = empty(case["m"], case["n"], dtype="bf16")
        if case.get("pre"):
            t["pre_gate"], t["pre_up"] = torch.zeros_like(t["y"]), torch.zeros_like(t["y"])
    s = State(case, t)
    if own:
        _arguments(s)
    torch.cuda.synchronize()  # the inputs are made on torch's stream, a context has its own
    return s


_OUT = {"layer_norm": ("sum", "y", "scales"), "layer_norm_backward": ("dx", "dweight", "dbias"), "gated": ("y", "pre_gate", "pre_up"),
        "gated_backward": ("dx", "dw_gate", "dw_up", "dbias_gate", "dbias_up"), "linear_blocks": ("y",), "quantize_blocks": ("q", "scales")}


def run(s):
    if not own:
        return _plain(s)
    ctx, kind = context(), s.case["kind"]
    if kind == "layer_norm":
        ctx.layer_norm(s.args)
    elif kind == "layer_norm_backward":
        ctx.layer_norm_backward(s.args)
    elif kind == "gated":
        ctx.gated_linear(s.args)
    elif kind == "gated_backward":
        ctx.gated_linear_backward(s.args)
    elif kind == "linear_blocks":
        ctx.linear_blocks(s.args)
    else:
        ctx.quantize_fp8_blocks(s.args["x"], s.args["q"], s.args["scales"])
    return {name: s.t[name] for name in _OUT[kind] if name in s.t}


def work(case):
    """Bytes and operations that no implementation can do without: each input read and each output
    written once."""
    kind = case["kind"]
    if kind in ("layer_norm", "layer_norm_backward", "quantize_blocks"):
        rows, cols, size = case["rows"], case["cols"], 2 if case["dtype"] == "bf16" else 4
        blocks = (cols + BLOCK - 1) // BLOCK
        if kind == "layer_norm":
            out = rows * (cols + 4) if case["out"] == "fp8" else rows * cols * size
            return {"bytes": 3 * rows * cols * size + 2 * cols * size + out, "flops": 8 * rows * cols}
        if kind == "layer_norm_backward":
            return {"bytes": 4 * rows * cols * size + cols * (size + 8), "flops": 16 * rows * cols}
        return {"bytes": rows * cols * (size + 1) + rows * blocks, "flops": 2 * rows * cols}
    m, n, k = case["m"], case["n"], case["k"]
    if kind == "gated_backward":
        return {"bytes": 2 * (3 * m * n + 2 * m * k + 4 * n * k) + 8 * n, "flops": 8 * m * n * k}
    weights = 1 if kind == "linear_blocks" else 2
    dtype = "blocks" if kind == "linear_blocks" else case["dtype"]
    rows = m + weights * n
    scales = {"bf16": 0, "fp8": 4 * rows, "blocks": rows * ((k + BLOCK - 1) // BLOCK)}[dtype]
    results = 1 + (2 if case.get("pre") else 0) + (1 if case.get("residual") else 0)
    return {"bytes": (2 if dtype == "bf16" else 1) * rows * k + scales + 2 * weights * n + 2 * m * n * results,
            "flops": 2 * weights * m * n * k}


# ---- the same results in 64 bits, from the operators' definitions -----------------------------------


def _sigmoid_part(name, z):
    """act(z) = z s(u(z)): (s, u'(z)) for the activations that have this form."""
    if name == "silu":
        return torch.sigmoid(z), torch.ones_like(z)
    c = 2 * math.sqrt(2 / math.pi)
    return torch.sigmoid(c * (z + 0.044715 * z ** 3)), c * (1 + 0.134145 * z * z)


def _act64(name, z):
    if name == "none":
        return z
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    return z * (torch.special.ndtr(z) if name == "gelu" else _sigmoid_part(name, z)[0])


def _slope64(name, z):
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return torch.where(z > 0, 1.0, 0.0)
    if name == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    s, du = _sigmoid_part(name, z)
    return s + z * s * (1 - s) * du


def _values64(t, name, scales, dtype):
    v = t[name].float().double() if t[name].dtype == _T["fp8"] else t[name].double()
    if dtype == "fp8":
        return v * t[scales].double()[:, None]
    if dtype == "blocks":
        each = torch.pow(2.0, t[scales].double() - 127).t()
        return v * each.repeat_interleave(BLOCK, dim=1)[:, :v.shape[1]]
    return v


def exact(case, seed):
    kind, t = case["kind"], _inputs(case, seed)
    if kind in ("layer_norm", "layer_norm_backward"):
        d, n = {name: v.double() for name, v in t.items()}, case["cols"]
        h = d["x"] + d["residual"] if kind == "layer_norm" else d["x"]
        var, mean = torch.var_mean(h, dim=1, keepdim=True, correction=0)
        root = torch.sqrt(var + EPS)
        unit = (h - mean) / root
        if kind == "layer_norm_backward":
            g = d["dy"] * d["weight"]
            flat = g.sum(1, keepdim=True) / n + unit * ((g * unit).sum(1, keepdim=True) / n)
            return {"dx": (g - flat) / root + d["residual"], "dweight": (d["dy"] * unit).sum(0), "dbias": d["dy"].sum(0)}
        y = torch.addcmul(d["bias"], unit, d["weight"])
        if case["out"] == "same":
            return {"sum": h, "y": y}
        scales = y.abs().max(dim=1).values / TOP
        return {"sum": h, "y": y / scales[:, None], "scales": scales}
    if kind == "quantize_blocks":
        b = _blocks_of(t["x"].double())
        top = b.abs().max(dim=2).values
        e = torch.ceil(torch.log2(top.clamp(min=1e-300) / TOP))
        # (a logarithm next to a whole number may be rounded over it)
        e = torch.where(top > TOP * torch.pow(2.0, e), e + 1, torch.where(top <= TOP * torch.pow(2.0, e - 1), e - 1, e)).clamp(min=-127.0)
        q = (b / torch.pow(2.0, e)[:, :, None]).reshape(b.shape[0], -1)[:, :case["cols"]]
        return {"q": q, "scales": None}
    if kind == "gated_backward":
        d = {name: v.double() for name, v in t.items()}
        dg = d["dy"] * d["pre_up"] * _slope64(case["act"], d["pre_gate"])
        du = d["dy"] * _act64(case["act"], d["pre_gate"])
        return {"dx": torch.addmm(torch.mm(dg, d["w_gate"]), du, d["w_up"]), "dw_gate": torch.mm(dg.t(), d["x"]),
                "dw_up": torch.mm(du.t(), d["x"]), "dbias_gate": dg.sum(0), "dbias_up": du.sum(0)}
    dtype = "blocks" if kind == "linear_blocks" else case["dtype"]
    x = _values64(t, "x", "x_scales", dtype)
    if kind == "linear_blocks":
        y = _act64(case["act"], torch.addmm(t["bias"].double(), x, _values64(t, "w", "w_scales", dtype).t()))
        return {"y": y + t["residual"].double() if case["residual"] else y}
    g = torch.addmm(t["bias_gate"].double(), x, _values64(t, "w_gate", "gate_scales", dtype).t())
    u = torch.addmm(t["bias_up"].double(), x, _values64(t, "w_up", "up_scales", dtype).t())
    out = {"y": _act64(case["act"], g) * u}
    if case["pre"]:
        out["pre_gate"], out["pre_up"] = g, u
    return out

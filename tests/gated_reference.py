"""The gated feed-forward block's operators in float64 numpy, and 8-bit rows with a scale for each 128 elements: what the kernels are tested
against. Written from the formulas alone; shares no code with the library."""
import numpy as np

import ffn_reference as ref

BLOCK = 128


# ---- block scales --------------------------------------------------------------------------------
def blocks(cols):
    return -(-cols // BLOCK)


def _blocked(x):
    return np.pad(x, ((0, 0), (0, -x.shape[1] % BLOCK))).reshape(x.shape[0], -1, BLOCK)


def scale_of(top):
    """The byte s of the least 2^(s - 127) >= top / 448, s >= 0; 255 where top is not finite."""
    top = np.asarray(top, np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        s = np.clip(np.ceil(np.log2(top / ref.TOP)), -400, 400)
    s = np.where(np.isfinite(top) & (top > 0), s, -400.0)
    s = np.where(top > ref.TOP * np.exp2(s), s + 1, s)  # (a logarithm next to a whole number may be rounded over it)
    s = np.where(top <= ref.TOP * np.exp2(s - 1), s - 1, s)
    return np.where(np.isfinite(top), np.maximum(s + 127, 0), 255).astype(np.uint8)


def scale_value(s):
    return np.where(np.asarray(s) == 255, np.nan, np.exp2(np.asarray(s, np.float64) - 127))


def rows_fp8(x):
    """Rows of x in e4m3 with block scales: (codes, scales [blocks][rows])."""
    b = _blocked(np.asarray(x, np.float64))
    s = scale_of(np.max(np.abs(b), axis=2))
    with np.errstate(invalid="ignore"):
        q = ref.to_fp8((b / scale_value(s)[:, :, None]).reshape(x.shape[0], -1)[:, :x.shape[1]])
    return q, np.ascontiguousarray(s.T)


def values(q, scales):
    """What codes [rows][cols] with block scales [blocks][rows] stand for."""
    each = np.repeat(scale_value(scales).T, BLOCK, axis=1)[:, :q.shape[1]]
    return ref.from_fp8(q).astype(np.float64) * each


# ---- operators -----------------------------------------------------------------------------------
def layer_norm(x, weight, bias, eps, residual=None):
    h = x if residual is None else x + residual
    d = h - np.mean(h, axis=1, keepdims=True)
    y = d / np.sqrt(np.mean(d * d, axis=1, keepdims=True) + eps) * weight
    return h, y if bias is None else y + bias


def layer_norm_grad(dy, h, weight, eps, dh=0.0):
    d = h - np.mean(h, axis=1, keepdims=True)
    s = 1.0 / np.sqrt(np.mean(d * d, axis=1, keepdims=True) + eps)
    g, u = dy * weight, d * s
    dx = s * (g - np.mean(g, axis=1, keepdims=True) - u * np.mean(g * u, axis=1, keepdims=True)) + dh
    return dx, np.sum(dy * u, axis=0), np.sum(dy, axis=0)


def gated(x, w_gate, w_up, bias_gate=None, bias_up=None, activation="silu"):
    g, _ = ref.linear(x, w_gate, bias_gate)
    u, _ = ref.linear(x, w_up, bias_up)
    return g, u, ref.act(activation, g) * u


def gated_grad(dy, x, w_gate, w_up, g, u, activation="silu"):
    dg, du = dy * u * ref.act_slope(activation, g), dy * ref.act(activation, g)
    return dg @ w_gate + du @ w_up, dg.T @ x, du.T @ x, dg.sum(axis=0), du.sum(axis=0)

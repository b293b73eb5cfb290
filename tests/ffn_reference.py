"""The feed-forward block's operators in float64 numpy, and the element types around them: what the
kernels are tested against. Written from the formulas alone; shares no code with the library."""
import math

import numpy as np
from scipy.special import erf, expit

TOP, LEAST, BLOCK = 448.0, 2.0 ** -9, 256
# Rounding to the nearest of 8 significant bits (bf16) moves a value by at most this part of it; of 4 bits (e4m3) by
# at most that, or by half of the smallest value.
BF16, FP8 = 2.0 ** -8, 2.0 ** -4


# ---- element types -------------------------------------------------------------------------------
def to_bf16(x):
    """float -> bf16 bits, to the nearest, ties to even; NaN stays NaN."""
    x = np.asarray(x, np.float32)
    u = x.view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bf16(b):
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def _fp8_values():
    v = np.empty(256, np.float32)
    for c in range(256):
        e, f = (c >> 3) & 15, c & 7
        a = f * 2.0 ** -9 if e == 0 else (8 + f) * 2.0 ** (e - 10)
        v[c] = math.nan if (c & 127) == 127 else (-a if c & 128 else a)
    return v


FP8_VALUES = _fp8_values()


def from_fp8(c):
    return FP8_VALUES[np.asarray(c, np.uint8)]


def to_fp8(x):
    """float -> e4m3 codes, to the nearest, ties to an even code, at most 448; NaN stays NaN."""
    x = np.asarray(x, np.float64)
    pos = FP8_VALUES[:127].astype(np.float64)
    a = np.minimum(np.where(np.isnan(x), 0.0, np.abs(x)), TOP)
    hi = np.clip(np.searchsorted(pos, a), 1, 126)
    lo = hi - 1
    down, up = a - pos[lo], pos[hi] - a
    code = np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi).astype(np.uint8)
    code = np.where(np.isnan(x), np.uint8(127), code)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def rows_fp8(x):
    """Rows of x (float32) in e4m3: (codes, float32 scales). The factor and the products are rounded to float32."""
    top = np.max(np.abs(x), axis=1, initial=0.0).astype(np.float32)
    with np.errstate(divide="ignore", over="ignore", invalid="ignore"):
        f = np.minimum(np.float32(TOP) / top, np.finfo(np.float32).max)
    return to_fp8(np.asarray(x, np.float32) * f[:, None]), top / np.float32(TOP)


# ---- operators -----------------------------------------------------------------------------------
def rms_norm(x, weight, eps, residual=None):
    h = x if residual is None else x + residual
    s = 1.0 / np.sqrt(np.mean(h * h, axis=1, keepdims=True) + eps)
    return h, h * s * weight


def rms_norm_grad(dy, h, weight, eps, dh=0.0):
    s = 1.0 / np.sqrt(np.mean(h * h, axis=1, keepdims=True) + eps)
    g, unit = dy * weight, h * s
    return s * (g - unit * np.mean(g * unit, axis=1, keepdims=True)) + dh, np.sum(dy * unit, axis=0)


_C = math.sqrt(2.0 / math.pi)


def act(name, z):
    if name == "none":
        return z
    if name == "relu":
        return np.where(z > 0, z, 0.0 * z)
    if name == "gelu":
        return 0.5 * z * (1.0 + erf(z / math.sqrt(2.0)))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + np.tanh(_C * (z + 0.044715 * z ** 3)))
    return z * expit(z)


def act_slope(name, z):
    if name == "none":
        return np.ones_like(z)
    if name == "relu":
        return (z > 0).astype(z.dtype)
    if name == "gelu":
        return 0.5 * (1.0 + erf(z / math.sqrt(2.0))) + z * np.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if name == "gelu_tanh":
        t = np.tanh(_C * (z + 0.044715 * z ** 3))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * _C * (1.0 + 0.134145 * z * z)
    s = expit(z)
    return s * (1.0 + z * (1.0 - s))


def linear(x, w, bias=None, activation="none", residual=None):
    z = x @ w.T
    if bias is not None:
        z = z + bias
    y = act(activation, z)
    return z, y if residual is None else y + residual


def linear_grad(dy, x, w, pre, activation="none"):
    dz = dy * act_slope(activation, pre)
    return dz @ w, dz.T @ x, dz.sum(axis=0)


def adamw(p, g, m, v, lr, beta1, beta2, eps, weight_decay, step, grad_scale=1.0):
    g = g * grad_scale
    m, v = beta1 * m + (1 - beta1) * g, beta2 * v + (1 - beta2) * g * g
    mh, vh = m / (1 - beta1 ** step), v / (1 - beta2 ** step)
    return p * (1 - lr * weight_decay) - lr * mh / (np.sqrt(vh) + eps), m, v

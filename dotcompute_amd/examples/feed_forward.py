"""A pre-norm feed-forward block with a linear head, trained and then served, everything on the device:

    n1 = norm(x)   z = n1 W1^T + b1   a = silu(z)   s = x + a W2^T + b2   n2 = norm(s)   y = n2 H^T

Training runs the products in bf16 and steps float32 parameters with AdamW on 8-bit states. The head's epilogue subtracts the
target (it is the head's residual with the sign turned), so that its result is the error e, which is also the gradient of
the loss |e|^2 / 2 by y: no other kernel is needed. Serving runs the same block on a few rows with the weights, and what the
norms write, in 8 bits.

    python -m dotcompute_amd.examples.feed_forward --rows 4096 --width 1024 --hidden 4096 --steps 100
"""
from __future__ import annotations

import argparse
import time

import numpy as np

from dotcompute_amd import hip

ACTIVATION = "silu"


def to_bf16(x: np.ndarray) -> np.ndarray:
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(b: np.ndarray) -> np.ndarray:
    return (b.astype(np.uint32) << 16).view(np.float32)


class Model:
    """The parameters in float32, their bf16 copies, gradients and AdamW states."""

    def __init__(self, ctx: hip.Context, width: int, hidden: int, outputs: int, seed: int = 0):
        self.ctx, self.width, self.hidden, self.outputs = ctx, width, hidden, outputs
        rng = np.random.default_rng(seed)
        shapes = {"norm1": (width,), "w1": (hidden, width), "b1": (hidden,), "w2": (width, hidden), "b2": (width,), "norm2": (width,),
                  "head": (outputs, width)}
        self.copy, self.grad, parts = {}, {}, []
        for name, shape in shapes.items():
            if len(shape) == 2:
                host = rng.normal(size=shape).astype(np.float32) * np.float32(shape[1] ** -0.5)
            else:
                host = np.full(shape, 1.0 if name.startswith("norm") else 0.0, np.float32)
            n = host.size
            blocks = -(-n // hip.ADAMW_BLOCK)
            self.copy[name] = ctx.to_device(to_bf16(host))
            self.grad[name] = ctx.empty(shape, np.uint16 if len(shape) == 2 else np.float32)
            state = {s: ctx.to_device(np.zeros(n, np.uint8)) for s in ("m", "v")}
            state.update({s: ctx.to_device(np.zeros(blocks, np.float32)) for s in ("m_scales", "v_scales")})
            parts.append(dict(param=ctx.to_device(host), grad=self.grad[name], copy=self.copy[name], **state))
        self.tensors = hip.AdamWTensors.of(parts)
        self.steps = 0

    def step(self, lr: float, rows: int) -> None:
        self.steps += 1
        self.ctx.adamw_step(hip.AdamW.of(lr=lr, step=self.steps, grad_scale=1.0 / rows), self.tensors)


class Trainer:
    """The buffers and argument blocks of a step on `x` and `target` (bf16, one row a token)."""

    def __init__(self, model: Model, x: np.ndarray, target: np.ndarray):
        self.model = model
        ctx, p, g = model.ctx, model.copy, model.grad
        rows, (d, h, o) = x.shape[0], (model.width, model.hidden, model.outputs)
        self.rows = rows
        bf16 = lambda cols: ctx.empty((rows, cols), np.uint16)  # noqa: E731
        self.x, target = ctx.to_device(x), ctx.to_device(target ^ np.uint16(0x8000))
        n1, z, a, branch, s, n2 = bf16(d), bf16(h), bf16(h), bf16(d), bf16(d), bf16(d)
        self.error, dn2, ds, da, dn1 = bf16(o), bf16(d), bf16(d), bf16(h), bf16(d)
        self.forward = [
            (ctx.rms_norm, hip.RmsNorm.of(self.x, p["norm1"], n1)),
            (ctx.linear, hip.Linear.of(n1, p["w1"], a, bias=p["b1"], pre=z, activation=ACTIVATION)),
            (ctx.linear, hip.Linear.of(a, p["w2"], branch, bias=p["b2"])),
            (ctx.rms_norm, hip.RmsNorm.of(branch, p["norm2"], n2, residual=self.x, sum=s)),
            (ctx.linear, hip.Linear.of(n2, p["head"], self.error, residual=target)),
        ]
        self.backward = [
            (ctx.linear_backward, hip.LinearGrad.of(self.error, n2, p["head"], dx=dn2, dw=g["head"])),
            (ctx.rms_norm_backward, hip.RmsNormGrad.of(dn2, s, p["norm2"], dx=ds, dweight=g["norm2"])),
            (ctx.linear_backward, hip.LinearGrad.of(ds, a, p["w2"], dx=da, dw=g["w2"], dbias=g["b2"])),
            (ctx.linear_backward, hip.LinearGrad.of(da, n1, p["w1"], pre=z, dx=dn1, dw=g["w1"], dbias=g["b1"], activation=ACTIVATION)),
            (ctx.rms_norm_backward, hip.RmsNormGrad.of(dn1, self.x, p["norm1"], dweight=g["norm1"])),
        ]

    def run(self, lr: float) -> None:
        for call, args in self.forward + self.backward:
            call(args)
        self.model.step(lr, self.rows)

    def loss(self) -> float:
        """Of the last step's forward pass."""
        e = from_bf16(self.error.to_host()).astype(np.float64)
        return float((e * e).sum() / (2 * self.rows))


class Server:
    """The model on at most `rows` rows at a time. In 8 bits its weights are laid out once, here."""

    def __init__(self, model: Model, rows: int, fp8: bool = True):
        ctx, p = model.ctx, model.copy
        d, h, o = model.width, model.hidden, model.outputs
        bf16 = lambda cols: ctx.empty((rows, cols), np.uint16)  # noqa: E731
        self.ctx, self.x, self.y = ctx, bf16(d), ctx.empty((rows, o), np.float32)
        a, branch, s = bf16(h), bf16(d), bf16(d)
        if not fp8:
            n1, n2 = bf16(d), bf16(d)
            self.calls = [
                (ctx.rms_norm, (hip.RmsNorm.of(self.x, p["norm1"], n1),)),
                (ctx.linear, (hip.Linear.of(n1, p["w1"], a, bias=p["b1"], activation=ACTIVATION),)),
                (ctx.linear, (hip.Linear.of(a, p["w2"], branch, bias=p["b2"]),)),
                (ctx.rms_norm, (hip.RmsNorm.of(branch, p["norm2"], n2, residual=self.x, sum=s),)),
                (ctx.linear, (hip.Linear.of(n2, p["head"], self.y),)),
            ]
            return
        codes = lambda r, c: (ctx.empty((r, c), np.uint8), ctx.empty(r, np.float32))  # noqa: E731
        w = {name: codes(*p[name].shape) for name in ("w1", "w2", "head")}
        for name, (q, scales) in w.items():
            ctx.quantize_fp8(p[name], q, scales)
        (n1, s1), (aq, sa), (n2, s2) = codes(rows, d), codes(rows, h), codes(rows, d)
        self.calls = [
            (ctx.rms_norm, (hip.RmsNorm.of(self.x, p["norm1"], n1, scales=s1),)),
            (ctx.linear, (hip.Linear.of(n1, w["w1"][0], a, bias=p["b1"], x_scales=s1, w_scales=w["w1"][1], activation=ACTIVATION),)),
            (ctx.quantize_fp8, (a, aq, sa)),
            (ctx.linear, (hip.Linear.of(aq, w["w2"][0], branch, bias=p["b2"], x_scales=sa, w_scales=w["w2"][1]),)),
            (ctx.rms_norm, (hip.RmsNorm.of(branch, p["norm2"], n2, residual=self.x, sum=s, scales=s2),)),
            (ctx.linear, (hip.Linear.of(n2, w["head"][0], self.y, x_scales=s2, w_scales=w["head"][1]),)),
        ]

    def run(self) -> None:
        for call, args in self.calls:
            call(*args)

    def __call__(self, x: np.ndarray) -> np.ndarray:
        self.x.copy_from(x)
        self.run()
        return self.y.to_host()


def data(rows: int, width: int, outputs: int, seed: int = 1) -> tuple:
    """Rows and what a fixed random function of them asks for, in bf16."""
    rng = np.random.default_rng(seed)
    x = from_bf16(to_bf16(rng.normal(size=(rows, width))))
    w = np.random.default_rng(2).normal(size=(outputs, width)).astype(np.float32) * np.float32(width ** -0.5)
    return to_bf16(x), to_bf16(np.tanh(x @ w.T))


def main() -> None:
    args = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("rows", 4096), ("width", 1024), ("hidden", 4096), ("outputs", 256), ("steps", 100), ("serve", 8)):
        args.add_argument("--" + name, type=int, default=value)
    args.add_argument("--lr", type=float, default=1e-3)
    o = args.parse_args()
    with hip.Context() as ctx:
        model = Model(ctx, o.width, o.hidden, o.outputs)
        x, target = data(o.rows, o.width, o.outputs)
        trainer = Trainer(model, x, target)
        for t in range(o.steps + 1):
            trainer.run(o.lr)
            if t % max(1, o.steps // 5) == 0:
                print(f"step {t}: loss {trainer.loss():.4f}", flush=True)
        timed = time.perf_counter()
        for _ in range(20):
            trainer.run(o.lr)
        ctx.synchronize()
        print(f"a step: {(time.perf_counter() - timed) / 20 * 1e6:.0f} us")
        results = {}
        for fp8 in (False, True):
            server = Server(model, o.serve, fp8)
            results[fp8] = server(x[:o.serve])
            timed = time.perf_counter()
            for _ in range(200):
                server.run()
            ctx.synchronize()
            print(f"{o.serve} rows {'in 8 bits' if fp8 else 'in bf16'}: {(time.perf_counter() - timed) / 200 * 1e6:.0f} us")
        off = np.linalg.norm(results[True] - results[False]) / np.linalg.norm(results[False])
        print(f"8 bits against bf16: {off:.4f} apart")


if __name__ == "__main__":
    main()

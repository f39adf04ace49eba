"""Plain implementations in 64 bits of the mixture of experts, and layers for its tests."""
import math

import numpy as np

from helpers import GGML_ID, random_valid_blocks


def dequantised(fmt, raw, *shape):
    from oracle import oracle
    return oracle.dequantize(GGML_ID[fmt], raw, int(np.prod(shape))).astype(np.float64).reshape(shape)


def activate(name, v):
    from scipy.special import expit, ndtr
    with np.errstate(over="ignore"):
        return {None: lambda z: z, "none": lambda z: z, "relu": lambda z: np.maximum(z, 0), "silu": lambda z: z / (1 + np.exp(-z)), "gelu": lambda z: z * ndtr(z),
                "gelu_tanh": lambda z: z * expit(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))}[name](v)


def route(x, w, used, gating="softmax", normalise=True, scale=1.0, bias=None):
    l = np.asarray(x, dtype=np.float64) @ np.asarray(w, dtype=np.float64).T
    with np.errstate(over="ignore", invalid="ignore"):
        p = np.exp(l - l.max(1, keepdims=True))
        p = p / p.sum(1, keepdims=True) if gating == "softmax" else 1 / (1 + np.exp(-l))
        by = l if bias is None else p + np.asarray(bias, dtype=np.float64)
        by = np.where(np.isnan(by), -np.inf, by)
        ids = np.argsort(-by, axis=1, kind="stable")[:, :used]
        chosen = np.take_along_axis(p, ids, 1)
        return ids, scale * (chosen / chosen.sum(1, keepdims=True) if normalise else chosen)


class Layer:
    """Random experts, their values and the package's tensors of them."""

    def __init__(self, rng, experts, used, d, ffn, up="Q4_K", down="Q6_K", gate=None, activation="silu", **routing):
        self.experts, self.used, self.d, self.ffn, self.activation, self.routing = experts, used, d, ffn, activation, routing
        self.formats = (gate or up, up, down)
        self.tolerance = tolerance(self.formats)
        self.shapes = ((experts, ffn, d), (experts, ffn, d), (experts, d, ffn))
        self.raw = [random_valid_blocks(rng, f, s[0] * s[1], s[2]) for f, s in zip(self.formats, self.shapes)]
        # (random blocks of any format: the rows brought to about one, so that the gates are neither open nor shut)
        self.values = [dequantised(f, r, *s) for f, r, s in zip(self.formats, self.raw, self.shapes)]
        self.size = 1.0 / (np.sqrt((self.values[0] ** 2).mean()) * math.sqrt(d))
        self.router = (rng.standard_normal((experts, d)) / math.sqrt(d)).astype(np.float32)

    def input(self, rng, tokens):
        return (self.size * rng.standard_normal((tokens, self.d))).astype(np.float32)

    def make(self, jn):
        w = [jn.Tensor.quantized(jn.DType[f], r, *s) for f, r, s in zip(self.formats, self.raw, self.shapes)]
        scaled = self.router / self.size
        r = jn.Router(scaled, self.used, gating=self.routing.get("gating", "softmax"), normalise=self.routing.get("normalise", True),
                      scale=self.routing.get("scale", 1.0), selection_bias=self.routing.get("bias"))
        return jn.Moe(r, *w, activation=self.activation)

    def route(self, x):
        return route(x, self.router / self.size, self.used, **self.routing)

    def experts_of(self, x, ids, weights, residual=None):
        x = np.asarray(x, dtype=np.float64)
        y = np.zeros_like(x) if residual is None else np.asarray(residual, dtype=np.float64).copy()
        for t in range(len(x)):
            for e, w in zip(ids[t], weights[t]):
                if 0 <= e < self.experts:
                    h = activate(self.activation, self.values[0][e] @ x[t]) * (self.values[1][e] @ x[t])
                    y[t] += w * (self.values[2][e] @ h)
        return y


# How many times the terms of a product with an offset are what they leave (2-norm): quants around 32, 8 or 7.5 less that offset, 2 at most for blocks of
# quants that are spread over their whole range.  Q3_K blocks run as Q6_K blocks whose quants are 28 to 35: sqrt(mean of q^2 / mean of (q - 32)^2) =
# sqrt(1029.5 / 5.5) = 13.7 with q spread evenly.
OFFSET = {"Q3_K": 14}


def offset(fmt):
    return OFFSET.get(fmt, 4)


# How far a layer may be off (2-norm over 2-norm).  The operands of a product hold a value to 2^-20 of itself (two FP16 parts, both cut) or to 2^-22 of the
# largest of 64 (three bytes), FP32 sums of some hundred terms add as much again, both count as often as offset() says; three products follow one
# another, errors of the first two meet in one.
def tolerance(formats):
    return 2 * sum(offset(f) for f in formats) * 2.0 ** -22


def close(got, want, tolerance):
    got, want = np.asarray(got, dtype=np.float64), np.asarray(want, dtype=np.float64)
    norm = np.linalg.norm(want)
    assert np.isfinite(got).all()
    off = np.linalg.norm(got - want)
    assert off <= tolerance * norm, (off / norm, tolerance)
    # one value among many: its share of the norm is about one in the root of their number
    assert np.abs(got - want).max() <= 40 * tolerance * norm / math.sqrt(want.size)

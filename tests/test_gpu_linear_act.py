"""Linears with bias, activation and residual against plain implementations in 64 bits."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import experts_reference as ref
from helpers import random_valid_blocks

pytestmark = pytest.mark.gpu

ACTIVATIONS = [None, "relu", "silu", "gelu", "gelu_tanh"]


@pytest.fixture(scope="module")
def jn():
    import jitnn_amd
    jitnn_amd.init()
    return jitnn_amd


class Case:
    def __init__(self, rng, fmt, n, k, rows, bias=True, residual=True):
        self.fmt, self.n, self.k, self.rows = fmt, n, k, rows
        self.raw = random_valid_blocks(rng, fmt, n, k)
        self.values = ref.dequantised(fmt, self.raw, n, k)
        size = 1.0 / (np.sqrt((self.values ** 2).mean()) * math.sqrt(k))
        self.x = (2 * size * rng.standard_normal((rows, k))).astype(np.float32)
        self.bias = rng.standard_normal(n).astype(np.float32) if bias else None
        self.residual = rng.standard_normal((rows, n)).astype(np.float32) if residual else None

    def weight(self, jn):
        return jn.Tensor.quantized(jn.DType[self.fmt], self.raw, self.n, self.k)

    def want(self, act):
        z = self.x.astype(np.float64) @ self.values.T
        y = ref.activate(act, z if self.bias is None else z + self.bias)
        return y if self.residual is None else y + self.residual

    # Up to 64 rows a sum is off by some 2^-20 (2-norm; ref.offset says how many times its terms are what they leave, FP32 sums add as much again), more rows round both operands to FP16, 2^-11 each at most.  An activation's slope is at most 1.13, and a gate that shuts leaves
    # less than went in, so errors count against the larger of what goes in and what comes out.
    def check(self, got, act):
        z = self.x.astype(np.float64) @ self.values.T
        tol = 2 * ref.offset(self.fmt) * 2.0 ** -22 if self.rows <= 64 else 2 * 2.0 ** -11
        want = self.want(act)
        norm = max(np.linalg.norm(want), np.linalg.norm(z))
        off = np.abs(got - want)
        assert np.isfinite(got).all()
        assert np.linalg.norm(off) <= 1.13 * tol * norm, (np.linalg.norm(off) / norm, tol)
        assert off.max() <= 40 * tol * norm / math.sqrt(want.size)


def call(jn, w, x, bias, act, residual, n, stream=0, shift=0):
    """On device memory; shift: outputs and residuals that are aligned to 4 bytes only."""
    t = [None if a is None else torch.as_tensor(a).cuda() for a in (x, bias)]
    y = torch.full((x.shape[0] * n + 8,), 7.0, device="cuda")
    r = None
    if residual is not None:
        r = torch.full((residual.size + 8,), 9.0, device="cuda")
        r[shift:shift + residual.size] = torch.as_tensor(residual).cuda().reshape(-1)
    jn.linear_dev(w, t[0].data_ptr(), x.shape[0], y.data_ptr() + 4 * shift, 0 if bias is None else t[1].data_ptr(), act, 0 if r is None else r.data_ptr() + 4 * shift, stream)
    torch.cuda.synchronize()
    assert (y[:shift] == 7).all() and (y[shift + x.shape[0] * n:] == 7).all()
    return y[shift:shift + x.shape[0] * n].reshape(x.shape[0], n).cpu().numpy()


@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("fmt", ["Q8_0", "Q4_0", "Q4_1", "Q4_K", "Q5_K", "Q6_K", "Q5_0", "Q5_1", "Q2_K", "Q3_K"])
@pytest.mark.parametrize("rows", [1, 2, 4, 7, 13, 40, 64, 96, 600])
def test_formats(jn, fmt, act, rows):
    rng = np.random.default_rng(rows)
    c = Case(rng, fmt, 272, 1024, rows)
    c.check(call(jn, c.weight(jn), c.x, c.bias, act, c.residual, c.n), act)


@pytest.mark.parametrize("fmt,n,k", [("Q8_0", 4096, 4096), ("Q4_0", 250, 96), ("Q4_1", 1000, 5120 + 32), ("Q6_K", 128, 14336), ("Q4_K", 3, 256), ("Q8_0", 1, 32), ("Q5_K", 61, 5120),
                                     ("Q4_0", 400, 1504), ("Q5_1", 100, 288), ("Q2_K", 36, 4608), ("Q4_K", 5000, 2048), ("Q8_0", 777, 17408)])
@pytest.mark.parametrize("rows", [1, 3, 8, 9, 31, 64, 70])
@pytest.mark.parametrize("bias,residual", [(True, True), (False, True), (True, False), (False, False)])
def test_shapes(jn, fmt, n, k, rows, bias, residual):
    rng = np.random.default_rng(n + k)
    c = Case(rng, fmt, n, k, rows, bias, residual)
    c.check(call(jn, c.weight(jn), c.x, c.bias, "silu", c.residual, n, shift=1), "silu")


@pytest.mark.parametrize("rows", [1, 2, 6, 20, 64, 100])
def test_without_an_epilogue_it_is_the_linear(jn, rows):
    from jitnn_amd import _lib
    rng = np.random.default_rng(rows)
    c = Case(rng, "Q4_K", 512, 2048, rows)
    w = c.weight(jn)
    x, b, y = torch.as_tensor(c.x).cuda(), torch.as_tensor(c.bias).cuda(), torch.empty(rows, c.n, device="cuda")
    _lib.check(_lib.lib.jitnn_hip_linear_dev(w.handle, x.data_ptr(), rows, b.data_ptr(), y.data_ptr(), None), "jitnn_hip_linear_dev")
    torch.cuda.synchronize()
    assert np.array_equal(call(jn, w, c.x, c.bias, None, None, c.n), y.cpu().numpy())


@pytest.mark.parametrize("rows", [1, 4, 8, 30, 64, 200])
@pytest.mark.parametrize("fmt,k", [("Q4_K", 1024), ("Q8_0", 1056), ("Q6_K", 12288)])
def test_host_streams_and_graphs(jn, fmt, k, rows):
    rng = np.random.default_rng(rows)
    cases = [Case(rng, fmt, 300, k, rows) for _ in range(3)]
    w = cases[0].weight(jn)
    want = [call(jn, w, c.x, c.bias, "gelu", c.residual, 300) for c in cases]
    host = jn.Gguf.linear(jn.Tensor.of(cases[0].x), w, jn.Tensor.of(cases[0].bias), activation="gelu", residual=jn.Tensor.of(cases[0].residual))
    assert np.array_equal(host.numpy(), want[0])
    t = [torch.as_tensor(a).cuda() for a in (cases[0].x, cases[0].bias, cases[0].residual)]
    y = torch.empty(rows, 300, device="cuda")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    jn.linear_dev(w, t[0].data_ptr(), rows, y.data_ptr(), t[1].data_ptr(), "gelu", t[2].data_ptr(), stream.cuda_stream)
    torch.cuda.synchronize()
    assert np.array_equal(y.cpu().numpy(), want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        jn.linear_dev(w, t[0].data_ptr(), rows, y.data_ptr(), t[1].data_ptr(), "gelu", t[2].data_ptr(), torch.cuda.current_stream().cuda_stream)
    for c, v in zip(cases, want):
        for dst, src in zip(t, (c.x, c.bias, c.residual)):
            dst.copy_(torch.as_tensor(src))
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(y.cpu().numpy(), v)
        assert np.array_equal(call(jn, w, cases[2].x, cases[2].bias, "gelu", cases[2].residual, 300), want[2])


@pytest.mark.parametrize("rows", [1, 3, 8, 20, 100])
def test_activations_of_odd_numbers(jn, rows):
    """Sums that are infinite or no number, far out on both sides of an activation, and zero."""
    w = jn.Tensor.quantized(jn.DType.Q8_0, np.zeros(34 * 16 * 8, dtype=np.uint8), 16, 256)
    bias = np.array([np.nan, np.inf, 1e30, 100, 20, 5, 1e-3, 0, -1e-3, -5, -9, -20, -100, -1e30, 1, -1], dtype=np.float32)
    x = np.ones((rows, 256), dtype=np.float32)
    for act in ACTIVATIONS:
        got = call(jn, w, x, bias, act, None, 16)
        assert (got == got[0]).all(axis=0)[1:].all()
        want = ref.activate(act, bias.astype(np.float64))
        assert np.isnan(got[0, 0]) and got[0, 1] == np.inf
        # An activation is some roundings of its own, 2^-21, and exp of an exponent that is off by two roundings of itself: -v for SiLU, about -v^2 / 2 for the
        # normal distribution's tail (its argument, off by 2^-24 and 1.7e-8 of itself, counts squared: 2^-23 v^2), -2 u for the form with tanh.
        v = bias[2:].astype(np.float64)
        exponent = {None: 0 * v, "relu": 0 * v, "silu": np.abs(v), "gelu": v * v, "gelu_tanh": np.abs(v) * (1.6 + 0.0714 * v * v)}[act]
        assert (np.abs(got[0, 2:] - want[2:]) <= (2.0 ** -21 + 2.0 ** -23 * np.minimum(exponent, 1e3)) * np.abs(want[2:]) + 1e-37).all(), (act, got[0], want)


def test_refusals(jn):
    from jitnn_amd import _lib
    rng = np.random.default_rng(0)
    c = Case(rng, "Q8_0", 64, 64, 4)
    w = c.weight(jn)
    x, y = torch.as_tensor(c.x).cuda(), torch.full((8, 64), 5.0, device="cuda")
    p, q = x.data_ptr(), y.data_ptr()
    for bad in (dict(x_ptr=0), dict(y_ptr=0), dict(rows=0), dict(rows=-3), dict(activation="tanh"), dict(residual_ptr=q), dict(residual_ptr=q + 4 * 255), dict(residual_ptr=q - 4)):
        with pytest.raises(ValueError):
            jn.linear_dev(**{**dict(w=w, x_ptr=p, rows=4, y_ptr=q), **bad})
    torch.cuda.synchronize()
    assert (y == 5).all()
    jn.linear_dev(w, p, 4, q, residual_ptr=q + 4 * 256)  # right behind it
    torch.cuda.synchronize()
    assert (y[4:] == 5).all()
    call_c = _lib.lib.jitnn_hip_linear_act_dev
    assert call_c(None, p, 1, None, 0, None, q, None) == _lib.EINVAL and call_c(w.handle, p, 1, None, 5, None, q, None) == _lib.EINVAL
    assert call_c(w.handle, p, 1, None, -1, None, q, None) == _lib.EINVAL
    t = jn.Tensor.of
    for bad in (dict(residual=t(np.zeros((4, 63)))), dict(residual=t(np.zeros(64))), dict(activation="x"), dict(bias=t(np.zeros(3)))):
        with pytest.raises(ValueError):
            jn.Gguf.linear(t(c.x), w, **bad)

"""Mixtures of experts on quantised weights (jitnn_hip_router_*, jitnn_hip_moe_*): the router, the experts' products, the whole layer.  `*_ptr` arguments are
addresses in device memory, `stream_ptr` a hipStream_t (0: the null stream); those calls only enqueue.  What each does, checks and leaves alone is said in
include/jitnn_hip.h.  The reference has no such layer."""
from __future__ import annotations

import ctypes as C
import weakref

import numpy as np

from . import _lib
from .serving import DeviceArray
from .tensor import Tensor

GATINGS = {"softmax": 0, "sigmoid": 1}


def _bytes(n: int, what: str) -> int:
    if n < 0:
        _lib.check(n, what)
    return n


class Router:
    """Which `used` of the experts a token goes to, and with which weights: weights [experts, d_model], gating "softmax" or "sigmoid" of the logits,
    normalise: the chosen ones' weights sum to `scale`; selection_bias [experts] is added for the choice alone."""

    def __init__(self, weights, used: int, gating: str = "softmax", normalise: bool = True, scale: float = 1.0, selection_bias=None):
        w = np.ascontiguousarray(weights, dtype=np.float32)
        if w.ndim != 2:
            raise ValueError(f"router weights of shape {w.shape} ([experts, d_model])")
        if gating not in GATINGS:
            raise ValueError(f"gating {gating!r} ('softmax' and 'sigmoid' are built)")
        bias = None if selection_bias is None else np.ascontiguousarray(selection_bias, dtype=np.float32).reshape(-1)
        if bias is not None and bias.size != w.shape[0]:
            raise ValueError(f"{bias.size} selection biases for {w.shape[0]} experts")
        _lib.init()
        fp, h = C.POINTER(C.c_float), C.c_void_p()
        _lib.check(_lib.lib.jitnn_hip_router_create(w.shape[0], w.shape[1], used, GATINGS[gating], bool(normalise), scale, w.ctypes.data_as(fp),
                                                    None if bias is None else bias.ctypes.data_as(fp), C.byref(h)), "jitnn_hip_router_create")
        self.experts, self.d_model, self.used, self._h = w.shape[0], w.shape[1], used, h
        weakref.finalize(self, _lib.lib.jitnn_hip_router_free, h)

    @property
    def handle(self):
        return self._h

    def workspace(self, tokens: int) -> int:
        """Bytes of device memory that route_dev needs."""
        return _bytes(_lib.lib.jitnn_hip_router_workspace(self._h, tokens), "jitnn_hip_router_workspace")

    def route_dev(self, x_ptr: int, tokens: int, ids_ptr: int, weights_ptr: int, workspace_ptr: int = 0, workspace_bytes: int = 0, stream_ptr: int = 0) -> None:
        """ids (32-bit whole numbers) and weights [tokens, used] of x [tokens, d_model]."""
        rc = _lib.lib.jitnn_hip_router_dev(self._h, x_ptr, tokens, ids_ptr, weights_ptr, workspace_ptr, workspace_bytes, stream_ptr)
        if rc:
            _lib.check(rc, "jitnn_hip_router_dev")

    def route(self, x):
        """The same on a host array: (ids, weights)."""
        a = np.ascontiguousarray(x, dtype=np.float32).reshape(-1, self.d_model)
        n, count = self.workspace(len(a)), len(a) * self.used
        xd, ids, weights, space = DeviceArray(a.size, np.float32).put(a), DeviceArray(count, np.int32), DeviceArray(count, np.float32), DeviceArray(n, np.uint8)
        self.route_dev(xd.ptr, len(a), ids.ptr, weights.ptr, space.ptr, n)
        return ids.get(count).reshape(-1, self.used), weights.get(count).reshape(-1, self.used)


class Moe:
    """A layer of experts: gate and up [experts, ffn, d_model], down [experts, d_model, ffn] in block formats (kept alive by this object)."""

    def __init__(self, router: Router, gate: Tensor, up: Tensor, down: Tensor, activation: str | None = "silu"):
        e, d = router.experts, router.d_model
        for w, what in ((gate, "gate"), (up, "up"), (down, "down")):
            if w.rank() != 3 or w.dim(0) != e or w.handle is None:
                raise ValueError(f"{what} of shape {list(w.shape())}: block-quantised experts [{e}, rows, values]")
        if gate.shape() != up.shape() or gate.dim(2) != d or down.dim(1) != d or down.dim(2) != gate.dim(1):
            raise ValueError(f"experts of shapes {list(gate.shape())}, {list(up.shape())}, {list(down.shape())} on {d} values")
        h = C.c_void_p()
        _lib.check(_lib.lib.jitnn_hip_moe_create(router.handle, gate.handle, up.handle, down.handle, _lib.activation_id(activation), C.byref(h)), "jitnn_hip_moe_create")
        self.router, self.d_model, self.ffn, self._keep, self._h = router, d, gate.dim(1), (gate, up, down), h
        weakref.finalize(self, _lib.lib.jitnn_hip_moe_free, h)

    @property
    def handle(self):
        return self._h

    def workspace(self, tokens: int) -> int:
        """Bytes of device memory that layer_dev and experts_dev need."""
        return _bytes(_lib.lib.jitnn_hip_moe_workspace(self._h, tokens), "jitnn_hip_moe_workspace")

    def layer_dev(self, x_ptr: int, tokens: int, y_ptr: int, workspace_ptr: int, workspace_bytes: int, residual_ptr: int = 0, stream_ptr: int = 0) -> None:
        """y [tokens, d_model] = residual + the experts that the router chooses, each times its weight; y may be x or the residual."""
        rc = _lib.lib.jitnn_hip_moe_dev(self._h, x_ptr, tokens, residual_ptr or None, y_ptr, workspace_ptr, workspace_bytes, stream_ptr)
        if rc:
            _lib.check(rc, "jitnn_hip_moe_dev")

    def experts_dev(self, x_ptr: int, tokens: int, ids_ptr: int, weights_ptr: int, y_ptr: int, workspace_ptr: int, workspace_bytes: int, residual_ptr: int = 0,
                    stream_ptr: int = 0) -> None:
        """The same for ids and weights [tokens, used] that somebody else chose."""
        rc = _lib.lib.jitnn_hip_moe_experts_dev(self._h, x_ptr, tokens, ids_ptr, weights_ptr, residual_ptr or None, y_ptr, workspace_ptr, workspace_bytes, stream_ptr)
        if rc:
            _lib.check(rc, "jitnn_hip_moe_experts_dev")

    def layer(self, x, residual=None) -> np.ndarray:
        """layer_dev on host arrays."""
        a = np.ascontiguousarray(x, dtype=np.float32).reshape(-1, self.d_model)
        r = None if residual is None else np.ascontiguousarray(residual, dtype=np.float32).reshape(a.shape)
        n = self.workspace(len(a))
        xd, yd, space = DeviceArray(a.size, np.float32).put(a), DeviceArray(a.size, np.float32), DeviceArray(n, np.uint8)
        if r is not None:
            yd.put(r)
        self.layer_dev(xd.ptr, len(a), yd.ptr, space.ptr, n, yd.ptr if r is not None else 0)
        return yd.get(a.size).reshape(np.shape(x))

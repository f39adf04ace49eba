"""What the router and the layer of experts refuse before any device is needed."""
import ctypes as C

import numpy as np
import pytest


@pytest.fixture(scope="module")
def lib():
    from jitnn_amd import _lib
    return _lib


def test_router_arguments(lib):
    w = np.zeros((8, 16), dtype=np.float32)
    p = w.ctypes.data_as(C.POINTER(C.c_float))
    h = C.c_void_p()

    def create(experts=8, d=16, used=2, gating=0, scale=1.0, weights=p, out=h):
        return lib.lib.jitnn_hip_router_create(experts, d, used, gating, 1, scale, weights, None, None if out is None else C.byref(out))

    for bad in (dict(experts=0), dict(experts=513), dict(experts=-1), dict(used=0), dict(used=9), dict(d=0), dict(d=18), dict(d=-4), dict(gating=2), dict(gating=-1),
                dict(scale=float("inf")), dict(weights=None), dict(out=None), dict(experts=100, used=65)):
        assert create(**bad) == lib.EINVAL, bad
    assert h.value is None
    f = lib.lib
    assert f.jitnn_hip_router_free(None) == 0 and f.jitnn_hip_moe_free(None) == 0
    assert f.jitnn_hip_router_workspace(None, 1) == lib.EINVAL and f.jitnn_hip_moe_workspace(None, 1) == lib.EINVAL
    assert f.jitnn_hip_router_dev(None, 16, 1, 16, 16, 16, 16, None) == lib.EINVAL
    assert f.jitnn_hip_moe_dev(None, 16, 1, None, 16, 16, 16, None) == lib.EINVAL
    assert f.jitnn_hip_moe_experts_dev(None, 16, 1, 16, 16, None, 16, 16, 16, None) == lib.EINVAL
    assert f.jitnn_hip_moe_create(None, None, None, None, 0, C.byref(h)) == lib.EINVAL and f.jitnn_hip_moe_create(None, None, None, None, 0, None) == lib.EINVAL


def test_host_side():
    import jitnn_amd
    with pytest.raises(ValueError, match="gating"):
        jitnn_amd.Router(np.zeros((4, 8)), 2, gating="hash")
    with pytest.raises(ValueError, match="shape"):
        jitnn_amd.Router(np.zeros(8), 2)
    with pytest.raises(ValueError, match="biases"):
        jitnn_amd.Router(np.zeros((4, 8)), 2, selection_bias=np.zeros(5))
    from jitnn_amd._lib import activation_id
    assert activation_id(None) == 0 and activation_id("gelu_tanh") == 4
    with pytest.raises(ValueError, match="activation"):
        activation_id("swish")

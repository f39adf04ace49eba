"""Layers of experts at their borders: matrices beyond 2 GiB whose rows are no whole columns, inputs next to a power of two and to the largest FP32 value, overlapping buffers."""
import numpy as np
import pytest
import torch

import experts_reference as ref
from test_gpu_experts import Call

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def jn():
    import jitnn_amd
    jitnn_amd.init()
    return jitnn_amd


def test_ragged_rows_of_weights_beyond_31_bits(jn):
    """Matrices of more than 2 GiB whose rows end inside a column of 256 values: the experts at their start, which stand further than 31 bits in front of the matrix's end, as well as the last ones."""
    experts, d, ffn, used, tokens = 128, 2880, 5760, 2, 70
    gen = torch.Generator(device="cuda").manual_seed(2)
    scales = torch.tensor([0.01], dtype=torch.float16).view(torch.uint8).cuda()
    shapes, matrices = ((ffn, d), (ffn, d), (d, ffn)), []
    for _ in shapes:
        raw = torch.empty(experts * d * ffn // 32, 34, dtype=torch.uint8, device="cuda").random_(0, 256, generator=gen)
        raw[:, :2] = scales
        matrices.append(raw)
    assert matrices[0].numel() > 1 << 31
    router = jn.Router(np.zeros((experts, d), dtype=np.float32), used)
    moe = jn.Moe(router, *(jn.Tensor.wrap_dev(jn.DType.Q8_0, m.data_ptr(), experts, *s) for m, s in zip(matrices, shapes)))
    some = [0, 1, 5, 60, 126, 127]
    values = {e: [m.reshape(experts, -1, 34)[e, :, 2:].contiguous().view(torch.int8).double().mul(float(np.float16(0.01))).reshape(s).cpu().numpy() for m, s in zip(matrices, shapes)]
              for e in some}
    rng = np.random.default_rng(3)
    x = (0.025 * rng.standard_normal((tokens, d))).astype(np.float32)  # (the quants' mean square is 74^2: rows of about one)
    ids = np.array(some)[rng.integers(0, len(some), (tokens, used))]
    weights = rng.standard_normal((tokens, used)).astype(np.float32)
    want = np.zeros(x.shape)
    for e, (gate, up, down) in values.items():
        share = np.where(ids == e, weights, 0).sum(1, keepdims=True, dtype=np.float64)
        want += share * ((ref.activate("silu", x.astype(np.float64) @ gate.T) * (x.astype(np.float64) @ up.T)) @ down.T)
    ref.close(Call(moe, x, None, ids, weights).result(), want, ref.tolerance(["Q8_0"] * 3))

"""Layers of experts at their borders: matrices beyond 2 GiB whose rows are no whole columns, inputs next to a power of two and to the largest FP32 value, outputs that overlap."""
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


def q6_k(quants):
    """Q6_K blocks of whole numbers -32..31, [rows, a multiple of 256]: every scale 1."""
    q = (np.asarray(quants, dtype=np.int32) + 32).astype(np.uint8).reshape(-1, 2, 4, 32)  # [block, half, quarter, place]
    low = np.stack([q[:, :, 0] & 15 | (q[:, :, 2] & 15) << 4, q[:, :, 1] & 15 | (q[:, :, 3] & 15) << 4], axis=2)
    high = q[:, :, 0] >> 4 | (q[:, :, 1] >> 4) << 2 | (q[:, :, 2] >> 4) << 4 | (q[:, :, 3] >> 4) << 6
    n = len(q)
    return np.concatenate([low.reshape(n, 128), high.reshape(n, 64), np.ones((n, 16), dtype=np.uint8), np.full((n, 1), np.float16(1)).view(np.uint8)], axis=1).astype(np.uint8)


def q8_0(quants, scale):
    q = np.asarray(quants, dtype=np.int8).reshape(-1, 32)
    return np.concatenate([np.full((len(q), 1), np.float16(scale)).view(np.uint8), q.view(np.uint8)], axis=1)


def one_expert(jn, d, fmt, gate, up, down):
    router = jn.Router(np.zeros((1, d), dtype=np.float32), 1)
    return jn.Moe(router, *(jn.Tensor.quantized(jn.DType[fmt], w.reshape(-1), 1, d, d) for w in (gate, up, down)), activation=None)


@pytest.mark.parametrize("tokens", [1, 3])
def test_inputs_next_to_a_power_of_two(jn, tokens):
    """A value that rounds up to the next power of two beside values of half a step: what is rounded counts with the quant less its offset of 32, so sixteen values of half a step, 2^-22 of
    the largest each, that meet a weight of 1 may go missing, and no more."""
    d = 256
    quants = np.zeros((3, d, d), dtype=np.int32)
    quants[0, :, 32:48] = 1  # gate: the sixteen small values
    quants[1, :, 0] = 1      # up: the largest one
    np.fill_diagonal(quants[2], 1)
    raw = [q6_k(q) for q in quants]
    assert all(np.array_equal(ref.dequantised("Q6_K", r.reshape(-1), d, d), q) for r, q in zip(raw, quants))
    x = np.zeros((tokens, d), dtype=np.float32)
    x[:, 0] = np.nextafter(np.float32(2), np.float32(0))
    x[:, 32:48] = 2.0 ** -21
    got = Call(one_expert(jn, d, "Q6_K", *raw), x, None, np.zeros((tokens, 1)), np.ones((tokens, 1))).result()
    want = x[:, :1].astype(np.float64) * 16 * 2.0 ** -21
    assert (np.abs(got - want) <= 2 * 16 * (2 * 2.0 ** -22) * (1 + 2.0 ** -18)).all(), got[0, 0]


@pytest.mark.parametrize("tokens", [1, 5, 70])
@pytest.mark.parametrize("bits", [0x7f7fffff, 0x7f7ffffe, 0x7f7ffffd, 0xff7fffff])
def test_inputs_next_to_the_largest_value(jn, bits, tokens):
    """The largest FP32 values are finite, and so are the products that they make."""
    d = 128
    quants = np.zeros((3, d, d), dtype=np.int32)
    quants[0, :, 0] = 1   # gate: the large value
    quants[1, :, 70] = 1  # up: a small one
    np.fill_diagonal(quants[2], 1)
    scales = (2.0 ** -24, 1.0, 1.0)
    raw = [q8_0(q, s) for q, s in zip(quants, scales)]
    x = np.zeros((tokens, d), dtype=np.float32)
    x[:, 0] = np.array([bits], dtype=np.uint32).view(np.float32)[0]
    x[:, 70] = 2.0 ** -60
    got = Call(one_expert(jn, d, "Q8_0", *raw), x, None, np.zeros((tokens, 1)), np.ones((tokens, 1))).result()
    # (the matrix cores' route scales 256 values by their largest and keeps two FP16 parts of each: the small one beside it, 2^-188 of it, is zero there, and so are the products)
    want = np.full((tokens, d), x[0, 0].astype(np.float64) * 2.0 ** -84)
    assert np.isfinite(got).all()
    if tokens <= 5:
        ref.close(got, want, ref.tolerance(["Q8_0"] * 3))


@pytest.mark.parametrize("tokens", [4, 70])
def test_outputs_that_overlap_in_part(jn, tokens):
    """An output shifted against the input or the residual would be written where rows are still to be read; beside them it is an output like any other."""
    d = 256
    layer = ref.Layer(np.random.default_rng(1), 4, 2, d, 512)
    moe = layer.make(jn)
    n = moe.workspace(tokens)
    buffer, ws = torch.full((3 * tokens, d), 3.0, device="cuda"), torch.empty(n, dtype=torch.uint8, device="cuda")
    other, ids, weights = torch.zeros(tokens, d, device="cuda"), torch.zeros(tokens, 2, dtype=torch.int32, device="cuda"), torch.ones(tokens, 2, device="cuda")

    def both(x, y, res=0):
        moe.layer_dev(x, tokens, y, ws.data_ptr(), n, res)
        moe.experts_dev(x, tokens, ids.data_ptr(), weights.data_ptr(), y, ws.data_ptr(), n, res)

    at = lambda row, values=0: buffer.data_ptr() + 4 * (row * d + values)
    for shifted in (at(tokens, 4), at(tokens, -4), at(tokens + 1), at(2 * tokens - 1), at(1), at(2 * tokens, -4)):
        for args in ((at(tokens), shifted), (other.data_ptr(), shifted, at(tokens)), (shifted, shifted, at(tokens))):
            with pytest.raises(ValueError, match="overlaps"):
                both(*args)
    torch.cuda.synchronize()
    assert (buffer == 3).all()
    both(at(tokens), at(2 * tokens), at(0))
    both(at(tokens), at(0), at(2 * tokens))
    both(at(0), at(tokens))
    torch.cuda.synchronize()
    assert torch.isfinite(buffer).all()


def test_the_workspace_of_a_pair(jn):
    """Gate and up of one format run as a pair and never leave registers; of two formats each has an array of its own in the workspace."""
    experts, used, d, ffn, tokens = 4, 2, 256, 1024, 2048
    rng = np.random.default_rng(1)
    pair, apart = ref.Layer(rng, experts, used, d, ffn, up="Q4_K").make(jn), ref.Layer(rng, experts, used, d, ffn, up="Q5_K", gate="Q4_K").make(jn)
    array = tokens * used * ffn * 4
    # (the same operands, lists and sums in both; chunks are no smaller in the second)
    assert apart.workspace(tokens) - pair.workspace(tokens) >= array - 65536
    # of one pass beside the array itself: operands of x and of the gated values (1152 bytes and a scale per 256 values), the products (rows of four columns are not shared out), choices
    # and logits
    most = array + (tokens * d + tokens * used * ffn) // 256 * 1156 + tokens * used * d * 4 + tokens * (experts * 8 * 8 + used * 16) + 65536
    assert pair.workspace(tokens) <= most

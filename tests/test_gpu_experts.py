"""The router of a mixture of experts, its experts' products and the whole layer against plain implementations in 64 bits."""
import numpy as np
import pytest
import torch

import experts_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def jn():
    import jitnn_amd
    jitnn_amd.init()
    return jitnn_amd


def dev(a, dtype=None):
    t = torch.as_tensor(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


def space(n):
    return torch.full((max(16, n),), 0xA5, dtype=torch.uint8, device="cuda")


class Call:
    """A layer's call on tensors of its own."""

    def __init__(self, moe, x, residual=None, ids=None, weights=None, room=0):
        self.moe, self.tokens = moe, len(x)
        self.x, self.y = dev(x), torch.full((len(x) + room, moe.d_model), 7.0, device="cuda")
        self.residual = None if residual is None else dev(residual)
        self.ids, self.weights = (None, None) if ids is None else (dev(ids, torch.int32), dev(weights, torch.float32))
        self.space = space(moe.workspace(len(x)))

    def __call__(self, stream=0, y=None):
        y = self.y if y is None else y
        r = 0 if self.residual is None else self.residual.data_ptr()
        if self.ids is None:
            self.moe.layer_dev(self.x.data_ptr(), self.tokens, y.data_ptr(), self.space.data_ptr(), self.space.numel(), r, stream)
        else:
            self.moe.experts_dev(self.x.data_ptr(), self.tokens, self.ids.data_ptr(), self.weights.data_ptr(), y.data_ptr(), self.space.data_ptr(), self.space.numel(), r, stream)
        return y

    def result(self):
        self()
        torch.cuda.synchronize()
        return self.y[:self.tokens].cpu().numpy()


# ---------------------------------------------------------------------------------------------- the router

def route_dev(r, x):
    n = r.workspace(len(x))
    xd, ids, w, s = dev(x), torch.full((len(x), r.used), -7, dtype=torch.int32, device="cuda"), torch.full((len(x), r.used), 7.0, device="cuda"), space(n)
    r.route_dev(xd.data_ptr(), len(x), ids.data_ptr(), w.data_ptr(), s.data_ptr(), n)
    torch.cuda.synchronize()
    return ids.cpu().numpy(), w.cpu().numpy()


def check_route(got, want):
    ids, w = got
    assert np.array_equal(ids, want[0])
    # FP64 up to the last step, rounded once: half a step of FP32, and what sums of some thousand products in another order make of an exponent
    assert (np.abs(w - want[1]) <= (2.0 ** -24 + 2.0 ** -40) * np.abs(want[1]) + 1e-44).all()


@pytest.mark.parametrize("gating,normalise,scale,biased", [("softmax", True, 1.0, False), ("softmax", False, 2.5, False), ("softmax", True, 1.0, True),
                                                           ("softmax", False, 1.0, True), ("sigmoid", True, 2.5, True), ("sigmoid", False, 1.0, False)])
@pytest.mark.parametrize("tokens,experts,used,d", [(1, 8, 2, 4096), (1, 128, 8, 2048), (3, 5, 5, 12), (7, 65, 3, 1028), (9, 8, 1, 64), (16, 16, 4, 16), (17, 100, 64, 404),
                                                   (64, 200, 6, 96), (65, 64, 64, 132), (300, 512, 10, 256), (1, 1, 1, 4), (40, 2, 2, 4100)])
def test_route(jn, tokens, experts, used, d, gating, normalise, scale, biased):
    rng = np.random.default_rng(tokens * experts + used)
    w = (rng.standard_normal((experts, d)) * 3 / np.sqrt(d)).astype(np.float32)
    bias = (0.2 * rng.standard_normal(experts)).astype(np.float32) if biased else None
    x = rng.standard_normal((tokens, d)).astype(np.float32)
    r = jn.Router(w, used, gating=gating, normalise=normalise, scale=scale, selection_bias=bias)
    check_route(route_dev(r, x), ref.route(x, w, used, gating, normalise, scale, bias))


def test_route_host_and_passes(jn):
    rng = np.random.default_rng(5)
    w, x = rng.standard_normal((6, 32)).astype(np.float32), rng.standard_normal((8192 + 33, 32)).astype(np.float32)
    r = jn.Router(w, 2)
    check_route(r.route(x), ref.route(x, w, 2))
    ids, weights = r.route(x[:1])
    check_route((ids, weights), ref.route(x[:1], w, 2))
    assert r.route(x[:0])[0].shape == (0, 2)


@pytest.mark.parametrize("tokens", [1, 20, 100])
def test_route_ties_and_odd_numbers(jn, tokens):
    """Equal logits go to the lowest index; logits that are not numbers come last; infinite ones are the largest."""
    d, experts = 64, 96
    w = np.zeros((experts, d), dtype=np.float32)
    w[70, 0] = w[80, 0] = w[7, 0] = 1.0
    x = np.zeros((tokens, d), dtype=np.float32)
    x[:, 0] = 1.0
    r = jn.Router(w, 5)
    ids, weights = route_dev(r, x)
    assert (ids == [7, 70, 80, 0, 1]).all()
    w2 = w.copy()
    w2[0], w2[1, 3], w2[2, 0] = np.nan, np.nan, -0.0
    ids, weights = route_dev(jn.Router(w2, 5), x)
    assert (ids == [7, 70, 80, 2, 3]).all() and np.isfinite(weights).all()
    w2[90, 0] = np.inf
    ids, _ = route_dev(jn.Router(w2, 64), x)
    assert (ids == ([90, 7, 70, 80] + [i for i in range(2, 96) if i not in (7, 70, 80, 90)])[:64]).all()
    w3 = np.zeros((6, d), dtype=np.float32)
    w3[:, 0] = [np.nan, -np.inf, 1, np.nan, np.inf, 0]
    assert (route_dev(jn.Router(w3, 6), x)[0] == [4, 2, 5, 1, 0, 3]).all()
    x[0] = np.nan
    ids, weights = route_dev(r, x)
    assert (ids[0] == range(5)).all() and np.isnan(weights[0]).all()
    assert (ids[1:] == [7, 70, 80, 0, 1]).all() and np.isfinite(weights[1:]).all()


def test_route_next_to_a_border(jn):
    """Two experts whose logits differ by less than FP32 sums can tell: the same choice at one token and in a batch."""
    rng = np.random.default_rng(8)
    d, experts = 2048, 32
    w = rng.standard_normal((experts, d)).astype(np.float32)
    x = rng.standard_normal((200, d)).astype(np.float32)
    for e in range(1, experts, 2):  # pairs a last bit of one value apart
        w[e] = w[e - 1]
        w[e, e] = np.nextafter(w[e, e], np.float32(9))
    r = jn.Router(w, 3)
    want = ref.route(x, w, 3)
    check_route(route_dev(r, x), want)
    check_route(tuple(np.concatenate(v) for v in zip(*(route_dev(r, x[t:t + 1]) for t in range(20)))), tuple(v[:20] for v in want))


# ---------------------------------------------------------------------------------------------- the experts

FORMATS = [("Q4_K", "Q6_K"), ("Q5_K", "Q5_K"), ("Q6_K", "Q4_K"), ("Q8_0", "Q8_0"), ("Q4_0", "Q4_1"), ("Q4_1", "Q4_0"), ("Q5_1", "Q2_K"), ("Q2_K", "Q5_1"), ("Q5_0", "Q3_K"), ("Q3_K", "Q5_0")]


@pytest.mark.parametrize("up,down", FORMATS)
@pytest.mark.parametrize("tokens", [1, 2, 5, 9, 40, 130])
def test_formats(jn, up, down, tokens):
    rng = np.random.default_rng(tokens)
    layer = ref.Layer(rng, 6, 2, 512, 256, up, down)
    moe = layer.make(jn)
    x = layer.input(rng, tokens)
    res = 0.1 * rng.standard_normal(x.shape).astype(np.float32)
    ref.close(Call(moe, x, res).result(), layer.experts_of(x, *layer.route(x), res), layer.tolerance)


@pytest.mark.parametrize("experts,used,d,ffn,up,down", [
    (8, 2, 4096, 1024, "Q4_K", "Q6_K"), (64, 6, 256, 1408, "Q8_0", "Q8_0"), (128, 8, 768, 256, "Q4_K", "Q4_K"), (3, 3, 32, 32, "Q8_0", "Q4_0"),
    (5, 1, 96, 64, "Q4_0", "Q5_1"), (4, 2, 2048, 96, "Q4_1", "Q8_0"), (7, 4, 1056, 2080, "Q4_0", "Q4_1"), (2, 2, 1280, 768, "Q6_K", "Q6_K"), (1, 1, 512, 512, "Q5_K", "Q2_K"),
    (16, 12, 256, 512, "Q6_K", "Q6_K"), (9, 2, 288, 32, "Q5_1", "Q5_1"), (4, 2, 5120, 320, "Q8_0", "Q8_0")])
@pytest.mark.parametrize("tokens", [1, 3, 8, 17, 70])
def test_shapes(jn, experts, used, d, ffn, up, down, tokens):
    rng = np.random.default_rng(experts + tokens)
    layer = ref.Layer(rng, experts, used, d, ffn, up, down, gating="sigmoid", normalise=True, scale=2.5, bias=(0.1 * rng.standard_normal(experts)).astype(np.float32))
    moe = layer.make(jn)
    x = layer.input(rng, tokens)
    ref.close(Call(moe, x).result(), layer.experts_of(x, *layer.route(x)), layer.tolerance)


@pytest.mark.parametrize("activation", [None, "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("tokens", [1, 12])
def test_activations(jn, activation, tokens):
    rng = np.random.default_rng(3)
    layer = ref.Layer(rng, 4, 2, 512, 768, activation=activation, normalise=False)
    x = 3 * layer.input(rng, tokens)
    ref.close(Call(layer.make(jn), x).result(), layer.experts_of(x, *layer.route(x)), layer.tolerance)


@pytest.mark.parametrize("tokens", [1, 11, 90])
def test_gate_and_up_of_two_formats(jn, tokens):
    rng = np.random.default_rng(4)
    layer = ref.Layer(rng, 4, 2, 512, 512, up="Q6_K", gate="Q4_K", down="Q8_0")
    x = layer.input(rng, tokens)
    ref.close(Call(layer.make(jn), x).result(), layer.experts_of(x, *layer.route(x)), layer.tolerance)


@pytest.mark.parametrize("tokens", [1, 4, 33, 200])
def test_given_choices(jn, tokens):
    """Ids from elsewhere: the same expert twice, ids that are no expert's, tokens of no expert, everybody at one expert."""
    rng = np.random.default_rng(tokens)
    layer = ref.Layer(rng, 5, 4, 256, 512)
    moe = layer.make(jn)
    x = layer.input(rng, tokens)
    ids = rng.integers(-2, 8, (tokens, 4))
    ids[0] = [3, 3, 3, -1]
    weights = rng.standard_normal((tokens, 4)).astype(np.float32)
    res = rng.standard_normal(x.shape).astype(np.float32)
    ref.close(Call(moe, x, res, ids, weights).result(), layer.experts_of(x, ids, weights, res), layer.tolerance)
    ids[:] = [9, -1, 1 << 30, -(1 << 31)]
    assert np.array_equal(Call(moe, x, res, ids, weights).result(), res)
    assert not Call(moe, x, None, ids, weights).result().any()
    ids[:] = 2
    ref.close(Call(moe, x, None, ids, weights).result(), layer.experts_of(x, ids, weights), layer.tolerance)


def test_rows_behind_the_last_and_passes(jn):
    """Some thousand tokens: more than one pass, and nothing is written behind them."""
    rng = np.random.default_rng(9)
    layer = ref.Layer(rng, 16, 8, 256, 256)
    moe = layer.make(jn)
    x = layer.input(rng, 512 + 261)
    call = Call(moe, x, room=2)
    got = call.result()
    assert (call.y[-2:] == 7).all()
    some = [0, 1, 100, 511, 512, 513, 772]
    ref.close(got[some], layer.experts_of(x[some], *layer.route(x[some])), layer.tolerance)
    assert moe.workspace(512 + 261) == moe.workspace(512) == moe.workspace(100000)


@pytest.mark.parametrize("tokens", [1, 6, 40])
def test_in_place_and_repeatable(jn, tokens):
    rng = np.random.default_rng(tokens)
    layer = ref.Layer(rng, 8, 2, 512, 256)
    moe = layer.make(jn)
    x = layer.input(rng, tokens)
    call = Call(moe, x, x)
    first = call.result()
    assert np.array_equal(call.result(), first)
    call.residual = call.x
    call(y=call.x)  # y, x and the residual all one
    assert np.array_equal(call.x.cpu().numpy(), first)
    assert np.array_equal(moe.layer(x, x), first)


@pytest.mark.parametrize("tokens", [1, 5, 30, 100])
def test_rows_that_are_not_numbers(jn, tokens):
    """A token with an infinite value or none at all gives a row that is not finite, and leaves the others' rows as they are."""
    rng = np.random.default_rng(tokens)
    layer = ref.Layer(rng, 4, 2, 512, 512)
    moe = layer.make(jn)
    x = layer.input(rng, tokens)
    clean = Call(moe, x).result()
    for bad in (np.nan, np.inf, -np.inf):
        z = x.copy()
        z[tokens // 2, 300] = bad
        got = Call(moe, z).result()
        keep = np.arange(tokens) != tokens // 2
        assert np.array_equal(got[keep], clean[keep])
        assert not np.isfinite(got[tokens // 2]).any()


def test_large_and_small_inputs(jn):
    """Inputs from 2^-60 to 2^40: the sums scale with them where there is no activation."""
    rng = np.random.default_rng(6)
    layer = ref.Layer(rng, 4, 2, 256, 512, activation=None)
    moe = layer.make(jn)
    ids, weights = np.tile([1, 3], (5, 1)), np.full((5, 2), 0.5, dtype=np.float32)
    x = layer.input(rng, 5)
    for s in (2.0 ** -60, 2.0 ** -20, 2.0 ** 20, 2.0 ** 40):
        z = (x * np.float32(s)).astype(np.float32)
        ref.close(Call(moe, z, None, ids, weights).result() / s ** 2, layer.experts_of(x, ids, weights), layer.tolerance)
        ref.close(Call(moe, z[:1], None, ids[:1], weights[:1]).result() / s ** 2, layer.experts_of(x[:1], ids[:1], weights[:1]), layer.tolerance)
    assert not Call(moe, np.zeros_like(x)).result().any()


@pytest.mark.parametrize("tokens", [1, 4, 24, 96])
def test_streams_and_graphs(jn, tokens):
    """Two layers at once on two streams; a recorded call, replayed with other inputs between eager work."""
    rng = np.random.default_rng(tokens)
    layer = ref.Layer(rng, 8, 2, 512, 512)
    moe = layer.make(jn)
    xs = [layer.input(rng, tokens) for _ in range(4)]
    want = [Call(moe, x).result() for x in xs]
    streams, calls = [torch.cuda.Stream() for _ in range(2)], [Call(moe, x) for x in xs[:2]]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, c in zip(streams, calls):
            c(s.cuda_stream)
    torch.cuda.synchronize()
    for c, w in zip(calls, want):
        assert np.array_equal(c.y.cpu().numpy(), w)
    call = Call(moe, xs[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(torch.cuda.current_stream().cuda_stream)
    for x, w in zip(xs, want):
        call.x.copy_(dev(x))
        call.space.fill_(0x5A)
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(call.y.cpu().numpy(), w)
        assert np.array_equal(Call(moe, xs[3]).result(), want[3])


def test_refusals(jn):
    rng = np.random.default_rng(1)
    layer = ref.Layer(rng, 4, 2, 256, 512)
    moe = layer.make(jn)
    x, y, ws = torch.zeros(8, 256, device="cuda"), torch.full((8, 256), 3.0, device="cuda"), space(moe.workspace(8))
    p, q, s, n = x.data_ptr(), y.data_ptr(), ws.data_ptr(), moe.workspace(8)
    for bad in (lambda: moe.layer_dev(0, 8, q, s, n), lambda: moe.layer_dev(p, 8, 0, s, n), lambda: moe.layer_dev(p, 8, q, 0, n), lambda: moe.layer_dev(p, 8, q, s, n - 1),
                lambda: moe.layer_dev(p + 4, 7, q, s, n), lambda: moe.layer_dev(p, 7, q + 8, s, n), lambda: moe.layer_dev(p, 7, q, s + 8, n), lambda: moe.layer_dev(p, -1, q, s, n),
                lambda: moe.layer_dev(p, 7, q, s, n, residual_ptr=p + 4), lambda: moe.experts_dev(p, 8, 0, p, q, s, n), lambda: moe.experts_dev(p, 8, p, 0, q, s, n),
                lambda: moe.workspace(-1), lambda: moe.router.workspace(-1), lambda: moe.router.route_dev(p, -1, q, q, s, n), lambda: moe.router.route_dev(p + 4, 1, q, q, s, n),
                lambda: moe.router.route_dev(0, 1, q, q, s, n), lambda: moe.router.route_dev(p, 1, 0, q, s, n), lambda: moe.router.route_dev(p, 8, q, 0, s, n),
                lambda: moe.router.route_dev(p, 100, q, q, 0, 0)):
        with pytest.raises(ValueError):
            bad()
    moe.layer_dev(0, 0, 0, 0, 0)
    moe.router.route_dev(0, 0, 0, 0)
    torch.cuda.synchronize()
    assert (y == 3).all() and moe.workspace(0) == 0
    w = np.zeros((4, 256), dtype=np.float32)
    for bad in (dict(used=0), dict(used=5), dict(used=2, gating="other"), dict(used=2, scale=float("nan")), dict(used=2, selection_bias=np.zeros(3)), dict(used=-1)):
        with pytest.raises(ValueError):
            jn.Router(w, **bad)
    for shape in ((513, 4), (4, 6), (4,), (0, 8)):
        with pytest.raises(ValueError):
            jn.Router(np.zeros(shape, dtype=np.float32), 1)
    gate, up, down = moe._keep
    other = jn.Router(np.zeros((4, 512), dtype=np.float32), 2)
    for bad in ((other, gate, up, down), (moe.router, gate, down, down), (moe.router, down, down, down), (moe.router, gate, up, up), (jn.Router(w[:2], 1), gate, up, down)):
        with pytest.raises(ValueError):
            jn.Moe(*bad)
    with pytest.raises(ValueError):
        jn.Moe(moe.router, gate, up, down, activation="swish2")
    with pytest.raises(ValueError):
        jn.Tensor.wrap_dev(jn.DType.Q4_K, p, 4, 100)
    with pytest.raises(ValueError):
        jn.Tensor.wrap_dev(jn.DType.Q4_K, p + 8, 4, 256)


@pytest.mark.parametrize("experts,used,d,ffn,up,down", [(8, 2, 512, 2048, "Q4_K", "Q6_K"), (64, 6, 256, 1408, "Q8_0", "Q8_0"), (100, 1, 64, 64, "Q5_0", "Q4_0")])
def test_a_workspace_does_for_fewer_tokens(jn, experts, used, d, ffn, up, down):
    rng = np.random.default_rng(2)
    layer = ref.Layer(rng, experts, used, d, ffn, up, down)
    moe = layer.make(jn)
    most = 150
    x, y, ws = dev(layer.input(rng, most)), torch.empty(most, d, device="cuda"), space(moe.workspace(most))
    ids, weights, rs = torch.empty(most, used, dtype=torch.int32, device="cuda"), torch.empty(most, used, device="cuda"), space(moe.router.workspace(most))
    for tokens in (1, 2, 7, 16, 17, 18, 25, 33, 64, 65, 149):
        moe.layer_dev(x.data_ptr(), tokens, y.data_ptr(), ws.data_ptr(), moe.workspace(most))
        moe.router.route_dev(x.data_ptr(), tokens, ids.data_ptr(), weights.data_ptr(), rs.data_ptr(), moe.router.workspace(most))
        moe.experts_dev(x.data_ptr(), tokens, ids.data_ptr(), weights.data_ptr(), (z := torch.empty(tokens, d, device="cuda")).data_ptr(), ws.data_ptr(), moe.workspace(most))
        torch.cuda.synchronize()
        assert torch.equal(y[:tokens], z)


@pytest.mark.parametrize("up,down", [("Q4_K", "Q2_K"), ("Q5_K", "Q6_K"), ("Q6_K", "Q4_K"), ("Q2_K", "Q5_K"), ("Q8_0", "Q4_0"), ("Q4_1", "Q5_1")])
@pytest.mark.parametrize("tokens", [65, 171, 300])
def test_many_rows_of_an_expert(jn, up, down, tokens):
    """More rows than a chunk holds, chunks of every number of groups; an expert of one row beside them, one of none."""
    rng = np.random.default_rng(tokens)
    layer = ref.Layer(rng, 4, 1, 256, 768, up, down)
    moe = layer.make(jn)
    x = layer.input(rng, tokens)
    ids = (rng.random((tokens, 1)) < 0.35).astype(np.int32) * 2
    ids[tokens // 3] = 1
    weights = rng.standard_normal((tokens, 1)).astype(np.float32)
    ref.close(Call(moe, x, None, ids, weights).result(), layer.experts_of(x, ids, weights), layer.tolerance)


@pytest.mark.parametrize("experts", [129, 200, 512])
@pytest.mark.parametrize("tokens", [1, 3, 16, 40, 70])
def test_many_experts(jn, experts, tokens):
    rng = np.random.default_rng(experts + tokens)
    layer = ref.Layer(rng, experts, 5, 256, 64, "Q4_0", "Q8_0", bias=(0.1 * rng.standard_normal(experts)).astype(np.float32))
    x = layer.input(rng, tokens)
    ref.close(Call(layer.make(jn), x).result(), layer.experts_of(x, *layer.route(x)), layer.tolerance)


def test_weights_beyond_31_bits(jn):
    """Experts that stand more than 2 GiB into their matrices: the results of a layer that has them alone, at one token bit for bit."""
    experts, d, ffn = 63, 4096, 8192
    gen = torch.Generator(device="cuda").manual_seed(1)
    scales = torch.tensor([0.01], dtype=torch.float16).view(torch.uint8).cuda()

    def blocks(count):
        raw = torch.empty(count, 34, dtype=torch.uint8, device="cuda").random_(0, 256, generator=gen)
        raw[:, :2] = scales
        return raw

    big = [blocks(experts * d * ffn // 32) for _ in range(3)]
    assert big[0].numel() > 1 << 31
    last = [61, 62]
    small = [b.reshape(experts, -1)[last].contiguous() for b in big]
    shapes = ((ffn, d), (ffn, d), (d, ffn))
    layers = []
    for count, parts in ((experts, big), (2, small)):
        router = jn.Router(np.zeros((count, d), dtype=np.float32), 2)
        layers.append(jn.Moe(router, *(jn.Tensor.wrap_dev(jn.DType.Q8_0, p.data_ptr(), count, *s) for p, s in zip(parts, shapes))))
    rng = np.random.default_rng(1)
    for tokens in (1, 5, 20):
        x = (0.001 * rng.standard_normal((tokens, d))).astype(np.float32)
        ids = rng.integers(0, 2, (tokens, 2))
        weights = rng.standard_normal((tokens, 2)).astype(np.float32)
        got, want = Call(layers[0], x, None, ids + 61, weights).result(), Call(layers[1], x, None, ids, weights).result()
        assert np.isfinite(want).all() and want.any()
        if tokens == 1:
            assert np.array_equal(got, want)
        else:  # (two experts and 63 may go another way, or come in another number of parts: either is off by one tolerance at most)
            ref.close(got, want, 2 * ref.tolerance(["Q8_0"] * 3))


@pytest.mark.parametrize("up,down", [f for f in FORMATS if "Q5_0" not in f])
@pytest.mark.parametrize("experts,used", [(200, 1), (20, 2)])
def test_few_rows_of_an_expert(jn, experts, used, up, down):
    """More tokens than the INT8 products are for, over so many experts that each has a row or a few: chunks of one group and of two."""
    rng = np.random.default_rng(experts)
    layer = ref.Layer(rng, experts, used, 256, 256, up, down)
    x = layer.input(rng, 67)
    ref.close(Call(layer.make(jn), x).result(), layer.experts_of(x, *layer.route(x)), layer.tolerance)


@pytest.mark.parametrize("gate,up,down", [("Q5_0", "Q5_0", "Q3_K"), ("Q3_K", "Q8_0", "Q5_0"), ("Q4_K", "Q3_K", "Q6_K"), ("Q4_K", "Q4_K", "Q5_0")])
@pytest.mark.parametrize("tokens", [1, 9, 70])
def test_blocks_that_are_left_as_they_are(jn, gate, up, down, tokens):
    """Q5_0 and Q3_K blocks in the caller's device memory, which nobody rewrites, beside formats that the matrix cores' kernels take."""
    rng = np.random.default_rng(tokens)
    layer = ref.Layer(rng, 5, 2, 256, 512, up=up, down=down, gate=gate)
    raw = [dev(r) for r in layer.raw]
    router = jn.Router(layer.router / layer.size, 2)
    moe = jn.Moe(router, *(jn.Tensor.wrap_dev(jn.DType[f], r.data_ptr(), *s) for f, r, s in zip(layer.formats, raw, layer.shapes)))
    x = layer.input(rng, tokens)
    res = rng.standard_normal(x.shape).astype(np.float32)
    ref.close(Call(moe, x, res).result(), layer.experts_of(x, *layer.route(x), res), layer.tolerance)


@pytest.mark.parametrize("experts,used,d,ffn,up,down", [(9, 8, 256, 4352, "Q4_K", "Q6_K"), (5, 4, 64, 10752, "Q8_0", "Q4_0"), (6, 5, 512, 13312, "Q5_K", "Q2_K"), (40, 33, 128, 6400, "Q4_1", "Q8_0")])
@pytest.mark.parametrize("tokens", [1, 3])
def test_long_rows_in_parts(jn, experts, used, d, ffn, up, down, tokens):
    """Down projections of one token that are longer than a workgroup takes: parts, the last of them ragged, that a launch more adds up with the residual."""
    rng = np.random.default_rng(ffn)
    layer = ref.Layer(rng, experts, used, d, ffn, up, down)
    moe = layer.make(jn)
    x = layer.input(rng, tokens)
    res = rng.standard_normal(x.shape).astype(np.float32)
    ids, weights = layer.route(x)
    want = layer.experts_of(x, ids, weights, res)
    call = Call(moe, x, res)
    ref.close(call.result(), want, layer.tolerance)
    call.y.copy_(call.residual)
    call.residual = call.y  # y is the residual
    ref.close(call.result(), want, layer.tolerance)
    bad = ids.copy()
    bad[0] = -1
    assert np.array_equal(Call(moe, x, res, bad, weights).result()[0], res[0])


@pytest.mark.parametrize("up,down", [f for f in FORMATS if "Q5_0" not in f])
@pytest.mark.parametrize("tokens", [20, 45, 70, 201])
def test_large_chunks(jn, up, down, tokens):
    """So many rows of weights that chunks are as large as a kernel holds: groups in one set, in two and three, the last one ragged, and experts of several chunks."""
    rng = np.random.default_rng(tokens)
    layer = ref.Layer(rng, 2, 2, 256, 12288, up, down)
    x = layer.input(rng, tokens)
    ids, weights = np.tile([1, 0], (tokens, 1)), rng.standard_normal((tokens, 2)).astype(np.float32)
    want = np.zeros(x.shape)
    for j, e in enumerate((1, 0)):
        gate, up_, down_ = (v[e] for v in layer.values)
        want += weights[:, j:j + 1] * ((ref.activate("silu", x.astype(np.float64) @ gate.T) * (x.astype(np.float64) @ up_.T)) @ down_.T)
    ref.close(Call(layer.make(jn), x, None, ids, weights).result(), want, layer.tolerance)

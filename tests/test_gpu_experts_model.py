"""Mixtures of experts in the layers of a model: decode steps, prompts, served batches, files, recorded passes - against the oracle's operators and against one another."""
import numpy as np
import pytest
import torch

import experts_reference as ref
import test_llm
from decode_oracle import SLOTS
from gguf_writer import write_gguf
from helpers import GGML_ID, norm_err
from oracle import oracle
from test_gpu_decode import build

pytestmark = pytest.mark.gpu

CFG = dict(layers=3, d_model=256, heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=300, max_ctx=160, rms_eps=1e-5, rope_theta=1e4)


@pytest.fixture(scope="module")
def jn():
    import jitnn_amd
    jitnn_amd.init()
    return jitnn_amd


def with_experts(jn, dec, layers, at, seed, **kw):
    """Puts random experts into the layers `at`; their inputs, the normalised rows, brought to the size the experts are made for."""
    rng = np.random.default_rng(seed)
    for l in at:
        moe = ref.Layer(rng, d=dec.cfg["d_model"], **kw)
        layers[l]["moe"] = moe
        layers[l]["ffn_norm"] = (layers[l]["ffn_norm"] * moe.size).astype(np.float32)
        dec.set_norm(l, 1, layers[l]["ffn_norm"])
        dec.set_moe(l, moe.make(jn))


def forward(cfg, layers, out_norm, out_w, kc, vc, x, pos0):
    """As decode_oracle.prefill_ref, with experts where a layer has them; -> (logits of every token, the smallest gap between a chosen expert's score and one that was
    not, over the logits' spread)."""
    heads, kv, hd, eps, theta = cfg["heads"], cfg["kv_heads"], cfg["head_dim"], cfg["rms_eps"], np.float32(cfg["rope_theta"])

    def lin(w, a):
        fid, raw, n, k = w
        return (a.astype(np.float64) @ oracle.dequantize(fid, raw, n * k).reshape(n, k).astype(np.float64).T).astype(np.float32)

    x, gap = np.ascontiguousarray(x, dtype=np.float32), np.inf
    T = len(x)
    for li, L in enumerate(layers):
        n = oracle.rms_norm(x, L["attn_norm"], eps)
        q = oracle.rope(lin(L["attn_q"], n).reshape(T, heads, hd), theta, pos0, False, True)
        k = oracle.rope(lin(L["attn_k"], n).reshape(T, kv, hd), theta, pos0, False, True)
        kc[li, pos0:pos0 + T], vc[li, pos0:pos0 + T] = k, lin(L["attn_v"], n).reshape(T, kv, hd)
        att = np.stack([oracle.attention_decode(q[t], kc[li, :pos0 + t + 1], vc[li, :pos0 + t + 1]).reshape(-1) for t in range(T)])
        x = oracle.add(x, lin(L["attn_o"], att))
        m = oracle.rms_norm(x, L["ffn_norm"], eps)
        if "moe" in L:
            e = L["moe"]
            ids, weights = e.route(m)
            x = e.experts_of(m, ids, weights, x).astype(np.float32)
            if e.used < e.experts:
                z = np.sort(m.astype(np.float64) @ (e.router / e.size).astype(np.float64).T, axis=1)[:, ::-1]
                gap = min(gap, ((z[:, e.used - 1] - z[:, e.used]) / z.std(axis=1)).min())
        else:
            x = oracle.add(x, lin(L["ffn_down"], oracle.swiglu(lin(L["ffn_gate"], m), lin(L["ffn_up"], m))))
    return lin(out_w, oracle.rms_norm(x, out_norm, eps)), gap


def caches(cfg):
    kc = np.zeros((cfg["layers"], cfg["max_ctx"], cfg["kv_heads"], cfg["head_dim"]), dtype=np.float32)
    return kc, np.zeros_like(kc)


# Up to 64 tokens every linear is FP32-grade, the bar of the dense model's test; beyond, the attention's linears have FP16 operands, 2e-3 each and 1e-2 on the logits of
# two layers: half as much again for three.  There every expert is used, for the choice is no continuous function of its input.
@pytest.mark.parametrize("experts,used,ffn,up,down", [(8, 2, 512, "Q4_K", "Q6_K"), (12, 5, 288, "Q8_0", "Q8_0"), (5, 2, 256, "Q5_0", "Q3_K")])
@pytest.mark.parametrize("tokens", [1, 2, 11, 40])
def test_decode_and_prompt(jn, experts, used, ffn, up, down, tokens):
    dec, layers, out_norm, out_w = build(jn, CFG, 11)
    with_experts(jn, dec, layers, (1, 2), experts, experts=experts, used=used, ffn=ffn, up=up, down=down)
    x = np.random.default_rng(tokens).standard_normal((tokens + 3, CFG["d_model"])).astype(np.float32)
    kc, vc = caches(CFG)
    want, gap = forward(CFG, layers, out_norm, out_w, kc, vc, x, 0)
    assert gap > 1e-4  # (an error of 1e-5 cannot change a choice)
    got = dec.prefill(x[:tokens], 0) if tokens > 1 else dec.decode(x[0], 0)
    assert norm_err(got, want[tokens - 1]) <= 1e-4
    for t in range(tokens, tokens + 3):
        assert norm_err(dec.decode(x[t], t), want[t]) <= 1e-4
    for l in range(CFG["layers"]):
        k, v = dec.kv_read(l, 0, tokens + 3)
        assert norm_err(k, kc[l, :tokens + 3]) <= 1e-4 and norm_err(v, vc[l, :tokens + 3]) <= 1e-4
    dec.close()


@pytest.mark.parametrize("tokens", [70, 130])
def test_long_prompt(jn, tokens):
    dec, layers, out_norm, out_w = build(jn, CFG, 12)
    with_experts(jn, dec, layers, (0, 2), 3, experts=3, used=3, ffn=512)
    x = np.random.default_rng(tokens).standard_normal((tokens, CFG["d_model"])).astype(np.float32)
    want, _ = forward(CFG, layers, out_norm, out_w, *caches(CFG), x, 0)
    assert norm_err(dec.prefill(x, 0), want[-1]) <= 1.5e-2
    dec.close()


def leading(rng, dec, layers, at, tokens, experts=6, used=2):
    """Experts that a token's own value leads to, past what the layers in between add -> the tokens' rows, each along two of the routers' directions."""
    d = dec.cfg["d_model"]
    rows, largest = rng.standard_normal((experts, d)) / np.sqrt(d), 0.0
    for l in at:
        moe = ref.Layer(rng, experts, used, d, 512)
        moe.router = (rows / 4).astype(np.float32)
        largest = max(largest, np.sqrt((moe.values[2] ** 2).mean() * moe.ffn))
        layers[l]["moe"] = moe
        layers[l]["ffn_norm"] = (layers[l]["ffn_norm"] * moe.size).astype(np.float32)
        dec.set_norm(l, 1, layers[l]["ffn_norm"])
    pairs = np.array([rng.permutation(experts)[:2] for _ in range(tokens)])
    return (largest * (np.sqrt(d / 2) * rows[pairs].sum(1) + 0.3 * rng.standard_normal((tokens, d)))).astype(np.float32)


# The linears of the attention have FP16 operands here, so that what reaches the router differs between a token by itself and a prompt: logits that lie closer together than that may be chosen
# either way.  These lie apart: logits of about 4 whose input is off by three linears' 2e-3 at most are off by 0.024 against a gap of about a standard deviation, one, and the choice of every token
# is the plain one.  The weights of two experts change by a quarter of what their logits do, 0.6 % a layer beside test_long_prompt's 1.5 % of FP16 linears: 3 % in all.  (Another second expert
# changes a token's logits by 5.8 % at least.)
@pytest.mark.parametrize("tokens", [70, 130])
def test_choices_of_a_long_prompt(jn, tokens):
    dec, layers, out_norm, out_w = build(jn, CFG, 16)
    rng = np.random.default_rng(tokens)
    x = leading(rng, dec, layers, (0, 2), tokens)
    for l in (0, 2):
        dec.set_moe(l, layers[l]["moe"].make(jn))
    want, gap = forward(CFG, layers, out_norm, out_w, *caches(CFG), x, 0)
    assert gap > 0.9
    table, starts, lens = (torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([[0, 1, 2]], [0, tokens], [tokens]))
    cache = jn.PagedCache(CFG["layers"], CFG["kv_heads"], CFG["head_dim"], 3, 64, 0)
    batch = jn.Batch(1, tokens, tokens, 192, table.data_ptr(), 3, starts.data_ptr(), lens.data_ptr())
    xd, rows, logits = torch.from_numpy(x).cuda(), torch.arange(tokens, dtype=torch.int32, device="cuda"), torch.empty(tokens, CFG["vocab"], device="cuda")
    dec.step_dev(cache, batch, xd.data_ptr(), rows.data_ptr(), tokens, logits.data_ptr(), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    got = logits.cpu().numpy()
    assert all(norm_err(g, w) <= 3e-2 for g, w in zip(got, want))
    assert norm_err(dec.prefill(x, 0), want[-1]) <= 3e-2
    dec.close()


def test_layers_change_places(jn):
    """Experts in, experts out: the dense layer's results come back bit for bit, and a model without dense weights where experts stand runs."""
    dec, layers, out_norm, out_w = build(jn, CFG, 13)
    x = np.random.default_rng(0).standard_normal((20, CFG["d_model"])).astype(np.float32)
    dense, one = dec.prefill(x, 0), dec.decode(x[0], 20)
    moe = ref.Layer(np.random.default_rng(1), 6, 2, CFG["d_model"], 512)
    dec.set_moe(1, moe.make(jn))
    mixed = dec.prefill(x, 0)
    assert norm_err(mixed, dense) > 1e-3
    dec.set_moe(1, None)
    assert np.array_equal(dec.prefill(x, 0), dense) and np.array_equal(dec.decode(x[0], 20), one)
    other = ref.Layer(np.random.default_rng(1), 2, 2, 512, 256).make(jn)
    for layer, e in ((3, moe.make(jn)), (-1, None), (0, other)):
        with pytest.raises(ValueError):
            dec.set_moe(layer, e)
    bare = jn.LlamaDecoder(**{**CFG, "layers": 1})
    for slot in range(4):
        fid, raw, n, k = layers[0][SLOTS[slot]]
        bare.set_weight(0, slot, jn.Tensor.quantized(next(t for t in jn.DType if t.ggml_id == fid), raw, n, k))
    fid, raw, n, k = out_w
    bare.set_weight(0, 7, jn.Tensor.quantized(next(t for t in jn.DType if t.ggml_id == fid), raw, n, k))
    for which in range(3):
        bare.set_norm(0, which, out_norm)
    with pytest.raises(ValueError):
        bare.decode(x[0], 0)  # (no gate, up and down, no experts)
    bare.set_moe(0, moe.make(jn))
    assert np.isfinite(bare.decode(x[0], 0)).all()
    bare.close()
    dec.close()


@pytest.mark.parametrize("tokens", [1, 3, 20])
def test_recorded_passes(jn, tokens):
    """A decode step and a pass of a batch, recorded and replayed between eager passes that are longer than any before."""
    dec, layers, _, _ = build(jn, CFG, 14)
    with_experts(jn, dec, layers, (0, 1), 4, experts=8, used=2, ffn=256)
    rng = np.random.default_rng(tokens)
    table, starts, lens = (torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([[0, 1]], [0, tokens], [tokens]))
    cache = jn.PagedCache(CFG["layers"], CFG["kv_heads"], CFG["head_dim"], 2, 64, 0)
    batch = jn.Batch(1, tokens, tokens, 64, table.data_ptr(), 2, starts.data_ptr(), lens.data_ptr())
    x, rows = torch.empty(tokens, CFG["d_model"], device="cuda"), torch.arange(tokens, dtype=torch.int32, device="cuda")
    logits, one = torch.empty(tokens, CFG["vocab"], device="cuda"), torch.empty(CFG["vocab"], device="cuda")

    def run():
        s = torch.cuda.current_stream().cuda_stream
        dec.step_dev(cache, batch, x.data_ptr(), rows.data_ptr(), tokens, logits.data_ptr(), s)
        dec.decode_dev(x.data_ptr(), 0, one.data_ptr(), s)

    inputs, want = [rng.standard_normal((tokens, CFG["d_model"])).astype(np.float32) for _ in range(4)], []
    for a in inputs:
        x.copy_(torch.from_numpy(a))
        run()
        torch.cuda.synchronize()
        want.append((logits.cpu().numpy(), one.cpu().numpy()))
        assert norm_err(want[-1][0][0], want[-1][1]) <= 1e-4  # (a sequence's first row is the token by itself)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for i, (a, w) in enumerate(zip(inputs, want)):
        x.copy_(torch.from_numpy(a))
        logits.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(logits.cpu().numpy(), w[0]) and np.array_equal(one.cpu().numpy(), w[1])
        dec.prefill(np.tile(inputs[0], (40, 1))[:21 + 30 * i], 1, logits=False)  # (a larger workspace takes the place of the one the replays use)
    torch.cuda.synchronize()
    dec.close()


def test_a_pass_is_recorded_after_experts_change(jn):
    """Experts that need no more than the workspace there is, and a layer that is dense again: a pass of a size that has run may be recorded as before."""
    dec, layers, _, _ = build(jn, CFG, 15)
    tokens = 20
    table, starts, lens = (torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([[0, 1]], [0, tokens], [tokens]))
    cache = jn.PagedCache(CFG["layers"], CFG["kv_heads"], CFG["head_dim"], 2, 64, 0)
    batch = jn.Batch(1, tokens, tokens, 64, table.data_ptr(), 2, starts.data_ptr(), lens.data_ptr())
    x, rows = torch.randn(tokens, CFG["d_model"], device="cuda"), torch.arange(tokens, dtype=torch.int32, device="cuda")
    logits = torch.empty(tokens, CFG["vocab"], device="cuda")

    def run():
        dec.step_dev(cache, batch, x.data_ptr(), rows.data_ptr(), tokens, logits.data_ptr(), torch.cuda.current_stream().cuda_stream)
        return logits

    moes = [ref.Layer(np.random.default_rng(s), 6, 2, CFG["d_model"], 512).make(jn) for s in (1, 2)]
    dec.set_moe(1, moes[0])
    run()
    torch.cuda.synchronize()
    for moe in (moes[1], None, moes[0]):
        dec.set_moe(1, moe)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        logits.fill_(0)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            replayed = logits.cpu().numpy()
            assert np.array_equal(run().cpu().numpy(), replayed) and replayed.any()
        del graph
    # more than there is room for: refused, and nothing is recorded
    dec.set_moe(1, ref.Layer(np.random.default_rng(3), 6, 6, CFG["d_model"], 2048).make(jn))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError, match="recording"):
            run()
        logits.fill_(1)
    graph.replay()
    torch.cuda.synchronize()
    assert (logits == 1).all()
    assert np.isfinite(run().cpu().numpy()).all()
    dec.close()


# ---------------------------------------------------------------------------------------------- files

def write_experts(path, monkeypatch, experts=6, used=2, ffn=256, meta=(), extra=(), drop=(), router_type="F32", bias=False, layers=(0, 1)):
    """test_llm's model with experts in `layers`."""
    rng = np.random.default_rng(3)
    d, made = test_llm.CFG["d_model"], {}

    def write(p, m, tensors):
        tensors = [t for t in tensors if not any(t[0] == f"blk.{l}.{n}.weight" for l in layers for n in ("ffn_gate", "ffn_up", "ffn_down"))]
        for l in layers:
            e = made[l] = ref.Layer(rng, experts, used, d, ffn, bias=(0.1 * rng.standard_normal(experts)).astype(np.float32) if bias else None)
            router = (e.router / e.size).astype(np.float32)
            if router_type == "F16":
                router = router.astype(np.float16)
            e.in_file = router.astype(np.float32)
            norm = next(i for i, t in enumerate(tensors) if t[0] == f"blk.{l}.ffn_norm.weight")
            tensors[norm] = (*tensors[norm][:3], (tensors[norm][3] * e.size).astype(np.float32))
            e.norm = tensors[norm][3]
            tensors.append((f"blk.{l}.ffn_gate_inp.weight", router.shape, {"F32": 0, "F16": 1}[router_type], router))
            for n, raw, fmt, shape in zip(("ffn_gate_exps", "ffn_up_exps", "ffn_down_exps"), e.raw, e.formats, e.shapes):
                tensors.append((f"blk.{l}.{n}.weight", shape, GGML_ID[fmt], raw))
            if bias:
                tensors.append((f"blk.{l}.exp_probs_b.bias", (experts,), 0, e.routing["bias"]))
        tensors = [t for t in tensors if t[0] not in drop] + list(extra)
        write_gguf(p, {**m, "llama.expert_count": experts, "llama.expert_used_count": used, **dict(meta)}, tensors)

    monkeypatch.setattr(test_llm, "write_gguf", write)
    model = test_llm.write_model(path, "llama", 11)
    for l, e in made.items():
        model["layers"][l]["ffn_norm"] = e.norm
    return model, made


@pytest.mark.parametrize("case", ["plain", "sigmoid", "a dense layer", "not normalised"])
def test_files(jn, tmp_path, monkeypatch, case):
    """A file's experts: metadata and tensors as they should be, every logit against the same layers put together by hand."""
    kw = {"plain": {}, "sigmoid": dict(meta={"llama.expert_gating_func": 2, "llama.expert_weights_norm": True, "llama.expert_weights_scale": 2.5}.items(), bias=True, router_type="F16"),
          "a dense layer": dict(layers=(1,)), "not normalised": dict(meta={"llama.expert_weights_norm": False, "llama.expert_feed_forward_length": 256}.items())}[case]
    routing = {"sigmoid": dict(gating="sigmoid", scale=2.5), "not normalised": dict(normalise=False)}.get(case, {})
    model, made = write_experts(tmp_path / "e.gguf", monkeypatch, **kw)
    for e in made.values():
        e.routing = {**{k: v for k, v in e.routing.items() if v is not None}, **routing}
    with jn.Llm.load(tmp_path / "e.gguf") as llm:
        assert "Q4_K" in llm.info().quantisation and llm.info().ffn == 512
        dec, vocab = llm.model(), llm.info().vocab
        table = dec.embed(np.arange(vocab))
        own = jn.LlamaDecoder(**dict(test_llm.CFG, vocab=vocab))
        own.set_rope_interleaved(True)
        by_id = {t.ggml_id: t for t in jn.DType}
        for l, L in enumerate(model["layers"]):
            for slot, name in enumerate(SLOTS):
                fid, raw, n, k = L[name]
                if slot < 4 or l not in made:
                    own.set_weight(l, slot, jn.Tensor.quantized(by_id[fid], raw, n, k))
            own.set_norm(l, 0, L["attn_norm"])
            own.set_norm(l, 1, L["ffn_norm"])
            if l in made:
                e, r = made[l], made[l].routing
                router = jn.Router(e.in_file, e.used, r.get("gating", "softmax"), r.get("normalise", True), r.get("scale", 1.0), r.get("bias"))
                own.set_moe(l, jn.Moe(router, *(jn.Tensor.quantized(jn.DType[f], raw, *shape) for f, raw, shape in zip(e.formats, e.raw, e.shapes))))
        own.set_norm(0, 2, model["out_norm"])
        fid, raw, n, k = model["out_w"]
        own.set_weight(0, 7, jn.Tensor.quantized(by_id[fid], raw, n, k))
        ids = [1, 40, 7, 90, 33]
        assert norm_err(dec.prefill(table[ids], 0), own.prefill(table[ids], 0)) <= 1e-6
        assert norm_err(dec.decode(table[5], 5), own.decode(table[5], 5)) <= 1e-6
        # greedy text: deterministic, the streamed pieces add up
        streamed = []
        text = llm.generate("the cat sat on the", 10, streamed.append)
        assert text == "".join(streamed) == llm.generate("the cat sat on the", 10)
        own.close()


def test_a_served_batch(jn, tmp_path, monkeypatch):
    """Sequences from one prompt, decoded together: every row's logits as if it had run alone; continuations follow the greedy loop."""
    write_experts(tmp_path / "e.gguf", monkeypatch, bias=True)
    rng = np.random.default_rng(2)
    with jn.Llm.load(tmp_path / "e.gguf") as llm:
        dec, vocab = llm.model(), llm.info().vocab
        table = dec.embed(np.arange(vocab))
        prompt = [int(t) for t in rng.integers(0, vocab, 21)]

        def alone(tokens):
            dec.prefill(table[tokens[:-1]], 0, logits=False)
            return dec.decode(table[tokens[-1]], len(tokens) - 1)

        run = jn.SharedPrompt(dec, prompt, 5, 60, rows=3, page_tokens=16, ggml_type=0)
        assert norm_err(run.prompt_logits, alone(prompt)) <= 1e-4
        known = [list(prompt) for _ in range(5)]
        for which, counts in (([0, 1, 2, 3, 4], [1, 1, 1, 1, 1]), ([3, 0, 4], [3, 1, 2]), ([1], [2])):
            tokens = [[int(t) for t in rng.integers(0, vocab, c)] for c in counts]
            got, at = run.step(which, tokens), 0
            for i, ts in zip(which, tokens):
                for t in ts:
                    known[i].append(t)
                    assert norm_err(got[at], alone(known[i])) <= 1e-4
                    at += 1
        request = jn.GenerationRequest("the dog ran to", 12)
        assert all(r.tokens == llm.generate(request).tokens for r in llm.continuations(request, 3, cache_type=0))


def test_files_that_are_refused(jn, tmp_path, monkeypatch):
    f32 = np.zeros(4, dtype=np.float32)
    for i, kw in enumerate((dict(meta={"llama.expert_gating_func": 3}.items()), dict(meta={"llama.expert_group_count": 4}.items()), dict(meta={"llama.expert_count": 7}.items()),
                            dict(meta={"llama.expert_used_count": 0}.items()), dict(meta={"llama.expert_used_count": 7}.items()),
                            dict(extra=[("blk.1.ffn_up_shexp.weight", (4,), 0, f32)]), dict(drop=("blk.1.ffn_down_exps.weight",)), dict(drop=("blk.0.ffn_gate_inp.weight",)))):
        write_experts(tmp_path / f"{i}.gguf", monkeypatch, **kw)
        with pytest.raises(ValueError):
            jn.Llm.load(tmp_path / f"{i}.gguf")

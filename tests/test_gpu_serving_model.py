"""A batch through the whole model over a paged cache, against the model's own cache and loop: the step, shared prompts, continuations, drafts, rotary scaling."""
import ctypes as C

import numpy as np
import pytest
import torch

import serving_reference as ref
import test_llm
from gguf_writer import write_gguf
from helpers import norm_err

pytestmark = pytest.mark.gpu

# FP32-grade linears and attention on both sides: the bar of the few-row linears.  FP16 pages: half a step, 2^-11, on values, and on scores of up to about 8 the same
# share of them, 2^-8 in a weight; two layers of both: 2 (2^-8 + 2^-11) = 0.9 %.
BAR = {0: 1e-4, 1: 9e-3}


@pytest.fixture(scope="module")
def jn():
    import jitnn_amd
    jitnn_amd.init()
    return jitnn_amd


@pytest.fixture(scope="module")
def model_file(tmp_path_factory):
    path = tmp_path_factory.mktemp("serving") / "tiny.gguf"
    test_llm.write_model(path, "llama", 11)
    return path


def own_logits(dec, table, tokens, count):
    """The model's own cache: logits after each of the last `count` tokens."""
    out = []
    head = tokens[: len(tokens) - count]
    if head:
        dec.prefill(table[head], 0, logits=False)
    for pos in range(len(head), len(tokens)):
        out.append(dec.decode(table[tokens[pos]], pos))
    return np.stack(out)


@pytest.mark.parametrize("cache_type", [0, 1])
@pytest.mark.parametrize("page", [16, 64])
def test_step_against_the_models_own_cache(jn, model_file, cache_type, page):
    """Three sequences of other lengths with other numbers of new tokens, a fourth without any, a row of nobody at the end; then another pass on top."""
    rng = np.random.default_rng(0)
    with jn.Llm.load(model_file) as llm:
        dec, vocab = llm.model(), llm.info().vocab
        table = dec.embed(np.arange(vocab))
        lens = [37, 1, 20, 0]
        known = [list(rng.integers(0, vocab, n)) for n in lens]
        b = ref.Batch(rng, [37, 1, 20, 0], lens, page, pad_rows=1, max_len=60)
        cache = jn.PagedCache(2, 2, 64, b.pages, page, cache_type)
        for counts in ([37, 1, 20, 0], [1, 3, 2, 4]):
            if counts != [37, 1, 20, 0]:
                for k, c in zip(known, counts):
                    k.extend(int(t) for t in rng.integers(0, vocab, c))
            starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
            rows = int(starts[-1]) + 1
            flat = [t for k, c in zip(known, counts) for t in k[len(k) - c:]]
            x = torch.zeros(rows, 256, device="cuda")
            x[:-1] = torch.from_numpy(table[np.array(flat, dtype=np.int64)]).cuda()
            keep = [torch.from_numpy(a).cuda() for a in (b.tables, starts, np.array([len(k) for k in known], dtype=np.int32))]
            nb = jn.Batch(4, rows, max(counts), 60, keep[0].data_ptr(), b.width, keep[1].data_ptr(), keep[2].data_ptr())
            want_rows = [int(s) - 1 for s, c in zip(starts[1:], counts) if c]
            pick = torch.tensor(want_rows + [rows, -1], dtype=torch.int32, device="cuda")
            logits = torch.empty(len(pick), vocab, device="cuda")
            dec.step_dev(cache, nb, x.data_ptr(), pick.data_ptr(), len(pick), logits.data_ptr())
            torch.cuda.synchronize()
            got = logits.cpu().numpy()
            assert np.isnan(got[-2:]).all()  # rows outside the batch
            at = 0
            for k, c in zip(known, counts):
                if c:
                    assert norm_err(got[at], own_logits(dec, table, k, 1)[0]) <= BAR[cache_type]
                    at += 1


@pytest.mark.parametrize("cache_type", [0, 1])
@pytest.mark.parametrize("prompt_len", [1, 16, 37])
def test_shared_prompt(jn, model_file, cache_type, prompt_len):
    """Five sequences from one prompt that ends on a page's border, inside a page or inside the first: every row's logits as if each had run alone."""
    rng = np.random.default_rng(prompt_len)
    with jn.Llm.load(model_file) as llm:
        dec, vocab = llm.model(), llm.info().vocab
        table = dec.embed(np.arange(vocab))
        prompt = [int(t) for t in rng.integers(0, vocab, prompt_len)]
        run = jn.SharedPrompt(dec, prompt, 5, 60, rows=3, page_tokens=16, ggml_type=cache_type)
        assert norm_err(run.prompt_logits, own_logits(dec, table, prompt, 1)[0]) <= BAR[cache_type]
        known = [list(prompt) for _ in range(5)]
        for which, counts in (([0, 1, 2, 3, 4], [1, 1, 1, 1, 1]), ([3, 0, 4], [3, 1, 2]), ([1], [2]), ([4, 2], [1, 3])):
            tokens = [[int(t) for t in rng.integers(0, vocab, c)] for c in counts]
            got, at = run.step(which, tokens), 0
            for i, ts in zip(which, tokens):
                known[i] += ts
                assert norm_err(got[at:at + len(ts)], own_logits(dec, table, known[i], len(ts))) <= BAR[cache_type]
                at += len(ts)
            assert run.lens == [len(k) for k in known]
        for bad in (([0, 0], [[1], [1]]), ([0], [[]]), ([0], [[1, 2, 3, 4]]), ([0], [[vocab]]), ([], [])):
            with pytest.raises(ValueError):
                run.step(*bad)


def test_verified_drafts_leave_the_cache_as_if_they_had_not_been(jn, model_file):
    """Passes with drafts, some kept and some not, then logits: those of the kept tokens alone."""
    rng = np.random.default_rng(5)
    with jn.Llm.load(model_file) as llm:
        dec, vocab = llm.model(), llm.info().vocab
        table = dec.embed(np.arange(vocab))
        prompt = [int(t) for t in rng.integers(0, vocab, 18)]
        run = jn.SharedPrompt(dec, prompt, 3, 60, rows=4, page_tokens=16, ggml_type=0)
        known = [list(prompt) + [int(np.argmax(run.prompt_logits))] for _ in range(3)]
        kept_ever = 0
        for turn in range(4):
            tokens = []
            for i, k in enumerate(known):
                # sequence 0 drafts what the model will say, sequence 1 its first token only, sequence 2 nonsense
                right, ctx = [], list(k)
                for _ in range(3):
                    right.append(int(np.argmax(own_logits(dec, table, ctx, 1)[0])))
                    ctx.append(right[-1])
                wrong = [(t + 1) % vocab for t in right]
                tokens.append([k[-1]] + (right if i == 0 else [right[0]] + wrong[1:] if i == 1 else wrong[: 1 + turn % 3]))
            got = run.verify([0, 1, 2], tokens, [0.0] * 3, rng.random((sum(len(t) for t in tokens), 2)))
            assert [kept for kept, _ in got] == [3, 1, 0]
            for i, (kept, token) in enumerate(got):
                assert token == int(np.argmax(own_logits(dec, table, known[i] + tokens[i][1:1 + kept], 1)[0]))
                known[i] += tokens[i][1:1 + kept] + [token]
                kept_ever += kept
            assert run.lens == [len(k) - 1 for k in known]
        logits = run.step([0, 1, 2], [[k[-1]] for k in known])
        for i, k in enumerate(known):
            assert norm_err(logits[i], own_logits(dec, table, k, 1)[0]) <= 1e-4
        assert kept_ever == 16


def test_continuations_and_drafts(jn, model_file):
    from jitnn_amd import GenerationRequest
    prompt = "the cat sat on the mat and the cat sat on"
    with jn.Llm.load(model_file) as llm:
        ids = llm.tokenizer().encode(prompt)
        greedy = llm.generate(GenerationRequest(prompt, 20))
        for kw in (dict(), dict(draft_tokens=3), dict(draft_tokens=7)):
            for r in llm.continuations(GenerationRequest(prompt, 20, **kw), 3, page_tokens=16, cache_type=0):
                assert (r.tokens, r.text, r.finish_reason, r.prompt_tokens) == (greedy.tokens, greedy.text, greedy.finish_reason, len(ids))
        streamed = []
        r = llm.generate(GenerationRequest(prompt, 20, draft_tokens=4, on_token=streamed.append))
        assert r.tokens == greedy.tokens and r.text == greedy.text == "".join(streamed)
        # sampled: each sequence draws what a request of its own seed draws, alone
        many = llm.continuations(GenerationRequest(prompt, 12, temperature=0.9, top_k=40, top_p=0.95, seed=3), 4, cache_type=0)
        for i, r in enumerate(many):
            assert r.tokens == llm.generate(GenerationRequest(prompt, 12, temperature=0.9, top_k=40, top_p=0.95, seed=3 + i)).tokens
        a = llm.continuations(GenerationRequest(prompt, 12, temperature=0.9, seed=3, draft_tokens=3), 4)
        b = llm.continuations(GenerationRequest(prompt, 12, temperature=0.9, seed=3, draft_tokens=3), 4)
        assert [r.tokens for r in a] == [r.tokens for r in b] and len({tuple(r.tokens) for r in a}) > 1
        assert all(len(r.tokens) == 12 or r.finish_reason == "eos" for r in a)
        if len(greedy.text) >= 6:
            stop = greedy.text[len(greedy.text) // 2:len(greedy.text) // 2 + 3]
            s = llm.continuations(GenerationRequest(prompt, 20, stop=[stop], draft_tokens=3), 2, cache_type=0)
            assert all(r.finish_reason == "stop" and r.text == greedy.text[:greedy.text.find(stop)] for r in s)
        assert [r.tokens for r in llm.continuations(GenerationRequest(prompt, 0), 2)] == [[], []]
        for bad in ((GenerationRequest(prompt, 10 ** 6), 1), (GenerationRequest(prompt, 4), 0), (GenerationRequest(prompt, 4, on_token=print), 1)):
            with pytest.raises(ValueError):
                llm.continuations(*bad)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("kind,kw", [("linear", dict(factor=2.5)), ("yarn", dict(factor=4.0, original_context=16)), ("factors", {}), ("part", {})])
def test_scaled_positions_in_the_model(jn, model_file, interleaved, kind, kw):
    """The keys that both caches hold of layer 0, which depend on the token alone: that of position 0, turned."""
    if kind == "part" and not interleaved:
        with jn.Llm.load(model_file) as llm, pytest.raises(ValueError, match="interleaved"):
            llm.model().set_rope(jn.Rope(32))
        return
    rot = 32 if kind == "part" else 64
    factors = (1 + np.arange(rot // 2) / 5).astype(np.float32) if kind == "factors" else None
    f, m = ref.rope_frequencies(rot, 10000.0, kind, kw.get("factor", 1.0), kw.get("original_context", 0), factors=factors)
    with jn.Llm.load(model_file) as llm:
        dec, vocab = llm.model(), llm.info().vocab
        dec.set_rope(jn.Rope(rot, 10000.0, interleaved, kind if kind in ("linear", "yarn") else None, freq_factors=factors, **kw))
        x = dec.embed([7])
        first = dec.decode(x[0], 0)
        raw = dec.kv_read(0, 0, 1)[0][0].astype(np.float64)
        raw[:, :rot] /= m
        positions = [0, 1, 5, 33]
        for p in positions:
            dec.decode(x[0], p)
        dec.prefill(np.repeat(x, 4, 0), 40, logits=False)
        pool = [torch.zeros(2, 4, 2, 16, 64, device="cuda") for _ in range(2)]
        cache = jn.PagedCache.wrap_dev(pool[0].data_ptr(), pool[1].data_ptr(), 2, 2, 64, 4, 16, 0)
        keep = [torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([2, 0, 3], [0, 40], [40], [0])]
        nb = jn.Batch(1, 40, 40, 40, keep[0].data_ptr(), 3, keep[1].data_ptr(), keep[2].data_ptr())
        xs, logits = torch.from_numpy(np.repeat(x, 40, 0)).cuda(), torch.empty(1, vocab, device="cuda")
        dec.step_dev(cache, nb, xs.data_ptr(), keep[3].data_ptr(), 1, logits.data_ptr())
        torch.cuda.synchronize()
        assert norm_err(logits[0].cpu().numpy(), first) <= 1e-4
        paged = pool[0][0, [2, 0, 3]].transpose(0, 1).reshape(2, 48, 64).cpu().numpy()
        scale = np.abs(raw).max()
        for p in positions + [40, 43]:
            want = ref.rotate(raw[None], [p], f, m, interleaved)[0]
            assert np.abs(dec.kv_read(0, p, 1)[0][0] - want).max() <= 1e-5 * scale   # (the few-row linears' 1e-6 beside the rotation's)
            if p < 40:
                assert np.abs(paged[:, p] - want).max() <= 1e-5 * scale


def test_files_that_scale_their_positions(jn, tmp_path, monkeypatch):
    """rope.scaling.*, rope.dimension_count and rope_freqs.weight of a file are what the model turns by; without them it turns as before."""
    factors = np.linspace(1, 8, 32).astype(np.float32)
    cases = {"plain": ({}, []), "linear": ({"llama.rope.scaling.type": "linear", "llama.rope.scaling.factor": 4.0}, []),
             "yarn": ({"llama.rope.scaling.type": "yarn", "llama.rope.scaling.factor": 4.0, "llama.rope.scaling.original_context_length": 16}, []),
             "factors": ({}, [("rope_freqs.weight", (32,), 0, factors)]), "part": ({"llama.rope.dimension_count": 32}, []),
             "magnitude": ({"llama.rope.scaling.attn_factor": 1.5}, []),
             "yarn with one": ({"llama.rope.scaling.type": "yarn", "llama.rope.scaling.factor": 4.0, "llama.rope.scaling.original_context_length": 16,
                                "llama.rope.scaling.attn_factor": 0.5, "llama.rope.scaling.yarn_beta_fast": 8.0}, []),
             "whole": ({"llama.rope.dimension_count": 64, "llama.rope.scaling.type": "none"}, [])}
    want = {"linear": dict(kind="linear", factor=4.0), "yarn": dict(kind="yarn", factor=4.0, original=16), "factors": dict(factors=factors),
            "yarn with one": dict(kind="yarn", factor=4.0, original=16, beta_fast=8.0)}
    gain = {"magnitude": 1.5, "yarn with one": 0.5}  # (on top of the scaling's own)
    for name, (meta, tensors) in cases.items():
        monkeypatch.setattr(test_llm, "write_gguf", lambda p, m, t: write_gguf(p, {**m, **meta}, t + tensors))
        path = tmp_path / f"{name}.gguf"
        test_llm.write_model(path, "llama", 11)
        rot = 32 if name == "part" else 64
        f, m = ref.rope_frequencies(rot, 10000.0, **want.get(name, {}))
        m *= gain.get(name, 1.0)
        with jn.Llm.load(path) as llm:
            dec = llm.model()
            x = dec.embed([7])[0]
            dec.decode(x, 0)
            raw = dec.kv_read(0, 0, 1)[0][0].astype(np.float64)
            raw[:, :rot] /= m
            dec.decode(x, 29)
            assert np.abs(dec.kv_read(0, 29, 1)[0][0] - ref.rotate(raw[None], [29], f, m, True)[0]).max() <= 1e-5 * np.abs(raw).max(), name
    monkeypatch.setattr(test_llm, "write_gguf", lambda p, m, t: write_gguf(p, {**m, "llama.rope.scaling.type": "longrope"}, t))
    test_llm.write_model(tmp_path / "other.gguf", "llama", 11)
    with pytest.warns(UserWarning, match="longrope"), jn.Llm.load(tmp_path / "other.gguf") as other, jn.Llm.load(tmp_path / "plain.gguf") as plain:
        x = plain.model().embed([7])[0]
        for llm in (other, plain):
            llm.model().decode(x, 29)
        assert np.array_equal(other.model().kv_read(0, 29, 1)[0], plain.model().kv_read(0, 29, 1)[0])


def test_recorded_step(jn, model_file):
    """A decode step of a batch recorded once and replayed with eager passes in between, each replay against an eager one; a larger pass cannot be recorded."""
    from jitnn_amd import _lib
    rng = np.random.default_rng(3)
    with jn.Llm.load(model_file) as llm:
        dec, vocab = llm.model(), llm.info().vocab
        b = ref.Batch(rng, [1] * 4, [9, 20, 33, 40], 16, shared=0, max_len=48)
        pool = [torch.randn(2, b.pages, 2, 16, 64, device="cuda") for _ in range(2)]
        cache = jn.PagedCache.wrap_dev(pool[0].data_ptr(), pool[1].data_ptr(), 2, 2, 64, b.pages, 16, 0)
        keep = [torch.from_numpy(a).cuda() for a in (b.tables, b.starts, np.array(b.lens, dtype=np.int32), np.arange(4, dtype=np.int32))]
        nb = jn.Batch(4, 4, 1, 48, keep[0].data_ptr(), b.width, keep[1].data_ptr(), keep[2].data_ptr())
        x, y, z = torch.randn(4, 256, device="cuda"), torch.empty(4, vocab, device="cuda"), torch.empty(4, vocab, device="cuda")
        side = torch.cuda.Stream()

        def step(out, stream):
            dec.step_dev(cache, nb, x.data_ptr(), keep[3].data_ptr(), 4, out.data_ptr(), stream.cuda_stream)

        with torch.cuda.stream(side):
            step(z, side)
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step(y, side)
            for i in range(4):
                x.normal_()
                keep[2].add_(i % 2)
                y.fill_(float("nan"))
                graph.replay()
                side.synchronize()
                step(z, side)
                side.synchronize()
                assert torch.equal(y, z) and torch.isfinite(y).all()
            graph2 = torch.cuda.CUDAGraph()
            wide = jn.Batch(1, 900, 900, 48, keep[0].data_ptr(), b.width, keep[1].data_ptr(), keep[2].data_ptr())
            with torch.cuda.graph(graph2, stream=side):
                rc = _lib.lib.jitnn_hip_llama_step_dev(dec.handle, cache.handle, wide, x.data_ptr(), None, 0, None, side.cuda_stream)
                y.add_(0)  # (a recording of something)
            assert rc == _lib.EINVAL and "recording" in _lib.last_error()
            # an eager pass that takes larger buffers, and a replay on those it was recorded with
            many = torch.zeros(900, 256, device="cuda")
            large = jn.Batch(1, 900, 900, 48, keep[0].data_ptr(), b.width, keep[1].data_ptr(), keep[2].data_ptr())
            dec.step_dev(cache, large, many.data_ptr(), 0, 0, 0, side.cuda_stream)
            side.synchronize()
            filler = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(8)]
            for _ in range(2):
                x.normal_()
                graph.replay()
                side.synchronize()
                step(z, side)
                side.synchronize()
                assert torch.equal(y, z) and torch.isfinite(y).all()
            del filler


def test_step_refusals(jn, model_file):
    from jitnn_amd import _lib
    with jn.Llm.load(model_file) as llm:
        dec = llm.model()
        x = torch.zeros(1024, device="cuda")
        p = x.data_ptr()
        nb = jn.Batch(1, 1, 1, 16, p, 1, p, p)
        call = _lib.lib.jitnn_hip_llama_step_dev
        for shape in ((3, 2, 64), (2, 4, 64), (2, 2, 128)):
            other = jn.PagedCache(*shape, 1, 16, 0)
            assert call(dec.handle, other.handle, nb, p, None, 0, None, None) == _lib.EINVAL, shape
        cache = jn.PagedCache(2, 2, 64, 1, 16, 0)
        assert call(dec.handle, cache.handle, nb, p, p, 2, p, None) == _lib.EINVAL
        assert call(dec.handle, cache.handle, nb, p, None, 1, p, None) == _lib.EINVAL
        assert call(dec.handle, cache.handle, nb, None, None, 0, None, None) == _lib.EINVAL
        assert call(dec.handle, None, nb, p, None, 0, None, None) == _lib.EINVAL
        with pytest.raises(ValueError):
            dec.set_rope(jn.Rope(128))
        dec.set_rope(jn.Rope(32, interleaved=True))
        with pytest.raises(ValueError, match="interleaved"):
            dec.set_rope_interleaved(False)

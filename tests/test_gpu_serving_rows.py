"""Rows of a pass that belong to no sequence, and sequences that cannot be attended, beside others: what they leave behind and that they reach nobody else."""
import numpy as np
import pytest
import torch

import serving_reference as ref
import test_llm
from helpers import norm_err

pytestmark = pytest.mark.gpu

TWICE = {False: 2e-4, True: 1e-2}  # the bars of few-row and many-row linears, for two results that may both be off by one


@pytest.fixture(scope="module")
def jn():
    import jitnn_amd
    jitnn_amd.init()
    return jitnn_amd


@pytest.fixture(scope="module")
def model_file(tmp_path_factory):
    path = tmp_path_factory.mktemp("rows") / "tiny.gguf"
    test_llm.write_model(path, "llama", 11)
    return path


# rows in front, rows of each sequence, rows behind: few-row linears, many-row ones, and a pass of nobody's rows alone
@pytest.mark.parametrize("front,counts,behind", [(0, [3, 1], 2), (2, [1, 4], 3), (5, [30, 25, 1], 4), (7, [90, 60], 9), (1, [1], 0), (3, [0, 0], 2), (40, [], 60)])
def test_rows_of_no_sequence_have_no_logits(jn, model_file, front, counts, behind):
    """NaN, whatever an earlier pass left in the model's buffers; and what they hold themselves reaches no row of a sequence."""
    rng = np.random.default_rng(front + behind)
    with jn.Llm.load(model_file) as llm:
        dec, vocab = llm.model(), llm.info().vocab
        table = torch.from_numpy(dec.embed(np.arange(vocab))).cuda()
        rows = front + sum(counts) + behind
        own = list(range(front, front + sum(counts)))
        b = ref.Batch(rng, counts, [c + 5 for c in counts], 16, max_len=128)
        starts = (b.starts + front).astype(np.int32)
        first = None
        for fill in (0.0, 3.0, float("nan"), float("inf")):
            pool = [torch.ones(2, b.pages, 2, 16, 64, device="cuda") * 0.1 for _ in range(2)]
            cache = jn.PagedCache.wrap_dev(pool[0].data_ptr(), pool[1].data_ptr(), 2, 2, 64, b.pages, 16, 0)
            x = torch.full((rows, 256), fill, device="cuda")
            if own:
                x[own] = table[torch.arange(len(own), device="cuda") * 7 % vocab]
            keep = [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (b.tables, starts, np.array(b.lens, dtype=np.int32), np.arange(rows, dtype=np.int32))]
            nb = jn.Batch(len(counts), rows, max([1] + counts), 128, keep[0].data_ptr(), b.width, keep[1].data_ptr(), keep[2].data_ptr())
            logits = torch.full((rows, vocab), 7.0, device="cuda")
            dec.step_dev(cache, nb, x.data_ptr(), keep[3].data_ptr(), rows, logits.data_ptr())
            torch.cuda.synchronize()
            stray = [r for r in range(rows) if r not in own]
            assert torch.isnan(logits[stray]).all()
            assert torch.isfinite(logits[own]).all()
            first = logits[own].clone() if first is None else first
            if np.isfinite(fill):
                assert torch.equal(logits[own], first)
            elif own:  # (a linear may take another way to the same result beside a row that is not finite)
                assert norm_err(logits[own].cpu().numpy(), first.cpu().numpy()) <= TWICE[rows > 64]


@pytest.mark.parametrize("counts", [[3, 1, 2], [30, 25, 40]])
def test_a_sequence_on_a_bad_page_reaches_no_other(jn, model_file, counts):
    """Its own rows are NaN through all layers; the logits of the other sequences' rows are those of a pass in which it is sound."""
    rng = np.random.default_rng(5)
    with jn.Llm.load(model_file) as llm:
        dec, vocab = llm.model(), llm.info().vocab
        table = torch.from_numpy(dec.embed(np.arange(vocab))).cuda()
        b = ref.Batch(rng, counts, [c + 20 for c in counts], 16, max_len=64)
        bad = list(range(int(b.starts[1]), int(b.starts[2])))
        out = []
        for page in (None, b.pages):
            pool = [torch.ones(2, b.pages, 2, 16, 64, device="cuda") * 0.1 for _ in range(2)]
            cache = jn.PagedCache.wrap_dev(pool[0].data_ptr(), pool[1].data_ptr(), 2, 2, 64, b.pages, 16, 0)
            tables = b.tables.copy()
            if page is not None:
                tables[1, 0] = page
            keep = [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (tables, b.starts, np.array(b.lens, dtype=np.int32), np.arange(b.tokens, dtype=np.int32))]
            nb = jn.Batch(3, b.tokens, max(counts), 64, keep[0].data_ptr(), b.width, keep[1].data_ptr(), keep[2].data_ptr())
            x, logits = table[torch.arange(b.tokens, device="cuda") * 5 % vocab].contiguous(), torch.empty(b.tokens, vocab, device="cuda")
            dec.step_dev(cache, nb, x.data_ptr(), keep[3].data_ptr(), b.tokens, logits.data_ptr())
            torch.cuda.synchronize()
            out.append(logits)
        others = [r for r in range(b.tokens) if r not in bad]
        assert torch.isnan(out[1][bad]).all() and torch.isfinite(out[0]).all()
        assert norm_err(out[1][others].cpu().numpy(), out[0][others].cpu().numpy()) <= TWICE[b.tokens > 64]


@pytest.mark.parametrize("length", [512, 513, 700])
def test_a_prompt_of_several_passes(jn, model_file, monkeypatch, length):
    """As many rows a pass as the default, and 16 of them: the same logits of the token after it, and of one more of each sequence (few-row linears on one side, many-row ones on the other)."""
    rng = np.random.default_rng(length)
    with jn.Llm.load(model_file) as llm:
        dec, vocab = llm.model(), llm.info().vocab
        prompt = [int(t) for t in rng.integers(0, vocab, length)]
        out = []
        for rows in (jn.SharedPrompt.PROMPT_ROWS, 16):
            monkeypatch.setattr(jn.SharedPrompt, "PROMPT_ROWS", rows)
            run = jn.SharedPrompt(dec, prompt, 3, length + 20, page_tokens=32, ggml_type=0)
            out.append((run.prompt_logits, run.step([0, 1, 2], [[5], [6], [7]])))
        assert norm_err(out[0][0], out[1][0]) <= TWICE[True] and norm_err(out[0][1], out[1][1]) <= TWICE[True]


@pytest.mark.parametrize("sequences", [4, 16, 90])
def test_a_pass_recorded_on_another_stream_than_it_ran_on(jn, model_file, sequences):
    """Run on the default stream, recorded on a stream of its own, replayed there, with eager passes on the default stream in between: every replay against an eager pass."""
    rng = np.random.default_rng(sequences)
    with jn.Llm.load(model_file) as llm:
        dec, vocab = llm.model(), llm.info().vocab
        b = ref.Batch(rng, [1] * sequences, [9 + i % 30 for i in range(sequences)], 16, max_len=48)
        pool = [torch.randn(2, b.pages, 2, 16, 64, device="cuda") for _ in range(2)]
        cache = jn.PagedCache.wrap_dev(pool[0].data_ptr(), pool[1].data_ptr(), 2, 2, 64, b.pages, 16, 0)
        keep = [torch.from_numpy(a).cuda() for a in (b.tables, b.starts, np.array(b.lens, dtype=np.int32), np.arange(sequences, dtype=np.int32))]
        nb = jn.Batch(sequences, sequences, 1, 48, keep[0].data_ptr(), b.width, keep[1].data_ptr(), keep[2].data_ptr())
        x, y, z = torch.randn(sequences, 256, device="cuda"), torch.empty(sequences, vocab, device="cuda"), torch.empty(sequences, vocab, device="cuda")

        def step(out):
            dec.step_dev(cache, nb, x.data_ptr(), keep[3].data_ptr(), sequences, out.data_ptr(), torch.cuda.current_stream().cuda_stream)

        step(z)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(y)
        for _ in range(4):
            x.normal_()
            y.fill_(float("nan"))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            step(z)
            torch.cuda.synchronize()
            assert torch.equal(y, z) and torch.isfinite(y).all()

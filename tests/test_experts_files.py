"""Files with experts that load refuses before it asks for a device."""
import numpy as np
import pytest

import test_gpu_experts_model as model_files
import test_llm

write_experts = model_files.write_experts


def refused(path, match):
    import jitnn_amd
    with pytest.raises(ValueError, match=match):
        jitnn_amd.Llm.load(path)


def without(monkeypatch, *keys):
    """write_gguf without these keys of the metadata, for files that a test makes from now on."""
    write = test_llm.write_gguf
    monkeypatch.setattr(test_llm, "write_gguf", lambda p, m, tensors: write(p, {k: v for k, v in m.items() if k not in keys}, tensors))


def test_a_file_without_a_length_of_its_layers(tmp_path, monkeypatch):
    """A dense file is asked for the length of dense layers, a file with experts for theirs where it has no other."""
    without(monkeypatch, "llama.feed_forward_length")
    test_llm.write_model(tmp_path / "dense.gguf", "llama", 3)
    refused(tmp_path / "dense.gguf", "no metadata key llama.feed_forward_length")


F32 = np.zeros(64, dtype=np.float32)


@pytest.mark.parametrize("name", ["blk.1.attn_q_norm.weight", "blk.0.attn_k_norm.weight", "blk.1.attn_q.bias", "blk.0.attn_output.bias", "blk.1.attn_sinks.weight", "blk.1.ffn_gate_inp.bias",
                                  "blk.0.ffn_gate_exps.bias", "blk.1.ffn_down_exps.bias", "blk.1.ffn_up_shexp.weight", "blk.0.ffn_gate_inp_shexp.weight", "blk.1.ffn_gate.weight",
                                  "blk.1.post_ffw_norm.weight", "blk.2.attn_q.weight", "output.bias", "token_embd_norm.weight"])
def test_tensors_that_nothing_reads(tmp_path, monkeypatch, name):
    """A file with experts whose layers have more than the decoder computes."""
    write_experts(tmp_path / "e.gguf", monkeypatch, extra=[(name, F32.shape, 0, F32)])
    refused(tmp_path / "e.gguf", name)


def test_every_layer_of_a_file_with_experts_is_looked_at(tmp_path, monkeypatch):
    """Dense layers in front of those with experts too; several names, the first ones of many."""
    write_experts(tmp_path / "e.gguf", monkeypatch, layers=(1,), extra=[("blk.0.attn_q.bias", F32.shape, 0, F32)])
    refused(tmp_path / "e.gguf", "blk.0.attn_q.bias")
    names = [f"blk.{l}.attn_{n}.bias" for l in (0, 1) for n in "qkv"]
    write_experts(tmp_path / "f.gguf", monkeypatch, extra=[(n, F32.shape, 0, F32) for n in names])
    refused(tmp_path / "f.gguf", "and 2 more")


def test_what_a_file_may_have(tmp_path, monkeypatch):
    """All that is read, and the rotary positions' own tensors: nothing left over.  A dense file goes on with a warning."""
    from jitnn_amd.gguf_file import GgufFile
    from jitnn_amd.llm import Llm
    write_experts(tmp_path / "e.gguf", monkeypatch, bias=True, layers=(1,), extra=[("rope_freqs.weight", (32,), 0, np.ones(32, dtype=np.float32))])
    f = GgufFile.open(tmp_path / "e.gguf")
    assert Llm._unread(f, 2, {1}) == [] and len(Llm._unread(f, 2, set())) == 5 and len(Llm._unread(f, 1, set())) == 4 + 2 + 5
    f.close()
    monkeypatch.undo()
    write = test_llm.write_gguf
    monkeypatch.setattr(test_llm, "write_gguf", lambda p, m, tensors: write(p, m, tensors + [("blk.0.attn_q.bias", F32.shape, 0, F32)]))
    test_llm.write_model(tmp_path / "dense.gguf", "llama", 3)
    import jitnn_amd
    with pytest.warns(UserWarning, match="blk.0.attn_q.bias"):
        try:
            jitnn_amd.Llm.load(tmp_path / "dense.gguf").close()
        except Exception as e:  # (no device here)
            assert not isinstance(e, ValueError), e


def test_whether_weights_sum_to_one(tmp_path, monkeypatch):
    """Without the key only where the architecture says so; with it whatever the file says."""
    from jitnn_amd.gguf_file import GgufFile
    from jitnn_amd.llm import Llm

    def routing(name):
        f = GgufFile.open(tmp_path / name)
        try:
            return Llm._routing(f, f.architecture())
        finally:
            f.close()

    write_experts(tmp_path / "a.gguf", monkeypatch)
    assert routing("a.gguf") == dict(used=2, gating="softmax", normalise=True, scale=1.0)
    write_experts(tmp_path / "b.gguf", monkeypatch, meta={"llama.expert_weights_norm": False, "llama.expert_weights_scale": 2.5, "llama.expert_gating_func": 2}.items())
    assert routing("b.gguf") == dict(used=2, gating="sigmoid", normalise=False, scale=2.5)
    monkeypatch.setattr(model_files, "write_gguf", lambda p, m, tensors, write=model_files.write_gguf: write(
        p, {k.replace("llama.", "testarch.", 1): "testarch" if k == "general.architecture" else v for k, v in m.items()}, tensors))
    write_experts(tmp_path / "c.gguf", monkeypatch)
    refused(tmp_path / "c.gguf", "no testarch.expert_weights_norm")
    for norm in (True, False):
        write_experts(tmp_path / "d.gguf", monkeypatch, meta={"llama.expert_weights_norm": norm}.items())
        assert routing("d.gguf")["normalise"] is norm

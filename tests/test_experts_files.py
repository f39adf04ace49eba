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

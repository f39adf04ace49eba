"""Files whose rotary metadata no rotary positions can be made of: they load with a warning and turn by the plain positions, as they did before that metadata was read."""
import numpy as np
import pytest

import test_llm
from gguf_writer import write_gguf

pytestmark = pytest.mark.gpu

S = "llama.rope.scaling."
ODD = {
    "no dimensions": ({"llama.rope.dimension_count": 0}, []),
    "an odd number of dimensions": ({"llama.rope.dimension_count": 33}, []),
    "dimensions that are no number": ({"llama.rope.dimension_count": "64"}, []),
    "yarn without a context": ({S + "type": "yarn", S + "factor": 4.0, S + "original_context_length": 0}, []),
    "yarn by a negative factor": ({S + "type": "yarn", S + "factor": -4.0, S + "original_context_length": 16, S + "attn_factor": 0.5}, []),
    "yarn without a slow end": ({S + "type": "yarn", S + "factor": 4.0, S + "original_context_length": 16, S + "yarn_beta_slow": 0.0}, []),
    "a negative factor": ({S + "type": "linear", S + "factor": -2.0}, []),
    "an infinite factor": ({S + "type": "linear", S + "factor": float("inf")}, []),
    "a negative gain": ({S + "attn_factor": -1.5}, []),
    "a kind that is no text": ({S + "type": 3}, []),
    "a frequency factor of 0": ({}, [("rope_freqs.weight", (32,), 0, np.array([1.0] * 31 + [0.0], dtype=np.float32))]),
    "a negative frequency factor": ({}, [("rope_freqs.weight", (32,), 0, np.array([-1.0] + [2.0] * 31, dtype=np.float32))]),
    "too few frequency factors": ({}, [("rope_freqs.weight", (31,), 0, np.ones(31, dtype=np.float32))]),
    "frequency factors in 16 bits": ({}, [("rope_freqs.weight", (32,), 1, np.ones(32, dtype=np.float16))]),
}


@pytest.mark.parametrize("case", ODD)
def test_files_of_odd_rotary_metadata_load(tmp_path, monkeypatch, case):
    import jitnn_amd as jn
    jn.init()
    read = {}
    for name, (meta, tensors) in (("plain", ({}, [])), ("odd", ODD[case])):
        monkeypatch.setattr(test_llm, "write_gguf", lambda p, m, t: write_gguf(p, {**m, **meta}, t + tensors))
        test_llm.write_model(tmp_path / f"{name}.gguf", "llama", 11)
    with pytest.warns(UserWarning, match="rotary"), jn.Llm.load(tmp_path / "odd.gguf") as odd, jn.Llm.load(tmp_path / "plain.gguf") as plain:
        for name, llm in (("odd", odd), ("plain", plain)):
            dec = llm.model()
            dec.decode(dec.embed([7])[0], 29)
            read[name] = dec.kv_read(0, 29, 1)[0]
    assert np.array_equal(read["odd"], read["plain"])

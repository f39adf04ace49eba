"""The host side of a served batch: what a shared prompt's steps take and refuse before anything is launched.  No device needed."""
import numpy as np
import pytest


@pytest.fixture
def run():
    """Three sequences behind a prompt of 20 tokens whose passes are only written down."""
    from jitnn_amd.serving import SharedPrompt

    class Logits:
        ptr = 0

        @staticmethod
        def get(n):
            return np.zeros(n, dtype=np.float32)

    s = SharedPrompt.__new__(SharedPrompt)
    s._vocab, s._rows, s.max_len, s.shared = 50, 4, 40, 1
    s._tables, s._verify, s._logits = np.zeros((3, 3), dtype=np.int32), None, Logits
    s.lens, s.passes = [20, 20, 20], []
    s._pass = lambda which, tokens, lens, shared, rows: s.passes.append((list(which), tokens, lens))
    return s


def test_a_step_advances_the_sequences_that_an_iterator_names(run):
    assert run.step(iter([2, 0]), [[1, 2], [3]]).shape == (3, 50)
    assert run.lens == [21, 20, 22] and [p[2] for p in run.passes] == [[22, 21]]
    run.step((i for i in (0, 1)), [[1], [2]])
    assert run.lens == [22, 21, 22]


def test_a_sequence_counted_from_the_end_is_the_same_one(run):
    """Named twice, once so and once so, it would write two tokens to one position."""
    for call in (lambda w, t: run.step(w, t), lambda w, t: run.verify(w, t, [0.0] * 2, np.zeros((2, 2)))):
        with pytest.raises(ValueError, match="sequences"):
            call([-1, 2], [[1], [2]])
        with pytest.raises(IndexError):
            call([0, 3], [[1], [2]])
    assert run.passes == []
    run.step([-1], [[1]])
    assert run.lens == [20, 20, 21] and run.passes[0][0] == [2]


@pytest.mark.parametrize("temperatures,uniforms", [([1.0], np.zeros((3, 2))), ([1.0, 0.5, 0.2], np.zeros((3, 2))), ([], np.zeros((3, 2))), ([1.0, 0.5], np.zeros((2, 2))),
                                                   ([1.0, 0.5], np.zeros((4, 2))), ([1.0, 0.5], np.zeros(5)), ([1.0, 0.5], np.zeros((3, 1))), ([1.0, 0.5], np.zeros((2, 3)))])
def test_verification_refuses_other_numbers_of_numbers(run, temperatures, uniforms):
    """Before the pass: too few would leave those of an earlier call in use."""
    with pytest.raises(ValueError, match="temperatures"):
        run.verify([0, 2], [[1, 2], [3]], temperatures, uniforms)
    assert run.passes == [] and run.lens == [20, 20, 20]


def test_numbers_just_below_one_stay_below_it(run, monkeypatch):
    """64-bit numbers in [0, 1) that 32 bits would round up to 1, which no longer keeps a certain draft."""
    from jitnn_amd import serving
    seen = {}

    class Array:
        def __init__(self, count, dtype):
            self.count, self.ptr = count, 0

        def put(self, values):
            seen[self.count] = np.array(values)
            return self

        def get(self, n):
            return np.zeros(n, dtype=np.int32)

    monkeypatch.setattr(serving, "DeviceArray", Array)
    monkeypatch.setattr(serving, "verify_workspace", lambda *a: 999)
    monkeypatch.setattr(serving, "verify_drafts_dev", lambda *a: None)
    run._ints, run._tok = [Array(1, np.int32)] * 4, Array(1, np.int32)
    run.verify([0], [[1, 2]], [1.0], [[1 - 2.0 ** -30, 0.25], [0.5, 1 - 2.0 ** -53]])
    assert seen[24].dtype == np.float32 and seen[24].max() == np.float32(1 - 2.0 ** -24) and seen[24].shape == (2, 2)

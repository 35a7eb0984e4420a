"""Engine.score_tokens' arguments, with a stand-in for the library's handle: what the kernels are given holds a value for
each position, and a call that is refused has not touched the sequence."""
import numpy as np
import pytest
import torch

from lpta.engine import Engine


class Handle:
    device = 0

    def __init__(self):
        self.calls = []

    def call(self, name, *args):
        self.calls.append((name, args))


@pytest.fixture
def engine(monkeypatch):
    monkeypatch.setattr(torch, "device", lambda *_: "cpu")
    eng = Engine.__new__(Engine)
    eng.cfg, eng.rt = {"vocab": 50}, Handle()
    return eng


@pytest.mark.parametrize("shape", [(6,), (1, 6), (2, 3), (6, 1)])
def test_a_target_for_each_position(engine, shape):
    got = engine.score_tokens(np.arange(6, dtype=np.int64).reshape(shape), top=3)
    (prefill, (seq, tokens, n, _)), (score, args) = engine.rt.calls
    assert (prefill, score, seq, n) == ("tl_prefill_logits", "tl_token_logprobs", 0, 6)
    logits, vocab, _, rows, width, targets, top, *out = args
    assert tokens.tolist() == list(range(6)) and logits.shape == (6, 50) and (rows, vocab, width, top) == (6, 50, 50, 3)
    assert targets.tolist() == [1, 2, 3, 4, 5, -1]
    assert [tuple(o.shape) for o in out] == [(6,), (6,), (6, 3), (6, 3)] and got["top_ids"].shape == (6, 3)


@pytest.mark.parametrize("top", [-1, 33, 51])
def test_refused_before_the_prompt_runs(engine, top):
    with pytest.raises(ValueError, match="top"):
        engine.score_tokens([1, 2, 3], top=top)
    assert engine.rt.calls == []

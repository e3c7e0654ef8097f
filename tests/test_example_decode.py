"""The example of a token decoder runs, keeps to its grammar and repeats itself."""
import importlib.util
import os

import numpy as np
import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


def test_decode_tokens(gpu):
    spec = importlib.util.spec_from_file_location("decode_tokens", os.path.join(ROOT, "examples", "decode_tokens.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    model = example.Decoder(0, layers=2, heads=4, vocabulary=301)
    r = np.random.default_rng(1)
    states = r.normal(size=(3, 40, model.width)).astype(np.float32)
    lengths, prompt = np.array([40, 1, 23], np.int32), r.integers(1, 301, (3, 9))
    first, seconds = example.generate(model, states, lengths, prompt, 20, block=16)
    assert first.shape == (3, 20) and len(seconds) == 20
    assert (first[:, :-1] != model.END).all() and (first >= 0).all() and (first < 301).all()
    again, _ = example.generate(model, states, lengths, prompt, 20, block=16)
    assert np.array_equal(first, again)
    # an utterance's tokens are its own: alone, they are the same
    alone, _ = example.generate(model, states[2:], lengths[2:], prompt[2:], 20, block=16)
    assert np.array_equal(alone[0], first[2])

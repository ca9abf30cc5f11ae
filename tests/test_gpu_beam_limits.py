"""Beam search and moved rows at their limits, on the GPU: searches with fewer texts than beams, indices out of range,
extreme values."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import beam_reference as ref
from test_gpu_beam_model import _cache, _ids, _model

pytestmark = pytest.mark.gpu


def _only(*tokens, words=16):
    mask = torch.zeros(words, dtype=torch.int32)
    for t in tokens:
        mask[t // 32] |= 1 << (t % 32)
    return mask


def test_generate_beam_of_fewer_texts_than_beams():
    """One continuation in all: it comes once, the other places hold the prompt, padded, with score -inf."""
    model = _model()
    ids = _ids(2)
    for eos, tail in ((None, [7] * 4), (7, [7])):
        got, scores = model.generate_beam(ids, 4, num_beams=3, num_return_sequences=3, allowed=_only(7), eos_token_id=eos,
                                          pad_token_id=500, return_scores=True)
        for b in range(2):
            text = ids[b].tolist() + tail
            assert got[3 * b].tolist() == text
            for i in (1, 2):
                assert got[3 * b + i].tolist() == ids[b].tolist() + [500] * len(tail)
        assert torch.isfinite(scores[::3]).all() and (scores.view(2, 3)[:, 1:] == -float("inf")).all()


def test_generate_beam_of_nan_logits_keeps_the_prompt():
    model = _model()
    ids = _ids(2)
    bias = torch.zeros(512)
    bias[3] = float("nan")
    got, scores = model.generate_beam(ids, 4, num_beams=2, num_return_sequences=2, bias=bias, return_scores=True)
    assert got.shape[1] == 6 and torch.equal(got[:, :5], ids.repeat_interleave(2, 0)) and scores.isnan().all()


@pytest.mark.parametrize("use_graph", [True, False])
def test_generate_beam_with_a_filler_outside_the_vocabulary(use_graph):
    """Prompts that end at different steps: the filler stands in the result alone."""
    model = _model()
    ids = _ids(3)
    want = model.generate_beam(ids, 12, num_beams=2, eos_token_id=80, pad_token_id=0, use_graph=use_graph, return_scores=True)
    got = model.generate_beam(ids, 12, num_beams=2, eos_token_id=80, pad_token_id=-100, use_graph=use_graph, return_scores=True)
    assert torch.equal(torch.where(got[0] == -100, 0, got[0]), want[0]) and torch.equal(got[1], want[1])

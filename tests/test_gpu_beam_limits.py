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


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_select_of_values_whose_parts_leave_fp32(dtype):
    """Scores near the type's lowest value under logits near its highest: s + (x - lse) is finite in 64 bits where
    s - lse alone is not in 32, and has the order of its 64-bit value."""
    import rwkv7mi as mi

    top = 3.0e38
    x = torch.full((4, 9000), -2.0e38)
    x[:, 4000:4012] = top - torch.arange(12) * 2.0 ** 121  # (steps that both types hold)
    x[2:] = x[2:].flip(1)
    x = x.to(torch.float32 if dtype == "fp32" else torch.bfloat16)
    s = torch.tensor([[-2.9e38, -1.0], [-3.0e38, -3.1e38]])
    for m in (2, 12, 64):
        v = ref.values(x.double().numpy().reshape(2, 2, 9000), s.numpy())
        with np.errstate(over="ignore"):
            v = np.where(np.isfinite(v.astype(np.float32)), v, -np.inf)  # (what rounds to -inf comes by index)
        want = ref.select(v, m)
        val, tok, row = (t.cpu().numpy() for t in mi.beam_select(x.cuda(), s.cuda(), m))
        assert np.array_equal(tok, want[1]) and np.array_equal(row - 2 * np.arange(2)[:, None], want[2])
        fine = np.isfinite(want[0])
        assert np.array_equal(np.isneginf(val), ~fine)
        # rounded once; lse is the row's maximum to the last bit here
        assert (np.abs(val[fine] - want[0][fine]) <= 2.0 ** -24 * np.abs(want[0][fine])).all()

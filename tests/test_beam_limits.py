"""Beam search and moved rows at their limits, on the CPU: searches with fewer texts than beams, states and buffers
that a call has to refuse, caches that the kernels do not serve."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import beam_reference as ref

KEYS = ("tokens", "lengths", "scores", "prompt_lengths", "finished_tokens", "finished_lengths", "finished_scores", "done")


def _search(mi, ids, beams, room, logits, ends=(), steps=None):
    """The state behind ``steps`` steps (default: until the rows are full) over ``logits [beams, n]``."""
    start = mi.BeamState.start(torch.tensor(ids), beams, room)
    s = {k: getattr(start, k).numpy().copy() for k in KEYS}
    prompts = len(ids)
    x = np.broadcast_to(np.asarray(logits, np.float64), (prompts, beams, len(logits[0]) if np.ndim(logits) > 1 else len(logits)))
    for _ in range(room - len(ids[0]) if steps is None else steps):
        val, tok, beam = ref.select(ref.values(x, s["scores"]), (1 + len(ends)) * beams)
        _, _, s = ref.step((val.astype(np.float32), tok, beam), s, ends, 1.0, False)
    return mi.BeamState(**{k: torch.from_numpy(v) for k, v in s.items()})


def _texts(found, prompt=0):
    tokens, lengths, scores = found
    return [(t[:n].tolist(), float(s)) for t, n, s in zip(tokens[prompt], lengths[prompt], scores[prompt])]


ONE = np.where(np.arange(8) == 5, 0.0, -np.inf)  # one token can follow


def test_best_of_a_full_search_gives_no_text_twice():
    import rwkv7mi as mi

    s = _search(mi, [[1, 2]], 3, 4, ONE)
    assert s.done.all()
    # one text in all: the places that are left hold the prompt
    assert _texts(s.best(3)) == [([1, 2, 5, 5], 0.0), ([1, 2], -np.inf), ([1, 2], -np.inf)]
    assert _texts(s.best(1)) == [([1, 2, 5, 5], 0.0)]


def test_best_of_a_search_that_ended_early():
    import rwkv7mi as mi

    s = _search(mi, [[1, 2], [3, 4]], 3, 9, ONE, ends=(5,))
    assert s.done.all()
    for b, prompt in enumerate(([1, 2], [3, 4])):
        assert _texts(s.best(3), b) == [(prompt + [5], 0.0), (prompt, -np.inf), (prompt, -np.inf)]


def test_best_of_a_running_search_with_fewer_texts_than_beams():
    import rwkv7mi as mi

    s = _search(mi, [[1, 2]], 3, 9, ONE, steps=2)
    assert not s.done.any()
    assert _texts(s.best(3)) == [([1, 2, 5, 5], 0.0), ([1, 2], -np.inf), ([1, 2], -np.inf)]
    # before the first step: the prompt itself
    assert _texts(mi.BeamState.start(torch.tensor([[1, 2]]), 3, 9).best(2)) == [([1, 2], 0.0), ([1, 2], -np.inf)]


def test_best_where_the_logits_are_nan():
    """A search that met NaN is over without hypotheses: its texts, their scores NaN, not rows of nothing."""
    import rwkv7mi as mi

    s = _search(mi, [[1, 2]], 3, 9, np.full(8, np.nan), steps=1)
    assert s.done.all()
    got = _texts(s.best(2))
    assert all(t[:2] == [1, 2] and len(t) == 3 and np.isnan(v) for t, v in got) and got[0][0] != got[1][0]


def test_best_without_room_for_a_token():
    import rwkv7mi as mi

    s = mi.BeamState.start(torch.tensor([[1, 2]]), 2, 2)
    s.done.fill_(True)
    assert _texts(s.best(2)) == [([1, 2], 0.0), ([1, 2], -np.inf)]


def test_best_where_the_penalty_outgrows_fp32():
    """Running texts whose scores round to -inf under the penalty are texts all the same."""
    import rwkv7mi as mi

    s = _search(mi, [[1, 2]], 2, 9, np.array([0.0, 1.0, 2.0]), steps=3)
    assert [len(t) for t, _ in _texts(s.best(2, length_penalty=-400.0))] == [5, 5]


class _Searcher:
    """What ``generate_beam`` needs of a model, on the CPU: logits that end prompt 0 at once, and a record of
    the tokens that it is fed."""

    class config:
        vocab_size = 8

    device = torch.device("cpu")

    def __init__(self):
        self.fed = []

    def forward(self, ids, past_key_values=None, use_graph=None):
        from types import SimpleNamespace as Of

        self.fed.append(ids.clone())
        x = torch.full((ids.shape[0], 1, 8), -2.0)
        first = (ids == 1).any(1) if past_key_values is None else torch.arange(ids.shape[0]) < ids.shape[0] // 2
        x[first, :, 7] = 9.0
        cache = Of(batch_repeat_interleave=lambda k: None, reorder_cache=lambda rows: None)
        return Of(logits=x, past_key_values=cache)


@pytest.mark.parametrize("pad", [-100, -1, 0, 7, 1 << 40])
def test_generate_beam_feeds_the_model_tokens_of_its_own(monkeypatch, pad):
    """A filler of any value: done prompts are padded with it, and the model never sees it."""
    import rwkv7mi as mi
    from rwkv7mi import model as module

    def step(logits, state, *, next_tokens, rows, workspace, eos_token_id, length_penalty, early_stopping, pad_token_id):
        s = {k: getattr(state, k).numpy() for k in KEYS}
        x = logits.double().numpy().reshape(*s["scores"].shape, -1)
        val, tok, beam = ref.select(ref.values(x, s["scores"]), (1 + len(eos_token_id)) * s["scores"].shape[1])
        nxt, at, new = ref.step((val.astype(np.float32), tok, beam), s, eos_token_id, length_penalty, early_stopping,
                                pad_token_id)
        for k, v in new.items():
            getattr(state, k).copy_(torch.from_numpy(v))
        next_tokens.copy_(torch.from_numpy(nxt))
        rows.copy_(torch.from_numpy(at))

    monkeypatch.setattr(module, "beam_step", step)
    model = _Searcher()
    got = mi.model.NativeRWKV7ForCausalLM.generate_beam(model, torch.tensor([[1, 1], [2, 2]]), 5, num_beams=1, eos_token_id=7,
                                                        pad_token_id=pad, use_graph=False)
    assert got[0].tolist() == [1, 1, 7] + [pad] * 4 and got[1, :2].tolist() == [2, 2] and got.shape == (2, 7)
    assert len(model.fed) == 5 and all(((0 <= t) & (t < 8)).all() for t in model.fed)


@pytest.fixture
def calls(monkeypatch):
    """The library calls, recorded instead of run."""
    from rwkv7mi import _lib

    made = []
    monkeypatch.setattr(_lib, "require_same_device", lambda *t, name: None)
    monkeypatch.setattr(_lib, "stream_of", lambda t: 0)
    monkeypatch.setattr(_lib, "on_device", lambda t: _lib._HERE)
    monkeypatch.setattr(_lib, "call", lambda name, *args: made.append((name, args)))
    return made


def _state(mi, room=9):
    return mi.BeamState.start(torch.zeros(2, 4, dtype=torch.int64), 3, room)


@pytest.mark.parametrize("key", KEYS)
def test_a_state_whose_memory_was_replaced_is_refused(calls, key):
    """resize_, set_ and .data give a tensor other memory or another room: the state's addresses are not its own."""
    import rwkv7mi as mi

    x = torch.zeros(6, 50)
    for change in (lambda t: t.resize_(4096), lambda t: t.set_(t.clone()), lambda t: setattr(t, "data", t.clone()),
                   lambda t: t.untyped_storage().resize_(0)):
        for side in ("in", "out"):
            s, o = _state(mi), _state(mi)
            change(getattr(s if side == "in" else o, key))
            with pytest.raises(ValueError, match="BeamState"):
                mi.beam_step(x, s, out=o)
    assert not calls
    s = _state(mi)
    s.tokens.resize_(2, 3, 5)  # (less room in the same memory)
    with pytest.raises(ValueError, match="BeamState"):
        mi.beam_step(x, s)
    assert not calls
    s = _state(mi)
    s.tokens.fill_(3)  # (written into: still its own)
    mi.beam_step(x, s)
    assert len(calls) == 1


def test_a_state_is_copied_and_pickled():
    import copy
    import pickle

    import rwkv7mi as mi

    s = _state(mi)
    s.tokens.random_(0, 9)
    same = copy.copy(s)
    assert type(same) is mi.BeamState and all(getattr(same, k).data_ptr() == getattr(s, k).data_ptr() for k in KEYS)
    for other in (copy.deepcopy(s), pickle.loads(pickle.dumps(s))):
        assert type(other) is mi.BeamState and other._addresses != s._addresses and other._shape == s._shape
        assert all(torch.equal(getattr(other, k), getattr(s, k)) for k in KEYS)
        other.tokens.zero_()
        assert s.tokens.any()


def test_beam_select_refuses_outputs_among_what_it_reads(calls):
    import rwkv7mi as mi

    s = torch.zeros(2, 3)
    tok, row = (torch.zeros(2, 6, dtype=torch.int64) for _ in range(2))
    need = mi.beam.beam_workspace_bytes(6, 50, 6)
    big = torch.zeros(1 << 16)
    x = big[:300].view(6, 50)
    bytes_ = big.view(torch.uint8)
    for args, kw in (((x, big[400:406].view(2, 3)), dict(out=(big[400:412].view(2, 6), tok, row))),  # the scores
                     ((x, s), dict(out=(big[290:302].view(2, 6), tok, row))),                        # the logits
                     ((x, s), dict(workspace=bytes_[:need])),
                     ((x, big[402:408].view(2, 3)), dict(workspace=bytes_[1600:])),
                     ((x, s), dict(out=(big[500:512].view(2, 6), tok, row), workspace=bytes_[2000:])),
                     ((x, s), dict(out=(big[500:512].view(2, 6), *torch.zeros(1, 24, dtype=torch.int64).expand(2, 24).reshape(-1)
                                        .as_strided((2, 2, 6), (6, 6, 1)).unbind(0))))):
        with pytest.raises(ValueError, match="overlap"):
            mi.beam_select(*args, **kw)
    assert not calls
    mi.beam_select(x, s, out=(big[500:512].view(2, 6), tok, row), workspace=bytes_[2048:])
    mi.beam_select(x[:0], s[:0], out=(big[:0].view(0, 6), tok[:0], row[:0]))
    assert len(calls) == 2


def test_beam_step_refuses_buffers_among_its_state(calls):
    import rwkv7mi as mi

    x, s, o = torch.zeros(6, 50), _state(mi), _state(mi)
    need = mi.beam.beam_workspace_bytes(6, 50, 3)
    room = torch.zeros(need + 4096, dtype=torch.int64)
    for kw in (dict(next_tokens=s.tokens.view(-1)[:6]), dict(rows=s.tokens.view(-1)[5:11]),
               dict(rows=s.finished_tokens.view(-1)[-6:]), dict(out=o, next_tokens=o.tokens.view(-1)[:6]),
               dict(workspace=room.view(torch.uint8), rows=room[:6]), dict(workspace=room.view(torch.uint8), next_tokens=room[9:15]),
               dict(next_tokens=room[:6], rows=room[5:11])):
        with pytest.raises(ValueError, match="overlap"):
            mi.beam_step(x, s, **kw)
    shared = torch.zeros(1 << 16, dtype=torch.uint8)
    parts = dict(scores=shared[64:88].view(torch.float32).view(2, 3))
    in_shared = mi.BeamState(**{**{k: getattr(_state(mi), k) for k in KEYS}, **parts})
    for args, kw in (((x, in_shared), dict(workspace=shared)),
                     ((shared[:1200].view(torch.float32).view(6, 50), s), dict(workspace=shared)),
                     ((shared[:1200].view(torch.float32).view(6, 50), s), dict(rows=shared[800:848].view(torch.int64)))):
        with pytest.raises(ValueError, match="overlap"):
            mi.beam_step(*args, **kw)
    assert not calls
    mi.beam_step(x, s, out=o, workspace=room.view(torch.uint8)[128:], rows=room[:6], next_tokens=room[6:12])
    mi.beam_step(x, in_shared, workspace=shared[88:], rows=shared[:48].view(torch.int64))
    assert len(calls) == 2


def test_lengths_lie_within_the_ids():
    import rwkv7mi as mi

    ids = torch.zeros(2, 4, dtype=torch.int64)
    for bad in ([5, 2], [2, 9], [50, 1], [-1, 2], torch.tensor([2, 5]), np.array([2, -3]), [2], [1, 2, 3], 2, [[1, 2]], [1 << 33, 1]):
        with pytest.raises((ValueError, OverflowError)):
            mi.BeamState.start(ids, 3, 9, lengths=bad)
    for good in ([4, 0], torch.tensor([1, 4], dtype=torch.int32), np.array([2, 3])):
        s = mi.BeamState.start(ids, 3, 9, lengths=good)
        assert s.prompt_lengths.tolist() == [int(n) for n in good] and s.lengths.tolist() == [int(n) for n in good for _ in range(3)]


def test_scores_made_contiguous_live_until_the_launch(monkeypatch, calls):
    import weakref

    import rwkv7mi as mi
    from rwkv7mi import _lib

    made, alive = [], []
    plain = torch.Tensor.contiguous

    def contiguous(t, *args, **kw):
        out = plain(t, *args, **kw)
        made.append((weakref.ref(out), out.data_ptr()))
        return out

    monkeypatch.setattr(torch.Tensor, "contiguous", contiguous)
    monkeypatch.setattr(_lib, "call", lambda name, *args: alive.extend(r() is not None for r, at in made if at in args))
    mi.beam_select(torch.zeros(6, 50), torch.zeros(3, 2).t())
    assert alive == [True]


@pytest.mark.parametrize("room", [(1 << 30) + 1, 2 ** 31 - 512, 2 ** 31 - 2])
def test_rooms_that_pass_32_bits_are_refused(room):
    """(the lanes' offsets into a text, steps of 512 tokens, are 32 bits wide)"""
    import ctypes

    from rwkv7mi import _lib

    state = (ctypes.c_void_p * 8)(*[(1 << 20) + 4096 * i for i in range(8)])
    other = (ctypes.c_void_p * 8)(*[(1 << 21) + 4096 * i for i in range(8)])
    at = 1 << 22
    assert _lib.load().rwkv7mi_beam_step(at, 2, 3, 100, 100, 1, 0, None, 0, 1.0, 0, 0, state, other, room, at, at, at, 1 << 20,
                                         None) == -1
    assert b"room" in _lib.load().rwkv7mi_last_error()

"""Refusals of the beam search's and the moved rows' entry points, on the CPU: no call here reaches a
launch.  The plain reference's own rules are checked too."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import beam_reference as ref

A = 1 << 20  # an aligned address that is never read


def _lib():
    from rwkv7mi import _lib

    return _lib.load()


def _select(x=A, prompts=2, beams=3, n=100, ldx=100, dt=1, scores=A, m=6, o1=A, o2=A, o3=A, ws=A, nws=1 << 20):
    return _lib().rwkv7mi_beam_select(x, prompts, beams, n, ldx, dt, scores, 0, m, o1, o2, o3, ws, nws, None)


@pytest.mark.parametrize("kw", [dict(x=0), dict(scores=0), dict(o1=0), dict(o2=0), dict(o3=0), dict(prompts=-1), dict(beams=0),
                                dict(n=0), dict(ldx=-1), dict(dt=5), dict(m=0), dict(m=129), dict(beams=129, m=4),
                                dict(n=2, m=7), dict(n=1 << 23), dict(prompts=65536, beams=1), dict(x=A + 1)])
def test_select_entry_refuses(kw):
    assert _select(**kw) == -1


@pytest.mark.parametrize("prompts,beams", [(2 ** 57, 128), (2 ** 62, 4), (16384, 4), (65536, 1)])
def test_entries_count_rows_without_wrapping(prompts, beams):
    for call in (_select, lambda **kw: _step(ends=(), **kw)):
        assert call(prompts=prompts, beams=beams) == -1
        assert b"65535 rows" in _lib().rwkv7mi_last_error()


def test_select_entry_wants_its_workspace():
    need = _lib().rwkv7mi_beam_workspace_bytes(6, 100, 6)
    assert need >= 6 * 6 * 8
    assert _select(ws=None) == -3 and _select(ws=A + 4) == -3 and _select(nws=need - 1) == -3
    assert _select(prompts=0, ws=None) == 0
    assert _lib().rwkv7mi_beam_workspace_bytes(0, 100, 6) == 0


def _step(ends=(1,), n_ends=None, prompts=2, beams=3, room=9, lp=1.0, early=0, hole=None, nxt=A, rows=A, ws=A, nws=1 << 20,
          n=100):
    sides = [(ctypes.c_void_p * 8)(*[A + 4096 * i for i in range(8)]) for _ in range(2)]
    if hole is not None:
        sides[hole // 8][hole % 8] = None
    return _lib().rwkv7mi_beam_step(A, prompts, beams, n, n, 1, 0, (ctypes.c_int64 * max(len(ends), 1))(*ends),
                                    len(ends) if n_ends is None else n_ends, lp, early, 0, *sides, room, nxt, rows, ws, nws,
                                    None)


@pytest.mark.parametrize("kw", [dict(n_ends=-1), dict(ends=range(9)), dict(beams=64, ends=(1, 2)), dict(room=0), dict(early=3),
                                dict(early=-1), dict(lp=float("nan")), dict(nxt=0), dict(rows=0), dict(n=1, ends=(0, 0)),
                                dict(hole=0), dict(hole=7), dict(hole=8), dict(hole=13)])
def test_step_entry_refuses(kw):
    assert _step(**kw) == -1


def test_step_entry_wants_its_workspace():
    assert _step(ws=None) == -3 and _step(nws=100) == -3 and _step(prompts=0, ws=None) == 0


def _move(t=((A, 1 << 30, 64, 16, 64, 16, 16, 1),), n=None, src_rows=4, dst_rows=4, nrows=4, si=None, di=None, sl=None, dl=None,
          disjoint=0):
    flat = [v for q in t for v in q]
    lst = lambda v: None if v is None else (ctypes.c_int64 * len(v))(*v)  # noqa: E731
    return _lib().rwkv7mi_rows_move(len(t) if n is None else n, (ctypes.c_int64 * len(flat))(*flat), src_rows, dst_rows, nrows,
                                    si, di, lst(sl), lst(dl), disjoint, None)


def _t(src=A, dst=1 << 30, so=64, sr=16, do=64, dr=16, size=16, outer=1):
    return (src, dst, so, sr, do, dr, size, outer)


@pytest.mark.parametrize("kw", [dict(n=-1), dict(t=[_t()] * 25), dict(src_rows=-1), dict(dst_rows=1 << 31), dict(nrows=-1),
                                dict(t=[_t(src=0)]), dict(t=[_t(dst=0)]), dict(t=[_t(size=-1)]), dict(t=[_t(outer=-1)]),
                                dict(sl=[0] * 193, nrows=193), dict(sl=[0] * 4, si=A), dict(dl=[0] * 4, di=A),
                                dict(t=[_t(src=A, dst=A, sr=16, dr=32)]), dict(t=[_t(src=A, dst=A)], nrows=2049),
                                dict(t=[_t(size=1 << 40)]), dict(t=[_t(outer=1 << 40)])])
def test_rows_entry_refuses(kw):
    assert _move(**kw) == -1


def test_rows_of_nothing_launch_nothing():
    assert _move(n=0) == 0 and _move(nrows=0) == 0 and _move(t=[_t(size=0)]) == 0 and _move(t=[_t(outer=0)]) == 0


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


def test_beam_select_refuses(calls):
    import rwkv7mi as mi

    x, s = torch.zeros(6, 50), torch.zeros(2, 3)
    for args, kw in (((x, s.double()), {}), ((x, s[0]), {}), ((x[:5], s), {}), ((x.view(3, 2, 50), s), {}),
                     ((x.to(torch.float64), s), {}), ((x[:, :0], s), {}), ((x, s), dict(out=(s, s, s))),
                     ((x, s), dict(workspace=torch.zeros(8, dtype=torch.uint8))), ((x, s, 0), {}), ((x, s, -3), {}),
                     ((x, s), dict(out=(torch.zeros(2, 6), *[torch.zeros(2, 6, dtype=torch.int64)] * 2)))):
        with pytest.raises(ValueError):
            mi.beam_select(*args, **kw)
    assert not calls
    got = mi.beam_select(x, s)
    assert [t.shape for t in got] == [(2, 6)] * 3 and len(calls) == 1


def _state(mi, **kw):
    return mi.BeamState.start(torch.zeros(2, 4, dtype=torch.int64), 3, 9, **kw)


def test_beam_state_is_checked_once():
    import rwkv7mi as mi

    s = _state(mi, lengths=[2, 4])
    assert s.lengths.tolist() == [2, 2, 2, 4, 4, 4] and s.scores.tolist()[0] == [0.0, -np.inf, -np.inf]
    with pytest.raises(AttributeError):
        s.tokens = s.finished_tokens
    keys = mi.BeamState.__slots__[:8]
    good = {k: getattr(s, k) for k in keys}
    mi.BeamState(**good)
    for key, bad in (("tokens", s.tokens[0]), ("tokens", s.tokens.int()), ("lengths", s.lengths[:5]), ("done", s.done.byte()),
                     ("lengths", s.lengths.long()), ("scores", s.scores.t()), ("finished_tokens", s.tokens),
                     ("finished_scores", s.scores), ("prompt_lengths", s.lengths[:2]), ("finished_lengths", s.lengths)):
        with pytest.raises(ValueError):
            mi.BeamState(**{**good, key: bad})
    with pytest.raises(ValueError):
        mi.BeamState.start(torch.zeros(2, 10, dtype=torch.int64), 3, 9)
    with pytest.raises(ValueError):
        s.best(4)


def test_beam_step_refuses(calls):
    import rwkv7mi as mi

    x, s = torch.zeros(6, 50), _state(mi)
    other = mi.BeamState.start(torch.zeros(2, 4, dtype=torch.int64), 3, 10)
    mixed = mi.BeamState(**{**{k: getattr(_state(mi), k) for k in mi.BeamState.__slots__[:8]}, "scores": s.scores})
    for kw in (dict(eos_token_id=list(range(9))), dict(early_stopping="maybe"), dict(length_penalty=float("inf")),
               dict(out=other), dict(out=mixed), dict(next_tokens=torch.zeros(5, dtype=torch.int64)),
               dict(rows=torch.zeros(6, dtype=torch.int32)), dict(workspace=torch.zeros(4, dtype=torch.uint8))):
        with pytest.raises(ValueError):
            mi.beam_step(x, s, **kw)
    both = torch.zeros(7, dtype=torch.int64)
    with pytest.raises(ValueError, match="overlap"):
        mi.beam_step(x, s, next_tokens=both[:6], rows=both[1:])
    with pytest.raises(ValueError):
        mi.beam_step(torch.zeros(80, 50), mi.BeamState.start(torch.zeros(1, 2, dtype=torch.int64), 80, 9), eos_token_id=1)
    with pytest.raises(ValueError):
        mi.beam_step(x[:4], s)
    assert not calls
    assert mi.beam_step(x, s)[2] is s and len(calls) == 1
    for eos in (3, [3, 4], (3, 4), torch.tensor([3, 4]), torch.tensor(3)):  # (the library's 9th and 8th arguments)
        mi.beam_step(x, s, eos_token_id=eos)
        args = calls[-1][1]
        assert list(args[7]) == ([3] if args[8] == 1 else [3, 4])


def test_rows_refuse(calls):
    import rwkv7mi as mi

    t, u = torch.zeros(2, 5, 8), torch.zeros(3, 5)
    base = torch.zeros(5, 8)
    for args, kw in ((([], [0]), {}), (([t, u[:, :4]], [0]), dict(dim=1)), (([t], [0]), dict(dim=3)), (([t], [0]), dict(dim=-1)),
                     (([t], torch.zeros(2)), dict(dim=1)), (([t], torch.zeros(2, 1, dtype=torch.long)), dict(dim=1)),
                     (([t], [0]), dict(dim=1, out=[torch.zeros(2, 2, 8)])), (([t], [0]), dict(dim=1, out=[])),
                     (([t], [0]), dict(dim=1, out=[t[:, :1]])), (([u], [0]), dict(dim=1, out=[torch.zeros(1, 1).expand(3, 1)])),
                     (([t], [0]), dict(dim=1, out=[torch.zeros(2, 1, 8, dtype=torch.half)]))):
        with pytest.raises(ValueError):
            mi.select_rows(*args, **kw)
    for args, kw in ((([], [0]), {}), (([t], [0, 1]), dict(dim=1)), (([t], [0, 1], [2]), dict(dim=1)),
                     (([t], [0, 1], [2, 2]), dict(dim=1)), (([t[..., ::2]], [0] * 5), dict(dim=1)),
                     (([base.expand(5, 8).as_strided((5, 8), (4, 1))], [0] * 5), {}), (([t, t], [0] * 5), dict(dim=1)),
                     (([base[0].expand(5, 8)], [0] * 5), {}), (([base, base[:, :3]], [0] * 5), {}),
                     (([torch.zeros(3000, 1)], [1] * 3000), {})):
        with pytest.raises(ValueError):
            mi.move_rows_(*args, **kw)
    for f in (lambda: mi.select_rows([t], [5], dim=1), lambda: mi.select_rows([t], [-2], dim=1),
              lambda: mi.move_rows_([t], [5], [0], dim=1), lambda: mi.move_rows_([t], [0], [5], dim=1),
              lambda: mi.move_rows_([t], [0], [-1], dim=1)):
        with pytest.raises(IndexError):
            f()
    assert not calls
    mi.move_rows_([t, u], [1, 0, -1, 3, 3], dim=1)
    assert [t.shape for t in mi.select_rows([t, u], [0, 0, -1], dim=1)] == [(2, 3, 8), (3, 3)]
    mi.move_rows_([torch.zeros(4, 3)], [], [])
    mi.move_rows_([torch.zeros(3000, 1)], list(range(3000)))  # nothing trades places
    assert len(calls) == 3
    flat = calls[0][1][1]
    assert list(flat[2:8]) == [160, 32, 160, 32, 32, 2] and list(flat[10:16]) == [20, 4, 20, 4, 4, 3]


def test_cpu_tensors_are_refused():
    import rwkv7mi as mi

    with pytest.raises(RuntimeError, match="GPU only"):
        mi.beam_select(torch.zeros(6, 50), torch.zeros(2, 3))
    with pytest.raises(RuntimeError, match="GPU only"):
        mi.beam_step(torch.zeros(6, 50), _state(mi))
    with pytest.raises(RuntimeError, match="GPU only"):
        mi.move_rows_([torch.zeros(5, 2)], [0] * 5)
    with pytest.raises(RuntimeError, match="GPU only"):
        mi.select_rows([torch.zeros(5, 2)], [0])


def test_the_plain_step():
    """The written-out step on a case small enough to see."""
    v = ref.values(np.log(np.array([[[0.5, 0.3, 0.2], [0.6, 0.1, 0.3]]])), np.array([[-1.0, -2.0]]))
    assert np.allclose(np.exp(v[0]), np.exp([[-1.0], [-2.0]]) * np.array([[0.5, 0.3, 0.2], [0.6, 0.1, 0.3]]))
    found = ref.select(v, 4)
    assert found[1].tolist() == [[0, 1, 0, 2]] and found[2].tolist() == [[0, 0, 1, 0]]
    state = dict(tokens=np.array([[[7, 0, 0], [8, 0, 0]]]), lengths=np.array([1, 1]), scores=np.array([[-1.0, -2.0]]),
                 prompt_lengths=np.array([1]), finished_tokens=np.zeros((1, 2, 3), int), finished_lengths=np.zeros((1, 2), int),
                 finished_scores=np.full((1, 2), -np.inf), done=np.array([False]))
    nxt, rows, new = ref.step(found, state, (1,), 1.0, False)
    # token 1 of beam 0 ends as the second best; token 0 of beam 0 and of beam 1 live on
    assert nxt.tolist() == [0, 0] and rows.tolist() == [0, 1]
    assert new["tokens"][0].tolist() == [[7, 0, 0], [8, 0, 0]] and new["lengths"].tolist() == [2, 2]
    # (of two empty places the first stays empty)
    assert new["finished_tokens"][0, 1].tolist() == [7, 1, 0] and new["finished_lengths"][0].tolist() == [0, 2]
    assert np.isclose(new["finished_scores"][0, 1], np.log(0.3) - 1.0) and not new["done"][0]


def test_custom_ops_give_shapes():
    import rwkv7mi  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        out = torch.ops.rwkv7mi.beam_select(torch.empty(6, 50), torch.empty(2, 3), 7, False)
        assert [t.shape for t in out] == [(2, 7)] * 3 and out[1].dtype is torch.int64
        rows = torch.ops.rwkv7mi.select_rows([torch.empty(2, 5, 3), torch.empty(1, 5)], torch.zeros(4, dtype=torch.long), 1)
        assert [t.shape for t in rows] == [(2, 4, 3), (1, 4)]
    with pytest.raises(RuntimeError, match="GPU only"):
        torch.ops.rwkv7mi.move_rows_([torch.zeros(3, 2)], torch.zeros(3, dtype=torch.long), 0)

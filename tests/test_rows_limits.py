"""Moved rows and the caches that use them at their limits, on the CPU: tensors of other kinds, layouts and lifetimes."""
from __future__ import annotations

import pytest
import torch


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


def _config(layers=2):
    from rwkv7mi.model import NativeRWKV7Config

    return NativeRWKV7Config(vocab_size=64, hidden_size=128, num_hidden_layers=layers, intermediate_size=256,
                             decay_low_rank_dim=32, a_low_rank_dim=32, gate_low_rank_dim=64, v_low_rank_dim=32)


@pytest.mark.parametrize("state", [torch.float32, torch.float16])
def test_cache_edits_of_fake_tensors_give_shapes(calls, state):
    """A GPU cache under a fake mode: its tensors have no memory that a kernel could read."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from rwkv7mi.model import NativeRWKV7Cache

    with FakeTensorMode():
        c = NativeRWKV7Cache.zeros(_config(), 3, "cuda", state_dtype=state)
        c.batch_repeat_interleave(2)
        assert c.get_batch_size() == 6 and all(t.shape[0] == 6 for t in c._all_tensors())
        d = c.select_batch([4, 0], inplace=False)
        assert d.get_batch_size() == 2 and c.get_batch_size() == 6
        c.reorder_cache(torch.tensor([5, 5, 1, 0], device="cuda"))
        assert [t.shape[0] for t in c._all_tensors()] == [4] * len(c._all_tensors())
        assert c._state[1].shape == (4, 2, 64, 64) and c._state[1].dtype is state
    assert not calls


def test_cache_edits_keep_the_graph(calls, monkeypatch):
    """Cache tensors that require grad: selection and repeat are differentiable (CPU tensors in the place of GPU
    ones); without grad mode they are moved."""
    from rwkv7mi.model import NativeRWKV7Cache

    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    c = NativeRWKV7Cache.zeros(_config(), 3, "cpu")
    c._map(lambda t: t.float().requires_grad_())
    leaves = c._all_tensors()
    c.batch_repeat_interleave(2)
    c.select_batch([0, 0, 5, 2])
    sum((t * (i + 1)).sum() for i, t in enumerate(c._all_tensors())).backward()
    for i, t in enumerate(leaves):
        want = torch.tensor([2.0, 1.0, 1.0]) * (i + 1)  # rows 0, 0, 2, 1 of the three
        assert torch.equal(t.grad, want.view(3, *[1] * (t.dim() - 1)).expand_as(t))
    assert not calls
    with torch.no_grad():
        c.select_batch([1, 0])
    assert calls and not any(t.requires_grad for t in c._all_tensors())


def test_moved_rows_have_no_gradient_and_say_so(calls):
    import rwkv7mi as mi

    t, u = torch.zeros(3, 4), torch.zeros(3, 5, requires_grad=True)
    for f in (lambda: mi.select_rows([t, u], [0, 1]), lambda: mi.move_rows_([t, u * 2], [1, 0, 2]),
              lambda: mi.select_rows([t], [0], out=[torch.zeros(1, 4, requires_grad=True)])):
        with pytest.raises(RuntimeError, match="no gradient"):
            f()
    assert not calls
    with torch.no_grad():
        assert not mi.select_rows([t, u], [0, 1])[1].requires_grad
        mi.move_rows_([t, u], [1, 0, 2])
    assert len(calls) == 2


def test_rows_moved_in_place_are_a_change_to_autograd(calls):
    """A tensor that a backward pass saved and whose rows then move: an error, as for torch's own in-place operations."""
    import rwkv7mi as mi

    x, w, aside = torch.ones(3, 4), torch.ones(3, 4, requires_grad=True), torch.ones(2, 3)
    y = (w * x).sum()
    mi.move_rows_([x], [1, 0, 2])
    assert x._version == 1 and aside._version == 0
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    out = torch.empty(2, 4)
    mi.select_rows([x], [1, 0], out=[out])
    assert out._version == 1 and x._version == 1
    mi.move_rows_([x], [], [])
    with torch.inference_mode():
        mi.move_rows_([torch.zeros(3, 4)], [1, 0, 2])
    assert len(calls) == 3


def test_conjugate_and_negative_views_are_selected_by_value(calls):
    """The bytes of such a view are not its values: they are taken from a plain copy, and written nowhere."""
    import rwkv7mi as mi

    x = torch.randn(4, 3, dtype=torch.complex64)
    for view in (x.conj(), x.conj().imag):
        assert view.is_conj() or view.is_neg()
        (out,) = mi.select_rows([view], [1, 0])
        assert not out.is_conj() and not out.is_neg()
        address, end = calls[-1][1][1][0], view.data_ptr() + view.untyped_storage().nbytes()
        assert not view.data_ptr() <= address < end  # (not the view's own memory)
        with pytest.raises(ValueError, match="conjugate"):
            mi.select_rows([view.clone()], [1, 0], out=[view[:2]])
    y = x.conj()
    mi.move_rows_([y], [1, 0, 2, 3])  # (rows of one view: its bytes trade places as its values do)
    assert list(calls[-1][1][1][:2]) == [x.data_ptr()] * 2


def test_rows_apart_are_moved_whatever_follows_them(calls):
    """Every other row of an odd number: the last one ends before the next part begins."""
    import rwkv7mi as mi

    for rows in range(1, 8):
        for step in (1, 2, 3):
            base = torch.zeros(3, rows, 4)
            view = base[:, ::step]
            mi.move_rows_([view], list(range(view.shape[1] - 1, -1, -1)), dim=1)
            mi.select_rows([base], [0] * view.shape[1], dim=1, out=[view.clone()])
    # rows outermost in memory, parts of them in use
    view = torch.zeros(5, 7, 4).transpose(0, 1)[::3, ::2]
    mi.move_rows_([view], [2, 1, 0], dim=1)
    done = len(calls)
    for bad in (torch.zeros(30).as_strided((3, 3, 4), (8, 4, 1)),      # a part's last row is the next one's first
                torch.zeros(30).as_strided((3, 3, 4), (7, 4, 1)), torch.zeros(30).as_strided((3, 2, 4), (4, 4, 1)),
                torch.zeros(40).as_strided((3, 3, 4), (12, 3, 1))):
        with pytest.raises(ValueError, match="apart"):
            mi.move_rows_([bad], [0] * bad.shape[1], dim=1)
    assert len(calls) == done


def test_an_index_out_of_range_is_marked_in_cache_edits(calls, monkeypatch):
    from rwkv7mi.model import NativeRWKV7Cache

    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    c = NativeRWKV7Cache.zeros(_config(), 3, "cpu")
    c.select_batch([1, 0])
    assert calls[-1][1][9] == 3  # (poison, and nothing trades places)
    c._map(lambda t: t.clone())
    c.select_batch([1, 0])
    assert calls[-1][1][9] == 3
    import rwkv7mi as mi

    mi.select_rows([torch.zeros(3, 4)], [0, -1])
    assert calls[-1][1][9] == 1
    mi.move_rows_([torch.zeros(3, 4)], [1, 0, -1])
    assert calls[-1][1][9] == 0
    mi.move_rows_([torch.zeros(3, 4)], [1, 0, -1], poison=True)
    assert calls[-1][1][9] == 2


def test_no_rows_are_moved(calls):
    """Tensors without rows, without parts, or with rows of nothing: all apart, and nothing is launched for no index."""
    import rwkv7mi as mi

    for t in (torch.empty(3, 0, 5), torch.empty(0, 4, 5), torch.empty(3, 4, 0), torch.empty(3, 8, 5)[:, 8:]):
        mi.move_rows_([t], list(range(t.shape[1])), dim=1)
        mi.move_rows_([t], [], [], dim=1)
        mi.select_rows([torch.empty(3, 2, 5)[:, :0], ], [], dim=1, out=[torch.empty(3, 0, 5)])

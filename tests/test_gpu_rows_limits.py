"""Moved rows at their limits, on the GPU: layouts, indices out of range, empty tensors, gradients."""
from __future__ import annotations

import pytest
import torch

from test_gpu_beam_model import _cache, _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.uint8])
def test_rows_apart_move_in_place(dtype):
    import rwkv7mi as mi

    g = torch.Generator("cuda").manual_seed(2)
    for rows, width in ((5, 12), (7, 33), (9, 4096)):
        base = torch.randint(0, 99, (3, rows, width), device="cuda", generator=g).to(dtype)
        view, keep = base[:, ::2], base.clone()
        n = view.shape[1]
        idx = list(range(1, n)) + [-1]
        for index in (idx, torch.tensor(idx, device="cuda")):
            base.copy_(keep)
            mi.move_rows_([view], index, dim=1)
            assert torch.equal(view[:, :-1], keep[:, 2::2]) and not view[:, -1].any()
            assert torch.equal(base[:, 1::2], keep[:, 1::2])


def test_conjugate_and_negative_views():
    import rwkv7mi as mi

    x = torch.randn(4, 3, dtype=torch.complex64, device="cuda")
    for view in (x.conj(), x.conj().imag):
        (got,) = mi.select_rows([view], [2, -1, 0])
        assert torch.equal(got[[0, 2]], view[[2, 0]]) and not got[1].any()
    y = x.clone().conj()
    want = y[[3, 0, 1, 2]].clone()
    mi.move_rows_([y], [3, 0, 1, 2])
    assert torch.equal(y, want)


def test_cache_edits_are_differentiable():
    model = _model()
    c = _cache(model, 3)
    c._map(lambda t: t.float().requires_grad_())
    leaves = c._all_tensors()
    c.batch_repeat_interleave(2)
    c.reorder_cache(torch.tensor([0, 0, 5, 2], device="cuda"))
    sum(t.sum() for t in c._all_tensors()).backward()
    for t in leaves:
        want = torch.tensor([2.0, 1.0, 1.0], device="cuda").view(3, *[1] * (t.dim() - 1)).expand_as(t)
        assert torch.equal(t.grad, want)


def test_rows_of_empty_tensors_are_zeros():
    """A tensor without rows has no memory: every index is out of range."""
    import rwkv7mi as mi

    e, full = torch.empty(3, 0, 5, device="cuda"), torch.empty(2, 0, 40, device="cuda", dtype=torch.half)
    for index in ([-1, -1], torch.tensor([-1, 3], device="cuda")):
        got = mi.select_rows([e, full], index, dim=1)
        assert [t.shape for t in got] == [(3, 2, 5), (2, 2, 40)] and not any(t.any() for t in got)
    mi.move_rows_([e, full], [], dim=1)


@pytest.mark.parametrize("state", [torch.float32, torch.float16])
def test_cache_edits_by_a_wrong_index_on_the_gpu(state):
    """Nothing waits to look at an index on the GPU: a row out of range is NaN, not a state to go on with."""
    model = _model()
    model.state_dtype = state
    for scattered in (False, True):
        c = _cache(model, 4)
        if scattered:
            c._map(lambda t: t.clone())
        old = [t.clone() for t in c._all_tensors()]
        c.reorder_cache(torch.tensor([2, 4, -1, 0, 1 << 40], device="cuda"))
        for t, o in zip(c._all_tensors(), old):
            assert torch.equal(t[[0, 3]], o[[2, 0]])
            bad = t[[1, 2, 4]]
            assert bad.isnan().all() if t.is_floating_point() else (bad == -1).all()
    runner = model.graph_runner(3)
    c = _cache(model, 3)
    runner.replay(torch.zeros(3, dtype=torch.long, device="cuda"), c)
    old = [t.clone() for t in runner.cache._all_tensors()]
    c.reorder_cache(torch.tensor([1, 3, 1], device="cuda"))
    assert c._native_graph_bound_to(runner)
    for t, o in zip(runner.cache._all_tensors(), old):
        assert torch.equal(t[[0, 2]], o[[1, 1]])
        assert t[1].isnan().all() if t.is_floating_point() else (t[1] == -1).all()
    logits = runner.replay(torch.zeros(3, dtype=torch.long, device="cuda"), c)
    assert logits[1].isnan().all() and not logits[[0, 2]].isnan().any()
    runner.cache.zero_()


def test_rows_of_all_kinds_poisoned():
    import rwkv7mi as mi
    from test_gpu_state_rows import _tensors

    for rows in (3, 70, 200):
        ts = _tensors(rows)
        idx = torch.arange(rows, device="cuda").flip(0)
        idx[1::3] = torch.tensor([-1, rows, -5, 1 << 50], device="cuda").repeat(rows)[:len(idx[1::3])]
        good = (idx >= 0) & (idx < rows)
        old = [t.clone() for t in ts]
        new = mi.select_rows(ts, idx, dim=1, poison=True)
        mi.move_rows_(ts, idx, dim=1, poison=True)
        for a, b, o in zip(new, ts, old):
            assert torch.equal(a[:, good], o[:, idx[good]]) and torch.equal(b[:, good], o[:, idx[good]])
            for t in (a[:, ~good], b[:, ~good]):
                assert t.isnan().all() if t.is_floating_point() else (t == -1).all()
        assert not any(t[:, ~good].any() for t in mi.select_rows(old, idx, dim=1))

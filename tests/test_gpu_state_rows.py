"""Rows of several tensors moved by one index in one launch, against torch's indexing: bytes, so equal."""
from __future__ import annotations

import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def _tensors(rows, seed=0):
    """Rows along dimension 1 of all kinds: wide and narrow, odd lengths, one byte, unaligned views."""
    g = torch.Generator("cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    ints = lambda *s: torch.randint(-99, 99, s, device="cuda", generator=g)  # noqa: E731
    wide = torch.zeros(3, rows + 4, 4, 64, 64, device="cuda")
    wide.normal_(generator=g)
    return [wide[:, 2:rows + 2], rnd(3, rows, 129).half(), rnd(1, rows, 1000).bfloat16(), ints(1, rows, 501),
            ints(1, rows, 1).to(torch.int32), ints(2, rows, 7).to(torch.int8), rnd(2, 3, rows, 5).reshape(6, rows, 5),
            rnd(1, 2 * rows, 3)[:, ::2], ints(2, rows, 33).to(torch.int16)[..., 1:]]


def _want(ts, src, dst):
    out = [t.clone() for t in ts]
    for t, o in zip(ts, out):
        for s, d in zip(src, dst):
            o[:, d] = t[:, s] if 0 <= s < t.shape[1] else 0
    return out


@pytest.mark.parametrize("rows", [1, 2, 3, 7, 32, 64, 65, 100, 300])
def test_select_rows(rows):
    import rwkv7mi as mi

    ts = [t for t in _tensors(rows)]
    r = random.Random(rows)
    for n in (1, 5, rows, 2 * rows + 3):
        idx = [r.randrange(-1, rows) for _ in range(n)]
        want = [torch.stack([t[:, i] if i >= 0 else torch.zeros_like(t[:, 0]) for i in idx], 1) for t in ts]
        for index in (idx, torch.tensor(idx), torch.tensor(idx, device="cuda"),
                      torch.tensor(idx, device="cuda", dtype=torch.int32)):
            got = mi.select_rows(ts, index, dim=1)
            assert all(torch.equal(a, b) and a.dtype == b.dtype for a, b in zip(got, want))
        out = [torch.empty(t.shape[0], n + 2, *t.shape[2:], dtype=t.dtype, device="cuda")[:, 1:-1] for t in ts]
        assert mi.select_rows(ts, idx, dim=1, out=out) is not None
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    # on the device an index out of range is a row of zeros
    got = mi.select_rows(ts[:1], torch.tensor([rows, -7, 0, 1 << 40], device="cuda"), dim=1)[0]
    assert not got[:, [0, 1, 3]].any() and torch.equal(got[:, 2], ts[0][:, 0])


@pytest.mark.parametrize("rows", [1, 2, 4, 31, 64, 65, 200, 513])
@pytest.mark.parametrize("how", ["permute", "any", "cycle", "same"])
def test_move_rows_in_place(rows, how):
    """Rows that trade places, rows read many times, zeros, rows left alone."""
    import rwkv7mi as mi

    r = random.Random(rows)
    src = list(range(rows))
    if how == "permute":
        r.shuffle(src)
    elif how == "any":
        src = [r.randrange(-1, rows) for _ in range(rows)]
    elif how == "cycle":
        src = src[1:] + src[:1]
    for k, index in enumerate((src, torch.tensor(src, device="cuda"))):
        ts = _tensors(rows, k)
        around = ts[0]._base.clone()
        want = _want(ts, src, range(rows))
        mi.move_rows_(ts, index, dim=1)
        assert all(torch.equal(a, b) for a, b in zip(ts, want))
        assert torch.equal(ts[0]._base[:, :2], around[:, :2]) and torch.equal(ts[0]._base[:, -2:], around[:, -2:])


def test_move_rows_to_destinations():
    """Forks, compaction with fresh rows, swaps of a few: the other rows stay."""
    import rwkv7mi as mi

    for rows, src, dst in ((9, [3] * 5, [0, 2, 4, 6, 8]), (33, [30, 31, 32, -1, -1], [2, 5, 7, 30, 1]),
                           (6, [1, 4], [4, 1]), (6, [], []), (250, list(range(210)), list(range(40, 250))),
                           (250, list(range(100)) * 2, list(range(50, 250)))):
        ts = _tensors(rows)
        want = _want(ts, src, dst)
        mi.move_rows_(ts, src, dst, dim=1)
        assert all(torch.equal(a, b) for a, b in zip(ts, want)), (rows, src, dst)
    # sources on the device
    ts = _tensors(20)
    want = _want(ts, [5, -1, 99, 7], [7, 0, 3, 5])
    mi.move_rows_(ts, torch.tensor([5, -1, 99, 7], device="cuda"), [7, 0, 3, 5], dim=1)
    assert all(torch.equal(a, b) for a, b in zip(ts, want))


def test_move_many_rows():
    """2048 rows that trade places; more where no source is a destination; more than 24 tensors."""
    import rwkv7mi as mi

    g = torch.Generator("cuda").manual_seed(1)
    ts = [torch.randn(2, 2048, 40, device="cuda", generator=g), torch.randn(1, 2048, 3, device="cuda", generator=g)]
    perm = torch.randperm(2048, device="cuda", generator=g)
    want = [t[:, perm] for t in ts]
    mi.move_rows_(ts, perm, dim=1)
    assert all(torch.equal(a, b) for a, b in zip(ts, want))
    t = torch.randn(1, 9000, 33, device="cuda", generator=g)
    want = t.clone()
    want[:, :4000] = t[:, 5000:]
    mi.move_rows_([t], list(range(5000, 9000)), list(range(4000)), dim=1)
    assert torch.equal(t, want)
    many = [torch.randn(5, 10 + i, device="cuda", generator=g) for i in range(60)]
    idx = torch.tensor([4, 0, 0, 1, 2], device="cuda")
    want = [m[idx] for m in many]
    assert all(torch.equal(a, b) for a, b in zip(mi.select_rows(many, idx), want))
    mi.move_rows_(many, idx)
    assert all(torch.equal(a, b) for a, b in zip(many, want))


def test_rows_as_outermost_and_between():
    """dim 0; rows outside their outer dimension in memory (a transposed pool); empty tensors."""
    import rwkv7mi as mi

    t = torch.randn(7, 5, 12, device="cuda")
    want = t.clone()
    want[:, [4, 1, 0]] = t[:, [0, 1, 4]]
    u = t.clone().transpose(0, 1).contiguous().transpose(0, 1)  # rows outermost in memory
    mi.move_rows_([u], [4, 1, 2, 3, 0], dim=1)
    assert torch.equal(u, want)
    v = torch.randn(6, device="cuda")
    w = v.clone()
    mi.move_rows_([v], [5, 4, 3, 2, 1, 0])
    assert torch.equal(v, w.flip(0))
    e = torch.empty(3, 0, device="cuda")
    assert mi.select_rows([e], [0, 2])[0].shape == (2, 0)
    assert mi.select_rows([v], [])[0].shape == (0,)


def test_move_rows_on_a_stream_and_captured():
    import rwkv7mi as mi

    ts = _tensors(12)
    idx = torch.arange(12, device="cuda")
    side = torch.cuda.Stream()
    want = _want(ts, list(range(11, -1, -1)), range(12))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mi.move_rows_(ts, list(range(11, -1, -1)), dim=1)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(ts, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        mi.move_rows_(ts, idx, dim=1)
        new = mi.select_rows(ts, [3, 3, 0], dim=1)
    r = random.Random(0)
    for _ in range(5):
        src = [r.randrange(12) for _ in range(12)]
        idx.copy_(torch.tensor(src))
        want = _want(ts, src, range(12))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ts, want))
        assert all(torch.equal(a, b[:, [3, 3, 0]]) for a, b in zip(new, want))


def test_an_index_among_what_is_moved():
    """The index's own rows move too: it counts as it was before the call."""
    import rwkv7mi as mi

    for _ in range(3):
        t = torch.randn(500, 3000, device="cuda")
        idx = torch.randperm(500, device="cuda")
        want = (t[idx], idx[idx])
        mi.move_rows_([t, idx], idx)
        assert torch.equal(t, want[0]) and torch.equal(idx, want[1])
    with pytest.raises(ValueError):
        mi.select_rows([t[:, 0].long().contiguous()], idx, out=[idx])


def test_custom_ops():
    import rwkv7mi as mi

    ts = _tensors(5)
    idx = torch.tensor([4, 0, 0, 1, 2], device="cuda")
    new = torch.ops.rwkv7mi.select_rows(ts, idx, 1)
    torch.ops.rwkv7mi.move_rows_(ts, idx, 1)
    assert all(torch.equal(a, b) for a, b in zip(new, ts))
    x, s = torch.randn(6, 300, device="cuda"), torch.zeros(2, 3, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(torch.ops.rwkv7mi.beam_select(x, s, 5, False), mi.beam_select(x, s, 5)))

"""Beam search on the device (selection, step) against plain 64-bit numpy."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import beam_reference as ref

pytestmark = pytest.mark.gpu
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
INF = float("inf")
# The 64-bit sum of a row is made of fp32 terms: an exponential is off by its argument's rounding
# (|d| 2^-24, which e^d outweighs) and two steps, 32 of them a lane and 10 partial sums follow one
# another in fp32: lse is off by less than 46 2^-24.  The result is rounded once.
LSE = 46 * 2.0 ** -24
HALF = 2.0 ** -24


def _case(rng, prompts, beams, n, dtype, scale=3.0):
    x = torch.from_numpy(rng.standard_normal((prompts * beams, n)) * scale).to(DTYPES[dtype])
    s = torch.from_numpy(rng.standard_normal((prompts, beams)) * 2 - 20).float()
    return x, s


def _check(got, x, s, m, normalized=False):
    """Values, tokens and rows of a selection: each value is its token's, none comes twice, and they are
    the best in order, as far as the error of lse (the same within a row) can tell."""
    prompts, beams = s.shape
    n = x.shape[1]
    v = ref.values(x.double().numpy().reshape(prompts, beams, n), s.numpy(), normalized)
    want, wtok, wbeam = ref.select(v, m)
    val, tok, row = (t.cpu().numpy() for t in got)
    assert val.shape == tok.shape == row.shape == (prompts, m)
    for b in range(prompts):
        beam = row[b] - b * beams
        assert ((0 <= beam) & (beam < beams) & (0 <= tok[b]) & (tok[b] < n)).all()
        assert len(set(zip(beam, tok[b]))) == m
        own = v[b, beam, tok[b]]
        fine = np.isfinite(want[b])
        assert np.array_equal(np.isnan(val[b]), np.isnan(want[b]))
        assert np.array_equal(np.isneginf(val[b]), np.isneginf(want[b]))
        tol = LSE + (np.abs(want[b][fine]) + LSE) * HALF
        assert (np.abs(val[b][fine] - own[fine]) <= tol).all()
        assert (np.abs(want[b][fine] - own[fine]) <= 2 * LSE).all()
        # what has no value comes in the order of the indices
        assert np.array_equal(beam[~fine], wbeam[b][~fine]) and np.array_equal(tok[b][~fine], wtok[b][~fine])
        for k in range(beams):  # inside a row the order is the logits'
            mine = tok[b][(beam == k) & fine]
            logits = x[b * beams + k].double().numpy()[mine]
            assert all(a > c or (a == c and i < j) for a, c, i, j in zip(logits, logits[1:], mine, mine[1:]))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("prompts,beams,n,m", [
    (1, 1, 1, 1), (1, 1, 7, 7), (2, 3, 33, 6), (1, 4, 1000, 8), (3, 5, 8191, 10), (2, 2, 8193, 128), (7, 1, 8200, 3),
    (1, 128, 300, 128), (2, 32, 4099, 64), (5, 2, 50277, 4), (1, 4, 65536, 8), (1, 2, 200003, 5)])
def test_select_against_64_bits(prompts, beams, n, m, dtype):
    import rwkv7mi as mi

    rng = np.random.default_rng(prompts * n + m)
    x, s = _case(rng, prompts, beams, n, dtype)
    _check(mi.beam_select(x.cuda(), s.cuda(), m), x, s, m)
    _check(mi.beam_select(x.cuda().view(prompts, beams, n), s.cuda(), m, normalized=True), x, s, m, True)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_select_rows_anywhere_in_memory(dtype):
    """Rows that start at any element and lie any distance apart; transposed logits; scores of any stride."""
    import rwkv7mi as mi

    rng = np.random.default_rng(3)
    for offset, gap in ((0, 0), (1, 0), (3, 5), (7, 1), (2, 16)):
        for n in (515, 9001):
            big = torch.from_numpy(rng.standard_normal(offset + 6 * (n + gap)) * 3).to(DTYPES[dtype]).cuda()
            big[: offset] = INF  # (in no row)
            x = big.as_strided((6, n), (n + gap, 1), offset)
            if gap:
                big.as_strided((6, gap), (n + gap, 1), offset + n).fill_(float("nan"))
            s = torch.randn(4, 3, generator=torch.Generator().manual_seed(offset))[::2]
            _check(mi.beam_select(x, s.cuda()[:, :], 9), x.cpu(), s, 9)
    x = torch.from_numpy(rng.standard_normal((40, 6))).to(DTYPES[dtype]).cuda().t()
    s = torch.randn(3, 2).cuda().t()
    _check(mi.beam_select(x, s, 4), x.cpu(), s.cpu(), 4)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_select_takes_nothing_from_around_a_row(dtype):
    """NaN or +inf in the elements before and behind every row, at each alignment; logits of large
    magnitude too (they leave no rounding of their own: the differences are exact)."""
    import rwkv7mi as mi

    rng = np.random.default_rng(9)
    for n in (1, 3, 16, 4097, 16385):
        for offset in range(9):
            for poison, shift in ((float("nan"), 0.0), (INF, 30000.0), (INF, -30000.0)):
                x = torch.from_numpy(rng.standard_normal((4, n)) * 3 + shift).to(DTYPES[dtype])
                big = torch.full((16 + offset + 4 * (n + 17) + 16,), poison, dtype=DTYPES[dtype], device="cuda")
                rows = big.as_strided((4, n), (n + 17, 1), 16 + offset)
                rows.copy_(x)
                s = torch.from_numpy(rng.standard_normal((2, 2)) - 5).float()
                m = min(4, 2 * n)
                _check(mi.beam_select(rows, s.cuda(), m), x, s, m)


def test_select_equal_values_by_index():
    """Equal beams, equal logits, more of them than a workgroup gathers: exactly the first indices."""
    import rwkv7mi as mi

    s = torch.full((2, 3), -1.5)
    for n in (40, 5000, 20000):
        for fill in ("constant", "steps", "zeros", "top"):
            x = torch.zeros(6, n)
            if fill == "constant":
                x += 2.5
            elif fill == "steps":  # long runs of equal values
                x += (torch.arange(n) * 7 // n).float()
            elif fill == "zeros":  # +0 and -0 are equal
                x[:, ::2] = -0.0
            else:
                x[:, n // 2:] = 1.0
            for dt in DTYPES.values():
                y = x.to(dt)
                v = ref.values(y.double().numpy().reshape(2, 3, n), s.numpy())
                for m in (1, 16, 100):
                    want = ref.select(v, m)
                    val, tok, row = mi.beam_select(y.cuda(), s.cuda(), m)
                    assert np.array_equal(tok.cpu().numpy(), want[1]), (n, fill, m)
                    assert np.array_equal(row.cpu().numpy() - 3 * np.arange(2)[:, None], want[2])
                    assert np.allclose(val.cpu().numpy(), want[0], rtol=0, atol=LSE + HALF * 20)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_select_sorted_and_shifted_rows(dtype):
    """Ascending, descending and far-off logits: many values of one lane, little between the values."""
    import rwkv7mi as mi

    rng = np.random.default_rng(5)
    n = 30000
    base = np.sort(rng.standard_normal((4, n)) * 3, axis=1)
    for x in (base, base[:, ::-1].copy(), base - 900.0, base * 1e-3 + 300.0, base * 1e-30):
        t = torch.from_numpy(x).to(DTYPES[dtype])
        s = torch.tensor([[-500.0, -501.0], [-3.0, -3.5]])
        for m in (4, 64, 128):
            _check(mi.beam_select(t.cuda(), s.cuda(), m), t, s, m)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_select_where_few_beams_hold_the_best(dtype):
    """All that is wanted comes from one or two of many beams, more of it than a workgroup gathers."""
    import rwkv7mi as mi

    rng = np.random.default_rng(9)
    for beams, n, good in ((64, 65536, 2), (64, 30001, 1), (128, 9000, 9), (40, 65536, 3)):
        x, s = _case(rng, 2, beams, n, dtype, 0.5 if good == 9 else 3.0)
        s[:] = s - 500.0
        s[:, rng.choice(beams, good, replace=False)] = -3.0
        for m in (128, 60):
            _check(mi.beam_select(x.cuda(), s.cuda(), m), x, s, m)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_select_masks(dtype):
    """Masks that leave a few tokens, one, or none; the type's lowest value; beams that have not begun."""
    import rwkv7mi as mi

    rng = np.random.default_rng(6)
    dt = DTYPES[dtype]
    for n in (50, 9000, 20001):
        x, s = _case(rng, 6, 4, n, dtype)
        keep = rng.random((24, n)) < np.array([1, 0.5, 0.01, 0.0])[rng.integers(0, 4, 24)][:, None]
        keep[4:8] = False                       # a prompt with nothing left
        keep[8:12] = False
        keep[9, n - 1] = keep[11, 0] = True     # two tokens in all
        x[torch.from_numpy(~keep)] = -INF
        x[12:16, : n // 2] = torch.finfo(dt).min
        s[3, 1:] = -INF
        s[4] = -INF
        for m in (1, 8, 100):
            _check(mi.beam_select(x.cuda(), s.cuda(), m), x, s, m)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_select_nan_and_infinities(dtype):
    """A row with NaN or +inf, or such a score, is NaN throughout and ranks first."""
    import rwkv7mi as mi

    rng = np.random.default_rng(7)
    for n in (5, 3000, 17000):
        x, s = _case(rng, 8, 3, n, dtype)
        x[1, 0] = float("nan")
        x[4, n - 1] = INF
        x[7, n // 2], x[8, 0] = float("nan"), INF
        s[3, 1], s[4, 2], s[5, 0] = float("nan"), INF, -INF
        x[17] = -INF
        x[18, 1], x[19] = float("nan"), -INF
        x[21, 2], s[7, 0] = float("nan"), -INF
        for m in (1, 6, min(3 * n, 128)):
            _check(mi.beam_select(x.cuda(), s.cuda(), m), x, s, m)


def test_select_outputs_streams_and_graphs():
    import rwkv7mi as mi

    rng = np.random.default_rng(8)
    x, s = _case(rng, 3, 4, 12345, "fp16")
    want = [t.clone() for t in mi.beam_select(x.cuda(), s.cuda())]
    assert all(t.shape == (3, 8) for t in want)
    xc, sc = x.cuda(), s.cuda()
    out = (torch.empty(3, 8, device="cuda"), *(torch.empty(3, 8, dtype=torch.int64, device="cuda") for _ in range(2)))
    ws = torch.empty(mi.beam.beam_workspace_bytes(12, 12345, 8), dtype=torch.uint8, device="cuda")
    ws.fill_(255)
    assert mi.beam_select(xc, sc, out=out, workspace=ws) is not None
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mi.beam_select(xc, sc)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        mi.beam_select(xc, sc, out=out, workspace=ws)
    for i in range(4):
        y, z = _case(rng, 3, 4, 12345, "fp16")
        xc.copy_(y)
        sc.copy_(z)
        g.replay()
        eager = mi.beam_select(xc, sc)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
        _check(eager, y, z, 8)
    assert mi.beam_select(xc[:0], sc[:0])[0].shape == (0, 8)


# ------------------------------------------------------------------ the step
KEYS = ("tokens", "lengths", "scores", "prompt_lengths", "finished_tokens", "finished_lengths", "finished_scores", "done")


def _state(mi, arrays):
    t = {k: torch.from_numpy(v.copy()).cuda() for k, v in arrays.items()}
    return mi.BeamState(**t)


def _arrays(state):
    return {k: getattr(state, k).cpu().numpy().copy() for k in KEYS}


def _same(state, want):
    for k in KEYS:
        got = getattr(state, k).cpu().numpy()
        if k.endswith("scores"):
            fine = np.isfinite(want[k])
            assert np.array_equal(np.where(fine, 0, got), np.where(fine, 0, want[k]), equal_nan=True), k
            assert (np.abs(got[fine] - want[k][fine]) <= 4 * HALF * np.abs(want[k][fine])).all(), k
        else:
            assert np.array_equal(got, want[k]), (k, got, want[k])


@pytest.mark.parametrize("prompts,beams,n,room,ends,penalty,early", [
    (1, 1, 30, 12, (3,), 1.0, False), (3, 2, 40, 16, (3,), 0.0, True), (4, 4, 60, 14, (3, 9), 1.0, "never"),
    (5, 3, 9000, 25, (), 1.0, False), (6, 8, 25, 19, (1, 2, 3), 2.0, False), (2, 32, 50, 10, (5, 6, 7), 0.6, True),
    (3, 5, 100, 21, (3, 3), -1.0, "never"), (2, 16, 3, 9, (0,), 1.0, False), (2, 128, 40, 6, (), 1.0, False)])
@pytest.mark.parametrize("in_place", [True, False])
def test_step_follows_the_definition(prompts, beams, n, room, ends, penalty, early, in_place):
    """Steps from a prompt to full rows: each against the plain one, from the state that it found.  The
    kernel's own selection (tested above) gives the candidates, so that no rounding decides here."""
    import rwkv7mi as mi

    rng = np.random.default_rng(prompts * n + room)
    ids = torch.from_numpy(rng.integers(0, n, (prompts, 4)))
    state = mi.BeamState.start(ids.cuda(), beams, room, lengths=rng.integers(1, 5, prompts))
    for _ in range(room):
        x = rng.standard_normal((prompts * beams, n)) * 2
        if ends:  # ends come and go
            x[:, list(ends)] += np.where(rng.random((prompts * beams, 1)) < 0.4, 4.0, -4.0)
        if rng.random() < 0.2:
            x[rng.random(x.shape) < 0.9] = -np.inf
        x = torch.from_numpy(x).half().cuda()
        before = _arrays(state)
        found = mi.beam_select(x, state.scores, (1 + len(ends)) * beams)
        val, tok, row = (t.cpu().numpy() for t in found)
        nxt, rows, want = ref.step((val, tok, row - beams * np.arange(prompts)[:, None]), before, ends, penalty, early, 7)
        how = dict(eos_token_id=list(ends) or None, length_penalty=penalty, early_stopping=early, pad_token_id=7)
        if in_place:
            got, at, new = mi.beam_step(x, state, **how)
            assert new is state
        else:
            other = _state(mi, {k: (np.zeros_like(v) if k != "finished_scores" else np.full_like(v, -5)) for k, v in before.items()})
            got, at, new = mi.beam_step(x, state, out=other, **how)
            assert new is other
            for k in KEYS:
                assert np.array_equal(getattr(state, k).cpu().numpy(), before[k], equal_nan=k.endswith("scores")), k
            # only the texts are written: what is behind them is zero here
            for key, lens in (("tokens", want["lengths"].reshape(prompts, beams)), ("finished_tokens", want["finished_lengths"])):
                want[key] = np.where(np.arange(room) < lens[..., None], want[key], 0)
        assert np.array_equal(got.cpu().numpy(), nxt) and np.array_equal(at.cpu().numpy(), rows)
        _same(new, want)
        moved = rows.reshape(prompts, beams)
        assert all((m[m - b * beams] == m).all() for b, m in enumerate(moved))  # what is read stays where it is
        state = new
    assert bool(state.done.all())


@pytest.mark.parametrize("prompts,beams,room", [(3, 4, 700), (2, 16, 2049), (1, 32, 1024), (3, 40, 999), (2, 8, 4096)])
def test_step_into_another_state_is_the_step_in_place(prompts, beams, room):
    """Long texts and hypotheses of all lengths, prompts that are done and full ones: the same state in
    place and into another one, whichever way its texts are copied, and the rest of the rows as it was."""
    import rwkv7mi as mi

    rng = np.random.default_rng(beams * room)
    n, ends = 400, [3, 5]
    length = rng.integers(room // 2, room, prompts)
    if prompts > 1:
        length[1] = room
    held = rng.integers(0, room + 1, (prompts, beams))
    has = rng.random((prompts, beams)) < 0.7
    arrays = dict(tokens=rng.integers(0, n, (prompts, beams, room)), lengths=np.repeat(length, beams).astype(np.int32),
                  scores=(rng.standard_normal((prompts, beams)) - 9).astype(np.float32),
                  prompt_lengths=(length // 2).astype(np.int32), finished_tokens=rng.integers(0, n, (prompts, beams, room)),
                  finished_lengths=held.astype(np.int32),
                  finished_scores=np.where(has, rng.standard_normal((prompts, beams)) * 0.02 - 0.05, -np.inf).astype(np.float32),
                  done=np.arange(prompts) == 2)
    x = rng.standard_normal((prompts * beams, n)) * 2
    x[:, ends] += 4.0 * (rng.random((prompts * beams, 1)) < 0.3)
    x = torch.from_numpy(x).half().cuda()
    ends = ends[: 2 if beams <= 40 else 1]
    here, there = _state(mi, arrays), _state(mi, arrays)
    other = _state(mi, {k: np.full_like(v, 7) if v.dtype != bool else v for k, v in arrays.items()})
    a = mi.beam_step(x, here, eos_token_id=ends)
    b = mi.beam_step(x, there, eos_token_id=ends, out=other)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for k in KEYS:
        assert np.array_equal(getattr(there, k).cpu().numpy(), arrays[k]), k
        got, want = getattr(other, k).cpu().numpy(), getattr(here, k).cpu().numpy()
        if k.endswith("tokens"):
            lens = (here.lengths.view(prompts, beams) if k == "tokens" else here.finished_lengths).cpu().numpy()
            want = np.where(np.arange(room) < lens[..., None], want, 7)
        assert np.array_equal(got, want), k
    val, tok, row = (t.cpu().numpy() for t in mi.beam_select(x, there.scores, (1 + len(ends)) * beams))
    nxt, rows, want = ref.step((val, tok, row - beams * np.arange(prompts)[:, None]), arrays, tuple(ends), 1.0, False)
    assert np.array_equal(a[0].cpu().numpy(), nxt) and np.array_equal(a[1].cpu().numpy(), rows)
    _same(here, want)


def test_step_one_end_token_as_a_number_and_logits_per_prompt():
    import rwkv7mi as mi

    x, _ = _case(np.random.default_rng(2), 2, 3, 50, "fp32")
    ids = torch.tensor([[1, 2], [3, 4]], device="cuda")
    a, b = (mi.BeamState.start(ids, 3, 9) for _ in range(2))
    r1 = mi.beam_step(x.cuda(), a, eos_token_id=5)
    nxt, rows = torch.empty(6, dtype=torch.int64, device="cuda"), torch.empty(6, dtype=torch.int64, device="cuda")
    ws = torch.empty(mi.beam.beam_workspace_bytes(6, 50, 6), dtype=torch.uint8, device="cuda")
    r2 = mi.beam_step(x.cuda().view(2, 3, 50), b, eos_token_id=[5], next_tokens=nxt, rows=rows, workspace=ws)
    assert r2[0] is nxt and r2[1] is rows
    assert torch.equal(r1[0], nxt) and torch.equal(r1[1], rows) and torch.equal(a.tokens, b.tokens)


def test_step_captured():
    """A captured step in place, replayed with eager steps of another search between."""
    import rwkv7mi as mi

    rng = np.random.default_rng(11)
    ids = torch.from_numpy(rng.integers(0, 500, (3, 2))).cuda()
    a, b = (mi.BeamState.start(ids, 4, 12) for _ in range(2))
    x = torch.empty(12, 500, device="cuda", dtype=torch.float16)
    nxt, rows = (torch.empty(12, dtype=torch.int64, device="cuda") for _ in range(2))
    keep = _arrays(a)
    x.normal_()
    mi.beam_step(x, a, eos_token_id=3, next_tokens=nxt, rows=rows)
    for k in KEYS:
        getattr(a, k).copy_(torch.from_numpy(keep[k]))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        mi.beam_step(x, a, eos_token_id=3, next_tokens=nxt, rows=rows)
    for _ in range(11):
        y = torch.from_numpy(rng.standard_normal((12, 500)) * 2).half()
        x.copy_(y)
        g.replay()
        n2, r2, _ = mi.beam_step(y.cuda(), b, eos_token_id=3)
        torch.cuda.synchronize()
        assert torch.equal(nxt, n2) and torch.equal(rows, r2)
        for k in KEYS:
            assert torch.equal(getattr(a, k), getattr(b, k)), k


def test_best_hypotheses():
    import rwkv7mi as mi

    ids = torch.tensor([[1], [2]], device="cuda")
    s = mi.BeamState.start(ids, 2, 4)
    s.finished_scores[0, 1], s.finished_lengths[0, 1] = -1.0, 3
    s.finished_tokens[0, 1, :3] = torch.tensor([1, 8, 9], device="cuda")
    s.scores.copy_(torch.tensor([[-0.5, -0.6], [-3.0, -2.0]]))
    s.lengths.fill_(3)
    s.tokens[1, 1, :3] = torch.tensor([2, 6, 7], device="cuda")
    tok, length, score = s.best(2)
    assert tok[0, 0, :3].tolist() == [1, 8, 9] and tok[1, 0, :3].tolist() == [2, 6, 7]
    assert torch.allclose(score.cpu(), torch.tensor([[-1.0, -0.25], [-1.0, -1.5]]))
    assert length.tolist() == [[3, 3], [3, 3]]

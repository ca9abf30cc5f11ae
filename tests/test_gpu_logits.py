"""The logits step (penalties, bias, mask, greedy token) against plain 64-bit numpy."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _words(bits: np.ndarray) -> torch.Tensor:
    """Boolean [rows, n] -> int32 words, bit t % 32 of word t // 32."""
    rows, n = bits.shape
    full = np.zeros((rows, (n + 31) // 32 * 32), dtype=bool)
    full[:, :n] = bits
    return torch.from_numpy(np.packbits(full, axis=1, bitorder="little").view(np.int32).copy())


def _reference(x, hist, lengths, pen, bias, bits):
    """64-bit result and an error bound: five fp32 operations on values no larger than
    the sum of all magnitudes (and 2^-40 an occurrence in a count, here 5 x 2^-24 x 2^-16
    or more), then one rounding."""
    y = x.double().numpy().copy()
    rows, n = y.shape
    mag = np.abs(np.where(np.isfinite(y), y, 0.0))
    for r in range(rows):
        theta, pres, freq, decay = (float(p[r]) for p in pen)
        h = hist[r, :lengths[r]]
        w = decay ** np.arange(len(h), dtype=np.float64)[::-1]
        keep = (h >= 0) & (h < n)
        c, k = np.zeros(n), np.zeros(n, dtype=int)
        np.add.at(c, h[keep], w[keep])
        np.add.at(k, h[keep], 1)
        seen = k > 0
        v = y[r]
        v = np.where(seen, np.where(v > 0, v / theta, v * theta), v)
        v = np.where(seen, v - pres - freq * c, v)
        y[r] = v
        mag[r] = np.where(seen, mag[r] * max(theta, 1 / theta) + abs(pres) + abs(freq) * (c + k * 2.0 ** -16),
                          mag[r])
    if bias is not None:
        y, mag = y + bias, mag + np.abs(bias)
    if bits is not None:
        y[~bits] = -np.inf
    return y, 5 * 2.0 ** -24 * mag


def _first_max(t: torch.Tensor) -> torch.Tensor:
    v = t.detach().cpu().double().numpy()
    return torch.tensor([int(np.argmax(np.isnan(r))) if np.isnan(r).any() else int(np.argmax(r)) for r in v])


def _check(got, want, bound, dt):
    got = got.cpu().double().numpy()
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    tol = bound + (np.abs(np.where(fine, want, 0)) + bound) * (torch.finfo(dt).eps / 2)
    assert (np.abs(got - want)[fine] <= tol[fine]).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,n,length", [(1, 1, 3), (1, 31, 5), (2, 33, 0), (3, 1000, 40), (7, 4096, 300),
                                           (4, 4097, 1), (5, 8191, 2000), (2, 65536, 700), (33, 5003, 64)])
@pytest.mark.parametrize("decayed", [False, True])
def test_process_logits_against_64_bits(rows, n, length, dtype, decayed):
    import rwkv7mi as mi

    rng = np.random.default_rng(rows * n + length + decayed)
    dt = DTYPES[dtype]
    x = torch.from_numpy(rng.standard_normal((rows, n)) * 4).to(dt)
    hist = (n * rng.random((rows, length)) ** 3).astype(np.int64)
    hist[rng.random(hist.shape) < 0.05] = -1
    hist[rng.random(hist.shape) < 0.05] = n + 5
    lengths = rng.integers(0, length + 1, rows)
    lengths[0] = length
    pen = [rng.uniform(0.8, 1.6, rows), rng.uniform(-0.2, 0.8, rows), rng.uniform(0, 0.5, rows),
           rng.uniform(0.9, 1.0, rows) if decayed else np.ones(rows)]
    pen = [p.astype(np.float32) for p in pen]
    dev = [torch.from_numpy(p).cuda() for p in pen]
    bits = rng.random((rows, n)) < 0.4
    bits[-1] = False
    for bias, mask, bits32 in ((None, None, False), (rng.standard_normal(n).astype(np.float32), bits, True),
                               (rng.standard_normal((rows, n)).astype(np.float32), bits[:1], False)):
        whole = None if mask is None else np.broadcast_to(mask, (rows, n))
        want, bound = _reference(x, hist, lengths, pen, bias, whole)
        h = torch.from_numpy(hist).cuda()
        nxt = torch.empty(rows, device="cuda", dtype=torch.int64)
        kw = dict(history=h.int() if bits32 else h, lengths=torch.from_numpy(lengths).int().cuda(),
                  repetition_penalty=dev[0], presence_penalty=dev[1], frequency_penalty=dev[2],
                  penalty_decay=dev[3] if decayed else 1.0, bias=None if bias is None else torch.from_numpy(bias).cuda(),
                  allowed=None if mask is None else _words(mask).cuda())
        got = mi.process_logits(x.cuda(), next_tokens=nxt, **kw)
        assert got.dtype == dt
        _check(got, want, bound, dt)
        assert torch.equal(nxt.cpu(), _first_max(got))
        wide = torch.empty(rows, n, device="cuda")
        mi.process_logits(x.cuda(), out=wide, **kw)
        _check(wide, want, bound, torch.float32)
        same = x.cuda()
        mi.process_logits(same, out=same, **kw)
        assert torch.equal(same.cpu().nan_to_num(), got.cpu().nan_to_num())


def test_masked_infinities_and_nans():
    """A masked place is -inf whatever it or its bias holds; an unmasked NaN stays and counts
    as the maximum; a row with nothing allowed is all -inf and gives token 0."""
    import rwkv7mi as mi

    n = 700
    x = torch.randn(4, n)
    low = torch.finfo(torch.float32).min
    x[0, 10], x[0, 20], x[0, 30], x[0, 40] = float("nan"), float("inf"), float("-inf"), low
    x[2, 50] = float("nan")
    x[3, 60], x[3, 5] = float("inf"), low
    bits = np.ones((4, n), dtype=bool)
    bits[0, [10, 20, 30, 40]] = False
    bits[1] = False
    bias = torch.zeros(n)
    bias[20] = float("nan")
    bias[60] = low
    bits[2:, 20] = False
    nxt = torch.empty(4, device="cuda", dtype=torch.int64)
    got = mi.process_logits(x.cuda(), bias=bias.cuda(), allowed=_words(bits).cuda(), next_tokens=nxt).cpu()
    assert (got[0, [10, 20, 30, 40]] == float("-inf")).all() and not torch.isnan(got[0]).any()
    assert (got[1] == float("-inf")).all() and int(nxt[1]) == 0
    assert torch.isnan(got[2, 50]) and int(nxt[2]) == 50
    assert got[3, 60] == float("inf") and int(nxt[3]) == 60 and got[3, 5] == low
    assert torch.equal(nxt.cpu(), _first_max(got))


def test_numbers_equal_tensors_and_defaults_change_nothing():
    import rwkv7mi as mi

    x = torch.randn(5, 3001).half().cuda()
    h = torch.randint(0, 3001, (5, 90), device="cuda")
    assert torch.equal(mi.process_logits(x, history=h), x)
    full = lambda v: torch.full((5,), v, device="cuda")
    a = mi.process_logits(x, history=h, repetition_penalty=1.25, presence_penalty=0.5, frequency_penalty=0.25,
                          penalty_decay=0.5)
    b = mi.process_logits(x, history=h, repetition_penalty=full(1.25), presence_penalty=full(0.5),
                          frequency_penalty=full(0.25), penalty_decay=full(0.5))
    assert torch.equal(a, b) and not torch.equal(a, x)
    assert mi.process_logits(x[:0], history=h[:0]).shape == (0, 3001)


def test_strided_logits_and_rows_behind():
    import rwkv7mi as mi

    buf = torch.randn(6, 2, 1031).half().cuda()
    view = buf[:, 1]  # rows 2062 apart, at odd offsets
    h = torch.randint(0, 1031, (6, 33), device="cuda")
    kw = dict(history=h[:, :30], presence_penalty=1.0, lengths=torch.full((6,), 29, device="cuda", dtype=torch.int32))
    want = mi.process_logits(view.contiguous(), **kw)
    assert torch.equal(mi.process_logits(view, **kw), want)
    out = torch.full((8, 1040), 3.0, device="cuda", dtype=torch.float16)
    mi.process_logits(view, out=out[1:7, 5:1036], **kw)
    assert torch.equal(out[1:7, 5:1036], want)
    assert (out[0] == 3).all() and (out[7] == 3).all() and (out[:, :5] == 3).all() and (out[:, 1036:] == 3).all()
    one = torch.randn(1, 1031).half().cuda().expand(6, 1031)
    assert torch.equal(mi.process_logits(one, **kw), mi.process_logits(one.contiguous(), **kw))
    mi.process_logits(view, out=view, **kw)
    assert torch.equal(view, want)


def test_append_grows_the_history_and_stops_at_its_end():
    import rwkv7mi as mi

    for dt in (torch.int64, torch.int32):
        n, cap = 300, 6
        h = torch.full((3, cap + 2), -7, device="cuda", dtype=dt)
        lengths = torch.tensor([0, 5, 6], device="cuda", dtype=torch.int32)
        nxt = torch.empty(3, device="cuda", dtype=torch.int64)
        again = torch.empty(3, device="cuda", dtype=torch.int64)
        for step in range(3):
            x = torch.randn(3, n).cuda()
            before, at = h.clone(), lengths.tolist()
            mi.process_logits(x, history=h[:, :cap], lengths=lengths, repetition_penalty=2.0, next_tokens=nxt,
                              next_tokens2=again, append=True)
            assert torch.equal(nxt, again)
            for r in range(3):
                if at[r] < cap:
                    before[r, at[r]] = nxt[r].to(dt)
            assert torch.equal(h, before)
            assert lengths.tolist() == [min(a + 1, cap) for a in at]


def test_step_in_a_graph():
    """A captured step that appends its token: every replay equals the eager step."""
    import rwkv7mi as mi

    n, cap = 5000, 40
    x = torch.randn(4, n, device="cuda").half()
    state = lambda: (torch.zeros(4, cap, device="cuda", dtype=torch.int64), torch.zeros(4, device="cuda", dtype=torch.int32),
                     torch.empty(4, device="cuda", dtype=torch.int64))
    def step(h, m, t):
        return mi.process_logits(x, history=h, lengths=m, repetition_penalty=1.5, frequency_penalty=0.5,
                                 penalty_decay=0.9, next_tokens=t, append=True)
    eager, captured = state(), state()
    step(*state())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = step(*captured)
    for k in range(4):
        x.copy_(torch.randn(4, n, device="cuda").half())
        want = step(*eager)
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and all(torch.equal(a, b) for a, b in zip(eager, captured))
    assert captured[1].tolist() == [4] * 4


@pytest.mark.parametrize("n", [3001, 2048])
def test_many_entries_of_one_token_and_of_one_slice(n):
    """More decayed entries in 2048 tokens than are gathered at once: all of one token, and all
    of a few neighbours; counts against the sums of the powers."""
    import rwkv7mi as mi

    L, decay = 5000, 0.999
    hist = torch.full((3, L), 7, dtype=torch.long)
    hist[1] = torch.arange(L) % 97 + 1000
    hist[2, ::2] = n  # outside the vocabulary
    hist[2, 1::4] = -(2 ** 63)
    y = mi.process_logits(torch.zeros(3, n, device="cuda"), history=hist.cuda(), frequency_penalty=1.0, penalty_decay=decay)
    age = torch.arange(L - 1, -1, -1, dtype=torch.float64)
    want = torch.zeros(3, n, dtype=torch.float64)
    for r in range(3):
        ok = (hist[r] >= 0) & (hist[r] < n)
        want[r].index_add_(0, hist[r][ok], -(decay ** age)[ok])
    # steps of 2^-40 for each of 5000 entries, decay rounded to fp32 (5000 x 2^-24 of a power), one fp32 rounding
    bound = L * 2.0 ** -41 + want.abs() * (L * 2.0 ** -24 + 2.0 ** -24)
    assert ((y.cpu().double() - want).abs() <= bound).all()


def test_settings_of_one_row_shared_and_two_streams():
    """Every penalty as a tensor of one value, one bias and mask for all rows, an expanded row
    of logits, and two steps at once on two streams with a history each."""
    import rwkv7mi as mi

    g = torch.Generator().manual_seed(3)
    n = 2500
    row = torch.randn(1, n, generator=g).cuda()
    hist = torch.randint(0, n, (4, 50), generator=g).cuda()
    bias = torch.randn(n, generator=g).cuda()
    words = torch.randint(-2 ** 31, 2 ** 31, ((n + 31) // 32,), generator=g).to(torch.int32).cuda()
    one = lambda v: torch.tensor(v, device="cuda")
    want = mi.process_logits(row.repeat(4, 1), history=hist, repetition_penalty=1.3, presence_penalty=0.5,
                             frequency_penalty=0.25, penalty_decay=0.75, bias=bias.repeat(4, 1), allowed=words.repeat(4, 1))
    got = mi.process_logits(row.expand(4, n), history=hist, repetition_penalty=one(1.3), presence_penalty=one(0.5),
                            frequency_penalty=one(0.25), penalty_decay=one(0.75), bias=bias, allowed=words)
    assert torch.equal(got, want)
    sides = []
    for k in range(2):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        state = (torch.zeros(4, 80, dtype=torch.long, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"),
                 torch.zeros(4, dtype=torch.long, device="cuda"))
        sides.append((s, state))
    torch.cuda.synchronize()
    for _ in range(20):
        for s, (h, lengths, nxt) in sides:
            with torch.cuda.stream(s):
                mi.process_logits(row.expand(4, n), history=h, lengths=lengths, presence_penalty=3.0, next_tokens=nxt,
                                  append=True)
    torch.cuda.synchronize()
    (_, a), (_, b) = sides
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and a[1].tolist() == [20] * 4
    order = torch.argsort(row[0], descending=True, stable=True)
    assert a[0][0, 0] == order[0]

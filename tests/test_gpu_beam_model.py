"""Beam search through the model, the cache and the state pool: the whole search against one written out
over single forwards, against transformers' own, and the caches' rows against torch's indexing."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import beam_reference as ref

pytestmark = pytest.mark.gpu


def _config(layers=2, vocab=512):
    from rwkv7mi.model import NativeRWKV7Config

    return NativeRWKV7Config(vocab_size=vocab, hidden_size=128, num_hidden_layers=layers, intermediate_size=256,
                             decay_low_rank_dim=32, a_low_rank_dim=32, gate_low_rank_dim=64, v_low_rank_dim=32)


def _model(dtype=torch.float16, **kw):
    from rwkv7mi.model import NativeRWKV7ForCausalLM, random_weights

    cfg = _config(**kw)
    w = random_weights(cfg, seed=0, device="cpu", dtype=dtype)
    w["lm_head.weight"] = w["lm_head.weight"] * 20  # (logits that tell tokens apart)
    return NativeRWKV7ForCausalLM(cfg, w, device="cuda", dtype=dtype)


def _ids(rows, t=5, seed=1, vocab=512):
    return torch.randint(0, vocab, (rows, t), generator=torch.Generator().manual_seed(seed)).cuda()


def _cache(model, rows, seed=0):
    c = model.new_cache(rows)
    g = torch.Generator("cuda").manual_seed(seed)
    for t in c._all_tensors():
        t.copy_(torch.randn(t.shape, device="cuda", generator=g) * 5)
    return c


def _plain_search(model, ids, beams, steps, ends, penalty, early, change=None):
    """The search over eager forwards of a cache whose rows torch's indexing moves."""
    p, t = ids.shape
    out = model(ids)
    cache = out.past_key_values
    pick = lambda idx: cache._map(lambda v: v[idx])  # noqa: E731
    pick(torch.arange(p, device="cuda").repeat_interleave(beams))
    logits = out.logits[:, -1].repeat_interleave(beams, 0)
    ids = ids.cpu().numpy()
    s = dict(tokens=np.zeros((p, beams, t + steps), np.int64), lengths=np.full(p * beams, t, np.int32),
             scores=np.where(np.arange(beams) == 0, 0, -np.inf).astype(np.float32)[None].repeat(p, 0),
             prompt_lengths=np.full(p, t, np.int32), finished_tokens=np.zeros((p, beams, t + steps), np.int64),
             finished_lengths=np.zeros((p, beams), np.int32),
             finished_scores=np.full((p, beams), -np.inf, np.float32), done=np.zeros(p, bool))
    s["tokens"][:, :, :t] = ids[:, None]
    for _ in range(steps):
        x = (logits if change is None else change(logits, s)).double().cpu().numpy().reshape(p, beams, -1)
        val, tok, beam = ref.select(ref.values(x, s["scores"]), (1 + len(ends)) * beams)
        nxt, rows, s = ref.step((val.astype(np.float32), tok, beam), s, ends, penalty, early)
        pick(torch.from_numpy(rows).cuda())
        logits = model(torch.from_numpy(nxt)[:, None].cuda(), past_key_values=cache, use_graph=False).logits[:, -1]
    return s


@pytest.mark.parametrize("beams,ends,penalty,early", [(1, (), 1.0, False), (4, (7,), 1.0, False), (3, (7, 80), 0.5, True),
                                                      (5, (3, 9), 2.0, "never")])
@pytest.mark.parametrize("use_graph", [True, False])
def test_generate_beam_follows_the_search(beams, ends, penalty, early, use_graph):
    model = _model()
    ids = _ids(3)
    s = _plain_search(model, ids, beams, 12, ends, penalty, early)
    got, scores = model.generate_beam(ids, 12, num_beams=beams, eos_token_id=list(ends) or None, length_penalty=penalty,
                                      early_stopping=early, num_return_sequences=beams, use_graph=use_graph, pad_token_id=511,
                                      return_scores=True)
    order = np.argsort(-s["finished_scores"], axis=1, kind="stable")
    n = int(s["finished_lengths"].max())
    assert got.shape == (3 * beams, n) and np.isfinite(s["finished_scores"]).all()
    for i, (b, k) in enumerate((b, k) for b in range(3) for k in order[b]):
        length = s["finished_lengths"][b, k]
        assert got[i, :length].tolist() == s["finished_tokens"][b, k, :length].tolist()
        assert (got[i, length:] == 511).all()
        # 12 sums of log-probabilities, each rounded to fp32 behind a 64-bit sum off by the fp32 lse (46 2^-24)
        value = s["finished_scores"][b, k]
        assert abs(float(scores[i]) - value) <= 12 * 46 * 2.0 ** -24 + 13 * 2.0 ** -24 * abs(value)
    best = model.generate_beam(ids, 12, num_beams=beams, eos_token_id=list(ends) or None, length_penalty=penalty,
                               early_stopping=early, use_graph=use_graph, pad_token_id=511)
    assert best.shape[0] == 3 and all(a[:n].tolist() == b[:n].tolist() for a, b in
                                      zip(best, got[::beams, :best.shape[1]]) for n in [best.shape[1]])


@pytest.mark.parametrize("beams,eos,penalty,early", [(2, None, 1.0, False), (4, 7, 1.0, False), (4, 7, 0.5, True), (3, 80, 1.5, "never")])
def test_generate_beam_matches_transformers(beams, eos, penalty, early):
    model = _model(torch.float32)
    ids = _ids(2, 6, 4)
    mine = model.generate_beam(ids, 10, num_beams=beams, eos_token_id=eos, length_penalty=penalty, early_stopping=early,
                               num_return_sequences=beams, pad_token_id=0)
    theirs = model.generate(ids, max_new_tokens=10, num_beams=beams, do_sample=False, eos_token_id=eos, length_penalty=penalty,
                            early_stopping=early, num_return_sequences=beams, pad_token_id=0,
                            attention_mask=torch.ones_like(ids))
    n = min(mine.shape[1], theirs.shape[1])
    assert torch.equal(mine[:, :n], theirs[:, :n]) and not mine[:, n:].any() and not theirs[:, n:].any()


def test_generate_beam_under_penalties_and_masks():
    import rwkv7mi as mi

    model = _model()
    ids = _ids(2)
    words = torch.full((16,), -1, dtype=torch.int32)
    words[3] = 0  # tokens 96..127 are not allowed
    bias = torch.zeros(512)
    bias[40:60] = 2.0

    def change(logits, s):
        h = torch.from_numpy(s["tokens"].reshape(-1, s["tokens"].shape[2])).cuda()
        return mi.process_logits(logits.contiguous(), history=h, lengths=torch.from_numpy(s["lengths"]).cuda(), out=torch.empty(
            logits.shape, device="cuda"), repetition_penalty=1.4, presence_penalty=0.3, bias=bias.cuda(), allowed=words.cuda())

    s = _plain_search(model, ids, 3, 9, (7,), 1.0, False, change)
    got = model.generate_beam(ids, 9, num_beams=3, eos_token_id=7, repetition_penalty=1.4, presence_penalty=0.3, bias=bias,
                              allowed=words)
    for b in range(2):
        k = int(np.argmax(s["finished_scores"][b]))
        length = s["finished_lengths"][b, k]
        assert got[b, :length].tolist() == s["finished_tokens"][b, k, :length].tolist()
    assert not ((got[:, 5:] >= 96) & (got[:, 5:] < 128)).any()


def test_generate_beam_of_one_beam_is_greedy_and_short_runs():
    model = _model()
    ids = _ids(2)
    assert torch.equal(model.generate_beam(ids, 8, num_beams=1), model.generate_greedy(ids, 8))
    assert model.generate_beam(ids, 1, num_beams=4).shape == (2, 6)
    with pytest.raises(ValueError):
        model.generate_beam(ids, 0)
    with pytest.raises(ValueError):
        model.generate_beam(ids, 4, num_beams=2, num_return_sequences=3)


def test_generate_beam_stops_when_all_are_done():
    """Every continuation but the end is masked away: the search ends long before its room."""
    model = _model()
    words = torch.zeros(16, dtype=torch.int32)
    words[0] = 1 << 7
    model.generate_beam(_ids(1), 2, num_beams=3)  # (captures the graph)
    runner = model.graph_runner(3)
    before = runner.replays
    got = model.generate_beam(_ids(1), 60, num_beams=3, eos_token_id=7, allowed=words)
    assert got.tolist() == [_ids(1)[0].tolist() + [7]] and runner.replays - before <= 8


def test_fp16_state_beams():
    """The fp16-state lane's decay phase follows the beams with the state."""
    model = _model()
    model.state_dtype = torch.float16
    ids = _ids(2)
    s = _plain_search(model, ids, 3, 7, (), 1.0, False)
    got = model.generate_beam(ids, 7, num_beams=3)
    for b in range(2):
        assert got[b].tolist() == s["finished_tokens"][b, int(np.argmax(s["finished_scores"][b]))].tolist()


@pytest.mark.parametrize("state", [torch.float32, torch.float16])
def test_cache_rows(state):
    """select, reorder, repeat of a cache in one allocation, of one in many, and of part of one."""
    model = _model()
    model.state_dtype = state
    for idx in ([2, 0], [1], [0, 0, 3, 2, 1], torch.tensor([3, 3], device="cuda"), torch.tensor([1, 0, 2, 3])):
        for scattered in (False, True):
            c = _cache(model, 4)
            if scattered:
                c._map(lambda t: t.clone())
            old = [t.clone() for t in c._all_tensors()]
            at = torch.as_tensor(idx).cuda()
            kept = c.select_batch(idx, inplace=False)
            assert all(torch.equal(a, b) for a, b in zip(c._all_tensors(), old))
            assert all(torch.equal(a, b[at]) and a.is_contiguous() for a, b in zip(kept._all_tensors(), old))
            assert (kept._stacked() is not None) == (not scattered)
            view = list(c._all_tensors())
            c.reorder_cache(idx)
            assert all(torch.equal(a, b[at]) for a, b in zip(c._all_tensors(), old))
            assert all(torch.equal(a, b) for a, b in zip(view, old))  # (new tensors: others may hold the old)
            c.batch_repeat_interleave(3)
            assert all(torch.equal(a, b[at].repeat_interleave(3, 0)) for a, b in zip(c._all_tensors(), old))
    c = _cache(model, 4)
    assert c.select_batch([], inplace=False).get_batch_size() == 0
    for bad in ([4], [-1], torch.tensor([0, -1]), torch.zeros(1, 2, dtype=torch.long, device="cuda")):
        with pytest.raises(IndexError):
            c.select_batch(bad)


def test_bound_cache_rows_trade_places():
    model = _model()
    runner = model.graph_runner(6)
    c = _cache(model, 6)
    runner.replay(_ids(1, 6)[0], c)
    for idx in ([5, 4, 3, 2, 1, 0], [0, 0, 0, 5, 5, 1], [0, 1, 2, 3, 4, 5]):
        for at in (torch.tensor(idx), torch.tensor(idx, device="cuda")):
            old = [t.clone() for t in runner.cache._all_tensors()]
            c.reorder_cache(at)
            assert c._native_graph_bound_to(runner)
            assert all(torch.equal(a, b[torch.tensor(idx)]) for a, b in zip(runner.cache._all_tensors(), old))
    with pytest.raises(IndexError):
        c.reorder_cache(torch.tensor([0, 1, 2, 3, 4, 6]))
    assert c._native_graph_bound_to(runner)


def _pool(capacity=6, seed=0):
    from rwkv7mi.state_pool import RWKV7StatePool

    pool = RWKV7StatePool(_config(), capacity, device="cuda")
    g = torch.Generator("cuda").manual_seed(seed)
    for t in pool._tensors():
        t[:, :capacity].copy_(torch.randn(t[:, :capacity].shape, device="cuda", generator=g))
    return pool


def _copy(pool):
    return [t.clone() for t in pool._tensors()]


def test_pool_fork():
    pool = _pool()
    (s, g), (s2, g2) = pool.allocate(["p", "q"])
    pool.state[:, s].normal_()
    pool.seen_tokens[s] = 17
    old = _copy(pool)
    new = pool.fork(s, g, ["a", "b", "c"])
    assert [n for n, _ in new] == [2, 3, 4] and [pool.seen_tokens[n] for n, _ in new] == [17] * 3
    for t, o in zip(pool._tensors(), old):
        assert torch.equal(t[:, 2:5], o[:, s:s + 1].expand_as(t[:, 2:5]))
        assert torch.equal(t[:, [0, 1, 5, 6]], o[:, [0, 1, 5, 6]])
    pool.free([s], [g])
    with pytest.raises(ValueError):
        pool.fork(s, g, ["d"])
    with pytest.raises(RuntimeError):
        pool.fork(s2, g2, ["d", "e", "f"])
    assert pool.fork(s2, g2, []) == []


def test_pool_reorder():
    pool = _pool()
    slots, gens = zip(*pool.allocate(list("abcde")))
    order = [4, 1, 3]  # slots of a search, in any order
    for parents, seen in (([1, 1, 0], [5, 6, 7]), (torch.tensor([2, 0, 0], device="cuda"), [5, 5, 5]), ([0, 1, 2], [1, 2, 3])):
        for t in pool._tensors():
            t.normal_()
        for s, n in zip(order, seen):
            pool.seen_tokens[s] = n
        old = _copy(pool)
        pool.reorder(order, [gens[s] for s in order], parents)
        at = [int(p) for p in parents]
        for t, o in zip(pool._tensors(), old):
            assert torch.equal(t[:, order], o[:, [order[p] for p in at]])
            assert torch.equal(t[:, [0, 2, 5, 6]], o[:, [0, 2, 5, 6]])
        assert [pool.seen_tokens[s] for s in order] == [seen[p] for p in at]
    for bad in ([0, 1], [0, 1, 3], [0, 1, -1], torch.zeros(2, dtype=torch.long, device="cuda")):
        with pytest.raises(ValueError):
            pool.reorder(order, [gens[s] for s in order], bad)
    with pytest.raises(ValueError):  # seen_tokens differ and the host does not know who follows whom
        pool.reorder(order, [gens[s] for s in order], torch.zeros(3, dtype=torch.long, device="cuda"))
    with pytest.raises(ValueError):
        pool.reorder(order, [9, 9, 9], [0, 1, 2])


def test_pool_compact_and_resize():
    pool = _pool(8)
    handles = pool.allocate(list("abcdefgh"))
    for t in pool._tensors():
        t[:, :8].normal_()
    for s in range(8):
        pool.seen_tokens[s] = 10 + s
    pool.free([0, 3, 5], [handles[s][1] for s in (0, 3, 5)])
    old = _copy(pool)
    with pytest.raises(ValueError):
        pool.resize(5)
    moved = pool.compact()
    assert moved == {5 + 1: (0, 1), 7: (3, 1)} and pool.free_slots() == 3
    for t, o in zip(pool._tensors(), old):
        assert torch.equal(t[:, :5], o[:, [6, 1, 2, 7, 4]])
    assert pool.seen_tokens[:5] == [16, 11, 12, 17, 14] and pool.owner == {0: "g", 1: "b", 2: "c", 3: "h", 4: "e"}
    pool.check([0, 1, 2, 3, 4], [1, 0, 0, 1, 0])
    with pytest.raises(ValueError):
        pool.check([6])
    assert pool.compact() == {}
    pool.resize(5)
    assert pool.capacity == 5 and pool.scratch_slot == 5 and pool.state.shape[1] == 6 and not pool.state[:, 5].any()
    for t, o in zip(pool._tensors(), old):
        assert torch.equal(t[:, :5], o[:, [6, 1, 2, 7, 4]])
    with pytest.raises(RuntimeError):
        pool.allocate(["x"])
    pool.resize(9)
    assert pool.free_slots() == 4 and not any(t[:, 5:].any() for t in pool._tensors())
    new = pool.allocate(list("wxyz"))
    # numbers that come back keep counting: the handles of before the pool shrank fit nothing
    assert new == [(5, 1), (6, 1), (7, 1), (8, 0)]
    for s, g in handles[5:]:
        with pytest.raises(ValueError):
            pool.check([s], [g])


def test_beams_in_the_pool():
    """A search over pool slots: fork, step, reorder, as a scheduler would, against the model's own."""
    from rwkv7mi import BeamState, beam_step
    from rwkv7mi.state_pool import PooledDecoder, RWKV7StatePool

    model = _model()
    ids = _ids(1)
    pool = RWKV7StatePool(model.config, 7, device="cuda")
    dec = PooledDecoder(model, pool)
    pool.allocate(["other"])
    (s, g), = pool.allocate(["p"])
    logits = dec.prefill([s], [g], ids)
    handles = [(s, g)] + pool.fork(s, g, ["1", "2", "3"])
    slots, gens = zip(*handles)
    state = BeamState.start(ids, 4, 5 + 9)
    nxt, rows, _ = beam_step(logits.expand(4, -1), state, eos_token_id=7)
    for _ in range(8):
        nxt, rows, _ = beam_step(dec.step(slots, gens, nxt), state, eos_token_id=7)
        pool.reorder(slots, gens, rows)
    tokens, lengths, _ = state.best(2)
    want = model.generate_beam(ids, 9, num_beams=4, eos_token_id=7, num_return_sequences=2)
    for i in range(2):
        n = int(lengths[0, i])
        assert tokens[0, i, :n].tolist() == want[i, :n].tolist()

"""Performance cases of beam search and of the state rows that it moves.

Four operators, each as a serving program calls it:

* ``select``: the best candidates of each prompt over its beams and the vocabulary;
* ``step``: the same with all that follows from it: ends, finished hypotheses, which row each
  surviving beam takes, the token rows;
* ``expand``: a cache's rows by an index into a new cache (prompts to beams, live rows of a batch);
* ``move``: rows of a recurrent state and its companions moved in place (beams, forks of a slot,
  compaction and fresh slots of a pool).

``listed()`` gives the fixed cases, ``draw(rng)`` one more of the same ranges, ``prepare`` the
inputs, ``run`` one pass (``own`` False: plain torch; True: this package's kernels), ``exact`` the
pass in 64 bits, ``work`` the bytes and operations that a pass cannot do without.
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
VOCAB = 65536
HEAD = 64
#: (layers, hidden) of the 0.1B, 1.5B, 2.9B and 7.2B models
MODELS = {"0.1B": (12, 768), "1.5B": (24, 2048), "2.9B": (32, 2560), "7.2B": (32, 4096)}


def _own():
    """This package's entry points (imported only where they are measured)."""
    if "rwkv7mi" not in sys.modules:
        sys.path.insert(0, str(Path.cwd() / "hf-adapter_amd"))
    import rwkv7mi

    return rwkv7mi


# ------------------------------------------------------------------ the cases
def _select(name, prompts, beams, vocab, dtype, candidates, masked=False):
    return {"name": name, "kind": "select", "prompts": prompts, "beams": beams, "vocab": vocab, "dtype": dtype,
            "candidates": candidates, "masked": masked}


def _step(name, prompts, beams, vocab, dtype, room, ends, penalty, early):
    return {"name": name, "kind": "step", "prompts": prompts, "beams": beams, "vocab": vocab, "dtype": dtype,
            "room": room, "ends": ends, "penalty": penalty, "early": early}


def _expand(name, model, rows, out, state):
    return {"name": name, "kind": "expand", "model": model, "rows": rows, "out": out, "state": state}


def _move(name, model, rows, group, pattern, moved, state):
    return {"name": name, "kind": "move", "model": model, "rows": rows, "group": group, "pattern": pattern,
            "moved": moved, "state": state}


def listed():
    return [
        # One chat's step with four beams: latency.
        _select("select_chat_1x4", 1, 4, VOCAB, "fp16", 8),
        # A few prompts, an odd vocabulary and an odd number of beams.
        _select("select_ragged_7x5", 7, 5, 50277, "bf16", 10),
        # Wide beams over fp32 scores that a grammar has masked, some beams not begun.
        _select("select_wide_4x32", 4, 32, VOCAB, "fp32", 64, True),
        # 64 prompts of 8 beams: the largest selection.
        _select("select_batch_64x8", 64, 8, VOCAB, "fp16", 16),
        # The whole step of one chat.
        _step("step_chat_1x4", 1, 4, VOCAB, "fp16", 500, 1, 1.0, False),
        # The whole step of a batch with long texts and two end tokens.
        _step("step_batch_64x8", 64, 8, VOCAB, "fp16", 4096, 2, 0.6, False),
        # Two prompts' states of the 7.2B model, each to four beams.
        _expand("expand_prompts_2_to_8", "7.2B", 2, 8, "fp32"),
        # The rows of a small model's batch that still run.
        _expand("expand_live_64_to_37", "0.1B", 64, 37, "fp32"),
        # One chat's four beams of the small model: latency.
        _move("move_beams_small_4", "0.1B", 4, 4, "beams", 3, "fp32"),
        # Eight chats of four beams of the 7.2B model: rows in the order of their scores.
        _move("move_beams_32", "7.2B", 32, 4, "beams", 3, "fp32"),
        # A long prompt's slot forked to eight requests.
        _move("move_fork_8", "7.2B", 17, 17, "fork", 8, "fp32"),
        # A pool of half-precision states: 9 slots move down into holes, 5 are made fresh.
        _move("move_compact_33", "2.9B", 33, 33, "compact", 9, "fp16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _row_bytes(model, state):
    layers, hidden = MODELS[model]
    return layers * hidden * HEAD * (4 if state == "fp32" else 2) + (2 * layers + 1) * hidden * 2


def draw(rng):
    kind = rng.choice(["select", "select", "select", "step", "step", "expand", "move", "move"])
    if kind in ("select", "step"):
        while True:
            prompts, beams = _log_int(rng, 1, 64), _log_int(rng, 1, 32)
            if prompts * beams <= 512:
                break
        vocab = VOCAB if rng.random() < 0.5 else _log_int(rng, 1000, VOCAB)
        # (at 512 rows fp32 logits would weigh more than the largest listed case)
        dtype = rng.choice(["fp16", "fp16", "bf16", "fp32" if prompts * beams <= 256 else "bf16"])
        if kind == "select":
            return {"kind": kind, "prompts": prompts, "beams": beams, "vocab": vocab, "dtype": dtype,
                    "candidates": rng.choice([beams, 2 * beams, 2 * beams, 3 * beams]), "masked": rng.random() < 0.3}
        return {"kind": kind, "prompts": prompts, "beams": beams, "vocab": vocab, "dtype": dtype,
                "room": _log_int(rng, 16, 4096), "ends": rng.choice([1, 1, 2, 3]),
                "penalty": rng.choice([1.0, 1.0, 0.0, 0.6, 2.0]), "early": rng.random() < 0.3}
    while True:
        model, state = rng.choice(list(MODELS)), rng.choice(["fp32", "fp32", "fp16"])
        if kind == "expand":
            rows, out = _log_int(rng, 1, 64), _log_int(rng, 1, 64)
            if max(rows, out) * _row_bytes(model, state) <= 0.5e9:
                return {"kind": kind, "model": model, "rows": rows, "out": out, "state": state}
            continue
        pattern = rng.choice(["beams", "beams", "fork", "compact"])
        group = rng.randint(2, 16) if pattern == "beams" else _log_int(rng, 4, 64)
        rows = group * rng.randint(1, 8) if pattern == "beams" else group
        most = group if pattern == "beams" else (group - 1 if pattern == "fork" else group // 2)
        if rows * _row_bytes(model, state) <= 0.9e9:
            return {"kind": kind, "model": model, "rows": rows, "group": group, "pattern": pattern,
                    "moved": rng.randint(1, most), "state": state}


# ------------------------------------------------------------------ inputs
def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFF)
    return g


def prepare(case, seed):
    if case["kind"] in ("select", "step"):
        return _prepare_search(case, _gen(seed, 1))
    return _prepare_rows(case, seed, _gen(seed, 2))


def _prepare_search(case, g):
    prompts, beams, vocab = case["prompts"], case["beams"], case["vocab"]
    rows = prompts * beams
    dt = DTYPES[case["dtype"]]
    x = torch.randn(rows, vocab, generator=g, device=DEV).mul_(3.0)
    scores = -40.0 + 2.0 * torch.randn(prompts, beams, generator=g, device=DEV)
    # a prompt's first step has one beam to go on from
    fresh = torch.rand(prompts, generator=g, device=DEV) < 0.1
    scores[:, 1:] = torch.where(fresh[:, None], -math.inf, scores[:, 1:])
    st = {"kind": case["kind"]}
    if case["kind"] == "select":
        if case["masked"]:  # grammars from free text to a few tokens, one row in twenty finished
            share = torch.tensor([1.0, 0.3, 0.001, 1.0], device=DEV)[torch.arange(rows, device=DEV) % 4]
            share = torch.where(torch.rand(rows, generator=g, device=DEV) < 0.05, 0.0, share)
            x.masked_fill_(torch.rand(rows, vocab, generator=g, device=DEV) >= share[:, None], -math.inf)
        st.update(logits=x.to(dt), scores=scores, candidates=case["candidates"])
        return st
    room, ends = case["room"], case["ends"]
    # texts end now and then: an end token near the top of a row's logits
    at = 5 + torch.arange(ends, device=DEV) * 7
    x[:, at] = torch.where(torch.rand(rows, ends, generator=g, device=DEV) < 0.25,
                           10.0 + 3.0 * torch.rand(rows, ends, generator=g, device=DEV), x[:, at])
    half = room // 2
    length = half + (torch.rand(prompts, generator=g, device=DEV) * (room - half - 1)).long()
    prompt = (length * torch.rand(prompts, generator=g, device=DEV)).long()
    pos = torch.arange(room, device=DEV)
    tokens = (torch.rand(prompts, beams, room, generator=g, device=DEV) * vocab).long().clamp_(max=vocab - 1)
    tokens = torch.where(pos < length[:, None, None], tokens, 0)
    # hypotheses found so far, in the first few places, each shorter than the texts now
    found = (torch.rand(prompts, generator=g, device=DEV) * (beams + 1)).long()
    has = torch.arange(beams, device=DEV) < found[:, None]
    flen = prompt[:, None] + 1 + (torch.rand(prompts, beams, generator=g, device=DEV)
                                  * (length - prompt)[:, None]).long()
    flen = torch.where(has, flen, 0)
    ftok = (torch.rand(prompts, beams, room, generator=g, device=DEV) * vocab).long().clamp_(max=vocab - 1)
    fscore = -42.0 + 2.0 * torch.randn(prompts, beams, generator=g, device=DEV)
    span = (flen - prompt[:, None]).clamp(min=1).float()
    state = {
        "tokens": tokens, "lengths": length[:, None].expand(prompts, beams).reshape(-1).to(torch.int32).contiguous(),
        "prompt_lengths": prompt.to(torch.int32), "scores": scores,
        "finished_tokens": torch.where(pos < flen[..., None], ftok, 0), "finished_lengths": flen.to(torch.int32),
        "finished_scores": torch.where(has, fscore / span ** case["penalty"], -math.inf),
        "done": torch.rand(prompts, generator=g, device=DEV) < (0.1 if prompts >= 8 else 0.0),
    }
    st.update(logits=x.to(dt), state=state, next={k: torch.zeros_like(v) for k, v in state.items()},
              ends=[int(t) for t in range(5, 5 + 7 * ends, 7)], penalty=case["penalty"], early=case["early"])
    return st


def _prepare_rows(case, seed, g):
    layers, hidden = MODELS[case["model"]]
    rows, heads = case["rows"], hidden // HEAD
    sd = DTYPES[case["state"]]
    state = torch.empty(layers, rows, heads, HEAD, HEAD, device=DEV, dtype=sd)
    state.normal_(generator=g)
    shift = torch.randn(2 * layers, rows, hidden, generator=g, device=DEV).half()
    v_first = torch.randn(1, rows, hidden, generator=g, device=DEV).half()
    ts = [state, shift[:layers], shift[layers:], v_first]
    if case["kind"] == "expand":
        r = random.Random(seed * 7 + 1)
        out = case["out"]
        if out >= rows:  # each row to its beams, in order
            src = [i * rows // out for i in range(out)]
        else:
            src = sorted(r.sample(range(rows), out))
        return {"kind": "expand", "tensors": ts, "index": torch.tensor(src, device=DEV)}
    # the rows' texts, and the phase that a half-precision state carries, follow the beams
    ts.append((torch.rand(1, rows, 501, generator=g, device=DEV) * VOCAB).long())
    if case["state"] == "fp16":
        ts.append((torch.rand(1, rows, 1, generator=g, device=DEV) * 4096).to(torch.int32))
    src, dst = _moves(case)
    names = list(range(rows))  # which row is which, another way each seed
    r = random.Random(seed * 7 + 3)
    for at in range(0, rows, case["group"]):
        part = names[at:at + case["group"]]
        r.shuffle(part)
        names[at:at + case["group"]] = part
    src, dst = [s if s < 0 else names[s] for s in src], [names[d] for d in dst]
    if case["pattern"] == "beams":
        by = dict(zip(dst, src))
        return {"kind": "move", "tensors": ts, "sources": torch.tensor([by[i] for i in range(rows)], device=DEV),
                "destinations": None}
    return {"kind": "move", "tensors": ts, "sources": src, "destinations": dst}


def _moves(case):
    """(sources, destinations) of a move; -1: a fresh row."""
    rows, group, moved = case["rows"], case["group"], case["moved"]
    if case["pattern"] == "fork":
        return [0] * moved, list(range(1, 1 + moved))
    if case["pattern"] == "compact":  # the holes below, the slots above them; half as many made fresh
        fresh = min(moved // 2 + 1, rows - 2 * moved)
        return list(range(rows - moved, rows)) + [-1] * fresh, list(range(moved + fresh))
    r = random.Random(1000 * rows + 10 * group + moved)
    src = []
    for at in range(0, rows, group):
        keep = max(1, group - moved)
        part = [r.randrange(min(group, keep + 1)) for _ in range(moved)] + list(range(moved, group))
        src += [at + p for p in part]
    return src, list(range(rows))


# ------------------------------------------------------------------ the pass
def run(state):
    return {"select": _run_select, "step": _run_step, "expand": _run_expand, "move": _run_move}[state["kind"]](state)


def _run_select(st):
    if own:
        return list(_own().beam_select(st["logits"], st["scores"], st["candidates"]))
    value, token, row = _best(st["logits"], st["scores"], st["candidates"])
    return [value.float(), token, row]


def _run_step(st):
    if own:
        mi = _own()
        nxt, rows, new = mi.beam_step(st["logits"], mi.BeamState(**st["state"]), eos_token_id=st["ends"],
                                      length_penalty=st["penalty"], early_stopping=st["early"],
                                      out=mi.BeamState(**st["next"]))
        return {"next": nxt, "rows": rows, "tokens": new.tokens, "lengths": new.lengths, "scores": new.scores,
                "finished_tokens": new.finished_tokens, "finished_lengths": new.finished_lengths,
                "finished_scores": new.finished_scores, "done": new.done}
    return _plain_step(st)


def _run_expand(st):
    if own:
        return list(_own().select_rows(st["tensors"], st["index"], dim=1))
    return [t.index_select(1, st["index"]) for t in st["tensors"]]


def _run_move(st):
    src, dst, ts = st["sources"], st["destinations"], st["tensors"]
    if own:
        _own().move_rows_(ts, src, dst, dim=1)
        return ts
    if dst is None:
        return [t.copy_(t.index_select(1, src)) for t in ts]
    s, d = torch.tensor(src, device=DEV), torch.tensor(dst, device=DEV)
    none = s < 0
    return [t.index_copy_(1, d, torch.where(none.view(-1, *[1] * (t.dim() - 2)), 0,
                                            t.index_select(1, s.clamp(min=0)))) for t in ts]


# ------------------------------------------------------------------ beam search in plain torch
def _best(logits, scores, m):
    """The ``m`` best of each prompt's beams x vocabulary: 64-bit values, tokens, rows.
    Equal values: the lower (beam, token) first."""
    prompts, beams = scores.shape
    n = logits.shape[1]
    # (which of two close candidates comes first hangs on the last bits: 64 of them)
    x = logits.double()
    top = x.amax(1, keepdim=True)
    lse = top + (x - top).exp().sum(1, keepdim=True).log()
    y = (scores.double().view(-1, 1) + (x - lse)).view(prompts, beams * n)
    # what cannot be chosen comes last, by its index (an empty row's NaN too)
    index = torch.arange(beams * n, device=y.device, dtype=torch.float64)
    key = torch.where(y > -math.inf, y, -1e15 - index)
    # a few more than wanted, so that equal values at the border are all there to be put in order
    some = key.topk(min(2 * m + 64, beams * n), dim=1, sorted=False).indices.sort(1).values
    order = key.gather(1, some).sort(dim=1, descending=True, stable=True).indices[:, :m]
    at = some.gather(1, order)
    value = key.gather(1, at)
    value = torch.where(value < -1e14, -math.inf, value)
    return value, at % n, torch.arange(prompts, device=y.device)[:, None] * beams + at // n


def _plain_step(st):
    s, lp = st["state"], st["penalty"]
    prompts, beams = s["scores"].shape
    room, dev = s["tokens"].shape[2], s["scores"].device
    count = (1 + len(st["ends"])) * beams
    value, token, row = _best(st["logits"], s["scores"], count)
    value, beam = value.float(), row % beams
    first = torch.arange(prompts, device=dev)[:, None]
    length = s["lengths"].long().view(prompts, beams)[:, :1]
    gen = (length + 1 - s["prompt_lengths"].long()[:, None]).double()
    end = torch.isin(token, torch.tensor(st["ends"], device=dev)) & (value > -math.inf)
    # the hypotheses that end here, among those found before: the best stay, the newcomers
    # take the places of those that go
    hyp = end[:, :beams]
    score = torch.where(hyp, (value[:, :beams].double() / gen ** lp).float(), -math.inf)
    best = torch.cat([s["finished_scores"], score], 1).sort(dim=1, descending=True, stable=True).indices[:, :beams]
    keep = torch.zeros(prompts, 2 * beams, dtype=torch.bool, device=dev).scatter_(1, best, True)
    gone = (~keep[:, :beams]).int().sort(dim=1, descending=True, stable=True).indices   # free places first
    new = keep[:, beams:].int().sort(dim=1, descending=True, stable=True).indices       # newcomers first
    take = torch.arange(beams, device=dev) < keep[:, beams:].sum(1, keepdim=True)
    from_ = torch.full((prompts, beams), -1, device=dev).scatter_(1, gone, torch.where(take, new, -1))
    is_new, who = from_ >= 0, from_.clamp(min=0)
    pos = torch.arange(room, device=dev)
    ended = torch.where(pos == length[..., None], token.gather(1, who)[..., None], s["tokens"][first, beam.gather(1, who)])
    ftok = torch.where(is_new[..., None], ended, s["finished_tokens"])
    flen = torch.where(is_new, (length + 1).int(), s["finished_lengths"])
    fscore = torch.where(is_new, score.gather(1, who), s["finished_scores"])
    # the beams that live on: the first child of a beam keeps its row, the others take the free rows
    live = end.int().sort(dim=1, stable=True).indices[:, :beams]
    par, tok, val = beam.gather(1, live), token.gather(1, live), value.gather(1, live)
    twin = (par[:, :, None] == par[:, None, :]).tril(-1).any(2)
    used = torch.zeros(prompts, beams, dtype=torch.bool, device=dev).scatter_(1, par, True)
    free = used.int().sort(dim=1, stable=True).indices
    dest = torch.where(twin, free.gather(1, (twin.long().cumsum(1) - 1).clamp(min=0)), par)
    put = lambda v: torch.empty_like(v).scatter_(1, dest, v)  # noqa: E731
    par, tok, val = put(par), put(tok), put(val)
    tokens = torch.where(pos == length[..., None], tok[..., None], s["tokens"][first, par])
    worst = fscore.amin(1)
    over = (worst > -math.inf) if st["early"] else ~((val.amax(1).double() / gen[:, 0] ** lp).float() > worst)
    over = over | (length[:, 0] + 1 >= room)
    d = s["done"]
    was = lambda a, b: torch.where(d.view(-1, *[1] * (a.dim() - 1)), a, b)  # noqa: E731
    rows = was(torch.arange(beams, device=dev).expand(prompts, beams), par) + first * beams
    return {"next": was(torch.zeros_like(tok), tok).view(-1), "rows": rows.view(-1), "tokens": was(s["tokens"], tokens),
            "lengths": (s["lengths"].view(prompts, beams) + (~d)[:, None].int()).view(-1),
            "scores": was(s["scores"], val), "finished_tokens": was(s["finished_tokens"], ftok),
            "finished_lengths": was(s["finished_lengths"], flen), "finished_scores": was(s["finished_scores"], fscore),
            "done": d | over}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    if case["kind"] in ("expand", "move"):
        return None  # (moved, not computed)
    st = prepare(case, seed)
    scores = (st["scores"] if case["kind"] == "select" else st["state"]["scores"]).double().cpu().numpy()
    prompts, beams = scores.shape
    n = case["vocab"]
    m = case["candidates"] if case["kind"] == "select" else (1 + case["ends"]) * beams
    found = []
    for b in range(prompts):
        x = st["logits"][b * beams:(b + 1) * beams].double().cpu().numpy()
        top = x.max(1, keepdims=True)
        with np.errstate(invalid="ignore", divide="ignore"):
            y = scores[b][:, None] + x - top - np.log(np.exp(x - top).sum(1, keepdims=True))
        y = np.where(np.isnan(y), -np.inf, y).reshape(-1)
        border = np.partition(y, y.size - m)[y.size - m]
        at = np.flatnonzero(y >= border) if border > -np.inf else np.arange(y.size)
        at = at[np.lexsort((at, -y[at]))[:m]]
        found.append([(y[i], int(i % n), int(i // n)) for i in at])
    if case["kind"] == "select":
        return [torch.tensor([[c[0] for c in f] for f in found], dtype=torch.float64),
                torch.tensor([[c[1] for c in f] for f in found]),
                torch.tensor([[b * beams + c[2] for c in f] for b, f in enumerate(found)])]
    return _exact_step(st, found)


def _exact_step(st, found):
    s = {k: (v.double() if v.is_floating_point() else v).cpu().numpy().copy() for k, v in st["state"].items()}
    prompts, beams, room = s["tokens"].shape
    nxt, rows = np.zeros((prompts, beams), np.int64), np.arange(prompts * beams).reshape(prompts, beams)
    lengths = s["lengths"].reshape(prompts, beams)
    for b in range(prompts):
        if s["done"][b]:
            continue
        old, at = s["tokens"][b].copy(), int(lengths[b, 0])
        span = float(at + 1 - s["prompt_lengths"][b]) ** st["penalty"]
        hyps, live = [(v, i, None) for i, v in enumerate(s["finished_scores"][b])], []
        for rank, (v, t, k) in enumerate(found[b]):
            if t in st["ends"] and v > -np.inf:
                if rank < beams:
                    hyps.append((v / span, rank, (t, k)))
            elif len(live) < beams:
                live.append((v, t, k))
        best = sorted(hyps, key=lambda h: -h[0])[:beams]
        stay = {h[1] for h in best if h[2] is None}
        places = [i for i in range(beams) if i not in stay]
        for place, (v, _, (t, k)) in zip(places, sorted((h for h in best if h[2]), key=lambda h: h[1])):
            s["finished_scores"][b, place], s["finished_lengths"][b, place] = v, at + 1
            s["finished_tokens"][b, place] = old[k]
            s["finished_tokens"][b, place, at] = t
        spare = [i for i in range(beams) if i not in {k for _, _, k in live}]
        seen = set()
        for v, t, k in live:
            i = k if k not in seen else spare.pop(0)
            seen.add(k)
            nxt[b, i], rows[b, i], s["scores"][b, i] = t, b * beams + k, v
            s["tokens"][b, i] = old[k]
            s["tokens"][b, i, at] = t
        lengths[b] += 1
        worst = s["finished_scores"][b].min()
        s["done"][b] = (worst > -np.inf if st["early"] else not live[0][0] / span > worst) or at + 1 >= room
    out = {"next": nxt.reshape(-1), "rows": rows.reshape(-1), "tokens": s["tokens"], "lengths": lengths.reshape(-1),
           "scores": s["scores"], "finished_tokens": s["finished_tokens"], "finished_lengths": s["finished_lengths"],
           "finished_scores": s["finished_scores"], "done": s["done"]}
    return {k: torch.from_numpy(v) for k, v in out.items()}


# ------------------------------------------------------------------ the least work
def work(case):
    if case["kind"] in ("select", "step"):
        prompts, beams, n = case["prompts"], case["beams"], case["vocab"]
        es = 4 if case["dtype"] == "fp32" else 2
        b = prompts * beams * (n * es + 4)
        if case["kind"] == "select":
            b += prompts * case["candidates"] * (4 + 8 + 8)
        else:  # texts (three quarters of their room on the average) and as many hypotheses, read and written
            b += prompts * beams * (2 * 2 * 8 * 0.75 * case["room"] + 2 * (4 + 4 + 4 + 4) + 16)
        return {"bytes": b, "flops": 4 * prompts * beams * n}
    row = _row_bytes(case["model"], case["state"])
    if case["kind"] == "expand":
        return {"bytes": row * (min(case["rows"], case["out"]) + case["out"]), "flops": 0}
    row += 8 * 501 + (4 if case["state"] == "fp16" else 0)
    pairs = [(s, d) for s, d in zip(*_moves(case)) if s != d]
    return {"bytes": row * (len({s for s, _ in pairs if s >= 0}) + len(pairs)), "flops": 0}

"""Beam search's step written out in 64-bit numpy: the selection, the ends, the places of the beams."""
from __future__ import annotations

import numpy as np


def values(x, scores, normalized=False):
    """``x [prompts, beams, n]``, ``scores [prompts, beams]`` (any floats) -> the 64-bit value of each
    continuation: NaN throughout a row that holds NaN or +inf or has such a score, -inf where the
    logit, the whole row or the score is."""
    x, scores = x.astype(np.float64), scores.astype(np.float64)
    out = np.empty_like(x)
    for i in np.ndindex(scores.shape):
        row, s = x[i], scores[i]
        if not (row < np.inf).all() or not s < np.inf:
            out[i] = np.nan
        elif s == -np.inf or (row == -np.inf).all():
            out[i] = -np.inf
        else:
            top = row.max()
            lse = 0.0 if normalized else top + np.log(np.exp(row - top).sum())
            out[i] = s + (row - lse)
    return out


def select(v, m):
    """The ``m`` best of each prompt: ``(values, tokens, beams)``; NaN first, equal ones by index."""
    p, k, n = v.shape
    flat = v.reshape(p, k * n)
    key = np.where(np.isnan(flat), np.inf, flat)
    order = np.argsort(-key, axis=1, kind="stable")[:, :m]
    return np.take_along_axis(flat, order, 1), order % n, order // n


def step(found, state, ends, penalty, early, pad=0):
    """``found`` (values as the kernel rounds them, tokens, beams, by prompt) applied to ``state`` (a dict of
    numpy arrays, left as it is): ``(next, rows, new state)``."""
    s = {k: v.copy() for k, v in state.items()}
    p, k, room = s["tokens"].shape
    nxt = np.full((p, k), pad, np.int64)
    rows = np.arange(p * k).reshape(p, k)
    length = s["lengths"].reshape(p, k)
    for b in range(p):
        at = int(length[b, 0])
        if s["done"][b] or at >= room:
            s["done"][b] = True
            continue
        val, tok, beam = (f[b] for f in found)
        texts = s["tokens"][b].copy()
        gen = max(at + 1 - int(s["prompt_lengths"][b]), 1)
        pool = [(float(v), 0, i) for i, v in enumerate(s["finished_scores"][b])]
        live = []
        for r in range(len(val)):
            end = tok[r] in ends and val[r] > -np.inf
            if r < k and (end or (at + 1 >= room and val[r] > -np.inf)):
                h = float(np.float32(np.float64(val[r]) / np.float64(gen) ** penalty))
                if h > -np.inf:
                    pool.append((h, 1, r))
            if not end and len(live) < k:
                live.append(r)
        best = sorted(pool, key=lambda e: (-e[0], e[1], e[2]))[:k]
        stay = {i for _, new, i in best if not new}
        free = [i for i in range(k) if i not in stay]
        for slot, (h, _, r) in zip(free, sorted((e for e in best if e[1]), key=lambda e: e[2])):
            s["finished_scores"][b, slot], s["finished_lengths"][b, slot] = h, at + 1
            s["finished_tokens"][b, slot, :at] = texts[beam[r], :at]
            s["finished_tokens"][b, slot, at] = tok[r]
        parents = [int(beam[r]) for r in live]
        spare = [i for i in range(k) if i not in parents]
        seen = set()
        for r, parent in zip(live, parents):
            i = spare.pop(0) if parent in seen else parent
            seen.add(parent)
            nxt[b, i], rows[b, i], s["scores"][b, i] = tok[r], b * k + parent, val[r]
            s["tokens"][b, i, :at] = texts[parent, :at]
            s["tokens"][b, i, at] = tok[r]
        length[b] += 1
        worst = s["finished_scores"][b].min()
        ahead = max(room - int(s["prompt_lengths"][b]), 1) if early == "never" and penalty > 0 else gen
        can = np.float32(np.float64(val[live[0]]) / np.float64(ahead) ** penalty)
        s["done"][b] = (worst > -np.inf if early is True else not can > worst) or at + 1 >= room
    s["lengths"] = length.reshape(-1)
    return nxt.reshape(-1), rows.reshape(-1), s

"""Beam search on the device: the selection over beams and vocabulary
(``rwkv7mi_beam_select``) and the whole step with its bookkeeping
(``rwkv7mi_beam_step``).  The cache rows that follow the beams are moved by
:func:`~.state_rows.move_rows_` (``NativeRWKV7Cache.reorder_cache``), the whole
search is ``NativeRWKV7ForCausalLM.generate_beam``."""
from __future__ import annotations

import bisect
import ctypes
import functools
import math

import torch

from . import _lib

MAX_CANDIDATES = 128
MAX_ENDS = 8


@functools.lru_cache(maxsize=4096)
def _workspace(rows: int, n: int, candidates: int) -> int:
    return int(_lib.load().rwkv7mi_beam_workspace_bytes(rows, n, candidates))


def beam_workspace_bytes(rows: int, n: int, candidates: int) -> int:
    """Workspace bytes of :func:`beam_select` and :func:`beam_step` for ``rows`` rows of
    ``n`` logits and ``candidates`` candidates a prompt."""
    return _workspace(int(rows), int(n), int(candidates))


def _logits(logits: torch.Tensor, prompts: int, beams: int, name: str) -> torch.Tensor:
    if logits.dim() == 3 and logits.shape[0] == prompts and logits.shape[1] == beams:
        logits = logits.reshape(prompts * beams, logits.shape[2])
    if logits.dim() != 2 or logits.shape[0] != prompts * beams or logits.shape[1] == 0:
        raise ValueError(f"{name}: logits must be [prompts * beams, n] or [prompts, beams, n]")
    if logits.shape[1] > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    return logits


def _scratch(workspace, need, like, name):
    if workspace is None:
        return like.new_empty(need, dtype=torch.uint8)
    if (not workspace.is_contiguous() or workspace.numel() * workspace.element_size() < need
            or workspace.data_ptr() % 8):
        raise ValueError(f"{name}: workspace must be contiguous, 8-byte aligned, of at least beam_workspace_bytes bytes")
    return workspace


def _rows_range(t: torch.Tensor):
    """The addresses of a matrix whose rows are any distance apart."""
    at, (rows, n) = t.data_ptr(), t.shape
    return at, at + (((rows - 1) * t.stride(0) + (n - 1) * t.stride(1) + 1) * t.element_size() if rows and n else 0)


def _clear(name: str, written, sizes, read, states=()) -> None:
    """Refuses tensors of ``written`` (None: not given; dense, of which ``sizes`` bytes count) that meet another one,
    a range of ``read``, or one of the states' (sorted, apart from each other)."""
    taken = list(read)
    for t, size in zip(written, sizes):
        if t is None or not size:
            continue
        a = t.data_ptr()
        b = a + size
        for c, d in taken:
            if c < b and a < d:
                break
        else:
            for ends in states:
                k = bisect.bisect_left(ends, (b,))
                if k and ends[k - 1][1] > a:
                    break
            else:
                taken.append((a, b))
                continue
        raise ValueError(f"{name}: outputs or workspace overlap each other or what is read")


def beam_select(logits: torch.Tensor, scores: torch.Tensor, candidates: int | None = None, *, normalized: bool = False,
                out=None, workspace: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``candidates`` (default twice the beams; 128, and the continuations there are, at most)
    best continuations of each prompt: ``logits [prompts * beams, n]`` (fp16, bf16 or fp32; or
    ``[prompts, beams, n]``; at most 65535 rows), ``scores [prompts, beams]`` (fp32) the beams'
    running sums of log-probabilities.

    Returns ``(scores fp32, tokens int64, rows int64)``, each ``[prompts, candidates]``, best
    first, equal ones by beam, then logit, then token; ``rows`` are rows of ``logits``.  A continuation's
    score is ``scores + (logit - logsumexp(row))`` in 64 bits (the exponentials and their sums over
    parts of a row in 32), rounded once (``normalized``: the logits are log-probabilities as they are).  A row that holds NaN
    or +inf, or whose score is one, counts as NaN throughout, which ranks first; a logit of
    -inf, a row of nothing else and a score of -inf (a beam that has not begun) give -inf, in
    the order of their indices.  No host synchronisation; capturable.  ``out``: three tensors
    to write; ``workspace`` (:func:`beam_workspace_bytes`) is allocated when not given.  They share no
    memory with each other, the logits or the scores.
    """
    name = "beam_select"
    if scores.dim() != 2 or scores.dtype is not torch.float32:
        raise ValueError(f"{name}: scores must be fp32 [prompts, beams]")
    prompts, beams = scores.shape
    logits = _logits(logits, prompts, beams, name)
    dt = _lib.dtype_code(logits)
    m = 2 * beams if candidates is None else int(candidates)
    if m < 1:
        raise ValueError(f"{name}: candidates must be positive")
    _lib.require_same_device(logits, scores, *(out or ()), workspace, name=name)
    given = out is not None
    if out is None:
        out = (scores.new_empty((prompts, m)), scores.new_empty((prompts, m), dtype=torch.int64),
               scores.new_empty((prompts, m), dtype=torch.int64))
    else:
        out = tuple(out)
        if len(out) != 3:
            raise ValueError(f"{name}: out must be three tensors")
        for t, want in zip(out, (torch.float32, torch.int64, torch.int64)):
            if tuple(t.shape) != (prompts, m) or t.dtype is not want or not t.is_contiguous():
                raise ValueError(f"{name}: out must be contiguous fp32, int64, int64 [prompts, candidates]")
    rows, n = logits.shape
    need = _workspace(rows, n, m)
    if given or workspace is not None:
        size = 8 * prompts * m
        _clear(name, (*out, workspace) if given else (None, None, None, workspace), (size // 2, size, size, need),
               (_rows_range(logits), _rows_range(scores)))
    workspace = _scratch(workspace, need, logits, name)
    scores = scores.contiguous()  # (a copy lives until the launch)
    with _lib.on_device(logits):
        _lib.call("rwkv7mi_beam_select", logits.data_ptr(), prompts, beams, n, logits.stride(0), dt,
                  scores.data_ptr(), 1 if normalized else 0, m, out[0].data_ptr(), out[1].data_ptr(),
                  out[2].data_ptr(), workspace.data_ptr(), need, _lib.stream_of(logits))
    return out


_Pointers = ctypes.c_void_p * 8


def _meet(ranges) -> bool:
    """Whether two of the sorted address ranges meet."""
    last = 0
    for start, end in ranges:
        if start < last:
            return True
        last = end
    return False


class BeamState:
    """The state of a beam search over ``prompts`` prompts with ``beams`` beams each, on one
    GPU: contiguous tensors, checked once and not replaced afterwards (a step refuses a state
    whose tensors were given other memory).

    ``tokens`` int64 ``[prompts, beams, room]`` (room at most 2^30) and ``lengths`` int32 ``[prompts * beams]``
    (the beams of a prompt are equally long): the texts, prompt included (also a history
    that :func:`~.sampling.process_logits` takes); ``scores`` fp32 ``[prompts, beams]`` their
    log-probabilities; ``prompt_lengths`` int32 ``[prompts]``; ``finished_tokens``,
    ``finished_lengths`` (int32) and ``finished_scores`` (fp32, -inf: none) the same of the
    hypotheses that have ended, in no order; ``done`` bool ``[prompts]``."""

    __slots__ = ("tokens", "lengths", "scores", "prompt_lengths", "finished_tokens", "finished_lengths",
                 "finished_scores", "done", "_pointers", "_addresses", "_shape", "_ends")

    def __init__(self, *, tokens, lengths, scores, prompt_lengths, finished_tokens, finished_lengths, finished_scores,
                 done):
        name = "BeamState"
        if tokens.dim() != 3:
            raise ValueError(f"{name}: tokens must be [prompts, beams, room]")
        p, k, _ = shape = tuple(tokens.shape)
        given = (("tokens", tokens, torch.int64, shape), ("lengths", lengths, torch.int32, (p * k,)),
                 ("scores", scores, torch.float32, (p, k)), ("prompt_lengths", prompt_lengths, torch.int32, (p,)),
                 ("finished_tokens", finished_tokens, torch.int64, shape),
                 ("finished_lengths", finished_lengths, torch.int32, (p, k)),
                 ("finished_scores", finished_scores, torch.float32, (p, k)), ("done", done, torch.bool, (p,)))
        put, where = object.__setattr__, tokens.get_device()
        ends, at = [], []
        for key, t, dtype, want in given:
            if t.dtype is not dtype or t.shape != want or not t.is_contiguous() or t.get_device() != where:
                raise ValueError(f"{name}: {key} must be a contiguous {dtype} tensor {list(want)} on {tokens.device}")
            put(self, key, t)
            p = t.data_ptr()
            at.append(p)
            ends.append((p, p + t.nbytes))
        ends.sort()
        if _meet(ends):
            raise ValueError(f"{name}: tensors overlap")
        put(self, "_pointers", _Pointers(*at))
        put(self, "_addresses", tuple(at))
        put(self, "_shape", shape)
        put(self, "_ends", ends)

    def _check(self, name: str) -> None:
        """The tensors lie where they did when they were checked (``resize_``, ``set_`` and ``.data`` move
        them), with the room that they had."""
        at = (self.tokens.data_ptr(), self.lengths.data_ptr(), self.scores.data_ptr(), self.prompt_lengths.data_ptr(),
              self.finished_tokens.data_ptr(), self.finished_lengths.data_ptr(), self.finished_scores.data_ptr(),
              self.done.data_ptr())
        if at != self._addresses or self.tokens.shape != self._shape:
            raise ValueError(f"{name}: a tensor of the BeamState was given other memory or another shape")

    def __setattr__(self, key, value):
        raise AttributeError(f"BeamState.{key} is not replaced (write into the tensor)")

    def __reduce__(self):
        """Copied and pickled by its tensors: a copy of other tensors has addresses of its own."""
        return _rebuilt, tuple(getattr(self, key) for key in self.__slots__[:8])

    @classmethod
    def start(cls, input_ids: torch.Tensor, beams: int, room: int, *, lengths=None) -> "BeamState":
        """The state behind the prompts ``input_ids [prompts, T]`` (the first ``lengths``
        tokens of each, default all; read on the host), with one live beam each and rows of ``room``
        tokens."""
        if input_ids.dim() != 2 or input_ids.shape[1] > room or beams < 1:
            raise ValueError("BeamState.start: input_ids must be [prompts, T] with T <= room, beams positive")
        dev, (p, t) = input_ids.device, input_ids.shape
        tokens = torch.zeros(p, beams, room, dtype=torch.int64, device=dev)
        tokens[:, :, :t] = input_ids[:, None]
        if lengths is None:
            n = torch.full((p,), t, dtype=torch.int32, device=dev)
        else:
            held = torch.as_tensor(lengths).tolist()
            if not isinstance(held, list) or len(held) != p or not all(isinstance(v, int) and 0 <= v <= t for v in held):
                raise ValueError(f"BeamState.start: lengths must be {p} numbers of 0..{t}")
            n = torch.tensor(held, dtype=torch.int32, device=dev)
        scores = torch.full((p, beams), -math.inf, device=dev)
        scores[:, 0] = 0.0
        return cls(tokens=tokens, lengths=n.repeat_interleave(beams), scores=scores,
                   prompt_lengths=n, finished_tokens=torch.zeros_like(tokens),
                   finished_lengths=torch.zeros(p, beams, dtype=torch.int32, device=dev),
                   finished_scores=torch.full((p, beams), -math.inf, device=dev),
                   done=torch.zeros(p, dtype=torch.bool, device=dev))

    def best(self, count: int = 1, *, length_penalty: float = 1.0):
        """``(tokens [prompts, count, room], lengths, scores)`` of each prompt's ``count`` best
        texts, best first: the hypotheses, then, of a search that is not over (or ended without a
        hypothesis) and has fewer, the running beams, by score / generated length ** length_penalty.
        Where there are not as many texts, the rest are the prompt alone, with the score -inf."""
        p, k, room = self.tokens.shape
        if not 1 <= count <= k:
            raise ValueError(f"BeamState.best: count must be 1..{k}")
        length = self.lengths.view(p, k)
        span = (length - self.prompt_lengths[:, None]).clamp(min=1).double()
        running = (self.scores.double() / span ** float(length_penalty)).float()
        ended = self.finished_scores > -math.inf
        # (what still ran when the last step filled the rows is among the hypotheses)
        open_ = ~(self.done & ended.any(1))[:, None] & (self.scores != -math.inf)
        kind = torch.cat([ended.int() * 2, open_.int()], 1)  # 2: a hypothesis, 1: a running text, 0: none
        score = torch.cat([self.finished_scores, running], 1)
        order = score.sort(dim=1, descending=True, stable=True).indices
        order = order.gather(1, kind.gather(1, order).sort(dim=1, descending=True, stable=True).indices)[:, :count]
        none = kind.gather(1, order) == 0
        order = order.masked_fill(none, k)  # (every running text begins with the prompt)
        tokens = torch.cat([self.finished_tokens, self.tokens], 1).gather(1, order[..., None].expand(p, count, room))
        lengths = torch.cat([self.finished_lengths, length], 1).gather(1, order)
        lengths = torch.where(none, self.prompt_lengths[:, None], lengths)
        tokens = tokens.masked_fill(none[..., None] & (torch.arange(room, device=tokens.device) >= lengths[..., None]), 0)
        return tokens, lengths, score.gather(1, order).masked_fill(none, -math.inf)


def _rebuilt(*tensors) -> BeamState:
    return BeamState(**dict(zip(BeamState.__slots__, tensors)))


def end_tokens(eos_token_id) -> list[int]:
    """The end tokens that ``eos_token_id`` names: none, one, or several (a sequence or a
    tensor)."""
    if eos_token_id is None:
        return []
    if isinstance(eos_token_id, torch.Tensor):
        eos_token_id = eos_token_id.reshape(-1).tolist()
    return [int(t) for t in eos_token_id] if isinstance(eos_token_id, (list, tuple)) else [int(eos_token_id)]


def beam_step(logits: torch.Tensor, state: BeamState, *, eos_token_id=None, length_penalty: float = 1.0,
              early_stopping=False, pad_token_id: int = 0, normalized: bool = False, out: BeamState | None = None,
              next_tokens: torch.Tensor | None = None, rows: torch.Tensor | None = None,
              workspace: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, BeamState]:
    """One step of a beam search: ``logits [prompts * beams, n]`` of the last tokens of
    ``state``'s texts; returns ``(next_tokens, rows, state)``: int64 ``[prompts * beams]``,
    each row's token and the row that it continues (for ``reorder_cache``), and the new state:
    ``state`` itself, or ``out``, another one of the same sizes (then ``state`` stays as it
    is; of the rows in ``out`` only their texts are written).

    Per prompt that is not done, :func:`beam_select` over ``(1 + ends) * beams`` candidates
    (at most 128), then:

    * an end token (``eos_token_id``: none, one or up to 8) among the first ``beams``, and each of
      these where the rows become full, makes a hypothesis of score
      ``score / generated_tokens ** length_penalty``, its last token included; the ``beams`` best of these and the earlier ones stay, the earlier first where
      equal; newcomers take the places of those that go;
    * the first ``beams`` others live on.  A beam's best child stays in its row, the rest take
      the rows without a child, in order: ``rows`` names as few moved rows as there can be;
    * the prompt is done when its rows are full, or, ``early_stopping`` False: no running beam at
      its present length, ``"never"``: at the length that helps it most, beats the worst of
      ``beams`` hypotheses; True: there are ``beams`` hypotheses.

    A done prompt keeps its state; its next tokens are ``pad_token_id`` (one that the
    model takes, where they are fed to it), its rows their own. No host synchronisation; capturable.  ``next_tokens``, ``rows`` and ``workspace``
    (:func:`beam_workspace_bytes`) are allocated when not given; they share no memory with each
    other, the logits or a state.
    """
    name = "beam_step"
    prompts, beams, room = state._shape
    logits = _logits(logits, prompts, beams, name)
    dt = _lib.dtype_code(logits)
    ends = end_tokens(eos_token_id)
    m = (1 + len(ends)) * beams
    if len(ends) > MAX_ENDS or m > MAX_CANDIDATES:
        raise ValueError(f"{name}: at most {MAX_ENDS} end tokens and {MAX_CANDIDATES} candidates, "
                         f"(1 + ends) * beams; got {len(ends)} and {m}")
    how = {False: 0, True: 1, "never": 2}.get(early_stopping)
    if how is None:
        raise ValueError(f"{name}: early_stopping is False, True or 'never'")
    lp = float(length_penalty)
    if not math.isfinite(lp):
        raise ValueError(f"{name}: length_penalty = {lp}")
    to = state if out is None else out
    _lib.require_same_device(logits, state.tokens, to.tokens, next_tokens, rows, workspace, name=name)
    state._check(name)
    if to is not state:
        to._check(name)
        if to._shape != state._shape:
            raise ValueError(f"{name}: out has {list(to._shape)} tokens, state {list(state._shape)}")
        if _meet(sorted(state._ends + to._ends)):
            raise ValueError(f"{name}: out shares memory with state")
    total = prompts * beams
    for t in (next_tokens, rows):
        if t is not None and (t.dtype is not torch.int64 or t.numel() != total or not t.is_contiguous()):
            raise ValueError(f"{name}: next_tokens and rows must be contiguous int64 tensors of one entry per row")
    n = logits.shape[1]
    need = _workspace(total, n, m)
    if next_tokens is not None or rows is not None or workspace is not None:
        _clear(name, (next_tokens, rows, workspace), (8 * total, 8 * total, need), (_rows_range(logits),),
               (state._ends,) if to is state else (state._ends, to._ends))
    if next_tokens is None:
        next_tokens = state.tokens.new_empty(total)
    if rows is None:
        rows = state.tokens.new_empty(total)
    workspace = _scratch(workspace, need, logits, name)
    with _lib.on_device(logits):
        _lib.call("rwkv7mi_beam_step", logits.data_ptr(), prompts, beams, n, logits.stride(0), dt, 1 if normalized else 0,
                  (ctypes.c_int64 * len(ends))(*ends) if ends else None, len(ends), lp, how, int(pad_token_id),
                  state._pointers, to._pointers, room, next_tokens.data_ptr(), rows.data_ptr(), workspace.data_ptr(),
                  need, _lib.stream_of(logits))
    return next_tokens, rows, to


__all__ = ["BeamState", "beam_select", "beam_step", "beam_workspace_bytes"]

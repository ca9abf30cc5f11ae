"""Greedy token selection on the GPU (``rwkv7mi_argmax_rows``): the argmax of
each logits row as the reference's greedy loop takes it with torch
(bench/bench_native_quant_e2e_decode.py:424-437), so a captured decode graph
can end with its next tokens; and the logits step before it
(``rwkv7mi_process_logits``): penalties for repeated tokens, a bias and a grammar
mask, with the greedy token of what they leave."""
from __future__ import annotations

import functools
import math

import torch

from . import _lib


def argmax_workspace_bytes(rows: int, n: int, dtype: torch.dtype) -> int:
    """Workspace bytes of the many-workgroup argmax of ``rows`` rows of ``n``."""
    return int(_lib.load().rwkv7mi_argmax_workspace_bytes(int(rows), int(n), _lib._DTYPE_CODE[dtype]))


def argmax_rows(logits: torch.Tensor, *, out: torch.Tensor | None = None,
                out2: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``logits [rows, n]`` -> ``int64 [rows]``: the first index of each row's
    maximum (NaN counts as the maximum), written to ``out`` (and ``out2``)
    when given.  No host synchronisation; capturable.  Rows are split over
    many workgroups (two launches); ``workspace`` (a contiguous tensor of at
    least :func:`argmax_workspace_bytes` bytes) is allocated when not given."""
    if logits.dim() != 2:
        raise ValueError("argmax_rows: logits must be [rows, n]")
    _lib.require_gpu(logits, out, out2, name="argmax_rows")
    rows, n = (int(s) for s in logits.shape)
    if logits.stride(1) != 1 or logits.data_ptr() % 16 or (logits.stride(0) * logits.element_size()) % 16:
        logits = logits.contiguous()
        if logits.data_ptr() % 16 or (n * logits.element_size()) % 16:
            raise ValueError("argmax_rows: rows must be 16-byte aligned")
    for t in (out, out2):
        if t is not None and (t.dtype != torch.int64 or t.numel() != rows or not t.is_contiguous()):
            raise ValueError("argmax_rows: out must be a contiguous int64 tensor of one entry per row")
    if out is None:
        out = torch.empty(rows, device=logits.device, dtype=torch.int64)
    need = argmax_workspace_bytes(rows, n, logits.dtype)
    if workspace is None:
        workspace = torch.empty(need, device=logits.device, dtype=torch.uint8)
    elif (not workspace.is_contiguous() or workspace.numel() * workspace.element_size() < need
          or workspace.data_ptr() % 8):
        raise ValueError("argmax_rows: workspace must be contiguous, 8-byte aligned, "
                         "of at least argmax_workspace_bytes bytes")
    _lib.call("rwkv7mi_argmax_rows_ws", _lib.ptr(logits), rows, n, int(logits.stride(0)), _lib.dtype_code(logits),
              _lib.ptr(out), _lib.ptr(out2), _lib.ptr(workspace), workspace.numel() * workspace.element_size(),
              _lib.stream_of(logits))
    return out


@functools.lru_cache(maxsize=4096)
def _process_workspace(rows: int, n: int) -> int:
    return int(_lib.load().rwkv7mi_process_logits_workspace_bytes(rows, n))


def process_logits_workspace_bytes(rows: int, n: int) -> int:
    """Workspace bytes of :func:`process_logits` with ``next_tokens``."""
    return _process_workspace(int(rows), int(n))


def _row_values(value, rows: int, name: str, lo: float, hi: float, *, open_lo: bool = False):
    """A penalty as ``(device tensor [rows] or None, float)``; numbers are checked
    against ``lo``..``hi`` (``open_lo``: above ``lo``)."""
    if isinstance(value, torch.Tensor):
        if value.dtype is torch.float32 and value.shape == (rows,) and value.is_contiguous():
            return value, 0.0
        if value.numel() not in (1, rows) or value.dim() > 1 or not value.is_floating_point():
            raise ValueError(f"process_logits: {name} must be a number or a floating-point tensor of one value per row")
        return value.to(torch.float32).expand(rows).contiguous(), 0.0
    value = float(value)
    if not math.isfinite(value) or not lo <= value <= hi or (open_lo and value == lo):
        raise ValueError(f"process_logits: {name} = {value} is out of range")
    return None, value


def _shared_rows(t: torch.Tensor, rows: int, width: int, name: str):
    """``t`` ``[width]``, ``[1, width]`` or ``[rows, width]`` with dense rows, and its row
    stride (0: one row for all)."""
    if t.dim() == 1:
        t = t[None]
    if t.dim() != 2 or int(t.shape[0]) not in (1, rows) or int(t.shape[1]) < width:
        raise ValueError(f"process_logits: {name} must hold {width} entries, once or per row")
    if t.stride(1) != 1 and int(t.shape[1]) > 1:
        t = t.contiguous()
    return t, int(t.stride(0)) if int(t.shape[0]) == rows and rows > 1 else 0


def process_logits(logits: torch.Tensor, *, history: torch.Tensor | None = None,
                   lengths: torch.Tensor | None = None, repetition_penalty=1.0, presence_penalty=0.0,
                   frequency_penalty=0.0, penalty_decay=1.0, bias: torch.Tensor | None = None,
                   allowed: torch.Tensor | None = None, out: torch.Tensor | None = None,
                   next_tokens: torch.Tensor | None = None, next_tokens2: torch.Tensor | None = None,
                   append: bool = False, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``logits [rows, n]`` (fp16, bf16 or fp32) after penalties, bias and mask:

    * a token that occurs in its row's history is divided by ``repetition_penalty`` where
      positive, multiplied by it elsewhere, then lowered by ``presence_penalty`` and by
      ``frequency_penalty`` times its occurrences, the one ``k`` tokens before the newest
      counted as ``penalty_decay ** k``;
    * ``bias`` (``[n]`` or ``[rows, n]``) is added;
    * a token whose bit in ``allowed`` is clear becomes ``-inf``, whatever it held
      (int32 words ``[ceil(n / 32)]`` or one row of them each; bit ``t % 32`` of word ``t // 32``).

    ``history [rows, L]`` (at most 2^23 a row, 65535 rows) holds int32 or int64 tokens, of
    which the first ``lengths[row]`` (int32; default all) count; entries outside
    ``0..n-1`` are ignored.
    The penalties are numbers or one value per row (a ``penalty_decay`` tensor is clamped
    to 0..1).  The arithmetic is fp32, rounded once to ``out``'s type: ``logits``' own
    (the default) or fp32.  ``out`` may be ``logits`` itself.

    ``next_tokens`` (int64 ``[rows]``, and a second copy ``next_tokens2``) receives the first
    index of each row's maximum, as :func:`argmax_rows` of the result gives it: 0 where
    nothing is allowed.  ``append`` also writes it behind the row's history and adds one to
    ``lengths`` where ``L`` leaves room.  No host synchronisation; capturable.  ``workspace``
    (:func:`process_logits_workspace_bytes`) is allocated when not given and needed.
    """
    name = "process_logits"
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"{name}: logits must be [rows, n]")
    rows, n = logits.shape
    dt = _lib.dtype_code(logits)
    big = math.inf
    rep, rep_v = _row_values(repetition_penalty, rows, "repetition_penalty", 0.0, big, open_lo=True)
    pres, pres_v = _row_values(presence_penalty, rows, "presence_penalty", -big, big)
    freq, freq_v = _row_values(frequency_penalty, rows, "frequency_penalty", -big, big)
    dec, dec_v = _row_values(penalty_decay, rows, "penalty_decay", 0.0, 1.0)
    _lib.require_same_device(logits, history, lengths, rep, pres, freq, dec, bias, allowed, out, next_tokens, next_tokens2,
                             workspace, name=name)
    if n > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    if out is None:
        out = logits.new_empty((rows, n))
    elif (tuple(out.shape) != (rows, n) or out.dtype not in (logits.dtype, torch.float32)
          or (n > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < n)):
        raise ValueError(f"{name}: out must be [rows, n] with dense rows, of logits' dtype or fp32")
    elif _lib.overlap(out, logits) and not (out.data_ptr() == logits.data_ptr() and out.dtype == logits.dtype
                                            and (rows == 1 or out.stride(0) == logits.stride(0))):
        raise ValueError(f"{name}: out overlaps logits without being them")
    bits, ldh, cap = 64, 0, 0
    if history is not None:
        if history.dim() != 2 or history.shape[0] != rows or history.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{name}: history must be an int32 or int64 [rows, L] tensor")
        cap, bits = history.shape[1], 8 * history.element_size()
        if cap > 1 and history.stride(1) != 1:
            if append:
                raise ValueError(f"{name}: appending needs a history of dense rows")
            history = history.contiguous()
        ldh = history.stride(0)
    if lengths is not None:
        if history is None or lengths.shape != (rows,) or lengths.dtype is not torch.int32:
            raise ValueError(f"{name}: lengths must be int32 [rows], with a history")
        if not lengths.is_contiguous():
            if append:
                raise ValueError(f"{name}: appending needs contiguous lengths")
            lengths = lengths.contiguous()
    if append and (history is None or lengths is None or next_tokens is None):
        raise ValueError(f"{name}: append needs history, lengths and next_tokens")
    ldb = lda = 0
    if bias is not None:
        bias, ldb = _shared_rows(bias.to(torch.float32), rows, n, "bias")
    if allowed is not None:
        if allowed.dtype is not torch.int32:
            raise ValueError(f"{name}: allowed must hold int32 words")
        allowed, lda = _shared_rows(allowed, rows, (n + 31) // 32, "allowed")
    need = 0
    if next_tokens is not None:
        for t in (next_tokens, next_tokens2):
            if t is not None and (t.dtype is not torch.int64 or t.numel() != rows or not t.is_contiguous()):
                raise ValueError(f"{name}: next_tokens must be a contiguous int64 tensor of one entry per row")
        need = _process_workspace(rows, n)
    elif next_tokens2 is not None:
        raise ValueError(f"{name}: next_tokens2 is a second copy of next_tokens")
    if workspace is None:
        workspace = logits.new_empty(need, dtype=torch.uint8) if need else None
    elif (not workspace.is_contiguous() or workspace.numel() * workspace.element_size() < need
          or workspace.data_ptr() % 8):
        raise ValueError(f"{name}: workspace must be contiguous, 8-byte aligned, "
                         "of at least process_logits_workspace_bytes bytes")
    ptr = _lib.ptr
    with _lib.on_device(logits):
        _lib.call("rwkv7mi_process_logits", logits.data_ptr(), rows, n, logits.stride(0), dt, out.data_ptr(),
                  out.stride(0), _lib.dtype_code(out), ptr(history), bits, ldh, cap, ptr(lengths), ptr(rep), rep_v,
                  ptr(pres), pres_v, ptr(freq), freq_v, ptr(dec), dec_v, ptr(bias), ldb, ptr(allowed), lda,
                  ptr(next_tokens), ptr(next_tokens2), 1 if append else 0, ptr(workspace), need, _lib.stream_of(logits))
    return out


class NativeLogitsProcessor:
    """:func:`process_logits` as an entry of ``generate(logits_processor=[...])``: the ids so
    far (the prompt from ``prompt_ignore_length`` on) are the history.  ``allowed`` may be a
    callable that gives the words for ``input_ids``, for a mask that follows the text."""

    def __init__(self, *, repetition_penalty=1.0, presence_penalty=0.0, frequency_penalty=0.0, penalty_decay=1.0,
                 bias: torch.Tensor | None = None, allowed=None, prompt_ignore_length: int = 0):
        if int(prompt_ignore_length) < 0:
            raise ValueError("NativeLogitsProcessor: prompt_ignore_length must not be negative")
        self.how = dict(repetition_penalty=repetition_penalty, presence_penalty=presence_penalty,
                        frequency_penalty=frequency_penalty, penalty_decay=penalty_decay)
        self.bias, self.allowed, self.skip = bias, allowed, int(prompt_ignore_length)

    def __call__(self, input_ids: torch.Tensor, scores: torch.Tensor) -> torch.Tensor:
        allowed = self.allowed(input_ids) if callable(self.allowed) else self.allowed
        return process_logits(scores, history=input_ids[:, self.skip:], allowed=allowed, bias=self.bias, **self.how)


__all__ = ["argmax_rows", "argmax_workspace_bytes", "process_logits", "process_logits_workspace_bytes",
           "NativeLogitsProcessor"]

"""Rows of several tensors moved by one index in one launch
(``rwkv7mi_rows_move``): the batch edits of a recurrent cache (select, reorder,
repeat: rwkv7_hf/model_cache.py:335-343, 368) and the state pool's forks, moves
and fresh slots.  Byte moves, bit-exact, any dtype."""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

MAX_TENSORS = 24  # of a launch
MAX_LISTED = 192  # host indices that travel with the launch
MAX_TRADING = 2048  # rows that may trade places in place


def _family(t: torch.Tensor, dim: int, name: str):
    """``(address, outer stride, row stride, row bytes, outer count, rows, end)`` of ``t`` in
    bytes, the dimensions before ``dim`` as one and those behind it dense; None where they are
    not."""
    es, shape, at = t.element_size(), t.shape, t.data_ptr()
    if len(shape) <= dim:
        raise ValueError(f"{name}: a tensor of {len(shape)} dimensions has no rows along dimension {dim}")
    rows = shape[dim]
    if t.is_contiguous():
        size = math.prod(shape[dim + 1:]) * es
        return at, rows * size, size, size, math.prod(shape[:dim]), rows, at + t.numel() * es
    stride, dense = t.stride(), 1
    for i in range(len(shape) - 1, dim, -1):
        if shape[i] != 1 and stride[i] != dense:
            return None
        dense *= shape[i]
    outer, step = 1, 0
    for i in range(dim - 1, -1, -1):
        if shape[i] == 1:
            continue
        if outer > 1 and stride[i] != outer * step:
            return None
        if outer == 1:
            step = stride[i]
        outer *= shape[i]
    end = at + (1 + sum((k - 1) * s for k, s in zip(shape, stride))) * es if t.numel() else at
    return at, step * es, (stride[dim] if rows > 1 else dense) * es, dense * es, outer, rows, end


def _apart(f) -> bool:
    """Whether the rows of a family lie apart (they are written)."""
    _, step, row, size, outer, rows, _ = f
    if not (size and outer and rows):
        return True
    spans = ((row, rows), (step, outer)) if row <= step else ((step, outer), (row, rows))
    for s, k in spans:
        if k > 1:
            if s < size:
                return False
            size += s * (k - 1)
    return True


def _lap(families) -> bool:
    """Whether the address ranges of any two meet."""
    ends = sorted([(f[0], f[6]) for f in families if f[6] > f[0]])
    return any([b[0] < a[1] for a, b in zip(ends, ends[1:])])


def _within(index, families) -> bool:
    """Whether an index of the GPU lies in memory that is written."""
    if type(index) is list:
        return False
    a = index.data_ptr()
    b = a + 8 * index.numel()
    for f in families:
        if f[0] < b and a < f[6]:
            return True
    return False


def _index(index, name: str):
    """``index`` as a list of ints, or a one-dimensional int64 tensor of the GPU."""
    if isinstance(index, torch.Tensor):
        if index.dim() != 1 or index.is_floating_point() or index.is_complex() or index.dtype is torch.bool:
            raise ValueError(f"{name}: an index is a one-dimensional tensor of integers")
        return index.to(torch.int64).contiguous() if index.is_cuda else index.tolist()
    return [int(i) for i in index]


def _launch(families, src_rows, dst_rows, n, src, dst, disjoint, poison, where):
    """``families``: 8 numbers a tensor, as the library's ``rwkv7mi_rows``."""
    src_at = dst_at = src_list = dst_list = None
    if type(src) is not list:
        src_at = src.data_ptr()
    elif n <= MAX_LISTED:
        src_list = (ctypes.c_int64 * n)(*src)
    else:
        src = torch.tensor(src, dtype=torch.int64).to(where.device)
        src_at = src.data_ptr()
    if dst is not None:
        if n <= MAX_LISTED:
            dst_list = (ctypes.c_int64 * n)(*dst)
        else:
            dst = torch.tensor(dst, dtype=torch.int64).to(where.device)
            dst_at = dst.data_ptr()
    with _lib.on_device(where):
        stream = _lib.stream_of(where)
        for i in range(0, len(families), 8 * MAX_TENSORS):
            part = families[i:i + 8 * MAX_TENSORS]
            _lib.call("rwkv7mi_rows_move", len(part) // 8, (ctypes.c_int64 * len(part))(*part), src_rows, dst_rows, n,
                      src_at, dst_at, src_list, dst_list, (1 if disjoint else 0) + (2 if poison else 0), stream)


def _same_rows(families, name):
    rows = families[0][5]
    for f in families:
        if f[5] != rows:
            raise ValueError(f"{name}: tensors of {sorted({f[5] for f in families})} rows")
    return rows


def _on_gpu(tensors, index, name):
    if not tensors:
        raise ValueError(f"{name}: no tensors")
    _lib.require_same_device(*tensors, *((index,) if isinstance(index, torch.Tensor) else ()), name=name)


def _no_gradient(tensors, name):
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise RuntimeError(f"{name}: no gradient flows through moved rows (a tensor requires grad)")


_changed = torch.autograd.graph.increment_version  # (tells autograd that the tensors are written)


def select_rows(tensors, indices, *, dim: int = 0, out=None, poison: bool = False) -> list[torch.Tensor]:
    """``[t.index_select(dim, indices) for t in tensors]`` in one launch (24 tensors a
    launch): the rows along ``dim`` of tensors that have as many.  No gradient flows through:
    in grad mode tensors that require grad are refused.

    ``indices``: integers (checked) or a one-dimensional integer tensor; -1, and on the
    GPU any index out of range, gives a row of zeros; with ``poison`` one of bytes of 0xff, NaN
    in fp16, bf16 and fp32.  ``out``: tensors to write instead of new ones, whose ranges of
    memory do not meet those of ``tensors``.  At most 4194240 indices.  Capturable where
    ``indices`` are on the GPU or at most 192.
    """
    name = "select_rows"
    tensors = list(tensors)
    idx = _index(indices, name)
    _on_gpu(tensors, idx, name)
    _no_gradient(tensors, name)
    if dim < 0:
        raise ValueError(f"{name}: dim counts from the front")
    n = len(idx) if type(idx) is list else idx.shape[0]
    src = []
    for i, t in enumerate(tensors):
        if t.is_neg() or t.is_conj():  # (its bytes are not its values)
            tensors[i] = t = t.resolve_conj().resolve_neg()
        f = _family(t, dim, name)
        if f is None:
            tensors[i] = t = t.contiguous()
            f = _family(t, dim, name)
        src.append(f)
    rows = _same_rows(src, name)
    if type(idx) is list and not all(-1 <= i < rows for i in idx):
        raise IndexError(f"{name}: indices outside -1..{rows - 1}")
    flat = []
    if out is None:
        out = []
        for t, f in zip(tensors, src):
            shape, size = t.shape, f[3]
            o = t.new_empty((*shape[:dim], n, *shape[dim + 1:]))
            out.append(o)
            flat += (f[0], o.data_ptr(), f[1], f[2], n * size, size, size, f[4])
    else:
        out = list(out)
        if len(out) != len(tensors):
            raise ValueError(f"{name}: {len(out)} outputs for {len(tensors)} tensors")
        for o, t in zip(out, tensors):
            want = (*t.shape[:dim], n, *t.shape[dim + 1:])
            if tuple(o.shape) != want or o.dtype != t.dtype:
                raise ValueError(f"{name}: an output is {tuple(o.shape)} {o.dtype}, not {want} {t.dtype}")
        _on_gpu([tensors[0], *out], None, name)
        _no_gradient(out, name)
        if any(o.is_neg() or o.is_conj() for o in out):
            raise ValueError(f"{name}: an output is a conjugate or negative view")
        dst = [_family(o, dim, name) for o in out]
        if any(f is None or not _apart(f) for f in dst):
            raise ValueError(f"{name}: the rows of an output are dense and apart")
        if _lap(dst) or any(_lap((f, g)) for f in src for g in dst) or _within(idx, dst):
            raise ValueError(f"{name}: outputs overlap")
        for f, g in zip(src, dst):
            flat += (f[0], g[0], f[1], f[2], g[1], g[2], f[3], f[4])
        if n:
            _changed(out)
    if n:
        _launch(flat, rows, n, n, idx, None, True, poison, tensors[0])
    return out


def move_rows_(tensors, sources, destinations=None, *, dim: int = 0, poison: bool = False) -> None:
    """Row ``destinations[i]`` along ``dim`` of every tensor becomes what row
    ``sources[i]`` was before the call, in place and in one launch (24 tensors a launch);
    -1 makes a row of zeros (with ``poison`` of bytes of 0xff, NaN in fp16, bf16 and fp32).
    Rows may trade places, and a source serve many times.

    ``sources``: integers (checked), or a one-dimensional integer tensor of the GPU, whose
    indices out of range do the same.  ``destinations``: distinct integers, known to the
    host; default every row.  Up to 2048 rows may trade places; more where no source is
    another row's destination.  The tensors' rows are dense, and their memory neither
    overlaps nor interleaves.  Capturable where host indices are at most 192.  No gradient flows
    through: in grad mode tensors that require grad are refused, others count as changed.
    """
    name = "move_rows_"
    tensors = list(tensors)
    src = _index(sources, name)
    _on_gpu(tensors, src, name)
    _no_gradient(tensors, name)
    if dim < 0:
        raise ValueError(f"{name}: dim counts from the front")
    fams = [_family(t, dim, name) for t in tensors]
    for f in fams:
        if f is None or not _apart(f):
            raise ValueError(f"{name}: the rows of a tensor are dense and apart")
    rows = _same_rows(fams, name)
    if _within(src, fams):
        src = src.clone()  # (as if it was read first, like the rows)
    if len(fams) > 1 and _lap(fams):
        raise ValueError(f"{name}: tensors overlap or interleave")
    n = len(src) if type(src) is list else src.shape[0]
    if type(src) is list and not all(-1 <= i < rows for i in src):
        raise IndexError(f"{name}: sources outside -1..{rows - 1}")
    dst = None
    if destinations is None:
        if n != rows:
            raise ValueError(f"{name}: {n} sources for {rows} rows")
    else:
        dst = _index(destinations, name)
        if type(dst) is not list:
            raise ValueError(f"{name}: destinations are known to the host")
        if len(dst) != n:
            raise ValueError(f"{name}: {n} sources for {len(dst)} destinations")
        if not all(0 <= i < rows for i in dst):
            raise IndexError(f"{name}: destinations outside 0..{rows - 1}")
        if len(set(dst)) != n:
            raise ValueError(f"{name}: destinations {sorted(dst)} repeat")
    disjoint = type(src) is list and not {s for s, d in zip(src, dst or range(n)) if s != d} & set(dst or range(n))
    if not disjoint and n > MAX_TRADING:
        raise ValueError(f"{name}: at most {MAX_TRADING} rows trade places in one call")
    flat = []
    for f in fams:
        flat += (f[0], f[0], f[1], f[2], f[1], f[2], f[3], f[4])
    if n:
        _changed(tensors)
        _launch(flat, rows, rows, n, src, dst, disjoint, poison, tensors[0])


__all__ = ["select_rows", "move_rows_"]

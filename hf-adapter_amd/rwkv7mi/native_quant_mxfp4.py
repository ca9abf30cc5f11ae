"""Microscaled 4-bit floating point (MXFP4): quantiser, linear and module.

A weight row's blocks of 32 inputs share a power-of-two scale byte and hold a
4-bit e2m1 code each (0.53 bytes a weight).  :func:`mxfp4_linear` runs fp16 or
bf16 rows against such a weight; with ``quantize_input`` it quantises the rows
on the way and multiplies codes by codes on the scaled matrix instructions.
:class:`MXFP4Linear` and :func:`quantize_model_mxfp4` put it in the place of
``nn.Linear`` as :class:`~.native_quant_mm4.MM4Linear` does.  GPU tensors only.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from .native_quant_mm8 import invalidate_model_caches
from .native_quant_policy import normalize_native_mm_policy, should_quantize_linear

BLOCK = 32
EPILOGUES = {"none": _lib.EPI_NONE, "relu2": _lib.EPI_RELU2, "residual": _lib.EPI_RESIDUAL}


def _aligned(t: torch.Tensor, nbytes: int) -> torch.Tensor:
    """``t`` contiguous and starting on an ``nbytes`` boundary."""
    t = t.contiguous()
    return t if t.data_ptr() % nbytes == 0 else t.clone()


def quantize_mxfp4(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``x [..., I]`` (fp16, bf16 or fp32; ``I`` a multiple of 32) to MXFP4:
    ``(codes uint8 [..., I/2], scales uint8 [..., I/32])``, the even input in a
    byte's low nibble.

    A block's scale is ``2^(floor(log2 max|x|) - 2)`` (at least ``2^-127``), its
    codes round to nearest, ties to even, and stop at 6 times the scale.  A block
    that holds an infinity or a NaN gets the scale NaN (byte 255), so that it shows
    in what is computed from it.
    """
    if x.dim() < 1 or int(x.shape[-1]) == 0 or int(x.shape[-1]) % BLOCK:
        raise ValueError("quantize_mxfp4: the last dimension must be a multiple of 32")
    code = _lib.dtype_code(x)
    _lib.require_gpu(x, name="quantize_mxfp4")
    lead, width = x.shape[:-1], x.shape[-1]
    rows = x.numel() // width
    ld = width
    if not x.is_contiguous():
        x = x.reshape(rows, width)
        ld = x.stride(0)
        if x.stride(1) != 1 or ld < width or ld % (16 // x.element_size()):
            x, ld = x.contiguous(), width
    if x.data_ptr() % 16:
        x, ld = x.contiguous().clone(), width
    codes = x.new_empty((*lead, width // 2), dtype=torch.uint8)
    scales = x.new_empty((*lead, width // BLOCK), dtype=torch.uint8)
    with _lib.on_device(x):
        _lib.call("rwkv7mi_mxfp4_quantize", x.data_ptr(), rows, width, ld, code, codes.data_ptr(), scales.data_ptr(),
                  _lib.stream_of(x))
    return codes, scales


def dequantize_mxfp4(codes: torch.Tensor, scales: torch.Tensor,
                     out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """The values ``[..., I]`` of :func:`quantize_mxfp4`'s result, rounded to
    ``out_dtype`` (bf16 and fp32 hold each exactly below 2^128; past it they become
    infinite, which the scales 2^126 and 2^127 reach).  Products do not form them so."""
    _check_packed(codes, scales, "dequantize_mxfp4")
    _lib.require_same_device(codes, scales, name="dequantize_mxfp4")
    codes, scales = _aligned(codes, 4), scales.contiguous()
    width = 2 * codes.shape[-1]
    out = codes.new_empty((*codes.shape[:-1], width), dtype=out_dtype)
    with _lib.on_device(codes):
        _lib.call("rwkv7mi_mxfp4_dequantize", codes.data_ptr(), scales.data_ptr(), out.numel() // width, width,
                  out.data_ptr(), _lib.dtype_code(out), _lib.stream_of(codes))
    return out


def _check_packed(codes, scales, who):
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise ValueError(f"{who}: codes and scales are uint8")
    cs, ss = codes.shape, scales.shape
    if not cs or len(cs) != len(ss) or cs[:-1] != ss[:-1] or ss[-1] == 0 or cs[-1] != 16 * ss[-1]:
        raise ValueError(f"{who}: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not match "
                         "([..., I/2] and [..., I/32])")


@functools.lru_cache(maxsize=4096)
def _scratch(nprob: int, rows: int, out_features: int, in_features: int, dt: int, quantize_input: int, device: int) -> int:
    """Scratch bytes of a call (decided by its sizes alone)."""
    return int(_lib.load().rwkv7mi_mxfp4_linear_workspace_bytes(nprob, rows, out_features, in_features, dt,
                                                                quantize_input))


def mxfp4_linear_multi_into(xs, weights, outs, *, biases=None, residuals=None, epilogues=None,
                            quantize_input: bool = False):
    """Up to four products of one shape in one launch: ``outs[i] = epilogue(xs[i] @ W_i^T
    (+ bias) (+ residual))`` with ``xs[i] [rows, I]`` and ``outs[i] [rows, O]`` contiguous
    and of one type (fp16 or bf16), ``weights[i] = (codes [O, I/2], scales [O, I/32])``.
    A residual may be its output's own memory; no output overlaps an input or another output.  The call's
    scratch is its own (torch's allocator; under capture the graph's pool)."""
    k = len(xs)
    biases, residuals = biases or [None] * k, residuals or [None] * k
    epilogues = list(epilogues) if epilogues is not None else [
        _lib.EPI_NONE if r is None else _lib.EPI_RESIDUAL for r in residuals]
    if not 1 <= k <= 4 or not k == len(weights) == len(outs) == len(biases) == len(residuals) == len(epilogues):
        raise ValueError("mxfp4: 1 to 4 products, with lists of one length")
    x0 = xs[0]
    if x0.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"mxfp4: fp16 or bf16 activations, got {x0.dtype}")
    rows, n = (int(s) for s in x0.shape)
    m = int(weights[0][0].shape[0])
    for x, (c, s), o, b, r, e in zip(xs, weights, outs, biases, residuals, epilogues):
        _check_packed(c, s, "mxfp4")
        if c.dim() != 2 or tuple(c.shape) != (m, n // 2) or n % BLOCK:
            raise ValueError(f"mxfp4: codes {tuple(c.shape)} do not match {n} inputs and {m} outputs")
        if not (c.is_contiguous() and s.is_contiguous()) or c.data_ptr() % 16 or s.data_ptr() % 4:
            raise ValueError("mxfp4: codes and scales must be contiguous, 16- and 4-byte aligned")
        if tuple(x.shape) != (rows, n) or x.dtype != x0.dtype or not x.is_contiguous() or x.data_ptr() % 16:
            raise ValueError("mxfp4: inputs must be contiguous, 16-byte aligned, of one shape and dtype")
        if tuple(o.shape) != (rows, m) or o.dtype != x0.dtype or not o.is_contiguous():
            raise ValueError("mxfp4: out must be a contiguous [rows, O] tensor of x's dtype")
        if b is not None and (int(b.numel()) != m or b.dtype != x0.dtype or not b.is_contiguous()):
            raise ValueError("mxfp4: bias must be a contiguous [O] tensor of x's dtype")
        if (e == _lib.EPI_RESIDUAL) != (r is not None) or e not in EPILOGUES.values():
            raise ValueError("mxfp4: the residual goes with the residual epilogue, and with no other")
        if r is not None:
            if tuple(r.shape) != (rows, m) or r.dtype != x0.dtype or not r.is_contiguous():
                raise ValueError("mxfp4: residual must be a contiguous [rows, O] tensor of x's dtype")
            if r.data_ptr() != o.data_ptr() and _lib.overlap(r, o):
                raise ValueError("mxfp4: out overlaps the residual without being it")
        _lib.require_same_device(x0, x, c, s, o, b, r, name="mxfp4_linear")
        if any(_lib.overlap(o, t) for t in xs):
            raise ValueError("mxfp4: out overlaps an input")
    for i, o in enumerate(outs):
        if any(t is not None and j != i and _lib.overlap(o, t) for side in (outs, residuals) for j, t in enumerate(side)):
            raise ValueError("mxfp4: out overlaps another product's out or residual")
    if rows == 0 or m == 0:
        return outs
    need = _scratch(k, rows, m, n, _lib.dtype_code(x0), int(bool(quantize_input)), x0.get_device())
    ws = torch.empty(need, dtype=torch.uint8, device=x0.device) if need else None
    arr = _lib.ptr_array
    with _lib.on_device(x0):
        _lib.call("rwkv7mi_mxfp4_linear", k, arr(xs), arr([c for c, _ in weights]), arr([s for _, s in weights]),
                  arr(biases), arr(residuals), arr(outs), (ctypes.c_int * k)(*epilogues), rows, m, n,
                  _lib.dtype_code(x0), int(bool(quantize_input)), _lib.ptr(ws), need, _lib.stream_of(x0))
    return outs


def mxfp4_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, *, bias: torch.Tensor | None = None,
                 out: torch.Tensor | None = None, residual: torch.Tensor | None = None, epilogue: str = "none",
                 quantize_input: bool = False) -> torch.Tensor:
    """``y = x @ W^T (+ bias)`` with ``W [O, I]`` in MXFP4 (``codes``, ``scales``) and
    ``x [..., I]`` fp16 or bf16, summed in fp32 and rounded once.

    ``epilogue``: ``"none"``, ``"relu2"`` (``relu(y)^2``) or ``"residual"``
    (``y + residual``, in fp32).  ``quantize_input``: ``x`` is quantised to MXFP4 first,
    as :func:`quantize_mxfp4` does, and both operands run as codes.  ``out`` (contiguous,
    ``x``'s dtype) may be the residual itself, not overlap ``x``.
    """
    epi = EPILOGUES.get(epilogue)
    if epi is None:
        raise ValueError(f"mxfp4: unknown epilogue {epilogue!r}; expected one of {', '.join(EPILOGUES)}")
    if (epi == _lib.EPI_RESIDUAL) != (residual is not None):
        raise ValueError("mxfp4: the residual goes with epilogue='residual'")
    shape, cshape = x.shape, codes.shape
    if not shape:
        raise ValueError("mxfp4: x must be [..., I]")
    _check_packed(codes, scales, "mxfp4")
    _lib.require_same_device(x, codes, scales, bias, out, residual, name="mxfp4_linear")
    n = shape[-1]
    if len(cshape) != 2 or 2 * cshape[1] != n:
        raise ValueError(f"mxfp4: x has {n} features but codes are {tuple(cshape)}")
    dt = x.dtype
    if dt is not torch.float16 and dt is not torch.bfloat16:
        raise ValueError(f"mxfp4: fp16 or bf16 activations, got {dt}")
    m, rows, want = cshape[0], x.numel() // n, (*shape[:-1], cshape[0])
    if not x.is_contiguous() or x.data_ptr() % 16:
        x = _aligned(x, 16)
    if not codes.is_contiguous() or codes.data_ptr() % 16:
        codes = _aligned(codes, 16)
    if not scales.is_contiguous() or scales.data_ptr() % 4:
        scales = _aligned(scales, 4)
    if bias is not None:
        if bias.numel() != m:
            raise ValueError(f"mxfp4: bias must hold {m} entries")
        bias = bias.to(dt).contiguous()
    if residual is not None:
        if tuple(residual.shape) != want or residual.dtype is not dt:
            raise ValueError("mxfp4: residual must have out's shape and dtype")
        residual = residual.contiguous()
    if out is None:
        out = x.new_empty(want)
    else:
        if tuple(out.shape) != want or not out.is_contiguous() or out.dtype is not dt:
            raise ValueError("mxfp4: out must be a contiguous [..., O] tensor of x's dtype")
        if _lib.overlap(out, x):
            raise ValueError("mxfp4: out overlaps an input")
        if residual is not None and residual.data_ptr() != out.data_ptr() and _lib.overlap(out, residual):
            raise ValueError("mxfp4: out overlaps the residual without being it")
    if rows == 0 or m == 0:
        return out
    quant, code = int(bool(quantize_input)), _lib.dtype_code(x)
    need = _scratch(1, rows, m, n, code, quant, x.get_device())
    ws = x.new_empty(need, dtype=torch.uint8) if need else None
    with _lib.on_device(x):
        _lib.call("rwkv7mi_mxfp4_linear1", x.data_ptr(), codes.data_ptr(), scales.data_ptr(), _lib.ptr(bias),
                  _lib.ptr(residual), out.data_ptr(), epi, rows, m, n, code, quant, _lib.ptr(ws), need,
                  _lib.stream_of(x))
    return out


class MXFP4Linear(torch.nn.Module):
    """Drop-in for ``nn.Linear`` with an MXFP4 weight (buffers ``codes [out, in/2]`` and
    ``scales [out, in/32]``) and the quantised-module protocol of
    :class:`~.native_quant_mm8.MM8Linear`.  ``quantize_input``: the input rows are
    quantised to MXFP4 too, at every row count."""

    def __init__(self, linear: torch.nn.Linear, *, quantize_input: bool = False):
        super().__init__()
        w = linear.weight.data
        if int(w.shape[1]) % BLOCK:
            raise ValueError("MXFP4 needs in_features divisible by 32")
        codes, scales = quantize_mxfp4(w)
        self._take(codes, scales, None if linear.bias is None else linear.bias.data.clone(), quantize_input)

    @classmethod
    def from_packed(cls, codes: torch.Tensor, scales: torch.Tensor, bias: torch.Tensor | None = None, *,
                    quantize_input: bool = False) -> "MXFP4Linear":
        """A module over codes ``[out, in/2]`` and scales ``[out, in/32]`` as they are."""
        _check_packed(codes, scales, "MXFP4Linear")
        if codes.dim() != 2:
            raise ValueError("MXFP4Linear: codes must be [out, in/2]")
        self = cls.__new__(cls)
        torch.nn.Module.__init__(self)
        self._take(_aligned(codes, 16), _aligned(scales, 4), bias, quantize_input)
        return self

    def _take(self, codes, scales, bias, quantize_input):
        self.out_features, self.in_features = int(codes.shape[0]), 2 * int(codes.shape[1])
        self.quantize_input = bool(quantize_input)
        self.register_buffer("codes", codes)
        self.register_buffer("scales", scales)
        self.register_buffer("bias", bias)

    def _run(self, x, out=None, residual=None, epilogue="none"):
        return mxfp4_linear(x, self.codes, self.scales, bias=self.bias, out=out, residual=residual, epilogue=epilogue,
                            quantize_input=self.quantize_input)

    def forward(self, x):
        return self._run(x)

    def rwkv7_forward_into(self, x, out):
        return self._run(x, out=out)

    def rwkv7_forward_relu2(self, x):
        return self._run(x, epilogue="relu2")

    def rwkv7_forward_add(self, x, residual):
        return self._run(x, residual=residual, epilogue="residual")

    def extra_repr(self):
        return (f"in={self.in_features}, out={self.out_features}, "
                f"mxfp4(quantize_input={self.quantize_input}, hip=gfx950)")


def quantize_model_mxfp4(model, *, min_params: int = 8_000_000, policy: str = "memory",
                         quantize_input: bool = False) -> int:
    """Swap eligible ``nn.Linear`` modules for :class:`MXFP4Linear`; returns the count.
    Linears whose ``in_features`` is not a multiple of 32 stay.  Weights may be fp32, but
    the modules run on fp16 or bf16 activations: an fp32 model is converted (``model.half()``
    or ``model.bfloat16()``) before it is called."""
    policy = normalize_native_mm_policy(policy)
    targets = [n for n, m in model.named_modules()
               if isinstance(m, torch.nn.Linear) and int(m.weight.shape[1]) % BLOCK == 0
               and should_quantize_linear(n, int(m.weight.numel()), min_params=min_params, policy=policy)]
    for full_name in targets:
        parent_name, _, attr = full_name.rpartition(".")
        parent = model.get_submodule(parent_name) if parent_name else model
        setattr(parent, attr, MXFP4Linear(getattr(parent, attr), quantize_input=quantize_input))
    setattr(model, "_rwkv7_native_mm_quantization", "mxfp4")
    setattr(model, "_rwkv7_native_mm_replaced_modules", len(targets))
    setattr(model, "_rwkv7_native_mm_block_replaced_modules", sum(n.startswith("model.layers.") for n in targets))
    invalidate_model_caches(model)
    return len(targets)


__all__ = ["quantize_mxfp4", "dequantize_mxfp4", "mxfp4_linear", "mxfp4_linear_multi_into", "MXFP4Linear",
           "quantize_model_mxfp4"]

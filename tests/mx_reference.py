"""MXFP4 in plain 64-bit torch on the CPU, written from the format: a block of 32
values shares 2^(e - 127), its codes are e2m1."""
from __future__ import annotations

import torch

VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantize(x: torch.Tensor):
    """``x [rows, I]`` -> (codes one a byte [rows, I], scale bytes [rows, I/32])."""
    b = x.detach().cpu().double().reshape(x.shape[0], -1, 32)
    bad = ~torch.isfinite(b).all(-1)
    b = torch.where(bad[..., None], 0.0, b)
    amax = b.abs().amax(-1)
    floor_log2 = torch.frexp(amax).exponent - 1
    e = torch.where(amax > 0, (floor_log2 - 2 + 127).clamp(0, 254), 0)
    v = b / torch.exp2((e - 127).double())[..., None]
    # nearest of the eight magnitudes; of two equally near the even code
    dist = (v.abs()[..., None] - VALUES).abs()
    best = dist.amin(-1, keepdim=True)
    near = dist == best
    index = torch.arange(8)
    even = torch.where(near & (index % 2 == 0), index, 99).amin(-1)
    any_ = torch.where(near, index, 99).amin(-1)
    code = torch.where(even < 99, even, any_)
    code = torch.where(v.abs() > 6, 7, code)
    code = code + 8 * torch.signbit(v).long()
    code = torch.where(bad[..., None], 0, code)
    e = torch.where(bad, 255, e)
    return code.reshape(x.shape).to(torch.uint8), e.to(torch.uint8)


def pack(codes: torch.Tensor) -> torch.Tensor:
    """One code a byte -> two, the even input low."""
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).contiguous()


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """64-bit values of packed codes [rows, I/2] and scales [rows, I/32]."""
    codes, scales = codes.cpu(), scales.cpu()
    c = torch.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1).long()
    v = VALUES[c & 7] * torch.where(c >= 8, -1.0, 1.0).double()
    s = torch.where(scales == 255, torch.nan, torch.exp2(scales.double() - 127))
    return (v.reshape(codes.shape[0], -1, 32) * s[..., None]).reshape(codes.shape[0], -1)


def random_weight(rows: int, inputs: int, gen: torch.Generator, lo: int = 112, hi: int = 122):
    """Random codes and scale bytes in lo..hi."""
    codes = torch.randint(0, 256, (rows, inputs // 2), generator=gen, dtype=torch.uint8)
    scales = torch.randint(lo, hi + 1, (rows, inputs // 32), generator=gen, dtype=torch.uint8)
    return codes, scales


def product(x, w, bias=None, residual=None, epilogue="none"):
    """(64-bit result, error bound) of epilogue(x w^T + bias) for 16-bit ``x [rows, I]`` and 64-bit
    ``w [O, I]``, sums in fp32.

    The bound: products are exact in fp32 (11 by 3 bits); the sum of I of them runs
    through fp32 adders in chains of at most I / 32 instructions after at most 32 adds
    within one, then up to 64 adds over waves and splits, each off by at most
    2^-23 (a truncating adder) of the running sum of magnitudes; bias, residual and
    square add three roundings; the result is rounded to x's type."""
    eps = torch.finfo(x.dtype).eps / 2
    xd = x.detach().cpu().double()
    s = xd @ w.t()
    mag = xd.abs() @ w.abs().t()
    if bias is not None:
        s = s + bias.cpu().double()
        mag = mag + bias.cpu().double().abs()
    err = mag * (x.shape[1] / 32 + 32 + 64 + 3) * 2.0 ** -23
    if epilogue == "relu2":
        err = 2 * s.abs() * err + err * err
        s = s.clamp(min=0) ** 2
        err = err + s * 2.0 ** -24
    elif epilogue == "residual":
        s = s + residual.cpu().double()
        err = err + s.abs() * 2.0 ** -24
    tiny = torch.finfo(x.dtype).smallest_normal * eps  # half a step of the subnormals
    return s, err + (s.abs() + err) * eps + tiny

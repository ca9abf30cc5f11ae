"""Products with the largest scale bytes, 2^126 and 2^127 (253, 254): their larger codes pass
the range of bf16 and of fp32, so a weight must not be formed by itself."""
from __future__ import annotations

import pytest
import torch

import mx_reference as ref

pytestmark = pytest.mark.gpu


def _weight(m, n, seed):
    """Rows of codes whose scale bytes lie in 100..254; every third row below 253."""
    g = torch.Generator().manual_seed(seed)
    codes, scales = ref.random_weight(m, n, g, 100, 254)
    scales[::3] = scales[::3].clamp(max=252)
    scales[1, :] = 254
    return codes, scales, g


def _check(got, x, w, bias, quantize_input):
    if quantize_input:
        x = ref.values(*[t if i else ref.pack(t) for i, t in enumerate(ref.quantize(x))]).to(x.dtype)
    want, bound = ref.product(x, w, bias)
    assert torch.isfinite(got).all()
    worst = ((got.cpu().double() - want).abs() - bound).max().item()
    assert worst <= 0, worst


@pytest.mark.parametrize("quantize_input", [False, True])
@pytest.mark.parametrize("rows,n,m", [(1, 64, 17), (3, 4096, 48), (16, 16384, 40), (33, 1024, 100), (40, 288, 70),
                                      (600, 1056, 65), (600, 1024, 264), (520, 8704, 40), (2000, 8224, 1030)])
def test_bf16_rows_times_the_largest_scales(rows, n, m, quantize_input):
    """bf16 rows of magnitude 2^-120: products up to 2^10.  A row of zeros gives its bias."""
    import rwkv7mi as mi

    codes, scales, g = _weight(m, n, rows + n)
    x = (torch.randn(rows, n, generator=g) * 2.0 ** -120).bfloat16()
    x[rows // 2] = 0
    bias = torch.randn(m, generator=g).bfloat16()
    got = mi.mxfp4_linear(x.cuda(), codes.cuda(), scales.cuda(), bias=bias.cuda(), quantize_input=quantize_input)
    pick = slice(0, rows) if rows < 700 else slice(rows // 2 - 40, rows // 2 + 40)
    _check(got[pick], x[pick], ref.values(codes, scales), bias, quantize_input)
    assert torch.equal(got[rows // 2].cpu(), bias)


@pytest.mark.parametrize("n,m", [(96, 16325), (128, 16384)])
def test_a_long_bf16_batch_times_the_largest_scales(n, m):
    import rwkv7mi as mi

    rows = 4096
    codes, scales, g = _weight(m, n, n)
    x = (torch.randn(rows, n, generator=g) * 2.0 ** -120).bfloat16()
    x[300] = 0
    got = mi.mxfp4_linear(x.cuda(), codes.cuda(), scales.cuda())
    w = ref.values(codes, scales)
    for r in (290, 2000, 4080):
        _check(got[r:r + 16], x[r:r + 16], w, None, False)
    assert (got[300] == 0).all()


@pytest.mark.parametrize("rows", [1, 24, 90, 400, 600])
def test_fp16_zeros_times_the_largest_scales(rows):
    import rwkv7mi as mi

    codes, scales, g = _weight(70, 512, rows)
    bias = torch.randn(70, generator=g).half()
    got = mi.mxfp4_linear(torch.zeros(rows, 512, dtype=torch.float16, device="cuda"), codes.cuda(), scales.cuda(),
                          bias=bias.cuda())
    assert torch.equal(got.cpu(), bias.expand(rows, 70))


@pytest.mark.parametrize("rows", [1, 24, 90, 400, 600])
def test_nan_scales_beside_the_largest(rows):
    """Byte 255 in a row that also holds 254: NaN in that output and in no other."""
    import rwkv7mi as mi

    codes, scales, g = _weight(40, 512, rows)
    scales[11, 3] = 255
    x = (torch.randn(rows, 512, generator=g) * 2.0 ** -120).bfloat16()
    x[:, 96:128] = 0
    got = mi.mxfp4_linear(x.cuda(), codes.cuda(), scales.cuda()).cpu()
    assert torch.isnan(got[:, 11]).all()
    assert torch.isfinite(got[:, [i for i in range(40) if i != 11]]).all()


@pytest.mark.parametrize("rows", [1, 24, 90, 400, 600])
def test_bf16_rows_times_the_smallest_scales(rows):
    """Bytes 0 to 4 against rows of magnitude 2^100: the weights are bf16's subnormals."""
    import rwkv7mi as mi

    g = torch.Generator().manual_seed(rows)
    codes, scales = ref.random_weight(70, 512, g, 0, 4)
    x = (torch.randn(rows, 512, generator=g) * 2.0 ** 100).bfloat16()
    got = mi.mxfp4_linear(x.cuda(), codes.cuda(), scales.cuda())
    _check(got, x, ref.values(codes, scales), None, False)

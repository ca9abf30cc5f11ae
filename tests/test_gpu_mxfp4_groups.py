"""Grouped MXFP4 products whose K is split, and long batches (the weight written out in 16
bits), every output against 64 bits."""
from __future__ import annotations

import pytest
import torch

import mx_reference as ref

pytestmark = pytest.mark.gpu
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _problem(rows, n, m, dt, seed):
    g = torch.Generator().manual_seed(seed)
    codes, scales = ref.random_weight(m, n, g)
    return (torch.randn(rows, n, generator=g).to(dt), codes, scales, torch.randn(m, generator=g).to(dt),
            torch.randn(rows, m, generator=g).to(dt))


def _quantized(x):
    return ref.values(*[t if i else ref.pack(t) for i, t in enumerate(ref.quantize(x))]).to(x.dtype)


def _within(got, x, w, bias, residual, epilogue):
    want, bound = ref.product(x, w, bias, residual, epilogue)
    worst = ((got.cpu().double() - want).abs() - bound).max().item()
    assert worst <= 0, (epilogue, worst)


@pytest.mark.parametrize("quantize_input", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("rows,n,m", [(16, 16384, 40), (40, 8704, 40), (100, 8704, 40), (600, 8704, 40), (40, 8224, 24),
                                      (600, 8224, 40), (128, 4096, 520), (300, 4096, 70)])
def test_grouped_products_of_many_inputs(rows, n, m, dtype, quantize_input):
    """Inputs, weights, biases, residuals and epilogues of their own in every place."""
    from rwkv7mi import _lib
    from rwkv7mi.native_quant_mxfp4 import mxfp4_linear_multi_into

    dt = DTYPES[dtype]
    problems = [_problem(rows, n, m, dt, 10 * rows + n + i) for i in range(4)]
    gpu = [[t.cuda() for t in p] for p in problems]
    names = ["none", "residual", "relu2", "residual"]
    outs = [p[4].clone() if e == "residual" and i == 1 else torch.empty_like(p[4])
            for i, (p, e) in enumerate(zip(gpu, names))]
    residuals = [None, outs[1], None, gpu[3][4]]
    biases = [gpu[0][3], None, gpu[2][3], gpu[3][3]]
    mxfp4_linear_multi_into([p[0] for p in gpu], [(p[1], p[2]) for p in gpu], outs, biases=biases, residuals=residuals,
                            epilogues=[{"none": _lib.EPI_NONE, "relu2": _lib.EPI_RELU2,
                                        "residual": _lib.EPI_RESIDUAL}[e] for e in names],
                            quantize_input=quantize_input)
    for i, (x, codes, scales, bias, res) in enumerate(problems):
        _within(outs[i], _quantized(x) if quantize_input else x, ref.values(codes, scales),
                None if biases[i] is None else bias, res if names[i] == "residual" else None, names[i])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("epilogue", ["none", "relu2", "residual"])
@pytest.mark.parametrize("rows,n,m", [(4096, 128, 16384), (4001, 192, 16325), (16384, 4096, 4096)])
def test_long_batches_of_whole_steps(rows, n, m, epilogue, dtype):
    """1024 tiles of 256 x 256 and more, outputs that store whole and that do not; a residual in
    place, a NaN scale and a NaN row."""
    import rwkv7mi as mi

    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(n)
    codes, scales = ref.random_weight(m, n, g)
    scales[77, 1] = 255
    x = torch.randn(rows, n, generator=g).to(dt)
    x[257, 5] = float("nan")
    bias = torch.randn(m, generator=g).to(dt)
    residual = torch.randn(rows, m, generator=g).to(dt).cuda() if epilogue == "residual" else None
    before = None if residual is None else residual.clone()
    got = mi.mxfp4_linear(x.cuda(), codes.cuda(), scales.cuda(), bias=bias.cuda(), residual=residual, out=residual,
                          epilogue=epilogue)
    assert residual is None or got is residual
    keep = [o for o in range(m) if o != 77]
    assert torch.isnan(got[:, 77]).all() and torch.isnan(got[257]).all()
    assert not torch.isnan(got[:, keep][[r for r in range(rows) if r != 257]]).any()
    w = ref.values(codes, scales)[keep]
    for r in (0, 240, 1790, rows - 10):
        rs = [i for i in range(r, r + 10) if i != 257]
        _within(got[rs][:, keep], x[rs], w, bias[keep], None if before is None else before[rs][:, keep], epilogue)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_grouped_long_batches(dtype):
    """Three products of one launch, as R, K and V of a long prompt."""
    from rwkv7mi.native_quant_mxfp4 import mxfp4_linear_multi_into

    rows, n, m, dt = 4096, 320, 16384, DTYPES[dtype]
    problems = [_problem(rows, n, m, dt, i) for i in range(3)]
    outs = [torch.empty(rows, m, dtype=dt, device="cuda") for _ in range(3)]
    mxfp4_linear_multi_into([p[0].cuda() for p in problems], [(p[1].cuda(), p[2].cuda()) for p in problems], outs,
                            biases=[p[3].cuda() for p in problems])
    for out, (x, codes, scales, bias, _) in zip(outs, problems):
        w = ref.values(codes, scales)
        for r in (0, 2044, 4080):
            _within(out[r:r + 16], x[r:r + 16], w, bias, None, "none")


def test_rows_of_two_gigabytes():
    """Inputs past 2^31 bytes run in chunks of rows (of 261888 here)."""
    import rwkv7mi as mi

    rows, n, m = 262400, 4096, 16
    g = torch.Generator().manual_seed(1)
    codes, scales = ref.random_weight(m, n, g)
    x = torch.randn(512, n, generator=g).half().cuda().repeat((rows + 511) // 512, 1)[:rows]
    x.mul_((1 + torch.arange(rows, device="cuda") % 7)[:, None])  # (no two chunks alike)
    residual = torch.randn(rows, m, generator=g).half().cuda()
    got = mi.mxfp4_linear(x, codes.cuda(), scales.cuda(), residual=residual, epilogue="residual")
    w = ref.values(codes, scales)
    for r in (0, 130000, 261880, 262390):
        rs = slice(r, min(r + 16, rows))
        _within(got[rs], x[rs], w, None, residual[rs], "residual")


@pytest.mark.parametrize("last", ["bias", "codes", "scales"])
def test_linears_that_cannot_be_grouped_run_one_by_one(last):
    """A bias of another type, codes and scales off their boundary, in the third of three linears
    of a model: the results of the single products."""
    from rwkv7mi import MXFP4Linear
    from rwkv7mi.model import BlockFloatLinear, QuantLinear

    x, codes, scales, bias, _ = (t.cuda() for t in _problem(5, 256, 40, torch.float16, 1))
    mods = [MXFP4Linear.from_packed(codes, scales, bias) for _ in range(3)]
    want = [m(x) for m in mods]
    if last == "bias":
        mods[2].bias = bias.float()
    else:
        t = getattr(mods[2], last)
        moved = torch.zeros(t.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view_as(t)
        setattr(mods[2], last, moved.copy_(t))
    outs = [torch.empty(5, 40, dtype=torch.float16, device="cuda") for _ in range(3)]
    QuantLinear.apply_group([BlockFloatLinear(m) for m in mods], [x, x, x], outs)
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_modules_of_fp32_linears_run_in_16_bits():
    """An fp32 model is quantised from its fp32 weights and converted afterwards."""
    import rwkv7mi as mi

    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(64, 40), torch.nn.ReLU()).cuda()
    codes, scales = mi.quantize_mxfp4(net[0].weight.data)
    bias = net[0].bias.data.clone()
    x = torch.randn(5, 64, device="cuda")
    assert mi.quantize_model_mxfp4(net, min_params=1) == 1
    with pytest.raises(ValueError, match="fp16 or bf16"):
        net(x)
    for dt in (torch.float16, torch.bfloat16):
        bias = bias.to(dt)
        y = net.to(dt)(x.to(dt))
        assert torch.equal(net[0].bias, bias)
        assert torch.equal(y, mi.mxfp4_linear(x.to(dt), codes, scales, bias=bias).relu())

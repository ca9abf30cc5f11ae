"""MXFP4 quantiser, products and module against plain 64-bit torch."""
from __future__ import annotations

import pytest
import torch

import mx_reference as ref

pytestmark = pytest.mark.gpu
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ quantiser
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,width", [(1, 32), (3, 64), (37, 1056), (5, 2080), (256, 4096), (1, 65536)])
def test_quantize_matches_the_format(rows, width, dtype):
    import rwkv7mi as mi

    x = (torch.randn(rows, width, generator=_gen(rows + width)) * 3).to(DTYPES[dtype])
    codes, scales = mi.quantize_mxfp4(x.cuda())
    want_c, want_s = ref.quantize(x)
    assert torch.equal(scales.cpu(), want_s)
    assert torch.equal(codes.cpu(), ref.pack(want_c))
    back = mi.dequantize_mxfp4(codes, scales, out_dtype=DTYPES[dtype])
    assert torch.equal(back.cpu().double(), ref.values(codes, scales))


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_quantize_special_blocks(dtype):
    """Zeros, ties, saturation, one large value, the smallest and largest magnitudes,
    infinities and NaN; neighbours of a bad block keep their values."""
    import rwkv7mi as mi

    dt = DTYPES[dtype]
    info = torch.finfo(dt)
    x = torch.zeros(12, 32)
    x[1] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0] * 4)
    x[2] = -x[1]
    x[3] = torch.linspace(-7.9, 7.9, 32)
    x[4, 7] = 1000.0
    x[5] = info.tiny * torch.arange(32)
    x[6] = info.max * torch.linspace(-1, 1, 32)
    x[7, 3] = float("inf")
    x[7, 4] = 1.0
    x[8, 31] = float("nan")
    x[9] = -0.0
    x[10, 0] = torch.finfo(dt).smallest_normal / 4  # a subnormal
    x[11] = torch.randn(32, generator=_gen(1)) * 1e-3
    x = x.to(dt)
    codes, scales = mi.quantize_mxfp4(x.cuda())
    want_c, want_s = ref.quantize(x)
    assert torch.equal(scales.cpu(), want_s)
    assert torch.equal(codes.cpu(), ref.pack(want_c))
    back = mi.dequantize_mxfp4(codes, scales, out_dtype=torch.float32).cpu().double()
    want = ref.values(codes, scales)
    assert torch.equal(torch.isnan(back), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(back), torch.nan_to_num(want))
    assert torch.isnan(back[7]).all() and torch.isnan(back[8]).all() and not torch.isnan(back[[0, 1, 6, 9, 11]]).any()


def test_quantize_strides_and_ranks():
    import rwkv7mi as mi

    big = torch.randn(6, 5, 192, generator=_gen(2)).half().cuda()
    want = mi.quantize_mxfp4(big.reshape(30, 192).clone())
    for x in (big, big.transpose(0, 1).contiguous().transpose(0, 1)):
        c, s = mi.quantize_mxfp4(x)
        assert c.shape == (6, 5, 96) and s.shape == (6, 5, 6)
        assert torch.equal(c.reshape(30, 96), want[0]) and torch.equal(s.reshape(30, 6), want[1])
    rows = big.reshape(30, 192)
    for view in (rows[:, 64:128], rows[:, 1:65], rows[::2, :64], rows[:1, 3:35], rows[3]):
        a, b = mi.quantize_mxfp4(view), mi.quantize_mxfp4(view.contiguous().clone())
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    c, s = mi.quantize_mxfp4(big[:0])
    assert c.shape == (0, 5, 96) and s.shape == (0, 5, 6)
    assert mi.dequantize_mxfp4(c, s).shape == (0, 5, 192)


# ------------------------------------------------------------------ products
SHAPES = [(1, 32, 1), (1, 64, 17), (2, 96, 40), (16, 128, 16), (17, 160, 33), (1, 4096, 48), (5, 1056, 65),
          (33, 1024, 100), (40, 512, 300), (64, 2048, 96), (65, 288, 130), (129, 640, 257), (200, 2560, 512),
          (257, 1024, 520), (300, 96, 70), (520, 768, 264),
          (2, 8704, 30), (9, 16384, 40), (16, 8224, 24),
          (4, 8192, 40), (2, 7680, 24), (700, 608, 1100),
          (256, 2080, 40), (100, 9248, 30), (128, 768, 200), (250, 32, 9), (400, 544, 70),
          (513, 32, 1), (514, 160, 33), (520, 288, 130), (530, 640, 257), (600, 1056, 65), (521, 2080, 300),
          (516, 8224, 24), (515, 16384, 40)]


def _case(rows, n, m, dt, seed, *, lo=112, hi=122):
    g = _gen(seed)
    codes, scales = ref.random_weight(m, n, g, lo, hi)
    x = torch.randn(rows, n, generator=g).to(dt)
    return x, codes, scales, g


@pytest.mark.parametrize("quantize_input", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("rows,n,m", SHAPES)
def test_linear_against_64_bits(rows, n, m, dtype, quantize_input):
    import rwkv7mi as mi

    dt = DTYPES[dtype]
    x, codes, scales, g = _case(rows, n, m, dt, 7 * rows + n + m)
    w = ref.values(codes, scales)
    bias = torch.randn(m, generator=g).to(dt)
    residual = torch.randn(rows, m, generator=g).to(dt)
    xr = ref.values(*[t if i else ref.pack(t) for i, t in enumerate(ref.quantize(x))]).to(dt) if quantize_input else x
    for epilogue, b in (("none", None), ("relu2", None), ("residual", bias)):
        r = residual if epilogue == "residual" else None
        want, bound = ref.product(xr, w, b, r, epilogue)
        got = mi.mxfp4_linear(x.cuda(), codes.cuda(), scales.cuda(), bias=None if b is None else b.cuda(),
                              residual=None if r is None else r.cuda(), epilogue=epilogue,
                              quantize_input=quantize_input).cpu().double()
        worst = ((got - want).abs() - bound).max().item()
        assert worst <= 0, (epilogue, worst)


@pytest.mark.parametrize("dtype,epilogue", [("fp16", "relu2"), ("bf16", "residual")])
def test_linear_of_a_prefill_batch(dtype, epilogue):
    """1024 tiles of 256 x 256 and more, ragged on both sides and in K: the weight in 16 bits."""
    import rwkv7mi as mi

    rows, n, m, dt = 4001, 96, 16325, DTYPES[dtype]
    x, codes, scales, g = _case(rows, n, m, dt, 3)
    scales[7, 1] = 60
    x, codes, scales = x.cuda(), codes.cuda(), scales.cuda()
    bias = torch.randn(m, generator=g).to(dt).cuda()
    residual = torch.randn(rows, m, generator=g).to(dt).cuda() if epilogue == "residual" else None
    got = mi.mxfp4_linear(x, codes, scales, bias=bias, residual=residual, epilogue=epilogue)
    w = ref.values(codes, scales)
    for r in (0, 255, 1300, 3990):  # a few rows of several tiles, all columns
        rs = slice(r, min(r + 40, rows))
        want, bound = ref.product(x[rs], w, bias, None if residual is None else residual[rs], epilogue)
        assert ((got[rs].cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("quantize_input", [False, True])
@pytest.mark.parametrize("rows,n,m", [(5000, 1056, 1030), (5000, 2080, 2070), (2000, 8224, 1030), (4100, 8224, 1030),
                                      (1500, 16384, 2050), (2451, 13792, 1618)])
def test_linear_of_larger_tiles(rows, n, m, quantize_input):
    """128- and 256-row tiles, whole and split in K, ragged on all sides."""
    import rwkv7mi as mi

    x, codes, scales, g = _case(rows, n, m, torch.float16, n)
    bias = torch.randn(m, generator=g).half()
    got = mi.mxfp4_linear(x.cuda(), codes.cuda(), scales.cuda(), bias=bias.cuda(), epilogue="relu2",
                          quantize_input=quantize_input).cpu().double()
    w = ref.values(codes, scales)
    for r in (0, 120, 250, rows - 20):  # a few rows of several tiles, all columns
        xr = x[r:r + 20]
        if quantize_input:
            xr = ref.values(*[t if i else ref.pack(t) for i, t in enumerate(ref.quantize(xr))]).half()
        want, bound = ref.product(xr, w, bias, None, "relu2")
        assert ((got[r:r + 20] - want).abs() <= bound).all(), r


@pytest.mark.parametrize("rows", [1, 24, 90, 400, 600])
def test_linear_fp16_scales_far_apart(rows):
    """fp16 rows with block scales over 2^-100..2^-7: a row's largest scale is brought to
    2^13, where fp16's grid is 2^-24: smaller weights are off by at most half a step,
    2^-38 of the largest scale."""
    import rwkv7mi as mi

    n, m = 512, 70
    g = _gen(rows)
    codes, scales = ref.random_weight(m, n, g, 27, 60)
    scales[:, 5] = 120  # one block per row that decides
    scales[3] = 60
    scales[4, :] = 0
    x = (torch.randn(rows, n, generator=g) * 30).half()
    w = ref.values(codes, scales)
    want, bound = ref.product(x, w)
    top = torch.exp2(scales.amax(-1).double() - 127)
    bound = bound + torch.outer(x.double().abs().sum(-1), top) * 2.0 ** -38
    got = mi.mxfp4_linear(x.cuda(), codes.cuda(), scales.cuda()).cpu().double()
    assert ((got - want).abs() <= bound).all()


@pytest.mark.parametrize("quantize_input", [False, True])
@pytest.mark.parametrize("rows", [1, 20, 70, 300, 600])
def test_linear_nan_scale_stays_in_its_output(rows, quantize_input):
    import rwkv7mi as mi

    x, codes, scales, _ = _case(rows, 256, 40, torch.float16, rows)
    scales[11, 3] = 255
    x[0, 5] = 0.0
    got = mi.mxfp4_linear(x.cuda(), codes.cuda(), scales.cuda(), quantize_input=quantize_input,
                          epilogue="relu2").cpu()
    assert torch.isnan(got[:, 11]).all()
    assert not torch.isnan(got[:, [i for i in range(40) if i != 11]]).any()


@pytest.mark.parametrize("quantize_input", [False, True])
@pytest.mark.parametrize("rows", [3, 70, 300, 600])
def test_linear_bad_rows_stay_in_their_rows(rows, quantize_input):
    import rwkv7mi as mi

    x, codes, scales, _ = _case(rows, 256, 40, torch.bfloat16, rows)
    x[1, 7] = float("nan")
    got = mi.mxfp4_linear(x.cuda(), codes.cuda(), scales.cuda(), quantize_input=quantize_input).cpu()
    assert torch.isnan(got[1]).all() and not torch.isnan(got[[0] + list(range(2, rows))]).any()


@pytest.mark.parametrize("quantize_input", [False, True])
@pytest.mark.parametrize("rows", [1, 7, 16, 30, 64, 100, 300, 600])
def test_grouped_products_equal_single_ones(rows, quantize_input):
    """Three products of one launch, a residual in place, and a row's result alike in
    every launch of the same row count."""
    import rwkv7mi as mi
    from rwkv7mi.native_quant_mxfp4 import mxfp4_linear_multi_into

    n, m = 512, 320
    cases = [_case(rows, n, m, torch.float16, 100 * rows + i)[:3] for i in range(3)]
    xs = [c[0].cuda() for c in cases]
    ws = [(c[1].cuda(), c[2].cuda()) for c in cases]
    res = torch.randn(rows, m, generator=_gen(4)).half().cuda()
    outs = [torch.empty(rows, m, device="cuda", dtype=torch.float16) for _ in range(2)] + [res.clone()]
    mxfp4_linear_multi_into(xs, ws, outs, residuals=[None, None, outs[2]], quantize_input=quantize_input)
    for i in range(3):
        epilogue = "residual" if i == 2 else "none"
        x, codes, scales = cases[i]
        xr = ref.values(*[t if j else ref.pack(t) for j, t in enumerate(ref.quantize(x))]).half() if quantize_input else x
        want, bound = ref.product(xr, ref.values(codes, scales), None, res if i == 2 else None, epilogue)
        assert ((outs[i].cpu().double() - want).abs() <= bound).all()
    again = [torch.empty(rows, m, device="cuda", dtype=torch.float16) for _ in range(2)] + [res.clone()]
    mxfp4_linear_multi_into(xs, ws, again, residuals=[None, None, again[2]], quantize_input=quantize_input)
    assert all(torch.equal(a, b) for a, b in zip(outs, again))  # the same bits every time


def test_linear_strides_ranks_and_out():
    import rwkv7mi as mi

    x, codes, scales, _ = _case(24, 128, 50, torch.float16, 5)
    x, codes, scales = x.cuda(), codes.cuda(), scales.cuda()
    want = mi.mxfp4_linear(x, codes, scales)
    assert torch.equal(mi.mxfp4_linear(x.view(2, 3, 4, 128), codes, scales), want.view(2, 3, 4, 50))
    wide = torch.zeros(24, 200, device="cuda", dtype=torch.float16)
    wide[:, 7:135] = x
    assert torch.equal(mi.mxfp4_linear(wide[:, 7:135], codes, scales), want)
    shifted = torch.empty(codes.numel() + 1, device="cuda", dtype=torch.uint8)[1:].view_as(codes).copy_(codes)
    assert torch.equal(mi.mxfp4_linear(x, shifted, scales), want)
    out = torch.empty(24, 50, device="cuda", dtype=torch.float16)
    assert mi.mxfp4_linear(x, codes, scales, out=out) is out and torch.equal(out, want)
    guard = torch.full((26, 50), 7.0, device="cuda", dtype=torch.float16)
    mi.mxfp4_linear(x, codes, scales, out=guard[1:25])
    assert torch.equal(guard[1:25], want) and (guard[0] == 7).all() and (guard[25] == 7).all()
    one = mi.mxfp4_linear(x[3], codes, scales)
    assert one.shape == (50,)
    assert mi.mxfp4_linear(x[:0], codes, scales).shape == (0, 50)


@pytest.mark.parametrize("quantize_input", [False, True])
@pytest.mark.parametrize("rows", [1, 40, 300, 600])
def test_linear_in_a_graph_and_on_another_stream(rows, quantize_input):
    import rwkv7mi as mi

    x, codes, scales, _ = _case(rows, 1024, 640, torch.bfloat16, rows)
    x, codes, scales = x.cuda(), codes.cuda(), scales.cuda()
    call = lambda: mi.mxfp4_linear(x, codes, scales, epilogue="relu2", quantize_input=quantize_input)
    want = call()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = call()
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(got, want)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = call()
        graphs.append((g, y))
    for k in range(3):
        x.copy_(torch.randn(rows, 1024, generator=_gen(50 + k)).to(x.dtype))
        want = call()
        for g, y in graphs:
            y.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want)


# ------------------------------------------------------------------ module
def test_module_protocol_and_state_dict():
    import rwkv7mi as mi

    torch.manual_seed(0)
    lin = torch.nn.Linear(256, 96, bias=True, device="cuda", dtype=torch.float16)
    mod = mi.MXFP4Linear(lin)
    x = torch.randn(9, 256, device="cuda", dtype=torch.float16)
    c, s = mi.quantize_mxfp4(lin.weight.data)
    want, bound = ref.product(x, ref.values(c, s), lin.bias.data)
    y = mod(x)
    assert ((y.cpu().double() - want).abs() <= bound).all()
    out = torch.empty_like(y)
    assert torch.equal(mod.rwkv7_forward_into(x, out), y)
    want2, bound2 = ref.product(x, ref.values(c, s), lin.bias.data, None, "relu2")
    assert ((mod.rwkv7_forward_relu2(x).cpu().double() - want2).abs() <= bound2).all()
    want3, bound3 = ref.product(x, ref.values(c, s), lin.bias.data, y, "residual")
    assert ((mod.rwkv7_forward_add(x, y).cpu().double() - want3).abs() <= bound3).all()
    assert set(mod.state_dict()) == {"codes", "scales", "bias"}
    again = mi.MXFP4Linear(torch.nn.Linear(256, 96, bias=True, device="cuda", dtype=torch.float16))
    again.load_state_dict(mod.state_dict())
    assert torch.equal(again(x), y)
    packed = mi.MXFP4Linear.from_packed(c, s, lin.bias.data)
    assert torch.equal(packed(x), y)


def test_quantize_model_swaps_eligible_linears():
    import rwkv7mi as mi

    net = torch.nn.Sequential(torch.nn.Linear(128, 64), torch.nn.Linear(64, 20), torch.nn.Linear(20, 8)).cuda().half()
    x = torch.randn(4, 128, device="cuda", dtype=torch.float16)
    assert mi.quantize_model_mxfp4(net, min_params=1, quantize_input=True) == 2
    assert isinstance(net[0], mi.MXFP4Linear) and net[0].quantize_input and isinstance(net[2], torch.nn.Linear)
    assert net(x).shape == (4, 8)


@pytest.mark.parametrize("quantize_input", [False, True])
@pytest.mark.parametrize("rows", [1, 40, 600])
@pytest.mark.parametrize("n", [512, 640])
def test_scales_on_any_dword_and_outputs_on_any_element(rows, n, quantize_input):
    """Scales that start 4, 8 and 12 bytes behind a 16-byte boundary, and an output and a
    residual that start on an odd element: the same bits."""
    import rwkv7mi as mi

    m = 264
    x, codes, scales, g = _case(rows, n, m, torch.float16, rows + n)
    x, codes, scales = x.cuda(), codes.cuda(), scales.cuda()
    res = torch.randn(rows, m, generator=g).half().cuda()
    want = mi.mxfp4_linear(x, codes, scales, residual=res, epilogue="residual", quantize_input=quantize_input)
    for off in (4, 8, 12):
        moved = torch.zeros(scales.numel() + 16, dtype=torch.uint8, device="cuda")[off:off + scales.numel()]
        moved = moved.view_as(scales).copy_(scales)
        buf = torch.full((rows * m + 2,), 5.0, dtype=torch.float16, device="cuda")
        out = buf[1:-1].view(rows, m)
        out.copy_(res)  # in place of the residual
        got = mi.mxfp4_linear(x, codes, moved, residual=out, epilogue="residual", out=out, quantize_input=quantize_input)
        assert torch.equal(got, want) and buf[0] == 5 and buf[-1] == 5


@pytest.mark.parametrize("quantize_input", [False, True])
@pytest.mark.parametrize("rows", [40, 600])
def test_calls_on_two_streams_and_one_tensor_in_every_place(rows, quantize_input):
    """Two split products at once on two streams, and one weight and one input in all four
    places of a launch."""
    import rwkv7mi as mi
    from rwkv7mi.native_quant_mxfp4 import mxfp4_linear_multi_into

    x, codes, scales, _ = _case(rows, 8704, 40, torch.float16, rows)
    x, codes, scales = x.cuda(), codes.cuda(), scales.cuda()
    want = mi.mxfp4_linear(x, codes, scales, quantize_input=quantize_input)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(mi.mxfp4_linear(x, codes, scales, quantize_input=quantize_input))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for side in got for y in side)
    outs = [torch.empty_like(want) for _ in range(4)]
    mxfp4_linear_multi_into([x] * 4, [(codes, scales)] * 4, outs, quantize_input=quantize_input)
    again = [torch.empty_like(want) for _ in range(4)]
    mxfp4_linear_multi_into([x] * 4, [(codes, scales)] * 4, again, quantize_input=quantize_input)
    assert all(torch.equal(o, outs[0]) for o in outs + again)

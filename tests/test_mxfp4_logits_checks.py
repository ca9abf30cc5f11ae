"""Refusals of the MXFP4 and logits entry points, on the CPU: no call here reaches a launch."""
from __future__ import annotations

import ctypes

import pytest
import torch

P = ctypes.c_void_p


def _lib():
    from rwkv7mi import _lib

    return _lib.load()


def _arr(*v):
    return (P * len(v))(*v)


A = 1 << 20  # an aligned address that is never read


@pytest.mark.parametrize("rows,n,ld,dtype,x", [(2, 33, 33, 1, A), (2, 0, 0, 1, A), (-1, 32, 32, 1, A), (2, 32, 16, 1, A),
                                               (2, 32, 32, 7, A), (2, 32, 32, 1, 0), (2, 32, 32, 1, A + 2),
                                               (2, 32, 36, 1, A), (1 << 40, 1 << 20, 1 << 20, 1, A),
                                               (1 << 20, 1 << 15, 1 << 15, 1, A)])
def test_quantize_entry_refuses(rows, n, ld, dtype, x):
    assert _lib().rwkv7mi_mxfp4_quantize(x, rows, n, ld, dtype, A, A, None) == -1


@pytest.mark.parametrize("rows,n,dtype,y", [(2, 48, 1, A), (2, 32, 9, A), (2, 32, 1, 0), (2, 32, 1, A + 8)])
def test_dequantize_entry_refuses(rows, n, dtype, y):
    assert _lib().rwkv7mi_mxfp4_dequantize(A, A, rows, n, y, dtype, None) == -1


def _linear(nprob=1, x=A, codes=A, scales=A, y=A, epi=0, residual=None, rows=2, m=16, n=64, dt=1, quant=0, ws=None, nws=0):
    return _lib().rwkv7mi_mxfp4_linear(nprob, _arr(x), _arr(codes), _arr(scales), None,
                                       None if residual is None else _arr(residual), _arr(y), (ctypes.c_int * 1)(epi),
                                       rows, m, n, dt, quant, ws, nws, None)


@pytest.mark.parametrize("kw", [dict(nprob=0), dict(nprob=5), dict(x=0), dict(codes=0), dict(scales=0), dict(y=0),
                                dict(x=A + 4), dict(codes=A + 8), dict(scales=A + 1), dict(epi=3), dict(epi=2),
                                dict(rows=-1), dict(m=0), dict(n=48), dict(dt=0), dict(rows=1 << 22)])
def test_linear_entry_refuses(kw):
    assert _linear(**kw) == -1


def test_linear_entry_wants_its_workspace():
    need = _lib().rwkv7mi_mxfp4_linear_workspace_bytes(1, 2, 16, 64, 1, 1)
    assert need >= 2 * (32 + 2)
    assert _linear(quant=1) == -3
    assert _linear(quant=1, ws=A, nws=need - 1) == -3
    assert _linear(quant=1, ws=A + 8, nws=need) == -3


def test_empty_calls_launch_nothing():
    assert _linear(rows=0) == 0
    assert _lib().rwkv7mi_mxfp4_quantize(None, 0, 32, 32, 1, None, None, None) == 0
    assert _logits(rows=0) == 0


def _logits(x=A, rows=2, n=100, ldx=100, dt=1, out=A, ldo=100, odt=1, hist=None, bits=64, ldh=8, cap=8, lengths=None,
            bias=None, ldb=0, allowed=None, lda=0, nxt=None, nxt2=None, append=0, ws=None, nws=0):
    return _lib().rwkv7mi_process_logits(x, rows, n, ldx, dt, out, ldo, odt, hist, bits, ldh, cap, lengths, None, 2.0,
                                         None, 0.0, None, 0.0, None, 1.0, bias, ldb, allowed, lda, nxt, nxt2, append, ws,
                                         nws, None)


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(n=0), dict(ldx=-1), dict(ldo=50), dict(dt=5), dict(odt=2), dict(x=0),
                                dict(out=0), dict(bits=16), dict(hist=A, cap=-1), dict(hist=A, cap=(1 << 23) + 1),
                                dict(ldb=-1), dict(lda=-4), dict(nxt2=A), dict(rows=1 << 16),
                                dict(append=1), dict(append=1, hist=A, nxt=A), dict(append=1, hist=A, lengths=A),
                                dict(append=1, hist=A, lengths=A, nxt=A, ldh=0)])
def test_logits_entry_refuses(kw):
    assert _logits(**kw) == -1


def test_logits_entry_wants_its_workspace():
    need = _lib().rwkv7mi_process_logits_workspace_bytes(2, 100)
    assert need >= 16
    assert _logits(nxt=A) == -3 and _logits(nxt=A, ws=A, nws=need - 1) == -3 and _logits(nxt=A, ws=A + 4, nws=need) == -3


def test_cpu_tensors_are_refused():
    import rwkv7mi as mi

    x = torch.zeros(2, 64, dtype=torch.float16)
    c, s = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    for call in (lambda: mi.quantize_mxfp4(x), lambda: mi.dequantize_mxfp4(c, s), lambda: mi.mxfp4_linear(x, c, s),
                 lambda: mi.process_logits(x), lambda: mi.MXFP4Linear(torch.nn.Linear(64, 4))):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_python_refusals_before_any_device_work():
    import rwkv7mi as mi

    x = torch.zeros(2, 64, dtype=torch.float16)
    c, s = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    bad = [lambda: mi.quantize_mxfp4(torch.zeros(2, 40)), lambda: mi.quantize_mxfp4(torch.zeros(2, 64).int()),
           lambda: mi.quantize_mxfp4(torch.zeros(2, 0)), lambda: mi.dequantize_mxfp4(c, s[:2]),
           lambda: mi.dequantize_mxfp4(c.int(), s), lambda: mi.mxfp4_linear(x, c, s, epilogue="tanh"),
           lambda: mi.mxfp4_linear(x, c, s, epilogue="residual"), lambda: mi.mxfp4_linear(x, c, s, residual=x),
           lambda: mi.mxfp4_linear(x, c, s[:, :1]), lambda: mi.process_logits(x[0]),
           lambda: mi.MXFP4Linear(torch.nn.Linear(40, 4)), lambda: mi.MXFP4Linear.from_packed(c, s[:1])]
    for call in bad:
        with pytest.raises(ValueError):
            call()


def test_model_config_refusals():
    from rwkv7mi.model import NativeRWKV7Config, NativeRWKV7ForCausalLM

    def cfg(**kw):
        return NativeRWKV7Config(vocab_size=64, hidden_size=64, num_hidden_layers=1, use_native_mxfp4=True, **kw)

    with pytest.raises(ValueError, match="exclude each other"):
        NativeRWKV7ForCausalLM(cfg(use_native_mm8=True), device="cpu")
    with pytest.raises(ValueError, match="fp16 or bf16"):
        NativeRWKV7ForCausalLM(cfg(), device="cpu", dtype=torch.float32)
    back = NativeRWKV7Config(**{k: v for k, v in cfg(native_mxfp4_quantize_input=True).to_dict().items()
                                if k != "model_type"})
    assert back.use_native_mxfp4 and back.native_mxfp4_quantize_input


def test_prepacked_manifest_refusals():
    from rwkv7mi.converter import MXFP4_FORMAT, MXFP4_PACKER_VERSION, PACKER_VERSION, validate_manifest
    from rwkv7mi.model import NativeRWKV7Config

    cfg = NativeRWKV7Config(vocab_size=64, hidden_size=64, num_hidden_layers=1)
    entry = {"format": MXFP4_FORMAT, "module": "lm_head", "input_features": 64, "output_features": 64,
             "activation_dtype": "float16", "scale_dtype": "uint8", "blocked_shape": [64, 32],
             "packer_version": MXFP4_PACKER_VERSION}

    def check(dtype=torch.bfloat16, top=MXFP4_PACKER_VERSION, **kw):
        validate_manifest({"format": MXFP4_FORMAT, "packer_version": top, "modules": [{**entry, **kw}]}, cfg, dtype)

    check()
    check(torch.float16)
    for bad in (dict(dtype=torch.float32), dict(top=PACKER_VERSION), dict(blocked_shape=[64, 64]),
                dict(scale_dtype="float16"), dict(format="rwkv7mi.mm8_blocked.v1"), dict(input_features=32)):
        with pytest.raises(ValueError):
            check(**bad)


def test_fake_kernels_give_shapes():
    import rwkv7mi  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        codes, scales = torch.ops.rwkv7mi.quantize_mxfp4(torch.empty(7, 96, dtype=torch.float16))
        assert codes.shape == (7, 48) and scales.shape == (7, 3) and codes.dtype == scales.dtype == torch.uint8
        assert torch.ops.rwkv7mi.dequantize_mxfp4(codes, scales, torch.bfloat16).shape == (7, 96)
        y = torch.ops.rwkv7mi.mxfp4_linear(torch.empty(2, 5, 96, dtype=torch.float16), codes, scales, True)
        assert y.shape == (2, 5, 7)
        out, nxt = torch.ops.rwkv7mi.process_logits(y[0], None, None, 1.0, 0.0, 0.0, 1.0, None, None)
        assert out.shape == (5, 7) and nxt.shape == (5,) and nxt.dtype == torch.int64

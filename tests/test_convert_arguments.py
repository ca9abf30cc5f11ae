"""What the converter's entry accepts and refuses before it reads a checkpoint."""
from __future__ import annotations

import argparse

import pytest
import torch


def _args(tmp_path, **kw):
    base = dict(input=str(tmp_path / "missing.pth"), output=str(tmp_path / "out"), precision="fp16", low_memory=False,
                prepack_mm8=False, device="cpu")
    return argparse.Namespace(**{**base, **kw})


def test_arguments_of_a_caller_that_knows_no_mxfp4(tmp_path, monkeypatch):
    """``convert`` takes a Namespace without ``prepack_mxfp4``, as built before the option."""
    from rwkv7mi import converter
    from rwkv7mi.model import NativeRWKV7Config, parameter_shapes

    cfg = NativeRWKV7Config(vocab_size=64, hidden_size=64, num_hidden_layers=1, intermediate_size=128)
    state = {k: torch.zeros(s, dtype=torch.float16) for k, s in parameter_shapes(cfg).items()}
    monkeypatch.setattr(converter, "convert_state_dict", lambda weights, dtype: (cfg, state))
    torch.save({}, tmp_path / "model.pth")
    out = converter.convert(_args(tmp_path, input=str(tmp_path / "model.pth")))
    assert (out / "config.json").exists() and (out / "model.safetensors").exists()


def test_mxfp4_of_an_fp32_checkpoint_is_refused_before_anything_is_read(tmp_path):
    from rwkv7mi import converter

    with pytest.raises(ValueError, match="fp16 or bf16"):
        converter.convert(_args(tmp_path, precision="fp32", prepack_mxfp4=True))
    assert not (tmp_path / "out").exists()

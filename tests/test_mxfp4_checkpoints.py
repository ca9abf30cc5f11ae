"""Prepacked directories of models built from packs come back as the models that were saved
(built, saved and loaded on the CPU; no kernel runs)."""
from __future__ import annotations

import json

import pytest
import torch

import mx_reference as mx

RKVO, FFN = (20, 21, 22, 23), (38, 39)  # the projections' entries of a pack


def _pack_model(quantized, head=None):
    """A one-layer model over packs: ``quantized`` maps a projection's entry to its MXFP4
    module's quantize_input, ``head`` is the head's (None: a dense head)."""
    from rwkv7mi import MXFP4Linear
    from rwkv7mi.model import NativeRWKV7Config, NativeRWKV7ForCausalLM, random_weights

    cfg = NativeRWKV7Config(vocab_size=96, hidden_size=64, num_hidden_layers=1, intermediate_size=128,
                            decay_low_rank_dim=32, a_low_rank_dim=32, gate_low_rank_dim=32, v_low_rank_dim=32,
                            native_mxfp4_min_params=1)
    w = random_weights(cfg, seed=0, device="cpu", dtype=torch.float16)
    dense = NativeRWKV7ForCausalLM(cfg, w, device="cpu", dtype=torch.float16)
    packs, *_ = dense.extract_graph_packs()

    def module(weight, quantize_input):
        codes, scales = mx.quantize(weight)
        return MXFP4Linear.from_packed(mx.pack(codes), scales, quantize_input=quantize_input)

    pk = list(packs[0])
    for i, q in quantized.items():
        pk[i] = module(pk[i], q)
    lm = dense.lm_head.weight if head is None else module(dense.lm_head.weight, head)
    return NativeRWKV7ForCausalLM.from_graph_packs(cfg, [tuple(pk)], embeddings=dense.emb, norm_weight=dense.norm[0],
                                                   norm_bias=dense.norm[1], lm_head=lm, device="cpu")


def _load(path, **kw):
    from rwkv7mi.model import NativeRWKV7ForCausalLM

    return NativeRWKV7ForCausalLM.from_pretrained(path, device="cpu", **kw)


def _flags(model):
    from rwkv7mi.model import BlockFloatLinear

    return {n: lin.m.quantize_input for n, lin in model.named_linears() if isinstance(lin, BlockFloatLinear)}


def test_a_linear_saved_dense_stays_dense(tmp_path):
    """The head alone in MXFP4; the projections are large enough for the config's setting."""
    from rwkv7mi.model import DenseLinear

    model = _pack_model({}, head=True)
    model.save_pretrained(tmp_path)
    again = _load(tmp_path)
    assert list(_flags(again)) == ["lm_head"] and again._rwkv7_native_mm_replaced_modules == 1
    for (name, a), (_, b) in zip(model.named_linears(), again.named_linears()):
        if name != "lm_head":
            assert isinstance(b, DenseLinear) and torch.equal(a.weight, b.weight), name
        else:
            assert torch.equal(a.m.codes, b.m.codes) and torch.equal(a.m.scales, b.m.scales)


def test_every_module_keeps_its_quantize_input(tmp_path):
    model = _pack_model({**dict.fromkeys(RKVO, True), **dict.fromkeys(FFN, True)}, head=False)
    want = _flags(model)
    assert len(want) == 7 and not want["lm_head"] and sum(want.values()) == 6
    model.save_pretrained(tmp_path)
    assert _flags(_load(tmp_path)) == want
    assert set(_flags(_load(tmp_path, native_mxfp4_quantize_input=True)).values()) == {True}
    # a manifest without the entry: the config's setting for every module
    manifest = json.loads((tmp_path / "manifest.json").read_text())
    for e in manifest["modules"]:
        del e["quantize_input"]
    (tmp_path / "manifest.json").write_text(json.dumps(manifest))
    cj = json.loads((tmp_path / "config.json").read_text())
    for setting in (True, False):
        (tmp_path / "config.json").write_text(json.dumps({**cj, "native_mxfp4_quantize_input": setting}))
        assert set(_flags(_load(tmp_path)).values()) == {setting}


def test_a_manifest_entry_that_is_no_truth_value_is_refused(tmp_path):
    _pack_model({}, head=True).save_pretrained(tmp_path)
    manifest = json.loads((tmp_path / "manifest.json").read_text())
    manifest["modules"][0]["quantize_input"] = "yes"
    (tmp_path / "manifest.json").write_text(json.dumps(manifest))
    with pytest.raises(ValueError, match="quantize_input"):
        _load(tmp_path)


def test_a_prepacked_directory_is_not_taken_for_the_other_format(tmp_path):
    """Asked for the other quantisation by name or by a config, a prepacked directory is refused."""
    from rwkv7mi import converter as conv
    from rwkv7mi.model import NativeRWKV7Config

    _pack_model({}, head=True).save_pretrained(tmp_path)
    assert list(_flags(_load(tmp_path, use_native_mxfp4=True))) == ["lm_head"]
    with pytest.raises(ValueError, match="MXFP4"):
        _load(tmp_path, use_native_mm8=True)
    cfg = NativeRWKV7Config(vocab_size=96, hidden_size=64, num_hidden_layers=1, use_native_mm8=True)
    with pytest.raises(ValueError, match="MXFP4"):
        _load(tmp_path, config=cfg)
    manifest = {"format": conv.PREPACKED_FORMAT, "packer_version": conv.PACKER_VERSION, "modules": []}
    (tmp_path / "manifest.json").write_text(json.dumps(manifest))
    with pytest.raises(ValueError, match="MM8"):
        _load(tmp_path, use_native_mxfp4=True)


def test_the_directorys_own_config_keeps_each_modules_setting(tmp_path):
    """``AutoModelForCausalLM`` hands over the config it read from the directory; a config that
    says otherwise than the directory's is a setting for every module."""
    from rwkv7mi.model import NativeRWKV7Config

    model = _pack_model(dict.fromkeys(FFN, True), head=False)
    model.save_pretrained(tmp_path)
    own = NativeRWKV7Config.from_pretrained(tmp_path)
    assert own.use_native_mxfp4 and own.native_mxfp4_quantize_input
    assert _flags(_load(tmp_path, config=own)) == _flags(model)
    own.native_mxfp4_quantize_input = False
    assert set(_flags(_load(tmp_path, config=own)).values()) == {False}
    assert set(_flags(_load(tmp_path, config=own, native_mxfp4_quantize_input=True)).values()) == {True}

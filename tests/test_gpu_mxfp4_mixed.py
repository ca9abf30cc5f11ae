"""A model from packs that holds MM8, MXFP4 and dense projections at once, against the fp64
per-token oracle over the weights they stand for."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import mx_reference as mx

pytestmark = pytest.mark.gpu

LOGIT_REL = 2e-3  # of max|logit|, as the models of one format are held to


def _model():
    """R, K, V and O in MM8, the FFN's two in MXFP4, the head dense."""
    from oracle import oracle as o
    from oracle.model_oracle import ModelOracle
    from rwkv7mi import MM8Linear, MXFP4Linear, quantize_mxfp4
    from rwkv7mi.model import NativeRWKV7Config, NativeRWKV7ForCausalLM, random_weights

    cfg = NativeRWKV7Config(vocab_size=512, hidden_size=128, num_hidden_layers=2, intermediate_size=256,
                            decay_low_rank_dim=32, a_low_rank_dim=32, gate_low_rank_dim=64, v_low_rank_dim=32)
    w = random_weights(cfg, seed=0, device="cpu", dtype=torch.float16)
    dense = NativeRWKV7ForCausalLM(cfg, w, device="cuda", dtype=torch.float16)
    packs, *_ = dense.extract_graph_packs()
    override, mixed = {}, []
    for i, pk in enumerate(packs):
        pk = list(pk)
        for at, name in ((20, "attn.r_proj"), (21, "attn.k_proj"), (22, "attn.v_proj"), (23, "attn.o_proj")):
            lin = torch.nn.Linear(128, 128, bias=False, device="cuda", dtype=torch.float16)
            lin.weight.data.copy_(pk[at])
            m = pk[at] = MM8Linear(lin)
            override[f"model.layers.{i}.{name}"] = o.mm8_dequant(*(t.cpu().numpy() for t in (m.w_u8, m.mx, m.rx, m.my, m.ry)))
        for at, name in ((38, "ffn.key"), (39, "ffn.value")):
            codes, scales = quantize_mxfp4(pk[at])
            pk[at] = MXFP4Linear.from_packed(codes, scales)
            override[f"model.layers.{i}.{name}"] = mx.values(codes, scales).t().numpy()
        mixed.append(tuple(pk))
    model = NativeRWKV7ForCausalLM.from_graph_packs(cfg, mixed, embeddings=dense.emb, norm_weight=dense.norm[0],
                                                    norm_bias=dense.norm[1], lm_head=dense.lm_head.weight)
    return cfg, model, ModelOracle(cfg, {k: v.float().numpy() for k, v in w.items()}, override)


@pytest.mark.parametrize("B", [1, 3, 20])
def test_prefill_and_decode_match_the_oracle(B, tmp_path):
    cfg, model, ref = _model()
    assert model._rwkv7_native_mm_quantization == "mm8+mxfp4" and model._rwkv7_native_mm_replaced_modules == 12
    rng = np.random.default_rng(1)
    ids = rng.integers(0, cfg.vocab_size, (B, 37))
    want, st = ref.run(ids)
    out = model(torch.tensor(ids, device="cuda"))
    cache = out.past_key_values

    def close(got, ref):
        assert np.abs(got.double().cpu().numpy() - ref).max() <= LOGIT_REL * np.abs(ref).max()

    close(out.logits[:, -1], want[:, -1])
    runner, captured = model.graph_runner(B), cache.clone()
    for _ in range(3):
        nxt = rng.integers(0, cfg.vocab_size, (B,))
        r = ref.step(nxt, st)
        tok = torch.tensor(nxt, device="cuda")
        eager = model(tok[:, None], past_key_values=cache, use_graph=False).logits[:, -1]
        close(eager, r)
        assert torch.equal(runner.replay(tok, captured), eager)
    with pytest.raises(ValueError, match="both MM8 and MXFP4"):
        model.save_pretrained(tmp_path)

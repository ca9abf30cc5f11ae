"""Captured prefills of MXFP4 models: the scratch of their products comes from the graph's pool."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quantize_input,dtype", [(False, torch.float16), (False, torch.bfloat16), (True, torch.float16)])
@pytest.mark.parametrize("B,T", [(1, 16), (2, 64), (2, 304)])
def test_replays_equal_eager_prefills(B, T, quantize_input, dtype):
    """Two captured prompt shapes replayed in turn, eager work between them."""
    from rwkv7mi.model import NativeRWKV7Config, NativeRWKV7ForCausalLM, random_weights

    cfg = NativeRWKV7Config(vocab_size=512, hidden_size=512, num_hidden_layers=2, intermediate_size=2048,
                            decay_low_rank_dim=32, a_low_rank_dim=32, gate_low_rank_dim=64, v_low_rank_dim=32,
                            use_native_mxfp4=True, native_mxfp4_min_params=0, native_mxfp4_quantize_input=quantize_input)
    model = NativeRWKV7ForCausalLM(cfg, random_weights(cfg, seed=0, device="cpu", dtype=dtype), device="cuda", dtype=dtype)
    g = torch.Generator().manual_seed(T)
    runners = [(t, model.prefill_graph_runner(B, t, logits_to_keep=1, carry_state=False)) for t in (T, T + 32)]
    for _ in range(3):
        for t, runner in runners:
            ids = torch.randint(0, cfg.vocab_size, (B, t), generator=g).cuda()
            cache = model.new_cache(B)
            want = model.prefill_(ids, cache, logits_to_keep=1)
            got, state = runner.replay(ids)
            torch.cuda.synchronize()
            assert torch.equal(got, want)
            assert all(torch.equal(a, b) for a, b in zip(state._state, cache._state))

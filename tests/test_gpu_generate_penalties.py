"""Greedy generation under penalties given as one value per row."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _model():
    from rwkv7mi.model import NativeRWKV7Config, NativeRWKV7ForCausalLM, random_weights

    cfg = NativeRWKV7Config(vocab_size=512, hidden_size=128, num_hidden_layers=2, intermediate_size=256,
                            decay_low_rank_dim=32, a_low_rank_dim=32, gate_low_rank_dim=64, v_low_rank_dim=32)
    w = random_weights(cfg, seed=0, device="cpu", dtype=torch.float16)
    return NativeRWKV7ForCausalLM(cfg, w, device="cuda", dtype=torch.float16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_penalties_per_row_from_host_memory(dtype):
    """Penalties on the CPU are moved like the bias and the mask: each row as it goes by itself."""
    model = _model()
    ids = torch.randint(0, 512, (2, 9), generator=torch.Generator().manual_seed(3)).cuda()
    rows = dict(repetition_penalty=[1.3, 1.0], presence_penalty=[0.5, 2.0], frequency_penalty=[0.25, 0.0],
                penalty_decay=[0.9, 1.0])
    got = model.generate_greedy(ids, 16, **{k: torch.tensor(v, dtype=dtype) for k, v in rows.items()})
    on_gpu = model.generate_greedy(ids, 16, **{k: torch.tensor(v, dtype=dtype, device="cuda") for k, v in rows.items()})
    assert torch.equal(got, on_gpu)
    for b in range(2):
        alone = model.generate_greedy(ids, 16, **{k: v[b] for k, v in rows.items()})
        assert torch.equal(got[b], alone[b])

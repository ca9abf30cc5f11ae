"""MXFP4 projections and the logits step in the model: prefill, decode and graph decode
against the fp64 per-token oracle over the dequantised weights, greedy generation under
penalties against the formula in 64 bits, checkpoints, packs, custom ops.

The oracle's tolerance is that of the unquantised model's tests (2e-3 x max|logit|): the
weights' values are exact, the activations are fp16 as there.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import mx_reference as mx

pytestmark = pytest.mark.gpu

LOGIT_REL = 2e-3


def _cfg(quantize_input=False, **kw):
    from rwkv7mi.model import NativeRWKV7Config

    args = dict(vocab_size=512, hidden_size=128, num_hidden_layers=2, intermediate_size=256, decay_low_rank_dim=32,
                a_low_rank_dim=32, gate_low_rank_dim=64, v_low_rank_dim=32, use_native_mxfp4=True,
                native_mxfp4_min_params=0, native_mxfp4_quantize_input=quantize_input)
    return NativeRWKV7Config(**{**args, **kw})


def _model(quantize_input=False, dtype=torch.float16, seed=0, **kw):
    from rwkv7mi.model import NativeRWKV7ForCausalLM, random_weights

    cfg = _cfg(quantize_input, **kw)
    w = random_weights(cfg, seed=seed, device="cpu", dtype=dtype)
    return cfg, w, NativeRWKV7ForCausalLM(cfg, w, device="cuda", dtype=dtype)


@pytest.mark.parametrize("B", [1, 2, 20])
def test_prefill_then_decode_matches_oracle(B):
    from oracle.model_oracle import ModelOracle
    from rwkv7mi.model import BlockFloatLinear

    cfg, w, model = _model()
    assert model._rwkv7_native_mm_quantization == "mxfp4" and model._rwkv7_native_mm_replaced_modules == 13
    override = {}
    for name, lin in model.named_linears():
        assert isinstance(lin, BlockFloatLinear), name
        codes, scales = mx.quantize(w[name + ".weight"])
        assert torch.equal(lin.m.codes.cpu(), mx.pack(codes)) and torch.equal(lin.m.scales.cpu(), scales), name
        override[name] = mx.values(lin.m.codes, lin.m.scales).t().numpy()  # [in, out]
    ref = ModelOracle(cfg, {k: v.float().numpy() for k, v in w.items()}, override)
    rng = np.random.default_rng(1)
    ids = rng.integers(0, cfg.vocab_size, (B, 37))
    want, st = ref.run(ids)
    out = model(torch.tensor(ids, device="cuda"))
    cache = out.past_key_values

    def close(got, ref):
        got, scale = got.double().cpu().numpy(), np.abs(ref).max()
        assert np.abs(got - ref).max() <= LOGIT_REL * scale

    close(out.logits[:, -1], want[:, -1])
    for _ in range(4):
        nxt = rng.integers(0, cfg.vocab_size, (B,))
        r = ref.step(nxt, st)
        close(model(torch.tensor(nxt[:, None], device="cuda"), past_key_values=cache, use_graph=False).logits[:, -1], r)


@pytest.mark.parametrize("quantize_input,dtype", [(False, torch.float16), (True, torch.float16), (True, torch.bfloat16)])
@pytest.mark.parametrize("B", [3, 24])
def test_graph_decode_equals_eager_decode(B, quantize_input, dtype):
    cfg, _, model = _model(quantize_input, dtype)
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(0, cfg.vocab_size, (B, 9), generator=g).cuda()
    c1 = model(ids).past_key_values
    c2 = c1.clone()
    runner = model.graph_runner(B)
    for step in range(5):
        tok = torch.randint(0, cfg.vocab_size, (B,), generator=g).cuda()
        eager = model(tok[:, None], past_key_values=c1, use_graph=False).logits
        lg = runner.replay(tok, c2).clone()
        _ = torch.randn(64, device="cuda").sum()  # unrelated eager work between replays
        torch.cuda.synchronize()
        assert torch.equal(lg, eager[:, -1]), step


@pytest.mark.parametrize("rows", [5, 300])
def test_quantized_inputs_product_by_product(rows, monkeypatch):
    """Every projection of a prompt with quantised inputs against the 64-bit product of its
    own input, quantised as the format says."""
    from rwkv7mi.model import BlockFloatLinear

    cfg, _, model = _model(True)
    seen = []
    apply, group = BlockFloatLinear.apply, BlockFloatLinear.apply_group

    def rec_apply(self, x2, out, *, act=0, residual=None):
        before = None if residual is None else residual.clone()
        apply(self, x2, out, act=act, residual=residual)
        seen.append((self, x2.clone(), out.clone(), "relu2" if act == 3 else "residual" if residual is not None else "none",
                     before))
        return out

    def rec_group(lins, xs, outs):
        done = group(lins, xs, outs)
        assert done
        seen.extend((l, x.clone(), o.clone(), "none", None) for l, x, o in zip(lins, xs, outs))
        return done

    monkeypatch.setattr(BlockFloatLinear, "apply", rec_apply)
    monkeypatch.setattr(BlockFloatLinear, "apply_group", staticmethod(rec_group))
    model(torch.randint(0, cfg.vocab_size, (1, rows), device="cuda"))
    assert len(seen) == 13
    for lin, x, out, epilogue, residual in seen:
        codes, scales = mx.quantize(x)
        xq = mx.values(mx.pack(codes), scales)
        want, bound = mx.product(xq, mx.values(lin.m.codes, lin.m.scales), residual=residual, epilogue=epilogue)
        slack = bound + (want.abs() + bound) * torch.finfo(out.dtype).eps / 2 + 2.0 ** -25  # (fp16's last half step)
        assert bool(((out.cpu().double() - want).abs() <= slack).all()), (lin.out_features, epilogue)


def _processed(logits, ids, pen, bias, bits):
    """The scores of one row in 64 bits, by the formula."""
    rep, pres, freq, decay = pen
    s = logits.double().cpu().numpy().copy()
    count = np.zeros(s.shape[0])
    for k, t in enumerate(reversed(ids)):
        count[t] += decay ** k
    for t in set(ids):
        s[t] = (s[t] / rep if s[t] > 0 else s[t] * rep) - pres - freq * count[t]
    s += bias
    s[~bits] = -np.inf
    return s


@pytest.mark.parametrize("B,quantize_input", [(1, False), (3, True)])
def test_generate_under_penalties_bias_and_mask(B, quantize_input):
    cfg, _, model = _model(quantize_input)
    V, T, new = cfg.vocab_size, 11, 24
    rng = np.random.default_rng(5)
    ids = torch.tensor(rng.integers(0, V, (B, T)), device="cuda")
    pen = (1.3, 0.4, 0.25, 0.95)
    bias = rng.normal(0, 0.5, V).astype(np.float32)
    bits = rng.random(V) < 0.7
    words = torch.from_numpy(np.packbits(bits, bitorder="little").view(np.int32).copy())
    how = dict(repetition_penalty=pen[0], presence_penalty=pen[1], frequency_penalty=pen[2], penalty_decay=pen[3],
               bias=torch.from_numpy(bias), allowed=words)
    out = model.generate_greedy(ids, new, **how)
    assert out.shape == (B, T + new) and torch.equal(out[:, :T], ids)
    assert torch.equal(out, model.generate_greedy(ids, new, use_graph=False, **how))
    # each token has the formula's largest score, to fp32: the terms are below 2^6 in
    # magnitude and go through six roundings, 24 entries of a count through as many
    fed = model(ids)
    cache, logits = fed.past_key_values, fed.logits[:, -1]
    for t in range(new):
        for b in range(B):
            s = _processed(logits[b], out[b, :T + t].tolist(), pen, bias, bits)
            tok = int(out[b, T + t])
            assert bits[tok] and s[tok] >= s.max() - 2 * (6 + 35) * 64 * 2.0 ** -24, (t, b)
        logits = model(out[:, T + t, None], past_key_values=cache, use_graph=False).logits[:, -1]


def test_generate_with_neutral_settings_and_without_repeats():
    cfg, _, model = _model()
    ids = torch.randint(0, cfg.vocab_size, (2, 7), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    plain = model.generate_greedy(ids, 12)
    neutral = torch.zeros(cfg.vocab_size, device="cuda")
    assert torch.equal(plain, model.generate_greedy(ids, 12, bias=neutral))
    once = model.generate_greedy(ids, 12, presence_penalty=1e4)
    assert all(len(set(r)) == len(r) - (7 - len(set(r[:7]))) for r in once.tolist())
    assert model.generate_greedy(ids, 1, presence_penalty=1e4).shape == (2, 8)


def test_hugging_face_generate_with_the_processor():
    from rwkv7mi import NativeLogitsProcessor

    cfg, _, model = _model()
    g = torch.Generator().manual_seed(9)
    ids = torch.randint(0, cfg.vocab_size, (2, 9), generator=g).cuda()
    bias = torch.randn(cfg.vocab_size, generator=g).cuda()  # (no two scores alike)
    how = dict(repetition_penalty=1.2, presence_penalty=0.3, frequency_penalty=0.1, penalty_decay=0.9, bias=bias)
    want = model.generate_greedy(ids, 10, **how)
    got = model.generate(ids, max_new_tokens=10, do_sample=False, eos_token_id=None,
                         logits_processor=[NativeLogitsProcessor(**how)])
    assert torch.equal(got, want)
    # a mask that follows the text: no token twice in a row's generated part
    def fresh(so_far):
        bits = torch.ones(so_far.shape[0], 512, dtype=torch.int64)
        bits.scatter_(1, so_far[:, 9:].cpu(), 0)
        words = (bits.reshape(so_far.shape[0], 16, 32) << torch.arange(32)).sum(-1)
        return words.to(torch.int32).to(so_far.device)

    got = model.generate(ids, max_new_tokens=10, do_sample=False, eos_token_id=None,
                         logits_processor=[NativeLogitsProcessor(allowed=fresh)])
    assert all(len(set(r)) == 10 for r in got[:, 9:].tolist())
    # the prompt left out of the history
    only_new = NativeLogitsProcessor(presence_penalty=5.0, prompt_ignore_length=9)
    scores = torch.randn(2, 512, device="cuda")
    assert torch.equal(only_new(ids, scores), scores)


def test_prepacked_round_trip(tmp_path):
    from rwkv7mi.model import NativeRWKV7ForCausalLM

    cfg, _, model = _model(True)
    ids = torch.randint(0, cfg.vocab_size, (2, 21), device="cuda")
    want = model(ids).logits
    model.save_pretrained(tmp_path)
    again = NativeRWKV7ForCausalLM.from_pretrained(tmp_path)
    assert again._rwkv7_native_mm_quantization == "mxfp4" and again.lm_head.m.quantize_input
    assert torch.equal(again(ids).logits, want)
    plain = NativeRWKV7ForCausalLM.from_pretrained(tmp_path, native_mxfp4_quantize_input=False)
    assert not plain.lm_head.m.quantize_input and torch.equal(plain.lm_head.m.codes, model.lm_head.m.codes)
    assert NativeRWKV7ForCausalLM.from_pretrained(tmp_path, dtype=torch.bfloat16)(ids).logits.dtype == torch.bfloat16
    with pytest.raises(ValueError, match="MXFP4"):
        NativeRWKV7ForCausalLM.from_pretrained(tmp_path, dtype=torch.float32)


def test_head_only_policy_and_packs():
    from rwkv7mi.model import BlockFloatLinear, DenseLinear, NativeRWKV7ForCausalLM

    cfg, _, model = _model(native_mxfp4_policy="speed")
    assert isinstance(model.lm_head, BlockFloatLinear)
    assert all(isinstance(lin, DenseLinear) for name, lin in model.named_linears() if name != "lm_head")
    cfg, _, model = _model()
    packs, *_ = model.extract_graph_packs()
    twin = NativeRWKV7ForCausalLM.from_graph_packs(cfg, packs, embeddings=model.emb, norm_weight=model.norm[0],
                                                   norm_bias=model.norm[1], lm_head=model.lm_head.m)
    ids = torch.randint(0, cfg.vocab_size, (2, 5), device="cuda")
    assert torch.equal(twin(ids).logits, model(ids).logits)


def test_head_to_token_in_a_graph():
    """The serving step's end as one graph: the 4-bit head, the scores, the token, the
    history; four replays with eager work between them against the same calls made eagerly."""
    import rwkv7mi

    g = torch.Generator().manual_seed(4)
    B, D, V = 4, 256, 1003
    codes, scales = rwkv7mi.quantize_mxfp4(torch.randn(V, D, generator=g).half().cuda())
    hidden = torch.empty(B, D, device="cuda", dtype=torch.float16)
    words = torch.randint(-2 ** 31, 2 ** 31, ((V + 31) // 32,), generator=g).to(torch.int32).cuda()

    def state():
        return (torch.arange(20, device="cuda").expand(B, 20).contiguous(),
                torch.full((B,), 10, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.long, device="cuda"))

    def step(hist, lengths, nxt):
        logits = rwkv7mi.mxfp4_linear(hidden, codes, scales)
        return rwkv7mi.process_logits(logits, history=hist, lengths=lengths, repetition_penalty=1.2,
                                      frequency_penalty=0.2, penalty_decay=0.99, allowed=words, next_tokens=nxt,
                                      append=True)

    captured, eager = state(), state()
    hidden.copy_(torch.randn(B, D, generator=g).half())
    step(*state())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*captured)
    for _ in range(4):
        hidden.copy_(torch.randn(B, D, generator=g).half())
        graph.replay()
        want = step(*eager)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert all(torch.equal(a, b) for a, b in zip(captured, eager))
    assert captured[1].tolist() == [14] * B


def test_custom_ops_give_the_functions_results():
    import rwkv7mi

    g = torch.Generator().manual_seed(6)
    w, x = torch.randn(96, 64, generator=g).half().cuda(), torch.randn(3, 64, generator=g).half().cuda()
    ops = torch.ops.rwkv7mi
    codes, scales = ops.quantize_mxfp4(w)
    want = rwkv7mi.quantize_mxfp4(w)
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])
    assert torch.equal(ops.dequantize_mxfp4(codes, scales, torch.float32),
                       rwkv7mi.dequantize_mxfp4(codes, scales, out_dtype=torch.float32))
    for q in (False, True):
        assert torch.equal(ops.mxfp4_linear(x, codes, scales, q), rwkv7mi.mxfp4_linear(x, codes, scales, quantize_input=q))
    hist = torch.randint(0, 96, (3, 8), generator=g).cuda()
    y, nxt = ops.process_logits(rwkv7mi.mxfp4_linear(x, codes, scales), hist, None, 1.5, 0.1, 0.1, 1.0, None, None)
    assert torch.equal(nxt, rwkv7mi.argmax_rows(y))


def test_grouped_outputs_must_not_overlap():
    from rwkv7mi.native_quant_mxfp4 import mxfp4_linear_multi_into

    x = torch.zeros(2, 64, dtype=torch.float16, device="cuda")
    w = (torch.zeros(32, 32, dtype=torch.uint8, device="cuda"), torch.zeros(32, 2, dtype=torch.uint8, device="cuda"))
    o = torch.zeros(2, 32, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="another product"):
        mxfp4_linear_multi_into([x, x], [w, w], [o, o])
    with pytest.raises(ValueError, match="another product"):
        mxfp4_linear_multi_into([x, x], [w, w], [o, torch.zeros_like(o)], residuals=[None, o])


def test_settings_from_a_config_and_a_model_with_nothing_replaced(tmp_path):
    from rwkv7mi.converter import save_hf_directory, save_prepacked
    from rwkv7mi.model import BlockFloatLinear, NativeRWKV7ForCausalLM

    cfg, w, model = _model(native_mxfp4_min_params=10 ** 9)
    assert model._rwkv7_native_mm_quantization is None
    plain = tmp_path / "plain"
    save_hf_directory(plain, cfg, w)
    head = _cfg(True, native_mxfp4_policy="head")
    m = NativeRWKV7ForCausalLM.from_pretrained(plain, config=head)
    assert [n for n, lin in m.named_linears() if isinstance(lin, BlockFloatLinear)] == ["lm_head"]
    assert m.lm_head.m.quantize_input
    m = NativeRWKV7ForCausalLM.from_pretrained(plain, use_native_mxfp4=True, native_mxfp4_min_params=0)
    assert all(isinstance(lin, BlockFloatLinear) for _, lin in m.named_linears())
    empty = tmp_path / "empty"
    assert save_prepacked(model, empty)["modules"] == []
    again = NativeRWKV7ForCausalLM.from_pretrained(empty)
    assert again.config.use_native_mxfp4 and not again.config.use_native_mm8
    ids = torch.randint(0, cfg.vocab_size, (1, 5), device="cuda")
    assert torch.equal(again(ids).logits, model(ids).logits)

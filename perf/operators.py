"""Performance cases of the microscaled 4-bit linears and of the logits step.

Four operators, each as a serving program calls it:

* ``quantize``: values to MXFP4 (32-value blocks of e2m1 codes with a
  power-of-two scale) and back, as the values the codes stand for;
* ``linear``: 16-bit activations times an MXFP4 weight;
* ``linear4``: the same with the activations quantised to MXFP4 on the way;
* ``logits``: penalties for repeated tokens, biases and a grammar mask on a
  step's logits, with the greedy token.

``listed()`` gives the fixed cases, ``draw(rng)`` one more of the same ranges,
``prepare`` the inputs, ``run`` one pass (``own`` False: plain torch in 32
bits; True: this package's kernels), ``exact`` the pass in 64 bits, ``work``
the bytes and operations that a pass cannot do without.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
VOCAB = 65536
BLOCK = 32  # values of one scale


def _own():
    """This package's entry points (imported only where they are measured)."""
    path = str(Path.cwd() / "hf-adapter_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import rwkv7mi

    return rwkv7mi


# ------------------------------------------------------------------ the cases
def _quantize(name, rows, width, dtype):
    return {"name": name, "kind": "quantize", "rows": rows, "width": width, "dtype": dtype}


def _linear(name, kind, rows, inputs, outputs, dtype, epilogue="none"):
    return {"name": name, "kind": kind, "rows": rows, "inputs": inputs, "outputs": outputs, "dtype": dtype,
            "epilogue": epilogue}


def _logits(name, rows, vocab, history, dtype, bias, mask, decay):
    return {"name": name, "kind": "logits", "rows": rows, "vocab": vocab, "history": history, "dtype": dtype,
            "bias": bias, "mask": mask, "decay": decay}


def listed():
    return [
        # A feed-forward weight of the 7.2B width on its way to 4 bits, when a model is loaded.
        _quantize("quantize_weight_16384", 16384, 4096, "fp16"),
        # The rows of an ordinary prompt, as an input-quantising linear needs them.
        _quantize("quantize_prompt_1000", 1000, 2560, "bf16"),
        # A few rows of an odd number of blocks: latency.
        _quantize("quantize_few_37", 37, 1056, "fp16"),
        # One token of a single chat through the 7.2B feed-forward key: the
        # weight stream and the launch.
        _linear("linear_key_decode_1", "linear", 1, 4096, 16384, "fp16", "relu2"),
        # The vocabulary head with 8 chats decoding together.
        _linear("linear_head_decode_8", "linear", 8, 4096, VOCAB, "fp16"),
        # 40 chats through the 1.5B feed-forward value with its residual, bf16.
        _linear("linear_value_decode_40", "linear", 40, 8192, 2048, "bf16", "residual"),
        # A prompt of 1000 tokens through the 7.2B key.
        _linear("linear_key_prompt_1000", "linear", 1000, 4096, 16384, "fp16", "relu2"),
        # A prefill batch of 4 x 4096 tokens through the 7.2B key: the largest product.
        _linear("linear_key_batch_16384", "linear", 16384, 4096, 16384, "fp16", "relu2"),
        # A ragged prompt through the 2.9B key with 4-bit activations.
        _linear("linear4_key_prompt_300", "linear4", 300, 2560, 10240, "bf16", "relu2"),
        # The prefill batch with 4-bit activations.
        _linear("linear4_key_batch_16384", "linear4", 16384, 4096, 16384, "fp16", "relu2"),
        # One chat's next token after 500 tokens, greedy with penalties: latency.
        _logits("logits_chat_1", 1, VOCAB, 500, "fp16", False, False, 1.0),
        # 64 chats with long histories, decaying penalties, a shared bias and a grammar each.
        _logits("logits_batch_64", 64, VOCAB, 4000, "fp16", True, True, 0.996),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "linear", "linear4", "linear4", "logits", "logits"])
    if kind == "quantize":
        while True:
            rows, width = _log_int(rng, 1, 16384), BLOCK * _log_int(rng, 1, 512)
            if rows * width <= 16384 * 4096:
                return {"kind": kind, "rows": rows, "width": width, "dtype": rng.choice(["fp16", "bf16", "fp32"])}
    if kind == "logits":
        rows = _log_int(rng, 1, 64)
        vocab = VOCAB if rng.random() < 0.5 else _log_int(rng, 1000, VOCAB)
        return {"kind": kind, "rows": rows, "vocab": vocab, "history": _log_int(rng, 1, 4000),
                "dtype": rng.choice(["fp16", "fp16", "bf16", "fp32"]), "bias": rng.random() < 0.5,
                "mask": rng.random() < 0.5, "decay": rng.choice([1.0, 1.0, 0.996, 0.9])}
    hidden = rng.choice([2048, 2560, 4096])
    n, m = rng.choice([(hidden, hidden), (hidden, 4 * hidden), (4 * hidden, hidden), (4096, VOCAB),
                       (BLOCK * rng.randint(4, 300), rng.randint(16, 9000))])
    # only last tokens reach the vocabulary head: decode rows
    rows = _log_int(rng, 1, 64 if m == VOCAB else 8000)
    return {"kind": kind, "rows": rows, "inputs": n, "outputs": m, "dtype": rng.choice(["fp16", "fp16", "bf16"]),
            "epilogue": rng.choice(["none", "relu2", "residual"])}


# ------------------------------------------------------------------ inputs
def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFF)
    return g


def _randn(gen, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)


def _activations(gen, rows, width, dtype):
    """Normalised rows with a few channels that run large, as hidden states have."""
    gain = torch.where(torch.rand(width, generator=gen, device=DEV) < 0.01, 8.0, 1.0)
    return (torch.randn(rows, width, generator=gen, device=DEV) * gain).to(dtype)


def _mx_weight(gen, outputs, inputs):
    """``N(0, 0.02)`` quantised to MXFP4: ``(codes [O, I/2], scales [O, I/32])``."""
    codes = torch.empty(outputs, inputs // 2, device=DEV, dtype=torch.uint8)
    scales = torch.empty(outputs, inputs // BLOCK, device=DEV, dtype=torch.uint8)
    for r in range(0, outputs, 8192):
        c, s = _mx_codes(_randn(gen, min(8192, outputs - r), inputs, scale=0.02))
        codes[r:r + 8192] = c[:, 0::2] | (c[:, 1::2] << 4)
        scales[r:r + 8192] = s
    return codes, scales


def prepare(case, seed):
    g = _gen(seed, 1)
    if case["kind"] == "quantize":
        return {"kind": "quantize", "x": _activations(g, case["rows"], case["width"], DTYPES[case["dtype"]])}
    if case["kind"] == "logits":
        return _prepare_logits(case, g)
    dt, rows, n, m = DTYPES[case["dtype"]], case["rows"], case["inputs"], case["outputs"]
    codes, scales = _mx_weight(g, m, n)
    return {"kind": case["kind"], "x": _activations(g, rows, n, dt), "codes": codes, "scales": scales,
            "epilogue": case["epilogue"],
            "residual": _randn(g, rows, m, dtype=dt) if case["epilogue"] == "residual" else None}


def _prepare_logits(case, g):
    rows, vocab, cap = case["rows"], case["vocab"], case["history"]
    st = {"kind": "logits", "decay": case["decay"], "bias": None, "allowed": None,
          "logits": _randn(g, rows, vocab, scale=3.0, dtype=DTYPES[case["dtype"]])}
    # a skewed vocabulary, so that tokens repeat; entries past a row's length are unused
    u = torch.rand(rows, cap, generator=g, device=DEV)
    st["history"] = (u.pow(4) * vocab).long().clamp_(max=vocab - 1)
    lengths = (torch.rand(rows, generator=g, device=DEV) * (cap + 1)).long().clamp_(max=cap)
    lengths[0] = cap
    if rows > 2:
        lengths[1] = 0  # a chat that has just begun
    st["lengths"] = lengths.to(torch.int32)
    st["repetition"] = 1.0 + 0.5 * torch.rand(rows, generator=g, device=DEV)
    st["presence"] = 0.6 * torch.rand(rows, generator=g, device=DEV)
    st["frequency"] = 0.4 * torch.rand(rows, generator=g, device=DEV)
    if case["bias"]:  # the same few tokens pushed up or down for every chat
        hit = torch.rand(vocab, generator=g, device=DEV) < 0.01
        st["bias"] = torch.where(hit, 4.0 * torch.randn(vocab, generator=g, device=DEV), 0.0)
    if case["mask"]:
        # grammars from free text to a few dozen tokens; one finished row allows nothing
        share = torch.tensor([1.0, 0.3, 0.001], device=DEV)[torch.arange(rows, device=DEV) % 3]
        if rows >= 8:
            share[5] = 0.0
        words = (vocab + 31) // 32
        bits = (torch.rand(rows, words * 32, generator=g, device=DEV) < share[:, None]).view(rows, words, 32)
        value = (bits.long() << torch.arange(32, device=DEV)).sum(-1)
        st["allowed"] = torch.where(value >= 2 ** 31, value - 2 ** 32, value).to(torch.int32)
    return st


# ------------------------------------------------------------------ the pass
def run(state):
    kind = state["kind"]
    if kind == "logits":
        return _run_logits(state)
    if kind == "quantize":
        return _run_quantize(state)
    return _run_linear(state)


def _run_quantize(st):
    x = st["x"]
    if own:
        mi = _own()
        return mi.dequantize_mxfp4(*mi.quantize_mxfp4(x), out_dtype=x.dtype)
    return _mx_values(*_mx_codes(x.float())).to(x.dtype)


def _run_linear(st):
    if own:
        return _own().mxfp4_linear(st["x"], st["codes"], st["scales"], epilogue=st["epilogue"],
                                   residual=st["residual"], quantize_input=st["kind"] == "linear4")
    x = st["x"].float()
    if st["kind"] == "linear4":
        x = _mx_values(*_mx_codes(x))
    c = st["codes"]
    w = _mx_values(torch.stack((c & 15, c >> 4), -1).reshape(c.shape[0], -1), st["scales"])
    y = x @ w.t()
    if st["epilogue"] == "relu2":
        y = torch.relu(y).square()
    elif st["epilogue"] == "residual":
        y = y + st["residual"].float()
    return y.to(st["x"].dtype)


def _run_logits(st):
    x = st["logits"]
    if own:
        nxt = torch.empty(x.shape[0], device=x.device, dtype=torch.int64)
        out = _own().process_logits(x, history=st["history"], lengths=st["lengths"],
                                    repetition_penalty=st["repetition"], presence_penalty=st["presence"],
                                    frequency_penalty=st["frequency"], penalty_decay=st["decay"], bias=st["bias"],
                                    allowed=st["allowed"], next_tokens=nxt)
        return [out, nxt]
    rows, vocab = x.shape
    h, n = st["history"], st["lengths"].long()
    pos = torch.arange(h.shape[1], device=x.device)
    used = pos < n[:, None]
    age = (n[:, None] - 1 - pos).clamp(min=0)
    weight = torch.where(used, torch.pow(torch.tensor(st["decay"], dtype=torch.float64, device=x.device), age), 0.0)
    count = torch.zeros(rows, vocab, dtype=torch.float64, device=x.device).scatter_add_(1, h, weight).float()
    seen = torch.zeros(rows, vocab, dtype=torch.int32, device=x.device).scatter_add_(1, h, used.int()) > 0
    y = x.float()
    theta = st["repetition"][:, None]
    cut = torch.where(y > 0, y / theta, y * theta) - (st["presence"][:, None] + st["frequency"][:, None] * count)
    y = torch.where(seen, cut, y)
    if st["bias"] is not None:
        y = y + st["bias"]
    if st["allowed"] is not None:
        i = torch.arange(vocab, device=x.device)
        y = torch.where((st["allowed"][:, i >> 5] >> (i & 31)) & 1 != 0, y, -math.inf)
    y = y.to(x.dtype)
    first = torch.where(y == y.max(-1, keepdim=True).values, torch.arange(vocab, device=x.device), vocab)
    return [y, first.min(-1).values]


# ------------------------------------------------------------------ MXFP4 in plain torch
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _mx_codes(x):
    """``x [rows, width]`` (fp32) -> codes ``[rows, width]`` (one a byte) and
    scales ``[rows, width / 32]``, finite values: the block's scale is
    ``2^(floor(log2 amax) - 2)``, the codes round to nearest, ties to even,
    and stop at 6."""
    b = x.view(x.shape[0], -1, BLOCK)
    amax = b.abs().amax(-1)
    exponent = torch.frexp(amax).exponent.int() + (127 - 1 - 2)
    scales = torch.where(amax > 0, exponent.clamp(0, 254), 0)
    v = torch.ldexp(b, 127 - scales[..., None])
    a = v.abs()
    code = torch.zeros_like(a, dtype=torch.uint8)
    # halfway points: the tie goes to the even code, the lower one where it is even
    for i, mid in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
        code += (a > mid) if i % 2 == 0 else (a >= mid)
    code = torch.where(v < 0, code + 8, code)
    return code.view(x.shape), scales.to(torch.uint8)


def _mx_values(codes, scales):
    """The fp32 values of one-a-byte codes (scale bytes below 255)."""
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=codes.device)
    v = table[codes.int()].view(codes.shape[0], -1, BLOCK)
    return torch.ldexp(v, scales.int()[..., None] - 127).view(codes.shape)


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "quantize":
        return _exact_mx(st["x"])
    if case["kind"] == "logits":
        return _exact_logits(st)
    x = _exact_mx(st["x"]) if case["kind"] == "linear4" else st["x"].double()
    y = torch.empty(x.shape[0], case["outputs"], dtype=torch.float64, device=DEV)
    for r in range(0, case["outputs"], 8192):
        y[:, r:r + 8192] = x @ _exact_weight(st["codes"][r:r + 8192], st["scales"][r:r + 8192]).t().contiguous()
    if case["epilogue"] == "relu2":
        y = y.clamp(min=0) ** 2
    elif case["epilogue"] == "residual":
        y += st["residual"].double()
    return y


def _exact_mx(x):
    """Rounded to the block's grid: steps of half a unit below 2, of one below
    4, of two above, in units of the power of two two octaves under the block's
    largest value."""
    b = x.double().view(x.shape[0], -1, BLOCK)
    top = b.abs().amax(-1, keepdim=True)
    unit = torch.exp2(torch.floor(torch.log2(top.clamp(min=1e-300))).clamp(min=-125) - 2)
    v = b / unit
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0))
    v = (torch.round(v / step) * step).clamp(-6, 6) * unit
    return v.view(x.shape)


def _exact_weight(codes, scales):
    c = torch.stack((codes & 15, codes >> 4), -1).view(codes.shape[0], -1).int()
    e, m = (c >> 1) & 3, (c & 1).double()
    v = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2((e - 1).double())) * (1 - 2 * (c >> 3))
    v = v.view(codes.shape[0], -1, BLOCK) * torch.exp2(scales.double() - 127)[..., None]
    return v.view(codes.shape[0], -1)


def _exact_logits(st):
    x = st["logits"]
    y = x.double().cpu().numpy()
    hist, lengths = st["history"].cpu().numpy(), st["lengths"].cpu().numpy()
    row = {k: st[k].double().cpu().numpy() for k in ("repetition", "presence", "frequency")}
    for r in range(y.shape[0]):
        tokens = hist[r, :lengths[r]]
        weight = np.power(np.float64(st["decay"]), np.arange(len(tokens))[::-1])
        ids, where = np.unique(tokens, return_inverse=True)
        v = y[r, ids]
        v = np.where(v > 0, v / row["repetition"][r], v * row["repetition"][r])
        y[r, ids] = v - row["presence"][r] - row["frequency"][r] * np.bincount(where, weight, len(ids))
    if st["bias"] is not None:
        y += st["bias"].double().cpu().numpy()
    if st["allowed"] is not None:
        words = np.ascontiguousarray(st["allowed"].cpu().numpy())
        bits = np.unpackbits(words.view(np.uint8), axis=1, bitorder="little")[:, :y.shape[1]]
        y[bits == 0] = -np.inf
    y = torch.from_numpy(y)
    rounded = y.to(x.dtype).double().numpy()
    return [y, torch.from_numpy(np.argmax(rounded, axis=1))]  # (the first of the largest)


# ------------------------------------------------------------------ the least work
def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "quantize":
        n = case["rows"] * case["width"]
        return {"bytes": 2 * es * n, "flops": 4 * n}
    if case["kind"] == "logits":
        n = case["rows"] * case["vocab"]
        b = 2 * es * n + case["rows"] * (8 * case["history"] + 24)
        b += 4 * case["vocab"] if case["bias"] else 0
        b += n / 8 if case["mask"] else 0
        return {"bytes": b, "flops": 4 * n}
    rows, n, m = case["rows"], case["inputs"], case["outputs"]
    b = m * (n / 2 + n / BLOCK) + es * rows * (n + m * (2 if case["epilogue"] == "residual" else 1))
    return {"bytes": b, "flops": 2 * rows * n * m}

"""Log probabilities and 4-bit group-scaled weights: the calls whose speed is measured, and their plain forms.

Three operators that a serving or scoring program uses together:

``int4``      y = x @ W^T (+ bias) for W in 4-bit codes with a scale, and optionally a zero
              point, for each group of 32, 64 or 128 weights along a row (``quantized_linear`` of
              ``QuantizedWeight.from_int4_groups``).
``logprobs``  for each row of logits the log probability of a given token, the entropy of the
              distribution, the token's rank and the most likely alternatives
              (``token_logprobs``).
``head``      the same numbers straight from the hidden states, through an LM head of such
              weights (``linear_logprobs``).

``listed`` gives the fixed cases, ``draw`` further ones of the same ranges, ``prepare`` the
weights and inputs, ``run`` one pass (plain torch in 32 bits, or with ``own`` the library's
calls), ``work`` the bytes and operations a pass cannot do without, ``exact`` its result in 64
bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def int4(m, n, k, group, zeros=True, scale="f16", x="bf16", out="bf16", bias=False):
    return {"kind": "int4", "m": m, "n": n, "k": k, "group": group, "zeros": zeros, "scale": scale, "x": x,
            "out": out, "bias": bias}


def logprobs(m, vocab, dtype="f32", top=0, ranks=False, masked=False):
    return {"kind": "logprobs", "m": m, "vocab": vocab, "dtype": dtype, "top": top, "ranks": ranks, "masked": masked}


def head(m, vocab, k, group, zeros=True, scale="f16", x="bf16", top=0):
    return {"kind": "head", "m": m, "n": vocab, "k": k, "group": group, "zeros": zeros, "scale": scale, "x": x,
            "top": top}


def listed():
    cases = {
        # one token through an attention projection, f32 activations as the linear's default: the
        # smallest call, where latency counts
        "int4_decode_projection": int4(1, 4096, 4096, 128, zeros=False, x="f32", out="f32"),
        # one token through the fused gate | up projection: most of a decode step's bytes
        "int4_decode_gate_up": int4(1, 24576, 4096, 128),
        # five speculated tokens, short groups, a K that ends inside a 64-wide step, an odd number of rows
        "int4_batch5_odd": int4(5, 5751, 2880, 32, x="f32", out="f32", bias=True),
        # a served batch of a dozen sequences through the down projection
        "int4_batch12_down": int4(12, 4096, 12288, 64, scale="bf16", bias=True),
        # a prompt of odd length with f32 activations, symmetric codes
        "int4_prefill203_f32": int4(203, 4096, 12288, 128, zeros=False, x="f32", out="f32"),
        # a prompt of 512 tokens through the up projection
        "int4_prefill512": int4(512, 12288, 4096, 128),
        # the token just sampled in one sequence, with the twenty alternatives that an API returns
        "logprobs_decode_top20": logprobs(1, 151936, top=20, ranks=True),
        # a served batch under a grammar's mask, logits in bf16 (ties among the best are common)
        "logprobs_batch48_bf16": logprobs(48, 50257, dtype="bf16", top=5, ranks=True, masked=True),
        # a prompt's tokens scored with five alternatives each
        "logprobs_prompt301_top5": logprobs(301, 151936, top=5, ranks=True),
        # a long prompt for its perplexity: log probability and entropy only
        "logprobs_prompt512": logprobs(512, 151936),
        # one decode step's answer: 4-bit LM head, the token's log probability and alternatives
        "head_decode_top5": head(1, 151936, 4096, 128, top=5),
        # a prompt scored through the LM head
        "head_prompt300": head(300, 151936, 4096, 128),
    }
    return [dict(name=name, **case) for name, case in cases.items()]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("int4", "int4", "int4", "logprobs", "logprobs", "head"))
    group, zeros, scale = rng.choice((32, 64, 128, 128)), rng.random() < 0.6, rng.choice(("f16", "f16", "bf16"))
    x = rng.choice(("bf16", "bf16", "f32"))
    if kind == "int4":
        k = group * _log_uniform(rng, 512 // group, 12288 // group)
        n = _log_uniform(rng, 256, 24576)
        if rng.random() < 0.6:
            n = (n + 127) // 128 * 128  # models' widths; the rest any number of rows
        n = min(n, 100000000 // k)
        m = min(_log_uniform(rng, 1, 640), int(5e10 / (2 * n * k)))
        return int4(m, n, k, group, zeros, scale, x, rng.choice(("bf16", "f32")), rng.random() < 0.3)
    if kind == "logprobs":
        vocab = _log_uniform(rng, 1000, 151936)
        m = min(_log_uniform(rng, 1, 2048), 512 * 151936 // vocab)
        return logprobs(m, vocab, rng.choice(("f32", "f32", "bf16", "f16")), rng.choice((0, 1, 5, 20, 20)),
                        rng.random() < 0.6, rng.random() < 0.3)
    k = group * _log_uniform(rng, 512 // group, 4096 // group)
    m = _log_uniform(rng, 1, 300)
    return head(m, _log_uniform(rng, 8000, 151936), k, group, zeros, scale, x, rng.choice((0, 5)) if m <= 8 else 0)


# ---- inputs --------------------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _activations(g, m, k, dtype):
    """N(0, 1) tokens whose channels differ in size, as a model's hidden states do."""
    channel = torch.exp(0.5 * torch.randn(k, generator=g, device=DEV))
    return (torch.randn(m, k, generator=g, device=DEV) * channel).to(dtype)


def _weights(g, case):
    """4-bit codes of N(0, 0.02) rows: two codes to a byte (the even column in the low half), a scale
    and (asymmetric) a zero point for each group of a row."""
    n, k, groups = case["n"], case["k"], case["k"] // case["group"]
    packed = torch.empty(n, k // 2, dtype=torch.uint8, device=DEV)
    rows = max(1, (1 << 27) // k)
    for i in range(0, n, rows):  # a slab of rows at a time, so that an LM head's normals need little memory
        q = torch.randn(min(rows, n - i), k, generator=g, device=DEV, dtype=torch.float16).mul_(3.2).add_(8.0)
        q = q.round_().clamp_(0, 15).to(torch.uint8)
        packed[i:i + rows] = q[:, 0::2] | (q[:, 1::2] << 4)
    scales = 0.00625 * (0.7 + 0.6 * torch.rand(n, groups, generator=g, device=DEV))
    zeros = None
    if case["zeros"]:
        zeros = torch.randn(n, groups, generator=g, device=DEV).add_(8.0).round_().clamp_(4, 12).to(torch.uint8)
    return packed, scales.to(DTYPES[case["scale"]]), zeros


def _tokens(g, logits):
    """Half of the rows ask for their most likely token, as greedy decoding does, the rest for any."""
    m, vocab = logits.shape
    any_token = torch.randint(0, vocab, (m,), generator=g, device=DEV)
    return torch.where(torch.rand(m, generator=g, device=DEV) < 0.5, logits.float().max(1).indices, any_token)


def prepare(case, seed):
    g = _generator(seed)
    if case["kind"] == "logprobs":
        m, vocab = case["m"], case["vocab"]
        logits = torch.randn(m, vocab, generator=g, device=DEV).mul_(2.2)
        # each row favours a few tokens, some rows one token almost surely
        likely = torch.randint(0, vocab, (m, 8), generator=g, device=DEV)
        logits.scatter_add_(1, likely, 14.0 * torch.rand(m, 8, generator=g, device=DEV))
        if case["masked"]:
            allowed = torch.rand(vocab, generator=g, device=DEV) < 0.6
            allowed[likely[:, 0]] = True
            logits.masked_fill_(~allowed, -math.inf)
        logits = logits.to(DTYPES[case["dtype"]])
        return {"case": case, "logits": logits, "tokens": _tokens(g, logits)}
    packed, scales, zeros = _weights(g, case)
    state = {"case": case, "packed": packed, "scales": scales, "zeros": zeros,
             "x": _activations(g, case["m"], case["k"], DTYPES[case["x"]])}
    if case["kind"] == "int4":
        state["bias"] = torch.randn(case["n"], generator=g, device=DEV) if case["bias"] else None
    else:
        state["tokens"] = torch.randint(0, case["n"], (case["m"],), generator=g, device=DEV)
    if own:
        import nn_amd
        state["weight"] = nn_amd.QuantizedWeight.from_int4_groups(packed, scales, zeros, case["group"])
    return state


# ---- one pass ------------------------------------------------------------------------------


def _plain_weight(packed, scales, zeros, group):
    """W in 32 bits: (code - zero point) * scale, the zero point 8 where none is given."""
    q = torch.stack((packed & 15, packed >> 4), 2).reshape(packed.shape[0], -1).float()
    z = 8.0 if zeros is None else zeros.float().repeat_interleave(group, 1)
    return (q - z) * scales.float().repeat_interleave(group, 1)


def _plain_linear(state):
    case = state["case"]
    y = state["x"].float() @ _plain_weight(state["packed"], state["scales"], state["zeros"], case["group"]).t()
    return y if state.get("bias") is None else y + state["bias"]


def _plain_logprobs(logits, tokens, top, ranks):
    x = logits.float()
    d = x - x.max(1, keepdim=True).values
    e = torch.exp(d)
    total = e.sum(1)
    at = tokens[:, None]
    lse = torch.log(total)
    out = {"logprobs": d.gather(1, at)[:, 0] - lse,
           "entropy": lse - torch.where(e > 0, d * e, torch.zeros_like(e)).sum(1) / total}
    if ranks:
        mine = x.gather(1, at)
        before = torch.arange(x.shape[1], device=x.device)[None] < at
        out["ranks"] = ((x > mine) | ((x == mine) & before)).sum(1)
    if top:
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
        out["top_ids"] = ids
        out["top_logprobs"] = d.gather(1, ids) - lse[:, None]
    return out


def _results(r, ranks, top):
    out = {"logprobs": r.logprobs, "entropy": r.entropy}
    if ranks:
        out["ranks"] = r.ranks
    if top:
        out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
    return out


def run(state):
    case = state["case"]
    if case["kind"] == "int4":
        if own:
            import nn_amd
            return nn_amd.quantized_linear(state["x"], state["weight"], state["bias"], out_dtype=DTYPES[case["out"]])
        return _plain_linear(state).to(DTYPES[case["out"]])
    if case["kind"] == "logprobs":
        if own:
            import nn_amd
            r = nn_amd.token_logprobs(state["logits"], state["tokens"], top_n=case["top"], ranks=case["ranks"])
            return _results(r, case["ranks"], case["top"])
        return _plain_logprobs(state["logits"], state["tokens"], case["top"], case["ranks"])
    if own:
        import nn_amd
        r = nn_amd.linear_logprobs(state["x"], state["weight"], state["tokens"], top_n=case["top"])
        return _results(r, False, case["top"])
    return _plain_logprobs(_plain_linear(state), state["tokens"], case["top"], False)


# ---- bytes and operations --------------------------------------------------------------------


def _weight_bytes(case):
    n, k, groups = case["n"], case["k"], case["k"] // case["group"]
    return n * k // 2 + n * groups * (3 if case["zeros"] else 2)


def _answer_bytes(m, top, ranks):
    return m * (8 + 4 + 4 + (8 if ranks else 0) + 12 * top)  # token read; the rest written


def work(case):
    m = case["m"]
    if case["kind"] == "int4":
        n, k = case["n"], case["k"]
        return {"bytes": _weight_bytes(case) + m * k * BYTES[case["x"]] + m * n * BYTES[case["out"]] + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    if case["kind"] == "logprobs":  # per logit: difference, exp, two sums and a product
        vocab = case["vocab"]
        return {"bytes": m * vocab * BYTES[case["dtype"]] + _answer_bytes(m, case["top"], case["ranks"]), "flops": 5 * m * vocab}
    n, k = case["n"], case["k"]
    return {"bytes": _weight_bytes(case) + m * k * BYTES[case["x"]] + _answer_bytes(m, case["top"], False),
            "flops": 2 * m * n * k + 5 * m * n}


# ---- the definition in 64 bits -----------------------------------------------------------------


def _exact_linear(state, m, n, k, group):
    """sum over groups of scale * (sum of code * x - zero point * sum of x), a slab of rows at a time."""
    x = state["x"].double()
    sums = x.view(m, k // group, group).sum(2)
    y = torch.empty(m, n, dtype=torch.float64, device=DEV)
    rows = max(1, (1 << 27) // k)
    for i in range(0, n, rows):
        s = state["scales"][i:i + rows].double()
        c = torch.empty(s.shape[0], k, dtype=torch.float64, device=DEV)
        c[:, 0::2] = state["packed"][i:i + rows].bitwise_and(15).double()
        c[:, 1::2] = state["packed"][i:i + rows].div(16, rounding_mode="floor").double()
        c = (c.view(-1, k // group, group) * s[:, :, None]).view(-1, k)
        offset = 8 * s if state["zeros"] is None else s * state["zeros"][i:i + rows].double()
        y[:, i:i + rows] = x @ c.t() - sums @ offset.t()
    return y


def _exact_logprobs(x, tokens, top, ranks):
    x = x.double()
    m, vocab = x.shape
    p = torch.softmax(x, 1)
    lse = torch.logsumexp(x, 1)
    mine = x[torch.arange(m, device=DEV), tokens]
    out = {"logprobs": mine - lse, "entropy": torch.special.entr(p).sum(1)}
    order = torch.arange(vocab, device=DEV).expand(m, vocab)
    if ranks:
        ahead = (x > mine[:, None]).sum(1)
        out["ranks"] = ahead + ((x == mine[:, None]) & (order < tokens[:, None])).sum(1)
    if top:
        left, ids, values = x.clone(), [], []
        for _ in range(top):  # the largest that is left, the lowest index of its equals
            best = left.max(1).values
            at = torch.where(left == best[:, None], order, vocab).min(1).values
            ids.append(at)
            values.append(best - lse)
            left[torch.arange(m, device=DEV), at] = -math.inf
        out["top_ids"], out["top_logprobs"] = torch.stack(ids, 1), torch.stack(values, 1)
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "logprobs":
        return _exact_logprobs(state["logits"], state["tokens"], case["top"], case["ranks"])
    y = _exact_linear(state, case["m"], case["n"], case["k"], case["group"])
    if case["kind"] == "int4":
        return y if state["bias"] is None else y + state["bias"].double()
    return _exact_logprobs(y, state["tokens"], case["top"], False)

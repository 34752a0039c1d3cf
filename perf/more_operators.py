"""Microscaled 4-bit floating point and beam search: the calls whose speed is measured, and their plain forms.

Five operators that a program decoding several beams over an MXFP4 model uses together:

``quantize``  rows of activations to MXFP4 (e2m1 codes, a power of two for each 32 of a row) and the
              values they stand for (``quantize_mxfp4_rows``).
``linear``    y = x @ W^T (+ bias) for W in MXFP4, x in full precision (``quantized_linear`` of
              ``QuantizedWeight.from_mxfp4_rows``).
``product``   the same with x quantized to MXFP4 too: a product of 4-bit operands (``mxfp4_linear``).
``select``    a beam search's step: of all continuations of a batch item's beams the k with the
              largest sum of the beam's score and the token's log probability (``beam_select``).
``reorder``   the caches that follow: each slot of a batch item gets its parent's state, in place
              (``beam_reorder``).

``listed`` gives the fixed cases, ``draw`` further ones of the same ranges, ``prepare`` the
weights and inputs, ``run`` one pass (plain torch, or with ``own`` the library's calls), ``work``
the bytes and operations a pass cannot do without, ``exact`` its result in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def quantize(m, k, x="bf16", rule="ceil"):
    return {"kind": "quantize", "m": m, "k": k, "x": x, "rule": rule}


def linear(m, n, k, x="bf16", out="bf16", bias=False):
    return {"kind": "linear", "m": m, "n": n, "k": k, "x": x, "out": out, "bias": bias}


def product(m, n, k, x="bf16", out="bf16", bias=False, rule="ceil"):
    return {"kind": "product", "m": m, "n": n, "k": k, "x": x, "out": out, "bias": bias, "rule": rule}


def select(batch, beams, vocab, keep, dtype="f32", masked=False, finished=False, first=False):
    return {"kind": "select", "batch": batch, "beams": beams, "vocab": vocab, "keep": keep, "dtype": dtype,
            "masked": masked, "finished": finished, "first": first}


def reorder(batch, beams, heads, room, used, width, tensors, moved, parents, dtype="bf16"):
    return {"kind": "reorder", "batch": batch, "beams": beams, "heads": heads, "room": room, "used": used,
            "width": width, "tensors": tensors, "moved": moved, "parents": parents, "dtype": dtype}


def listed():
    cases = {
        # one token's hidden state before a projection: the smallest call, where latency counts
        "quantize_token": quantize(1, 4096),
        # a prompt of odd length before the down projection, f32 activations
        "quantize_prompt2011_f32": quantize(2011, 12288, x="f32"),
        # one token through the down projection, f32 activations as the linear's default
        "linear_decode_down_f32": linear(1, 4096, 12288, x="f32", out="f32"),
        # a dozen beams through the fused gate | up projection
        "linear_batch12_gate_up": linear(12, 24576, 4096, bias=True),
        # a prompt of 512 tokens through the up projection
        "linear_prefill512": linear(512, 12288, 4096),
        # eight sequences' tokens through the down projection, both sides in 4 bits
        "product_batch8_down": product(8, 4096, 12288),
        # a prompt of odd length, K that ends inside a 128-wide step, an odd number of output columns
        "product_prefill301_odd": product(301, 5751, 2880, x="f32", out="f32", bias=True),
        # a long prompt through the fused gate | up projection
        "product_prefill2048": product(2048, 24576, 4096, rule="floor"),
        # one sequence's four beams over a large vocabulary, two candidates a beam
        "select_four_beams": select(1, 4, 151936, 8),
        # a served batch under a grammar's mask, some beams at their end, logits in bf16 (ties are common)
        "select_batch24_bf16": select(24, 8, 50257, 16, dtype="bf16", masked=True, finished=True),
        # a short cache of one sequence with four beams, one of which took another's place
        "reorder_short": reorder(1, 4, 8, 64, 37, 128, 4, 1, 1),
        # long caches of a served batch: three of four slots move
        "reorder_batch8_long": reorder(8, 4, 8, 2048, 1501, 128, 8, 3, 1),
    }
    return [dict(name=name, **case) for name, case in cases.items()]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_weight(rng):
    k = 32 * _log_uniform(rng, 8, 384)
    n = _log_uniform(rng, 256, 24576)
    if rng.random() < 0.6:
        n = (n + 127) // 128 * 128  # models' widths; the rest any number of rows
    return min(n, 100000000 // k), k


def draw(rng):
    kind = rng.choice(("quantize", "linear", "linear", "product", "product", "select", "select", "reorder"))
    x, out = rng.choice(("bf16", "bf16", "f32")), rng.choice(("bf16", "f32"))
    rule = rng.choice(("ceil", "ceil", "floor"))
    if kind == "quantize":
        k = 32 * _log_uniform(rng, 2, 512)
        return quantize(min(_log_uniform(rng, 1, 8192), 2011 * 12288 // k), k, x, rule)
    if kind == "linear":
        n, k = _draw_weight(rng)
        return linear(min(_log_uniform(rng, 1, 640), int(5e10 / (2 * n * k))), n, k, x, out, rng.random() < 0.3)
    if kind == "product":
        n, k = _draw_weight(rng)
        return product(min(_log_uniform(rng, 1, 4096), int(4e11 / (2 * n * k))), n, k, x, out, rng.random() < 0.3, rule)
    if kind == "select":
        beams, vocab = rng.randint(1, 16), _log_uniform(rng, 1000, 151936)
        batch = min(_log_uniform(rng, 1, 64), max(1, 24 * 8 * 50257 // (beams * vocab)))
        return select(batch, beams, vocab, rng.randint(beams, min(32, 2 * beams)), rng.choice(("f32", "f32", "bf16", "f16")),
                      rng.random() < 0.3, rng.random() < 0.4, rng.random() < 0.2)
    beams, width, heads = rng.randint(2, 12), rng.choice((64, 80, 128)), rng.randint(1, 8)
    moved, dtype = rng.randint(1, beams - 1), rng.choice(("bf16", "bf16", "f32"))
    parents = rng.randint(1, min(moved, beams - moved))
    batch, tensors = _log_uniform(rng, 1, 16), rng.randint(1, 8)
    most = 8 * 8 * 1501 * 128 * 8 * 2 * 4 // (batch * tensors * heads * width * BYTES[dtype] * (moved + parents))
    used = max(1, min(_log_uniform(rng, 1, 2048), most))
    return reorder(batch, beams, heads, used + rng.randint(0, 64), used, width, tensors, moved, parents, dtype)


# ---- inputs --------------------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _activations(g, m, k, dtype):
    """N(0, 1) tokens whose channels differ in size, as a model's hidden states do."""
    channel = torch.exp(0.5 * torch.randn(k, generator=g, device=DEV))
    return (torch.randn(m, k, generator=g, device=DEV) * channel).to(dtype)


def _weights(g, n, k):
    """The MXFP4 form of N(0, 0.02) rows: two codes to a byte, the even column in the low half, and a
    biased exponent for each 32 columns."""
    codes = torch.empty(n, k // 2, dtype=torch.uint8, device=DEV)
    scales = torch.empty(n, k // 32, dtype=torch.uint8, device=DEV)
    rows = max(1, (1 << 26) // k)
    for i in range(0, n, rows):  # a slab of rows at a time, so that the normals need little memory
        w = torch.randn(min(rows, n - i), k, generator=g, device=DEV).mul_(0.02)
        values, e = _plain_quantize(w, "ceil")
        index = _plain_index(values.abs()) + torch.where(values < 0, 8, 0)
        codes[i:i + rows] = (index[:, 0::2] | (index[:, 1::2] << 4)).to(torch.uint8)
        scales[i:i + rows] = (e + 127).to(torch.uint8)
    return codes, scales


def _logits(g, case):
    batch, beams, vocab = case["batch"], case["beams"], case["vocab"]
    logits = torch.randn(batch, beams, vocab, generator=g, device=DEV).mul_(2.2)
    # each beam favours a few tokens, some beams one token almost surely
    likely = torch.randint(0, vocab, (batch, beams, 8), generator=g, device=DEV)
    logits.scatter_add_(2, likely, 14.0 * torch.rand(batch, beams, 8, generator=g, device=DEV))
    if case["masked"]:
        allowed = torch.rand(vocab, generator=g, device=DEV) < 0.6
        allowed[likely[:, :, 0].reshape(-1)] = True
        logits.masked_fill_(~allowed, -math.inf)
    return logits.to(DTYPES[case["dtype"]])


def prepare(case, seed):
    g = _generator(seed)
    state = {"case": case}
    if case["kind"] in ("quantize", "linear", "product"):
        if case["kind"] != "quantize":
            codes, scales = _weights(g, case["n"], case["k"])
            state |= {"codes": codes, "scales": scales}
            state["bias"] = torch.randn(case["n"], generator=g, device=DEV) if case["bias"] else None
            if own:
                import nn_amd
                state["weight"] = nn_amd.QuantizedWeight.from_mxfp4_rows(codes, scales)
        state["x"] = _activations(g, case["m"], case["k"], DTYPES[case["x"]])
        return state
    batch, beams = case["batch"], case["beams"]
    if case["kind"] == "select":
        state["logits"] = _logits(g, case)
        scores = -30.0 + 3.0 * torch.randn(batch, beams, generator=g, device=DEV)
        scores = scores.sort(1, descending=True).values
        if case["first"]:  # the first step: all beams hold the prompt, and one counts
            scores[:, 1:] = -math.inf
        state["scores"] = scores
        state["finished"] = torch.rand(batch, beams, generator=g, device=DEV) < 0.25 if case["finished"] else None
        state["end"] = case["vocab"] - 1
        return state
    # which slots move, and which of the others they copy (those stay)
    order = torch.rand(batch, beams, generator=g, device=DEV).argsort(1)
    moved, stay = order[:, :case["moved"]], order[:, case["moved"]:]
    parents = torch.arange(beams, device=DEV).repeat(batch, 1)
    of = torch.arange(case["moved"], device=DEV) % case["parents"]
    state["parents"] = parents.scatter(1, moved, stay[:, of])
    shape = (batch * beams, case["heads"], case["room"], case["width"])
    state["caches"] = [torch.randn(shape, generator=g, device=DEV, dtype=DTYPES[case["dtype"]]) for _ in range(case["tensors"])]
    return state


# ---- one pass ------------------------------------------------------------------------------


def _plain_index(a):
    """The place of magnitudes that are on the grid 0, 0.5, 1, 1.5, 2, 3, 4, 6."""
    return torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.int64)


def _plain_quantize(x, rule):
    """(values on the e2m1 grid, exponents per 32): scale 2^e, e from the block's largest magnitude f * 2^p with
    f in [0.5, 1): "floor" p - 3, above 6 saturating; "ceil" the smallest that brings it to at most 6."""
    b = x.float().unflatten(1, (-1, 32))
    f, p = torch.frexp(b.abs().amax(2))
    e = p - 3 if rule == "floor" else torch.where(f <= 0.75, p - 3, p - 2)
    e = torch.where(f == 0, -127, e.clamp(-127, 125))
    half = torch.ldexp(torch.ones_like(f), -torch.div(e, 2, rounding_mode="floor"))  # 2^-e in two exact factors
    v = b * half[:, :, None] * torch.ldexp(torch.ones_like(f), -(e - torch.div(e, 2, rounding_mode="floor")))[:, :, None]
    a = v.abs()
    # steps of 0.5 up to 2, of 1 up to 4, of 2 above; to the nearest, halves to even
    q = torch.where(a < 2, (2 * a).round() / 2, torch.where(a < 4, a.round(), 2 * (a / 2).round()))
    return (q.clamp(max=6.0) * torch.sign(v)).flatten(1), e


def _plain_values(x, rule):
    values, e = _plain_quantize(x, rule)
    h = torch.div(e, 2, rounding_mode="floor")
    one = torch.ones_like(e, dtype=torch.float32)
    return (values.unflatten(1, (-1, 32)) * torch.ldexp(one, h)[:, :, None] * torch.ldexp(one, e - h)[:, :, None]).flatten(1)


def _plain_weight(codes, scales):
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    grid = torch.cat((grid, -grid))
    w = torch.stack((grid[(codes & 15).long()], grid[(codes >> 4).long()]), 2).flatten(1)
    scale = torch.ldexp(torch.ones(scales.shape, device=codes.device), scales.int() - 127)
    return (w.unflatten(1, (-1, 32)) * scale[:, :, None]).flatten(1)


def _plain_linear(state, x):
    y = x @ _plain_weight(state["codes"], state["scales"]).t()
    return (y if state["bias"] is None else y + state["bias"]).to(DTYPES[state["case"]["out"]])


def _plain_select(state):
    """In 64 bits: continuations of two beams may be nearly equal."""
    x, case = state["logits"].double(), state["case"]
    d = x - x.amax(2, keepdim=True)
    value = state["scores"].double()[:, :, None] + (d - torch.log(torch.exp(d).sum(2, keepdim=True)))
    if state["finished"] is not None:  # an ended beam stays as it is, with the end token
        end = torch.full_like(value, -math.inf)
        end[:, :, state["end"]] = state["scores"].double()
        value = torch.where(state["finished"][:, :, None], end, value)
    value, at = torch.sort(value.flatten(1), dim=1, descending=True, stable=True)
    value, at = value[:, :case["keep"]], at[:, :case["keep"]]
    none = value == -math.inf
    return {"scores": value.float(), "parents": torch.where(none, -1, at // case["vocab"]),
            "tokens": torch.where(none, -1, at % case["vocab"])}


def _plain_reorder(state):
    case, caches = state["case"], state["caches"]
    batch, beams, used = case["batch"], case["beams"], case["used"]
    rows = (state["parents"] + beams * torch.arange(batch, device=DEV)[:, None]).reshape(-1)
    for c in caches:
        c[:, :, :used] = c[rows, :, :used]
    return caches


def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        if kind == "quantize":
            return _plain_values(state["x"], case["rule"])
        if kind == "linear":
            return _plain_linear(state, state["x"].float())
        if kind == "product":
            return _plain_linear(state, _plain_values(state["x"], case["rule"]))
        return _plain_select(state) if kind == "select" else _plain_reorder(state)
    import nn_amd
    if kind == "quantize":
        return nn_amd.quantize_mxfp4_rows(state["x"], case["rule"]).dequantize()
    if kind == "linear":
        return nn_amd.quantized_linear(state["x"], state["weight"], state["bias"], out_dtype=DTYPES[case["out"]])
    if kind == "product":
        return nn_amd.mxfp4_linear(state["x"], state["weight"], state["bias"], out_dtype=DTYPES[case["out"]],
                                   scale_rule=case["rule"])
    if kind == "select":
        r = nn_amd.beam_select(state["logits"], state["scores"], case["keep"], finished=state["finished"],
                               end_token=state["end"])
        return {"scores": r.scores, "parents": r.parents, "tokens": r.tokens}
    nn_amd.beam_reorder([c[:, :, :case["used"]] for c in state["caches"]], state["parents"])
    return state["caches"]


# ---- bytes and operations --------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "quantize":  # x read; codes, exponents and f32 values written
        n = case["m"] * case["k"]
        return {"bytes": n * BYTES[case["x"]] + n // 2 + n // 32 + 4 * n, "flops": 4 * n}
    if kind in ("linear", "product"):
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k // 2 + n * k // 32 + m * k * BYTES[case["x"]] + m * n * BYTES[case["out"]] + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    if kind == "select":  # per logit: difference, exp, sum
        rows = case["batch"] * case["beams"]
        return {"bytes": rows * case["vocab"] * BYTES[case["dtype"]] + 5 * rows + 20 * case["batch"] * case["keep"],
                "flops": 3 * rows * case["vocab"]}
    row = case["tensors"] * case["heads"] * case["used"] * case["width"] * BYTES[case["dtype"]]
    return {"bytes": case["batch"] * (row * (case["moved"] + case["parents"]) + 8 * case["beams"]), "flops": 0}


# ---- the definition in 64 bits -----------------------------------------------------------------

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_quantize(x, rule):
    """Each block's exponent by comparison with powers of two, each magnitude by the midpoints of the grid."""
    b = x.double().view(x.shape[0], -1, 32)
    largest = b.abs().amax(2)
    powers = torch.ldexp(torch.ones(253, dtype=torch.float64, device=DEV), torch.arange(-127, 126, device=DEV))
    if rule == "floor":  # the largest s with 4 * 2^s <= largest
        at = torch.searchsorted(4 * powers, largest, right=True) - 1
    else:  # the smallest s with largest <= 6 * 2^s
        at = torch.searchsorted(6 * powers, largest)
    scale = powers[at.clamp(0, 252)][:, :, None]
    grid = torch.tensor(GRID, dtype=torch.float64, device=DEV)
    a = (b.abs() / scale).contiguous()
    mid = (grid[1:] + grid[:-1]) / 2
    low, high = torch.searchsorted(mid, a), torch.searchsorted(mid, a, right=True)  # differ on a midpoint
    i = torch.where(low % 2 == 0, low, high)
    return (torch.where(b < 0, -grid[i], grid[i]) * scale).view(x.shape)


def _exact_linear(state, x):
    case = state["case"]
    grid = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float64, device=DEV)
    y = torch.empty(case["m"], case["n"], dtype=torch.float64, device=DEV)
    rows = max(1, (1 << 26) // case["k"])
    for i in range(0, case["n"], rows):
        c = state["codes"][i:i + rows]
        w = torch.empty(c.shape[0], case["k"], dtype=torch.float64, device=DEV)
        w[:, 0::2], w[:, 1::2] = grid[c.long() % 16], grid[c.long() // 16]
        w *= torch.pow(2.0, state["scales"][i:i + rows].double() - 127).repeat_interleave(32, 1)
        y[:, i:i + rows] = x.double() @ w.t()
    return y if state["bias"] is None else y + state["bias"].double()


def _exact_select(state):
    case = state["case"]
    x = state["logits"].double()
    value = torch.log_softmax(x, 2) + state["scores"].double()[:, :, None]
    if state["finished"] is not None:
        token = torch.arange(case["vocab"], device=DEV)
        value = torch.where(state["finished"][:, :, None],
                            torch.where(token == state["end"], state["scores"].double()[:, :, None], -math.inf), value)
    value = value.flatten(1)
    place = torch.arange(value.shape[1], device=DEV)
    scores, parents, tokens = [], [], []
    for _ in range(case["keep"]):  # the largest that is left, the lowest place of its equals
        best = value.amax(1, keepdim=True)
        at = torch.where(value == best, place, value.shape[1]).amin(1, keepdim=True)
        none = best == -math.inf
        scores.append(best)
        parents.append(torch.where(none, -1, at // case["vocab"]))
        tokens.append(torch.where(none, -1, at % case["vocab"]))
        value = value.scatter(1, at, -math.inf)
    return {"scores": torch.cat(scores, 1), "parents": torch.cat(parents, 1), "tokens": torch.cat(tokens, 1)}


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "quantize":
        return _exact_quantize(state["x"], case["rule"])
    if case["kind"] == "linear":
        return _exact_linear(state, state["x"])
    if case["kind"] == "product":
        return _exact_linear(state, _exact_quantize(state["x"], case["rule"]))
    if case["kind"] == "select":
        return _exact_select(state)
    after = [c.double() for c in state["caches"]]
    for i, row in enumerate(state["parents"].tolist()):
        for j, parent in enumerate(row):
            for old, new in zip(state["caches"], after):
                at = case["beams"] * i
                new[at + j].narrow(1, 0, case["used"]).copy_(old[at + parent].narrow(1, 0, case["used"]))
    return after

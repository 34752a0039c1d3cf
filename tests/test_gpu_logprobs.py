"""GPU parity of token_logprobs and linear_logprobs against the definitions in 64 bits.

Whole numbers (ranks, ids) are equal.  Bars for the floats, d the distance of a logit to its row's largest:
a logit's d carries 2^-24 |d|; a term e^d of the sum R carries (1.5 |d| + 2) 2^-24 from its argument and the
exponential and some 45 roundings of the sums, so log1p(R) is off by at most (1.5 * 30 + 47) 2^-24 = 5.5e-6
where terms down to d = -30 count (those below add less than their own size), plus its own 2^-23 of at
most 12; the last subtraction rounds at 2^-24 of the result.  So |error| <= 1e-5 + 2^-23 |log p|, and for
the entropy, whose S has the same relative error, 1e-5 (1 + H).  For rows with one nearly certain token
both are relative: R and S themselves, to 1e-5."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module", autouse=True)
def dev():
    import nn_amd
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    nn_amd.init(0)
    return torch.device("cuda:0")


def plain(logits, tokens, top):
    """The definitions in 64 bits on the host: dict of logprobs, entropy, ranks, top_ids, top_logprobs."""
    x = logits.double().cpu()
    m, n = x.shape
    t = tokens.cpu()
    mx = x.max(1, keepdim=True).values
    d = x - mx
    e = torch.exp(d)
    z = e.sum(1)
    lz = torch.log(z)
    # log Z of a row that one token dominates, without its 1: log1p of the rest
    best = torch.argmax(x, 1)
    rest = e.clone()
    rest[torch.arange(m), best] = 0
    r = rest.sum(1)
    lz = torch.where(r < 0.5, torch.log1p(r), lz)
    ok = (t >= 0) & (t < n)
    tc = t.clamp(0, n - 1)
    mine = x[torch.arange(m), tc]
    bad = ~torch.isfinite(mx[:, 0]) | torch.isnan(z)
    lp = torch.where(ok & ~bad, mine - mx[:, 0] - lz, NAN)
    ent = torch.where(bad, NAN, lz - torch.where(e > 0, d * e, 0.0).sum(1) / z)
    before = (x > mine[:, None]).sum(1) + ((x == mine[:, None]) & (torch.arange(n) < tc[:, None])).sum(1)
    order = torch.sort(torch.where(torch.isnan(x), -INF, x), dim=1, descending=True, stable=True).indices[:, :top]
    vals = x.gather(1, order)
    none = ~(vals > -INF)
    tlp = torch.where(none, -INF, vals - mx - lz[:, None])
    return {"logprobs": lp, "entropy": ent, "ranks": torch.where(torch.isnan(lp), -1, before),
            "top_ids": torch.where(none, -1, order), "top_logprobs": torch.where(bad[:, None], NAN, tlp), "bad": bad}


def near(a, b, atol, rtol):
    a = a.double().cpu()
    assert a.shape == b.shape
    assert torch.equal(torch.isnan(a), torch.isnan(b)), "NaN at other places"
    fin = torch.isfinite(b)
    assert torch.equal(a[~fin & ~torch.isnan(b)], b[~fin & ~torch.isnan(b)])
    err = (a - b)[fin].abs() - rtol * b[fin].abs()
    assert err.numel() == 0 or err.max().item() <= atol, f"off by {err.max().item():.2e} more than allowed"


def check(r, ref, top, ids=True):
    near(r.logprobs, ref["logprobs"], 1e-5, 2 ** -23)
    near(r.entropy, ref["entropy"], 1e-5, 1e-5)
    if r.ranks is not None:
        assert torch.equal(r.ranks.cpu(), ref["ranks"])
    if top:
        near(r.top_logprobs, ref["top_logprobs"], 1e-5, 2 ** -23)
        if ids:
            good = ~ref["bad"]  # a row of NaN has no order to speak of
            assert torch.equal(r.top_ids.cpu()[good], ref["top_ids"][good])


def draw(m, n, dtype=F32, seed=0, spread=3.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = (torch.randn(m, n, generator=g, device="cuda") * spread).to(dtype)
    return x, torch.randint(0, n, (m,), generator=g, device="cuda")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,n", [(1, 1), (3, 2), (2, 7), (5, 63), (4, 64), (3, 1000), (2, 2045), (2, 2048), (3, 2049), (2, 8191),
                                 (2, 8193), (7, 50257), (2, 151936)])
def test_against_64_bits(m, n, dtype):
    import nn_amd
    x, t = draw(m, n, dtype, seed=n)
    top = min(20, n)
    ref = plain(x, t, top)
    check(nn_amd.token_logprobs(x, t, top_n=top, ranks=True), ref, top)
    for kw in ({}, {"ranks": True}, {"top_n": min(3, n)}):  # the kernel's other forms
        r = nn_amd.token_logprobs(x, t, **kw)
        near(r.logprobs, ref["logprobs"], 1e-5, 2 ** -23)
        assert (r.ranks is None) == ("ranks" not in kw) and (r.top_ids is None) == ("top_n" not in kw)
        if r.ranks is not None:
            assert torch.equal(r.ranks.cpu(), ref["ranks"])
        if r.top_ids is not None:
            assert torch.equal(r.top_ids.cpu(), ref["top_ids"][:, :kw["top_n"]])


@pytest.mark.parametrize("top", [1, 5, 32])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_ties(top, dtype):
    """Few distinct values, all equal, equal but for one, a sorted row (a segment's largest in one lane), and
    zeros of both signs: the lowest index comes first."""
    import nn_amd
    n = 9000
    x, t = draw(6, n, dtype, seed=3)
    x[0] = x[0].round()
    x[1] = 1.25
    x[2] = 1.25
    x[2, 7001] = 2.0
    x[3] = torch.sort(x[3], descending=True).values
    x[4] = torch.where(torch.arange(n, device="cuda") % 2 == 0, 0.0, -0.0).to(dtype)
    x[5] = torch.sort(x[5]).values
    t[1], t[4] = 8999, 5001
    check(nn_amd.token_logprobs(x, t, top_n=top, ranks=True), plain(x, t, top), top)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("top", [1, 5, 20, 32])
def test_candidates_around_the_slots(dtype, top):
    """From fewer than a segment's slots to more than a wave's lanes reach the bound, all equal or not: copies of
    the largest value, logits far from 0, masks of the type's lowest value, the largest in one run of the row."""
    import nn_amd
    n = 5000
    rows = []
    g = torch.Generator(device="cuda")
    g.manual_seed(top)
    base = torch.randn(n, generator=g, device="cuda")
    for k in (3, 9, 30, 40, 63, 64, 65, 200):
        r = base.clone()
        r[torch.randperm(2040, generator=g, device="cuda")[:k]] = 6.0  # in the first segment
        rows.append(r)
    rows += [base + 300.0, base * 1e-3 + 3000.0, base * 1e-30]
    low = torch.full((n,), torch.finfo(dtype).min, device="cuda")
    few = torch.randperm(n, generator=g, device="cuda")
    for k in (0, 1, top - 1, top, 90):
        r = low.clone()
        r[few[:k]] = base[few[:k]]
        rows.append(r)
    r = base.clone()
    r[1000:1100] = 10.0 - torch.arange(100, device="cuda") / 16  # lanes of 4 or 8 hold all of the largest
    rows.append(r)
    rows.append(-torch.arange(n, device="cuda") / 32.0)
    x = torch.stack(rows).to(dtype)
    t = torch.randint(0, n, (len(rows),), generator=g, device="cuda")
    check(nn_amd.token_logprobs(x, t, top_n=top, ranks=True), plain(x, t, top), top)
    check(nn_amd.token_logprobs(x[:, 1:], t.clamp(max=n - 2), top_n=top, ranks=True), plain(x[:, 1:], t.clamp(max=n - 2), top), top)


def test_many_equal_logits_over_many_segments():
    """Every segment offers as many candidates as it may, all equal: more than the join's list holds."""
    import nn_amd
    n = 151936
    x = torch.zeros(2, n, device="cuda")
    x[1] = torch.arange(n, device="cuda") % 3
    t = torch.tensor([151935, 0], device="cuda")
    for top in (1, 32):
        check(nn_amd.token_logprobs(x, t, top_n=top, ranks=True), plain(x, t, top), top)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_masks(dtype):
    """-inf over most of a row, over all but fewer tokens than alternatives are asked for, over all but one,
    over the whole row; the token itself masked; and the type's lowest value as the mask."""
    import nn_amd
    n, top = 5000, 8
    x, t = draw(7, n, dtype, seed=5)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x[0][torch.rand(n, generator=g, device="cuda") < 0.95] = -INF
    keep = torch.tensor([4999, 17, 2050], device="cuda")
    for r in (1, 6):
        kept = x[r, keep].clone()
        x[r] = -INF
        x[r, keep] = kept
    x[2] = -INF
    x[2, 3000] = 1.5
    x[3] = -INF
    x[4, t[4]] = -INF
    x[5, 100:] = torch.finfo(dtype).min
    t[1], t[2], t[6] = 17, 3000, 18
    r = nn_amd.token_logprobs(x, t, top_n=top, ranks=True)
    check(r, plain(x, t, top), top)
    assert r.logprobs[2] == 0 and r.entropy[2] == 0 and r.top_ids[2].tolist() == [3000] + [-1] * 7
    assert torch.isnan(r.logprobs[3]) and r.ranks[3] == -1 and (r.top_ids[3] == -1).all() and torch.isnan(r.top_logprobs[3]).all()
    assert r.logprobs[4] == -INF and r.logprobs[6] == -INF


def test_nan_and_infinity_rows():
    import nn_amd
    x, t = draw(6, 4100, F32, seed=6)
    x[0, 4099] = NAN
    x[1, 5] = INF
    x[2] = NAN
    x[3, 7], x[3, 3000] = INF, NAN
    x[4, 9], x[4, 10] = INF, INF
    r = nn_amd.token_logprobs(x, t, top_n=4, ranks=True)
    ref = plain(x, t, 4)
    ref["bad"][:5] = True
    for k in ("logprobs", "entropy", "top_logprobs"):
        ref[k][:5] = NAN
    ref["ranks"][:5] = -1
    check(r, ref, 4)


def test_nearly_certain_tokens():
    """Log probabilities and entropies near 0, relative to themselves: R and S are held without the 1."""
    import nn_amd
    n = 4500
    x = torch.full((3, n), -50.0, device="cuda")
    x[0, 4321] = 0.0
    x[0, 7] = -18.0
    x[1] = -25.0
    x[1, 0] = 3.0
    x[2] = -40.0
    x[2, 2100] = 1.0
    t = torch.tensor([4321, 0, 2100], device="cuda")
    r = nn_amd.token_logprobs(x, t)
    ref = plain(x, t, 1)
    assert (ref["logprobs"] > -1e-7).all() and (ref["logprobs"] < 0).all()
    near(r.logprobs, ref["logprobs"], 0.0, 1e-5)
    near(r.entropy, ref["entropy"], 0.0, 1e-5)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_one_term_beside_the_largest(dtype):
    """Two logits an exact distance d apart, d = -1 to -86: R is the one term e^d, and log1p(R) and the entropy are
    as good as that and log1p.  Bar: e^d to 2^-22 (the hardware's 2^p to a unit in the last place, 2^-23, one
    rounding of the correction, 2^-24, its terms left out below that), log1p to 2 units, 2^-22; the entropy's
    other part -d R / (1 + R) has e^d's 2^-22 and four roundings of at most 2^-24, its last addition one more.
    So 9 x 2^-24 relative for both."""
    import nn_amd
    d = torch.arange(1, 87, device="cuda")
    x = torch.stack([torch.zeros_like(d), -d], 1).to(dtype)
    t = torch.zeros(86, dtype=torch.int64, device="cuda")
    r = nn_amd.token_logprobs(x, t)
    ref = plain(x, t, 1)
    near(r.logprobs, ref["logprobs"], 0.0, 9 * 2 ** -24)
    near(r.entropy, ref["entropy"], 0.0, 9 * 2 ** -24)


def test_tokens_outside_the_vocabulary():
    import nn_amd
    x, _ = draw(5, 3000, F32, seed=8)
    t = torch.tensor([-100, 0, 3000, 2999, 1 << 40], device="cuda")
    r = nn_amd.token_logprobs(x, t, top_n=2, ranks=True)
    check(r, plain(x, t, 2), 2)
    assert torch.isnan(r.logprobs[[0, 2, 4]]).all() and r.ranks[[0, 2, 4]].tolist() == [-1] * 3
    assert torch.isfinite(r.entropy).all() and torch.isfinite(r.top_logprobs).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views(dtype):
    """Rows that start anywhere in a 16-byte word, a row stride of its own, repeated rows, a transposed tensor,
    leading dimensions, one row without a batch, no rows; int32 and host tokens."""
    import nn_amd
    x, t = draw(9, 3001, dtype, seed=9)
    big = torch.full((9, 3333), 60.0, device="cuda", dtype=dtype)  # what lies around the rows is larger
    for off in range(9):
        v = big[:, off:off + 3001]
        v.copy_(x)
        check(nn_amd.token_logprobs(v, t, top_n=6, ranks=True), plain(x, t, 6), 6)
        big.fill_(60.0)
    check(nn_amd.token_logprobs(x[::2], t[::2], top_n=3), plain(x[::2], t[::2], 3), 3)
    e = x[:1].expand(5, 3001)
    check(nn_amd.token_logprobs(e, t[:5], top_n=3, ranks=True), plain(e, t[:5], 3), 3)
    check(nn_amd.token_logprobs(x.t().contiguous().t(), t, top_n=3), plain(x, t, 3), 3)
    r = nn_amd.token_logprobs(x.view(3, 3, 3001), t.view(3, 3), top_n=4, ranks=True)
    assert r.logprobs.shape == r.entropy.shape == r.ranks.shape == (3, 3) and r.top_ids.shape == (3, 3, 4)
    check(type(r)(r.logprobs.view(9), r.entropy.view(9), r.ranks.view(9), r.top_logprobs.view(9, 4), r.top_ids.view(9, 4)),
          plain(x, t, 4), 4)
    one = nn_amd.token_logprobs(x[2], t[2], top_n=4)
    assert one.logprobs.shape == () and one.top_ids.shape == (4,) and torch.equal(one.logprobs, r.logprobs.view(9)[2])
    none = nn_amd.token_logprobs(x[:0], t[:0], top_n=4, ranks=True)
    assert none.logprobs.shape == (0,) and none.top_ids.shape == (0, 4)
    a = nn_amd.token_logprobs(x, t.int())
    b = nn_amd.token_logprobs(x, t.tolist())
    assert torch.equal(a.logprobs, b.logprobs)
    with pytest.raises(nn_amd.InvalidShape):
        nn_amd.token_logprobs(x, t, top_n=33)
    with pytest.raises(nn_amd.ShapeMismatch):
        nn_amd.token_logprobs(x, t[:-1])


def test_no_rows():
    import nn_amd
    x, _ = draw(2, 5003, F32, seed=2)
    for r in (nn_amd.token_logprobs(x[:0], [], top_n=4, ranks=True),
              nn_amd.linear_logprobs(torch.zeros(0, 512, device="cuda"), head("int4", 5003, 512), [], top_n=4, ranks=True)):
        assert r.logprobs.shape == r.entropy.shape == r.ranks.shape == (0,) and r.top_ids.shape == (0, 4)


def test_more_rows_than_one_launch_takes():
    """70000 rows: two launches; and few long rows whose candidates pass one launch's scratch."""
    import nn_amd
    x, t = draw(70000, 40, F32, seed=10)
    check(nn_amd.token_logprobs(x, t, top_n=2, ranks=True), plain(x, t, 2), 2)
    x, t = draw(2100, 20000, BF16, seed=11)
    rows = torch.tensor([0, 1, 1500, 1999, 2099], device="cuda")
    r = nn_amd.token_logprobs(x, t, top_n=32, ranks=True)
    some = type(r)(*(None if v is None else v[rows] for v in r))
    check(some, plain(x[rows], t[rows], 32), 32)


def test_offsets_past_32_bits():
    """A row that starts more than 2^32 bytes into its tensor."""
    import nn_amd
    x = torch.empty(9, 1 << 27, device="cuda")
    rows = x[:, :3000]
    src, t = draw(9, 3000, F32, seed=12)
    rows.copy_(src)
    assert rows.stride(0) * 4 * 8 >= 1 << 32
    check(nn_amd.token_logprobs(rows, t, top_n=3, ranks=True), plain(src, t, 3), 3)


def test_captured_graph_and_repeats():
    import nn_amd
    x, t = draw(33, 9001, BF16, seed=13)
    nn_amd.token_logprobs(x, t, top_n=5, ranks=True)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = nn_amd.token_logprobs(x, t, top_n=5, ranks=True)
    for i in range(4):
        x2, t2 = draw(33, 9001, BF16, seed=40 + i)
        x.copy_(x2)
        t.copy_(t2)
        nn_amd.token_logprobs(draw(400, 20000, F32, seed=i)[0], [0] * 400, top_n=32)
        g.replay()
        torch.cuda.synchronize()
        e = nn_amd.token_logprobs(x, t, top_n=5, ranks=True)
        for a, b in zip(r[:5], e[:5]):
            assert torch.equal(a, b)
        check(r, plain(x, t, 5), 5)


# ---- through an LM head ---------------------------------------------------------------------


def head(fmt, n, k, seed=21):
    import nn_amd
    from test_gpu_int4 import make
    if fmt == "int4":
        return make(n, k, 128, seed=seed)[0]
    quant = {"q8_0": nn_amd.quantize_q8_0, "q4_k": nn_amd.quantize_q4_k, "q6_k": nn_amd.quantize_q6_k}[fmt]
    layout = nn_amd.Layout.NN_GGUF if fmt == "q6_k" else nn_amd.Layout.GGUF
    qt = {"q8_0": nn_amd.QuantType.Q8_0, "q4_k": nn_amd.QuantType.Q4_K, "q6_k": nn_amd.QuantType.Q6_K}[fmt]
    return nn_amd.QuantizedWeight.from_quantized(quant(nn_amd.synth_normal(seed, 1, (n, k), 0.05)), qt, (n, k), layout=layout)


@pytest.mark.parametrize("xdt", [F32, BF16])
@pytest.mark.parametrize("m", [1, 2, 9, 40, 150])
@pytest.mark.parametrize("fmt", ["int4", "q8_0", "q4_k", "q6_k"])
def test_linear_logprobs(fmt, m, xdt):
    """The same numbers as the log probabilities of the linear's own logits (bit for bit), which are the
    definition's on those logits."""
    import nn_amd
    n, k = 5003, 512
    w = head(fmt, n, k)
    g = torch.Generator(device="cuda")
    g.manual_seed(m)
    x = torch.randn(m, k, generator=g, device="cuda").to(xdt)
    t = torch.randint(0, n, (m,), generator=g, device="cuda")
    bias = torch.randn(n, generator=g, device="cuda")
    y = nn_amd.quantized_linear(x, w, bias)
    a = nn_amd.token_logprobs(y, t, top_n=7, ranks=True)
    b = nn_amd.linear_logprobs(x, w, t, bias, top_n=7, ranks=True, return_logits=True)
    c = nn_amd.linear_logprobs(x, w, t, bias, top_n=7, ranks=True)
    assert torch.equal(b.logits, y) and c.logits is None
    for u, v, s in zip(a[:5], b[:5], c[:5]):
        assert torch.equal(u, v) and torch.equal(u, s)
    check(a, plain(y, t, 7), 7)


def test_linear_logprobs_in_chunks():
    """More rows than one chunk of logits holds (n = 1200001: 64 rows), the last chunk shorter; x misaligned."""
    import nn_amd
    n, k, m = 1200001, 128, 150
    w = head("int4", n, k)
    flat = torch.randn(m * k + 1, device="cuda")
    x = flat[1:].view(m, k)
    t = torch.arange(m, device="cuda") * 4000
    r = nn_amd.linear_logprobs(x, w, t, top_n=3, ranks=True)
    for i in (0, 63, 64, 65, 127, 128, 149):
        y = nn_amd.quantized_linear(x[i:i + 1], w)
        ref = plain(y, t[i:i + 1], 3)
        # (one row takes another kernel than many: sums in another order, 1e-5 of the logits' size)
        tol = 3e-5 * y.abs().max().item()
        near(r.logprobs[i:i + 1], ref["logprobs"], 1e-5 + tol, 2 ** -23)
        near(r.top_logprobs[i:i + 1], ref["top_logprobs"], 1e-5 + tol, 2 ** -23)


def test_every_output_of_several_chunks():
    """Rows in three chunks, the logits asked for or kept in the workspace: each of the five outputs is, bit for
    bit, what token_logprobs gives for those logits in one call, and the definition's in rows of every chunk."""
    import nn_amd
    n, k, m = 1200001, 128, 150
    w = head("int4", n, k)
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    x = torch.randn(m, k, generator=g, device="cuda")
    t = torch.randint(0, n, (m,), generator=g, device="cuda")
    bias = torch.randn(n, generator=g, device="cuda")
    kept = nn_amd.linear_logprobs(x, w, t, bias, top_n=3, ranks=True, return_logits=True)
    inner = nn_amd.linear_logprobs(x, w, t, bias, top_n=3, ranks=True)
    whole = nn_amd.token_logprobs(kept.logits, t, top_n=3, ranks=True)
    assert kept.logits.shape == (m, n) and inner.logits is None
    for name, a, b, c in zip(whole._fields, whole[:5], kept[:5], inner[:5]):
        assert torch.equal(a, b) and torch.equal(a, c), name
    rows = torch.tensor([0, 63, 64, 127, 128, 149], device="cuda")
    some = type(kept)(*(v[rows] for v in kept[:5]))
    check(some, plain(kept.logits[rows], t[rows], 3), 3)
    # (the logits are the linear's: one row takes another kernel than many, sums in another order)
    for i in (0, 64, 149):
        y = nn_amd.quantized_linear(x[i:i + 1], w, bias)
        assert (y[0] - kept.logits[i]).abs().max() <= 2e-5 * y.abs().max()


def test_scoring_loop_as_a_server_runs_it():
    """A prompt scored, then tokens sampled one at a time with their log probabilities, nothing returning to the
    host in between; the last step captured in a graph and replayed."""
    import nn_amd
    n, k = 8200, 1024
    w = head("int4", n, k)
    prompt = torch.randn(37, k, device="cuda").to(BF16)
    ids = torch.randint(0, n, (37,), device="cuda")
    scored = nn_amd.linear_logprobs(prompt, w, ids, top_n=5)
    y = nn_amd.quantized_linear(prompt, w)
    check(scored, plain(y, ids, 5), 5)
    hidden = torch.randn(k, device="cuda")
    for step in range(3):
        logits, tok = nn_amd.linear_sample(hidden, w, seed=step)
        r = nn_amd.token_logprobs(logits, tok, top_n=5, ranks=True)
        ref = plain(logits[None], tok[None], 5)
        assert r.ranks.item() == ref["ranks"][0].item() < 50
        near(r.logprobs[None], ref["logprobs"], 1e-5, 2 ** -23)
        hidden = torch.roll(hidden, 1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        nn_amd.linear_logprobs(hidden[None], w, ids[:1], top_n=5)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    one = ids[:1].clone()
    with torch.cuda.graph(g):
        r = nn_amd.linear_logprobs(hidden[None], w, one, top_n=5, ranks=True)
    for i in range(3):
        hidden.copy_(torch.randn(k, device="cuda"))
        one.copy_(ids[i:i + 1])
        g.replay()
        torch.cuda.synchronize()
        e = nn_amd.linear_logprobs(hidden[None], w, one, top_n=5, ranks=True)
        for a, b in zip(r[:5], e[:5]):
            assert torch.equal(a, b)


def test_entropy_of_a_uniform_row():
    import nn_amd
    r = nn_amd.token_logprobs(torch.zeros(1, 50000, device="cuda"), [3])
    assert abs(r.entropy.item() - math.log(50000)) < 1e-5 and abs(r.logprobs.item() + math.log(50000)) < 1e-5

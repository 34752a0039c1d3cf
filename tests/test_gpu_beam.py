"""GPU parity of beam_select and beam_reorder against their definitions in 64 bits, and a beam search over an MXFP4 head.

Parents and tokens are equal: equal values go by beam, then token, and on the seeded inputs no two others are nearer than
the kernel's sums are exact.  Scores: the sum over a row carries 2^-22 a term and its additions in f32, as
token_logprobs' does (1e-5 there, with the sums joined in f32), and the result's rounding to f32 2^-24."""
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


def plain(logits, scores, keep, finished=None, end=0):
    """[batch, beams, n], [batch, beams] on the host -> scores (f64), parents, tokens"""
    x, s = logits.double().cpu(), scores.double().cpu()
    batch, beams, n = x.shape
    out = torch.full((batch, keep), -INF, dtype=torch.float64)
    parents = torch.full((batch, keep), -1)
    tokens = torch.full((batch, keep), -1)
    for b in range(batch):
        cands = []
        for j in range(beams):
            if not math.isfinite(s[b, j]):
                continue
            if finished is not None and finished[b, j]:
                cands.append((-s[b, j].item(), j, 0, end))
                continue
            row = x[b, j]
            if torch.isnan(row).any() or (row == INF).any() or not (row > -INF).any():
                continue
            v = s[b, j] + torch.log_softmax(row, 0)
            order = torch.sort(row, descending=True, stable=True).indices[:keep]
            cands += [(-v[t].item(), j, i, int(t)) for i, t in enumerate(order) if row[t] > -INF]
        for i, (v, j, _, t) in enumerate(sorted(cands)[:keep]):
            out[b, i], parents[b, i], tokens[b, i] = -v, j, t
    return out, parents, tokens


def check(r, ref):
    out, parents, tokens = ref
    assert torch.equal(r.parents.cpu(), parents)
    assert torch.equal(r.tokens.cpu(), tokens)
    got = r.scores.double().cpu()
    fin = torch.isfinite(out)
    assert torch.equal(got[~fin], out[~fin])
    assert ((got - out)[fin].abs() <= 1e-5 + 2.0 ** -24 * out[fin].abs()).all()


def inputs(batch, beams, n, dtype=F32, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed + 1000 * n + beams)
    logits = (torch.randn(batch, beams, n, generator=g) * spread).to(dtype)
    scores = torch.sort(-20 + 3 * torch.randn(batch, beams, generator=g), 1, descending=True).values
    return logits, scores


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("batch,beams,n,keep", [(1, 1, 1, 1), (1, 2, 3, 4), (2, 3, 7, 32), (1, 4, 2047, 8), (3, 5, 2049, 5),
                                                (2, 4, 8193, 8), (7, 8, 5000, 16), (1, 32, 3001, 32), (2, 16, 50257, 32),
                                                (1, 1, 151936, 1), (1, 4, 151936, 8), (1, 16, 90001, 32), (2, 23, 40000, 17), (9, 6, 32000, 12)])
def test_select(batch, beams, n, keep, dtype):
    import nn_amd
    logits, scores = inputs(batch, beams, n, dtype)
    r = nn_amd.beam_select(logits.cuda(), scores.cuda(), keep)
    assert r.scores.dtype is F32 and r.parents.dtype is torch.int64 and r.scores.shape == (batch, keep)
    check(r, plain(logits, scores, keep))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("beams,keep", [(2, 31), (15, 30), (32, 32)])
@pytest.mark.parametrize("n", [63, 64, 200, 255, 257, 511, 512, 1000, 1621, 2048 + 40, 2048 + 212, 4096 + 500])
def test_select_rows_that_end_early(n, beams, keep, dtype):
    """few lanes of a row's last segment hold logits, and few of the join's candidates; also with equal logits"""
    import nn_amd
    logits, scores = inputs(2, beams, n, dtype)
    logits[1] = logits[1].float().round().to(dtype)
    check(nn_amd.beam_select(logits.cuda(), scores.cuda(), keep), plain(logits, scores, keep))


@pytest.mark.parametrize("n", [5, 3000, 20000])
def test_select_ties_go_by_beam_then_token(n):
    """identical beams: every continuation of one ties with the others'; whole-number logits tie within a beam"""
    import nn_amd
    g = torch.Generator().manual_seed(n)
    row = torch.randint(-3, 4, (n,), generator=g).float()
    logits = row.expand(2, 6, n).contiguous()
    scores = torch.full((2, 6), -7.25)
    for keep in (1, 6, 32):
        check(nn_amd.beam_select(logits.cuda(), scores.cuda(), keep), plain(logits, scores, keep))
    # all logits equal: the first tokens of the first beams
    flat = torch.zeros(1, 3, n)
    check(nn_amd.beam_select(flat.cuda(), torch.zeros(1, 3).cuda(), 32), plain(flat, torch.zeros(1, 3), 32))
    # rows at odd places: the sums of equal rows are equal wherever they lie
    wide = torch.empty(2, 6, n + 3, device="cuda")
    wide[:, :, 1:1 + n] = logits.cuda()
    check(nn_amd.beam_select(wide[:, :, 1:1 + n], scores.cuda(), 32), plain(logits, scores, 32))


def test_select_first_step_finished_and_masked_beams():
    import nn_amd
    batch, beams, n = 6, 5, 4099
    logits, scores = inputs(batch, beams, n)
    first = scores.clone()
    first[:, 1:] = -INF
    check(nn_amd.beam_select(logits.cuda(), first.cuda(), 10), plain(logits, first, 10))
    g = torch.Generator().manual_seed(3)
    mask = torch.rand(batch, beams, n, generator=g) < 0.9995
    masked = logits.masked_fill(mask, -INF)
    masked[0, 1] = -INF
    masked[5] = -INF
    masked[5, 2, 17] = 0.5  # one continuation in all
    check(nn_amd.beam_select(masked.cuda(), scores.cuda(), 20), plain(masked, scores, 20))
    finished = torch.rand(batch, beams, generator=g) < 0.5
    finished[1], finished[2] = True, False
    scores[3, 0], scores[4, 4] = NAN, INF
    scores[0, 2] = -INF
    finished[3, 0], finished[0, 2] = True, True
    for f in (finished, None):
        check(nn_amd.beam_select(masked.cuda(), scores.cuda(), 9, finished=None if f is None else f.cuda(), end_token=4098),
              plain(masked, scores, 9, f, 4098))
    lowest = logits.masked_fill(mask, torch.finfo(F32).min)  # masked by the type's lowest value
    check(nn_amd.beam_select(lowest.cuda(), scores.cuda(), 9), plain(lowest, scores, 9))


def test_select_bad_rows_offer_nothing():
    import nn_amd
    logits, scores = inputs(4, 3, 3000)
    logits[0, 0, 5], logits[1, 2, 2999], logits[2, 1, 0] = NAN, INF, NAN
    logits[3] = NAN
    for dt in (F32, BF16):
        check(nn_amd.beam_select(logits.to(dt).cuda(), scores.cuda(), 6), plain(logits.to(dt), scores, 6))


def test_select_peaked_and_far_rows():
    """a token with all the probability, logits around 300 and -1e4, scores far apart"""
    import nn_amd
    logits, scores = inputs(4, 4, 6007)
    logits[0, :, 77] += 60
    logits[1] += 300
    logits[2] -= 1e4
    logits[3] *= 30
    scores[1, 3] = -4e4
    scores[2] = torch.tensor([0.0, -1e-3, -1e5, -3e38])
    check(nn_amd.beam_select(logits.cuda(), scores.cuda(), 12), plain(logits, scores, 12))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_select_strides_and_shapes(dtype):
    import nn_amd
    logits, scores = inputs(4, 3, 2500, dtype)
    ref = plain(logits, scores, 6)
    wide = torch.full((4, 5, 2511), NAN, dtype=dtype, device="cuda")
    for at in (0, 1, 3, 11):
        wide[:, 1:4, at:at + 2500] = logits.cuda()
        check(nn_amd.beam_select(wide[:, 1:4, at:at + 2500], scores.cuda(), 6), ref)
    check(nn_amd.beam_select(logits.cuda().transpose(0, 1).contiguous().transpose(0, 1), scores.cuda(), 6), ref)
    check(nn_amd.beam_select(logits.cuda().transpose(1, 2).contiguous().transpose(1, 2), scores.cuda().double(), 6), ref)
    r = nn_amd.beam_select(logits.cuda().view(2, 2, 3, 2500), scores.cuda().view(2, 2, 3), 6)
    assert r.tokens.shape == (2, 2, 6)
    check(nn_amd.BeamSelection(*(t.view(4, 6) for t in r)), ref)
    r = nn_amd.beam_select(logits[0].cuda(), scores[0].cuda())
    assert r.scores.shape == (3,)
    check(nn_amd.BeamSelection(*(t[None] for t in r)), plain(logits[:1], scores[:1], 3))
    r = nn_amd.beam_select(logits[:0].cuda(), scores[:0].cuda(), 6)
    assert r.scores.shape == (0, 6)
    shared = logits[:1, :1].cuda().expand(4, 3, 2500)  # one row for all beams
    check(nn_amd.beam_select(shared, scores.cuda(), 6), plain(logits[:1, :1].expand(4, 3, 2500), scores, 6))


def test_select_many_items_and_many_ties():
    """more items than one launch's scratch holds; segments whose every logit is a candidate"""
    import nn_amd
    batch, beams, n = 700, 2, 33000
    g = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.randn(batch, beams, n, generator=g, device="cuda")
    scores = -torch.rand(batch, beams, generator=g, device="cuda")
    r = nn_amd.beam_select(logits, scores, 32)
    at = [0, 1, 350, batch - 1]
    check(nn_amd.BeamSelection(*(t[at] for t in r)), plain(logits[at], scores[at], 32))
    flat = torch.zeros(2, 8, 60000, device="cuda")
    flat[1, 5, 59990:] = 1.0
    s = torch.zeros(2, 8, device="cuda")
    check(nn_amd.beam_select(flat, s, 32), plain(flat, s, 32))


def test_select_in_a_graph_and_on_streams():
    import nn_amd
    logits = torch.zeros(3, 4, 9001, device="cuda")
    scores = torch.zeros(3, 4, device="cuda")
    state = torch.zeros(12, 6, 40, device="cuda")

    def step():
        r = nn_amd.beam_select(logits, scores, 4)
        nn_amd.beam_reorder(state, r.parents)
        return r

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = step()
    for i in range(3):
        x, sc = inputs(3, 4, 9001, seed=i)
        logits.copy_(x)
        scores.copy_(sc)
        before = torch.randn(12, 6, 40, generator=torch.Generator().manual_seed(i))
        state.copy_(before)
        ref = plain(x, sc, 4)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(out, ref)
        assert torch.equal(state.cpu(), moved(before, ref[1], 0))
        check(nn_amd.beam_select(logits, scores, 4), ref)  # eager work between the replays


# ---- states -------------------------------------------------------------------------------


def moved(state, parents, dim):
    parents = parents.cpu()
    batch, beams = parents.shape if parents.dim() == 2 else (1, parents.shape[0])
    p = parents.view(batch, beams).clone()
    own = torch.arange(beams).expand(batch, beams)
    p = torch.where((p < 0) | (p >= beams), own, p)
    return state.index_select(dim, (p + beams * torch.arange(batch)[:, None]).reshape(-1).to(state.device))


def parents_of(batch, beams, seed):
    g = torch.Generator().manual_seed(seed)
    p = torch.randint(0, beams, (batch, beams), generator=g)
    p[0] = torch.randperm(beams, generator=g)  # cycles
    if batch > 1:
        p[1] = torch.arange(beams)
    if batch > 2:
        p[2] = -1
        p[2, 0] = beams - 1
    if batch > 3:
        p[3, 0] = beams + 5
        p[3, -1] = -(1 << 40)
    return p


@pytest.mark.parametrize("dtype", [F32, BF16, torch.uint8, torch.int64, torch.complex128])
@pytest.mark.parametrize("batch,beams", [(1, 1), (1, 2), (4, 3), (5, 4), (3, 7), (2, 8), (4, 12), (2, 32)])
def test_reorder(batch, beams, dtype):
    import nn_amd
    p = parents_of(batch, beams, batch + beams)
    for shape in ((), (1,), (3, 5), (2, 9, 16), (4, 700)):
        t = (torch.randn(batch * beams, *shape, generator=torch.Generator().manual_seed(3)) * 50).to(dtype)
        d = t.cuda()
        assert nn_amd.beam_reorder(d, p.cuda()) is None
        assert torch.equal(d.cpu(), moved(t, p, 0))


@pytest.mark.parametrize("beams", [4, 11])
def test_reorder_views_leave_the_rest(beams):
    import nn_amd
    batch = 3
    p = parents_of(batch, beams, 9)
    cache = torch.randn(2, batch * beams, 3, 20, 24, generator=torch.Generator().manual_seed(1)).to(BF16)
    cases = [lambda c: (c, 1), lambda c: (c[:, :, :, :13], 1), lambda c: (c[0, :, :, :1], 0), lambda c: (c[1, :, 2, 5:9, 3:8], 0),
             lambda c: (c[:, :, :, ::3, 1:2], 1), lambda c: (c.permute(3, 2, 0, 4, 1)[:7], -1), lambda c: (c[:, :, :0], 1),
             lambda c: (c[:, :, :, :, ::2], 1)]
    for view in cases:
        want = cache.clone()
        v, dim = view(want)
        v.copy_(moved(v.clone(), p, dim))
        got = cache.cuda()
        v, dim = view(got)
        nn_amd.beam_reorder(v, p.cuda(), dim)
        assert torch.equal(got.cpu(), want)


def test_reorder_several_states_and_integer_types():
    import nn_amd
    p = parents_of(4, 5, 2)
    shapes = [(20, 8, 16)] * 40 + [(20, 3), (20,)]  # more than one launch takes
    dtypes = [BF16] * 20 + [F32] * 20 + [torch.int32, torch.bool]
    ts = [(torch.randn(*s, generator=torch.Generator().manual_seed(i)) * 9).to(d) for i, (s, d) in enumerate(zip(shapes, dtypes))]
    ds = [t.cuda() for t in ts]
    nn_amd.beam_reorder(ds, p.clamp(-2, 9).to(torch.int32).cuda())
    for t, d in zip(ts, ds):
        assert torch.equal(d.cpu(), moved(t, p.clamp(-2, 9), 0))
    one = ts[0][:5].cuda()
    nn_amd.beam_reorder(one, p[0].cuda())
    assert torch.equal(one.cpu(), moved(ts[0][:5], p[0], 0))
    nn_amd.beam_reorder([], p.cuda())
    nn_amd.beam_reorder(ts[0][:0].cuda(), p[:0].cuda())
    strided = torch.stack((p, p + 1), -1).cuda()[..., 0]
    d = ts[1].cuda()
    nn_amd.beam_reorder(d, strided)
    assert torch.equal(d.cpu(), moved(ts[1], p, 0))


@pytest.mark.parametrize("batch,beams,shape,dtype", [(12300, 2, (300, 8), BF16), (12300, 4, (3, 211), torch.uint8),
                                                     (70001, 3, (5,), BF16), (40, 4, (8, 5000, 6), F32)])
def test_reorder_many_pieces(batch, beams, shape, dtype):
    import nn_amd
    p = parents_of(batch, beams, 6)
    cache = torch.randint(0, 100, (batch * beams, *shape[:-1], shape[-1] + 4), generator=torch.Generator().manual_seed(2)).to(dtype)
    for used in (shape[-1] + 4, shape[-1]):
        got = cache.cuda()
        nn_amd.beam_reorder(got[..., :used], p.cuda())
        want = cache.cuda()
        want[..., :used] = moved(want[..., :used], p, 0)
        assert torch.equal(got, want)


def test_reorder_beyond_32_bit_offsets():
    import nn_amd
    state = torch.zeros(4, 3, 1 << 30, dtype=torch.uint8, device="cuda")  # 12 GiB, one item a leading index
    for j in range(3):
        state[2, j] = j + 1
        state[3, j, -5:] = j + 7
    nn_amd.beam_reorder(state, torch.tensor([2, 0, 1], device="cuda"), dim=1)
    for j, parent in enumerate((2, 0, 1)):
        assert int(state[2, j].min()) == int(state[2, j].max()) == parent + 1
        assert int(state[3, j, -5]) == parent + 7 and int(state[3, j, -6]) == 0


def test_refusals():
    import nn_amd
    x, s = torch.randn(2, 3, 50, device="cuda"), torch.zeros(2, 3, device="cuda")
    for bad in (0, 33, -1):
        with pytest.raises(nn_amd.InvalidShape):
            nn_amd.beam_select(x, s, bad)
    with pytest.raises(nn_amd.InvalidShape):
        nn_amd.beam_select(torch.zeros(33, 8, device="cuda"), torch.zeros(33, device="cuda"), 4)
    with pytest.raises(nn_amd.ShapeMismatch):
        nn_amd.beam_select(x, s[:, :2])
    with pytest.raises(nn_amd.ShapeMismatch):
        nn_amd.beam_select(x, s, finished=torch.zeros(2, 3, device="cuda"))
    with pytest.raises(nn_amd.TensorError):
        nn_amd.beam_select(x, s, finished=torch.zeros(2, 3, dtype=torch.bool, device="cuda"), end_token=-1)
    with pytest.raises(nn_amd.Unsupported):
        nn_amd.beam_select(x.cpu(), s)
    with pytest.raises(nn_amd.InvalidShape):
        nn_amd.beam_select(x[..., :0], s)
    p = torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    t = torch.randn(6, 4, device="cuda")
    with pytest.raises(nn_amd.ShapeMismatch):
        nn_amd.beam_reorder(t[:5], p)
    with pytest.raises(nn_amd.RankMismatch):
        nn_amd.beam_reorder(t, p, 2)
    with pytest.raises(nn_amd.Unsupported):
        nn_amd.beam_reorder(t, p.float())
    with pytest.raises(nn_amd.Unsupported):
        nn_amd.beam_reorder(t.cpu(), p)
    with pytest.raises(nn_amd.TensorError, match="twice"):
        nn_amd.beam_reorder([t, t], p)
    with pytest.raises(nn_amd.TensorError, match="overlap"):
        nn_amd.beam_reorder(t[:1].expand(6, 4), p)
    with pytest.raises(nn_amd.TensorError, match="overlap"):
        nn_amd.beam_reorder(torch.zeros(60, device="cuda").as_strided((6, 4), (2, 1)), p)
    with pytest.raises(nn_amd.Unsupported, match="4 dimensions"):
        nn_amd.beam_reorder(torch.zeros(6, 3, 3, 3, 3, 3, device="cuda")[:, :2, :2, :2, :2, :2], p)


def test_reorder_moves_all_states_or_none():
    import nn_amd
    p = torch.tensor([[1, 2, 0], [0, 0, 0]], device="cuda")
    for bad in (torch.randn(1, 4, device="cuda").expand(6, 4), torch.zeros(6, 3, 3, 3, 3, 3, device="cuda")[:, :2, :2, :2, :2, :2],
                torch.zeros(6, *(1,) * 9, device="cuda")):
        good = torch.randn(6, 5, device="cuda")
        was = good.clone()
        with pytest.raises((nn_amd.TensorError, nn_amd.Unsupported)):
            nn_amd.beam_reorder([good, bad], p)
        assert torch.equal(good, was)


# ---- together -------------------------------------------------------------------------------


def test_a_beam_search_over_an_mxfp4_head():
    """Five steps of two sequences with three beams: a hidden state that follows the tokens, logits through an MXFP4 head,
    selection and reordering, against the same search in 64 bits that scores every continuation."""
    import nn_amd
    batch, beams, n, k, steps, end = 2, 3, 997, 128, 5, 11
    g = torch.Generator().manual_seed(4)
    head = nn_amd.quantize_mxfp4_rows(torch.randn(n, k, generator=g).cuda())
    w = nn_amd.QuantizedWeight.from_mxfp4_rows(head.codes, head.scales)
    w64 = head.dequantize().double().cpu()
    embed = (torch.randn(n, k, generator=g) * 0.3).cuda()
    hidden0 = (torch.randn(batch, 1, k, generator=g) * 0.3).cuda().expand(batch, beams, k).reshape(batch * beams, k)

    hidden, history = hidden0.clone(), torch.full((batch * beams, steps), -1, dtype=torch.int64, device="cuda")
    scores = torch.full((batch, beams), -INF, device="cuda")
    scores[:, 0] = 0
    finished = torch.zeros(batch, beams, dtype=torch.bool, device="cuda")
    sums = hidden0.double().cpu().view(batch, beams, k)
    ref = [[(0.0 if j == 0 else -INF, sums[b, j], [], False) for j in range(beams)] for b in range(batch)]
    for step in range(steps):
        logits = nn_amd.quantized_linear(hidden, w).view(batch, beams, n)
        r = nn_amd.beam_select(logits, scores, beams, finished=finished, end_token=end)
        nn_amd.beam_reorder([hidden, history], r.parents)
        nn_amd.beam_reorder(finished.view(-1), r.parents)
        history[:, step] = r.tokens.view(-1)
        hidden += embed[r.tokens.view(-1)]
        finished |= r.tokens == end
        scores = r.scores
        for b in range(batch):
            cands = []
            for j, (s, h, seq, fin) in enumerate(ref[b]):
                if s == -INF:
                    continue
                v = torch.log_softmax(w64 @ h, 0) + s
                cands += [(-s, j, end)] if fin else [(-v[t].item(), j, int(t)) for t in v.topk(beams).indices]
            cands.sort()
            ref[b] = [(-v, ref[b][j][1] + embed[t].double().cpu(), ref[b][j][2] + [t], ref[b][j][3] or t == end) for v, j, t in cands[:beams]]
    for b in range(batch):
        for j in range(beams):
            s, h, seq, fin = ref[b][j]
            assert history[b * beams + j].tolist() == seq
            assert abs(scores[b, j].item() - s) < steps * 1e-4
            assert bool(finished[b, j]) == fin
            assert torch.allclose(hidden[b * beams + j].double().cpu(), h, atol=1e-5)

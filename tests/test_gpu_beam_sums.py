"""How exact beam_select's row sums are: exponentials to 2^-22 of themselves, also where an f32 product d log2(e) is off by
its most, as in token_logprobs."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.fixture(scope="module", autouse=True)
def dev():
    import nn_amd
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    nn_amd.init(0)
    return torch.device("cuda:0")


def hard_differences(lo, hi, sign, g):
    """f32 numbers d in [lo, hi] whose d log2(e) lies nearly half a step from the next f32, on the side of `sign`"""
    d = (lo + (hi - lo) * torch.rand(400000, generator=g, dtype=torch.float64)).float()
    p = d.double() * math.log2(math.e)
    half = 2.0 ** (torch.floor(torch.log2(p.abs())) - 24)  # half of p's step
    off = (p.float().double() - p) / half
    return d[sign * off > 0.9]


@pytest.mark.parametrize("sign", [1, -1])
def test_exponentials_of_far_logits(sign):
    """Segments of one logit of 0 and 2047 some 5.6 below: together they weigh seven times what the one does, and an
    exponential of the rounded product would be off by up to 2^-21 ln 2 = 3.3e-7, all to one side.  The exponential's instruction
    is exact to a step (2^-23) and an FMA rounds it (2^-24); the additions' roundings go either way (6e-9 of a row's sum as
    computed in f32).  A score of the logarithm of the row's sum leaves the selected value near 0, where its own rounding
    is nothing: what it is off by is the sum's relative error."""
    import nn_amd
    g = torch.Generator().manual_seed(7 + sign)
    d = hard_differences(-6.0, -5.56, sign, g)
    assert len(d) > 1000
    rows, n = 64, 38 * 2048
    logits = d[torch.randint(0, len(d), (rows, 38, 2048), generator=g)]
    logits.scatter_(2, torch.randint(0, 2048, (rows, 38, 1), generator=g), 0.0)
    logits = logits.view(rows, 1, n)
    lse = torch.logsumexp(logits.double(), 2)
    scores = lse.float()
    r = nn_amd.beam_select(logits.cuda(), scores.cuda(), 1)
    off = r.scores.double().cpu() - (scores.double() - lse)
    assert abs(off.mean().item()) <= 2.0 ** -23 + 2.0 ** -24, off.mean().item()


def test_sums_of_rows_with_far_masked_and_equal_logits():
    """-inf, the lowest f32 and differences beyond 1e30 count nothing; rows of equal logits are exact"""
    import nn_amd
    n = 5000
    rows = torch.full((6, 1, n), -INF)
    rows[0, 0, 17] = 2.5  # one continuation: its log probability is 0
    rows[1, 0, :] = torch.finfo(torch.float32).min
    rows[1, 0, 4999] = -1.0
    rows[2, 0, ::3] = 3e38
    rows[2, 0, 1::3] = -3e38
    rows[3, 0, :] = -3e38
    rows[4, 0, :2048] = -100.0
    rows[4, 0, 2100:2102] = 30.0
    rows[5, 0, 1:4097] = 7.0
    r = nn_amd.beam_select(rows.cuda(), torch.zeros(6, 1).cuda(), 1)
    want = [0.0, 0.0, -math.log((n + 2) // 3), -math.log(n), -math.log(2), -math.log(4096)]
    assert r.tokens[:, 0].tolist() == [17, 4999, 0, 0, 2100, 1]
    for got, ref in zip(r.scores[:, 0].tolist(), want):
        assert abs(got - ref) <= 2.0 ** -22 + 2.0 ** -24 * abs(ref)

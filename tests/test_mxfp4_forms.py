"""Every form of the linears over MXFP4 rows (tiles of the GEMMs, pairs of units of the rows kernel, K in one or several
parts) on operands whose products and sums are exact in f32 in any order, so that the outputs are equal to the
definition's, and f32 x in its norm.

Exactness: a weight row has up to 16 values of +-0.5, 1 or 2 (codes and scales vary) and is zero elsewhere.  x: f32 odd
integers of 17 bits (all three bf16 parts of each count), bf16 integers of 8, or, where it is quantized, blocks that the
grid of their scale holds.  Sums are then multiples of 0.5 below 16 * 2 * 2^17 + 2^10 < 2^23."""
import ctypes
import math
import random

import pytest
import torch

from nn_amd import _lib

F32, BF16, QUANT_BF16, QUANT_F32 = 1, 0, 2, 3  # kinds of x (MxInput); the codes themselves are kind 4
CODES = 4

# (m, n, k): m no multiple of 32, most n odd, stages of K even and odd in number, rows that end inside a unit
CASES = {
    BF16: [
        (17, 94, 1504), (19, 64, 416), (17, 83, 1312), (17, 66, 288), (1399, 263, 3360), (816, 2355, 416),
        (1468, 257, 3200), (1396, 1281, 288), (677, 781, 6528), (2852, 771, 416), (699, 781, 5696), (2837, 771, 288),
        (1025, 1801, 6880), (1348, 2848, 416), (1032, 1913, 7392), (2722, 1329, 288), (1, 64, 32), (16, 237, 3616),
        (1, 64, 288), (6, 1044, 16576), (3, 533, 8288), (4, 777, 12384), (1, 1281, 20480), (12, 6001, 2048),
        (1, 20000, 512),
    ],
    F32: [
        (17, 64, 960), (18, 66, 416), (17, 66, 864), (20, 65, 288), (393, 1027, 2016), (1638, 1075, 416),
        (411, 1063, 2336), (1156, 1549, 288), (15, 805, 12416), (6, 64, 32), (16, 71, 1056), (6, 64, 288),
        (1, 64, 32), (5, 261, 3872), (1, 66, 288), (2, 1055, 16416), (2, 531, 8352), (1, 795, 12704),
        (1, 1281, 20480),
    ],
    QUANT_BF16: [
        (652, 1899, 19200), (1233, 3099, 832), (654, 1836, 20096), (1250, 3129, 544), (1, 64, 32), (16, 941, 14432),
        (1, 64, 288), (15, 1045, 16576), (3, 517, 8256), (1, 796, 12480), (1, 1281, 20480),
    ],
    QUANT_F32: [
        (19, 441, 7008), (18, 65, 800), (18, 241, 3616), (17, 65, 544), (905, 519, 8096), (1161, 1593, 800),
        (683, 771, 8384), (1196, 1539, 544), (1175, 1540, 17280), (2317, 2365, 800), (1155, 1573, 17728),
        (2314, 2343, 544), (1, 64, 32), (16, 909, 14368), (2, 67, 288), (14, 1053, 16544), (3, 515, 8224),
        (5, 777, 12320),
    ],
}


def form(m, n, k, x):
    """(kernel and kind of x, its template's sizes), (K's parts, stages of the smallest)"""
    lib = _lib.load()
    lib.nnq_rule_mx.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_int, ctypes.POINTER(ctypes.c_int)]
    f = (ctypes.c_int * 4)()
    if lib.nnq_rule_mx(m, n, k, x, f):
        kind = x if x != F32 else "one MFMA" if m <= 5 else "planes"
        return ("rows", kind, f[0]), (f[3], 1)
    return ("gemm", min(x, QUANT_BF16), f[0], f[1]), (f[2], f[3])


def test_the_cases_take_every_form():
    """also where the plans change: any form that some shape takes is a case's, GEMMs with K in one part and in several and
    stages even and odd in number"""
    got = {x: [form(m, n, k, x) for m, n, k in shapes] for x, shapes in CASES.items()}
    got[CODES] = [form(m, n, k, CODES) for x in (QUANT_BF16, QUANT_F32) for m, n, k in CASES[x]]
    seen = {f for forms in got.values() for f, _ in forms}
    rng = random.Random(11)
    log = lambda lo, hi: round(lo * (hi / lo) ** rng.random())
    for _ in range(100000):
        m, n, k, x = rng.choice((log(1, 16), log(17, 9000))), log(1, 300000), 32 * log(1, 1 << 15), rng.randrange(5)
        assert form(m, n, k, x)[0] in seen, (m, n, k, x, form(m, n, k, x))
    for f in (f for f in seen if f[0] == "gemm"):
        turns = {(parts > 1, stages % 2) for forms in got.values() for g, (parts, stages) in forms if g == f}
        assert turns == {(False, 0), (False, 1), (True, 0), (True, 1)}, (f, turns)
        assert all(stages >= 3 for forms in got.values() for g, (_, stages) in forms if g == f)


def sparse_weight(n, k, g):
    """codes, scales and (columns, values) of the weights that are not zero"""
    hot = min(k, 16, max(4, -(-k // n)))
    start = torch.randperm(k, generator=g)
    cols = start[(torch.arange(n)[:, None] * hot + torch.arange(hot)) % k]
    e = torch.randint(-2, 2, (n, k // 32), generator=g)
    # codes of powers of two (1, 2, 4, 6 for 0.5, 1, 2, 4) that the block's scale brings to 0.5, 1 or 2
    low, high = torch.tensor([2, 1, 0, 0]), torch.tensor([3, 3, 2, 1])
    at = e.gather(1, cols // 32)
    pick = low[at + 2] + (torch.rand(n, hot, generator=g) * (high - low + 1)[at + 2]).long()
    sign = torch.randint(0, 2, (n, hot), generator=g)
    code = torch.zeros(n, k, dtype=torch.uint8)
    code.scatter_(1, cols, (torch.tensor([1, 2, 4, 6])[pick] + 8 * sign).to(torch.uint8))
    values = (0.5 * 2.0 ** pick.double()) * 2.0 ** at.double() * (1 - 2 * sign)
    assert values.abs().min() >= 0.5 and values.abs().max() <= 2
    return (code[:, 0::2] | code[:, 1::2] << 4).cuda(), (e + 127).to(torch.uint8).cuda(), cols.cuda(), values.cuda()


def exact_x(m, k, kind, g):
    sign = 1 - 2 * torch.randint(0, 2, (m, k), generator=g)
    if kind == F32:
        return (sign * (2 ** 16 + 1 + 2 * torch.randint(0, 2 ** 15, (m, k), generator=g))).float().cuda()
    if kind == BF16:
        return (sign * torch.randint(128, 256, (m, k), generator=g)).bfloat16().cuda()
    q = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])[torch.randint(0, 8, (m, k), generator=g)].view(m, -1, 32)
    q.scatter_(2, torch.randint(0, 32, (m, k // 32, 1), generator=g), 6.0)  # (each scale is the block's own)
    x = (q * 2.0 ** torch.randint(0, 4, (m, k // 32, 1), generator=g)).view(m, k) * sign
    return x.to(torch.bfloat16 if kind == QUANT_BF16 else torch.float32).cuda()


def product(x, cols, values):
    """x @ W^T in 64 bits, for the weights that are not zero"""
    y = torch.zeros(x.shape[0], cols.shape[0], dtype=torch.float64, device="cuda")
    for j in range(cols.shape[1]):
        y += x.double()[:, cols[:, j]] * values[:, j]
    return y


@pytest.mark.gpu
@pytest.mark.parametrize("kind,shape", [(x, s) for x, shapes in CASES.items() for s in shapes])
def test_every_form_is_exact(kind, shape):
    import nn_amd
    m, n, k = shape
    g = torch.Generator().manual_seed(m + 3 * n + 7 * k + kind)
    codes, scales, cols, values = sparse_weight(n, k, g)
    w = nn_amd.QuantizedWeight.from_mxfp4_rows(codes, scales)
    x = exact_x(m, k, kind, g)
    bias = torch.randint(-1024, 1025, (n,), generator=g).float().cuda()
    ref = product(x, cols, values)
    assert ref.abs().max() + 1024 < 2 ** 23 and torch.equal(ref.float().double(), ref)
    calls = [lambda *a, **o: nn_amd.quantized_linear(x, w, *a, **o)]
    if kind >= QUANT_BF16:
        q = nn_amd.quantize_mxfp4_rows(x)
        assert torch.equal(q.dequantize(), x.float())
        calls = [lambda *a, **o: nn_amd.mxfp4_linear(x, w, *a, **o), lambda *a, **o: nn_amd.mxfp4_linear(q, w, *a, **o),
                 lambda *a, **o: nn_amd.mxfp4_linear(x, w, *a, scale_rule="floor", **o)]
    for call in calls:
        for b, out in ((None, torch.float32), (bias, torch.bfloat16), (bias, torch.float32)):
            want = (ref if b is None else ref + b.double()).float().to(out)
            y = call(b, out_dtype=out)
            assert y.dtype is out and torch.equal(y, want), (out, (y != want).nonzero()[:4].tolist())


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 301, 4096), (3, 77, 8224), (5, 261, 3872), (6, 64, 288), (11, 500, 2880), (16, 71, 1056),
                                   (20, 65, 288), (33, 300, 2880), (393, 1027, 2016), (1156, 1549, 288)])
def test_f32_rows_in_their_norm(m, n, k):
    """Dense random operands: 3 K / 16 + 40 roundings to 2^-24 of a partial sum, whose size grows as a random walk's, are
    2^-24 sqrt(N / 6) of the result in the mean; allowed is twice that.  x without its third part would be off by more."""
    import nn_amd
    g = torch.Generator().manual_seed(m + n + k)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8).cuda()
    scales = torch.randint(121, 124, (n, k // 32), generator=g).to(torch.uint8).cuda()
    w = nn_amd.QuantizedWeight.from_mxfp4_rows(codes, scales)
    x = torch.randn(m, k, generator=g).cuda()
    full = w.dequantize().double()
    ref = x.double() @ full.t()
    bar = 2 * 2.0 ** -24 * math.sqrt((3 * k / 16 + 40) / 6)
    cut = (x.view(torch.int32) & ~0xFF).view(torch.float32)
    assert (cut.double() @ full.t() - ref).norm() > bar * ref.norm()
    y = nn_amd.quantized_linear(x, w)
    assert (y.double() - ref).norm() <= bar * ref.norm(), ((y.double() - ref).norm() / ref.norm()).item()

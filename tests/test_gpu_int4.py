"""GPU parity of linears over 4-bit codes with group scales against a plain product in 64 bits, at the
edges of the kernels' forms: one row, two, eight and nine (f32 x as row pairs or as planes), sixteen and
seventeen and prefills; N below a tile, past one, no whole number of tiles, more tiles than two per CU; K
of one group, inside a unit of 128, one pass, several passes; each group size, scale type, with and
without zero points.

Bar (f32 outputs): every product of an integer and an f16 is exact in f32; f32 x enters as an f16 hi + lo
pair that drops at most 2^-22 of it.  What is left is rounding of f32 sums and scalings, 2^-24 each of
partial sums that stay within a few times the output's own size, some 40 in line: max |error| <= 1e-5 of
the output's root mean square.  A bf16 output is the f32 result rounded once, bit for bit."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def dev():
    import nn_amd
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    nn_amd.init(0)
    return torch.device("cuda:0")


def make(n, k, group, zeros=True, scale=F16, seed=1):
    """(weight, W in 64 bits)"""
    import nn_amd
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    q = torch.randint(0, 16, (n, k), generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
    s = (0.004 + 0.008 * torch.rand(n, k // group, generator=g, device="cuda")).to(scale)
    s = s * torch.where(torch.rand(n, k // group, generator=g, device="cuda") < 0.1, -1.0, 1.0).to(scale)
    z = torch.randint(0, 17, (n, k // group), generator=g, device="cuda") if zeros else None
    w = nn_amd.QuantizedWeight.from_int4_groups(q[:, 0::2] | (q[:, 1::2] << 4), s, z, group)
    zz = 8.0 if z is None else z.double().repeat_interleave(group, 1)
    return w, (q.double() - zz) * s.double().repeat_interleave(group, 1)


def tokens(m, k, dtype, seed=2):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(m, k, generator=g, device="cuda") * torch.exp(torch.randn(k, generator=g, device="cuda"))).to(dtype)


def check(y, ref, what="", bias=None):
    """``bias`` was added to ``ref``'s product: it may cancel the product (one output: to any extent), whose
    rounding errors are of its own size and stay, and the addition rounds once, 2^-24 of at most the two's
    sum.  So the size that counts is then the root mean square of the product and of the bias together."""
    assert y.shape == ref.shape and torch.isfinite(y).all()
    size = ref.pow(2).mean()
    if bias is not None:
        b = bias.double()
        size = (ref - b).pow(2).mean() + b.pow(2).mean()
    err = (y.double() - ref).abs().max().item() / size.sqrt().item()
    assert err <= 1e-5, f"{what} max error {err:.2e} of the output's rms"


@pytest.mark.parametrize("n,k,group,zeros,scale", [(1, 32, 32, True, F16), (17, 160, 32, False, BF16), (16, 128, 128, True, BF16),
                                                   (100, 2880, 64, True, F16), (33, 1152, 128, False, F16)])
def test_dequantize_is_exact(n, k, group, zeros, scale):
    w, ref = make(n, k, group, zeros, scale)
    assert w.shape == (n, k) and w.quant_type == 1000
    assert torch.equal(w.dequantize().double(), ref)  # 5 bits times 11 (8): no rounding


@pytest.mark.parametrize("zeros", [True, False])
@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (17, 160, 32), (16, 128, 128), (100, 2880, 64), (333, 1152, 128), (8209, 4224, 32)])
def test_image_made_on_the_device(n, k, group, zeros):
    """The same weight from host arrays, device arrays and an odd view of them."""
    import nn_amd
    g = torch.Generator()
    g.manual_seed(n)
    flat = torch.randint(0, 256, (n * k // 2 + 1,), generator=g, dtype=torch.int32).to(torch.uint8)
    c = flat[1:].view(n, k // 2)
    s = (0.01 * torch.randn(n, k // group, generator=g)).half()
    z = torch.randint(0, 17, (n, k // group), generator=g) if zeros else None
    make = lambda *t: nn_amd.QuantizedWeight.from_int4_groups(*t, group)  # noqa: E731
    host, x = make(c, s, z), tokens(20, k, BF16)
    ref, y = host.dequantize(), nn_amd.quantized_linear(x, host)
    cz = None if z is None else z.cuda()
    for w in (make(c.cuda(), s.cuda(), cz), make(flat.cuda()[1:].view(n, k // 2), s, z), make(c, s.cuda(), cz)):
        assert torch.equal(w.dequantize(), ref) and torch.equal(nn_amd.quantized_linear(x, w), y)
    bad = s.clone()
    bad[n // 2, -1] = float("inf")
    with pytest.raises(nn_amd.NonFiniteData, match=str((n // 2 + 1) * (k // group) - 1)):
        make(c.cuda(), bad, z)
    if zeros:
        bad = z.to(torch.uint8)
        bad[-1, 0] = 17
        with pytest.raises(nn_amd.TensorError, match="zero point"):
            make(c.cuda(), s, bad)


SHAPES = [(1, 1, 32, 32), (1, 5, 64, 64), (2, 40, 128, 128), (3, 16, 160, 32), (1, 300, 2880, 64), (8, 33, 1152, 128),
          (9, 100, 2912, 32), (16, 257, 4096, 128), (1, 8209, 640, 128), (5, 8304, 4096, 64), (12, 8193, 5120, 32),
          (7, 64, 12288, 128), (16, 48, 8320, 64), (1, 9000, 4224, 128)]


@pytest.mark.parametrize("xdt", [F32, BF16])
@pytest.mark.parametrize("zeros,scale", [(True, F16), (False, F16), (True, BF16)])
@pytest.mark.parametrize("m,n,k,group", SHAPES)
def test_rows(m, n, k, group, zeros, scale, xdt):
    import nn_amd
    w, ref = make(n, k, group, zeros, scale)
    x = tokens(m, k, xdt)
    bias = torch.randn(n, device="cuda")
    ref = x.double() @ ref.t()
    check(nn_amd.quantized_linear(x, w), ref)
    y = nn_amd.quantized_linear(x, w, bias)
    check(y, ref + bias.double(), bias=bias)
    assert torch.equal(nn_amd.quantized_linear(x, w, bias, out_dtype=BF16), y.to(BF16))


# up to 16 units of K: one a wave, with one tile at a time or two, in workgroups of 16, 8 and 4 waves
SHORT_K = [(1, 8304, 2048, 64), (4, 8193, 1984, 32), (3, 17000, 1024, 128), (2, 33025, 512, 128), (1, 40000, 96, 32),
           (7, 9000, 1920, 64), (8, 300, 2048, 128), (13, 8300, 2048, 128), (16, 500, 1152, 128), (5, 16500, 640, 128)]


@pytest.mark.parametrize("xdt", [F32, BF16])
@pytest.mark.parametrize("zeros", [True, False])
@pytest.mark.parametrize("m,n,k,group", SHORT_K)
def test_rows_of_a_short_k(m, n, k, group, zeros, xdt):
    import nn_amd
    w, ref = make(n, k, group, zeros)
    x = tokens(m, k, xdt)
    y = nn_amd.quantized_linear(x, w)
    check(y, x.double() @ ref.t())
    if m == 1 and xdt is F32:
        logits, idx = nn_amd.linear_argmax(x, w)
        assert torch.equal(logits, y[0]) and idx.item() == int(torch.nonzero(y[0] == y.max())[0])


PREFILL = [(17, 16, 128, 128), (33, 300, 160, 32), (48, 129, 2880, 64), (64, 257, 1152, 128), (130, 1000, 4096, 128),
           (203, 512, 2912, 32), (300, 4100, 640, 64), (513, 264, 4224, 128), (1, 512, 1024, 128)]


@pytest.mark.parametrize("xdt", [F32, BF16])
@pytest.mark.parametrize("zeros", [True, False])
@pytest.mark.parametrize("m,n,k,group", PREFILL)
def test_prefill(m, n, k, group, zeros, xdt):
    import nn_amd
    w, ref = make(n, k, group, zeros, BF16 if n % 2 else F16)
    x = tokens(m, k, xdt)
    bias = torch.randn(n, device="cuda")
    ref = x.double() @ ref.t() + bias.double()
    y = nn_amd.quantized_linear(x, w, bias)
    check(y, ref)
    assert torch.equal(nn_amd.quantized_linear(x, w, bias, out_dtype=BF16), y.to(BF16))


def test_leading_dimensions_views_and_empty():
    import nn_amd
    w, ref = make(70, 256, 64)
    x = tokens(12, 512, F32)
    y = nn_amd.quantized_linear(x[:, :256].view(3, 4, 256), w)  # strided rows
    check(y, (x[:, :256].double() @ ref.t()).view(3, 4, 70))
    flat = torch.empty(2 * 256 + 1, device="cuda")
    v = flat[1:].view(2, 256)  # 4 bytes past an aligned address
    v.copy_(x[:2, :256])
    check(nn_amd.quantized_linear(v, w), v.double() @ ref.t())
    check(nn_amd.quantized_linear(x[:, :256].half(), w), x[:, :256].half().double() @ ref.t())
    assert nn_amd.quantized_linear(x[:0, :256], w).shape == (0, 70)
    with pytest.raises(nn_amd.ShapeMismatch):
        nn_amd.quantized_linear(x, w)


@pytest.mark.parametrize("m", [1, 16, 40])
@pytest.mark.parametrize("xdt", [F32, BF16])
def test_activation_range(m, xdt):
    """Rows of very small and very large activations, a row of zeros, and one with zeros but for one value: the
    power of two of a row and unit keeps each row's precision its own."""
    import nn_amd
    w, ref = make(48, 384, 128)
    x = tokens(m, 384, xdt)
    x = x * torch.tensor([1e-30, 1.0, 1e30, 0.0] * 10, device="cuda")[:m, None].to(xdt)
    if m > 4:
        x[4] = 0
        x[4, 200] = 3.0
    y = nn_amd.quantized_linear(x, w)
    r = x.double() @ ref.t()
    for t in range(m):
        rms = r[t].pow(2).mean().sqrt().item()
        assert (y[t].double() - r[t]).abs().max().item() <= 1e-5 * rms, t


@pytest.mark.parametrize("m", [1, 6, 12, 40])
def test_smallest_and_largest_scales(m):
    """f16 scales below the smallest normal one and at the largest, each the only ones of a weight."""
    import nn_amd
    for value in (2.0 ** -24, 3 * 2.0 ** -20, 65504.0):
        q = torch.randint(0, 256, (50, 192), dtype=torch.int32).to(torch.uint8)
        s = torch.full((50, 6), value, dtype=F16)
        w = nn_amd.QuantizedWeight.from_int4_groups(q.cuda(), s, None, 64)
        codes = torch.stack([q & 15, q >> 4], 2).view(50, 384).double().cuda() - 8
        assert torch.equal(w.dequantize().double(), codes * value)
        for xdt in (F32, BF16):
            x = tokens(m, 384, xdt)
            check(nn_amd.quantized_linear(x, w), x.double() @ (codes * value).t(), value)


@pytest.mark.parametrize("m", [1, 6, 12, 40])
def test_smallest_and_largest_bf16_scales(m):
    """The smallest subnormal one, the smallest normal one and the largest that is taken, each the only ones of a
    weight; and the smallest that is refused, from host and device arrays.  (x brings the results to where f32 is
    normal.)"""
    import nn_amd
    q = torch.randint(0, 256, (50, 192), generator=torch.Generator().manual_seed(m), dtype=torch.int32).to(torch.uint8)
    codes = torch.stack([q & 15, q >> 4], 2).view(50, 384).double().cuda() - 8
    for value, size in ((2.0 ** -133, 2.0 ** 40), (2.0 ** -126, 2.0 ** 40), (255 * 2.0 ** 80, 1.0), (255 * 2.0 ** 80, 2.0 ** -30)):
        s = torch.full((50, 6), value, dtype=BF16)
        assert s[0, 0].double().item() == value
        w = nn_amd.QuantizedWeight.from_int4_groups(q.cuda(), s, None, 64)
        assert torch.equal(w.dequantize().double(), codes * value)
        for xdt in (F32, BF16):
            x = tokens(m, 384, xdt) * size
            check(nn_amd.quantized_linear(x, w), x.double() @ (codes * value).t(), value)
    for bad in (2.0 ** 88, -2.0 ** 110):
        s[7, 3] = bad
        for c in (q, q.cuda()):
            with pytest.raises(nn_amd.Unsupported, match="scale 45 "):
                nn_amd.QuantizedWeight.from_int4_groups(c, s, None, 64)


@pytest.mark.parametrize("m", [1, 6, 12, 40])
@pytest.mark.parametrize("xdt", [F32, BF16])
def test_largest_finite_activations(m, xdt):
    """Activations up to the type's largest value are numbers, not infinities: rows of 3.1e38 to 3.38e38 beside
    ordinary ones, scales that keep the results in f32's range."""
    import nn_amd
    g = torch.Generator(device="cuda")
    g.manual_seed(m)
    q = torch.randint(0, 256, (50, 192), generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
    codes = torch.stack([q & 15, q >> 4], 2).view(50, 384).double() - 8
    w = nn_amd.QuantizedWeight.from_int4_groups(q, torch.full((50, 3), 2.0 ** -24, dtype=F16), None, 128)
    x = tokens(m, 384, xdt)
    big = 3.1e38 + 0.28e38 * torch.rand(384, generator=g, device="cuda")
    x[0] = big.to(xdt) * torch.where(torch.rand(384, generator=g, device="cuda") < 0.5, -1.0, 1.0).to(xdt)
    x[m // 2, 100] = torch.finfo(xdt).max
    assert torch.isfinite(x).all()
    y, ref = nn_amd.quantized_linear(x, w), x.double() @ (codes * 2.0 ** -24).t()
    for t in range(m):
        check(y[t], ref[t], t)


@pytest.mark.parametrize("m", [1, 6, 12, 40])
def test_activations_below_the_smallest_normal(m):
    """f32 x of multiples of 2^-140 (subnormal: nine bits are left), scales that bring the result back up."""
    import nn_amd
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    q = torch.randint(0, 256, (40, 128), generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
    w = nn_amd.QuantizedWeight.from_int4_groups(q, torch.full((40, 2), 65504.0, dtype=F16), None, 128)
    codes = torch.stack([q & 15, q >> 4], 2).view(40, 256).double() - 8
    x = torch.randint(-400, 401, (m, 256), generator=g, device="cuda").float() * 2.0 ** -140
    assert x.abs().max() < torch.finfo(F32).tiny and x.abs().max() > 0
    check(nn_amd.quantized_linear(x, w), x.double() @ (codes * 65504.0).t())


def test_threads_on_their_own_streams_and_on_one():
    """Calls of two host threads, each on a stream of its own, then both on one."""
    import threading
    import nn_amd
    w, _ = make(4500, 9600, 64)
    xs = [tokens(m, 9600, F32, seed=m) for m in (7, 40)]
    want = [nn_amd.quantized_linear(x, w) for x in xs]
    torch.cuda.synchronize()
    one = torch.cuda.Stream()
    for streams in ([torch.cuda.Stream(), torch.cuda.Stream()], [one, one]):
        bad = []

        def loop(i):
            with torch.cuda.stream(streams[i]):
                for _ in range(30):
                    if not torch.equal(nn_amd.quantized_linear(xs[i], w), want[i]):
                        bad.append(i)

        threads = [threading.Thread(target=loop, args=(i,)) for i in range(2)]
        [t.start() for t in threads]
        [t.join() for t in threads]
        torch.cuda.synchronize()
        assert not bad


@pytest.mark.parametrize("m", [1, 3, 12, 30])
def test_non_finite_activations_stay_in_their_row(m):
    import nn_amd
    w, ref = make(40, 512, 64)
    for bad in (float("nan"), float("inf"), -float("inf")):
        for xdt in (F32, BF16):
            x = tokens(m, 512, xdt)
            x[m // 2, 77] = bad
            y = nn_amd.quantized_linear(x, w)
            assert torch.isnan(y[m // 2]).all()
            keep = [t for t in range(m) if t != m // 2]
            if keep:
                check(y[keep], x[keep].double() @ ref.t())


def test_argmax_and_sampling_through_an_int4_head():
    import nn_amd
    for n, k, group in ((1, 128, 128), (50, 256, 32), (9001, 512, 64), (32017, 4224, 128)):
        w, ref = make(n, k, group)
        x = tokens(1, k, F32)
        y = nn_amd.quantized_linear(x, w)[0]
        logits, idx = nn_amd.linear_argmax(x, w)
        assert torch.equal(logits, y) and idx.item() == int(torch.nonzero(y == y.max())[0])
        logits, tok = nn_amd.linear_sample(x, w, temperature=1e-6, top_k=1, top_p=None)
        assert torch.equal(logits, y) and y[tok] == y.max()
    x[0, 3] = float("nan")
    with pytest.raises(nn_amd.NonFiniteData):
        nn_amd.linear_argmax(x, w)


@pytest.mark.parametrize("m", [5, 9, 16])
@pytest.mark.parametrize("xdt", [F32, BF16])
def test_rows_over_a_split_k(m, xdt):
    """K split over workgroups: a row of NaN stays a row of NaN, the others and a replayed graph are right."""
    import nn_amd
    w, ref = make(4500, 9600, 64)  # 75 units: parts of unequal length
    x = tokens(m, 9600, xdt)
    x[m // 2, 9599] = float("nan")
    keep = [t for t in range(m) if t != m // 2]
    nn_amd.quantized_linear(x, w)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = nn_amd.quantized_linear(x, w)
    for i in range(3):
        x[keep] = tokens(m, 9600, xdt, seed=20 + i)[keep]
        eager = nn_amd.quantized_linear(x, w)
        g.replay()
        torch.cuda.synchronize()
        assert torch.isnan(y[m // 2]).all() and torch.equal(y[keep], eager[keep])
        check(y[keep], x[keep].double() @ ref.t())


def test_rows_in_several_launches():
    """More rows than one launch stages: the rows on both sides of the edge, the first and the last."""
    import nn_amd
    w, ref = make(24, 32768, 128)
    x = tokens(8200, 32768, BF16)
    y = nn_amd.quantized_linear(x, w)
    rows = list(range(0, 8200, 411)) + list(range(8050, 8080)) + [8199]
    check(y[rows], x[rows].double() @ ref.t())


def test_outputs_past_32_bits():
    import nn_amd
    w, ref = make(17000, 128, 64)
    x = tokens(66000, 128, BF16)
    y = nn_amd.quantized_linear(x, w)  # 4.5 GB
    rows = [0, 31999, 65535, 65536, 65999] + list(range(63150, 63180))  # 63161 x 17000 x 4 bytes is 2^32
    check(y[rows], x[rows].double() @ ref.t())


def test_sampling_without_allocation_through_an_int4_head():
    from nn_amd import _lib
    w, _ = make(9001, 4224, 64)
    x = tokens(1, 4224, F32)[0].contiguous()
    for top_k, top_p, seed in ((20, 0.9, 3), (50, 1.0, 8)):
        cfg = _lib.Sampling(0.7, top_k, 1, top_p, 1.0, 0.0, seed)
        out = []
        for name in ("nnq_linear_sample", "nnq_linear_sample_noalloc"):
            logits, tok = torch.empty(9001, device="cuda"), torch.full((1,), -1, dtype=torch.int32, device="cuda")
            rc = getattr(_lib.load(), name)(w.handle, x.data_ptr(), 4224, None, 0, logits.data_ptr(), None, 0,
                                            ctypes.byref(cfg), tok.data_ptr(), torch.cuda.current_stream().cuda_stream)
            assert rc == 0, _lib.last_error()
            out.append((logits, int(tok)))
        assert torch.equal(out[0][0], out[1][0]) and out[0][1] == out[1][1] >= 0


@pytest.mark.parametrize("m", [1, 16, 40, 200])
def test_captured_graph_beside_eager_calls(m):
    """A captured linear replayed with new inputs, eager calls of other sizes on the stream between the replays."""
    import nn_amd
    w, ref = make(500, 1152, 128)
    w2, _ = make(64, 4096, 64, seed=9)
    x = tokens(m, 1152, BF16)
    nn_amd.quantized_linear(x, w)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = nn_amd.quantized_linear(x, w)
    for i in range(4):
        x.copy_(tokens(m, 1152, BF16, seed=50 + i))
        nn_amd.quantized_linear(tokens(300, 4096, F32, seed=i), w2)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, nn_amd.quantized_linear(x, w)), i
        check(y, x.double() @ ref.t())


def test_same_results_every_time_and_on_another_stream():
    import nn_amd
    w, _ = make(8300, 4224, 64)
    for m in (1, 13, 100):
        x = tokens(m, 4224, F32)
        y = nn_amd.quantized_linear(x, w)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            z = nn_amd.quantized_linear(x, w)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(y, z) and torch.equal(y, nn_amd.quantized_linear(x, w))

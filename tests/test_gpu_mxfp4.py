"""GPU parity of MXFP4 rows against their definitions in 64 bits: quantization and its inverse (equal), the linears over
an MXFP4 weight with x as it is and with x quantized too.

Bars of the linears: a product of an activation (bf16: 8 significant bits, an f32's three parts 8 each, a code 2) and a
weight (2 bits) is exact in f32, so only the sums round.  An MFMA adds its 16 to 128 products to the running sum in at
most four roundings or cuts of 2^-23 of the magnitudes in play, which are at most S = sum |x| |w| (3 S for the three
parts' separate sums, whose magnitudes add to at most 2 |x|); a row of K has at most K / 16 of them a part, and up to 40
further additions join waves, parts of K and the bias: |error| <= (3 * 4 K / 16 + 40) 2^-23 (S + |bias|), plus 2^-8 of
the result where it is rounded to bf16."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
INF, NAN = float("inf"), float("nan")
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


@pytest.fixture(scope="module", autouse=True)
def dev():
    import nn_amd
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    nn_amd.init(0)
    return torch.device("cuda:0")


def decode(codes, scales):
    """f64 values on the host; a block of scale 255 is NaN"""
    c, s = codes.cpu().long(), scales.cpu().double()
    g = torch.cat((GRID, -GRID))
    v = torch.stack((g[c & 15], g[c >> 4]), -1).flatten(-2)
    s = torch.where(s == 255, NAN, 2.0 ** (s - 127))
    return v * s.repeat_interleave(32, -1)


def quantize(x, rule):
    """(values, scale bytes) in f64 on the host, straight from the definition"""
    b = x.double().cpu().unflatten(-1, (-1, 32))
    m = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    s = torch.full_like(m, -127.0)
    for e in range(-127, 126):  # floor: the largest e with 4 * 2^e <= m; ceil: the smallest with m <= 6 * 2^e
        if rule == "floor":
            s = torch.where(m >= 4 * 2.0 ** e, float(e), s)
        elif e > -127:
            s = torch.where(m > 6 * 2.0 ** (e - 1), float(e), s)
    v = b / (2.0 ** s)[..., None]
    d = (v.abs()[..., None] - GRID).abs()
    lo = d.argmin(-1)
    near = d.gather(-1, lo[..., None])[..., 0]
    up = (lo + 1).clamp(max=7)
    tie = (d.gather(-1, up[..., None])[..., 0] == near) & (up > lo) & (lo % 2 == 1)
    q = GRID[torch.where(tie, up, lo)] * torch.sign(v)
    values = torch.where(bad[..., None], NAN, q * (2.0 ** s)[..., None]).flatten(-2)
    return values, torch.where(bad, 255, (s + 127)).to(torch.uint8)


def same(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    assert a.shape == b.shape
    assert torch.equal(torch.isnan(a), torch.isnan(b))
    ok = ~torch.isnan(b)
    assert torch.equal(a[ok], b[ok])


def hard_rows(k, g):
    """rows of many magnitudes: ordinary, tiny, subnormal, huge, on the grid and on its midpoints, zeros"""
    n = k // 32
    rows = [torch.randn(k, generator=g) * 2.0 ** p for p in (0, -20, -126, -140, -149, 60, 120)]
    grid = (torch.randint(-28, 29, (k,), generator=g).double() / 4).float()
    rows += [grid, grid * 2.0 ** -90, grid * 2.0 ** 100, torch.zeros(k), torch.sign(torch.randn(k, generator=g)) * 3.4e38]
    one = torch.zeros(k)
    one[torch.randint(0, k, (n,), generator=g)] = -7.0
    rows += [one, torch.nextafter(grid, torch.tensor(INF)), torch.nextafter(grid, torch.tensor(-INF))]
    spread = torch.randn(k, generator=g) * 2.0 ** torch.randint(-30, 30, (k,), generator=g).float()
    return torch.stack(rows + [spread])


@pytest.mark.parametrize("rule", ["ceil", "floor"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("k", [32, 96, 2080])
def test_quantize_hard_values(dtype, rule, k):
    import nn_amd
    x = hard_rows(k, torch.Generator().manual_seed(k)).to(dtype)
    r = nn_amd.quantize_mxfp4_rows(x.cuda(), rule)
    values, scales = quantize(x, rule)
    assert torch.equal(r.scales.cpu(), scales)
    same(decode(r.codes, r.scales), values)
    same(r.dequantize(), values)
    assert r.dequantize(BF16).dtype is BF16
    same(r.dequantize(BF16), values)


@pytest.mark.parametrize("rows,k", [(1, 32), (1, 4096), (3, 2880), (517, 160), (2049, 64), (70000, 32)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize_sizes(rows, k, dtype):
    import nn_amd
    x = torch.randn(rows, k, generator=torch.Generator().manual_seed(rows)).to(dtype)
    r = nn_amd.quantize_mxfp4_rows(x.cuda())
    values, scales = quantize(x, "ceil")
    assert torch.equal(r.scales.cpu(), scales)
    same(r.dequantize(), values)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize_bad_values_stay_in_their_block(dtype):
    import nn_amd
    x = torch.randn(4, 128, generator=torch.Generator().manual_seed(5)).to(dtype)
    x[0, 3], x[1, 64], x[2, 127], x[3, 40] = NAN, INF, -INF, NAN
    r = nn_amd.quantize_mxfp4_rows(x.cuda())
    values, scales = quantize(x, "ceil")
    assert torch.equal(r.scales.cpu(), scales) and int((r.scales == 255).sum()) == 4
    assert not r.codes.view(4, 4, 16)[r.scales == 255].any()
    same(r.dequantize(), values)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize_strides_and_shapes(dtype):
    import nn_amd
    base = torch.randn(9, 5, 203, generator=torch.Generator().manual_seed(1)).cuda().to(dtype)
    for x in (base[:, 1, 3:195], base[:, :, :192], base[2, 0, 1:161], base[:0, :, :64], base.transpose(0, 2)[:, :, :0].transpose(0, 2)[:, :, :32],
              base[:, 2, :192].expand(9, 192), base[3:4, 0, 7:167], base[::2, ::2, 11:171], base[0, :, :192:2].contiguous()):
        r = nn_amd.quantize_mxfp4_rows(x)
        assert r.codes.shape == (*x.shape[:-1], x.shape[-1] // 2) and r.scales.shape == (*x.shape[:-1], x.shape[-1] // 32)
        if x.numel():
            same(r.dequantize(), quantize(x, "ceil")[0])
    t = torch.randn(64, 96, generator=torch.Generator().manual_seed(2)).cuda().to(dtype).t()[:, :32]  # columns apart
    same(nn_amd.quantize_mxfp4_rows(t).dequantize(), quantize(t, "ceil")[0])
    same(nn_amd.quantize_mxfp4_rows(base[1, :1, :32].expand(6, 32)).dequantize(), quantize(base[1, :1, :32].expand(6, 32), "ceil")[0])
    h = torch.randn(3, 64, generator=torch.Generator().manual_seed(3)).half().cuda()  # widened
    same(nn_amd.quantize_mxfp4_rows(h).dequantize(), quantize(h, "ceil")[0])


def test_quantize_agrees_with_the_host_encoder_off_the_midpoints():
    """the blocks of quantize_mxfp4_ocp, whose halves go to the smaller magnitude: continuous values have none"""
    import nn_amd
    x = torch.randn(40, 256, generator=torch.Generator().manual_seed(8)) * 0.02
    r = nn_amd.quantize_mxfp4_rows(x.cuda())
    blocks = torch.from_numpy(nn_amd.quantize_mxfp4_ocp(x.numpy())).view(-1, 17)
    assert torch.equal(r.scales.cpu().view(-1), blocks[:, 0])
    assert torch.equal(r.codes.cpu().view(-1, 16), blocks[:, 1:])
    same(r.dequantize().view(-1), nn_amd.dequantize_mxfp4_ocp(blocks.numpy(), x.numel()))


# ---- linears ------------------------------------------------------------------------------


def weight(n, k, seed, spread=6, on="cuda"):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(121 - spread, 121 + spread, (n, k // 32), generator=g).to(torch.uint8)
    return codes.to(on), scales.to(on)


def bar(x, w, bias, y, out):
    s = x.abs().double() @ w.abs().t() + (0 if bias is None else bias.abs().double())
    b = (3 * 4 * w.shape[1] / 16 + 40) * 2.0 ** -23 * s
    return b + (2.0 ** -8 * (y.abs() + b) if out is BF16 else 0)


def check_linear(y, x, w, bias, out):
    """y against x @ w^T + bias in f64, x and w the values that are multiplied"""
    x, w = x.double().cpu(), w.double().cpu()
    ref = x @ w.t() + (0 if bias is None else bias.double().cpu())
    err = (y.double().cpu() - ref).abs()
    over = err - bar(x, w, None if bias is None else bias.cpu(), ref, out)
    assert y.dtype is out and y.shape == ref.shape
    assert torch.isfinite(y).all()
    assert over.max().item() <= 0, f"over the bar by {over.max().item():.2e}"


# (few and many columns, K in one to several parts, units that end inside a pair, f32 rows whose planes share an MFMA and
# those that do not; the larger tiles and longer rows that test_mxfp4_forms.py lists are not among them)
SHAPES = [(1, 1, 32), (1, 16, 128), (2, 33, 96), (3, 300, 2880), (5, 129, 4128), (6, 257, 2112), (8, 512, 8192), (13, 40, 224),
          (16, 1000, 512), (17, 64, 32), (31, 129, 160), (33, 300, 2880), (64, 255, 384), (65, 513, 1056), (130, 70, 4096),
          (200, 1025, 640), (301, 384, 2208), (4, 9000, 288), (12, 6001, 1024), (7, 5000, 5152), (9, 4100, 9216), (16, 8200, 4096),
          (40, 13000, 1024), (260, 6200, 512), (520, 4200, 256)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("x_dtype", [F32, BF16])
def test_linear(m, n, k, x_dtype):
    import nn_amd
    codes, scales = weight(n, k, n + k)
    w = nn_amd.QuantizedWeight.from_mxfp4_rows(codes, scales)
    assert w.shape == (n, k) and w.quant_type == nn_amd.QuantType.MXFP4 and w.layout == nn_amd.Layout.ROWS
    ref = decode(codes, scales)
    same(w.dequantize(), ref)
    g = torch.Generator().manual_seed(m)
    x = (torch.randn(m, k, generator=g) * torch.exp(torch.randn(k, generator=g))).to(x_dtype)
    bias = torch.randn(n, generator=g)
    check_linear(nn_amd.quantized_linear(x.cuda(), w), x, ref, None, F32)
    check_linear(nn_amd.quantized_linear(x.cuda(), w, bias.cuda(), out_dtype=BF16), x, ref, bias, BF16)


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("x_dtype", [F32, BF16])
def test_product_of_4_bit_operands(m, n, k, x_dtype):
    import nn_amd
    codes, scales = weight(n, k, 2 * n + k)
    w = nn_amd.QuantizedWeight.from_mxfp4_rows(codes, scales)
    ref = decode(codes, scales)
    g = torch.Generator().manual_seed(m + 1)
    x = (torch.randn(m, k, generator=g) * torch.exp(torch.randn(k, generator=g))).to(x_dtype)
    bias = torch.randn(n, generator=g)
    for rule in ("ceil", "floor"):
        q = quantize(x, rule)[0]
        check_linear(nn_amd.mxfp4_linear(x.cuda(), w, scale_rule=rule), q, ref, None, F32)
    y = nn_amd.mxfp4_linear(x.cuda(), w, bias.cuda(), out_dtype=BF16)
    check_linear(y, quantize(x, "ceil")[0], ref, bias, BF16)
    # rows quantized before are the same product
    assert torch.equal(y, nn_amd.mxfp4_linear(nn_amd.quantize_mxfp4_rows(x.cuda()), w, bias.cuda(), out_dtype=BF16))


def test_linear_extreme_scales():
    """weights from 2^-128 to 6 * 2^125, activations of the opposite size: bf16 holds every factor exactly"""
    import nn_amd
    k = 256
    codes, _ = weight(48, k, 3)
    for byte, size in ((0, 2.0 ** 120), (1, 2.0 ** 100), (60, 2.0 ** 60), (200, 2.0 ** -80), (252, 2.0 ** -110)):
        scales = torch.full((48, k // 32), byte, dtype=torch.uint8, device="cuda")
        w = nn_amd.QuantizedWeight.from_mxfp4_rows(codes, scales)
        ref = decode(codes, scales)
        same(w.dequantize(), ref)
        for m in (2, 20):
            for dt in (F32, BF16):
                x = (torch.randn(m, k, generator=torch.Generator().manual_seed(m)) * size).to(dt)
                check_linear(nn_amd.quantized_linear(x.cuda(), w), x, ref, None, F32)
                check_linear(nn_amd.mxfp4_linear(x.cuda(), w), quantize(x, "ceil")[0], ref, None, F32)


@pytest.mark.parametrize("m", [1, 5, 12, 40, 200])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_of_nan_and_infinity_keep_to_themselves(m, dtype):
    """K ends inside a unit and a bad row is a neighbour of every other one"""
    import nn_amd
    n, k = 70, 2080
    codes, scales = weight(n, k, 9)
    w = nn_amd.QuantizedWeight.from_mxfp4_rows(codes, scales)
    ref = decode(codes, scales)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(m)).to(dtype)
    bad = list(range(0, m, 2)) if m > 1 else [0]
    full = torch.full((m, k), NAN, dtype=dtype, device="cuda")
    nn_amd.quantized_linear(full, w), nn_amd.mxfp4_linear(full, w)  # (what they leave on the chip is NaN)
    x[bad[0], 0] = INF
    for r in bad[1:]:
        x[r, -1] = NAN
    good = [r for r in range(m) if r not in bad]
    y = nn_amd.quantized_linear(x.cuda(), w)
    z = nn_amd.mxfp4_linear(x.cuda(), w)
    assert torch.isnan(z[bad]).all() and not torch.isfinite(y[bad]).any()
    if good:
        check_linear(y[good], x[good], ref, None, F32)
        check_linear(z[good], quantize(x[good], "ceil")[0], ref, None, F32)


def test_linear_misaligned_strided_and_batched_inputs():
    import nn_amd
    n, k = 130, 416
    codes, scales = weight(n, k, 4)
    w = nn_amd.QuantizedWeight.from_mxfp4_rows(codes, scales)
    ref = decode(codes, scales)
    for dt in (F32, BF16):
        base = torch.randn(40, 2 * k + 3, generator=torch.Generator().manual_seed(7)).cuda().to(dt)
        flat = base.reshape(-1)
        for x in (base[:, 1:1 + k], base[::3, 3:3 + k], flat[1:1 + 3 * k].view(3, k), flat[3:3 + 24 * k].view(2, 3, 4, k), base[:0, :k]):
            y, z = nn_amd.quantized_linear(x, w), nn_amd.mxfp4_linear(x, w)
            assert y.shape == z.shape == (*x.shape[:-1], n)
            if x.numel():
                v = x.reshape(-1, k)
                check_linear(y.reshape(-1, n), v, ref, None, F32)
                check_linear(z.reshape(-1, n), quantize(v, "ceil")[0], ref, None, F32)
        q = nn_amd.quantize_mxfp4_rows(flat[:24 * k].view(2, 3, 4, k))
        z = nn_amd.mxfp4_linear(q, w)
        check_linear(z.reshape(-1, n), quantize(flat[:24 * k].view(-1, k), "ceil")[0], ref, None, F32)
        odd = torch.empty(q.codes.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view(q.codes.shape)
        odd.copy_(q.codes)
        assert torch.equal(z, nn_amd.mxfp4_linear(nn_amd.Mxfp4Rows(odd, q.scales), w))
        same(nn_amd.Mxfp4Rows(odd, q.scales).dequantize(), q.dequantize())


def test_weight_from_host_views_and_blocks():
    import nn_amd
    n, k = 75, 352
    codes, scales = weight(n, k, 6)
    ref = decode(codes, scales)
    same(nn_amd.QuantizedWeight.from_mxfp4_rows(codes.cpu(), scales.cpu()).dequantize(), ref)
    wide = torch.zeros(n, k // 2 + 5, dtype=torch.uint8, device="cuda")
    wide[:, 5:] = codes
    same(nn_amd.QuantizedWeight.from_mxfp4_rows(wide[:, 5:], scales).dequantize(), ref)
    flat = torch.zeros(n * k // 2 + 1, dtype=torch.uint8, device="cuda")
    flat[1:] = codes.view(-1)
    same(nn_amd.QuantizedWeight.from_mxfp4_rows(flat[1:].view(n, -1), scales.cpu()).dequantize(), ref)
    v = torch.randn(n, k, generator=torch.Generator().manual_seed(1)) * 0.02
    b = torch.from_numpy(nn_amd.quantize_mxfp4_ocp(v.numpy())).view(n, -1, 17)
    w = nn_amd.QuantizedWeight.from_mxfp4_rows(b[..., 1:].reshape(n, -1), b[..., 0].contiguous())
    same(w.dequantize().view(-1), nn_amd.dequantize_mxfp4_ocp(b.numpy(), n * k))


def test_weight_with_a_scale_over_252_is_refused():
    import nn_amd
    codes, scales = weight(20, 128, 1)
    for bad in (253, 255):
        s = scales.clone()
        s[7, 2] = bad
        for c, t in ((codes, s), (codes.cpu(), s.cpu())):
            with pytest.raises(nn_amd.NonFiniteData, match="30"):
                nn_amd.QuantizedWeight.from_mxfp4_rows(c, t)


def test_the_weight_in_the_calls_beside_the_linear():
    """argmax, sampling and log probabilities over the head's logits are those of the logits that quantized_linear gives"""
    import nn_amd
    n, k = 5003, 512
    codes, scales = weight(n, k, 12)
    w = nn_amd.QuantizedWeight.from_mxfp4_rows(codes, scales)
    x = torch.randn(1, k, generator=torch.Generator().manual_seed(3)).cuda() * 0.2
    bias = torch.randn(n, generator=torch.Generator().manual_seed(4)).cuda()
    logits, at = nn_amd.linear_argmax(x, w, bias)
    check_linear(logits[None], x, decode(codes, scales), bias, F32)
    assert int(at) == int(logits.argmax())
    lg, tok = nn_amd.linear_sample(x, w, bias, seed=77)
    assert torch.equal(lg, logits) and int(tok) == int(nn_amd.sample_token(lg, seed=77))
    xs = torch.randn(21, k, generator=torch.Generator().manual_seed(5)).cuda() * 0.2
    toks = torch.randint(0, n, (21,), generator=torch.Generator().manual_seed(6)).cuda()
    r = nn_amd.linear_logprobs(xs, w, toks, bias, top_n=4, ranks=True, return_logits=True)
    t = nn_amd.token_logprobs(r.logits, toks, top_n=4, ranks=True)
    check_linear(r.logits, xs, decode(codes, scales), bias, F32)
    for a, b in zip(r[:5], t[:5]):
        assert torch.equal(a, b)


def test_the_head_with_nan_and_without_allocation():
    import ctypes

    import nn_amd
    from nn_amd import _lib
    n, k = 3000, 12288 + 8192  # (x of a long row passes through LDS in chunks)
    codes, scales = weight(n, k, 13)
    w = nn_amd.QuantizedWeight.from_mxfp4_rows(codes, scales)
    x = torch.randn(k, generator=torch.Generator().manual_seed(9)).cuda() * 0.2
    logits, tok = nn_amd.linear_sample(x, w, seed=5, top_k=8)
    check_linear(logits[None], x[None], decode(codes, scales), None, F32)
    out, t = torch.empty(n, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
    cfg = _lib.Sampling(0.7, 8, 1, 0.9, 1.0, 0.0, 5)
    rc = _lib.load().nnq_linear_sample_noalloc(w.handle, x.data_ptr(), k, None, 0, out.data_ptr(), None, 0, ctypes.byref(cfg),
                                               t.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == _lib.OK
    assert torch.equal(out, logits) and int(t) == int(tok)
    x[77] = NAN
    with pytest.raises(nn_amd.NonFiniteData):
        nn_amd.linear_argmax(x, w)


def test_linears_captured_in_a_graph():
    import nn_amd
    n, k = 300, 1056
    codes, scales = weight(n, k, 21)
    w = nn_amd.QuantizedWeight.from_mxfp4_rows(codes, scales)
    for m in (1, 7, 50):
        for dt in (F32, BF16):
            x = torch.zeros(m, k, dtype=dt, device="cuda")

            def step():
                q = nn_amd.quantize_mxfp4_rows(x)
                return nn_amd.quantized_linear(x, w), nn_amd.mxfp4_linear(x, w), nn_amd.mxfp4_linear(q, w), q.dequantize()

            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                step()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                out = step()
            for i in range(3):
                x.copy_(torch.randn(m, k, generator=torch.Generator().manual_seed(i)).to(dt))
                eager = step()
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                for a, b in zip(out, eager):
                    assert torch.equal(a, b)


def test_two_streams_at_once():
    import nn_amd
    n, k, m = 700, 2048, 90
    codes, scales = weight(n, k, 31)
    w = nn_amd.QuantizedWeight.from_mxfp4_rows(codes, scales)
    xs = [torch.randn(m, k, generator=torch.Generator().manual_seed(i)).cuda() for i in range(2)]
    want = [(nn_amd.mxfp4_linear(x, w), nn_amd.quantized_linear(x, w)) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((nn_amd.mxfp4_linear(xs[i], w), nn_amd.quantized_linear(xs[i], w)))
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in got[i]:
            assert torch.equal(a, want[i][0]) and torch.equal(b, want[i][1])


def test_refusals():
    import nn_amd
    codes, scales = weight(32, 64, 2)
    w = nn_amd.QuantizedWeight.from_mxfp4_rows(codes, scales)
    x = torch.randn(2, 64, device="cuda")
    with pytest.raises(nn_amd.ShapeMismatch):
        nn_amd.mxfp4_linear(torch.randn(2, 96, device="cuda"), w)
    with pytest.raises(nn_amd.RankMismatch):
        nn_amd.mxfp4_linear(x[0], w)
    with pytest.raises(nn_amd.Unsupported):
        nn_amd.mxfp4_linear(x.cpu(), w)
    with pytest.raises(nn_amd.Unsupported):
        nn_amd.mxfp4_linear(x, w, out_dtype=torch.float16)
    with pytest.raises(nn_amd.BiasMismatch):
        nn_amd.mxfp4_linear(x, w, torch.zeros(31, device="cuda"))
    with pytest.raises(nn_amd.TensorError):
        nn_amd.mxfp4_linear(x, w, scale_rule="round")
    with pytest.raises(nn_amd.NotQuantized):
        nn_amd.mxfp4_linear(x, x)
    with pytest.raises(nn_amd.WrongQuantType):
        int4 = nn_amd.QuantizedWeight.from_int4_groups(codes, torch.ones(32, 2, dtype=torch.float16, device="cuda"), group_size=32)
        nn_amd.mxfp4_linear(x, int4)
    q = nn_amd.quantize_mxfp4_rows(x)
    with pytest.raises(nn_amd.ShapeMismatch):
        nn_amd.mxfp4_linear(nn_amd.Mxfp4Rows(q.codes, q.scales[:, :1]), w)
    with pytest.raises(nn_amd.Unsupported):
        nn_amd.mxfp4_linear(nn_amd.Mxfp4Rows(q.codes.cpu(), q.scales.cpu()), w)
    with pytest.raises(nn_amd.InvalidShape):
        nn_amd.quantize_mxfp4_rows(torch.randn(2, 40, device="cuda"))


def test_large_offsets():
    """outputs past 2^32 bytes, and a long row"""
    import nn_amd
    codes, scales = weight(40000, 32, 41)
    w = nn_amd.QuantizedWeight.from_mxfp4_rows(codes, scales)
    m = 30000
    x = torch.randn(m, 32, generator=torch.Generator().manual_seed(1)).cuda()
    ref, at = decode(codes, scales), [0, 1, 13000, 26900, m - 1]
    for y, v in ((nn_amd.quantized_linear(x, w), x[at]), (nn_amd.mxfp4_linear(x, w), quantize(x[at], "ceil")[0])):
        check_linear(y[at], v, ref, None, F32)
        del y
    k = 1 << 20
    codes, scales = weight(17, k, 42)
    w = nn_amd.QuantizedWeight.from_mxfp4_rows(codes, scales)
    for m in (3, 130):
        x = torch.randn(m, k, generator=torch.Generator().manual_seed(2)).cuda()
        check_linear(nn_amd.quantized_linear(x, w)[-3:], x[-3:], decode(codes, scales), None, F32)
        check_linear(nn_amd.mxfp4_linear(x, w)[-3:], quantize(x[-3:], "ceil")[0], decode(codes, scales), None, F32)

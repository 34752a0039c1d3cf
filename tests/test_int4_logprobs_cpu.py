"""Refusals of the 4-bit group-scaled weights and of the log probabilities that need no GPU, the host
repack of the 4-bit image against its description, and the plan of a log-probability call."""
import ctypes
import resource
import subprocess
import sys

import numpy as np
import pytest
import torch

import nn_amd
from nn_amd import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def create(lib, codes, scales, zeros, n, k, group, dtype=1):
    h = ctypes.c_void_p()
    ptr = lambda a: None if a is None else a.ctypes.data  # noqa: E731
    rc = lib.nnq_weight_create_int4(ptr(codes), ptr(scales), dtype, ptr(zeros), n, k, group, ctypes.byref(h))
    assert not h.value or rc == 0
    return rc


def test_int4_create_refusals(lib):
    c, s = np.zeros((4, 64), np.uint8), np.ones((4, 1), np.float16)
    z = np.full((4, 1), 8, np.uint8)
    assert lib.nnq_weight_create_int4(c.ctypes.data, s.ctypes.data, 1, None, 4, 128, 128, None) == _lib.ERR_INVALID_ARGUMENT
    assert create(lib, c, s, z, 0, 128, 128) == _lib.ERR_INVALID_ARGUMENT
    assert create(lib, c, s, z, 4, -128, 128) == _lib.ERR_INVALID_ARGUMENT
    for group in (0, 16, 48, 256, -32):
        assert create(lib, c, s, z, 4, 128, group) == _lib.ERR_INVALID_SHAPE, group
    assert create(lib, c, s, z, 4, 96, 64) == _lib.ERR_INVALID_SHAPE
    assert "96" in _lib.last_error()
    assert create(lib, c, s, z, 4, 128, 128, dtype=0) == _lib.ERR_UNSUPPORTED  # f32 scales
    assert create(lib, None, s, z, 4, 128, 128) == _lib.ERR_INVALID_ARGUMENT
    assert create(lib, c, None, z, 4, 128, 128) == _lib.ERR_INVALID_ARGUMENT
    z[2] = 17
    assert create(lib, c, s, z, 4, 128, 128) == _lib.ERR_INVALID_ARGUMENT
    assert "zero point 2" in _lib.last_error()
    for bad in (np.inf, -np.inf, np.nan):
        s2 = s.copy()
        s2[3] = bad
        assert create(lib, c, s2, None, 4, 128, 128) == _lib.ERR_NON_FINITE
    b = np.array([0x3F80, 0x7F80, 0x3F80, 0x3F80], np.uint16)  # bf16 infinity
    assert create(lib, c, b, None, 4, 128, 128, dtype=2) == _lib.ERR_NON_FINITE
    assert create(lib, c, s, None, 4, 1 << 21, 128) == _lib.ERR_UNSUPPORTED  # (nothing is read)
    # sizes whose product passes 64 bits are refused before anything is read
    assert create(lib, c, s, None, 1 << 40, 1 << 30, 128) == _lib.ERR_OUT_OF_MEMORY


def test_int4_scales_out_of_range(lib):
    """bf16 scales of 2^88 and more in magnitude; the largest below it passes (and the call goes on to the device)."""
    c = np.zeros((4, 64), np.uint8)
    for bits, refused in ((0x6B80, True), (0xEB80, True), (0x7F7F, True), (0xFF7F, True), (0x6B7F, False), (0xEB7F, False),
                          (0x0001, False)):
        s = np.array([0x3F80, 0x3F80, bits, 0x3F80], np.uint16)
        assert (create(lib, c, s, None, 4, 128, 128, dtype=2) == _lib.ERR_UNSUPPORTED) == refused, hex(bits)
        assert not refused or "scale 2 " in _lib.last_error()
    s = np.array([0x7BFF, 0x7BFF, 0xFBFF, 0x7BFF], np.uint16)  # f16 65504: the same bits would be too large in bf16
    assert create(lib, c, s, None, 4, 128, 128, dtype=1) != _lib.ERR_UNSUPPORTED


def test_int4_create_where_threads_cannot_start():
    """The host repack starts a thread per CPU.  Where only the first few start (stacks of 4 GiB in an address
    space that has room for two more), the call does the rest itself; a running thread must not be dropped,
    which would end the process."""
    child = '''
import ctypes, resource, sys
lib = ctypes.CDLL(sys.argv[1])
n, k = 32768, 32
codes, scales = (ctypes.c_uint8 * (n * k // 2))(), (ctypes.c_uint16 * n)(*[0x3C00] * n)
i64, h = ctypes.c_int64, ctypes.c_void_p()
used = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (used + (10 << 30),) * 2)
rc = lib.nnq_weight_create_int4(codes, scales, 1, None, i64(n), i64(k), i64(32), ctypes.byref(h))
print("returned", rc)
'''

    def limits():
        resource.setrlimit(resource.RLIMIT_STACK, (4 << 30, resource.getrlimit(resource.RLIMIT_STACK)[1]))

    r = subprocess.run([sys.executable, "-c", child, _lib.LIB_PATH], preexec_fn=limits, capture_output=True, text=True,
                       timeout=60)
    assert r.returncode == 0 and "returned" in r.stdout, (r.returncode, r.stderr[-500:])
    # (the device's refusal where there is none, but not the repack's)
    assert int(r.stdout.split()[-1]) != _lib.ERR_OUT_OF_MEMORY


def test_int4_device_create_refusals(lib):
    """What the device form refuses before it touches memory."""
    f, h = lib.nnq_weight_create_int4_device, ctypes.c_void_p()
    ok = [4096, 8192, 1, 12288, 4, 128, 128]
    for i, v, code in ((0, None, _lib.ERR_INVALID_ARGUMENT), (1, None, _lib.ERR_INVALID_ARGUMENT), (0, 4098, _lib.ERR_INVALID_ARGUMENT),
                       (1, 8193, _lib.ERR_INVALID_ARGUMENT), (2, 0, _lib.ERR_UNSUPPORTED), (4, 0, _lib.ERR_INVALID_ARGUMENT),
                       (5, 96, _lib.ERR_INVALID_SHAPE), (5, 1 << 21, _lib.ERR_UNSUPPORTED), (6, 16, _lib.ERR_INVALID_SHAPE),
                       (4, 1 << 60, _lib.ERR_OUT_OF_MEMORY)):
        args = list(ok)
        args[i] = v
        assert f(*args, ctypes.byref(h), None) == code, (i, v)
    assert f(*ok, None, None) == _lib.ERR_INVALID_ARGUMENT and not h.value


def test_from_int4_groups_refusals():
    with pytest.raises(nn_amd.Unsupported):
        nn_amd.QuantizedWeight.from_int4_groups(torch.zeros(4, 64, dtype=torch.uint8), torch.ones(4, 1).half(), [[8]] * 4)
    make = nn_amd.QuantizedWeight.from_int4_groups
    c, s = torch.zeros(4, 64, dtype=torch.uint8), torch.ones(4, 1, dtype=torch.float16)
    with pytest.raises(nn_amd.Unsupported):
        make(c.to(torch.int32), s)
    with pytest.raises(nn_amd.Unsupported):
        make(c, s.float())
    with pytest.raises(nn_amd.Unsupported):
        make(c.numpy(), s)
    with pytest.raises(nn_amd.WeightRank):
        make(c[0], s)
    for group in (16, 256, 0):
        with pytest.raises(nn_amd.InvalidShape):
            make(c, s, group_size=group)
    with pytest.raises(nn_amd.InvalidShape):
        make(c[:, :48], s, group_size=64)  # 96 columns
    with pytest.raises(nn_amd.InvalidShape):
        make(c[:0], s[:0])
    with pytest.raises(nn_amd.ShapeMismatch):
        make(c, s, group_size=64)
    with pytest.raises(nn_amd.ShapeMismatch):
        make(c, s, torch.zeros(4, 2, dtype=torch.uint8))
    with pytest.raises(nn_amd.Unsupported):
        make(c, s, torch.full((4, 1), 8.0))
    for z in (-1, 17, 300):
        with pytest.raises(nn_amd.TensorError):
            make(c, s, torch.full((4, 1), z, dtype=torch.int64))
    with pytest.raises(nn_amd.WrongQuantType):
        nn_amd.QuantizedWeight.from_quantized(np.zeros(64, np.uint8), nn_amd.QuantType.INT4G, (1, 128))


def test_int4g_has_no_blocks():
    q = nn_amd.QuantType.INT4G
    for call in (q.block_size, q.block_bytes, lambda: q.expected_bytes(256), lambda: q.expected_bytes(0),
                 lambda: q.expected_bytes(100)):
        with pytest.raises(nn_amd.WrongQuantType):
            call()
    assert [t.block_size() for t in nn_amd.QuantType if t != q] == [32, 256, 256, 32]
    assert [t.expected_bytes(512) for t in nn_amd.QuantType if t != q] == [544, 288, 420, 272]


class GemmPlan(ctypes.Structure):
    _fields_ = [(f, ctypes.c_int) for f in ("mt", "nt", "ks", "row_blocks", "col_blocks")] + \
               [(f, ctypes.c_size_t) for f in ("plane", "rowback", "slabs", "bytes")]


@pytest.mark.parametrize("xb", [0, 1])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_int4_plans(lib, xb, group):
    """Every shape has a tile that is built, workgroups that cover it, parts of K that none is empty of and
    scratch regions that hold what the launches write."""
    plan, split = lib._ZN3nnq14int4_gemm_planElllii, lib._ZN3nnq15int4_rows_splitEllli
    rows_scratch, chunk = lib._ZN3nnq17int4_rows_scratchEllli, lib._ZN3nnq15int4_chunk_rowsEll
    takes = lib._ZN3nnq15int4_takes_rowsEllli
    i64 = ctypes.c_int64
    takes.argtypes, takes.restype = [i64, i64, i64, ctypes.c_int], ctypes.c_bool
    plan.argtypes, plan.restype = [i64, i64, i64, ctypes.c_int, ctypes.c_int], GemmPlan
    split.argtypes, split.restype = [i64, i64, i64, ctypes.c_int], ctypes.c_int
    rows_scratch.argtypes, rows_scratch.restype = [i64, i64, i64, ctypes.c_int], ctypes.c_size_t
    chunk.argtypes, chunk.restype = [i64, i64], i64
    for n in (1, 16, 100, 4096, 12288, 151936):
        for k in (group, 128, 320 * group // 32, 4096, 12288, 1 << 20):
            units = (k + 127) // 128
            assert all(takes(m, n, k, xb) for m in (1, 4)) and not takes(17, n, k, xb)
            for m in (1, 4, 5, 8, 9, 16):
                ks = split(m, n, k, xb)
                assert 1 <= ks <= min(8, units) and (m > 4 or ks == 1)  # (one row: no scratch)
                assert rows_scratch(m, n, k, xb) == (ks * m * n * 4 if ks > 1 else 0)
            for m in (1, 17, 32, 33, 203, 640, 5000, 65536):
                r = chunk(m, k)
                assert 1 <= r <= m and (r == m or r % 128 == 0)
                p = plan(r, n, k, group, xb)
                assert p.mt in (1, 2) and p.nt in (1, 2) and not (p.mt == p.nt == 2 and (not xb or group == 32))
                assert 1 <= p.ks <= max(1, units // 2) and p.row_blocks * p.mt * 32 >= r and p.col_blocks * p.nt * 128 >= n
                planes, tiles = 1 if xb else 2, (r + 31) // 32
                assert p.plane == tiles * units * 8192 and planes * p.plane < 2 ** 31  # 32-bit offsets
                assert p.rowback == planes * p.plane and p.slabs >= p.rowback + tiles * 128 and p.slabs % 256 == 0
                assert p.bytes >= p.slabs + (p.ks * r * n * 4 if p.ks > 1 else 0)


def test_int4_few_rows_or_gemm(lib):
    """The rule's two sides, as measured (8 bf16 rows: 72 us against 77, 40 against 25; 16 f32 rows: 12
    against 13.6, 33 against 25)."""
    takes = lib._ZN3nnq15int4_takes_rowsEllli
    takes.argtypes, takes.restype = [ctypes.c_int64] * 3 + [ctypes.c_int], ctypes.c_bool
    for m, n, k, xb, rows in ((8, 151936, 4096, 1, 1), (8, 151936, 1024, 1, 0), (16, 4096, 4096, 0, 1),
                              (12, 4096, 12288, 1, 1), (16, 65536, 512, 1, 0), (5, 5751, 2880, 0, 1), (16, 24576, 4096, 0, 0)):
        assert takes(m, n, k, xb) == bool(rows), (m, n, k, xb)


def test_int4_gguf_formats_refuse_the_layout(lib):
    """The block-format entry points do not take the new format's id."""
    h = ctypes.c_void_p()
    buf = np.zeros(1024, np.uint8)
    vp = buf.ctypes.data
    assert lib.nnq_weight_create(1000, 4, vp, buf.size, 4, 128, ctypes.byref(h)) == _lib.ERR_WRONG_FORMAT
    assert lib.nnq_mlp_create(1000, 4, vp, vp, buf.size, 1000, 4, vp, buf.size, 128, 128,
                              ctypes.byref(h)) == _lib.ERR_WRONG_FORMAT


class Layout(ctypes.Structure):
    _fields_ = [("fmt", ctypes.c_int), ("layout", ctypes.c_int), ("n", ctypes.c_int64), ("k", ctypes.c_int64),
                ("ntile", ctypes.c_int64), ("nblk", ctypes.c_int64), ("qs", ctypes.c_size_t), ("hdr", ctypes.c_size_t),
                ("aux", ctypes.c_size_t), ("group", ctypes.c_int), ("zeros", ctypes.c_int), ("sbf", ctypes.c_int)]


@pytest.mark.parametrize("n,k,group,zeros", [(1, 32, 32, True), (16, 128, 128, False), (17, 160, 32, True),
                                             (33, 192, 64, False), (5, 2880, 64, True), (40, 384, 128, True)])
def test_int4_image(lib, n, k, group, zeros):
    """Every code, scale and zero point at the place the kernels read it, zeros elsewhere."""
    rng = np.random.default_rng(n * 1000 + k)
    q = rng.integers(0, 16, (n, k), dtype=np.uint8)
    codes = np.ascontiguousarray(q[:, 0::2] | (q[:, 1::2] << 4))
    scales = rng.integers(1, 0x7C00, (n, k // group)).astype(np.uint16)
    zp = rng.integers(0, 17, (n, k // group), dtype=np.uint8) if zeros else None
    L, err = Layout(), ctypes.c_char_p()
    make = lib._ZN3nnq16make_layout_int4EllliiPNS_6LayoutEPPKc
    make.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_int] * 2 + [ctypes.c_void_p] * 2
    make.restype = ctypes.c_bool
    assert make(n, k, group, int(zeros), 0, ctypes.byref(L), ctypes.byref(err))
    gpu, ub = 128 // group, 1024 + 16 * (128 // group) * (3 if zeros else 2)
    tiles, units = (n + 15) // 16, (k + 127) // 128
    assert (L.ntile, L.nblk, L.qs, L.hdr, L.aux) == (tiles, units, tiles * units * ub, 0, 0)
    img = np.full(L.qs + 64, 0xAB, np.uint8)
    rep = lib._ZN3nnq11repack_int4EPKhPKtS1_RKNS_6LayoutEllPh
    rep.argtypes = [ctypes.c_void_p] * 4 + [ctypes.c_int64] * 2 + [ctypes.c_void_p]
    for t in range(tiles):  # (tile by tile, as the threads of an upload do)
        rep(codes.ctypes.data, scales.ctypes.data, zp.ctypes.data if zeros else None, ctypes.byref(L), t, t + 1,
            img.ctypes.data)
    assert (img[L.qs:] == 0xAB).all()
    rec = img[:L.qs].reshape(tiles, units, ub)
    words = rec[:, :, :1024].copy().view(np.uint32).reshape(tiles, units, 4, 16, 4)  # [tile][unit][p][row][j]
    got = np.zeros((tiles * 16, units * 128), np.uint8)
    for p in range(4):
        for j in range(4):
            for e in range(8):
                col = 32 * j + 8 * p + e
                w = (words[:, :, p, :, j] >> (4 * (e // 2) + 16 * (e % 2))) & 15
                got[:, col::128] = w.transpose(0, 2, 1).reshape(tiles * 16, units)
    want = np.zeros_like(got)
    want[:n, :k] = q
    assert np.array_equal(got, want)

    def per_group(a):
        g = np.zeros((tiles * 16, units * gpu), a.dtype)
        g[:n, :k // group] = a
        return g.reshape(tiles, 16, units, gpu).transpose(0, 2, 1, 3)

    sc = rec[:, :, 1024:1024 + 32 * gpu].copy().view(np.uint16).reshape(tiles, units, 16, gpu)
    assert np.array_equal(sc, per_group(scales))
    if zeros:
        assert np.array_equal(rec[:, :, 1024 + 32 * gpu:].reshape(tiles, units, 16, gpu), per_group(zp))


def test_logprob_refusals(lib):
    f32, i64 = np.zeros(64, np.float32), np.zeros(64, np.int64)
    p, t = f32.ctypes.data, i64.ctypes.data

    def call(logits=p, dtype=0, m=2, n=8, stride=8, tokens=t, top=0, lp=p, ent=None, ranks=None, tlp=None, tid=None):
        return lib.nnq_token_logprobs(logits, dtype, m, n, stride, tokens, top, lp, ent, ranks, tlp, tid, None)

    assert call(dtype=3) == _lib.ERR_UNSUPPORTED
    assert call(m=-1) == _lib.ERR_INVALID_ARGUMENT
    assert call(n=0) == _lib.ERR_INVALID_SHAPE
    assert call(n=1 << 31) == _lib.ERR_UNSUPPORTED
    for top in (-1, 9, 33):
        assert call(top=top, tlp=p, tid=t) == _lib.ERR_INVALID_SHAPE, top
    assert call(n=64, stride=64, top=33, tlp=p, tid=t) == _lib.ERR_INVALID_SHAPE
    assert call(logits=None) == _lib.ERR_INVALID_ARGUMENT
    assert call(tokens=None) == _lib.ERR_INVALID_ARGUMENT
    assert call(lp=None) == _lib.ERR_INVALID_ARGUMENT
    assert call(top=2, tlp=p) == _lib.ERR_INVALID_ARGUMENT
    assert call(top=2, tid=t) == _lib.ERR_INVALID_ARGUMENT
    assert call(stride=-8) == _lib.ERR_INVALID_ARGUMENT
    assert call(logits=p + 2) == _lib.ERR_INVALID_ARGUMENT  # f32 logits at an odd half
    assert call(tokens=t + 4) == _lib.ERR_INVALID_ARGUMENT
    assert call(lp=p + 1) == _lib.ERR_INVALID_ARGUMENT
    assert call(m=0, logits=None, tokens=None, lp=None) == 0  # nothing to do
    assert lib.nnq_linear_logprobs(None, p, 0, 1, 8, None, 0, t, 0, None, p, None, None, None, None,
                                   None) == _lib.ERR_NOT_QUANTIZED


def test_python_logprob_refusals():
    with pytest.raises(nn_amd.Unsupported):
        nn_amd.token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64))  # host tensor
    w = nn_amd.QuantizedWeight(ctypes.c_void_p(), nn_amd.QuantType.INT4G, nn_amd.Layout.GROUPS, (16, 256), 0)
    with pytest.raises(nn_amd.Unsupported):
        nn_amd.linear_logprobs(torch.zeros(1, 256), w, [0])
    with pytest.raises(nn_amd.ShapeMismatch):
        nn_amd.linear_logprobs(torch.zeros(1, 128), w, [0])
    with pytest.raises(nn_amd.NotQuantized):
        nn_amd.linear_logprobs(torch.zeros(1, 256), torch.zeros(16, 256), [0])
    from nn_amd.quantized import _logprob_outputs, _token_ids
    for top in (-1, 33, 9):
        with pytest.raises(nn_amd.InvalidShape):
            _logprob_outputs((2,), 8 if top == 9 else 100, top, False, "cpu")
    with pytest.raises(nn_amd.ShapeMismatch):
        _token_ids(torch.zeros(3, dtype=torch.int64), (2,), "cpu")
    with pytest.raises(nn_amd.Unsupported):
        _token_ids(torch.zeros(2), (2,), "cpu")
    for batch in ((), (0,), (2, 3)):
        _, out = _logprob_outputs(batch, 8, 4, True, "cpu")
        assert out.logprobs.shape == out.entropy.shape == out.ranks.shape == batch
        assert out.top_ids.shape == out.top_logprobs.shape == (*batch, 4)


def test_no_tokens_from_a_list():
    """An empty batch is nothing to do, also where its tokens come as a list; an empty float tensor is a mistake."""
    from nn_amd.quantized import _token_ids
    for tokens, batch in (([], (0,)), ((), (0,)), ([[], []], (2, 0)), (np.zeros((0,), np.int32), (0,))):
        t = _token_ids(tokens, batch, torch.device("cpu"))
        assert t.dtype is torch.int64 and tuple(t.shape) == batch
    with pytest.raises(nn_amd.ShapeMismatch):
        _token_ids([], (1,), torch.device("cpu"))
    with pytest.raises(nn_amd.Unsupported):
        _token_ids(torch.zeros(0), (0,), torch.device("cpu"))
    with pytest.raises(nn_amd.Unsupported):
        _token_ids([0.5], (1,), torch.device("cpu"))


class OnOther(torch.Tensor):
    """A host tensor that says it is on the second device."""
    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda", 1))


def test_launches_are_made_on_the_device_of_their_tensors(monkeypatch):
    """The raw handle of a default stream is 0 and means the current device's: every call that takes a 4-bit weight
    or its logits makes its tensors' device current for the launch, and puts the caller's back."""
    from nn_amd import quantized
    now, calls = [0], []

    class Switch:
        def __init__(self, device):
            self.to = torch.device(device).index

        def __enter__(self):
            self.back, now[0] = now[0], self.to

        def __exit__(self, *exc):
            now[0] = self.back

    class Lib:
        def __getattr__(self, name):
            return lambda *args: calls.append((name, now[0])) or 0

    empty = torch.empty
    monkeypatch.setattr(quantized._lib, "load", lambda: Lib())
    monkeypatch.setattr(quantized, "_current_device", lambda: now[0], raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(quantized, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "device", Switch)
    monkeypatch.setattr(torch, "empty", lambda *a, device=None, **kw: empty(*a, **kw).as_subclass(OnOther))
    w = nn_amd.QuantizedWeight(ctypes.c_void_p(), nn_amd.QuantType.INT4G, nn_amd.Layout.GROUPS, (16, 256), 1)
    x = torch.zeros(2, 256).as_subclass(OnOther)
    logits, t = torch.zeros(16).as_subclass(OnOther), torch.zeros(2, dtype=torch.int64).as_subclass(OnOther)
    for call, name in ((lambda: nn_amd.quantized_linear(x, w), "nnq_linear"),
                       (lambda: nn_amd.linear_argmax(x[0], w, check=False), "nnq_linear_argmax_i64"),
                       (lambda: nn_amd.linear_sample(x[0], w), "nnq_linear_sample"),
                       (lambda: nn_amd.sample_token(logits), "nnq_sample_token"),
                       (lambda: nn_amd.token_logprobs(x, t, top_n=2), "nnq_token_logprobs"),
                       (lambda: nn_amd.linear_logprobs(x, w, t), "nnq_linear_logprobs"),
                       (w.dequantize, "nnq_dequant")):
        for current in (0, 1):
            calls.clear()
            now[0] = current
            call()
            assert calls == [(name, 1)] and now[0] == current


class Plan(ctypes.Structure):
    _fields_ = [("nseg", ctypes.c_int64), ("rows", ctypes.c_int64), ("slots", ctypes.c_int), ("bytes", ctypes.c_size_t)]


@pytest.mark.parametrize("elem", [2, 4])
@pytest.mark.parametrize("top", [0, 1, 5, 20, 32])
def test_logprob_plan(lib, top, elem):
    """The segments cover a row wherever it starts in a 16-byte word; slots hold the alternatives and fit a
    wave's lanes; rows fit the grid; the scratch stays bounded."""
    plan = lib._ZN3nnq12logprob_planEllii
    plan.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.c_int]
    plan.restype = Plan
    for n in (1, 2045, 2046, 2048, 2049, 8185, 8192, 50257, 151936, 2 ** 31 - 1):
        for m in (1, 7, 65536, 1 << 33):
            p = plan(m, n, top, elem)
            assert p.nseg % 4 == 0 and p.nseg * 2048 >= n + 16 // elem - 1
            assert top <= p.slots <= 64 and (top == 0) == (p.slots == 0)
            assert 1 <= p.rows <= min(m, 65535)
            assert p.bytes == p.rows * p.nseg * (20 + 8 * p.slots)
            assert p.rows == 1 or p.bytes <= 64 << 20
    chunk = lib._ZN3nnq15head_chunk_rowsEll
    chunk.argtypes, chunk.restype = [ctypes.c_int64] * 2, ctypes.c_int64
    for n in (1, 1000, 151936, 1 << 24):
        for m in (1, 15, 16, 300, 100000):
            r = chunk(m, n)
            assert 1 <= r <= m and (r == m or r % 16 == 0) and (r <= 16 or 4 * n * r <= 320 << 20)
            assert r == m or m // r >= 1 and (m + r - 1) // r * r - m < 64 * ((m + r - 1) // r)  # even chunks

"""MXFP4 rows and beam search without a device: what the C ABI and the Python calls refuse, before any device work."""
import ctypes

import numpy as np
import pytest
import torch

from nn_amd import _lib

P = ctypes.c_void_p(4096)  # an address that no refused call reads


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_weight_refusals(lib):
    h = ctypes.c_void_p(1)
    codes, scales = np.zeros((4, 32), np.uint8), np.full((4, 2), 127, np.uint8)

    def create(n, k, c=codes, s=scales, out=h):
        return lib.nnq_weight_create_mxfp4(None if c is None else c.ctypes.data, None if s is None else s.ctypes.data, n, k,
                                           ctypes.byref(out) if out is not None else None)

    assert create(4, 64, out=None) == _lib.ERR_INVALID_ARGUMENT
    assert create(0, 64) == _lib.ERR_INVALID_ARGUMENT and create(4, -32) == _lib.ERR_INVALID_ARGUMENT
    assert not h.value  # (cleared where the call is refused)
    assert create(4, 48) == _lib.ERR_INVALID_SHAPE and "multiple of 32" in _lib.last_error()
    assert create(4, (1 << 20) + 32) == _lib.ERR_UNSUPPORTED
    assert create(1 << 62, 64) == _lib.ERR_OUT_OF_MEMORY
    assert create(4, 64, c=None) == _lib.ERR_INVALID_ARGUMENT and create(4, 64, s=None) == _lib.ERR_INVALID_ARGUMENT
    for byte in (253, 254, 255):
        bad = scales.copy()
        bad[2, 1] = byte
        assert create(4, 64, s=bad) == _lib.ERR_NON_FINITE and "5" in _lib.last_error()
    for args in ((None, P, 4, 64), (P, None, 4, 64), (P, P, 4, 40), (P, P, 0, 64)):
        assert lib.nnq_weight_create_mxfp4_device(*args, ctypes.byref(h), None) in (_lib.ERR_INVALID_ARGUMENT, _lib.ERR_INVALID_SHAPE)


def test_quantize_refusals(lib):
    q = lambda x=P, dt=0, rows=2, k=64, stride=64, rule=0, c=P, s=P: lib.nnq_mxfp4_quantize(x, dt, rows, k, stride, rule, c, s, None)
    assert q(rows=-1) == _lib.ERR_INVALID_ARGUMENT
    for k in (0, -32, 16, 40):
        assert q(k=k) == _lib.ERR_INVALID_SHAPE
    assert q(dt=1) == _lib.ERR_UNSUPPORTED  # f16
    assert q(rule=2) == _lib.ERR_INVALID_ARGUMENT and q(stride=-1) == _lib.ERR_INVALID_ARGUMENT
    for null in ({"x": None}, {"c": None}, {"s": None}, {"x": ctypes.c_void_p(4098)}, {"c": ctypes.c_void_p(4098)}):
        assert q(**null) == _lib.ERR_INVALID_ARGUMENT
    assert q(rows=1 << 60) == _lib.ERR_OUT_OF_MEMORY
    assert q(x=None, rows=0) == _lib.OK
    d = lambda c=P, s=P, rows=2, k=64, out=P, dt=0: lib.nnq_mxfp4_dequantize(c, s, rows, k, out, dt, None)
    assert d(k=33) == _lib.ERR_INVALID_SHAPE and d(dt=1) == _lib.ERR_UNSUPPORTED and d(rows=-1) == _lib.ERR_INVALID_ARGUMENT
    for null in ({"c": None}, {"s": None}, {"out": None}, {"out": ctypes.c_void_p(4100)}):
        assert d(**null) == _lib.ERR_INVALID_ARGUMENT
    assert d(rows=0) == _lib.OK


def test_product_refusals(lib):
    assert lib.nnq_mxfp4_linear(None, P, 0, 1, 64, 0, None, 0, P, 0, None) == _lib.ERR_NOT_QUANTIZED
    assert lib.nnq_mxfp4_linear_codes(None, P, P, 1, 64, None, 0, P, 0, None) == _lib.ERR_NOT_QUANTIZED


def test_beam_select_refusals(lib):
    def s(logits=P, dt=0, batch=2, beams=3, n=50, bs=150, js=50, scores=P, fin=None, end=0, keep=4, out=P, parents=P, tokens=P):
        return lib.nnq_beam_select(logits, dt, batch, beams, n, bs, js, scores, fin, end, keep, out, parents, tokens, None)

    assert s(dt=3) == _lib.ERR_UNSUPPORTED and s(batch=-1) == _lib.ERR_INVALID_ARGUMENT
    for bad in (0, -1, 33):
        assert s(beams=bad) == _lib.ERR_INVALID_SHAPE and s(keep=bad) == _lib.ERR_INVALID_SHAPE
    assert s(n=0) == _lib.ERR_INVALID_SHAPE and s(n=1 << 31) == _lib.ERR_UNSUPPORTED
    assert s(bs=-1) == _lib.ERR_INVALID_ARGUMENT and s(js=-1) == _lib.ERR_INVALID_ARGUMENT
    assert s(fin=P, end=-1) == _lib.ERR_INVALID_ARGUMENT
    for null in ("logits", "scores", "out", "parents", "tokens"):
        assert s(**{null: None}) == _lib.ERR_INVALID_ARGUMENT
    for odd, at in (("logits", 4098), ("scores", 4098), ("out", 4097), ("parents", 4100), ("tokens", 4100)):
        assert s(**{odd: ctypes.c_void_p(at)}) == _lib.ERR_INVALID_ARGUMENT
    assert s(batch=0, logits=None) == _lib.OK


def reorder(lib, sizes=(4, 8), strides=(8, 1), slot=32, batch=2, beams=3, elem=2, states=(4096,), parents=P, ndim=None):
    arr = (ctypes.c_void_p * max(1, len(states)))(*states)
    n = len(sizes)
    return lib.nnq_beam_reorder(arr, len(states), batch, beams, slot, n if ndim is None else ndim, (ctypes.c_int64 * max(1, n))(*sizes),
                                (ctypes.c_int64 * max(1, n))(*strides), elem, parents, None)


def test_beam_reorder_refusals(lib):
    for bad in (0, 33):
        assert reorder(lib, beams=bad) == _lib.ERR_INVALID_SHAPE
    assert reorder(lib, batch=-1) == _lib.ERR_INVALID_ARGUMENT and reorder(lib, ndim=9) == _lib.ERR_INVALID_ARGUMENT
    assert reorder(lib, elem=0) == _lib.ERR_INVALID_ARGUMENT and reorder(lib, elem=17) == _lib.ERR_INVALID_ARGUMENT
    assert reorder(lib, slot=-1) == _lib.ERR_INVALID_ARGUMENT
    assert reorder(lib, states=(4096, 0)) == _lib.ERR_INVALID_ARGUMENT and reorder(lib, parents=None) == _lib.ERR_INVALID_ARGUMENT
    assert reorder(lib, parents=ctypes.c_void_p(4100)) == _lib.ERR_INVALID_ARGUMENT
    for sizes, strides, slot in (((4, 8), (8, 1), 31), ((4, 8), (7, 1), 32), ((4, 8), (0, 1), 32), ((4, 8), (8, 1), 0),
                                 ((4, 8), (48, 1), 5), ((-1, 8), (8, 1), 32), ((4, 8), (-8, 1), 32)):
        assert reorder(lib, sizes, strides, slot) == _lib.ERR_INVALID_ARGUMENT, (sizes, strides, slot)
    apart = (2,) * 5, (1000, 300, 90, 20, 3)
    assert reorder(lib, *apart, slot=4000) == _lib.ERR_UNSUPPORTED and "4 dimensions" in _lib.last_error()
    assert reorder(lib, (4, 8), (1 << 58, 1)) == _lib.ERR_OUT_OF_MEMORY
    # nothing to do: no states, no items, one beam, no elements
    assert reorder(lib, states=()) == _lib.OK and reorder(lib, batch=0) == _lib.OK and reorder(lib, beams=1) == _lib.OK
    assert reorder(lib, (0, 8), (8, 1)) == _lib.OK


def test_beam_reorder_checks_the_geometry_first(lib):
    for states, batch, beams in (((), 2, 3), ((4096,), 2, 1), ((4096,), 1, 3)):
        assert reorder(lib, (4, 8), (7, 1), states=states, batch=batch, beams=beams) == _lib.ERR_INVALID_ARGUMENT
        assert reorder(lib, (2,) * 5, (1000, 300, 90, 20, 3), slot=4000, states=states, batch=batch, beams=beams) == _lib.ERR_UNSUPPORTED


def test_python_refusals_without_a_device():
    import nn_amd
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    make = nn_amd.QuantizedWeight.from_mxfp4_rows
    with pytest.raises(nn_amd.Unsupported):
        make(codes.numpy(), scales)
    with pytest.raises(nn_amd.Unsupported):
        make(codes.int(), scales)
    with pytest.raises(nn_amd.InvalidShape):
        make(codes[:, :24], scales)
    with pytest.raises(nn_amd.ShapeMismatch):
        make(codes, scales[:3])
    with pytest.raises(nn_amd.WeightRank):
        make(codes[None], scales[None])
    with pytest.raises(nn_amd.InvalidShape):
        make(codes[:0], scales[:0])
    x = torch.zeros(2, 64)
    with pytest.raises(nn_amd.Unsupported):
        nn_amd.quantize_mxfp4_rows(x)
    with pytest.raises(nn_amd.TensorError):
        nn_amd.quantize_mxfp4_rows(x, "nearest")
    with pytest.raises(nn_amd.Unsupported):
        nn_amd.Mxfp4Rows(codes, scales).dequantize()
    with pytest.raises(nn_amd.NotQuantized):
        nn_amd.mxfp4_linear(x, x)
    with pytest.raises(nn_amd.Unsupported):
        nn_amd.beam_select(torch.zeros(2, 5), torch.zeros(2))
    with pytest.raises(nn_amd.Unsupported):
        nn_amd.beam_reorder(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(nn_amd.ShapeMismatch):
        nn_amd.beam_reorder(torch.zeros(2, 5), 1)
    # blocks of 17 bytes are the experts' and the host encoder's form; a linear weight has arrays of its own
    with pytest.raises(nn_amd.TensorError):
        nn_amd.QuantizedWeight.from_quantized(np.zeros(17 * 8, np.uint8), nn_amd.QuantType.MXFP4, (4, 64), nn_amd.Layout.OCP)

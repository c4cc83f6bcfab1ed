"""Dropout from counters against a restatement of its generator in numpy: which elements stay is compared exactly, their values to the roundings of one product and one sum (2^-23 of their magnitudes in fp32, 2^-8
of the value for bfloat16's own rounding)."""
import ctypes as C

import numpy as np
import pytest

from helpers import capi
from typed_arrays import UNIT, rounded
from test_rocm_residual_norm import Rows

gpu = pytest.mark.gpu


def kept(count, rate, seed, stream):
    """Philox4x32-10 in unsigned 64-bit arithmetic; element i: 16 bits, half i % 8 of group i / 8"""
    u, mask = np.uint64, np.uint64(0xFFFFFFFF)
    i = np.arange(-(-count // 8), dtype=np.uint64)
    x = [i & mask, i >> u(32), np.full_like(i, stream & 0xFFFFFFFF), np.full_like(i, stream >> 32)]
    for r in range(10):
        a, b = x[0] * u(0xD2511F53), x[2] * u(0xCD9E8D57)
        k = u(((seed & 0xFFFFFFFF) + r * 0x9E3779B9) & 0xFFFFFFFF), u(((seed >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)
        x = [(b >> u(32)) ^ x[1] ^ k[0], b & mask, (a >> u(32)) ^ x[3] ^ k[1], a & mask]
    return np.stack(x, 1).astype("<u4").view("<u2").reshape(-1)[:count] >= int(np.float32(rate) * 65536 + 0.5)


def reference(x, residual, rate, seed, stream):
    threshold = int(np.float32(rate) * 65536 + 0.5)
    keep = kept(x.size, rate, seed, stream).reshape(x.shape)
    y = np.where(keep, x * (65536 / (65536 - threshold) if threshold < 65536 else 0.0), 0.0)
    return keep, y if residual is None else residual + y, np.where(keep, 2 * np.abs(x) / max(1 - rate, 2.0 ** -16), 0.0) + (0.0 if residual is None else np.abs(residual))


def run(rocm, x, residual, dtype, rate, seed, stream, pad=0, offset=0, alias=None):
    a = Rows(rocm, x, dtype, pad, offset)
    r = Rows(rocm, residual, dtype, pad, offset) if residual is not None else None
    y = a if alias == "x" else r if alias == "residual" else Rows(rocm, x, dtype, pad, offset, 7.0)
    rocm.call("dropout", capi.TYPE[dtype], a.ptr, a.ld, r.ptr if r else None, r.ld if r else 0, y.ptr, y.ld, x.shape[0], x.shape[1], rate, seed, stream)
    rocm.sync()
    return y.numpy()


def check(got, x, residual, dtype, rate, seed, stream):
    keep, want, size = reference(x, residual, rate, seed, stream)
    if residual is None:
        assert np.array_equal(got != 0, keep & (x != 0))
    assert np.all(np.abs(got - want) <= 2.0 ** -23 * size + (UNIT[dtype] * np.abs(want) if dtype == "bfloat16" else 0.0))


def inputs(shape, dtype, residual, seed=0):
    rng = np.random.default_rng(seed)
    return rounded(rng.standard_normal(shape), dtype), rounded(rng.standard_normal(shape), dtype) if residual else None


def test_the_restated_generator_gives_the_published_vector():
    """counter and key of zero: 6627e8d5 e169c58d bc57ac4c 9b00dbd8 (Salmon et al., known answers of Philox4x32-10), compared half by half around its own values"""
    halves = np.array([0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8], "<u4").view("<u2")
    for h in halves:
        rate = h / 65536
        assert np.array_equal(kept(8, rate, 0, 0), halves >= h)


def test_the_share_that_stays():
    assert abs(kept(1 << 18, 0.3, 5, 6).mean() - 0.7) < 5 * np.sqrt(0.21 / (1 << 18))      # five standard deviations
    assert kept(1000, 0.0, 5, 6).all() and not kept(1000, 1.0, 5, 6).any()


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (3, 8), (5, 9), (256, 256), (129, 1023), (2, 5000), (4001, 24), (64, 4096)])
def test_sizes(rocm, shape, dtype, residual):
    print("case", shape, dtype, residual, flush=True)
    x, r = inputs(shape, dtype, residual, sum(shape))
    for rate, seed, stream in ((0.1, 3, 4), (0.5, (1 << 63) + 12345, (1 << 40) + 7)):
        check(run(rocm, x, r, dtype, rate, seed, stream), x, r, dtype, rate, seed, stream)


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("pad,offset", [(8, 0), (3, 0), (0, 1), (16, 8), (0, 8)])
@pytest.mark.parametrize("alias", [None, "x", "residual"])
def test_strides_alignments_and_in_place(rocm, dtype, pad, offset, alias):
    for shape in ((33, 120), (17, 61)):
        x, r = inputs(shape, dtype, True, 2)
        check(run(rocm, x, r, dtype, 0.25, 9, 10, pad, offset, alias), x, r, dtype, 0.25, 9, 10)
        check(run(rocm, x, None, dtype, 0.25, 9, 10, pad, offset, "x" if alias else None), x, None, dtype, 0.25, 9, 10)


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_rates_of_none_and_all_and_values_that_are_not_finite(rocm, dtype):
    x, r = inputs((20, 40), dtype, True)
    assert np.array_equal(run(rocm, x, None, dtype, 0.0, 1, 2), x)
    assert np.array_equal(run(rocm, x, r, dtype, 1.0, 1, 2), r) and not run(rocm, x, None, dtype, 1.0, 1, 2).any()
    keep = kept(800, 0.5, 1, 2).reshape(20, 40)
    x[~keep] = np.nan
    got = run(rocm, x, r, dtype, 0.5, 1, 2)
    assert np.array_equal(got[~keep], r[~keep]) and np.isfinite(got).all()      # a dropped element's value is not looked at


@gpu
def test_the_backward_call_drops_what_the_forward_call_dropped(rocm):
    x, d = inputs((50, 333), "float32", True, 4)
    forward, backward = run(rocm, x, None, "float32", 0.4, 21, 22), run(rocm, d, None, "float32", 0.4, 21, 22)
    assert np.array_equal(forward != 0, backward != 0)
    h = 2.0 ** -4      # a power of two: the differences of this piecewise linear function are exact up to the roundings of its values
    up = run(rocm, rounded(x + h * np.sign(d), "float32"), None, "float32", 0.4, 21, 22)
    numeric = ((up - forward) * d).sum() / h
    assert abs(numeric - (backward * np.sign(d)).sum()) <= 1e-4 * np.abs(backward).sum()


@gpu
def test_another_stream_number_draws_another_mask_and_the_offset_counts(rocm):
    x = np.ones((64, 64))
    a, b = run(rocm, x, None, "float32", 0.5, 1, 100), run(rocm, x, None, "float32", 0.5, 1, 101)
    assert 0.3 < ((a != 0) == (b != 0)).mean() < 0.7
    rocm.call("set_stream_offset", 1)
    try:
        assert np.array_equal(run(rocm, x, None, "float32", 0.5, 1, 100), b)
    finally:
        rocm.call("set_stream_offset", 0)


@gpu
def test_a_graph_draws_anew_with_each_replay(rocm):
    """the offset advances inside the graph, so the replays' masks are those of streams 50, 51, 52"""
    lib, h = rocm.device.lib, rocm.device.handle
    x, y = rocm.array(np.ones((40, 50), np.float32)), rocm.zeros((40, 50))
    rocm.sync()
    assert lib.rlt_rocm_graph_begin_capture(h) == 0
    rocm.call("dropout", capi.TYPE["float32"], x.ptr, 50, None, 0, y.ptr, 50, 40, 50, 0.5, 8, 50)
    rocm.call("advance_streams", 1)
    graph = C.c_void_p()
    assert lib.rlt_rocm_graph_end_capture(h, C.byref(graph)) == 0
    try:
        for replay in range(3):
            y.upload(np.zeros((40, 50), np.float32))
            assert lib.rlt_rocm_graph_launch(h, graph) == 0
            rocm.sync()
            assert np.array_equal(y.numpy().reshape(-1) != 0, kept(2000, 0.5, 8, 50 + replay))
    finally:
        rocm.call("set_stream_offset", 0)
        lib.rlt_rocm_graph_destroy(h, graph)


@gpu
def test_refusals(rocm):
    lib, h, x = rocm.device.lib, rocm.device.handle, rocm.zeros((4, 8))
    code = lambda type=0, x=x.ptr, ldx=8, r=None, ldr=0, y=x.ptr, ldy=8, rows=4, cols=8, rate=0.5: lib.rlt_rocm_dropout(h, type, x, ldx, r, ldr, y, ldy, rows, cols, rate, 1, 2)
    assert code() == 0
    for bad in (code(type=2), code(x=None), code(y=None), code(ldx=7), code(ldy=7), code(r=x.ptr, ldr=7), code(rows=0), code(cols=-1), code(rate=-0.1), code(rate=1.1), code(rate=float("nan"))):
        assert bad == capi.RLT_E_INVALID_ARGUMENT
    assert lib.rlt_rocm_dropout(None, 0, x.ptr, 8, None, 0, x.ptr, 8, 4, 8, 0.5, 1, 2) == capi.RLT_E_NOT_INITIALISED
    rocm.sync()

"""Linear attention where tensors, values and calls are out of the ordinary. The reference in 64 bits, the cases and the bounds are those of test_rocm_linear_attention."""
import ctypes as C

import numpy as np
import pytest

import helpers
from helpers import capi
from test_rocm_linear_attention import Tensor, bounds, case, check, layer_of, magnitudes, reference, strides_of, view, workspace
from typed_arrays import download, filled, rounded, upload

gpu = pytest.mark.gpu


class Backwards(Tensor):
    """A tensor whose axes of `axes` lie in memory from the last index to the first: the view starts at element (0, 0, 0, 0) and its strides there are negative."""

    def __init__(self, rocm, x, dtype, axes, value=None):
        self.rocm, self.dtype, self.axes = rocm, dtype, axes
        self.shape = self.padded = x.shape if value is None else x
        host = np.full(self.shape, value, np.float32) if value is not None else x
        self.array, strides = upload(rocm, np.flip(host, axes), dtype), strides_of(self.shape, (0, 1, 2))
        first = sum((self.shape[a] - 1) * strides[a] for a in axes)
        self.view = view(self.array, [-s if a in axes else s for a, s in enumerate(strides)], 4 if dtype == "float32" else 2, first)

    def whole(self):
        return np.flip(download(self.array, self.dtype).reshape(self.shape), self.axes)


def run(rocm, c, x, tensor=None, in_place=False):
    """forward and backward, all outputs in 64 bits; tensor(x or shape, value) makes the tensors of heads; in_place: the states' gradients in one buffer"""
    tensor = tensor or (lambda x, value=None: Tensor(rocm, x, c["dtype"], value=value))
    layer, steps = layer_of(rocm, c, x), c["steps"]
    t = {n: tensor(x[n]) for n in ("q", "k", "v", "d_output")}
    o = {n: tensor(s, 7.0) for n, s in (("output", x["d_output"].shape), ("d_q", x["q"].shape), ("d_k", x["k"].shape), ("d_v", x["v"].shape))}
    state, d_state, reset, lengths = (rocm.array(x[n]) if x.get(n) is not None else None for n in ("state", "d_state", "reset", "lengths"))
    ptr = lambda a: a.ptr if a is not None else None
    shape = (c["rows"], c["heads"], c["dk"], c["dv"])
    final, d_initial, d_rate = filled(rocm, shape, "float32"), d_state if in_place else filled(rocm, shape, "float32"), filled(rocm, (c["heads"],), "float32")
    w, n = workspace(rocm, layer, steps, 0)
    rocm.call("linear_attention_forward", C.byref(layer), t["q"].view, t["k"].view, t["v"].view, o["output"].view, ptr(state), final.ptr, ptr(reset), ptr(lengths), steps, w.ptr, n)
    w, n = workspace(rocm, layer, steps, 1)
    rocm.call("linear_attention_backward", C.byref(layer), t["q"].view, t["k"].view, t["v"].view, t["d_output"].view, o["d_q"].view, o["d_k"].view, o["d_v"].view, ptr(state), ptr(d_state),
              d_initial.ptr, d_rate.ptr, 0, ptr(reset), ptr(lengths), steps, w.ptr, n)
    rocm.sync()
    return dict({n: a.numpy() for n, a in o.items()}, **{n: a.numpy().astype(np.float64) for n, a in (("state", final), ("d_state", d_initial), ("d_log_decay", d_rate))})


# ------------------------------------------------------------------ roundings


@gpu
@pytest.mark.parametrize("steps,rows,heads,d", [(16, 256, 8, 32), (16, 64, 8, 64), (12, 40, 8, 128)])
def test_bfloat16_outputs_are_rounded_once(rocm, steps, rows, heads, d):
    """An output is the bfloat16 number nearest to the exact value unless the midpoint between two numbers lies between that value and the one in 32 bits, which it does with a probability of their distance in units of
    the last place. That distance: 4 steps + channels + 16 roundings to 24 bits, each independent of the others, of values as large as the outputs. Scores, states or weighted values of 16 bits are three times as far off."""
    c, x = case(47, "bfloat16", steps, rows, heads, heads, d, d)
    want, got = reference(c, x), run(rocm, c, x)
    for n in ("output", "d_q", "d_k", "d_v"):
        last_place = 2.0 ** (np.floor(np.log2(np.abs(want[n]))) - 7)
        off = 2.0 ** -24 * (4 * steps + d + 16) ** 0.5 * np.sqrt(np.mean(want[n] ** 2))
        expected = np.sum(np.minimum(1, off / last_place))
        others = np.sum(got[n] != rounded(want[n], "bfloat16"))
        print(n, want[n].size, "elements", others, "elsewhere, at most", expected, flush=True)
        assert others <= expected + 5 * expected ** 0.5, n


# ------------------------------------------------------------------ views


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dk,dv", [(32, 32), (64, 64), (128, 128), (24, 41)])
@pytest.mark.parametrize("steps,rows", [(130, 3), (900, 1)])
def test_views_that_go_back_in_memory(rocm, dk, dv, steps, rows, dtype):
    """steps, and steps, rows and heads, with strides below zero: heads of whole tiles and others, whole and cut chunks, one segment and several"""
    print("case", steps, rows, dk, dv, dtype, flush=True)
    c, x = case(43, dtype, steps, rows, 4, 2, dk, dv, resets=0.02, ragged=rows > 1)
    for axes in ((0,), (0, 1, 2)):
        check(c, x, run(rocm, c, x, lambda x, value=None: Backwards(rocm, x, dtype, axes, value)))


# ------------------------------------------------------------------ values that are not finite


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("steps,rows,dk,dv", [(200, 3, 32, 32), (200, 2, 64, 48), (150, 2, 128, 128), (90, 3, 24, 41), (20, 2, 64, 64), (900, 1, 128, 128)])
@pytest.mark.parametrize("name", ["q", "k", "v", "d_output"])
def test_values_that_are_not_finite_reach_what_sees_them(rocm, steps, rows, dk, dv, name, dtype):
    """One channel of one row and head at some steps, no resets: outputs of the steps before, gradients of the steps behind, and channels that the value has no part in are as if it were finite, the others are not finite. What
    is finite in the recurrence itself, step by step in 64 bits, is what the formulas leave alone."""
    print("case", steps, rows, dk, dv, name, dtype, flush=True)
    c, x = case(53, dtype, steps, rows, 2, 2, dk, dv)
    for at, value in ((0, np.inf), (steps // 2 + 3, np.nan), (min(63, steps - 1), -np.inf), (steps - 1, np.nan)):
        y = {n: a.copy() for n, a in x.items()}
        y[name][at, 0, 1, dv // 3 if name in ("v", "d_output") else dk // 3] = value
        with np.errstate(invalid="ignore"):
            want = reference(c, y)
        b, got = bounds(c, reference(c, x), magnitudes(c, x)), run(rocm, c, y)
        for n in ("output", "state", "d_q", "d_k", "d_v", "d_state"):
            finite = np.isfinite(want[n])
            assert np.array_equal(np.isfinite(got[n]), finite), (n, at, value)
            assert np.all(np.abs(got[n][finite] - want[n][finite]) <= b[n][finite]), (n, at, value)


@gpu
@pytest.mark.parametrize("log_decay,steps", [(0.02, 200), (0.5, 300), (2.0, 70), (30.0, 40)])
def test_states_that_grow_beyond_fp32_are_infinite(rocm, log_decay, steps):
    """A logarithm above zero and sums of products of numbers from 1 on alone, which pass fp32's largest number on their way: what is beyond it by more than its bound is infinite, not a NaN."""
    c, x = case(59, "float32", steps, 1, 2, 2, 32, 32, log_decay=[log_decay, log_decay / 2])
    x = {n: (a if n == "log_decay" else (np.abs(a) + 1).astype(np.float32).astype(a.dtype)) for n, a in x.items()}
    c["scale"] = 1.0
    with np.errstate(over="ignore", invalid="ignore"):
        want, got, largest = reference(c, x), run(rocm, c, x), float(np.finfo(np.float32).max)
        b = bounds(c, want, want)
        for n in ("output", "state", "d_q", "d_k", "d_v", "d_state"):
            surely, within = (want[n] - b[n] > largest) | np.isinf(want[n]), want[n] + b[n] < largest
            assert np.all(got[n][surely] == np.inf) and np.all(np.abs(got[n] - want[n])[within] <= b[n][within]), (n, log_decay)


# ------------------------------------------------------------------ buffers


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("steps,rows,heads,kv_heads,dk,dv", [(70, 300, 4, 4, 32, 32), (30, 200, 4, 2, 64, 48), (1, 900, 2, 2, 128, 128), (900, 1, 2, 2, 64, 64), (900, 1, 2, 1, 128, 96)])
def test_the_states_gradient_in_place(rocm, steps, rows, heads, kv_heads, dk, dv, dtype):
    """one buffer for the final and the initial state's gradient, bit for bit as two, in one segment and several"""
    c, x = case(61, dtype, steps, rows, heads, kv_heads, dk, dv, resets=0.02, ragged=True)
    two, one = run(rocm, c, x), run(rocm, c, x, in_place=True)
    for n in two:
        assert np.array_equal(two[n], one[n]), n


# ------------------------------------------------------------------ more rows and heads than a launch holds


MOST = [  # type, width, the most rows x heads: forward, backward, step
    ("float32", 128, 8388607, 4194296, 16777215), ("float32", 64, 16777215, 8388600, 16777215), ("float32", 32, 33554431, 16777208, 33554431),
    ("bfloat16", 128, 16777215, 8388600, 16777215), ("bfloat16", 64, 16777215, 8388600, 16777215), ("bfloat16", 32, 33554431, 16777208, 33554431)]


@pytest.mark.parametrize("dtype,width,forward,backward,step", MOST)
def test_scratch_memory_ends_where_launches_do(dtype, width, forward, backward, step):
    """fewer than 2^32 threads: two walks of 512, 256 or 128 threads for each eight heads' gradients (no GPU is asked)"""
    lib = helpers.package().load_library()
    of = lambda batch: lib.rlt_rocm_linear_attention_workspace_bytes(C.byref(capi.LinearAttention(scale=1.0, type=capi.TYPE[dtype], batch=batch, heads=1, kv_heads=1, key_dim=width, value_dim=width)), 2, 1)
    assert of(backward) > 0 and of(backward + 1) == 0 and of(33554432) == 0
    threads = {128: 512 if dtype == "float32" else 256, 64: 256, 32: 128}[width]
    assert -(-backward // 8) * 16 * threads < 2 ** 32 <= -(-(backward + 1) // 8) * 16 * threads


@gpu
@pytest.mark.parametrize("dtype,width,forward,backward,step", MOST)
def test_more_rows_and_heads_than_a_launch_holds_are_refused(rocm, dtype, width, forward, backward, step):
    """by the host, before the first launch: nothing is written"""
    lib, h = rocm.device.lib, rocm.device.handle
    decay, a = rocm.zeros((4,)), filled(rocm, (4096,), "float32")
    view = C.byref(capi.HeadView(a.ptr, 0, 0, 0))
    layer = lambda batch, heads=1: C.byref(capi.LinearAttention(log_decay=decay.ptr, scale=1.0, type=capi.TYPE[dtype], batch=batch, heads=heads, kv_heads=heads, key_dim=width, value_dim=width))
    for one in (layer(forward + 1), layer(33554432), layer(1 << 16, 1 << 16)):
        assert lib.rlt_rocm_linear_attention_forward(h, one, *[view] * 4, None, None, None, None, 2, a.ptr, 16384) == capi.RLT_E_UNSUPPORTED
    assert lib.rlt_rocm_linear_attention_forward(h, layer(step + 1), *[view] * 4, None, a.ptr, None, None, 1, a.ptr, 16384) == capi.RLT_E_UNSUPPORTED
    assert lib.rlt_rocm_linear_attention_step(h, layer(step + 1), *[view] * 4, a.ptr, a.ptr, None) == capi.RLT_E_UNSUPPORTED
    for one in (layer(backward + 1), layer(1, backward + 1)):
        for d_log_decay in (None, a.ptr):
            assert lib.rlt_rocm_linear_attention_backward(h, one, *[view] * 7, None, None, None, d_log_decay, 1, None, None, 2, a.ptr, 1 << 62) == capi.RLT_E_UNSUPPORTED
    assert lib.rlt_rocm_linear_attention_backward(h, layer(1, 8388608), *[view] * 7, None, None, None, a.ptr, 1, None, None, 2, a.ptr, 1 << 62) == capi.RLT_E_UNSUPPORTED      # a workgroup of 512 sums up a head's decay
    rocm.sync()
    assert np.all(a.numpy() == 7.0)


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("steps,rows,heads,kv_heads,dk,dv", [(66, 500, 128, 64, 4, 4), (33, 65, 64, 32, 33, 33)])
def test_shared_heads_of_more_tokens_than_the_grid(rocm, steps, rows, heads, kv_heads, dk, dv, dtype):
    """the sums over heads take 2,048 workgroups of 1,024 elements (or vectors of four) at a time"""
    elements = kv_heads * (dk // 4 if dk % 4 == 0 else dk)
    assert steps * rows > 2048 * max(1, 1024 // elements)
    c, x = case(67, dtype, steps, rows, heads, kv_heads, dk, dv, resets=0.02, ragged=True)
    got = run(rocm, c, x)
    check(c, x, got, ["d_k", "d_v"])

"""The short causal convolution, forward, backward and single steps, against the definition in 64 bits, step by step.

Bounds, set before the first run; u = 2^-24. With all factors replaced by their absolute values the reference gives the sum of the products' magnitudes, M. A sum before the activation has width + 1 roundings at most on the way of
a product: (width + 2) u M. z sigmoid(z) has a slope of at most 1.1, and its own exponential, sum, reciprocal and products are ten roundings (the exponential two units in the last place): the activated output is off by
(1.1 (width + 2) + 12) u M', M' the magnitude of z. Gradients before the activation: the slope's own slope is at most 0.5, so 0.5 (width + 2) u M' |d| + 14 u |d|; each then passes at most width + 1 roundings in the input's gradient and, in the sums over
steps and rows of the weights' gradient, at most one for each step and row that is added: (steps + rows + width + 16) u of the sum of magnitudes. bfloat16 adds the output's own rounding, 2^-8 of the value."""
import ctypes as C

import numpy as np
import pytest

from helpers import capi
from test_rocm_linear_attention import Tensor, strides_of, view
from typed_arrays import UNIT, filled, rounded, to_bits, upload

gpu = pytest.mark.gpu
U = 2.0 ** -24


def sigmoid(z):
    return np.where(z >= 0, 1 / (1 + np.exp(-np.abs(z))), np.exp(-np.abs(z)) / (1 + np.exp(-np.abs(z))))


def reference(c, x, pre=None):
    """Step by step in 64 bits: the window of the last inputs, which a reset empties; then its gradient from the last step to the first. pre: the values before the activation where those of x are not meant (magnitudes)."""
    steps, rows, w = c["steps"], c["rows"], c["width"]
    taps = x["weights"].T[:, None].astype(np.float64)      # [width, 1, channels], the step's own last
    bias = x["biases"] if x.get("biases") is not None else 0.0
    lengths = np.clip(x["lengths"], 0, steps) if x.get("lengths") is not None else np.full(rows, steps)
    window = np.zeros((w - 1, rows, c["channels"])) if x.get("state") is None else x["state"].transpose(1, 0, 2).astype(np.float64)
    z, out, kept = np.zeros_like(x["x"]), np.zeros_like(x["x"]), []
    for t in range(steps):
        live, begins = (t < lengths)[:, None], (x["reset"][t] != 0)[:, None] if x.get("reset") is not None else np.zeros((rows, 1), bool)
        full = np.concatenate([np.where(begins, 0.0, window), x["x"][t][None]])
        kept.append(full)
        with np.errstate(invalid="ignore"):
            z[t] = np.where(live, bias + (taps * full).sum(0), 0.0)
            out[t] = np.where(live, z[t] * sigmoid(z[t]) if c["silu"] and pre is None else z[t], 0.0)
        window = np.where(live, full[1:], window)
    state = window.transpose(1, 0, 2)
    at = z if pre is None else pre
    slope = sigmoid(at) * (1 + at * sigmoid(-at)) if c["silu"] else np.ones_like(z)
    slope = slope if pre is None else np.abs(slope)
    d_window = np.zeros_like(window) if x.get("d_state") is None else x["d_state"].transpose(1, 0, 2).astype(np.float64)
    d_x, d_taps, d_bias, d_z = np.zeros_like(x["x"]), np.zeros((w, c["channels"])), np.zeros(c["channels"]), np.zeros_like(x["x"])
    for t in reversed(range(steps)):
        live, begins = (t < lengths)[:, None], (x["reset"][t] != 0)[:, None] if x.get("reset") is not None else np.zeros((rows, 1), bool)
        d = d_z[t] = np.where(live, x["d_output"][t] * slope[t], 0.0)
        full = np.where(live, kept[t], 0.0)
        d_taps += (d * full).sum(1)
        d_bias += d.sum(0)
        d_full = np.concatenate([np.zeros((1, rows, c["channels"])), d_window]) + taps * d
        d_x[t] = np.where(live, d_full[-1], 0.0)
        d_window = np.where(live, np.where(begins, 0.0, d_full[:-1]), d_window)
    return dict(output=out, state=state, d_x=d_x, d_weights=d_taps.T, d_biases=d_bias, d_state=d_window.transpose(1, 0, 2), pre=z)


def case(seed, dtype, steps, rows, channels, width, resets=0.0, ragged=False, silu=1, with_state=True, biases=True):
    rng = np.random.default_rng(seed)
    n = lambda *shape: rounded(rng.standard_normal(shape), dtype)
    x = dict(x=n(steps, rows, channels), d_output=n(steps, rows, channels), weights=(rng.standard_normal((channels, width)) / np.sqrt(width)).astype(np.float32))
    if biases:
        x["biases"] = (0.3 * rng.standard_normal(channels)).astype(np.float32)
    if with_state:
        x["state"], x["d_state"] = (rng.standard_normal((rows, width - 1, channels)).astype(np.float32) for _ in range(2))
    if resets:
        x["reset"] = (rng.random((steps, rows)) < resets).astype(np.uint8)
    if ragged:
        x["lengths"] = rng.integers(0, steps + 1, rows).astype(np.int32)
        x["lengths"][0], x["lengths"][-1] = 0, steps + 5      # an empty row; one that claims more than there is
    return dict(dtype=dtype, steps=steps, rows=rows, channels=channels, width=width, silu=silu), x


def bounds(c, x, want):
    size = reference(c, {n: (a if n in ("reset", "lengths") else np.abs(a)) for n, a in x.items()}, pre=want["pre"])
    w = c["width"]
    z = (w + 2) * U * size["pre"]
    b = {"output": (1.1 * z + 12 * U * size["pre"]) if c["silu"] else z, "state": 0.0 * want["state"]}
    # the gradient before the activation: what its own error adds goes through the rest as another gradient
    slope_error = 0.5 * z + 14 * U if c["silu"] else 0.0 * z
    extra = reference(dict(c, silu=0), {n: (a if n in ("reset", "lengths") else np.abs(a)) for n, a in dict(x, d_output=np.abs(x["d_output"]) * slope_error, d_state=0.0 * size["state"]).items()})
    for n in ("d_x", "d_state"):
        b[n] = extra[n] + (w + 3) * U * size[n]
    for n in ("d_weights", "d_biases"):
        b[n] = extra[n] + (c["steps"] + c["rows"] + w + 16) * U * size[n]
    if c["dtype"] == "bfloat16":
        for n in ("output", "d_x"):
            b[n] = b[n] + UNIT["bfloat16"] * (np.abs(want[n]) + b[n])
    return b


def check(c, x, got, names=None):
    want = reference(c, x)
    b = bounds(c, x, want)
    for n in names or [n for n in want if n != "pre"]:
        off = np.abs(got[n] - want[n]) - b[n]
        assert np.all(off <= 0), (n, float(off.max()), float(np.abs(got[n] - want[n]).max()), float(np.abs(want[n]).max()))


def three(rocm, x, dtype, gap=0, offset=0, order=(0, 1, 2), value=None):
    """[steps, rows, channels] as a tensor of one head"""
    return Tensor(rocm, x[:, :, None] if value is None else tuple(x[:2]) + (1, x[2]), dtype, order, gap, value, offset)


def layer_of(rocm, c, x, keep, gradients=True, onto=7.0):
    up = lambda n: rocm.array(x[n]) if x.get(n) is not None else None
    keep["weights"], keep["biases"] = up("weights"), up("biases")
    keep["d_weights"], keep["d_biases"] = rocm.array(np.full((c["channels"], c["width"]), onto, np.float32)), rocm.array(np.full(c["channels"], onto, np.float32))
    ptr = lambda a: a.ptr if a is not None else None
    return capi.CausalConvolution(keep["weights"].ptr, ptr(keep["biases"]), keep["d_weights"].ptr if gradients else None, keep["d_biases"].ptr if gradients else None, capi.TYPE[c["dtype"]], c["rows"],
                                  c["channels"], c["width"], c["silu"], 0)


def workspace(rocm, layer, steps):
    n = rocm.device.lib.rlt_rocm_causal_convolution_workspace_bytes(C.byref(layer), steps)
    return rocm.device.empty((max(int(n), 16),), np.uint8), n


def run(rocm, c, x, gap=0, offset=0, order=(0, 1, 2), onto=None):
    keep, dtype, steps = {}, c["dtype"], c["steps"]
    layer = layer_of(rocm, c, x, keep, onto=7.0 if onto is None else onto)
    shape = (steps, c["rows"], c["channels"])
    t = {n: three(rocm, x[n], dtype, gap, offset, order) for n in ("x", "d_output")}
    o = {n: three(rocm, shape, dtype, gap, offset, order, value=7.0) for n in ("output", "d_x")}
    up = lambda n: rocm.array(x[n]) if x.get(n) is not None else None
    ptr = lambda a: a.ptr if a is not None else None
    state, d_state, reset, lengths = up("state"), up("d_state"), up("reset"), up("lengths")
    final, d_initial = (filled(rocm, (c["rows"], c["width"] - 1, c["channels"]), "float32") for _ in range(2))
    rocm.call("causal_convolution_forward", C.byref(layer), t["x"].view, o["output"].view, ptr(state), final.ptr, ptr(reset), ptr(lengths), steps)
    w, n = workspace(rocm, layer, steps)
    rocm.call("causal_convolution_backward", C.byref(layer), t["x"].view, t["d_output"].view, o["d_x"].view, ptr(state), ptr(d_state), d_initial.ptr, int(onto is not None), ptr(reset), ptr(lengths), steps, w.ptr, n)
    rocm.sync()
    for a in o.values():
        assert np.all(a.whole()[..., a.shape[3]:] == 7.0)      # nothing is written between the rows
    f = lambda a: a.numpy().astype(np.float64)
    return dict(output=o["output"].numpy()[:, :, 0], d_x=o["d_x"].numpy()[:, :, 0], state=f(final), d_state=f(d_initial), d_weights=f(keep["d_weights"]), d_biases=f(keep["d_biases"]))


def test_the_references_gradients_are_its_differences():
    c, x = case(0, "float32", 9, 3, 4, 3, resets=0.2, ragged=True)
    x = {n: (a.astype(np.float64) if a.dtype.kind == "f" else a) for n, a in x.items()}

    def loss(y):
        r = reference(c, y)
        return (r["output"] * x["d_output"]).sum() + (r["state"] * x["d_state"]).sum()
    got, rng = reference(c, x), np.random.default_rng(2)
    for name, grad in (("x", "d_x"), ("weights", "d_weights"), ("biases", "d_biases"), ("state", "d_state")):
        direction, h = rng.standard_normal(x[name].shape), 1e-5
        numeric = (loss(dict(x, **{name: x[name] + h * direction})) - loss(dict(x, **{name: x[name] - h * direction}))) / (2 * h)
        assert abs(numeric - (got[grad] * direction).sum()) <= 1e-7 * max(1.0, abs(numeric)), name


SHAPES = [  # steps, rows, channels, width
    (1, 1, 1, 2), (1, 3, 8, 4), (2, 2, 16, 4), (3, 2, 5, 8), (7, 3, 64, 3), (8, 2, 24, 8), (15, 1, 32, 5), (16, 4, 33, 4), (17, 2, 16, 6), (31, 3, 40, 2), (64, 2, 64, 4), (100, 3, 7, 7), (333, 2, 24, 3), (700, 1, 16, 4), (20, 300, 8, 4)]


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_backward(rocm, shape, dtype):
    print("case", shape, dtype, flush=True)
    c, x = case(sum(shape), dtype, *shape)
    check(c, x, run(rocm, c, x))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [(1, 5, 16, 4), (5, 4, 8, 8), (40, 6, 24, 4), (100, 5, 33, 3), (200, 3, 16, 7)])
@pytest.mark.parametrize("resets", [0.02, 0.3, 1.0])
def test_resets_and_lengths(rocm, shape, dtype, resets):
    print("case", shape, dtype, resets, flush=True)
    c, x = case(sum(shape), dtype, *shape, resets=resets, ragged=True)
    check(c, x, run(rocm, c, x))


@gpu
@pytest.mark.parametrize("shape,dtype", [((24, 140, 4096, 4), "float32"), ((24, 140, 4095, 4), "float32"), ((20, 140, 8192, 3), "bfloat16"), ((17, 140, 8191, 2), "bfloat16"), ((100, 34, 4096, 3), "float32")])
def test_rows_and_segments_that_a_thread_goes_through_one_after_the_other(rocm, shape, dtype):
    """more of them than lanes, and segments of more steps than are on their way at a time; what lies beyond a row's length is not looked at"""
    print("case", shape, dtype, flush=True)
    c, x = case(sum(shape), dtype, *shape, resets=0.05, ragged=True)
    beyond = np.arange(shape[0])[:, None] >= np.clip(x["lengths"], 0, shape[0])[None]
    layer = layer_of(rocm, c, x, {})
    assert workspace(rocm, layer, shape[0])[1] < shape[1] * (-(-shape[0] // 25)) * (shape[3] + 1) * shape[2] * 4      # fewer threads share a channel than there are rows and segments (of 25 steps at the most here)
    got = run(rocm, c, dict(x, x=np.where(beyond[..., None], np.nan, x["x"]), d_output=np.where(beyond[..., None], np.inf, x["d_output"]), reset=np.where(beyond, 1, x["reset"]).astype(np.uint8)))
    check(c, x, got)


@gpu
@pytest.mark.parametrize("gap,offset,order", [(5, 3, (0, 1, 2)), (8, 0, (0, 1, 2)), (1, 1, (1, 0, 2)), (0, 0, (1, 0, 2)), (16, 8, (1, 0, 2))])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_orders_gaps_and_alignments(rocm, gap, offset, order, dtype):
    print("case", gap, offset, order, dtype, flush=True)
    c, x = case(5, dtype, 50, 3, 32, 4, resets=0.1, ragged=True)
    check(c, x, run(rocm, c, x, gap, offset, order))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_sequence_backwards_in_memory(rocm, dtype):
    c, x = case(9, dtype, 70, 2, 16, 4)
    keep, item = {}, 4 if dtype == "float32" else 2
    layer = layer_of(rocm, c, x, keep)
    tensors = {n: upload(rocm, np.ascontiguousarray(x[n][::-1]), dtype) for n in ("x", "d_output")}
    outs = {n: filled(rocm, x["x"].shape, dtype) for n in ("output", "d_x")}
    back = lambda a: view(a, (-2 * 16, 16, 0), item, 69 * 2 * 16)
    state, d_state = rocm.array(x["state"]), rocm.array(x["d_state"])
    final, d_initial = filled(rocm, x["state"].shape, "float32"), filled(rocm, x["state"].shape, "float32")
    rocm.call("causal_convolution_forward", C.byref(layer), back(tensors["x"]), back(outs["output"]), state.ptr, final.ptr, None, None, 70)
    w, n = workspace(rocm, layer, 70)
    rocm.call("causal_convolution_backward", C.byref(layer), back(tensors["x"]), back(tensors["d_output"]), back(outs["d_x"]), state.ptr, d_state.ptr, d_initial.ptr, 0, None, None, 70, w.ptr, n)
    rocm.sync()
    from typed_arrays import download
    check(c, x, dict(output=download(outs["output"], dtype)[::-1], d_x=download(outs["d_x"], dtype)[::-1], state=final.numpy().astype(np.float64), d_state=d_initial.numpy().astype(np.float64),
                     d_weights=keep["d_weights"].numpy().astype(np.float64), d_biases=keep["d_biases"].numpy().astype(np.float64)))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("silu", [0, 1])
def test_without_states_biases_or_activation(rocm, dtype, silu):
    c, x = case(11, dtype, 40, 3, 24, 4, silu=silu, with_state=False, biases=False)
    check(c, x, run(rocm, c, x))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_what_lies_beyond_a_rows_length_or_before_a_reset_is_not_looked_at(rocm, dtype):
    c, x = case(17, dtype, 120, 6, 16, 4, ragged=True)
    x["reset"] = np.zeros((120, 6), np.uint8)
    x["reset"][0] = 1
    x["reset"][60, 5] = 1
    beyond = np.arange(120)[:, None] >= np.clip(x["lengths"], 0, 120)[None]
    clean = {n: a.copy() for n, a in x.items()}
    x["x"][beyond], x["d_output"][beyond] = np.nan, np.inf
    x["state"][1:] = np.nan
    clean["state"][1:] = 0.0
    got = run(rocm, c, x)
    names = ["output", "d_x", "d_weights", "d_biases", "d_state"]
    check(c, clean, got, names)
    full = np.clip(x["lengths"], 0, 120) > 0
    assert np.all(got["output"][beyond] == 0) and np.all(got["d_x"][beyond] == 0) and np.array_equal(got["state"][0], x["state"][0].astype(np.float64)) and np.isfinite(got["state"][full]).all()
    x, clean = clean, {n: a.copy() for n, a in clean.items()}
    x["x"][57, 5], x["d_output"][58, 5] = np.nan, np.nan      # values of the episode before: the next one is as if they were not
    got, want = run(rocm, c, x), reference(c, clean)
    b = bounds(c, clean, want)
    assert np.all(np.abs(got["output"][60:] - want["output"][60:]) <= b["output"][60:]) and np.all(np.abs(got["d_x"][60:] - want["d_x"][60:]) <= b["d_x"][60:])
    assert np.all(np.abs(got["output"][:, :5] - want["output"][:, :5]) <= b["output"][:, :5])


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,channels,width", [(1, 1, 2), (64, 32, 4), (3, 33, 3), (5, 8, 8), (300, 16, 4)])
@pytest.mark.parametrize("in_place", [False, True])
def test_steps_walk_a_sequence(rocm, rows, channels, width, dtype, in_place):
    print("case", rows, channels, width, dtype, in_place, flush=True)
    c, x = case(rows + width, dtype, 6, rows, channels, width, resets=0.3)
    x["reset"][0, 0] = 1
    clean = {n: a.copy() for n, a in x.items()}
    x["state"][0], clean["state"][0] = np.nan, 0.0
    want, keep = reference(c, clean), {}
    b, layer = bounds(c, clean, want), layer_of(rocm, c, x, keep)
    state, other, reset = rocm.array(x["state"]), filled(rocm, x["state"].shape, "float32"), rocm.array(x["reset"])
    inputs, out, item = three(rocm, x["x"], dtype), three(rocm, x["x"].shape, dtype, value=7.0), 4 if dtype == "float32" else 2
    for t in range(6):
        one = [view(a.array, strides_of(a.padded, a.order), item, t * rows * channels) for a in (inputs, out)]
        to = state if in_place else other
        rocm.call("causal_convolution_step", C.byref(layer), *one, state.ptr, to.ptr, reset.ptr + t * rows)
        if not in_place:
            state, other = other, state
    rocm.sync()
    assert np.all(np.abs(out.numpy()[:, :, 0] - want["output"]) <= b["output"]) and np.array_equal(state.numpy().astype(np.float64), want["state"])


@gpu
def test_gradients_add_up_and_runs_repeat_bit_for_bit(rocm):
    c, x = case(23, "float32", 200, 40, 24, 4, resets=0.02, ragged=True)
    first, second, onto = run(rocm, c, x), run(rocm, c, x), run(rocm, c, x, onto=3.0)
    for n in first:
        assert np.array_equal(first[n], second[n]), n
    for n in ("d_weights", "d_biases"):
        assert np.allclose(onto[n], first[n] + 3.0, rtol=2e-7, atol=0)


@gpu
@pytest.mark.parametrize("steps", [3, 200])
def test_the_states_buffer_may_be_the_same(rocm, steps):
    c, x = case(29, "float32", steps, 4, 16, 4, resets=0.05, ragged=True)
    want, keep = run(rocm, c, x), {}
    layer = layer_of(rocm, c, x, keep)
    inputs, out = three(rocm, x["x"], "float32"), three(rocm, x["x"].shape, "float32", value=7.0)
    state, reset, lengths = rocm.array(x["state"]), rocm.array(x["reset"]), rocm.array(x["lengths"])
    rocm.call("causal_convolution_forward", C.byref(layer), inputs.view, out.view, state.ptr, state.ptr, reset.ptr, lengths.ptr, steps)
    assert np.array_equal(out.numpy()[:, :, 0], want["output"]) and np.array_equal(state.numpy().astype(np.float64), want["state"])


@gpu
def test_a_graph_replays_forward_and_backward(rocm):
    lib, h, keep = rocm.device.lib, rocm.device.handle, {}
    c, x = case(31, "bfloat16", 100, 3, 64, 4, resets=0.02, ragged=True)
    want = run(rocm, c, x)
    layer = layer_of(rocm, c, x, keep)
    t = {n: three(rocm, x[n], "bfloat16") for n in ("x", "d_output")}
    o = {n: three(rocm, x["x"].shape, "bfloat16", value=7.0) for n in ("output", "d_x")}
    state, d_state, reset, lengths = (rocm.array(x[n]) for n in ("state", "d_state", "reset", "lengths"))
    final, d_initial = rocm.zeros(x["state"].shape), rocm.zeros(x["state"].shape)
    w, n = workspace(rocm, layer, 100)
    rocm.sync()
    assert lib.rlt_rocm_graph_begin_capture(h) == 0
    rocm.call("causal_convolution_forward", C.byref(layer), t["x"].view, o["output"].view, state.ptr, final.ptr, reset.ptr, lengths.ptr, 100)
    rocm.call("causal_convolution_backward", C.byref(layer), t["x"].view, t["d_output"].view, o["d_x"].view, state.ptr, d_state.ptr, d_initial.ptr, 0, reset.ptr, lengths.ptr, 100, w.ptr, n)
    graph = C.c_void_p()
    assert lib.rlt_rocm_graph_end_capture(h, C.byref(graph)) == 0
    for _ in range(3):
        for a in o.values():
            a.array.upload(to_bits(np.full(a.array.shape, 7.0, np.float32)))      # eager work between the replays
        assert lib.rlt_rocm_graph_launch(h, graph) == 0
        rocm.sync()
        for name, a in o.items():
            assert np.array_equal(a.numpy()[:, :, 0], want[name]), name
        assert np.array_equal(final.numpy().astype(np.float64), want["state"]) and np.array_equal(keep["d_weights"].numpy().astype(np.float64), want["d_weights"])
    lib.rlt_rocm_graph_destroy(h, graph)


def test_refusals_without_a_device():
    lib = __import__("helpers").package().load_library()
    good = capi.CausalConvolution(4096, None, 4096, None, 0, 2, 8, 4, 1, 0)
    size = lambda steps=10, **fields: lib.rlt_rocm_causal_convolution_workspace_bytes(C.byref(capi.CausalConvolution(**dict({n: getattr(good, n) for n, _ in good._fields_}, **fields))), steps)
    assert size() > 0
    assert size(d_weights=None) == size(0) == size(2 ** 30 + 1) == size(width=1) == size(width=9) == size(channels=0) == size(batch=-1) == size(type=2) == size(batch=2 ** 24, channels=2 ** 8) == size(batch=1, channels=2 ** 22 + 1) == size(batch=2 ** 24 + 1, channels=1) == 0
    assert lib.rlt_rocm_causal_convolution_forward(None, C.byref(good), None, None, None, None, None, None, 4) == capi.RLT_E_NOT_INITIALISED


@gpu
def test_refusals(rocm):
    lib, h, keep = rocm.device.lib, rocm.device.handle, {}
    c, x = case(37, "float32", 4, 2, 8, 4)
    good = layer_of(rocm, c, x, keep)
    t, out, state = three(rocm, x["x"], "float32"), three(rocm, x["x"].shape, "float32", value=7.0), rocm.array(x["state"])
    none = C.byref(capi.HeadView(None, 1, 1, 1))
    w, n = workspace(rocm, good, 4)

    def changed(**fields):
        return C.byref(capi.CausalConvolution(**dict({name: getattr(good, name) for name, _ in good._fields_}, **fields)))

    def forward(layer=C.byref(good), a=t.view, b=out.view, steps=4):
        return lib.rlt_rocm_causal_convolution_forward(h, layer, a, b, None, None, None, None, steps)

    def backward(layer=C.byref(good), a=t.view, b=t.view, d=out.view, entry=None, given=None, to=None, ptr=w.ptr, size=n):
        return lib.rlt_rocm_causal_convolution_backward(h, layer, a, b, d, entry, given, to, 0, None, None, 4, ptr, size)

    def step(layer=C.byref(good), a=t.view, b=out.view, state=state.ptr, to=state.ptr):
        return lib.rlt_rocm_causal_convolution_step(h, layer, a, b, state, to, None)
    assert forward() == backward() == step() == 0
    for call in (forward, backward, step):
        for layer in (None, changed(type=2), changed(batch=0), changed(channels=-1), changed(width=0), changed(weights=None)):
            assert call(layer) == capi.RLT_E_INVALID_ARGUMENT
        assert call(changed(width=1)) == call(changed(width=9)) == call(changed(batch=2 ** 24, channels=2 ** 20)) == capi.RLT_E_UNSUPPORTED
        assert call(a=none) == call(a=None) == call(b=none) == capi.RLT_E_INVALID_ARGUMENT
    assert forward(steps=0) == forward(steps=-3) == backward(ptr=None) == backward(size=n - 1) == backward(ptr=w.ptr + 4) == backward(d=none) == capi.RLT_E_INVALID_ARGUMENT
    assert forward(steps=2 ** 30 + 1) == capi.RLT_E_UNSUPPORTED
    assert backward(given=state.ptr, to=state.ptr) == backward(entry=state.ptr, to=state.ptr) == step(state=None) == step(to=None) == capi.RLT_E_INVALID_ARGUMENT
    rocm.sync()

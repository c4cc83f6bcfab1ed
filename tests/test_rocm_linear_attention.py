"""Linear attention with a decay for each head, forward, backward and single steps, against the recurrence in 64 bits.

Bounds, set before the first run. Every output is a sum of products; with all inputs replaced by their absolute values the reference gives the sum of the products' magnitudes, M. A product passes at most 4 roundings a
step (decay, its power's argument, product, sum) and the sums over a head's channels: (4 steps + channels + 16) * 2^-24 * M in fp32. bfloat16 adds the output's own rounding, 2^-8 of the value, and the kernels' operands in
two bfloat16 parts (16 bits) at two places in a row: 2^-15 * M. The decay's gradient adds the sums over steps, rows and workgroups of the same products: the same bound times two."""
import ctypes as C

import numpy as np
import pytest

from helpers import capi
from typed_arrays import UNIT, download, filled, rounded, to_bits, upload

gpu = pytest.mark.gpu


def reference(c, x):
    """x: q, k, v [steps, rows, heads, d], log_decay, state (or None), reset, lengths (or None), d_output, d_state (or None), in 64 bits. All outputs by the recurrence."""
    steps, rows, heads, dk = x["q"].shape
    group, dv = heads // x["k"].shape[2], x["v"].shape[3]
    k, v = np.repeat(x["k"], group, 2), np.repeat(x["v"], group, 2)
    lengths = np.clip(x["lengths"], 0, steps) if x.get("lengths") is not None else np.full(rows, steps)
    decay = np.exp(x["log_decay"].astype(np.float64))
    state = np.zeros((rows, heads, dk, dv)) if x.get("state") is None else x["state"].astype(np.float64)
    slope, d_rate = np.zeros_like(state), np.zeros((heads,))
    out, d = np.zeros((steps, rows, heads, dv)), c["scale"] * x["d_output"]
    d_q, d_k, d_v = np.zeros_like(x["q"]), np.zeros_like(k), np.zeros_like(v)
    kept = [np.where(x["reset"][t].astype(bool)[:, None] if x.get("reset") is not None else False, 0.0, decay[None])[..., None, None] for t in range(steps)]
    for t in range(steps):
        live = (t < lengths)[:, None, None, None]
        slope = np.where(live, kept[t] * (slope + state), slope)
        with np.errstate(invalid="ignore"):
            state = np.where(live, kept[t] * state + k[t][..., :, None] * v[t][..., None, :], state)
            out[t] = np.where(live[..., 0], c["scale"] * np.einsum("bhi,bhij->bhj", x["q"][t], state), 0.0)
            d_q[t] = np.where(live[..., 0], np.einsum("bhj,bhij->bhi", d[t], state), 0.0)
            d_rate += np.where(live, x["q"][t][..., :, None] * slope * d[t][..., None, :], 0.0).sum((0, 2, 3))
    grad = np.zeros_like(state) if x.get("d_state") is None else x["d_state"].astype(np.float64)
    d_rate += (grad * slope).sum((0, 2, 3))
    for t in reversed(range(steps)):
        live = (t < lengths)[:, None, None, None]
        here = grad + x["q"][t][..., :, None] * d[t][..., None, :]
        d_k[t] = np.where(live[..., 0], np.einsum("bhij,bhj->bhi", here, v[t]), 0.0)
        d_v[t] = np.where(live[..., 0], np.einsum("bhij,bhi->bhj", here, k[t]), 0.0)
        grad = np.where(live, kept[t] * here, grad)
    shared = lambda g: g.reshape(steps, rows, heads // group, group, -1).sum(3)
    return dict(output=out, state=state, d_q=d_q, d_k=shared(d_k), d_v=shared(d_v), d_state=grad, d_log_decay=d_rate)


def case(seed, dtype, steps, rows, heads, kv_heads, dk, dv, resets=0.0, ragged=False, with_state=True, log_decay=None):
    rng = np.random.default_rng(seed)
    n = lambda *shape: rounded(rng.standard_normal(shape), dtype)
    x = dict(q=n(steps, rows, heads, dk), k=n(steps, rows, kv_heads, dk), v=n(steps, rows, kv_heads, dv), d_output=n(steps, rows, heads, dv))
    x["log_decay"] = (np.log1p(-np.exp(rng.uniform(np.log(1 / 256), np.log(1 / 4), heads))) if log_decay is None else np.asarray(log_decay)).astype(np.float32)
    if with_state:
        x["state"], x["d_state"] = (rng.standard_normal((rows, heads, dk, dv)).astype(np.float32) for _ in range(2))
    if resets:
        x["reset"] = (rng.random((steps, rows)) < resets).astype(np.uint8)
    if ragged:
        x["lengths"] = rng.integers(0, steps + 1, rows).astype(np.int32)
        x["lengths"][0], x["lengths"][-1] = 0, steps + 5      # an empty row; one that claims more than there is
    return dict(dtype=dtype, steps=steps, rows=rows, heads=heads, kv_heads=kv_heads, dk=dk, dv=dv, scale=float(np.float32(dk ** -0.5))), x


def magnitudes(c, x):
    return reference(c, {n: (a if n in ("log_decay", "reset", "lengths") else np.abs(a)) for n, a in x.items()})


def bounds(c, want, size):
    steps = c["steps"]
    unit = (4 * steps + max(c["dk"], c["dv"]) + 16) * 2.0 ** -24
    b = {n: unit * m for n, m in size.items()}
    if c["dtype"] == "bfloat16":
        for n in ("output", "d_q", "d_k", "d_v"):
            b[n] = b[n] + UNIT["bfloat16"] * np.abs(want[n]) + 2.0 ** -15 * size[n]
        for n in ("state", "d_state", "d_log_decay"):
            b[n] = b[n] + 2.0 ** -15 * size[n]
    b["d_log_decay"] = 2 * b["d_log_decay"]
    return b


def view(array, strides, itemsize, offset=0):
    return C.byref(capi.HeadView(array.ptr + offset * itemsize, *strides))


def strides_of(shape, order):
    """element strides of [steps, rows, heads, channels] laid out with the axes of `order` from the slowest to the fastest (channels last)"""
    s, step = [0, 0, 0], shape[3]
    for axis in reversed(order):
        s[axis] = step
        step *= shape[axis]
    return tuple(s)


class Tensor:
    """A [steps, rows, heads, channels] tensor on the device in an order of its axes, `gap` elements behind every row of channels."""

    def __init__(self, rocm, x, dtype, order=(0, 1, 2), gap=0, value=None, offset=0):
        self.rocm, self.dtype, self.order, self.gap, self.offset = rocm, dtype, order, gap, offset
        self.shape = x.shape if value is None else x
        padded = tuple(self.shape[:3]) + (self.shape[3] + gap,)
        self.padded, host = padded, np.full(padded, 99.0 if value is None else value, np.float32)
        if value is None:
            host[..., :self.shape[3]] = x
        self.array = upload(rocm, np.concatenate([np.full(offset, 5.0, np.float32), host.transpose(*order, 3).reshape(-1)]), dtype)
        self.view = view(self.array, strides_of(padded, order), 4 if dtype == "float32" else 2, offset)

    def whole(self):
        flat = download(self.array, self.dtype)[self.offset:]
        moved = flat.reshape([self.padded[a] for a in self.order] + [self.padded[3]])
        return moved.transpose([self.order.index(a) for a in range(3)] + [3])

    def numpy(self):
        return self.whole()[..., :self.shape[3]]


def layer_of(rocm, c, x):
    decay = rocm.array(x["log_decay"])
    return capi.LinearAttention(log_decay=decay.ptr, scale=c["scale"], type=capi.TYPE[c["dtype"]], batch=c["rows"], heads=c["heads"], kv_heads=c["kv_heads"], key_dim=c["dk"], value_dim=c["dv"])


def workspace(rocm, layer, steps, backward):
    n = rocm.device.lib.rlt_rocm_linear_attention_workspace_bytes(C.byref(layer), steps, backward)
    return rocm.device.empty((max(int(n), 4),), np.uint8), n


def run(rocm, c, x, order=(0, 1, 2), gap=0, offset=0, accumulate_onto=None):
    layer, dtype, steps = layer_of(rocm, c, x), c["dtype"], c["steps"]
    t = {n: Tensor(rocm, x[n], dtype, order, gap, offset=offset) for n in ("q", "k", "v", "d_output")}
    o = {n: Tensor(rocm, s, dtype, order, gap, value=7.0, offset=offset) for n, s in (("output", x["d_output"].shape), ("d_q", x["q"].shape), ("d_k", x["k"].shape), ("d_v", x["v"].shape))}
    up = lambda n: rocm.array(x[n]) if x.get(n) is not None else None
    ptr = lambda a: a.ptr if a is not None else None
    state, d_state, reset, lengths = up("state"), up("d_state"), up("reset"), up("lengths")
    shape = (c["rows"], c["heads"], c["dk"], c["dv"])
    final, d_initial = filled(rocm, shape, "float32"), filled(rocm, shape, "float32")
    d_rate = rocm.array(np.full(c["heads"], 7.0 if accumulate_onto is None else accumulate_onto, np.float32))
    w, n = workspace(rocm, layer, steps, 0)
    rocm.call("linear_attention_forward", C.byref(layer), t["q"].view, t["k"].view, t["v"].view, o["output"].view, ptr(state), final.ptr, ptr(reset), ptr(lengths), steps, w.ptr, n)
    w, n = workspace(rocm, layer, steps, 1)
    rocm.call("linear_attention_backward", C.byref(layer), t["q"].view, t["k"].view, t["v"].view, t["d_output"].view, o["d_q"].view, o["d_k"].view, o["d_v"].view, ptr(state), ptr(d_state),
              d_initial.ptr, d_rate.ptr, int(accumulate_onto is not None), ptr(reset), ptr(lengths), steps, w.ptr, n)
    rocm.sync()
    got = {n: a.numpy() for n, a in o.items()}
    for a in o.values():
        assert np.all(a.whole()[..., a.shape[3]:] == 7.0)      # nothing is written between the rows
    return dict(got, state=final.numpy().astype(np.float64), d_state=d_initial.numpy().astype(np.float64), d_log_decay=d_rate.numpy().astype(np.float64))


def check(c, x, got, names=None):
    want, size = reference(c, x), magnitudes(c, x)
    b = bounds(c, want, size)
    for n in names or want:
        off = np.abs(got[n] - want[n]) - b[n]
        assert np.all(off <= 0), (n, float(off.max()), float(np.abs(got[n] - want[n]).max()), float(np.abs(want[n]).max()))


# ------------------------------------------------------------------ the reference itself (no GPU)


def test_the_references_gradients_are_its_differences():
    c, x = case(0, "float32", 7, 3, 4, 2, 3, 5, resets=0.2, ragged=True)
    x = {n: (a.astype(np.float64) if a.dtype.kind == "f" else a) for n, a in x.items()}
    w = np.random.default_rng(1).standard_normal(x["d_output"].shape)
    x["d_output"] = w

    def loss(y):
        r = reference(c, y)
        return (r["output"] * w).sum() + (r["state"] * x["d_state"]).sum()
    got = reference(c, x)
    rng = np.random.default_rng(2)
    for name, grad in (("q", "d_q"), ("k", "d_k"), ("v", "d_v"), ("state", "d_state"), ("log_decay", "d_log_decay")):
        direction = rng.standard_normal(x[name].shape)
        h = 1e-5
        numeric = (loss(dict(x, **{name: x[name] + h * direction})) - loss(dict(x, **{name: x[name] - h * direction}))) / (2 * h)
        assert abs(numeric - (got[grad] * direction).sum()) <= 1e-7 * max(1.0, abs(numeric)), name


# ------------------------------------------------------------------ sequences

SHAPES = [  # steps, rows, heads, kv_heads, dk, dv
    (1, 1, 1, 1, 1, 1), (1, 3, 2, 2, 32, 32), (2, 2, 2, 1, 16, 16), (15, 3, 2, 2, 8, 24), (16, 2, 3, 3, 64, 64), (17, 2, 3, 1, 64, 64), (63, 2, 2, 2, 33, 65), (64, 2, 4, 2, 32, 32),
    (65, 3, 2, 2, 128, 128), (100, 2, 6, 2, 24, 41), (127, 1, 2, 2, 128, 16), (128, 1, 2, 2, 16, 128), (129, 2, 1, 1, 127, 1), (300, 2, 2, 2, 64, 64), (40, 300, 2, 2, 16, 16), (641, 1, 3, 1, 48, 80), (700, 1, 2, 2, 128, 128), (1000, 1, 1, 1, 100, 128)]


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_backward(rocm, shape, dtype):
    print("case", shape, dtype, flush=True)
    c, x = case(sum(shape), dtype, *shape)
    check(c, x, run(rocm, c, x))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [(1, 5, 2, 2, 32, 32), (70, 5, 4, 2, 32, 48), (64, 9, 2, 2, 64, 64), (200, 4, 2, 1, 128, 96), (333, 7, 3, 3, 24, 41), (900, 2, 2, 2, 128, 128)])
@pytest.mark.parametrize("resets", [0.02, 0.3, 1.0])
def test_resets_and_lengths(rocm, shape, dtype, resets):
    print("case", shape, dtype, resets, flush=True)
    c, x = case(sum(shape), dtype, *shape, resets=resets, ragged=True)
    check(c, x, run(rocm, c, x))


@gpu
@pytest.mark.parametrize("order,gap,offset", [((1, 2, 0), 0, 0), ((2, 1, 0), 0, 0), ((1, 0, 2), 8, 0), ((0, 1, 2), 5, 3), ((0, 2, 1), 1, 1)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_orders_gaps_and_alignments(rocm, order, gap, offset, dtype):
    print("case", order, gap, offset, dtype, flush=True)
    c, x = case(7, dtype, 130, 3, 4, 2, 32, 64, resets=0.05, ragged=True)
    check(c, x, run(rocm, c, x, order, gap, offset))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_without_states(rocm, dtype):
    c, x = case(11, dtype, 90, 3, 2, 2, 48, 64, with_state=False)
    check(c, x, run(rocm, c, x))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_decays_from_none_to_all(rocm, dtype):
    """log decays of 0 (nothing fades), of -infinity (a step sees itself alone), and ones whose powers leave the range of fp32 within a chunk"""
    c, x = case(13, dtype, 150, 2, 4, 2, 32, 32, log_decay=[0.0, -3.0, -80.0, -1e-6])
    check(c, x, run(rocm, c, x))
    x["log_decay"] = np.array([-np.inf, 0.0, -np.inf, -0.5], np.float32)
    got = run(rocm, c, x)
    with np.errstate(invalid="ignore"):
        check(c, x, got, ["output", "state", "d_q", "d_k", "d_v", "d_state"])      # (the derivative by a logarithm of zero is left out)


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_what_lies_beyond_a_rows_length_is_not_looked_at(rocm, dtype):
    c, x = case(17, dtype, 150, 6, 2, 2, 32, 64, resets=0.05, ragged=True)
    beyond = np.arange(150)[:, None] >= np.clip(x["lengths"], 0, 150)[None]
    clean = {n: a.copy() for n, a in x.items()}
    for i, n in enumerate(("q", "k", "v", "d_output")):
        x[n][beyond] = (np.nan, np.inf, -np.inf, np.nan)[i]
    got = run(rocm, c, x)
    check(c, clean, got)
    for n in ("output", "d_q", "d_k", "d_v"):
        assert np.all(got[n][beyond] == 0.0)
    assert np.array_equal(got["state"][0], x["state"][0].astype(np.float64))      # the empty row's state, bit for bit
    assert np.array_equal(got["d_state"][0], x["d_state"][0].astype(np.float64))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("steps", [1, 100])
def test_a_reset_forgets_a_state_that_is_not_finite(rocm, dtype, steps):
    c, x = case(19, dtype, steps, 3, 2, 2, 32, 32)
    x["reset"] = np.zeros((steps, 3), np.uint8)
    x["reset"][0] = 1
    clean = {n: a.copy() for n, a in x.items()}
    x["state"][0], x["state"][1], x["state"][2] = np.nan, np.inf, -np.inf
    check(c, clean, run(rocm, c, x))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dk,dv", [(32, 32), (64, 48), (128, 128)])
def test_an_episode_does_not_see_values_of_another_that_are_not_finite(rocm, dtype, dk, dv):
    """row 0: a step of its first episode holds values that are not finite, in the chunk in which the second episode begins (and a third): from there on everything is as if they were"""
    c, x = case(41, dtype, 200, 3, 2, 2, dk, dv)
    x["reset"] = np.zeros((200, 3), np.uint8)
    x["reset"][[75, 90, 140], 0] = 1
    x["reset"][100, 1] = 1
    want, size = reference(c, x), magnitudes(c, x)
    b = bounds(c, want, size)
    for i, n in enumerate(("q", "k", "v", "d_output")):
        x[n][70, 0] = (np.nan, np.inf, np.nan, -np.inf)[i]
    got = run(rocm, c, x)
    for n in ("output", "d_q", "d_k", "d_v"):
        assert np.all(np.abs(got[n][75:] - want[n][75:]) <= b[n][75:]) and np.all(np.abs(got[n][:, 1:] - want[n][:, 1:]) <= b[n][:, 1:]), n
    assert np.all(np.abs(got["state"] - want["state"]) <= b["state"]) and np.all(np.abs(got["d_state"][1:] - want["d_state"][1:]) <= b["d_state"][1:])


@gpu
def test_the_decays_gradient_adds_up_and_runs_repeat_bit_for_bit(rocm):
    c, x = case(23, "float32", 200, 5, 4, 2, 32, 32, resets=0.02, ragged=True)
    first, second, onto = run(rocm, c, x), run(rocm, c, x), run(rocm, c, x, accumulate_onto=3.0)
    for n in first:
        assert np.array_equal(first[n], second[n]), n
    assert np.allclose(onto["d_log_decay"], first["d_log_decay"] + 3.0, rtol=2e-7, atol=0)


@gpu
def test_optional_arguments(rocm):
    """no final state, no gradient of the state or the decay; the initial state's buffer as the final one's"""
    c, x = case(29, "float32", 140, 3, 2, 2, 32, 32, resets=0.05)
    want = run(rocm, c, x)
    layer = layer_of(rocm, c, x)
    t = {n: Tensor(rocm, x[n], "float32") for n in ("q", "k", "v", "d_output")}
    o = {n: Tensor(rocm, s, "float32", value=7.0) for n, s in (("output", x["d_output"].shape), ("d_q", x["q"].shape), ("d_k", x["k"].shape), ("d_v", x["v"].shape))}
    state, d_state, reset = rocm.array(x["state"]), rocm.array(x["d_state"]), rocm.array(x["reset"])
    w, n = workspace(rocm, layer, 140, 0)
    rocm.call("linear_attention_forward", C.byref(layer), t["q"].view, t["k"].view, t["v"].view, o["output"].view, state.ptr, None, reset.ptr, None, 140, w.ptr, n)
    assert np.array_equal(o["output"].numpy(), want["output"])
    w2, n2 = workspace(rocm, layer, 140, 1)
    rocm.call("linear_attention_backward", C.byref(layer), t["q"].view, t["k"].view, t["v"].view, t["d_output"].view, o["d_q"].view, o["d_k"].view, o["d_v"].view, state.ptr, d_state.ptr, None, None, 0,
              reset.ptr, None, 140, w2.ptr, n2)
    for name in ("d_q", "d_k", "d_v"):
        assert np.allclose(o[name].numpy(), want[name], rtol=1e-5, atol=1e-5), name
    rocm.call("linear_attention_forward", C.byref(layer), t["q"].view, t["k"].view, t["v"].view, o["output"].view, state.ptr, state.ptr, reset.ptr, None, 140, w.ptr, n)
    assert np.array_equal(o["output"].numpy(), want["output"]) and np.array_equal(state.numpy(), want["state"].astype(np.float32))


# ------------------------------------------------------------------ single steps


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,heads,kv_heads,dk,dv", [(1, 1, 1, 1, 1), (64, 2, 2, 32, 32), (3, 6, 2, 24, 41), (5, 4, 4, 64, 64), (2, 3, 1, 128, 128), (7, 2, 2, 128, 20), (2, 2, 2, 7, 128), (300, 8, 8, 16, 16),
                                                       (3, 2, 2, 128, 101), (5, 3, 1, 5, 64), (2, 3, 3, 100, 1), (3, 2, 1, 8, 101), (1, 5, 5, 8, 100), (9, 1, 1, 17, 3)])
@pytest.mark.parametrize("in_place", [False, True])
def test_steps_walk_a_sequence(rocm, rows, heads, kv_heads, dk, dv, dtype, in_place):
    """five steps one by one against the recurrence, states that a reset drops included; a state that is not finite is dropped too"""
    print("case", rows, heads, kv_heads, dk, dv, dtype, in_place, flush=True)
    c, x = case(rows + dk, dtype, 5, rows, heads, kv_heads, dk, dv, resets=0.3)
    x["reset"][0, 0] = 1
    clean = {n: a.copy() for n, a in x.items()}
    x["state"][0] = np.nan
    want, size = reference(c, clean), magnitudes(c, clean)
    b, layer = bounds(c, want, size), layer_of(rocm, c, x)
    state, other = rocm.array(x["state"]), filled(rocm, x["state"].shape, "float32")
    reset = rocm.array(x["reset"])
    q, k, v = (Tensor(rocm, x[n], dtype) for n in ("q", "k", "v"))
    out = Tensor(rocm, x["d_output"].shape, dtype, value=7.0)
    item = 4 if dtype == "float32" else 2
    for t in range(5):
        one = [view(a.array, strides_of(a.padded, a.order), item, t * int(np.prod(a.padded[1:]))) for a in (q, k, v, out)]
        to = state if in_place else other
        rocm.call("linear_attention_step", C.byref(layer), *one, state.ptr, to.ptr, reset.ptr + t * rows)
        if not in_place:
            state, other = other, state
    rocm.sync()
    assert np.all(np.abs(out.numpy() - want["output"]) <= b["output"]) and np.all(np.abs(state.numpy() - want["state"]) <= b["state"])


# ------------------------------------------------------------------ graphs, streams, refusals


@gpu
def test_a_graph_replays_forward_and_backward(rocm):
    lib, h = rocm.device.lib, rocm.device.handle
    c, x = case(31, "bfloat16", 200, 3, 4, 2, 64, 64, resets=0.02, ragged=True)
    want = run(rocm, c, x)
    layer = layer_of(rocm, c, x)
    t = {n: Tensor(rocm, x[n], "bfloat16") for n in ("q", "k", "v", "d_output")}
    o = {n: Tensor(rocm, s, "bfloat16", value=7.0) for n, s in (("output", x["d_output"].shape), ("d_q", x["q"].shape), ("d_k", x["k"].shape), ("d_v", x["v"].shape))}
    state, d_state, reset, lengths = (rocm.array(x[n]) for n in ("state", "d_state", "reset", "lengths"))
    final, d_initial, d_rate = rocm.zeros(x["state"].shape), rocm.zeros(x["state"].shape), rocm.zeros((4,))
    w, n = workspace(rocm, layer, 200, 0)
    w2, n2 = workspace(rocm, layer, 200, 1)
    rocm.sync()
    assert lib.rlt_rocm_graph_begin_capture(h) == 0
    rocm.call("linear_attention_forward", C.byref(layer), t["q"].view, t["k"].view, t["v"].view, o["output"].view, state.ptr, final.ptr, reset.ptr, lengths.ptr, 200, w.ptr, n)
    rocm.call("linear_attention_backward", C.byref(layer), t["q"].view, t["k"].view, t["v"].view, t["d_output"].view, o["d_q"].view, o["d_k"].view, o["d_v"].view, state.ptr, d_state.ptr, d_initial.ptr,
              d_rate.ptr, 0, reset.ptr, lengths.ptr, 200, w2.ptr, n2)
    graph = C.c_void_p()
    assert lib.rlt_rocm_graph_end_capture(h, C.byref(graph)) == 0
    for _ in range(3):
        for a in o.values():
            a.array.upload(to_bits(np.full(a.array.shape, 7.0, np.float32)))      # eager work between the replays
        assert lib.rlt_rocm_graph_launch(h, graph) == 0
        rocm.sync()
        for name, a in o.items():
            assert np.array_equal(a.numpy(), want[name]), name
        assert np.array_equal(final.numpy(), want["state"].astype(np.float32)) and np.array_equal(d_rate.numpy(), want["d_log_decay"].astype(np.float32))
    lib.rlt_rocm_graph_destroy(h, graph)


@gpu
def test_refusals(rocm):
    lib, h = rocm.device.lib, rocm.device.handle
    c, x = case(37, "float32", 4, 2, 4, 2, 8, 8)
    t = {n: Tensor(rocm, x[n], "float32") for n in ("q", "k", "v")}
    out = Tensor(rocm, x["d_output"].shape, "float32", value=7.0)
    none = C.byref(capi.HeadView(None, 1, 1, 1))
    state = rocm.array(x["state"])
    good = layer_of(rocm, c, x)

    def forward(layer=good, q=t["q"].view, steps=4):
        w, n = workspace(rocm, good, 4, 0)
        return lib.rlt_rocm_linear_attention_forward(h, C.byref(layer) if layer is not None else None, q, t["k"].view, t["v"].view, out.view, None, None, None, None, steps, w.ptr, n)

    def changed(**fields):
        layer = layer_of(rocm, c, x)
        for name, value in fields.items():
            setattr(layer, name, value)
        return layer
    assert forward() == 0
    for layer in (None, changed(type=2), changed(type=-1), changed(batch=0), changed(heads=0), changed(kv_heads=0), changed(kv_heads=3), changed(key_dim=0), changed(value_dim=-1), changed(log_decay=None)):
        assert forward(layer) == capi.RLT_E_INVALID_ARGUMENT
    assert forward(q=none) == forward(q=None) == forward(steps=0) == capi.RLT_E_INVALID_ARGUMENT
    assert forward(changed(key_dim=129)) == forward(changed(value_dim=129)) == capi.RLT_E_UNSUPPORTED
    assert lib.rlt_rocm_linear_attention_forward(None, C.byref(good), t["q"].view, t["k"].view, t["v"].view, out.view, None, None, None, None, 4, None, 0) == capi.RLT_E_NOT_INITIALISED
    w, n = workspace(rocm, good, 4, 1)
    assert n > 0
    views = [t["q"].view, t["k"].view, t["v"].view, out.view, out.view, out.view, out.view]
    for ptr, size in ((None, n), (w.ptr, n - 1)):
        assert lib.rlt_rocm_linear_attention_backward(h, C.byref(good), *views, None, None, None, None, 0, None, None, 4, ptr, size) == capi.RLT_E_INVALID_ARGUMENT
    for i in range(7):
        assert lib.rlt_rocm_linear_attention_backward(h, C.byref(good), *(views[:i] + [none] + views[i + 1:]), None, None, None, None, 0, None, None, 4, w.ptr, n) == capi.RLT_E_INVALID_ARGUMENT
    assert lib.rlt_rocm_linear_attention_step(h, C.byref(good), t["q"].view, t["k"].view, t["v"].view, out.view, None, state.ptr, None) == capi.RLT_E_INVALID_ARGUMENT
    assert lib.rlt_rocm_linear_attention_step(h, C.byref(good), t["q"].view, t["k"].view, t["v"].view, out.view, state.ptr, None, None) == capi.RLT_E_INVALID_ARGUMENT
    assert lib.rlt_rocm_linear_attention_workspace_bytes(None, 4, 1) == lib.rlt_rocm_linear_attention_workspace_bytes(C.byref(good), 0, 1) == 0
    rocm.sync()


@gpu
def test_longer_sequences_than_an_index_holds_are_refused(rocm):
    c, x = case(2, "float32", 4, 2, 2, 2, 8, 8)
    layer, t = layer_of(rocm, c, x), {n: Tensor(rocm, x[n], "float32") for n in ("q", "k", "v", "d_output")}
    lib, h = rocm.device.lib, rocm.device.handle
    w = rocm.zeros((1024,))
    views = [t[n].view for n in ("q", "k", "v", "d_output")]
    for steps in (2 ** 30 + 1, 2 ** 31 - 1):
        assert lib.rlt_rocm_linear_attention_workspace_bytes(C.byref(layer), steps, 0) == lib.rlt_rocm_linear_attention_workspace_bytes(C.byref(layer), steps, 1) == 0
        assert lib.rlt_rocm_linear_attention_forward(h, C.byref(layer), *views, None, None, None, None, steps, w.ptr, 4096) == capi.RLT_E_UNSUPPORTED
        assert lib.rlt_rocm_linear_attention_backward(h, C.byref(layer), *views, *views[:3], None, None, None, None, 0, None, None, steps, w.ptr, 4096) == capi.RLT_E_UNSUPPORTED

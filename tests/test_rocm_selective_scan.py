"""The selective scan, forward, backward and single steps, against the recurrence in 64 bits.

Bounds, set before the first run; u = 2^-24. Every output is a sum of products; with the inputs, the gate's factors and the rates of the sums (not those of the exponents) replaced by their absolute values the reference gives the sum of the
products' magnitudes, M. A product holds up to `steps` decays, exp(-rate delta): its argument is off by at most 16 u of itself (delta: an exponential with a first-order correction, a reciprocal, a polynomial, sums: eight; the rate: an
exponential and its factor: four; the product and the power's own), the power itself by 2 u, and h's sum rounds once a step. With E the largest sum of rate * delta over a row's steps that is: (4 steps + 16 E) u, and the other factors (delta, the gate's
sigmoid and its slope, delta's slope: at most 12 u each, of which a product has at most four), the sums over states and channels add (64 + channels + states) u. Sums over steps and rows round once more for each: (steps + rows) u.
bfloat16 adds the output's own rounding, 2^-8 of the value."""
import ctypes as C

import numpy as np
import pytest

from helpers import capi, package
from test_rocm_linear_attention import Tensor, strides_of, view
from typed_arrays import UNIT, download, filled, rounded, to_bits, upload

gpu = pytest.mark.gpu
U = 2.0 ** -24
SEQUENCES = ("x", "delta", "b", "c", "gate", "d_output")
PARAMETERS = ("log_rates", "skip", "delta_biases")


def sigmoid(z):
    e = np.exp(-np.abs(z))
    return np.where(z >= 0, 1 / (1 + e), e / (1 + e))


def factors(x):
    """what the exponentials and the gate make of the inputs: delta and its slope, the gate's factor and its slope, the rates"""
    raw = x["delta"] + (x["delta_biases"].astype(np.float64) if x.get("delta_biases") is not None else 0.0)
    f = dict(delta=np.logaddexp(raw, 0.0), slope=sigmoid(raw), rates=np.exp(x["log_rates"].astype(np.float64)), factor=np.ones_like(raw), d_factor=np.zeros_like(raw))
    if x.get("gate") is not None:
        z = x["gate"]
        f.update(factor=z * sigmoid(z), d_factor=sigmoid(z) * (1 + z * sigmoid(-z)))
    return f


def reference(c, x, f=None, sign=-1.0):
    """All outputs by the recurrence in 64 bits. sign: of the rates in the sums (+1 for magnitudes)."""
    f = factors(x) if f is None else f
    steps, rows = c["steps"], c["rows"]
    shape = (rows, c["heads"], c["channels"], c["states"])
    rates, skip = f["rates"], x["skip"].astype(np.float64) if x.get("skip") is not None else np.zeros((c["heads"], c["channels"]))
    lengths = np.clip(x["lengths"], 0, steps) if x.get("lengths") is not None else np.full(rows, steps)
    h = np.zeros(shape) if x.get("state") is None else x["state"].astype(np.float64)
    d = {n: np.zeros(s) for n, s in (("x", x["x"].shape), ("delta", x["x"].shape), ("gate", x["x"].shape), ("b", x["b"].shape), ("c", x["b"].shape), ("log_rates", rates.shape), ("skip", skip.shape), ("delta_biases", skip.shape))}
    out, entries = np.zeros_like(x["x"]), []
    flags = lambda t: ((t < lengths)[:, None, None, None], (x["reset"][t] != 0)[:, None, None, None] if x.get("reset") is not None else np.zeros((rows, 1, 1, 1), bool))
    with np.errstate(invalid="ignore"):
        for t in range(steps):
            live, begins = flags(t)
            entries.append(np.where(begins, 0.0, h))
            after = np.exp(-rates * f["delta"][t][..., None]) * entries[-1] + (f["delta"][t] * x["x"][t])[..., None] * x["b"][t][:, :, None]
            out[t] = np.where(live[..., 0], ((x["c"][t][:, :, None] * after).sum(-1) + skip * x["x"][t]) * f["factor"][t], 0.0)
            h = np.where(live, after, h)
        grad = np.zeros(shape) if x.get("d_state") is None else x["d_state"].astype(np.float64)
        for t in reversed(range(steps)):
            live, begins = flags(t)
            decay, u = np.exp(-rates * f["delta"][t][..., None]), f["delta"][t] * x["x"][t]
            after = np.where(live, decay * entries[t] + u[..., None] * x["b"][t][:, :, None], 0.0)
            up = np.where(live[..., 0], x["d_output"][t], 0.0)
            on = lambda a: np.where(live[..., 0], a, 0.0)
            read, added, x_t = np.where(live, x["c"][t][:, :, None], 0.0), np.where(live, x["b"][t][:, :, None], 0.0), on(x["x"][t])
            d["gate"][t] = on(up * ((read * after).sum(-1) + skip * x_t) * f["d_factor"][t])
            g = on(up * f["factor"][t])
            d["skip"] += (g * x_t).sum(0)
            d["c"][t] = (g[..., None] * after).sum(2)
            here = np.where(live, grad + g[..., None] * read, 0.0)
            d["b"][t] = np.where(live, here * u[..., None], 0.0).sum(2)
            through = (here * added).sum(-1)
            d["x"][t] = on(through * f["delta"][t]) + skip * g
            q = np.where(live, here * decay * entries[t], 0.0)
            d["log_rates"] += sign * np.where(live, q * f["delta"][t][..., None] * rates, 0.0).sum(0)
            d["delta"][t] = on((through * x_t + sign * (q * rates).sum(-1)) * f["slope"][t])
            d["delta_biases"] += d["delta"][t].sum(0)
            grad = np.where(live, np.where(begins, 0.0, decay * here), grad)
    return dict({"d_" + n: a for n, a in d.items()}, output=out, state=h, d_state=grad)


def case(seed, dtype, steps, rows, heads, channels, states, resets=0.0, ragged=False, with_state=True, gate=True, parameters=True, size=0.3):
    rng = np.random.default_rng(seed)
    n = lambda *shape: rounded(rng.standard_normal(shape), dtype)
    wide, narrow = (steps, rows, heads, channels), (steps, rows, heads, states)
    x = dict(x=n(*wide), delta=n(*wide), b=n(*narrow), c=n(*narrow), d_output=n(*wide), log_rates=(np.log(np.arange(1, states + 1)) + 0.1 * rng.standard_normal((heads, channels, states))).astype(np.float32))
    if gate:
        x["gate"] = n(*wide)
    if parameters:
        x["skip"], x["delta_biases"] = rng.standard_normal((heads, channels)).astype(np.float32), (np.log(size) + rng.uniform(-2, 0, (heads, channels))).astype(np.float32)
    if with_state:
        x["state"], x["d_state"] = (rng.standard_normal((rows, heads, channels, states)).astype(np.float32) for _ in range(2))
    if resets:
        x["reset"] = (rng.random((steps, rows)) < resets).astype(np.uint8)
    if ragged:
        x["lengths"] = rng.integers(0, steps + 1, rows).astype(np.int32)
        x["lengths"][0], x["lengths"][-1] = 0, steps + 5      # an empty row; one that claims more than there is
    return dict(dtype=dtype, steps=steps, rows=rows, heads=heads, channels=channels, states=states), x


def magnitudes(c, x, f):
    """The gate's slope, s (1 + z (1 - s)) with s = sigmoid(z), is a sum whose terms cancel near z = -1.28: what its roundings are relative to is s (1 + |z| (1 - s)) there, not the slope itself."""
    sizes = {n: np.abs(a) for n, a in f.items()}
    if x.get("gate") is not None:
        sizes["d_factor"] = sigmoid(x["gate"]) * (1 + np.abs(x["gate"]) * sigmoid(-x["gate"]))
    return reference(c, {n: (a if n in ("reset", "lengths") else np.abs(a)) for n, a in x.items()}, sizes, 1.0)


def bounds(c, x, want):
    f = factors(x)
    size = magnitudes(c, x, f)
    E = (f["rates"] * f["delta"][..., None]).sum(0).max()
    unit = (4 * c["steps"] + 16 * E + 64 + c["channels"] + c["states"]) * U
    b = {n: unit * m for n, m in size.items()}
    for n in PARAMETERS:
        b["d_" + n] = b["d_" + n] + (c["steps"] + c["rows"]) * U * size["d_" + n]
    if c["dtype"] == "bfloat16":
        for n in ("output", "d_x", "d_delta", "d_b", "d_c", "d_gate"):
            b[n] = b[n] + UNIT["bfloat16"] * (np.abs(want[n]) + b[n])
    return b


def check(c, x, got, names=None, underflow=0.0):
    want = reference(c, x)
    b = bounds(c, x, want)
    for n in names or got:
        off = np.abs(got[n] - want[n]) - b[n] - underflow
        assert np.all(off <= 0), (n, float(off.max()), float(np.abs(got[n] - want[n]).max()), float(np.abs(want[n]).max()))


def layer_of(rocm, c, x, keep, onto=7.0, gradients=True):
    for n in PARAMETERS:
        keep[n] = rocm.array(x[n]) if x.get(n) is not None else None
        keep["d_" + n] = rocm.array(np.full((c["heads"], c["channels"]) + ((c["states"],) if n == "log_rates" else ()), onto, np.float32))
    ptr = lambda a: a.ptr if a is not None else None
    return capi.SelectiveScan(*[ptr(keep[n]) for n in PARAMETERS], *[keep["d_" + n].ptr if gradients else None for n in PARAMETERS], capi.TYPE[c["dtype"]], c["rows"], c["heads"], c["channels"], c["states"], 0)


class Buffers:
    """a case's tensors, states and scratch memory on the device"""

    def __init__(self, rocm, c, x, order=(0, 1, 2), gap=0, offset=0, onto=None):
        self.rocm, self.c, self.x, self.keep, self.onto = rocm, c, x, {}, onto
        self.layer = layer_of(rocm, c, x, self.keep, 7.0 if onto is None else onto)
        dtype, steps = c["dtype"], c["steps"]
        self.t = {n: Tensor(rocm, x[n], dtype, order, gap, offset=offset) for n in SEQUENCES if x.get(n) is not None}
        shapes = {"output": "x", "d_x": "x", "d_delta": "x", "d_b": "b", "d_c": "c", "d_gate": "gate"}
        self.o = {n: Tensor(rocm, x[like].shape, dtype, order, gap, value=7.0, offset=offset) for n, like in shapes.items() if x.get(like) is not None}
        up = lambda n: rocm.array(x[n]) if x.get(n) is not None else None
        self.state, self.d_state, self.reset, self.lengths = up("state"), up("d_state"), up("reset"), up("lengths")
        shape = (c["rows"], c["heads"], c["channels"], c["states"])
        self.final, self.d_initial = filled(rocm, shape, "float32"), filled(rocm, shape, "float32")
        lib, layer = rocm.device.lib, C.byref(self.layer)
        bytes_of = lambda n: rocm.device.empty((max(int(n), 16),), np.uint8)
        self.sizes = [lib.rlt_rocm_selective_scan_workspace_bytes(layer, steps, k) for k in (0, 1)]
        self.scratch = [bytes_of(n) for n in self.sizes]
        self.checkpoints = bytes_of(lib.rlt_rocm_selective_scan_checkpoint_bytes(layer, steps))

    def inputs(self):
        return [self.t[n].view if n in self.t else None for n in SEQUENCES[:5]]

    def tail(self, backward):
        ptr = lambda a: a.ptr if a is not None else None
        return ptr(self.reset), ptr(self.lengths), self.c["steps"], self.checkpoints.ptr, self.scratch[backward].ptr, self.sizes[backward]

    def forward(self):
        ptr = lambda a: a.ptr if a is not None else None
        self.rocm.call("selective_scan_forward", C.byref(self.layer), *self.inputs(), self.o["output"].view, ptr(self.state), self.final.ptr, *self.tail(0))

    def backward(self):
        ptr = lambda a: a.ptr if a is not None else None
        outs = [self.o[n].view if n in self.o else None for n in ("d_x", "d_delta", "d_b", "d_c", "d_gate")]
        self.rocm.call("selective_scan_backward", C.byref(self.layer), *self.inputs(), self.t["d_output"].view, *outs, ptr(self.d_state), self.d_initial.ptr, int(self.onto is not None), *self.tail(1))

    def results(self):
        f = lambda a: a.numpy().astype(np.float64)
        for a in self.o.values():
            assert np.all(a.whole()[..., a.shape[3]:] == 7.0)      # nothing is written between the rows
        return dict({n: a.numpy() for n, a in self.o.items()}, state=f(self.final), d_state=f(self.d_initial), **{"d_" + n: f(self.keep["d_" + n]) for n in PARAMETERS})


def run(rocm, c, x, **layout):
    b = Buffers(rocm, c, x, **layout)
    b.forward()
    b.backward()
    rocm.sync()
    return b.results()


# ------------------------------------------------------------------ the reference itself (no GPU)


def test_the_references_gradients_are_its_differences():
    c, x = case(0, "float32", 7, 3, 2, 3, 4, resets=0.2, ragged=True)
    x = {n: (a.astype(np.float64) if a.dtype.kind == "f" else a) for n, a in x.items()}

    def loss(y):
        r = reference(c, y)
        return (r["output"] * x["d_output"]).sum() + (r["state"] * x["d_state"]).sum()
    got, rng = reference(c, x), np.random.default_rng(2)
    for name in ("x", "delta", "b", "c", "gate", "state", "log_rates", "skip", "delta_biases"):
        direction, h = rng.standard_normal(x[name].shape), 1e-5
        numeric = (loss(dict(x, **{name: x[name] + h * direction})) - loss(dict(x, **{name: x[name] - h * direction}))) / (2 * h)
        assert abs(numeric - (got["d_" + name] * direction).sum()) <= 1e-7 * max(1.0, abs(numeric)), name


# ------------------------------------------------------------------ sequences

SHAPES = [  # steps, rows, heads, channels, states
    (1, 1, 1, 1, 1), (1, 3, 2, 16, 16), (2, 2, 1, 17, 4), (15, 3, 1, 64, 16), (16, 2, 2, 65, 16), (17, 2, 1, 63, 15), (31, 2, 1, 48, 8), (33, 3, 2, 24, 32), (64, 2, 1, 130, 16), (65, 1, 3, 40, 31), (100, 2, 1, 33, 9),
    (129, 1, 1, 16, 25), (300, 2, 1, 20, 16), (700, 1, 2, 16, 5), (900, 1, 1, 12, 20), (20, 300, 1, 8, 16), (3, 60, 40, 8, 4)]


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_backward(rocm, shape, dtype):
    print("case", shape, dtype, flush=True)
    c, x = case(sum(shape), dtype, *shape)
    check(c, x, run(rocm, c, x))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [(1, 5, 2, 16, 16), (40, 6, 1, 70, 16), (64, 9, 2, 16, 8), (200, 4, 1, 33, 32), (333, 5, 1, 24, 11), (600, 2, 1, 16, 16)])
@pytest.mark.parametrize("resets", [0.02, 0.3, 1.0])
def test_resets_and_lengths(rocm, shape, dtype, resets):
    print("case", shape, dtype, resets, flush=True)
    c, x = case(sum(shape), dtype, *shape, resets=resets, ragged=True)
    check(c, x, run(rocm, c, x))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [(1, 700, 1, 4, 16), (17, 330, 2, 7, 16), (70, 650, 1, 3, 9), (150, 340, 1, 5, 16), (40, 330, 1, 8, 25), (70, 330, 2, 4, 32)])
@pytest.mark.parametrize("resets", [0.0, 0.1])
def test_many_rows(rocm, shape, dtype, resets):
    """more channels and rows than segments are made for"""
    print("case", shape, dtype, resets, flush=True)
    c, x = case(sum(shape), dtype, *shape, resets=resets, ragged=resets > 0)
    if resets:      # what lies beyond a row's length is not looked at
        beyond = np.arange(shape[0])[:, None] >= np.clip(x["lengths"], 0, shape[0])[None]
        clean = {n: a.copy() for n, a in x.items()}
        for i, n in enumerate(SEQUENCES):
            x[n][beyond] = (np.nan, np.inf, -np.inf, np.nan, np.inf, -np.inf)[i]
        check(c, clean, run(rocm, c, x))
    else:
        check(c, x, run(rocm, c, x))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("states", [16, 20])
def test_many_rows_in_another_order_and_episodes_that_are_not_finite(rocm, dtype, states):
    c, x = case(43, dtype, 90, 330, 2, 4, states)
    check(c, x, run(rocm, c, x, order=(2, 1, 0), gap=3, offset=1))
    x["reset"] = np.zeros((90, 330), np.uint8)
    x["reset"][40, 0] = x["reset"][40, 2] = 1
    want = reference(c, x)
    b = bounds(c, x, want)
    for i, n in enumerate(SEQUENCES):
        x[n][38, 0] = (np.nan, np.inf, np.nan, -np.inf, np.nan, np.inf)[i]
        x[n][45, 2] = (np.nan, np.inf, np.nan, -np.inf, np.nan, np.inf)[i]
    got = run(rocm, c, x)
    for n in ("output", "d_x", "d_delta", "d_b", "d_c", "d_gate"):
        off = np.abs(got[n] - want[n]) <= b[n]
        assert np.all(off[40:, 0]) and np.all(off[:, 1]) and np.all(off[:40, 2]) and np.all(off[:, 3:]), n


SHORT = [(5, 300, 8, 65, 16), (8, 150, 16, 130, 16), (7, 130, 16, 64, 27), (6, 400, 8, 20, 8), (1, 600, 8, 40, 8), (1, 700, 4, 130, 16), (2, 300, 8, 65, 16), (3, 150, 16, 130, 16), (4, 120, 8, 300, 32), (4, 500, 16, 9, 5), (3, 330, 16, 64, 27), (2, 3, 1, 1, 1)]


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape,kind", [(s, dict(resets=0.3, ragged=True)) for s in SHORT] + [(s, dict()) for s in SHORT[::3]] + [(s, k) for s in SHORT[:2] + SHORT[-2:] for k in (dict(gate=False, with_state=False), dict(parameters=False, ragged=True))])
def test_few_steps_of_many_rows(rocm, shape, dtype, kind):
    """rows that a workgroup goes through one after the other, some of them empty; what lies beyond a row's length is not looked at"""
    print("case", shape, dtype, kind, flush=True)
    c, x = case(sum(shape), dtype, *shape, **kind)
    clean = {n: a.copy() for n, a in x.items()}
    if kind.get("ragged"):
        beyond = np.arange(shape[0])[:, None] >= np.clip(x["lengths"], 0, shape[0])[None]
        for i, n in enumerate(SEQUENCES):
            if n in x:
                x[n][beyond] = (np.nan, np.inf, -np.inf, np.nan, np.inf, -np.inf)[i]
    first, second = run(rocm, c, x), run(rocm, c, x)
    # Relative bounds end where fp32 does: states of rates up to 32 and deltas of three pass on e^-96 of a gradient a step, below 2^-126, where an operation's result may be zero instead, off by 2^-126 at most. On its way to an output such an error meets
    # decays, which are at most one, at most two of the inputs (m is the largest) and a rate, and as many of its kind as there are operations: eight for each step and state or channel of the sum.
    m, rate = max(np.abs(a).max() for n, a in clean.items() if n not in ("reset", "lengths", "log_rates")), np.exp(clean["log_rates"].max())
    check(c, clean, first, underflow=2.0 ** -126 * 8 * shape[0] * (shape[1] + shape[3] + shape[4]) * (1 + m) ** 2 * (1 + rate))
    assert all(np.array_equal(a, second[n]) for n, a in first.items())


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("steps", [1, 3, 4, 6, 8])
def test_few_steps_in_other_orders_and_states_that_a_reset_forgets(rocm, dtype, steps):
    c, x = case(47 + steps, dtype, steps, 300, 8, 24, 16, resets=0.1)
    check(c, x, run(rocm, c, x, order=(2, 1, 0), gap=3, offset=1))
    x["reset"][0, 5] = 1
    clean = run(rocm, c, x)
    x["state"][5] = np.inf
    got = run(rocm, c, x)
    assert all(np.array_equal(got[n], clean[n]) for n in got)


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [(3, 40, 1, 70, 16), (20, 5, 2, 70, 16), (300, 3, 1, 20, 12), (700, 1, 1, 70, 20)])
def test_rates_that_leave_the_range(rocm, shape, dtype):
    """a state that forgets all at every step that is there, and nothing at those that are not: exp(100) is infinite in 32 bits"""
    c, x = case(51, dtype, *shape, ragged=True)
    if shape[1] == 1:
        x["lengths"][:] = shape[0] - 9
    x["log_rates"][:, ::2, 1] = 100.0
    got, want, f = run(rocm, c, x), reference(c, x), factors(x)
    size = magnitudes(c, x, f)
    E = np.where(f["rates"] < 1e30, f["rates"] * f["delta"][..., None], 0.0).sum(0).max()
    unit = (4 * c["steps"] + 16 * E + 64 + c["channels"] + c["states"] + c["steps"] + c["rows"]) * U
    for n in got:
        limit = unit * size[n]
        if dtype == "bfloat16" and n in ("output", "d_x", "d_delta", "d_b", "d_c", "d_gate"):
            limit = limit + UNIT["bfloat16"] * (np.abs(want[n]) + limit)
        assert np.isfinite(got[n]).all() and np.all(np.abs(got[n] - want[n]) <= limit), n


ENDS = [(21, 12, 1, 20, 8), (21, 12, 2, 70, 16), (45, 12, 1, 16, 16), (22, 12, 1, 20, 20), (30, 12, 1, 70, 27), (700, 2, 1, 20, 16), (900, 2, 1, 70, 12), (6, 12, 2, 70, 16), (3, 12, 1, 20, 25)]


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", ENDS)
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_rows_that_end_in_a_state_or_a_gradient_that_is_not_finite(rocm, shape, dtype, bad):
    """steps behind a row's last are exact zeros then too, and so is what they add to the parameters' gradients"""
    print("case", shape, dtype, bad, flush=True)
    steps, rows = shape[:2]
    c, x = case(61 + sum(shape), dtype, *shape)
    x["lengths"] = np.maximum(steps - 1 - np.arange(rows) % 11, 1).astype(np.int32)
    beyond = np.arange(steps)[:, None] >= x["lengths"][None]
    # a state that is not finite from a row's last step on, by an input of that step: what it gives the rates is finite, as the state before it is
    clean = {n: a for n, a in x.items() if n != "d_state"}
    by_input = dict(clean, b=x["b"].copy())
    for r in range(rows):
        by_input["b"][x["lengths"][r] - 1, r, 0, 0] = bad
    want = reference(c, clean)
    limit = bounds(c, clean, want)
    got = run(rocm, c, by_input)
    for n in ("output", "d_x", "d_delta", "d_b", "d_c", "d_gate"):
        assert np.all(got[n][beyond] == 0.0), n
    for n in ("d_log_rates", "d_skip"):
        assert np.all(np.abs(got[n] - want[n]) <= limit[n]), n
    # the gradient of the state behind the last step is not finite
    by_gradient = dict(x, d_state=x["d_state"].copy())
    by_gradient["d_state"][:, 0, 0, 0] = bad
    got = run(rocm, c, by_gradient)
    for n in ("output", "d_x", "d_delta", "d_b", "d_c", "d_gate"):
        assert np.all(got[n][beyond] == 0.0), n
    # channels whose states are finite keep their outputs and gradients
    want = reference(c, x)
    limit = bounds(c, x, want)
    for n in ("output", "d_gate", "d_c"):      # (that need no gradient of the state)
        assert np.all(np.abs(got[n] - want[n]) <= limit[n]), n
    for n in ("d_x", "d_delta", "d_log_rates", "d_skip", "d_delta_biases"):
        others = np.ones(want[n].shape, bool)
        others[(Ellipsis, slice(0, 1), slice(0, 1), slice(None)) if n == "d_log_rates" else (Ellipsis, slice(0, 1), slice(0, 1))] = False
        assert np.all(np.abs(got[n] - want[n])[others] <= limit[n][others]), n


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", ENDS)
def test_an_infinite_state_of_the_last_channel_is_infinite_in_the_sums_over_channels(rocm, shape, dtype):
    """and no number where it is summed up with what lanes beyond the channels have"""
    print("case", shape, dtype, flush=True)
    c, x = case(63 + sum(shape), dtype, *shape)
    x["log_rates"][:], x["delta"][:] = np.log(0.1), rounded(np.full(x["delta"].shape, -2.0), dtype)      # nothing is forgotten that counts: infinite states stay so
    x["state"][:, :, -1, 0] = np.inf
    got, want = run(rocm, c, x), reference(c, x)
    assert np.isinf(want["d_c"][..., 0]).all() and np.array_equal(got["d_c"][..., 0], want["d_c"][..., 0])
    x["state"][:, :, -1, 0] = 1.0
    x["d_state"][:, :, -1, 0] = np.inf
    got, want = run(rocm, c, x), reference(c, x)
    assert np.isinf(want["d_b"][..., 0]).all() and np.array_equal(got["d_b"][..., 0], want["d_b"][..., 0])


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", ENDS)
def test_rates_that_leave_the_range_with_large_states_and_gradients(rocm, shape, dtype):
    """states and gradients of 1e5, whose product times the largest rate, 1e30, is beyond fp32: steps that are not there give nothing all the same"""
    print("case", shape, dtype, flush=True)
    c, x = case(67 + sum(shape), dtype, *shape)
    x["lengths"] = np.maximum(c["steps"] - 1 - np.arange(c["rows"]) % 11, 1).astype(np.int32)
    x["log_rates"][:, ::2, 1] = 100.0
    x["b"], x["d_state"] = rounded(1e5 * x["b"], dtype), 1e5 * x["d_state"]
    got, want, f = run(rocm, c, x), reference(c, x), factors(x)
    size = magnitudes(c, x, f)
    E = np.where(f["rates"] < 1e30, f["rates"] * f["delta"][..., None], 0.0).sum(0).max()
    unit = (4 * c["steps"] + 16 * E + 64 + c["channels"] + c["states"] + c["steps"] + c["rows"]) * U
    for n in got:
        limit = unit * size[n]
        if dtype == "bfloat16" and n in ("output", "d_x", "d_delta", "d_b", "d_c", "d_gate"):
            limit = limit + UNIT["bfloat16"] * (np.abs(want[n]) + limit)
        assert np.isfinite(got[n]).all() and np.all(np.abs(got[n] - want[n]) <= limit), n


@gpu
@pytest.mark.parametrize("order,gap,offset", [((1, 2, 0), 0, 0), ((2, 1, 0), 0, 0), ((1, 0, 2), 8, 0), ((0, 1, 2), 5, 3), ((0, 2, 1), 1, 1)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_orders_gaps_and_alignments(rocm, order, gap, offset, dtype):
    print("case", order, gap, offset, dtype, flush=True)
    c, x = case(7, dtype, 130, 3, 2, 80, 16, resets=0.05, ragged=True)
    check(c, x, run(rocm, c, x, order=order, gap=gap, offset=offset))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_sequence_backwards_in_memory(rocm, dtype):
    c, x = case(8, dtype, 150, 2, 1, 32, 16, ragged=True)
    b = Buffers(rocm, c, x)
    item, back = 4 if dtype == "float32" else 2, {}
    for n, a in list(b.t.items()) + list(b.o.items()):
        width = 2 * a.shape[3]
        if n in b.t:
            a.array.upload(x[n][::-1].astype(np.float32) if dtype == "float32" else to_bits(x[n][::-1].astype(np.float32)))
        a.view = view(a.array, (-width, a.shape[3], a.shape[3]), item, 149 * width)
    b.forward()
    b.backward()
    rocm.sync()
    got = b.results()
    check(c, x, {n: (a[::-1] if n in b.o else a) for n, a in got.items()})


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_without_states_gate_or_parameters(rocm, dtype):
    for kinds in (dict(with_state=False), dict(gate=False), dict(parameters=False), dict(with_state=False, gate=False, parameters=False)):
        c, x = case(11, dtype, 90, 3, 2, 48, 16, **kinds)
        got = run(rocm, c, x)
        check(c, x, got)


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_steps_from_tiny_to_huge_and_rates_from_none_to_all(rocm, dtype):
    """deltas whose exponentials leave the range of fp32 on either side, rates of zero and of infinity"""
    c, x = case(13, dtype, 60, 2, 1, 16, 16)
    x["delta"][:] = rounded(np.linspace(-120, 120, 16)[None, None, None] + np.zeros(x["delta"].shape), dtype)
    x["log_rates"][0, :, 0] = -np.inf
    x["log_rates"][0, :, 1] = 30.0
    x["gate"][:] = rounded(np.linspace(-100, 100, 60)[:, None, None, None] + np.zeros(x["gate"].shape), dtype)
    got, want = run(rocm, c, x), reference(c, x)
    f = factors(x)
    b = bounds(c, x, want)
    # E counts what decays to nothing: a state of a product e^-E is off by E e^-E at most, 0.37 of a unit each; 64 units more than cover it, and numbers below fp32's smallest normal one are zero
    unit = (4 * 60 + 16 * 60 + 64 + 32) * U
    size = magnitudes(c, x, f)
    for n in ("output", "state", "d_x", "d_b", "d_c", "d_gate", "d_state"):
        limit = unit * size[n] + 1e-35 * (1 + size[n]) * 1e3 + (UNIT["bfloat16"] * np.abs(want[n]) + 1e-38 if dtype == "bfloat16" and n not in ("state", "d_state") else 0.0)
        assert np.isfinite(got[n]).all() and np.all(np.abs(got[n] - want[n]) <= limit), n
    assert np.isfinite(got["d_delta"]).all() and b is not None


def underflow_of(c, x):
    """Relative bounds end where fp32 does: what decays below 2^-126 may be zero instead, off by 2^-126 at most. On its way to an output such an error meets decays, which are at most one, at most two of the inputs (m is the largest) and a rate, and as many of
    its kind as there are operations: eight for each step and state or channel of the sum."""
    m, rate = max(np.abs(a).max() for n, a in x.items() if n not in ("reset", "lengths", "log_rates")), np.exp(x["log_rates"].max())
    return 2.0 ** -126 * 8 * c["steps"] * (c["rows"] + c["channels"] + c["states"]) * (1 + m) ** 2 * (1 + rate)


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [(20, 330, 8, 5, 16), (17, 300, 8, 9, 27), (33, 400, 8, 9, 8), (20, 150, 8, 65, 16), (9, 150, 8, 66, 20), (25, 280, 8, 7, 3), (100, 260, 8, 3, 16)])
@pytest.mark.parametrize("kind", [dict(resets=0.1, ragged=True), dict(gate=False, with_state=False)])
def test_long_rows_that_a_workgroup_goes_through_one_after_the_other(rocm, shape, dtype, kind):
    """more rows than gradients' workgroups are made for, empty ones between full ones; what lies beyond a row's length is not looked at"""
    print("case", shape, dtype, kind, flush=True)
    steps, rows, heads, channels, states = shape
    groups = 2048 // (heads * ((channels + 63) // 64))
    assert groups < rows
    c, x = case(71 + sum(shape), dtype, *shape, **kind)
    if kind.get("ragged"):
        x["lengths"][groups::7], x["lengths"][3::groups] = 0, steps
    clean = {n: a.copy() for n, a in x.items()}
    if kind.get("ragged"):
        beyond = np.arange(steps)[:, None] >= np.clip(x["lengths"], 0, steps)[None]
        for i, n in enumerate(SEQUENCES):
            x[n][beyond] = (np.nan, np.inf, -np.inf, np.nan, np.inf, -np.inf)[i]
        x["reset"][beyond] = 1
    buffers = Buffers(rocm, c, x)
    wide = 8 if states <= 8 else 16 if states <= 16 else 32
    if channels <= 64:      # the workspace is for the workgroups' shares: fewer than there are rows
        assert buffers.sizes[1] < rows * heads * channels * (wide + 2) * 4
    first, second = run(rocm, c, x), run(rocm, c, x)
    check(c, clean, first, underflow=underflow_of(c, clean))
    assert all(np.array_equal(a, second[n]) for n, a in first.items())


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [(40, 3, 1, 580, 16), (6, 5, 1, 1100, 9), (300, 1, 2, 520, 20)])
def test_more_tiles_of_channels_than_are_added_up_at_a_time(rocm, shape, dtype):
    print("case", shape, dtype, flush=True)
    c, x = case(73 + sum(shape), dtype, *shape, resets=0.05, ragged=shape[1] > 1)
    check(c, x, run(rocm, c, x), underflow=underflow_of(c, x))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_gradients_of_steps_from_tiny_to_huge_and_of_rates_from_none_to_all(rocm, dtype):
    """as test_steps_from_tiny_to_huge_and_rates_from_none_to_all: what exponentials that leave the range of fp32 give delta and the parameters"""
    c, x = case(13, dtype, 60, 2, 1, 16, 16)
    x["delta"][:] = rounded(np.linspace(-120, 120, 16)[None, None, None] + np.zeros(x["delta"].shape), dtype)
    x["log_rates"][0, :, 0] = -np.inf
    x["log_rates"][0, :, 1] = 30.0
    x["gate"][:] = rounded(np.linspace(-100, 100, 60)[:, None, None, None] + np.zeros(x["gate"].shape), dtype)
    got, want, f = run(rocm, c, x), reference(c, x), factors(x)
    unit, size = (4 * 60 + 16 * 60 + 64 + 32 + 62) * U, magnitudes(c, x, f)
    # What is below fp32's smallest normal number, 2^-126, may be zero: a slope, off by 2^-126 at most, times what it is multiplied by, which are the magnitudes for a slope of one; a decay, in the product q = G decay h, and products with it on their way into the
    # sums. G is a sum over steps of c, d_output and the gate's factor and of the last state's gradient, h of delta, x and b and of the first state, whose decays are at most one; q is multiplied by the rate and, in the rates' gradient, by delta (in delta's by a
    # slope, at most one, and over the states). Four such roundings for each of 120 steps of rows.
    m = {n: np.abs(a).max() for n, a in list(x.items()) + [("factor", f["factor"]), ("step", f["delta"])]}
    G, h = 60 * m["c"] * m["d_output"] * m["factor"] + m["d_state"], 60 * m["step"] * m["x"] * m["b"] + m["state"]
    of_decays = 4 * G * h * (1 + m["step"]) * f["rates"][0]      # [channels, states]
    steep = magnitudes(c, x, dict(f, slope=np.ones_like(f["slope"])))["d_delta"] + of_decays.sum(-1)
    lost = dict(d_delta=steep, d_delta_biases=steep.sum((0, 1)), d_log_rates=120 * of_decays, d_skip=np.abs(x["d_output"] * x["gate"] * x["x"]).sum((0, 1)))
    for n, m in lost.items():
        limit = unit * size[n] + 2.0 ** -125 * m
        if dtype == "bfloat16" and n == "d_delta":
            limit = limit + UNIT["bfloat16"] * (np.abs(want[n]) + limit) + 2.0 ** -126      # (below the smallest normal number of that type, too)
        assert np.isfinite(got[n]).all() and np.all(np.abs(got[n] - want[n]) <= limit), (n, float((np.abs(got[n] - want[n]) - limit).max()))


def test_the_rows_that_a_launch_holds():
    """rows x heads below 2^24, beside the limits on elements"""
    lib = package().load_library()
    size = lambda *shape: lib.rlt_rocm_selective_scan_checkpoint_bytes(C.byref(capi.SelectiveScan(4096, None, None, None, None, None, 0, *shape, 0)), 4)
    assert size(2 ** 24 - 1, 1, 1, 1) == (2 ** 24 - 1) * 8 * 4 and size(2 ** 23 - 1, 2, 4, 2) == (2 ** 23 - 1) * 2 * 4 * 8 * 4
    assert size(2 ** 24, 1, 1, 1) == size(2 ** 23, 2, 4, 2) == 0


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("steps", [150, 900])
def test_what_lies_beyond_a_rows_length_is_not_looked_at(rocm, dtype, steps):
    c, x = case(17, dtype, steps, 6, 1, 20, 16, resets=0.05, ragged=True)
    beyond = np.arange(steps)[:, None] >= np.clip(x["lengths"], 0, steps)[None]
    clean = {n: a.copy() for n, a in x.items()}
    for i, n in enumerate(SEQUENCES):
        x[n][beyond] = (np.nan, np.inf, -np.inf, np.nan, np.inf, -np.inf)[i]
    x["reset"][beyond] = 1
    got = run(rocm, c, x)
    check(c, clean, got)
    for n in ("output", "d_x", "d_delta", "d_b", "d_c", "d_gate"):
        assert np.all(got[n][beyond] == 0.0), n
    assert np.array_equal(got["state"][0], x["state"][0].astype(np.float64))      # the empty row's state, bit for bit
    assert np.array_equal(got["d_state"][0], x["d_state"][0].astype(np.float64))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("steps", [1, 100, 700])
def test_a_reset_forgets_a_state_that_is_not_finite(rocm, dtype, steps):
    c, x = case(19, dtype, steps, 3, 1, 20, 16)
    x["reset"] = np.zeros((steps, 3), np.uint8)
    x["reset"][0] = 1
    clean = {n: a.copy() for n, a in x.items()}
    x["state"][0], x["state"][1], x["state"][2] = np.nan, np.inf, -np.inf
    check(c, clean, run(rocm, c, x))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("steps", [200, 800])
def test_an_episode_does_not_see_values_of_another_that_are_not_finite(rocm, dtype, steps):
    """row 0: a step of its first episode holds values that are not finite, in the chunk in which the second episode begins: from there on everything is as if they were. A later episode's do not reach the one before either"""
    c, x = case(41, dtype, steps, 3, 1, 24, 16)
    x["reset"] = np.zeros((steps, 3), np.uint8)
    x["reset"][[75, 90, 140], 0] = 1
    x["reset"][75, 2] = 1
    want = reference(c, x)
    b = bounds(c, x, want)
    for i, n in enumerate(SEQUENCES):
        x[n][70, 0] = (np.nan, np.inf, np.nan, -np.inf, np.nan, np.inf)[i]
        x[n][78, 2] = (np.nan, np.inf, np.nan, -np.inf, np.nan, np.inf)[i]
    got = run(rocm, c, x)
    for n in ("output", "d_x", "d_delta", "d_b", "d_c", "d_gate"):
        off = np.abs(got[n] - want[n]) <= b[n]
        assert np.all(off[75:, 0]) and np.all(off[:, 1]) and np.all(off[:75, 2]), n
    assert np.all(np.abs(got["state"] - want["state"])[:2] <= b["state"][:2]) and np.all(np.abs(got["d_state"] - want["d_state"])[1:] <= b["d_state"][1:])


@gpu
@pytest.mark.parametrize("shape", [(200, 5, 1, 70, 16), (700, 1, 1, 130, 16)])
def test_gradients_add_up_and_runs_repeat_bit_for_bit(rocm, shape):
    c, x = case(23, "float32", *shape, resets=0.02, ragged=shape[1] > 1)
    first, second, onto = run(rocm, c, x), run(rocm, c, x), run(rocm, c, x, onto=3.0)
    for n in first:
        assert np.array_equal(first[n], second[n]), n
    for n in PARAMETERS:
        assert np.allclose(onto["d_" + n], first["d_" + n] + 3.0, rtol=2e-7, atol=0), n


@gpu
@pytest.mark.parametrize("steps", [40, 700])
def test_optional_arguments_and_states_in_place(rocm, steps):
    c, x = case(29, "float32", steps, 2, 1, 20, 16, resets=0.02)
    want = run(rocm, c, x)
    b = Buffers(rocm, c, x)
    call, layer = rocm.device.lib, C.byref(b.layer)
    h = rocm.device.handle
    tail = list(b.tail(0))
    tail[3] = None      # no checkpoints
    assert call.rlt_rocm_selective_scan_forward(h, layer, *b.inputs(), b.o["output"].view, b.state.ptr, None, *tail) == 0
    assert np.array_equal(b.o["output"].numpy(), want["output"])
    assert call.rlt_rocm_selective_scan_forward(h, layer, *b.inputs(), b.o["output"].view, b.state.ptr, b.state.ptr, *b.tail(0)) == 0
    assert np.array_equal(b.o["output"].numpy(), want["output"]) and np.array_equal(b.state.numpy().astype(np.float64), want["state"])
    outs = [b.o[n].view for n in ("d_x", "d_delta", "d_b", "d_c", "d_gate")]
    assert call.rlt_rocm_selective_scan_backward(h, layer, *b.inputs(), b.t["d_output"].view, *outs, b.d_state.ptr, b.d_state.ptr, 0, *b.tail(1)) == 0
    assert np.array_equal(b.d_state.numpy().astype(np.float64), want["d_state"])
    for n in ("d_x", "d_delta", "d_b", "d_c", "d_gate"):
        assert np.array_equal(b.o[n].numpy(), want[n]), n
    bare = layer_of(rocm, c, x, {}, gradients=False)
    bare.log_rates, bare.skip, bare.delta_biases = b.layer.log_rates, b.layer.skip, b.layer.delta_biases
    d_state = rocm.array(x["d_state"])
    assert call.rlt_rocm_selective_scan_backward(h, C.byref(bare), *b.inputs(), b.t["d_output"].view, *outs, d_state.ptr, None, 0, *b.tail(1)) == 0
    rocm.sync()
    for n in ("d_x", "d_delta", "d_b", "d_c", "d_gate"):
        assert np.array_equal(b.o[n].numpy(), want[n]), n


# ------------------------------------------------------------------ single steps


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,heads,channels,states", [(1, 1, 1, 1), (64, 1, 64, 16), (3, 2, 24, 11), (5, 1, 33, 32), (7, 3, 5, 7), (300, 1, 16, 16), (2, 1, 64, 4), (2, 2, 9, 8)])
@pytest.mark.parametrize("in_place", [False, True])
def test_steps_walk_a_sequence(rocm, rows, heads, channels, states, dtype, in_place):
    print("case", rows, heads, channels, states, dtype, in_place, flush=True)
    c, x = case(rows + states, dtype, 5, rows, heads, channels, states, resets=0.3)
    x["reset"][0, 0] = 1
    clean = {n: a.copy() for n, a in x.items()}
    x["state"][0] = np.nan
    want = reference(c, clean)
    b, buffers = bounds(c, clean, want), Buffers(rocm, c, x)
    state, other, item = buffers.state, filled(rocm, x["state"].shape, "float32"), 4 if dtype == "float32" else 2
    for t in range(5):
        at = lambda a: view(a.array, strides_of(a.padded, a.order), item, t * int(np.prod(a.padded[1:])))
        to = state if in_place else other
        rocm.call("selective_scan_step", C.byref(buffers.layer), *[at(buffers.t[n]) for n in SEQUENCES[:5]], at(buffers.o["output"]), state.ptr, to.ptr, buffers.reset.ptr + t * rows)
        if not in_place:
            state, other = other, state
    rocm.sync()
    assert np.all(np.abs(buffers.o["output"].numpy() - want["output"]) <= b["output"]) and np.all(np.abs(state.numpy() - want["state"]) <= b["state"])


# ------------------------------------------------------------------ graphs, refusals


@gpu
@pytest.mark.parametrize("steps", [100, 700])
def test_a_graph_replays_forward_and_backward(rocm, steps):
    lib, h = rocm.device.lib, rocm.device.handle
    c, x = case(31, "bfloat16", steps, 2, 1, 80, 16, resets=0.02, ragged=True)
    want = run(rocm, c, x)
    b = Buffers(rocm, c, x)
    rocm.sync()
    assert lib.rlt_rocm_graph_begin_capture(h) == 0
    b.forward()
    b.backward()
    graph = C.c_void_p()
    assert lib.rlt_rocm_graph_end_capture(h, C.byref(graph)) == 0
    for _ in range(3):
        for a in b.o.values():
            a.array.upload(to_bits(np.full(a.array.shape, 7.0, np.float32)))      # eager work between the replays
        assert lib.rlt_rocm_graph_launch(h, graph) == 0
        rocm.sync()
        for name, a in b.results().items():
            assert np.array_equal(a, want[name]), name
    lib.rlt_rocm_graph_destroy(h, graph)


def changed(layer, **fields):
    return C.byref(capi.SelectiveScan(**dict({n: getattr(layer, n) for n, _ in layer._fields_}, **fields)))


def test_refusals_without_a_device():
    lib = package().load_library()
    good = capi.SelectiveScan(4096, None, None, None, None, None, 0, 2, 1, 100, 16, 0)
    for size in (lambda layer, steps: lib.rlt_rocm_selective_scan_workspace_bytes(layer, steps, 1), lib.rlt_rocm_selective_scan_checkpoint_bytes):
        assert size(C.byref(good), 40) > 0
        for layer in (None, changed(good, heads=2, channels=2 ** 20), changed(good, batch=1, heads=1, channels=2 ** 20 + 1), changed(good, states=33), changed(good, states=0), changed(good, channels=0), changed(good, type=2), changed(good, batch=2 ** 20, channels=2 ** 10), changed(good, batch=2 ** 30, heads=2 ** 30)):
            assert size(layer, 40) == 0
        assert size(C.byref(good), 0) == size(C.byref(good), 2 ** 30 + 1) == size(changed(good, batch=64), 2 ** 26) == 0
    assert lib.rlt_rocm_selective_scan_forward(None, C.byref(good), *[None] * 6, None, None, None, None, 4, None, None, 0) == capi.RLT_E_NOT_INITIALISED


@gpu
def test_refusals(rocm):
    lib, h = rocm.device.lib, rocm.device.handle
    c, x = case(37, "float32", 4, 2, 1, 70, 16)
    b = Buffers(rocm, c, x)
    none, good = C.byref(capi.HeadView(None, 1, 1, 1)), C.byref(b.layer)
    inputs, outs = b.inputs(), [b.o[n].view for n in ("d_x", "d_delta", "d_b", "d_c", "d_gate")]

    def forward(layer=good, views=inputs + [b.o["output"].view], steps=4, checkpoints=b.checkpoints.ptr):
        return lib.rlt_rocm_selective_scan_forward(h, layer, *views, None, None, None, None, steps, checkpoints, b.scratch[0].ptr, b.sizes[0])

    def backward(layer=good, views=inputs + [b.t["d_output"].view] + outs, steps=4, checkpoints=b.checkpoints.ptr, ptr=b.scratch[1].ptr, size=b.sizes[1]):
        return lib.rlt_rocm_selective_scan_backward(h, layer, *views, None, None, 0, None, None, steps, checkpoints, ptr, size)

    def step(layer=good, views=inputs + [b.o["output"].view], state=b.state.ptr, to=b.state.ptr):
        return lib.rlt_rocm_selective_scan_step(h, layer, *views, state, to, None)
    assert forward() == backward() == step() == 0
    for call, n in ((forward, 6), (backward, 11), (step, 6)):
        for layer in (None, changed(b.layer, type=2), changed(b.layer, batch=0), changed(b.layer, heads=0), changed(b.layer, channels=-1), changed(b.layer, states=0), changed(b.layer, log_rates=None)):
            assert call(layer) == capi.RLT_E_INVALID_ARGUMENT
        assert call(changed(b.layer, states=33)) == call(changed(b.layer, batch=2 ** 20, channels=2 ** 10)) == capi.RLT_E_UNSUPPORTED
        views = inputs + ([b.t["d_output"].view] + outs if n == 11 else [b.o["output"].view])
        for i in range(n):
            assert call(views=views[:i] + [none] + views[i + 1:]) == capi.RLT_E_INVALID_ARGUMENT
            if i != 4:      # (no gate is no error)
                assert call(views=views[:i] + [None] + views[i + 1:]) == capi.RLT_E_INVALID_ARGUMENT
    for call in (forward, backward):
        assert call(steps=0) == call(checkpoints=b.checkpoints.ptr + 4) == capi.RLT_E_INVALID_ARGUMENT
        assert call(steps=2 ** 30 + 1) == capi.RLT_E_UNSUPPORTED
        far = C.byref(capi.HeadView(b.t["x"].array.ptr, 2 ** 27 + 1, 1, 1))
        views = inputs + ([b.t["d_output"].view] + outs if call is backward else [b.o["output"].view])
        assert all(call(views=views[:i] + [far] + views[i + 1:]) == capi.RLT_E_UNSUPPORTED for i in range(len(views)))
    assert backward(checkpoints=None) == backward(ptr=None) == backward(size=b.sizes[1] - 1) == backward(ptr=b.scratch[1].ptr + 8) == capi.RLT_E_INVALID_ARGUMENT
    assert step(state=None) == step(to=None) == capi.RLT_E_INVALID_ARGUMENT
    long = case(38, "float32", 700, 1, 1, 16, 16)
    b2 = Buffers(rocm, *long)
    assert b2.sizes[0] > 0      # cut into segments: a forward call without its scratch memory is refused
    assert lib.rlt_rocm_selective_scan_forward(h, C.byref(b2.layer), *b2.inputs(), b2.o["output"].view, None, None, None, None, 700, None, None, 0) == capi.RLT_E_INVALID_ARGUMENT
    rocm.sync()

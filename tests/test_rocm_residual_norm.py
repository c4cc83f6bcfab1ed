"""The norms around a block with its gate and residual scale, forward and backward, against the formulas in 64 bits.

Bounds, set before the first run. An element passes at most 128 roundings (sums over a row are trees over threads that each add up at most 32 columns; activation functions to a few units): 128 * 2^-24 of the magnitudes
that meet in it, where subtracting a mean counts the row's values with theirs. Column sums add the rows up: (rows + 160) * 2^-24 of the summands' magnitudes times what those are off themselves (1 + 128 / (rows + 160)).
bfloat16 outputs add their own rounding, 2^-8 of the value."""
import ctypes as C

import numpy as np
import pytest

from helpers import capi
from typed_arrays import UNIT, download, filled, rounded, upload

gpu = pytest.mark.gpu
U = 128 * 2.0 ** -24
PARAMETERS = ["branch_weights", "branch_biases", "output_weights", "output_biases", "residual_scale"]


def act(x, kind):
    if kind == "relu":
        return np.maximum(x, 0), (x > 0).astype(float)
    if kind == "gelu":      # with the reference library's constant
        a, b = 0.3989422804014327, 0.044715
        t = np.tanh(a * (b * x ** 3 + x))
        return 0.5 * x * (1 + t), 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * a * (3 * b * x * x + 1)
    if kind == "tanh":
        return np.tanh(x), 1 - np.tanh(x) ** 2
    if kind == "fast_tanh":
        c = np.clip(x, -3, 3)
        t = c * (27 + c * c) / (27 + 9 * c * c)
        return t, 1 - t * t
    if kind == "sigmoid":
        s = 1 / (1 + np.exp(-x))
        return s, s * (1 - s)
    return x, np.ones_like(x)


def normalised(x, kind, epsilon):
    """x normalised, 1 / deviation, and what its elements may be off, relative to U (subtracting the mean counts the row's own magnitudes)"""
    if kind == "none":
        return x, np.ones((len(x), 1)), np.abs(x)
    centred = x - x.mean(1, keepdims=True) if kind == "layer" else x
    inverse = 1 / np.sqrt((centred ** 2).mean(1, keepdims=True) + epsilon)
    magnitude = np.abs(x) + (np.abs(x).mean(1, keepdims=True) if kind == "layer" else 0)
    return centred * inverse, inverse, magnitude * inverse * (1 + (np.abs(x).mean(1, keepdims=True) * inverse if kind == "layer" else 0))


def one(x, otherwise):
    return otherwise if x is None else x.astype(np.float64)


def forward(c, x):
    """outputs and the magnitudes of their bounds"""
    y, my = x["x"], np.abs(x["x"])
    if x.get("branch") is not None:
        n, _, mn = normalised(x["branch"], c["branch_norm"], c["epsilon"])
        w, b = one(x.get("branch_weights"), 1.0), one(x.get("branch_biases"), 0.0)
        m = act(x["gate"], c["activation"])[0] if x.get("gate") is not None else 1.0
        s = one(x.get("residual_scale"), 1.0)
        y, my = y + s * m * (n * w + b), my + np.abs(s) * (np.abs(m) + (1e-3 if x.get("gate") is not None else 0)) * (mn * np.abs(w) + np.abs(b))
    h, _, mh = normalised(y, c["output_norm"], c["epsilon"])
    # what y is off counts as its own magnitude does
    inverse = normalised(y, c["output_norm"], c["epsilon"])[1]
    mh = mh + my * inverse + np.abs(h) * np.sqrt((my ** 2).mean(1, keepdims=True)) * inverse * (c["output_norm"] != "none") + (my.mean(1, keepdims=True) * inverse if c["output_norm"] == "layer" else 0)
    w, b = one(x.get("output_weights"), 1.0), one(x.get("output_biases"), 0.0)
    return dict(y=y, h=h * w + b), dict(y=my, h=mh * np.abs(w) + np.abs(b))


def through_norm(d, md, n, mn, inverse, kind):
    if kind == "none":
        return d, md
    along, mean = (d * n).mean(1, keepdims=True), d.mean(1, keepdims=True) if kind == "layer" else 0.0
    m_along, m_mean = (md * mn).mean(1, keepdims=True), md.mean(1, keepdims=True) if kind == "layer" else 0.0
    return inverse * (d - n * along - mean), inverse * (md + mn * m_along + m_mean) * (1 + mn / np.maximum(1, np.abs(n)))


def backward(c, x):
    out, size = {}, {}
    d, md = (x["d_y"], np.abs(x["d_y"])) if x.get("d_y") is not None else (0.0, 0.0)
    rows = len(x["y"])
    if x.get("d_h") is not None:
        n, inverse, mn = normalised(x["y"], c["output_norm"], c["epsilon"])
        out["d_output_weights"], size["d_output_weights"] = (x["d_h"] * n).sum(0), (np.abs(x["d_h"]) * mn).sum(0)
        out["d_output_biases"], size["d_output_biases"] = x["d_h"].sum(0), np.abs(x["d_h"]).sum(0)
        e = x["d_h"] * one(x.get("output_weights"), 1.0)
        e, me = through_norm(e, np.abs(e), n, mn, inverse, c["output_norm"])
        d, md = d + e, md + me
    d, md = np.broadcast_to(d, x["y"].shape), np.broadcast_to(md, x["y"].shape)
    out["d_x"], size["d_x"] = d, md
    if x.get("branch") is not None:
        n, inverse, mn = normalised(x["branch"], c["branch_norm"], c["epsilon"])
        w, b, s = one(x.get("branch_weights"), 1.0), one(x.get("branch_biases"), 0.0), one(x.get("residual_scale"), 1.0)
        m, slope = act(x["gate"], c["activation"]) if x.get("gate") is not None else (1.0, 0.0)
        mm = np.abs(m) + (1e-3 if x.get("gate") is not None else 0)
        full, m_full = n * w + b, mn * np.abs(w) + np.abs(b)
        dn, mdn = d * s * m, md * np.abs(s) * mm
        for name, value, magnitude in (("d_branch_weights", dn * n, mdn * mn), ("d_branch_biases", dn, mdn), ("d_residual_scale", d * m * full, md * mm * m_full)):
            out[name], size[name] = value.sum(0), magnitude.sum(0)
        if x.get("gate") is not None:
            out["d_gate"], size["d_gate"] = d * s * full * slope, md * np.abs(s) * m_full * (np.abs(slope) + 1)
        out["d_branch"], size["d_branch"] = through_norm(dn * w, mdn * np.abs(w), n, mn, inverse, c["branch_norm"])
    for name in list(size):
        if name[2:] in PARAMETERS:
            size[name] = size[name] * (rows + 160 + 128) / 128
    return out, size


def case(seed, dtype, rows, dim, branch_norm="rms", output_norm="rms", activation="sigmoid", gate=True, parameters=PARAMETERS):
    rng = np.random.default_rng(seed)
    n = lambda scale=1.0, shift=0.0: rounded(scale * rng.standard_normal((rows, dim)) + shift, dtype)
    x = dict(x=n(), branch=n(2.0, 0.5), gate=n(1.5) if gate else None, y=n(1.5, -0.2), d_y=n(), d_h=n())
    for p in parameters:
        x[p] = (0.3 * rng.standard_normal(dim) + (0.0 if "biases" in p else 1.0)).astype(np.float32)
    return dict(dtype=dtype, rows=rows, dim=dim, branch_norm=branch_norm, output_norm=output_norm, activation=activation, epsilon=float(np.float32(1e-5))), x


class Rows:
    def __init__(self, rocm, x, dtype, pad=0, offset=0, fill=None):
        self.dtype, self.cols, self.ld, self.offset = dtype, x.shape[1], x.shape[1] + pad, offset
        host = np.full((x.shape[0], self.ld), 9.0, np.float32)
        host[:, :self.cols] = x if fill is None else fill
        self.array = upload(rocm, np.concatenate([np.full(offset, 9.0, np.float32), host.reshape(-1)]), dtype)
        self.ptr = self.array.ptr + offset * (4 if dtype == "float32" else 2)

    def numpy(self):
        whole = download(self.array, self.dtype)[self.offset:].reshape(-1, self.ld)
        assert np.all(whole[:, self.cols:] == 9.0)      # nothing is written between the rows
        return whole[:, :self.cols]


def layer_of(rocm, c, x, gradients=None):
    layer = capi.ResidualNorm(type=capi.TYPE[c["dtype"]], dim=c["dim"], branch_norm=capi.NORM[c["branch_norm"]], output_norm=capi.NORM[c["output_norm"]], gate_activation=capi.ACT[c["activation"]],
                              epsilon=c["epsilon"])
    for p in PARAMETERS:
        if x.get(p) is not None:
            setattr(layer, p, rocm.array(x[p]).ptr)
    for p, a in (gradients or {}).items():
        setattr(layer, p, a.ptr)
    return layer


def run_forward(rocm, c, x, pad=0, offset=0, in_place=False):
    layer = layer_of(rocm, c, x)
    rows = lambda n: Rows(rocm, x[n], c["dtype"], pad, offset) if x.get(n) is not None else None
    xs, u, g = rows("x"), rows("branch"), rows("gate")
    y, h = xs if in_place else Rows(rocm, x["x"], c["dtype"], pad, offset, 7.0), Rows(rocm, x["x"], c["dtype"], pad, offset, 7.0)
    at = lambda r: (r.ptr, r.ld) if r is not None else (None, 0)
    rocm.call("residual_norm_forward", C.byref(layer), *at(xs), *at(u), *at(g), *at(y), *at(h), c["rows"])
    rocm.sync()
    return dict(y=y.numpy(), h=h.numpy())


def run_backward(rocm, c, x, pad=0, offset=0, accumulate_onto=None, wanted=("d_x", "d_branch", "d_gate")):
    grads = {"d_" + p: rocm.array(np.full(c["dim"], 7.0 if accumulate_onto is None else accumulate_onto, np.float32)) for p in PARAMETERS
             if (x.get("d_h") is not None if "output" in p else x.get("branch") is not None)}
    layer = layer_of(rocm, c, x, grads)
    n = rocm.device.lib.rlt_rocm_residual_norm_workspace_bytes(C.byref(layer), c["rows"])
    w = rocm.device.empty((max(int(n), 4),), np.uint8)
    rows = lambda n: Rows(rocm, x[n], c["dtype"], pad, offset) if x.get(n) is not None else None
    at = lambda r: (r.ptr, r.ld) if r is not None else (None, 0)
    to = {n: Rows(rocm, x["y"], c["dtype"], pad, offset, 7.0) for n in wanted if n == "d_x" or x.get(n[2:]) is not None}
    rocm.call("residual_norm_backward", C.byref(layer), *at(rows("branch")), *at(rows("gate")), *at(rows("y")), *at(rows("d_y")), *at(rows("d_h")), *at(to.get("d_x")), *at(to.get("d_branch")),
              *at(to.get("d_gate")), c["rows"], int(accumulate_onto is not None), w.ptr, n)
    rocm.sync()
    return dict({n: r.numpy() for n, r in to.items()}, **{n: a.numpy().astype(np.float64) for n, a in grads.items()})


def check(c, got, want, size):
    for n, g in got.items():
        bound = U * size[n] + (UNIT["bfloat16"] * np.abs(want[n]) if c["dtype"] == "bfloat16" and n[2:] not in PARAMETERS else 0.0)
        off = np.abs(g - want[n]) - bound
        assert np.all(off <= 0), (n, float(off.max()), float(np.abs(want[n]).max()))


# ------------------------------------------------------------------ the reference itself (no GPU)


@pytest.mark.parametrize("activation", ["identity", "sigmoid", "tanh", "gelu"])
@pytest.mark.parametrize("norms", [("rms", "layer"), ("layer", "rms"), ("none", "layer"), ("rms", "none")])
def test_the_references_gradients_are_its_differences(norms, activation):
    c, x = case(0, "float32", 5, 7, *norms, activation)
    x = {n: a.astype(np.float64) for n, a in x.items()}
    x["y"] = forward(c, x)[0]["y"]
    got = backward(c, x)[0]
    loss = lambda z: sum((a * x["d_" + n]).sum() for n, a in forward(c, z)[0].items())
    rng = np.random.default_rng(1)
    for name in ["x", "branch", "gate"] + PARAMETERS:
        direction = rng.standard_normal(x[name].shape)
        numeric = (loss(dict(x, **{name: x[name] + 1e-6 * direction})) - loss(dict(x, **{name: x[name] - 1e-6 * direction}))) / 2e-6
        assert abs(numeric - (got["d_" + name] * direction).sum()) <= 1e-6 * max(1.0, abs(numeric)), name


# ------------------------------------------------------------------ on the card

SIZES = [(1, 1), (3, 2), (5, 7), (4, 8), (70, 64), (33, 63), (256, 256), (9, 511), (5, 512), (3, 513), (40, 1000), (7, 1024), (6, 2047), (3, 4096), (2, 4100), (3, 8192), (1500, 24), (5000, 8)]


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("norms", [("rms", "rms"), ("layer", "layer")])
def test_sizes(rocm, size, dtype, norms):
    print("case", size, dtype, norms, flush=True)
    c, x = case(sum(size), dtype, *size, *norms)
    check(c, run_forward(rocm, c, x), *forward(c, x))
    check(c, run_backward(rocm, c, x), *backward(c, x))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("norms", [("none", "none"), ("none", "rms"), ("layer", "none"), ("rms", "layer")])
@pytest.mark.parametrize("activation", ["identity", "relu", "gelu", "tanh", "fast_tanh", "sigmoid"])
def test_norms_and_activations(rocm, dtype, norms, activation):
    c, x = case(3, dtype, 37, 136, *norms, activation)
    check(c, run_forward(rocm, c, x), *forward(c, x))
    check(c, run_backward(rocm, c, x), *backward(c, x))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("pad,offset", [(8, 0), (3, 0), (0, 1), (8, 8), (5, 3)])
def test_strides_and_alignments(rocm, dtype, pad, offset):
    for dim in (120, 1032):
        c, x = case(5, dtype, 19, dim, "layer", "rms")
        check(c, run_forward(rocm, c, x, pad, offset), *forward(c, x))
        check(c, run_forward(rocm, c, x, pad, offset, in_place=True), *forward(c, x))
        check(c, run_backward(rocm, c, x, pad, offset), *backward(c, x))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("absent", [("gate",), ("branch", "gate"), ("d_y",), ("d_h",), ("branch", "gate", "d_y"), tuple(PARAMETERS)])
def test_what_may_be_absent(rocm, dtype, absent):
    c, x = case(7, dtype, 30, 200, "rms", "layer", parameters=[p for p in PARAMETERS if p not in absent])
    x.update({n: None for n in absent if n not in PARAMETERS})
    if not {"d_y", "d_h"} & set(absent):
        check(c, run_forward(rocm, c, x), *forward(c, x))
    check(c, run_backward(rocm, c, x), *backward(c, x))
    check(c, run_backward(rocm, c, x, wanted=("d_x",)), *backward(c, x))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_rows_without_content(rocm, dtype):
    """rows of zeros (a deviation of zero), rows whose mean is far from their spread, and rows that are not finite, which stay to themselves"""
    c, x = case(9, dtype, 12, 96, "layer", "rms")
    x["branch"][0], x["x"][0], x["y"][0] = 0.0, 0.0, 0.0
    x["branch"][1] = rounded(100 + np.random.default_rng(0).standard_normal(96), dtype)
    for n, value in (("branch", np.nan), ("d_h", np.inf)):
        x[n][5] = value
    finite = [r for r in range(12) if r != 5]
    few = dict({n: (a[finite] if a is not None and a.ndim == 2 else a) for n, a in x.items()})
    got = run_forward(rocm, c, x)
    check(c, {n: a[finite] for n, a in got.items()}, *forward(c, few))
    assert np.isnan(got["y"][5]).all()
    got = run_backward(rocm, c, x)
    want, size = backward(c, few)
    check(c, {n: got[n][finite] for n in ("d_x", "d_branch", "d_gate")}, want, size)


@gpu
def test_sums_accumulate_and_repeat_bit_for_bit(rocm):
    c, x = case(11, "bfloat16", 900, 320, "layer", "layer")
    first, second, onto = run_backward(rocm, c, x), run_backward(rocm, c, x), run_backward(rocm, c, x, accumulate_onto=2.0)
    for n in first:
        assert np.array_equal(first[n], second[n]), n
        if n[2:] in PARAMETERS:
            assert np.allclose(onto[n], first[n] + 2.0, rtol=2e-7, atol=2e-7), n


@gpu
def test_a_graph_replays_both_passes(rocm):
    lib, h = rocm.device.lib, rocm.device.handle
    c, x = case(13, "float32", 100, 260, "rms", "rms")
    want, want_back = run_forward(rocm, c, x), run_backward(rocm, c, x)
    grads = {"d_" + p: rocm.zeros((260,)) for p in PARAMETERS}
    layer = layer_of(rocm, c, x, grads)
    n = lib.rlt_rocm_residual_norm_workspace_bytes(C.byref(layer), 100)
    w = rocm.device.empty((int(n),), np.uint8)
    a = {k: rocm.array(x[k].astype(np.float32)) for k in ("x", "branch", "gate", "y", "d_y", "d_h")}
    y, hh, dx, db, dg = (rocm.zeros((100, 260)) for _ in range(5))
    rocm.sync()
    assert lib.rlt_rocm_graph_begin_capture(h) == 0
    rocm.call("residual_norm_forward", C.byref(layer), a["x"].ptr, 260, a["branch"].ptr, 260, a["gate"].ptr, 260, y.ptr, 260, hh.ptr, 260, 100)
    rocm.call("residual_norm_backward", C.byref(layer), a["branch"].ptr, 260, a["gate"].ptr, 260, a["y"].ptr, 260, a["d_y"].ptr, 260, a["d_h"].ptr, 260, dx.ptr, 260, db.ptr, 260, dg.ptr, 260, 100, 0,
              w.ptr, n)
    graph = C.c_void_p()
    assert lib.rlt_rocm_graph_end_capture(h, C.byref(graph)) == 0
    for _ in range(3):
        y.upload(np.zeros((100, 260), np.float32))
        assert lib.rlt_rocm_graph_launch(h, graph) == 0
        rocm.sync()
        assert np.array_equal(y.numpy(), want["y"]) and np.array_equal(hh.numpy(), want["h"]) and np.array_equal(db.numpy(), want_back["d_branch"])
        assert all(np.array_equal(grads[k].numpy(), want_back[k]) for k in grads)
    lib.rlt_rocm_graph_destroy(h, graph)


@gpu
def test_refusals(rocm):
    lib, h = rocm.device.lib, rocm.device.handle
    c, x = case(15, "float32", 4, 16)
    a = rocm.array(x["x"].astype(np.float32))
    g = {"d_branch_weights": rocm.zeros((16,))}

    def forward_code(layer, ld=16, x=a.ptr, y=a.ptr, rows=4, branch=a.ptr):
        return lib.rlt_rocm_residual_norm_forward(h, C.byref(layer) if layer is not None else None, x, ld, branch, 16, None, 0, y, 16, None, 0, rows)

    def changed(**fields):
        layer = layer_of(rocm, c, {})
        for name, value in fields.items():
            setattr(layer, name, value)
        return layer
    assert forward_code(changed()) == 0
    for layer in (None, changed(type=5), changed(dim=0), changed(branch_norm=3), changed(output_norm=-1), changed(gate_activation=6), changed(epsilon=0.0), changed(epsilon=float("nan"))):
        assert forward_code(layer) == capi.RLT_E_INVALID_ARGUMENT
    assert forward_code(changed(), ld=15) == forward_code(changed(), x=None) == forward_code(changed(), rows=0) == forward_code(changed(), y=None) == capi.RLT_E_INVALID_ARGUMENT
    big = rocm.zeros((1, 8200))
    assert lib.rlt_rocm_residual_norm_forward(h, C.byref(changed(dim=8193)), big.ptr, 8200, None, 0, None, 0, big.ptr, 8200, None, 0, 1) == capi.RLT_E_UNSUPPORTED
    assert lib.rlt_rocm_residual_norm_forward(None, C.byref(changed()), a.ptr, 16, None, 0, None, 0, a.ptr, 16, None, 0, 4) == capi.RLT_E_NOT_INITIALISED

    def backward_code(layer, branch=a.ptr, gate=None, y=a.ptr, d_y=a.ptr, d_h=a.ptr, d_branch=None, d_gate=None, w=None, n=0):
        return lib.rlt_rocm_residual_norm_backward(h, C.byref(layer), branch, 16, gate, 16, y, 16, d_y, 16, d_h, 16, None, 0, d_branch, 16, d_gate, 16, 4, 0, w, n)
    plain, summed = changed(), layer_of(rocm, c, {}, g)
    out = rocm.zeros((4, 16))
    assert backward_code(plain, d_branch=out.ptr) == 0
    need = lib.rlt_rocm_residual_norm_workspace_bytes(C.byref(summed), 4)
    w = rocm.device.empty((int(need),), np.uint8)
    assert need > 0 and backward_code(summed, w=w.ptr, n=need) == 0
    assert backward_code(summed) == backward_code(summed, w=w.ptr, n=need - 1) == capi.RLT_E_INVALID_ARGUMENT
    assert backward_code(summed, branch=None, w=w.ptr, n=need) == capi.RLT_E_INVALID_ARGUMENT      # nothing reaches the branch's weights
    assert backward_code(plain, d_y=None, d_h=None) == backward_code(plain, y=None) == backward_code(plain, d_gate=out.ptr) == backward_code(plain, branch=None, d_branch=out.ptr) == capi.RLT_E_INVALID_ARGUMENT
    rocm.sync()


@gpu
def test_more_rows_than_an_index_holds_are_refused(rocm):
    a = rocm.zeros((4, 16))
    layer = layer_of(rocm, dict(dtype="float32", dim=16, rows=4, branch_norm="rms", output_norm="rms", activation="sigmoid", epsilon=1e-5), {})
    lib, h = rocm.device.lib, rocm.device.handle
    for rows in (2 ** 30 + 1, 2 ** 31 - 1):
        assert lib.rlt_rocm_residual_norm_forward(h, C.byref(layer), a.ptr, 16, None, 0, None, 0, a.ptr, 16, None, 0, rows) == capi.RLT_E_UNSUPPORTED
        assert lib.rlt_rocm_residual_norm_backward(h, C.byref(layer), None, 0, None, 0, a.ptr, 16, a.ptr, 16, None, 0, a.ptr, 16, None, 0, None, 0, rows, 0, None, 0) == capi.RLT_E_UNSUPPORTED

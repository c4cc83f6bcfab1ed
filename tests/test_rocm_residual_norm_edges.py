"""The norms around a block where values and sizes are out of the ordinary. The reference in 64 bits, the cases and the bounds are those of test_rocm_residual_norm."""
import ctypes as C

import numpy as np
import pytest

from test_rocm_residual_norm import PARAMETERS, Rows, U, act, backward, case, check, forward, layer_of, run_backward, run_forward

gpu = pytest.mark.gpu


def gates_alone(rocm, gates, activation):
    """act(gate) and its derivative as the two passes form them: no norms, no parameters, a branch and gradients of ones"""
    x = dict(x=np.zeros_like(gates), branch=np.ones_like(gates), gate=gates, y=np.zeros_like(gates), d_y=np.ones_like(gates), d_h=None)
    c = dict(dtype="float32", rows=len(gates), dim=gates.shape[1], branch_norm="none", output_norm="none", activation=activation, epsilon=1e-5)
    return run_forward(rocm, c, x)["y"], run_backward(rocm, c, x)["d_gate"]


@gpu
def test_sigmoid_gates_keep_their_relative_accuracy(rocm):
    """The exponential to two units of 2^-24, the sum one, the quotient two, the product one, those with the scale and the branch two: eight of the value, for gates from -80 to 80 (beyond -87 it leaves fp32's range)."""
    gates = np.linspace(-80, 80, 64 * 250).astype(np.float32).astype(np.float64).reshape(64, 250)
    value, slope = gates_alone(rocm, gates, "sigmoid")
    small = 1 / (1 + np.exp(np.abs(gates)))      # the smaller of sigmoid(g) and 1 - sigmoid(g)
    want, want_slope = np.where(gates < 0, small, 1 - small), small * (1 - small)
    print("largest errors, units:", np.max(np.abs(value - want) / want) * 2 ** 24, np.max(np.abs(slope - want_slope) / want_slope) * 2 ** 24, flush=True)
    assert np.all(np.abs(value - want) <= 8 * 2.0 ** -24 * want) and np.all(np.abs(slope - want_slope) <= 8 * 2.0 ** -24 * want_slope)


@gpu
@pytest.mark.parametrize("activation", ["relu", "gelu", "tanh", "fast_tanh", "sigmoid"])
def test_gates_of_any_size(rocm, activation):
    """from the smallest numbers to the largest, of either sign: functions and derivatives as in 64 bits, to U = 128 units of the value and of one (the functions' own range)"""
    gates = np.concatenate([2.0 ** np.arange(-126, 128), [float(np.finfo(np.float32).max)] * 2])
    gates = np.stack([gates, -gates]).astype(np.float32).astype(np.float64)
    value, slope = gates_alone(rocm, gates, activation)
    with np.errstate(over="ignore"):
        want, want_slope = act(gates, activation)
    assert np.all(np.abs(value - want) <= U * (np.abs(want) + np.minimum(1, np.abs(gates))))
    assert np.all(np.abs(slope - want_slope) <= U * (np.abs(want_slope) + 1))


@gpu
@pytest.mark.parametrize("activation", ["gelu", "sigmoid", "tanh"])
def test_gates_that_are_not_numbers_stay_so(rocm, activation):
    value, slope = gates_alone(rocm, np.full((3, 50), np.nan), activation)
    assert np.isnan(value).all() and np.isnan(slope).all()


# ------------------------------------------------------------------ more rows than one turn of the grid takes
# backward: 512 workgroups of 16, 4 or 2 rows (up to 128, 512, 1,024 columns) or of one; forward: 2,048 of 16, 4 or one


def run_without_biases(rocm, c, x):
    """the backward pass's instances that have no biases and sum up none"""
    parameters = [p for p in PARAMETERS if "biases" not in p]
    grads = {"d_" + p: rocm.array(np.full(c["dim"], 7.0, np.float32)) for p in parameters}
    layer = layer_of(rocm, c, x, grads)
    n = rocm.device.lib.rlt_rocm_residual_norm_workspace_bytes(C.byref(layer), c["rows"])
    w = rocm.device.empty((int(n),), np.uint8)
    of = {n: Rows(rocm, x[n], c["dtype"]) for n in ("branch", "gate", "y", "d_y", "d_h")}
    to = {n: Rows(rocm, x["y"], c["dtype"], fill=7.0) for n in ("d_x", "d_branch", "d_gate")}
    at = lambda r: (r.ptr, r.ld)
    rocm.call("residual_norm_backward", C.byref(layer), *at(of["branch"]), *at(of["gate"]), *at(of["y"]), *at(of["d_y"]), *at(of["d_h"]), *at(to["d_x"]), *at(to["d_branch"]), *at(to["d_gate"]), c["rows"], 0, w.ptr, n)
    rocm.sync()
    return dict({n: r.numpy() for n, r in to.items()}, **{n: a.numpy().astype(np.float64) for n, a in grads.items()})


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,dim", [(17001, 24), (9000, 128), (5003, 320), (2500, 1000), (1200, 2047), (1100, 2048), (1300, 4095), (1100, 4096), (1025, 4100), (1027, 4099), (1100, 8192)])
@pytest.mark.parametrize("biases", [True, False])
def test_gradients_of_more_rows_than_the_grid(rocm, rows, dim, dtype, biases):
    print("case", rows, dim, dtype, biases, flush=True)
    c, x = case(rows + dim, dtype, rows, dim, "layer", "layer", parameters=[p for p in PARAMETERS if biases or "biases" not in p])
    check(c, run_backward(rocm, c, x) if biases else run_without_biases(rocm, c, x), *backward(c, x))


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,dim", [(40001, 24), (8500, 320), (4100, 511), (2100, 1000), (2050, 2047), (2100, 4096), (2049, 4100)])
def test_more_rows_than_the_grid(rocm, rows, dim, dtype):
    print("case", rows, dim, dtype, flush=True)
    c, x = case(rows + dim, dtype, rows, dim, "rms", "layer")
    check(c, run_forward(rocm, c, x), *forward(c, x))

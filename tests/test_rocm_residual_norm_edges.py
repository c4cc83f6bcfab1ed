"""The norms around a block where values and sizes are out of the ordinary. The reference in 64 bits, the cases and the bounds are those of test_rocm_residual_norm."""
import numpy as np
import pytest

from test_rocm_residual_norm import U, act, run_backward, run_forward

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

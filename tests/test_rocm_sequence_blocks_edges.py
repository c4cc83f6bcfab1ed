"""The stack of sequence blocks where training, acting and evaluation meet. Reference, cases and bounds are those of test_rocm_sequence_blocks."""
import numpy as np
import pytest

from test_rocm_sequence_blocks import case, reference

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dropout", [True, False])
@pytest.mark.parametrize("reset", [True, False])
def test_gradients_are_those_of_the_last_pass(rocm, dropout, reset):
    """what the forward call had (streams, resets, dropout or none) need not be said again"""
    c, p, x, resets, net, tolerance, rng = case(rocm, 5, 40, 6, 48, 3, 1, 2, dropout=0.4)
    net.forward(stream=3)
    got = net.forward(stream=8, reset=reset, dropout=dropout).numpy().reshape(x.shape)
    resets = resets if reset else np.zeros_like(resets)
    of = lambda p, x: reference(c, p, x, resets, 8 if dropout else None)
    want = of(p, x)
    assert np.max(np.abs(got - want)) <= tolerance * np.max(np.abs(want))
    d = rng.standard_normal(x.shape).astype(np.float32)
    net.zero_gradient()
    net.backward(rocm.array(d.reshape(-1, 48)))
    gradients = {n: v.numpy().astype(np.float64) for n, v in net.grad_views.items()}
    for name, g in list(gradients.items()) + [("x", net.d_stream.numpy().astype(np.float64).reshape(x.shape))]:
        along, step = rng.choice([-1.0, 1.0], g.shape), 1e-6
        at = lambda s: np.sum(d * (of(p, x + s * along) if name == "x" else of({**p, name: p[name] + s * along}, x)))
        quotient = (at(step) - at(-step)) / (2 * step)
        assert abs(np.sum(g * along) - quotient) <= (3 * tolerance + 1e-6) * max(np.linalg.norm(g) * np.linalg.norm(along), abs(quotient)), name

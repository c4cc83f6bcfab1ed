"""The stack of sequence blocks where training, acting and evaluation meet. Reference, cases and bounds are those of test_rocm_sequence_blocks."""
import ctypes as C

import numpy as np
import pytest

from helpers import capi
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


@gpu
def test_training_leaves_the_rollouts_states_alone(rocm):
    """steps with forward and backward passes between them against steps without, bit for bit; a pass without dropout leaves its own states, or not if it is asked so"""
    c, p, x, resets, net, tolerance, rng = case(rocm, 6, 30, 4, 32, 2, 2, 2, dropout=0.2)
    d = rocm.array(rng.standard_normal((30 * 4, 32)).astype(np.float32))

    def act(between):
        for s in net.states:
            s.upload(np.zeros(s.shape, np.float32))
        h = []
        for t in range(6):
            between()
            net.step_x.upload(x[t].astype(np.float32))
            net.step_reset.upload(resets[t])
            h.append(net.step().numpy())
        return np.stack(h)

    def train():
        net.forward(stream=2)
        net.zero_gradient()
        net.backward(d)
    alone = act(lambda: None)
    assert np.array_equal(alone, act(train)) and np.array_equal(alone, act(lambda: net.forward(dropout=False, keep_states=False)))
    final = [s.numpy() for s in net.states]
    net.forward(dropout=False)
    kept = [s.numpy() for s in net.states]
    assert all(not np.array_equal(a, b) for a, b in zip(final, kept))
    net.forward(stream=2, keep_states=True)
    assert all(not np.array_equal(a.numpy(), b) for a, b in zip(net.states[1:], kept[1:]))      # the second block's, behind a dropout


@gpu
@pytest.mark.parametrize("blocks,heads", [(1, 1), (2, 3), (3, 4)])
def test_decays_stay_decays(rocm, blocks, heads):
    """gradients that push every second logarithm up and the others down, in eager updates and in a graph's: none is above zero, the others are where Adam alone takes them"""
    c, p, x, resets, net, tolerance, rng = case(rocm, 7, 4, 2, 12 * heads, heads, 1, blocks)
    adam, names = capi.adam_parameters(alpha=3e-3), [f"log_decay{l}" for l in range(blocks)]
    up = np.arange(heads) % 2 == 0
    flat = np.zeros(net.total, np.float32)
    for n in names:
        flat[net.offsets[n]:net.offsets[n] + heads] = np.where(up, -1.0, 1.0)
    net.grads.upload(flat)
    before = {n: v.numpy() for n, v in net.param_views.items()}
    lib, h = rocm.device.lib, rocm.device.handle
    for i in range(20):
        net.update(adam)
    rocm.sync()
    assert lib.rlt_rocm_graph_begin_capture(h) == 0
    net.update(adam)
    graph = C.c_void_p()
    assert lib.rlt_rocm_graph_end_capture(h, C.byref(graph)) == 0
    for i in range(5):
        assert lib.rlt_rocm_graph_launch(h, graph) == 0
        rocm.sync()
        assert all(np.all(net.param_views[n].numpy() <= 0.0) for n in names)
    lib.rlt_rocm_graph_destroy(h, graph)
    for n in names:
        after = net.param_views[n].numpy()
        risen = before[n].astype(np.float64) + 25 * 3e-3      # a gradient of one sign and size moves a parameter by alpha an update, up to the epsilon beside its root
        assert np.all(np.abs(after[up] - np.minimum(risen[up], 0.0)) <= 1e-4) and np.all(np.abs(after[~up] - (before[n][~up] - 25 * 3e-3)) <= 1e-4)
        assert np.any(after[up] == 0.0) or heads == 1      # (a single head's decay starts too far below)
    assert all(np.array_equal(net.param_views[n].numpy(), before[n]) for n in before if n not in names)

"""The stack of blocks that runs the causal convolution, the selective scan, norms, dropout and both optimisers together (builders.SelectiveBlocks), against its formulas in 64 bits.

Bounds, set before the first run, as those of test_rocm_sequence_blocks: what leaves a norm is of order one; a value passes, per block, four dense products (inner or width + 4 roundings each), the convolution (12 + 1.1 taps), the scan (4 steps + 16 E + 64 + channels + states, where the decays'
exponents add up to E, whose products of a size that counts have E below 16) and two norms (128 each). Sums over magnitudes are at most 8 times what comes out of them at these sizes. A gradient meets those of the forward values and its own twice: three times that along a random direction, where it is
compared with the difference quotient of the 64-bit loss."""
import ctypes as C

import numpy as np
import pytest

import helpers
from helpers import capi
from test_rocm_dropout import kept
from test_rocm_muon import orthogonalised
from test_rocm_sequence_blocks import normalised

gpu = pytest.mark.gpu
SelectiveBlocks = helpers.package().builders.SelectiveBlocks


def silu(z):
    return z / (1 + np.exp(-z))


def reference(c, p, x, reset, stream=None):
    """h after the last block, all steps"""
    S, B, W = x.shape
    n, H, N, R, K = c["inner"], c["heads"], c["states"], c["rank"], c["taps"]
    D = n // H
    h = normalised(x, c["norm"], p["input_weights"], p["input_biases"])
    for l in range(c["blocks"]):
        projected = h @ p[f"in_w{l}"].T + p[f"in_b{l}"]
        u, gate = projected[..., :n], projected[..., n:]
        window, conv = np.zeros((K - 1, B, n)), np.zeros_like(u)
        for t in range(S):
            window = np.where(reset[t].astype(bool)[None, :, None], 0.0, window)
            full = np.concatenate([window, u[t][None]])
            conv[t] = silu((p[f"taps{l}"].T[:, None] * full).sum(0) + p[f"tap_b{l}"])
            window = full[1:]
        parts = conv @ p[f"x_w{l}"].T + p[f"x_b{l}"]
        delta = np.logaddexp(parts[..., :R] @ p[f"dt_w{l}"].T + p[f"dt_b{l}"], 0.0).reshape(S, B, H, D)
        b, read = parts[..., R:R + H * N].reshape(S, B, H, N), parts[..., R + H * N:].reshape(S, B, H, N)
        rates, state, o = np.exp(p[f"log_rates{l}"]).reshape(H, D, N), np.zeros((B, H, D, N)), np.zeros((S, B, H, D))
        v = conv.reshape(S, B, H, D)
        for t in range(S):
            state = np.where(reset[t].astype(bool)[:, None, None, None], 0.0, state) * np.exp(-rates * delta[t][..., None]) + (delta[t] * v[t])[..., None] * b[t][:, :, None]
            o[t] = (state * read[t][:, :, None]).sum(-1) + p[f"skip{l}"].reshape(H, D) * v[t]
        out = (o.reshape(S, B, n) * silu(gate)) @ p[f"out_w{l}"].T + p[f"out_b{l}"]
        if stream is not None and c["dropout"] > 0:
            threshold = int(np.float32(c["dropout"]) * 65536 + 0.5)
            out = np.where(kept(S * B * W, c["dropout"], c["seed"], stream + l).reshape(out.shape), out * (65536 / (65536 - threshold)), 0.0)
        x = x + p[f"residual_scale{l}"] * normalised(out, c["norm"], p[f"branch_weights{l}"], p[f"branch_biases{l}"])
        h = normalised(x, c["norm"], p[f"output_weights{l}"], p[f"output_biases{l}"])
    return h


def case(rocm, seed, steps, batch, width, inner, heads, states, rank, taps, blocks, dropout=0.0, norm="rms", resets=0.05):
    rng = np.random.default_rng(seed)
    sizes = dict(width=width, inner=inner, heads=heads, states=states, rank=rank, taps=taps, blocks=blocks)
    params = SelectiveBlocks.random(rng, **sizes)
    for name in params:      # no parameter at a value that hides it
        if params[name].ndim == 1 and not name.startswith("dt_b"):
            params[name] = (params[name] + rng.uniform(-0.2, 0.2, params[name].shape)).astype(np.float32)
    c = dict(sizes, steps=steps, batch=batch, dropout=dropout, seed=seed, norm=norm)
    x = rng.standard_normal((steps, batch, width)).astype(np.float32)
    reset = (rng.random((steps, batch)) < resets).astype(np.uint8)
    net = SelectiveBlocks(rocm, params, **c)
    net.x.upload(x)
    net.reset.upload(reset)
    tolerance = blocks * 8 * (4 * (max(width, inner) + 4) + 12 + 2 * taps + 4 * steps + 16 * 16 + 64 + inner // heads + states + 272) * 2.0 ** -24
    return c, {n: a.astype(np.float64) for n, a in params.items()}, x.astype(np.float64), reset, net, tolerance, rng


CASES = [  # steps, batch, width, inner, heads, states, rank, taps, blocks, dropout, norm
    (70, 5, 32, 64, 1, 16, 4, 4, 2, 0.1, "rms"), (130, 3, 24, 48, 2, 8, 3, 3, 1, 0.0, "layer"), (1, 9, 20, 40, 1, 4, 2, 2, 2, 0.3, "rms"), (400, 1, 16, 33, 1, 11, 5, 4, 1, 0.0, "rms"), (9, 4, 64, 128, 4, 20, 8, 8, 1, 0.5, "layer")]


@gpu
@pytest.mark.parametrize("sizes", CASES)
def test_sequences_and_gradients(rocm, sizes):
    print("case", sizes, flush=True)
    c, p, x, reset, net, tolerance, rng = case(rocm, sum(sizes[:4]), *sizes)
    got = net.forward(stream=40).numpy().reshape(x.shape)
    want = reference(c, p, x, reset, 40)
    assert np.max(np.abs(got - want)) <= tolerance * np.max(np.abs(want))
    d = rng.standard_normal(x.shape).astype(np.float32)
    net.zero_gradient()
    net.backward(rocm.array(d.reshape(-1, c["width"])))
    loss = lambda p, x: np.sum(d * reference(c, p, x, reset, 40))
    gradients = {n: v.numpy().astype(np.float64) for n, v in net.grad_views.items()}
    for name, g in list(gradients.items()) + [("x", net.d_stream.numpy().astype(np.float64).reshape(x.shape))]:
        along = rng.choice([-1.0, 1.0], g.shape)
        step = 1e-6
        def at(s):
            return loss(p, x + s * along) if name == "x" else loss({**p, name: p[name] + s * along}, x)
        quotient = (at(step) - at(-step)) / (2 * step)
        assert abs(np.sum(g * along) - quotient) <= (3 * tolerance + 1e-6) * max(np.linalg.norm(g) * np.linalg.norm(along), abs(quotient)), name
    before = net.grads.numpy()
    net.backward(rocm.array(d.reshape(-1, c["width"])))
    assert np.allclose(net.grads.numpy(), 2 * before, rtol=1e-4, atol=1e-4 * np.max(np.abs(before)))      # added to


@gpu
@pytest.mark.parametrize("sizes", CASES)
def test_steps_give_what_sequences_give(rocm, sizes):
    print("case", sizes, flush=True)
    c, p, x, reset, net, tolerance, rng = case(rocm, sum(sizes[:4]), *sizes)
    want = net.forward(dropout=False).numpy().reshape(x.shape)
    final = [s.numpy() for s in net.states + net.windows]
    for s in net.states + net.windows:
        s.upload(np.zeros(s.shape, np.float32))
    for t in range(c["steps"]):
        net.step_x.upload(x[t].astype(np.float32))
        net.step_reset.upload(reset[t])
        got = net.step().numpy()
        assert np.max(np.abs(got - want[t])) <= 2 * tolerance * np.max(np.abs(want)), t
    for a, b in zip(net.states + net.windows, final):
        assert np.max(np.abs(a.numpy() - b)) <= 2 * tolerance * max(np.max(np.abs(b)), 1.0)


@gpu
def test_training_leaves_the_rollouts_states_alone(rocm):
    c, p, x, reset, net, tolerance, rng = case(rocm, 5, 20, 3, 16, 32, 1, 16, 2, 4, 2, dropout=0.1)
    net.forward(dropout=False)
    before = [s.numpy() for s in net.states + net.windows]
    net.forward(stream=2)
    net.zero_gradient()
    net.backward(rocm.array(rng.standard_normal((60, 16)).astype(np.float32)))
    assert all(np.array_equal(a, b.numpy()) for a, b in zip(before, net.states + net.windows))


@gpu
def test_updates_by_both_optimisers_in_a_graph(rocm):
    """forward, backward and update captured once; every replay is what the same calls do eagerly, and the first update of the matrices is the definition's"""
    c, p, x, reset, net, tolerance, rng = case(rocm, 9, 40, 4, 32, 64, 1, 16, 4, 4, 2)
    twin = case(rocm, 9, 40, 4, 32, 64, 1, 16, 4, 4, 2)[4]
    adam, muon = capi.adam_parameters(alpha=1e-3), capi.MuonParameters(alpha=1 / 64, momentum=15 / 16, weight_decay=1 / 8, epsilon=2.0 ** -23, nesterov=1, iterations=5)
    d = rocm.array(rng.standard_normal((160, 32)).astype(np.float32))

    def train(n):
        n.zero_gradient()
        n.forward(stream=0)
        n.backward(d)
        n.update(adam, muon)
    train(twin)
    for name, view in twin.param_views.items():
        if name.rstrip("0123456789") in SelectiveBlocks.MATRICES:
            g = twin.grad_views[name].numpy().astype(np.float64)
            rows, cols = g.shape
            want = (1 - 1 / 512) * p[name] - np.sqrt(max(1.0, rows / cols)) / 64 * orthogonalised(g * (1 + 15 / 16), 2.0 ** -23, 5)
            off = (view.numpy() - want) * 64
            assert np.linalg.norm(off, 2) <= 960 * 2.0 ** -24 * (rows ** 0.5 + cols ** 0.5) * 200 * np.sqrt(max(1.0, rows / cols)) + 3 * 2.0 ** -24 * 64 * np.linalg.norm(p[name])
            assert np.allclose(twin.m.numpy()[twin.offsets[name]:twin.offsets[name] + g.size].reshape(g.shape), g, rtol=1e-6, atol=0)
    lib, h = rocm.device.lib, rocm.device.handle
    train(net)
    rocm.sync()
    assert np.array_equal(net.params.numpy(), twin.params.numpy())
    assert lib.rlt_rocm_graph_begin_capture(h) == 0
    train(net)
    graph = C.c_void_p()
    assert lib.rlt_rocm_graph_end_capture(h, C.byref(graph)) == 0
    for _ in range(3):
        train(twin)      # eager work between the replays
        assert lib.rlt_rocm_graph_launch(h, graph) == 0
        rocm.sync()
        assert np.array_equal(net.params.numpy(), twin.params.numpy()) and np.isfinite(net.params.numpy()).all()
    lib.rlt_rocm_graph_destroy(h, graph)


@gpu
@pytest.mark.parametrize("with_muon", [False, True])
def test_training_runs(rocm, with_muon):
    c, p, x, reset, net, tolerance, rng = case(rocm, 3, 24, 16, 32, 64, 1, 16, 4, 4, 2, dropout=0.05)
    adam, muon = capi.adam_parameters(alpha=1e-3), capi.MuonParameters(alpha=1e-2, momentum=0.95, weight_decay=0.0, epsilon=1e-7, nesterov=1, iterations=5)
    d = rocm.zeros((24 * 16, 32))
    for i in range(10):
        out = net.forward(stream=2 * i).numpy()
        d.upload((out - x.reshape(out.shape)).astype(np.float32) / out.size)
        net.zero_gradient()
        net.backward(d)
        net.update(adam, muon if with_muon else None)
    assert np.isfinite(net.params.numpy()).all() and not np.array_equal(net.params.numpy(), np.concatenate([a.ravel() for a in p.values()]).astype(np.float32)[:net.total])


@gpu
@pytest.mark.parametrize("with_muon", [False, True])
def test_every_tensor_moves_as_its_optimiser_says(rocm, with_muon):
    """Two updates in a row by the definitions in 64 bits. Adam: what its bias corrections lose, 2 u / (1 - beta_2) of them, and some ten roundings of the update; Muon: as in test_rocm_muon"""
    c, p, x, reset, net, tolerance, rng = case(rocm, 15, 24, 6, 32, 64, 1, 16, 4, 4, 2)
    adam, muon = capi.adam_parameters(alpha=1e-3), capi.MuonParameters(alpha=1 / 64, momentum=15 / 16, weight_decay=1 / 8, epsilon=2.0 ** -23, nesterov=1, iterations=5)
    u, one, two = 2.0 ** -24, np.float64(np.float32(0.9)), np.float64(np.float32(0.999))
    m, v = {n: np.zeros(a.shape) for n, a in p.items()}, {n: np.zeros(a.shape) for n, a in p.items()}
    for age in (1, 2):
        out = net.forward(stream=0).numpy()
        net.zero_gradient()
        net.backward(rocm.array((out - 0.5 * x.reshape(out.shape)).astype(np.float32)))
        before = {n: a.numpy().astype(np.float64) for n, a in net.param_views.items()}
        net.update(adam, muon if with_muon else None)
        for n, a in net.param_views.items():
            g, after = net.grad_views[n].numpy().astype(np.float64), a.numpy().astype(np.float64)
            assert np.any(after != before[n]), n
            if with_muon and n.rstrip("0123456789") in SelectiveBlocks.MATRICES:
                rows, cols = g.shape
                m[n] = 15 / 16 * m[n] + g
                scale = np.sqrt(max(1.0, rows / cols)) / 64
                want = (1 - 1 / 512) * before[n] - scale * orthogonalised(g + 15 / 16 * m[n], 2.0 ** -23, 5)
                assert np.linalg.norm((after - want) / scale, 2) <= 960 * u * (rows ** 0.5 + cols ** 0.5) * 200 + 3 * u / scale * np.linalg.norm(before[n]), n
            else:
                m[n], v[n] = one * m[n] + (1 - one) * g, two * v[n] + (1 - two) * g * g
                step = 1e-3 * m[n] / (1 - one ** age) / (np.sqrt(np.maximum(v[n] / (1 - two ** age), 1e-7)) + 1e-7)
                slack = 1e-3 * (np.abs(one * m[n]) + np.abs(g)) / (1 - one ** age) / (np.sqrt(np.maximum(v[n] / (1 - two ** age), 1e-7)) + 1e-7)
                assert np.all(np.abs(after - (before[n] - step)) <= (2 * u / (1 - two) + 2 * u / (1 - one) + 16 * u) * slack + 2 * u * np.abs(before[n])), n

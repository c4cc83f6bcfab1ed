"""The stack of blocks that runs norms, linear attention and dropout together (builders.SequenceBlocks), against its formulas in 64 bits.

Bounds, set before the first run. What leaves a norm is of order one; a value passes, per block, two dense products (width + 4 roundings each), the attention (4 steps + channels + 16) and two norms (128 each). Sums over
magnitudes are at most 8 times what comes out of them at these sizes: blocks * 8 * (2 (width + 4) + 4 steps + channels + 272) * 2^-24 of the largest output. A gradient meets those of the forward values that it is formed from and
its own twice (each product has two gradients): three times that, of the gradient's norm, along a random direction, where it is compared with the difference quotient of the 64-bit loss."""
import numpy as np
import pytest

import helpers
from helpers import capi
from test_rocm_dropout import kept

gpu = pytest.mark.gpu
SequenceBlocks = helpers.package().builders.SequenceBlocks


def normalised(x, kind, w, b, epsilon=1e-5):
    x = x - x.mean(-1, keepdims=True) if kind == "layer" else x
    return x / np.sqrt((x ** 2).mean(-1, keepdims=True) + epsilon) * w + b


def reference(c, p, x, reset, stream=None):
    """h after the last block, all steps"""
    S, B, W = x.shape
    H, K = c["heads"], c["kv_heads"]
    d, group = W // H, H // K
    h = normalised(x, c["norm"], p["input_weights"], p["input_biases"])
    for l in range(c["blocks"]):
        q, k, v, gate = np.split(h @ p[f"in_w{l}"].T + p[f"in_b{l}"], [W, W + K * d, W + 2 * K * d], -1)
        q, k, v = q.reshape(S, B, H, d), np.repeat(k.reshape(S, B, K, d), group, 2), np.repeat(v.reshape(S, B, K, d), group, 2)
        state, o = np.zeros((B, H, d, d)), np.zeros((S, B, H, d))
        decay = np.exp(p[f"log_decay{l}"])[None, :, None, None]
        for t in range(S):
            state = np.where(reset[t].astype(bool)[:, None, None, None], 0.0, state * decay) + k[t][..., :, None] * v[t][..., None, :]
            o[t] = np.einsum("bhi,bhij->bhj", q[t], state) * d ** -0.5
        out = o.reshape(S, B, W) @ p[f"out_w{l}"].T + p[f"out_b{l}"]
        if stream is not None and c["dropout"] > 0:
            threshold = int(np.float32(c["dropout"]) * 65536 + 0.5)
            out = np.where(kept(S * B * W, c["dropout"], c["seed"], stream + l).reshape(out.shape), out * (65536 / (65536 - threshold)), 0.0)
        x = x + p[f"residual_scale{l}"] / (1 + np.exp(-gate)) * normalised(out, c["norm"], p[f"branch_weights{l}"], p[f"branch_biases{l}"])
        h = normalised(x, c["norm"], p[f"output_weights{l}"], p[f"output_biases{l}"])
    return h


def case(rocm, seed, steps, batch, width, heads, kv_heads, blocks, dropout=0.0, norm="rms", resets=0.05):
    rng = np.random.default_rng(seed)
    params = SequenceBlocks.random(rng, width, heads, kv_heads, blocks)
    for name in params:      # no parameter at a value that hides it
        if params[name].ndim == 1 and not name.startswith("log_decay"):
            params[name] = (params[name] + rng.uniform(-0.2, 0.2, params[name].shape)).astype(np.float32)
    c = dict(steps=steps, batch=batch, width=width, heads=heads, kv_heads=kv_heads, blocks=blocks, dropout=dropout, seed=seed, norm=norm)
    x = rng.standard_normal((steps, batch, width)).astype(np.float32)
    reset = (rng.random((steps, batch)) < resets).astype(np.uint8)
    net = SequenceBlocks(rocm, params, **c)
    net.x.upload(x)
    net.reset.upload(reset)
    tolerance = blocks * 8 * (2 * (width + 4) + 4 * steps + width // heads + 272) * 2.0 ** -24
    return c, {n: a.astype(np.float64) for n, a in params.items()}, x.astype(np.float64), reset, net, tolerance, rng


CASES = [(70, 5, 48, 3, 1, 2, 0.1, "rms"), (130, 3, 64, 2, 2, 1, 0.0, "layer"), (1, 9, 20, 4, 2, 2, 0.3, "rms"), (33, 2, 36, 2, 1, 2, 0.5, "layer"), (9, 4, 128, 1, 1, 1, 0.0, "rms")]


@gpu
@pytest.mark.parametrize("steps,batch,width,heads,kv_heads,blocks,dropout,norm", CASES)
def test_sequences_and_gradients(rocm, steps, batch, width, heads, kv_heads, blocks, dropout, norm):
    print("case", steps, batch, width, heads, kv_heads, blocks, dropout, norm, flush=True)
    c, p, x, reset, net, tolerance, rng = case(rocm, steps + width, steps, batch, width, heads, kv_heads, blocks, dropout, norm)
    got = net.forward(stream=40).numpy().reshape(x.shape)
    want = reference(c, p, x, reset, 40)
    assert np.max(np.abs(got - want)) <= tolerance * np.max(np.abs(want))
    d = rng.standard_normal(x.shape).astype(np.float32)
    net.zero_gradient()
    net.backward(rocm.array(d.reshape(-1, width)), stream=40)
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
    net.backward(rocm.array(d.reshape(-1, width)), stream=40)
    assert np.allclose(net.grads.numpy(), 2 * before, rtol=1e-4, atol=1e-4 * np.max(np.abs(before)))      # added to


@gpu
@pytest.mark.parametrize("steps,batch,width,heads,kv_heads,blocks,dropout,norm", CASES)
def test_steps_give_what_sequences_give(rocm, steps, batch, width, heads, kv_heads, blocks, dropout, norm):
    print("case", steps, batch, width, heads, kv_heads, blocks, dropout, norm, flush=True)
    c, p, x, reset, net, tolerance, rng = case(rocm, steps + width, steps, batch, width, heads, kv_heads, blocks, dropout, norm)
    want = net.forward(dropout=False).numpy().reshape(x.shape)
    final = [s.numpy() for s in net.states]
    for s in net.states:
        s.upload(np.zeros(s.shape, np.float32))
    for t in range(steps):
        net.step_x.upload(x[t])
        net.step_reset.upload(reset[t])
        got = net.step().numpy()
        assert np.max(np.abs(got - want[t])) <= 2 * tolerance * np.max(np.abs(want)), t
    for a, b in zip(net.states, final):
        assert np.max(np.abs(a.numpy() - b)) <= 2 * tolerance * max(np.max(np.abs(b)), 1.0)


@gpu
def test_training_recalls_an_earlier_step(rocm):
    """Adam on a target that only memory reaches: the input of three steps ago. The loss of the best answer without memory is that of zeros, the targets' variance of 1, of which a mean over ten batches of 5,376 values
    is off by sqrt(2 / 53760) = 0.6 %: a loss below 1 by five of these has used the states."""
    c, p, x, reset, net, tolerance, rng = case(rocm, 3, 24, 64, 32, 2, 2, 2, dropout=0.05, resets=0.0)
    adam = capi.adam_parameters(alpha=3e-3)
    d = rocm.zeros((24 * 64, 32))
    losses = []
    for i in range(300):
        x = np.random.default_rng(i).standard_normal((24, 64, 32)).astype(np.float32)
        target = np.zeros_like(x); target[3:, :, :4] = x[:-3, :, :4]
        weight = np.zeros_like(x); weight[3:, :, :4] = 1
        net.x.upload(x)
        error = weight * (net.forward(stream=i * 2, reset=False).numpy().reshape(x.shape) - target)
        losses.append(np.sum(error ** 2) / np.sum(weight))
        d.upload((error / np.sum(weight) * 2).reshape(-1, 32))
        net.zero_gradient()
        net.backward(d, stream=i * 2, reset=False)
        net.update(adam)
    print("loss", losses[0], np.mean(losses[-10:]), flush=True)
    assert np.mean(losses[-10:]) < 1 - 5 * (2 / 53760) ** 0.5

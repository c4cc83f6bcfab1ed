"""Workloads of the sequence-block operators: linear attention with a decay for each head (training, prompts, single steps), the norms around a block with its
gate and residual scale, and dropout whose mask is drawn from counters.

listed() are sizes of this repository's recurrent and vectorised workloads next to generic ones; draw() spreads over the ranges that they stand for. prepare()
lays a case's tensors out in GPU memory, run() makes one pass: with `own` through the C ABI, otherwise in elementary torch operations in 32 bits. exact() computes
a case from the definitions in 64 bits (attention as the recurrence, step by step).
"""
import ctypes as C
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

# ------------------------------------------------------------------ the cases


def listed():
    return [
        # acting: one step of a small policy's layer in 64 environments, between two environment steps
        dict(name="attention_step_64", kind="step", type="float32", rows=64, heads=2, kv_heads=2, key=32, value=32),
        # vectorised collection / serving: one token for each of 4,096 rows, whose states fill half a gigabyte
        dict(name="attention_step_4096", kind="step", type="bfloat16", rows=4096, heads=8, kv_heads=8, key=64, value=64),
        # a training step of the recurrent workloads' shape (64 steps x 1,024 sequences, width 64) with episode ends inside the sequences: forward + backward
        dict(name="attention_train_64x1024", kind="train", type="float32", steps=64, rows=1024, heads=2, kv_heads=2, key=32, value=32, resets=True, ragged=False),
        # sequences of different lengths, some empty, odd widths, keys and values shared by three heads each: forward + backward
        dict(name="attention_train_ragged", kind="train", type="float32", steps=333, rows=37, heads=6, kv_heads=2, key=24, value=41, resets=True, ragged=True),
        # long sequences in 16 bits, few of them: forward + backward
        dict(name="attention_train_8192", kind="train", type="bfloat16", steps=8192, rows=4, heads=16, kv_heads=16, key=128, value=128, resets=False, ragged=False),
        # one long prompt: outputs and the state that single steps go on from
        dict(name="attention_prompt_16384", kind="prompt", type="bfloat16", steps=16384, rows=1, heads=16, kv_heads=16, key=128, value=128, resets=False, ragged=False),
        # the norms around a small policy's block over one batch of 256
        dict(name="norm_256x256", kind="norm", type="float32", rows=256, dim=256, norm="rms"),
        # gradients of a wide block over 16,384 tokens
        dict(name="norm_backward_16384x4096", kind="norm_backward", type="bfloat16", rows=16384, dim=4096, norm="rms"),
        # gradients with mean, deviation and biases over a batch and a width that fill no tile evenly
        dict(name="norm_backward_4001x1000", kind="norm_backward", type="float32", rows=4001, dim=1000, norm="layer"),
        # dropout between the layers of a critic over one batch of 256
        dict(name="dropout_256x256", kind="dropout", type="float32", rows=256, cols=256, rate=0.1, residual=False),
        # rows that no vector divides, added to the residual stream
        dict(name="dropout_4001x1023", kind="dropout", type="float32", rows=4001, cols=1023, rate=0.5, residual=True),
        # a block's output over 32,768 tokens
        dict(name="dropout_32768x4096", kind="dropout", type="bfloat16", rows=32768, cols=4096, rate=0.1, residual=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["step", "train", "train", "prompt", "norm", "norm_backward", "dropout"])
    dtype = rng.choice(["float32", "bfloat16"])
    if kind in ("step", "train", "prompt"):
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 1, 1, 2, 3])
        key = rng.choice([16, 32, 64, 64, 128, 128, rng.randint(8, 128)])
        value = key if rng.random() < 0.6 else rng.randint(8, 128)
        case = dict(kind=kind, type=dtype, heads=heads, kv_heads=kv_heads, key=key, value=value)
        if kind == "step":
            return dict(case, rows=min(_log(rng, 16, 4096), 4096 * 8 * 64 * 64 // (heads * key * value)))
        tokens = _log(rng, 64, 16384 * 16 * 128 // (heads * max(key, value)))
        steps = min(_log(rng, 1, 16384), tokens)
        rows = max(1, min(tokens // steps, 4096 * 8 * 64 * 64 // (heads * key * value)))
        return dict(case, steps=steps, rows=rows, resets=rng.random() < 0.5, ragged=rng.random() < 0.5)
    if kind == "dropout":
        cols = _log(rng, 16, 8192)
        return dict(kind=kind, type=dtype, rows=_log(rng, 64, max(64, min(65536, (1 << 26) // cols))), cols=cols, rate=rng.choice([0.01, 0.1, 0.5]), residual=rng.random() < 0.5)
    dim = _log(rng, 16, 8192)
    return dict(kind=kind, type=dtype, rows=_log(rng, 64, max(64, min(65536, (1 << 25) // dim))), dim=dim, norm=rng.choice(["rms", "layer"]))


def work(case):
    """Each input once, each output once; the recurrence's products (two per step forward: the state's update and its reading)."""
    c = case
    if c["kind"] == "dropout":
        n = c["rows"] * c["cols"]
        return {"bytes": n * _size(c) * (3 if c["residual"] else 2), "flops": n}
    if c["kind"] == "norm":
        n = c["rows"] * c["dim"]
        return {"bytes": 5 * n * _size(c), "flops": 12 * n}
    if c["kind"] == "norm_backward":
        n = c["rows"] * c["dim"]
        return {"bytes": 8 * n * _size(c), "flops": 30 * n}
    state, pairs = c["key"] * c["value"], c["rows"] * c["heads"]
    if c["kind"] == "step":
        per_row = c["heads"] * (c["key"] + c["value"]) + c["kv_heads"] * (c["key"] + c["value"])
        return {"bytes": 8 * pairs * state + c["rows"] * per_row * _size(c), "flops": 4 * pairs * state}
    queries, values = c["heads"] * c["key"], c["heads"] * c["value"]
    shared = c["kv_heads"] * (c["key"] + c["value"])
    tokens = c["steps"] * c["rows"]
    bytes_, flops = tokens * (queries + shared + values) * _size(c) + 4 * pairs * state, 4 * tokens * c["heads"] * state
    if c["kind"] == "train":
        bytes_ += tokens * (2 * queries + 2 * shared + values) * _size(c) + 4 * pairs * state
        flops += 12 * tokens * c["heads"] * state
    return {"bytes": bytes_, "flops": flops}


def _size(case):
    return 4 if case["type"] == "float32" else 2


# ------------------------------------------------------------------ inputs


def _type(case):
    return getattr(torch, case["type"])


def _log_decay(heads):
    """Decays from 7/8 to 511/512 per step, spread over the heads as memories of different reach are."""
    reach = torch.linspace(math.log(1 / 8), math.log(1 / 512), heads, dtype=torch.float64) if heads > 1 else torch.tensor([math.log(1 / 64)], dtype=torch.float64)
    return torch.log1p(-reach.exp()).float().cuda()


def _inputs(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)

    def randn(*shape, dtype=_type(case)):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)
    c, f32 = case, torch.float32
    if c["kind"] == "dropout":
        s = dict(x=randn(c["rows"], c["cols"]), seed=(seed * 7919 + 17) % (1 << 64), stream=((seed << 33) + 5) % (1 << 64))
        if c["residual"]:
            s["residual"] = randn(c["rows"], c["cols"])
        return s
    if c["kind"] in ("norm", "norm_backward"):
        r, d = c["rows"], c["dim"]
        s = dict(branch=randn(r, d), gate=randn(r, d), branch_weights=1 + 0.1 * randn(d, dtype=f32), output_weights=1 + 0.1 * randn(d, dtype=f32), scale=0.3 + 0.1 * randn(d, dtype=f32))
        if c["norm"] == "layer":
            s.update(branch_biases=0.1 * randn(d, dtype=f32), output_biases=0.1 * randn(d, dtype=f32))
        if c["kind"] == "norm":
            return dict(s, x=randn(r, d))
        return dict(s, y=(1.5 * randn(r, d, dtype=f32) + 0.1).to(_type(c)), d_y=randn(r, d), d_h=randn(r, d))
    h, hk, dk, dv = c["heads"], c["kv_heads"], c["key"], c["value"]
    lead = (c["rows"],) if c["kind"] == "step" else (c["steps"], c["rows"])
    s = dict(q=randn(*lead, h, dk), k=randn(*lead, hk, dk), v=randn(*lead, hk, dv), log_decay=_log_decay(h), state=randn(c["rows"], h, dk, dv, dtype=f32), scale=dk ** -0.5)
    if c["kind"] == "step":
        s["reset"] = (torch.rand(c["rows"], generator=g, device="cuda") < 0.02).to(torch.uint8)
        return s
    if c["resets"]:      # an episode ends every 50 steps
        s["reset"] = (torch.rand(lead, generator=g, device="cuda") < 0.02).to(torch.uint8)
    if c["ragged"]:
        s["lengths"] = torch.randint(0, c["steps"] + 1, (c["rows"],), generator=g, device="cuda").to(torch.int32)
    if c["kind"] == "train":
        s["d_output"], s["d_state"] = randn(*lead, h, dv), randn(c["rows"], h, dk, dv, dtype=f32)
    return s


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if own:
        s["run"] = _OWN[case["kind"]](s)
    torch.cuda.synchronize()      # torch filled the buffers on its stream, the library works on its own
    return s


def run(state):
    return state["run"]() if own else _PLAIN[state["case"]["kind"]](state)


# ------------------------------------------------------------------ through the framework

_device = None


def _handle():
    """The package and the library's handle of the GPU: one per process, as a program keeps it."""
    global _device
    if "rl_tools_amd" not in sys.modules:
        path = os.path.join(os.getcwd(), "rl-tools_amd")
        spec = importlib.util.spec_from_file_location("rl_tools_amd", os.path.join(path, "__init__.py"), submodule_search_locations=[path])
        module = importlib.util.module_from_spec(spec)
        sys.modules["rl_tools_amd"] = module
        spec.loader.exec_module(module)
    capi = sys.modules["rl_tools_amd"].capi
    if _device is None:
        _device = capi.Device(0)
    return capi, _device


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(device, name, *args):
    f, check, handle = getattr(device.lib, "rlt_rocm_" + name), device.check, device.handle

    def call():
        rc = f(handle, *args)
        if rc:
            check(rc)
    return call


def _view(capi, t):
    """[steps x rows x heads x channels], or [rows x heads x channels] for a single step"""
    strides = t.stride() if t.dim() == 4 else (0,) + t.stride()
    return C.byref(capi.HeadView(t.data_ptr(), strides[0], strides[1], strides[2]))


def _layer(capi, s):
    c = s["case"]
    rows = c["rows"]
    return capi.LinearAttention(log_decay=s["log_decay"].data_ptr(), scale=s["scale"], type=capi.TYPE[c["type"]], batch=rows, heads=c["heads"], kv_heads=c["kv_heads"], key_dim=c["key"],
                                value_dim=c["value"])


def _own_step(s):
    capi, device = _handle()
    layer = _layer(capi, s)
    out, state = torch.empty(s["v"].shape[:1] + (s["case"]["heads"], s["case"]["value"]), dtype=s["q"].dtype, device="cuda"), torch.empty_like(s["state"])
    step = _call(device, "linear_attention_step", C.byref(layer), _view(capi, s["q"]), _view(capi, s["k"]), _view(capi, s["v"]), _view(capi, out), _ptr(s["state"]), _ptr(state), _ptr(s["reset"]))

    def go():
        step()
        return {"output": out, "state": state}
    return go


def _own_attention(s):
    capi, device = _handle()
    c, layer = s["case"], _layer(capi, s)
    out, state = torch.empty((c["steps"], c["rows"], c["heads"], c["value"]), dtype=s["q"].dtype, device="cuda"), torch.empty_like(s["state"])
    train = c["kind"] == "train"
    nbytes = max(device.lib.rlt_rocm_linear_attention_workspace_bytes(C.byref(layer), c["steps"], k) for k in range(1 + train))
    s["workspace"] = torch.empty(max(nbytes, 4), dtype=torch.uint8, device="cuda")
    q, k, v, tail = _view(capi, s["q"]), _view(capi, s["k"]), _view(capi, s["v"]), (_ptr(s.get("reset")), _ptr(s.get("lengths")), c["steps"], s["workspace"].data_ptr(), nbytes)
    forward = _call(device, "linear_attention_forward", C.byref(layer), q, k, v, _view(capi, out), _ptr(s["state"]), _ptr(state), *tail)
    results = {"output": out, "state": state}
    if not train:
        def go():
            forward()
            return results
        return go
    d = {"d_" + n: torch.empty_like(s[n]) for n in ("q", "k", "v", "state", "log_decay")}
    backward = _call(device, "linear_attention_backward", C.byref(layer), q, k, v, _view(capi, s["d_output"]), _view(capi, d["d_q"]), _view(capi, d["d_k"]), _view(capi, d["d_v"]),
                     _ptr(s["state"]), _ptr(s["d_state"]), _ptr(d["d_state"]), _ptr(d["d_log_decay"]), 0, *tail)
    results.update(d)

    def both():
        forward()
        backward()
        return results
    return both


def _own_norm(s):
    capi, device = _handle()
    c = s["case"]
    d, backward = c["dim"], c["kind"] == "norm_backward"
    parameters = ["branch_weights", "output_weights", "scale"] + (["branch_biases", "output_biases"] if c["norm"] == "layer" else [])
    grads = {"d_" + n: torch.empty_like(s[n]) for n in parameters} if backward else {}
    at = lambda n: _ptr(s.get(n))  # noqa: E731
    to = lambda n: _ptr(grads.get(n))  # noqa: E731
    layer = capi.ResidualNorm(type=capi.TYPE[c["type"]], dim=d, branch_norm=capi.NORM[c["norm"]], output_norm=capi.NORM[c["norm"]], gate_activation=capi.ACT["sigmoid"], epsilon=1e-5,
                              branch_weights=at("branch_weights"), branch_biases=at("branch_biases"), output_weights=at("output_weights"), output_biases=at("output_biases"),
                              residual_scale=at("scale"), d_branch_weights=to("d_branch_weights"), d_branch_biases=to("d_branch_biases"), d_output_weights=to("d_output_weights"),
                              d_output_biases=to("d_output_biases"), d_residual_scale=to("d_scale"))
    if not backward:
        y, h = torch.empty_like(s["x"]), torch.empty_like(s["x"])
        call = _call(device, "residual_norm_forward", C.byref(layer), at("x"), d, at("branch"), d, at("gate"), d, _ptr(y), d, _ptr(h), d, c["rows"])
        results = {"y": y, "h": h}
    else:
        results = {n: torch.empty_like(s["y"]) for n in ("d_x", "d_branch", "d_gate")}
        nbytes = device.lib.rlt_rocm_residual_norm_workspace_bytes(C.byref(layer), c["rows"])
        s["workspace"] = torch.empty(max(nbytes, 4), dtype=torch.uint8, device="cuda")
        call = _call(device, "residual_norm_backward", C.byref(layer), at("branch"), d, at("gate"), d, at("y"), d, at("d_y"), d, at("d_h"), d, _ptr(results["d_x"]), d,
                     _ptr(results["d_branch"]), d, _ptr(results["d_gate"]), d, c["rows"], 0, s["workspace"].data_ptr(), nbytes)
        results.update(grads)

    def go():
        call()
        return results
    return go


def _own_dropout(s):
    capi, device = _handle()
    c = s["case"]
    y = torch.empty_like(s["x"])
    call = _call(device, "dropout", capi.TYPE[c["type"]], _ptr(s["x"]), c["cols"], _ptr(s.get("residual")), c["cols"], _ptr(y), c["cols"], c["rows"], c["cols"], c["rate"], s["seed"], s["stream"])

    def go():
        call()
        return y
    return go


_OWN = dict(step=_own_step, prompt=_own_attention, train=_own_attention, norm=_own_norm, norm_backward=_own_norm, dropout=_own_dropout)

# ------------------------------------------------------------------ plain forms


def _plain_step(s):
    c, group = s["case"], s["case"]["heads"] // s["case"]["kv_heads"]
    q, k, v = s["q"].float(), s["k"].float().repeat_interleave(group, 1), s["v"].float().repeat_interleave(group, 1)
    kept = torch.where(s["reset"].bool()[:, None, None, None], 0.0, s["state"] * s["log_decay"].exp()[:, None, None])
    state = kept + k[..., None] * v[..., None, :]
    out = s["scale"] * (q[..., None] * state).sum(2)
    return {"output": out.to(_type(c)), "state": state}


def _plain_attention(s):
    """In chunks of up to 64 steps: products within a chunk under the matrix of decays, and the state of the steps before it; only the states go chunk by chunk."""
    c = s["case"]
    t, b, h, group = c["steps"], c["rows"], c["heads"], c["heads"] // c["kv_heads"]
    size = min(64, t)
    n = -(-t // size)
    pad = n * size - t

    def chunks(x, repeat):      # [steps, rows, heads, d] -> [rows, heads, chunks, size, d] in 32 bits
        x = x.float().repeat_interleave(repeat, 2) if repeat > 1 else x.float()
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, 0, 0, pad)).permute(1, 2, 0, 3).reshape(b, h, n, size, x.shape[-1])
        return torch.where(valid[:, None, :, :, None], x, 0.0)

    def joined(x):
        return x.reshape(b, h, n * size, -1)[:, :, :t].permute(2, 0, 1, 3)

    at = torch.arange(size, device="cuda")
    lengths = s["lengths"].long() if "lengths" in s else torch.full((b,), t, device="cuda")
    count = (lengths[:, None] - size * torch.arange(n, device="cuda")).clamp(0, size)                                   # [rows, chunks] valid steps
    valid = at < count[:, :, None]
    episode = torch.zeros((b, n, size), dtype=torch.long, device="cuda")
    if "reset" in s:
        episode = torch.nn.functional.pad(s["reset"].long(), (0, 0, 0, pad)).t().reshape(b, n, size).cumsum(2)
    last = torch.where(count > 0, episode.gather(2, (count - 1).clamp(min=0)[:, :, None])[:, :, 0], 0)                      # the episode that the chunk ends in
    rate = s["log_decay"][:, None, None]
    lag = at[:, None] - at[None, :]
    within = (lag >= 0) & (episode[..., :, None] == episode[..., None, :])                                                  # [rows, chunks, size, size]
    decays = torch.where(within[:, None], torch.exp(rate * lag.clamp(min=0))[:, None], 0.0)                                 # [rows, heads, chunks, size, size]
    begin = torch.where(((episode == 0) & valid)[:, None], torch.exp(rate * (at + 1)), 0.0)[..., None]                      # weights of the state before the chunk
    left = (count[:, :, None] - 1 - at).clamp(min=0)
    end = torch.where(((episode == last[:, :, None]) & valid)[:, None], torch.exp(rate * left[:, None]), 0.0)[..., None]  # weights in the state after it
    keep = torch.where((last == 0)[:, None], torch.exp(s["log_decay"][:, None] * count[:, None]), 0.0)  # [rows, heads, chunks]

    q, k, v = chunks(s["q"], 1), chunks(s["k"], group), chunks(s["v"], group)
    scores = q @ k.transpose(-1, -2) * decays
    added = (k * end).transpose(-1, -2) @ v
    states, state = [], s["state"]
    for i in range(n):
        states.append(state)
        state = keep[:, :, i, None, None] * state + added[:, :, i]
    states = torch.stack(states, 2)
    out = s["scale"] * (scores @ v + (q * begin) @ states)
    results = {"output": joined(out).to(_type(c)), "state": state}
    if c["kind"] == "prompt":
        return results
    d = s["scale"] * chunks(s["d_output"], 1)
    d_scores = d @ v.transpose(-1, -2)
    weighted = d_scores * decays
    added = (q * begin).transpose(-1, -2) @ d
    d_states, d_state = [], s["d_state"]
    for i in reversed(range(n)):
        d_states.append(d_state)
        d_state = keep[:, :, i, None, None] * d_state + added[:, :, i]
    d_states = torch.stack(d_states[::-1], 2)
    d_q_before, d_k_after = (d @ states.transpose(-1, -2)) * begin, (v @ d_states.transpose(-1, -2)) * end
    d_k = weighted.transpose(-1, -2) @ q + d_k_after
    d_v = scores.transpose(-1, -2) @ d + (k @ d_states) * end
    d_rate = (lag * scores * d_scores).sum((0, 2, 3, 4)) + ((at + 1) * (q * d_q_before).sum(-1)).sum((0, 2, 3)) + (left[:, None] * (k * d_k_after).sum(-1)).sum((0, 2, 3)) \
        + (count[:, None] * keep * (states * d_states).sum((-1, -2))).sum((0, 2))
    shared = lambda x: joined(x).reshape(t, b, c["kv_heads"], group, -1).sum(3).to(_type(c))  # noqa: E731
    return dict(results, d_q=joined(weighted @ k + d_q_before).to(_type(c)), d_k=shared(d_k), d_v=shared(d_v), d_state=d_state, d_log_decay=d_rate)


def _plain_statistics(x, kind):
    """normalised x and 1 / deviation"""
    if kind == "layer":
        x = x - x.mean(1, keepdim=True)
    inverse = torch.rsqrt((x * x).mean(1, keepdim=True) + 1e-5)
    return x * inverse, inverse


def _plain_norm(s):
    c = s["case"]
    n, _ = _plain_statistics(s["branch"].float(), c["norm"])
    n = n * s["branch_weights"]
    if c["norm"] == "layer":
        n = n + s["branch_biases"]
    y = s["x"].float() + s["scale"] * (1 / (1 + torch.exp(-s["gate"].float()))) * n
    h = _plain_statistics(y, c["norm"])[0] * s["output_weights"]
    if c["norm"] == "layer":
        h = h + s["output_biases"]
    return {"y": y.to(_type(c)), "h": h.to(_type(c))}


def _plain_norm_gradient(d, x, inverse, kind):
    """gradient with respect to what a norm normalised; d: with respect to the normalised x"""
    d = d - x * (d * x).mean(1, keepdim=True) - (d.mean(1, keepdim=True) if kind == "layer" else 0.0)
    return d * inverse


def _plain_norm_backward(s):
    c, kind = s["case"], s["case"]["norm"]
    branch, branch_inverse = _plain_statistics(s["branch"].float(), kind)
    out, out_inverse = _plain_statistics(s["y"].float(), kind)
    d_h, gate = s["d_h"].float(), 1 / (1 + torch.exp(-s["gate"].float()))
    d_x = s["d_y"].float() + _plain_norm_gradient(d_h * s["output_weights"], out, out_inverse, kind)
    n = branch * s["branch_weights"]
    if kind == "layer":
        n = n + s["branch_biases"]
    d_n = d_x * s["scale"] * gate
    grads = dict(d_branch_weights=(d_n * branch).sum(0), d_output_weights=(d_h * out).sum(0), d_scale=(d_x * gate * n).sum(0))
    if kind == "layer":
        grads.update(d_branch_biases=d_n.sum(0), d_output_biases=d_h.sum(0))
    d_branch = _plain_norm_gradient(d_n * s["branch_weights"], branch, branch_inverse, kind)
    d_gate = d_x * s["scale"] * n * gate * (1 - gate)
    return dict(grads, d_x=d_x.to(_type(c)), d_branch=d_branch.to(_type(c)), d_gate=d_gate.to(_type(c)))


def _plain_words(seed, stream, groups):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC'11) on torch's 64-bit integers: [groups, 4] words; key = seed, counter = (group, stream)."""
    def product(a, b):      # high and low words of a 32 x 32 bit product, in steps that 63 bits hold
        t = a * (b & 0xFFFF)
        u = a * (b >> 16) + (t >> 16)
        return u >> 16, ((u & 0xFFFF) << 16) | (t & 0xFFFF)
    index = torch.arange(groups, device="cuda")
    c = [index & 0xFFFFFFFF, index >> 32, torch.full_like(index, stream & 0xFFFFFFFF), torch.full_like(index, (stream >> 32) & 0xFFFFFFFF)]
    key = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        (hi0, lo0), (hi1, lo1) = product(0xD2511F53, c[0]), product(0xCD9E8D57, c[2])
        c = [hi1 ^ c[1] ^ key[0], lo1, hi0 ^ c[3] ^ key[1], lo0]
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return torch.stack(c, 1)


def _plain_dropout(s):
    """Element i (row by row) goes by 16 bits: half i % 8 of group i / 8, the low half of a word first; it stays where they reach the threshold."""
    c, n = s["case"], s["x"].numel()
    words = _plain_words(s["seed"], s["stream"], -(-n // 8))
    halves = torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:n].reshape(s["x"].shape)
    threshold = int(c["rate"] * 65536 + 0.5)
    y = torch.where(halves >= threshold, s["x"].float() * (65536 / (65536 - threshold)), 0.0)
    if "residual" in s:
        y = s["residual"].float() + y
    return y.to(_type(c))


_PLAIN = dict(step=_plain_step, prompt=_plain_attention, train=_plain_attention, norm=_plain_norm, norm_backward=_plain_norm_backward, dropout=_plain_dropout)

# ------------------------------------------------------------------ in 64 bits


def exact(case, seed):
    s = _inputs(case, seed)
    return _EXACT[case["kind"]](case, s)


def _exact_attention(c, s):
    """The recurrence: S <- decay * S (nothing at a reset) + k^T v, o = scale * q S; its derivative by the decay's logarithm goes along as a second state; then back through time."""
    step = c["kind"] == "step"
    lead = (lambda x: x[None]) if step else (lambda x: x)
    group, heads = c["heads"] // c["kv_heads"], c["heads"]
    q, k, v = lead(s["q"]).double(), lead(s["k"]).double().repeat_interleave(group, 2), lead(s["v"]).double().repeat_interleave(group, 2)
    steps, rows = q.shape[:2]
    decay = s["log_decay"].double().exp()[None, :, None, None]
    reset = lead(s["reset"]).bool() if "reset" in s else torch.zeros((steps, rows), dtype=torch.bool, device="cuda")
    live = torch.arange(steps, device="cuda")[:, None] < (s["lengths"] if "lengths" in s else torch.full((rows,), steps, device="cuda"))[None]
    kept = torch.where(reset[..., None, None, None], torch.zeros_like(decay), decay)      # [steps, rows, heads, 1, 1]
    live = live[..., None, None, None]
    train = c["kind"] == "train"
    state = s["state"].double()
    slope = torch.zeros_like(state)
    out = torch.zeros((steps, rows, heads, c["value"]), dtype=torch.float64, device="cuda")
    if train:
        d = s["scale"] * lead(s["d_output"]).double()
        d_q, d_k, d_v = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        d_rate = torch.zeros(heads, dtype=torch.float64, device="cuda")
    for t in range(steps):
        if train:
            slope = torch.where(live[t], kept[t] * (slope + state), slope)
        state = torch.where(live[t], kept[t] * state + k[t][..., :, None] * v[t][..., None, :], state)
        out[t] = torch.where(live[t][..., 0], s["scale"] * (q[t][..., :, None] * state).sum(2), 0.0)
        if train:
            d_q[t] = torch.where(live[t][..., 0], (state * d[t][..., None, :]).sum(3), 0.0)
            d_rate += torch.where(live[t], q[t][..., :, None] * slope * d[t][..., None, :], 0.0).sum((0, 2, 3))
    results = {"output": out[0] if step else out, "state": state}
    if not train:
        return results
    grad = s["d_state"].double()
    d_rate += (grad * slope).sum((0, 2, 3))
    for t in reversed(range(steps)):
        here = grad + q[t][..., :, None] * d[t][..., None, :]
        d_k[t] = torch.where(live[t][..., 0], (here * v[t][..., None, :]).sum(3), 0.0)
        d_v[t] = torch.where(live[t][..., 0], (here * k[t][..., :, None]).sum(2), 0.0)
        grad = torch.where(live[t], kept[t] * here, grad)
    shared = lambda x: x.reshape(steps, rows, c["kv_heads"], group, -1).sum(3)  # noqa: E731
    return dict(results, d_q=d_q, d_k=shared(d_k), d_v=shared(d_v), d_state=grad, d_log_decay=d_rate)


def _exact_norm(c, s):
    """By differentiation of the definition in 64 bits where gradients are asked for: autograd over rows' formulas."""
    d = {n: (t.double() if isinstance(t, torch.Tensor) else t) for n, t in s.items()}
    layer = c["norm"] == "layer"

    def norm(x, w, b):
        centred = x - x.mean(-1, keepdim=True) if layer else x
        x = centred / ((centred ** 2).mean(-1, keepdim=True) + 1e-5).sqrt() * w
        return x + b if layer else x
    if c["kind"] == "norm":
        y = d["x"] + d["scale"] * torch.sigmoid(d["gate"]) * norm(d["branch"], d["branch_weights"], d.get("branch_biases"))
        return {"y": y, "h": norm(y, d["output_weights"], d.get("output_biases"))}
    names = ["branch_weights", "output_weights", "scale"] + (["branch_biases", "output_biases"] if layer else [])
    parameters = {n: d[n].requires_grad_() for n in names}
    results = {"d_" + n: torch.zeros_like(d[n]).detach() for n in names}
    parts = {n: [] for n in ("d_x", "d_branch", "d_gate")}
    size = max(1, (1 << 24) // c["dim"])
    for at in range(0, c["rows"], size):      # some rows at a time: autograd keeps what it passes over
        rows = slice(at, at + size)
        branch, gate, y = (d[n][rows].clone().requires_grad_() for n in ("branch", "gate", "y"))
        w = lambda n: parameters.get(n)  # noqa: E731
        # the gradient that reaches the residual stream: its own and the output norm's
        h = norm(y, w("output_weights"), w("output_biases"))
        first = [y] + [parameters[n] for n in names if n.startswith("output")]
        got = torch.autograd.grad(h, first, d["d_h"][rows])
        d_x = d["d_y"][rows] + got[0]
        for n, g in zip([n for n in names if n.startswith("output")], got[1:]):
            results["d_" + n] += g
        added = w("scale") * torch.sigmoid(gate) * norm(branch, w("branch_weights"), w("branch_biases"))
        rest = [n for n in names if not n.startswith("output")]
        got = torch.autograd.grad(added, [branch, gate] + [parameters[n] for n in rest], d_x)
        for n, g in zip(rest, got[2:]):
            results["d_" + n] += g
        parts["d_x"].append(d_x.detach()), parts["d_branch"].append(got[0]), parts["d_gate"].append(got[1])
    return dict(results, **{n: torch.cat(p) for n, p in parts.items()})


def _exact_dropout(c, s):
    """The generator in numpy's unsigned 64-bit arithmetic, the sum in 64 bits."""
    n, threshold, halves = s["x"].numel(), round(c["rate"] * 65536), []
    mask, u = np.uint64(0xFFFFFFFF), np.uint64
    for at in range(0, -(-n // 8), 1 << 21):
        index = np.arange(at, min(at + (1 << 21), -(-n // 8)), dtype=np.uint64)
        x0, x1, x2, x3 = index & mask, index >> u(32), np.full_like(index, s["stream"] & 0xFFFFFFFF), np.full_like(index, s["stream"] >> 32)
        for r in range(10):
            k0, k1 = u(((s["seed"] & 0xFFFFFFFF) + r * 0x9E3779B9) & 0xFFFFFFFF), u(((s["seed"] >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)
            a, b = x0 * u(0xD2511F53), x2 * u(0xCD9E8D57)
            x0, x1, x2, x3 = (b >> u(32)) ^ x1 ^ k0, b & mask, (a >> u(32)) ^ x3 ^ k1, a & mask
        words = np.stack([x0, x1, x2, x3], 1).astype("<u4")
        halves.append(words.view("<u2").reshape(-1))
    keep = torch.from_numpy((np.concatenate(halves)[:n] >= threshold)).cuda().reshape(s["x"].shape)
    y = torch.where(keep, s["x"].double() / (1 - threshold / 65536), 0.0)
    return y + s["residual"].double() if "residual" in s else y


_EXACT = dict(step=_exact_attention, prompt=_exact_attention, train=_exact_attention, norm=_exact_norm, norm_backward=_exact_norm, dropout=_exact_dropout)

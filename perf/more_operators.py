"""Workloads of the selective blocks' operators: the short causal convolution, the selective scan behind it (training, prompts, single steps), and the optimiser step
that orthogonalises the updates of matrices.

listed() are sizes of this repository's recurrent and vectorised workloads next to generic ones; draw() spreads over the ranges that they stand for. prepare()
lays a case's tensors out in GPU memory, run() makes one pass: with `own` through the C ABI, otherwise in elementary torch operations in 32 bits. exact() computes
a case from the definitions in 64 bits (sequences step by step).
"""
import ctypes as C
import importlib.util
import math
import os
import sys

import torch

own = False

# ------------------------------------------------------------------ the cases


def listed():
    return [
        # serving / vectorised collection: one token for each of 4,096 rows through a wide block's convolution
        dict(name="convolution_step_4096", kind="convolution_step", type="bfloat16", rows=4096, channels=2048, width=4),
        # sequences of different lengths, some empty, episodes that end inside them, a channel count that no vector divides: forward + backward
        dict(name="convolution_train_ragged", kind="convolution", type="float32", steps=333, rows=37, channels=201, width=3, resets=True, ragged=True),
        # long sequences in 16 bits: forward + backward
        dict(name="convolution_train_8192", kind="convolution", type="bfloat16", steps=8192, rows=4, channels=2048, width=4, resets=False, ragged=False),
        # acting: one step of a small policy's layer in 64 environments, between two environment steps
        dict(name="scan_step_64", kind="scan_step", type="float32", rows=64, heads=1, channels=64, states=16),
        # vectorised collection / serving: one token for each of 4,096 rows, whose states fill a quarter of a gigabyte
        dict(name="scan_step_4096", kind="scan_step", type="bfloat16", rows=4096, heads=1, channels=1024, states=16),
        # a training step of the recurrent workloads' shape (64 steps x 1,024 sequences, width 64) with episode ends inside the sequences: forward + backward
        dict(name="scan_train_64x1024", kind="scan", type="float32", steps=64, rows=1024, heads=1, channels=64, states=16, resets=True, ragged=False),
        # sequences of different lengths, some empty, two heads with inputs of their own, odd widths: forward + backward
        dict(name="scan_train_ragged", kind="scan", type="float32", steps=333, rows=37, heads=2, channels=101, states=11, resets=True, ragged=True),
        # long sequences in 16 bits, few of them: forward + backward
        dict(name="scan_train_8192", kind="scan", type="bfloat16", steps=8192, rows=2, heads=1, channels=2048, states=16, resets=False, ragged=False),
        # one long prompt: outputs and the state that single steps go on from
        dict(name="scan_prompt_16384", kind="scan_prompt", type="bfloat16", steps=16384, rows=1, heads=1, channels=4096, states=16, resets=False, ragged=False),
        # the matrices of the benchmark's network 17-256-256-6
        dict(name="muon_256", kind="muon", type="float32", shapes="256x17,256x256,6x256"),
        # the matrices of four selective blocks of width 512
        dict(name="muon_blocks", kind="muon", type="float32", shapes=",".join(["2048x512,64x1024,1024x32,512x1024"] * 4)),
        # two matrices of a wide model, one square, one tall
        dict(name="muon_4096", kind="muon", type="float32", shapes="4096x4096,16384x4096"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["convolution_step", "convolution", "scan_step", "scan", "scan", "scan_prompt", "muon"])
    dtype = rng.choice(["float32", "bfloat16"])
    if kind == "muon":
        shapes = []
        for _ in range(rng.randint(1, 8)):
            shapes.append((_log(rng, 6, 2048), _log(rng, 6, 2048)))
        return dict(kind=kind, type="float32", shapes=",".join(f"{a}x{b}" for a, b in shapes))
    if kind.startswith("convolution"):
        channels = rng.choice([64, 256, 1024, 2048, _log(rng, 16, 4096)])
        case = dict(kind=kind, type=dtype, channels=channels, width=rng.choice([2, 3, 4, 4]))
        if kind == "convolution_step":
            return dict(case, rows=min(_log(rng, 16, 4096), 4096 * 2048 // channels))
        tokens = _log(rng, 64, 8192 * 4 * 2048 // 2 // channels)
        steps = min(_log(rng, 1, 16384), tokens)
        return dict(case, steps=steps, rows=max(1, tokens // steps), resets=rng.random() < 0.5, ragged=rng.random() < 0.5)
    heads = rng.choice([1, 1, 1, 2, 4])
    states = rng.choice([16, 16, 16, 8, rng.randint(1, 32)])
    channels = rng.choice([64, 256, 1024, 2048, _log(rng, 16, 4096)]) // heads
    case = dict(kind=kind, type=dtype, heads=heads, channels=channels, states=states)
    if kind == "scan_step":
        return dict(case, rows=max(1, min(_log(rng, 16, 4096), 4096 * 1024 * 16 // (heads * channels * states))))
    most = (8192 * 2 * 2048 * 16 if kind == "scan" else 16384 * 4096 * 16) // 2
    tokens = _log(rng, 64, max(64, most // (heads * channels * max(states, 8))))
    steps = min(_log(rng, 1, 16384), tokens)
    rows = max(1, min(tokens // steps, 4096 * 1024 * 16 // (heads * channels * states)))
    return dict(case, steps=steps, rows=rows, resets=rng.random() < 0.5, ragged=rng.random() < 0.5)


def _shapes(case):
    return [tuple(int(n) for n in s.split("x")) for s in case["shapes"].split(",")]


def _size(case):
    return 4 if case["type"] == "float32" else 2


def work(case):
    """Each input once, each output once. The scan: per step, channel and state forward one exponential and the products of decay, input, state and output; backward those of
    the state again, of its gradient and of the five sums. Orthogonalising: five times A = X X' and A A (symmetric: half of them) and B X."""
    c = case
    if c["kind"] == "muon":
        elements = flops = 0
        for rows, cols in _shapes(c):
            m, n = min(rows, cols), max(rows, cols)
            elements += m * n
            flops += 5 * (3 * m * m * n + m * m * m)
        return {"bytes": 20 * elements, "flops": flops}
    if c["kind"].startswith("convolution"):
        n, state = c["rows"] * c["channels"], c["rows"] * c["channels"] * (c["width"] - 1)
        if c["kind"] == "convolution_step":
            return {"bytes": 2 * n * _size(c) + 8 * state, "flops": 2 * n * c["width"]}
        n *= c["steps"]
        return {"bytes": 5 * n * _size(c) + 16 * state, "flops": 8 * n * c["width"]}
    n, state = c["rows"] * c["heads"] * c["channels"], c["rows"] * c["heads"] * c["channels"] * c["states"]
    shared = c["rows"] * c["heads"] * c["states"]
    if c["kind"] == "scan_step":
        return {"bytes": (4 * n + 2 * shared) * _size(c) + 8 * state, "flops": 8 * state}
    n, shared = n * c["steps"], shared * c["steps"]
    bytes_, flops = (4 * n + 2 * shared) * _size(c) + 8 * state, 8 * state * c["steps"]
    if c["kind"] == "scan":
        bytes_ += (7 * n + 4 * shared) * _size(c) + 8 * state
        flops += 24 * state * c["steps"]
    return {"bytes": bytes_, "flops": flops}


# ------------------------------------------------------------------ inputs


def _type(case):
    return getattr(torch, case["type"])


def _inputs(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)

    def randn(*shape, dtype=_type(case)):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    def rand(*shape):
        return torch.rand(shape, generator=g, device="cuda")
    c, f32 = case, torch.float32
    if c["kind"] == "muon":      # gradients of batches of samples: some directions carry most of them, the others noise
        s = dict(parameters=[], gradient=[], momentum=[])
        for rows, cols in _shapes(c):
            rank = max(1, min(rows, cols) // 8)

            def gradient():
                return 1e-3 * (randn(rows, rank, dtype=f32) @ randn(rank, cols, dtype=f32) / math.sqrt(rank) + 0.3 * randn(rows, cols, dtype=f32))
            s["parameters"].append(randn(rows, cols, dtype=f32) / math.sqrt(cols))
            s["gradient"].append(gradient())
            s["momentum"].append(5 * gradient())
        return dict(s, alpha=1 / 64, momentum_factor=61 / 64, weight_decay=1 / 8, epsilon=1e-7)
    step = c["kind"].endswith("_step")
    lead = (c["rows"],) if step else (c["steps"], c["rows"])
    s = {}
    if step:
        s["reset"] = (rand(c["rows"]) < 0.02).to(torch.uint8)
    elif c["resets"]:      # an episode ends every 50 steps
        s["reset"] = (rand(*lead) < 0.02).to(torch.uint8)
    if not step and c["ragged"]:
        s["lengths"] = torch.randint(0, c["steps"] + 1, (c["rows"],), generator=g, device="cuda").to(torch.int32)
    if c["kind"].startswith("convolution"):
        w = c["width"]
        s.update(x=randn(*lead, c["channels"]), weights=randn(c["channels"], w, dtype=f32) / math.sqrt(w), biases=0.1 * randn(c["channels"], dtype=f32), state=randn(c["rows"], w - 1, c["channels"]).float())
        if not step:
            s.update(d_output=randn(*lead, c["channels"]), d_state=randn(c["rows"], w - 1, c["channels"], dtype=f32))
        return s
    h, d, n = c["heads"], c["channels"], c["states"]
    # rates 1 ... states, step sizes from 1e-3 to 1e-1 (logarithms even), as such layers are begun with and stay near
    sizes = torch.exp(math.log(1e-3) + rand(h, d) * math.log(1e2))
    s.update(x=randn(*lead, h, d), delta=(0.5 * randn(*lead, h, d, dtype=f32)).to(_type(c)), b=randn(*lead, h, n), c=randn(*lead, h, n), gate=randn(*lead, h, d),
             log_rates=torch.arange(1, n + 1, device="cuda").log().repeat(h, d, 1) + 0.1 * randn(h, d, n, dtype=f32), skip=1 + 0.1 * randn(h, d, dtype=f32), delta_biases=torch.log(torch.expm1(sizes)),
             state=0.3 * randn(c["rows"], h, d, n, dtype=f32))
    if c["kind"] == "scan":
        s.update(d_output=randn(*lead, h, d), d_state=0.3 * randn(c["rows"], h, d, n, dtype=f32))
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
    """[steps x] rows [x heads] x channels"""
    strides = t.stride()[:-1]
    if len(strides) == 1:
        return C.byref(capi.HeadView(t.data_ptr(), 0, strides[0], 0))
    return C.byref(capi.HeadView(t.data_ptr(), strides[0], strides[1], strides[2] if len(strides) == 3 else 0))


def _step_view(capi, t):
    return C.byref(capi.HeadView(t.data_ptr(), 0, t.stride(0), t.stride(1)))


def _scratch(s, name, nbytes):
    s[name] = torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device="cuda")
    return s[name].data_ptr()


def _own_convolution(s):
    capi, device = _handle()
    c = s["case"]
    out, state = torch.empty_like(s["x"]), torch.empty_like(s["state"])
    results = {"output": out, "state": state}
    grads = {}
    if c["kind"] == "convolution":
        grads = {"d_" + n: torch.empty_like(s[n]) for n in ("x", "weights", "biases", "state")}
        results.update(grads)
    layer = capi.CausalConvolution(weights=_ptr(s["weights"]), biases=_ptr(s["biases"]), d_weights=_ptr(grads.get("d_weights")), d_biases=_ptr(grads.get("d_biases")), type=capi.TYPE[c["type"]],
                                   batch=c["rows"], channels=c["channels"], width=c["width"], silu=1)
    L, x, o = C.byref(layer), _view(capi, s["x"]), _view(capi, out)
    if c["kind"] == "convolution_step":
        step = _call(device, "causal_convolution_step", L, x, o, _ptr(s["state"]), _ptr(state), _ptr(s["reset"]))

        def go():
            step()
            return results
        return go
    tail = (_ptr(s.get("reset")), _ptr(s.get("lengths")), c["steps"])
    forward = _call(device, "causal_convolution_forward", L, x, o, _ptr(s["state"]), _ptr(state), *tail)
    nbytes = device.lib.rlt_rocm_causal_convolution_workspace_bytes(L, c["steps"])
    backward = _call(device, "causal_convolution_backward", L, x, _view(capi, s["d_output"]), _view(capi, grads["d_x"]), _ptr(s["state"]), _ptr(s["d_state"]), _ptr(grads["d_state"]), 0, *tail,
                     _scratch(s, "workspace", nbytes), nbytes)

    def both():
        forward()
        backward()
        return results
    return both


def _scan_layer(capi, s, grads):
    c = s["case"]
    return capi.SelectiveScan(log_rates=_ptr(s["log_rates"]), skip=_ptr(s["skip"]), delta_biases=_ptr(s["delta_biases"]), d_log_rates=_ptr(grads.get("d_log_rates")), d_skip=_ptr(grads.get("d_skip")),
                              d_delta_biases=_ptr(grads.get("d_delta_biases")), type=capi.TYPE[c["type"]], batch=c["rows"], heads=c["heads"], channels=c["channels"], states=c["states"])


def _own_scan_step(s):
    capi, device = _handle()
    out, state = torch.empty_like(s["x"]), torch.empty_like(s["state"])
    v = lambda n: _step_view(capi, s[n])  # noqa: E731
    step = _call(device, "selective_scan_step", C.byref(_scan_layer(capi, s, {})), v("x"), v("delta"), v("b"), v("c"), v("gate"), _step_view(capi, out), _ptr(s["state"]), _ptr(state), _ptr(s["reset"]))

    def go():
        step()
        return {"output": out, "state": state}
    return go


def _own_scan(s):
    capi, device = _handle()
    c, train = s["case"], s["case"]["kind"] == "scan"
    out, state = torch.empty_like(s["x"]), torch.empty_like(s["state"])
    results = {"output": out, "state": state}
    grads = {"d_" + n: torch.empty_like(s[n]) for n in ("x", "delta", "b", "c", "gate", "state", "log_rates", "skip", "delta_biases")} if train else {}
    results.update(grads)
    layer = C.byref(_scan_layer(capi, s, grads))
    nbytes = max(device.lib.rlt_rocm_selective_scan_workspace_bytes(layer, c["steps"], k) for k in range(1 + train))
    workspace = (_scratch(s, "workspace", nbytes), nbytes)
    checkpoints = _scratch(s, "checkpoints", device.lib.rlt_rocm_selective_scan_checkpoint_bytes(layer, c["steps"])) if train else None
    v = lambda n: _view(capi, s[n])  # noqa: E731
    d = lambda n: _view(capi, grads["d_" + n])  # noqa: E731
    inputs, tail = (v("x"), v("delta"), v("b"), v("c"), v("gate")), (_ptr(s.get("reset")), _ptr(s.get("lengths")), c["steps"], checkpoints, *workspace)
    forward = _call(device, "selective_scan_forward", layer, *inputs, _view(capi, out), _ptr(s["state"]), _ptr(state), *tail)
    if not train:
        def go():
            forward()
            return results
        return go
    backward = _call(device, "selective_scan_backward", layer, *inputs, v("d_output"), d("x"), d("delta"), d("b"), d("c"), d("gate"), _ptr(s["d_state"]), _ptr(grads["d_state"]), 0, *tail)

    def both():
        forward()
        backward()
        return results
    return both


def _own_muon(s):
    capi, device = _handle()
    parameters, momentum = [torch.empty_like(t) for t in s["parameters"]], [torch.empty_like(t) for t in s["momentum"]]
    tensors = (capi.MuonTensor * len(parameters))(*[capi.MuonTensor(w.data_ptr(), g.data_ptr(), m.data_ptr(), nw.data_ptr(), nm.data_ptr(), *w.shape)
                                                    for w, g, m, nw, nm in zip(s["parameters"], s["gradient"], s["momentum"], parameters, momentum)])
    settings = capi.MuonParameters(alpha=s["alpha"], momentum=s["momentum_factor"], weight_decay=s["weight_decay"], epsilon=s["epsilon"], nesterov=1, iterations=5)
    nbytes = device.lib.rlt_rocm_muon_workspace_bytes(tensors, len(parameters))
    step = _call(device, "muon_step", tensors, len(parameters), C.byref(settings), _scratch(s, "workspace", nbytes), nbytes)

    def go():
        step()
        return {"parameters": parameters, "momentum": momentum}
    return go


_OWN = dict(convolution=_own_convolution, convolution_step=_own_convolution, scan=_own_scan, scan_prompt=_own_scan, scan_step=_own_scan_step, muon=_own_muon)

# ------------------------------------------------------------------ plain forms


def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _begins(s, steps, rows, first):
    """[steps, rows]: the step that the episode of a step begins with, `first` for the one that goes on from before"""
    if "reset" not in s:
        return torch.full((steps, rows), first, device="cuda")
    at = torch.arange(steps, device="cuda")[:, None]
    return torch.where(s["reset"].reshape(steps, rows).bool(), at, first).cummax(0).values


def _lengths(s, steps, rows):
    return s["lengths"].long() if "lengths" in s else torch.full((rows,), steps, device="cuda")


def _plain_convolution(s):
    c = s["case"]
    step, w = c["kind"] == "convolution_step", c["width"]
    x = (s["x"][None] if step else s["x"]).float()
    steps, rows = x.shape[:2]
    weights = s["weights"]
    begins, lengths = _begins(s, steps, rows, 1 - w), _lengths(s, steps, rows)
    at = torch.arange(steps, device="cuda")[:, None]
    live = (at < lengths)[..., None]
    longer = torch.cat([s["state"].permute(1, 0, 2), x])      # row i holds the input of step i - (w - 1)
    pre = s["biases"].expand(x.shape)
    for j in range(w):      # j steps back
        seen = (at - j >= begins)[..., None]
        pre = pre + weights[:, w - 1 - j] * torch.where(seen, longer[w - 1 - j:w - 1 - j + steps], 0.0)
    sigmoid = _sigmoid(pre)
    out = torch.where(live, pre * sigmoid, 0.0).to(_type(c))
    # the last w - 1 inputs of each row, of its last episode
    last = (lengths - 1).clamp(min=0)
    begin = torch.where(lengths > 0, begins.gather(0, last[None])[0], 1 - w)
    source = lengths[:, None] - (w - 1) + torch.arange(w - 1, device="cuda")      # [rows, w - 1] steps
    kept = (source >= begin[:, None])[..., None]
    row = torch.arange(rows, device="cuda")[:, None]
    state = torch.where(kept, longer[source + w - 1, row], 0.0)
    results = {"output": out[0] if step else out, "state": state}
    if step:
        return results
    d_pre = torch.where(live, s["d_output"].float() * sigmoid * (1 + pre * (1 - sigmoid)), 0.0)
    d_longer = torch.zeros_like(longer)
    d_weights = torch.empty_like(weights)
    for j in range(w):
        seen = (at - j >= begins)[..., None]
        d_weights[:, w - 1 - j] = (d_pre * torch.where(seen, longer[w - 1 - j:w - 1 - j + steps], 0.0)).sum((0, 1))
        d_longer[w - 1 - j:w - 1 - j + steps] += torch.where(seen, weights[:, w - 1 - j] * d_pre, 0.0)
    d_longer[source + w - 1, row] += torch.where(kept, s["d_state"], 0.0)
    return dict(results, d_x=d_longer[w - 1:].to(_type(c)), d_weights=d_weights, d_biases=d_pre.sum((0, 1)), d_state=d_longer[:w - 1].permute(1, 0, 2).contiguous())


def _recurrence(a, u, entry):
    """h_t = a_t h_{t-1} + u_t along the first axis, in place of u; chunks of up to 64 steps side by side, then from chunk to chunk"""
    steps = u.shape[0]
    size = max(1, min(64, int(math.sqrt(steps))))
    chunks = -(-steps // size)
    pad = chunks * size - steps
    if pad:
        a, u = torch.cat([a, a.new_ones((pad,) + a.shape[1:])]), torch.cat([u, u.new_zeros((pad,) + u.shape[1:])])
    else:
        a = a.clone()
    a, u = a.reshape((chunks, size) + a.shape[1:]), u.reshape((chunks, size) + u.shape[1:])
    for i in range(1, size):
        u[:, i] += a[:, i] * u[:, i - 1]
        a[:, i] *= a[:, i - 1]
    entries = [entry]
    for k in range(chunks - 1):
        entries.append(u[k, -1] + a[k, -1] * entries[-1])
    for i in range(size):
        u[:, i] += a[:, i] * torch.stack(entries)
    return u.reshape((chunks * size,) + u.shape[2:])[:steps]


def _plain_scan(s):
    c = s["case"]
    step, train = c["kind"] == "scan_step", c["kind"] == "scan"
    lead = (lambda t: t[None].float()) if step else (lambda t: t.float())
    x, raw, b, read, gate = (lead(s[n]) for n in ("x", "delta", "b", "c", "gate"))
    steps, rows = x.shape[:2]
    rates = -torch.exp(s["log_rates"])
    raw = raw + s["delta_biases"]
    delta = torch.logaddexp(raw, torch.zeros_like(raw))
    live = (torch.arange(steps, device="cuda")[:, None] < _lengths(s, steps, rows))[..., None, None]
    reset = s["reset"].reshape(steps, rows).bool()[..., None, None, None] if "reset" in s else None
    decay = torch.exp(delta[..., None] * rates)
    if reset is not None:
        decay = torch.where(reset, 0.0, decay)
    decay = torch.where(live[..., None], decay, 1.0)
    added = torch.where(live[..., None], (delta * x)[..., None] * b[:, :, :, None, :], 0.0)
    h = _recurrence(decay, added, s["state"])
    y = (h * read[:, :, :, None, :]).sum(-1)
    sigmoid = _sigmoid(gate)
    mixed = y + s["skip"] * x
    out = torch.where(live, mixed * gate * sigmoid, 0.0).to(_type(c))
    results = {"output": out[0] if step else out, "state": h[-1].clone()}
    if not train:
        return results
    d_out = torch.where(live, s["d_output"].float(), 0.0)
    d_gate = d_out * mixed * sigmoid * (1 + gate * (1 - sigmoid))
    d_y = d_out * gate * sigmoid
    d_c = (d_y[..., None] * h).sum(3)
    # the gradient of the state behind each step: from the last step to the first, the next step's decay with it
    later = torch.cat([decay[1:], torch.ones_like(decay[:1])]).flip(0)
    grad = _recurrence(later, (d_y[..., None] * read[:, :, :, None, :]).flip(0), s["d_state"]).flip(0)
    del later
    grad = torch.where(live[..., None], grad, 0.0)
    d_state = decay[0] * torch.where(live[0][..., None], grad[0], s["d_state"])
    d_u = (grad * b[:, :, :, None, :]).sum(-1)
    d_b = (grad * (delta * x)[..., None]).sum(3)
    grad *= decay * torch.cat([s["state"][None], h[:-1]])      # by the decay's exponent
    d_delta = torch.where(live, (grad * rates).sum(-1) + d_u * x, 0.0)
    d_log_rates = (grad * delta[..., None]).sum((0, 1)) * rates
    d_raw = d_delta * _sigmoid(raw)
    return dict(results, d_x=(d_u * delta + s["skip"] * d_y).to(_type(c)), d_delta=d_raw.to(_type(c)), d_b=d_b.to(_type(c)), d_c=d_c.to(_type(c)), d_gate=d_gate.to(_type(c)), d_state=d_state,
                d_log_rates=d_log_rates, d_skip=(d_y * x).sum((0, 1)), d_delta_biases=d_raw.sum((0, 1)))


def _plain_muon(s):
    parameters, momenta = [], []
    for w, g, m in zip(s["parameters"], s["gradient"], s["momentum"]):
        m = s["momentum_factor"] * m + g
        x = g + s["momentum_factor"] * m
        tall = w.shape[0] > w.shape[1]
        x = x.t() if tall else x
        x = x / ((x * x).sum().sqrt() + s["epsilon"])
        for _ in range(5):
            a = x @ x.t()
            x = 3.4445 * x + (-4.775 * a + 2.0315 * (a @ a)) @ x
        x = x.t() if tall else x
        parameters.append((1 - s["alpha"] * s["weight_decay"]) * w - s["alpha"] * math.sqrt(max(1.0, w.shape[0] / w.shape[1])) * x)
        momenta.append(m)
    return {"parameters": parameters, "momentum": momenta}


_PLAIN = dict(convolution=_plain_convolution, convolution_step=_plain_convolution, scan=_plain_scan, scan_prompt=_plain_scan, scan_step=_plain_scan, muon=_plain_muon)

# ------------------------------------------------------------------ in 64 bits


def exact(case, seed):
    s = _inputs(case, seed)
    return _EXACT[case["kind"].split("_")[0]](case, s)


def _flags(c, s, steps, rows):
    reset = s["reset"].reshape(steps, rows) != 0 if "reset" in s else torch.zeros((steps, rows), dtype=torch.bool, device="cuda")
    live = torch.ones((steps, rows), dtype=torch.bool, device="cuda")
    if "lengths" in s:
        live = torch.arange(steps, device="cuda")[:, None] < s["lengths"][None]
    return reset, live


def _exact_convolution(c, s):
    """Step by step with the window of the last inputs, which a reset empties; then the window's gradient from the last step to the first."""
    step = c["kind"] == "convolution_step"
    x = (s["x"][None] if step else s["x"]).double()
    steps, rows, channels = x.shape
    reset, live = _flags(c, s, steps, rows)
    taps, bias = s["weights"].double().t(), s["biases"].double()      # [width, channels], the step's own last
    window = s["state"].double()
    out, pres, seen = torch.zeros_like(x), torch.zeros_like(x), []
    for t in range(steps):
        window = window * (~reset[t] | ~live[t])[:, None, None]
        full = torch.cat([window, x[t][:, None]], 1)
        seen.append(full)
        pres[t] = bias + (taps * full).sum(1)
        out[t] = pres[t] / (1 + torch.exp(-pres[t])) * live[t][:, None]
        window = torch.where(live[t][:, None, None], full[:, 1:], window)
    results = {"output": out[0] if step else out, "state": window}
    if step:
        return results
    d_window, d_x, d_taps, d_bias = s["d_state"].double(), torch.zeros_like(x), torch.zeros_like(taps), torch.zeros_like(bias)
    nothing = torch.zeros((rows, 1, channels), dtype=torch.float64, device="cuda")
    for t in reversed(range(steps)):
        p = torch.sigmoid(pres[t])
        d = s["d_output"][t].double() * (p + pres[t] * p * (1 - p)) * live[t][:, None]
        d_taps += (d[:, None] * seen[t]).sum(0)
        d_bias += d.sum(0)
        d_full = torch.cat([nothing, d_window], 1) + taps * d[:, None]
        d_x[t] = d_full[:, -1] * live[t][:, None]
        d_window = torch.where(live[t][:, None, None], d_full[:, :-1] * (~reset[t])[:, None, None], d_window)
    return dict(results, d_x=d_x, d_weights=d_taps.t(), d_biases=d_bias, d_state=d_window)


def _exact_scan(c, s):
    """h <- exp(-exp(log_rates) delta) h (nothing at a reset) + delta x b; the states are kept in 64 bits where gradients are asked for."""
    step, train = c["kind"] == "scan_step", c["kind"] == "scan"
    if train and c["steps"] * c["rows"] * c["heads"] * c["channels"] * c["states"] * 8 > 48 << 30:
        return None
    lead = (lambda t: t[None]) if step else (lambda t: t)
    x, raw, b, read, gate = (lead(s[n]) for n in ("x", "delta", "b", "c", "gate"))
    steps, rows = x.shape[:2]
    reset, live = _flags(c, s, steps, rows)
    rates, skip, bias = -s["log_rates"].double().exp(), s["skip"].double(), s["delta_biases"].double()
    h = s["state"].double()
    kept = torch.empty((steps,) + h.shape, dtype=torch.float64, device="cuda") if train else None
    out = torch.zeros(x.shape, dtype=torch.float64, device="cuda")

    def at(t):
        raw_t = raw[t].double() + bias
        size = torch.nn.functional.softplus(raw_t, threshold=40.0)
        return x[t].double(), raw_t, size, b[t].double()[:, :, None], read[t].double()[:, :, None], gate[t].double(), torch.exp(size[..., None] * rates)
    for t in range(steps):
        x_t, _, size, b_t, c_t, z, decay = at(t)
        if train:
            kept[t] = h
        before = torch.where(reset[t][:, None, None, None], 0.0, h)
        h = torch.where(live[t][:, None, None, None], decay * before + (size * x_t)[..., None] * b_t, h)
        out[t] = torch.where(live[t][:, None, None], ((h * c_t).sum(-1) + skip * x_t) * z * torch.sigmoid(z), 0.0)
    results = {"output": out[0] if step else out, "state": h}
    if not train:
        return results
    grad = s["d_state"].double()
    d = {n: torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in ("x", "delta", "b", "c", "gate", "log_rates", "skip", "delta_biases")}
    for t in reversed(range(steps)):
        x_t, raw_t, size, b_t, c_t, z, decay = at(t)
        on, on4 = live[t][:, None, None], live[t][:, None, None, None]
        before = torch.where(reset[t][:, None, None, None], 0.0, kept[t])
        after = decay * before + (size * x_t)[..., None] * b_t
        up, p = torch.where(on, s["d_output"][t].double(), 0.0), torch.sigmoid(z)
        mixed = (after * c_t).sum(-1) + skip * x_t
        d["gate"][t] = up * mixed * (p + z * p * (1 - p))
        d_y = up * z * p
        d["skip"] += (d_y * x_t).sum(0)
        d["c"][t] = (d_y[..., None] * after).sum(2)
        here = torch.where(on4, grad + d_y[..., None] * c_t, 0.0)
        d["b"][t] = (here * (size * x_t)[..., None]).sum(2)
        through = (here * b_t).sum(-1)
        d["x"][t] = through * size + d_y * skip
        exponent = here * decay * before
        d_size = through * x_t + (exponent * rates).sum(-1)
        d["log_rates"] += (exponent * size[..., None]).sum(0) * rates
        d_raw = d_size * torch.sigmoid(raw_t)
        d["delta"][t] = d_raw
        d["delta_biases"] += d_raw.sum(0)
        grad = torch.where(on4, torch.where(reset[t][:, None, None, None], 0.0, decay * here), grad)
    return dict(results, d_state=grad, **{"d_" + n: t for n, t in d.items()})


def _exact_muon(c, s):
    parameters, momenta = [], []
    for w, g, m in zip(s["parameters"], s["gradient"], s["momentum"]):
        w, g, m = w.double(), g.double(), m.double()
        m = g + s["momentum_factor"] * m
        update = g + s["momentum_factor"] * m
        x = update / (torch.linalg.norm(update) + s["epsilon"])
        for _ in range(5):      # a x + b (x x') x + c (x x')^2 x, on the smaller side
            gram = x @ x.t() if x.shape[0] <= x.shape[1] else x.t() @ x
            inner = -4.775 * gram + 2.0315 * gram @ gram
            x = 3.4445 * x + (inner @ x if x.shape[0] <= x.shape[1] else x @ inner)
        parameters.append(w - s["alpha"] * (s["weight_decay"] * w + max(1.0, w.shape[0] / w.shape[1]) ** 0.5 * x))
        momenta.append(m)
    return {"parameters": parameters, "momentum": momenta}


_EXACT = dict(convolution=_exact_convolution, scan=_exact_scan, muon=_exact_muon)

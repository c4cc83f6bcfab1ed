"""Linear attention where tensors, values and calls are out of the ordinary. The reference in 64 bits, the cases and the bounds are those of test_rocm_linear_attention."""
import ctypes as C

import numpy as np
import pytest

from test_rocm_linear_attention import Tensor, case, layer_of, reference, workspace
from typed_arrays import filled, rounded

gpu = pytest.mark.gpu


def run(rocm, c, x, tensor=None):
    """forward and backward, all outputs in 64 bits; tensor(x or shape, value) makes the tensors of heads"""
    tensor = tensor or (lambda x, value=None: Tensor(rocm, x, c["dtype"], value=value))
    layer, steps = layer_of(rocm, c, x), c["steps"]
    t = {n: tensor(x[n]) for n in ("q", "k", "v", "d_output")}
    o = {n: tensor(s, 7.0) for n, s in (("output", x["d_output"].shape), ("d_q", x["q"].shape), ("d_k", x["k"].shape), ("d_v", x["v"].shape))}
    state, d_state, reset, lengths = (rocm.array(x[n]) if x.get(n) is not None else None for n in ("state", "d_state", "reset", "lengths"))
    ptr = lambda a: a.ptr if a is not None else None
    shape = (c["rows"], c["heads"], c["dk"], c["dv"])
    final, d_initial, d_rate = filled(rocm, shape, "float32"), filled(rocm, shape, "float32"), filled(rocm, (c["heads"],), "float32")
    w, n = workspace(rocm, layer, steps, 0)
    rocm.call("linear_attention_forward", C.byref(layer), t["q"].view, t["k"].view, t["v"].view, o["output"].view, ptr(state), final.ptr, ptr(reset), ptr(lengths), steps, w.ptr, n)
    w, n = workspace(rocm, layer, steps, 1)
    rocm.call("linear_attention_backward", C.byref(layer), t["q"].view, t["k"].view, t["v"].view, t["d_output"].view, o["d_q"].view, o["d_k"].view, o["d_v"].view, ptr(state), ptr(d_state),
              d_initial.ptr, d_rate.ptr, 0, ptr(reset), ptr(lengths), steps, w.ptr, n)
    rocm.sync()
    return dict({n: a.numpy() for n, a in o.items()}, **{n: a.numpy().astype(np.float64) for n, a in (("state", final), ("d_state", d_initial), ("d_log_decay", d_rate))})


# ------------------------------------------------------------------ roundings


@gpu
@pytest.mark.parametrize("steps,rows,heads,d", [(16, 256, 8, 32), (16, 64, 8, 64), (12, 40, 8, 128)])
def test_bfloat16_outputs_are_rounded_once(rocm, steps, rows, heads, d):
    """An output is the bfloat16 number nearest to the exact value unless the midpoint between two numbers lies between that value and the one in 32 bits, which it does with a probability of their distance in units of
    the last place. That distance: 4 steps + channels + 16 roundings to 24 bits, each independent of the others, of values as large as the outputs. Scores, states or weighted values of 16 bits are three times as far off."""
    c, x = case(47, "bfloat16", steps, rows, heads, heads, d, d)
    want, got = reference(c, x), run(rocm, c, x)
    for n in ("output", "d_q", "d_k", "d_v"):
        last_place = 2.0 ** (np.floor(np.log2(np.abs(want[n]))) - 7)
        off = 2.0 ** -24 * (4 * steps + d + 16) ** 0.5 * np.sqrt(np.mean(want[n] ** 2))
        expected = np.sum(np.minimum(1, off / last_place))
        others = np.sum(got[n] != rounded(want[n], "bfloat16"))
        print(n, want[n].size, "elements", others, "elsewhere, at most", expected, flush=True)
        assert others <= expected + 5 * expected ** 0.5, n

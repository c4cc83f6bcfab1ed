"""The optimiser step for matrices whose updates are orthogonalised, against the definition in 64 bits.

Bounds, set before the first run; u = 2^-24. The momentum has two roundings: 2 u (|f m| + |m'|). The rest in the spectral norm, which no element's error passes: X of norm at most 1.21 is held, and goes into products, with errors of at most 4 u of each
element (22 bits and a sign; the low parts' product is dropped), and a sum over K products rounds K times: an error matrix of elements at most e has a spectral norm of at most e sqrt(M N), but those of roundings are as good as random, and theirs is about
e (sqrt M + sqrt N) / 2: bounds take e = 4 u times the largest row norms that enter, 1.21 at most, whatever K is (sums over K of products of two rows of norm 1.21 have magnitudes of at most 1.5), and 8 as a factor of safety: one iteration adds
at most D = 8 * 4 u * (sqrt M + sqrt N) * 3 (three products, whose coefficients' sum 4.775 * 1.21 + 2.0315 * 1.8 ... is below 10: D = 960 u (sqrt M + sqrt N) at worst). An error before an iteration is amplified by at most the
polynomial's largest slope, 3.4445 (it is largest at zero): after five, D (1 + 3.4445 + ... + 3.4445^4) = 200 D. What is checked against that is the spectral norm of the error of X, whose own scale is 1;
and that the error's root mean square is no more than 4 times that of the same products in fp32."""
import ctypes as C

import numpy as np
import pytest

from helpers import capi, package

gpu = pytest.mark.gpu
U = 2.0 ** -24
COEFFICIENTS = (np.float64(np.float32(3.4445)), np.float64(np.float32(-4.775)), np.float64(np.float32(2.0315)))


def orthogonalised(u, epsilon, iterations, dtype=np.float64):
    a, b, c = (dtype(k) for k in COEFFICIENTS)
    x = (u.astype(np.float64) / (np.sqrt((u.astype(np.float64) ** 2).sum()) + epsilon)).astype(dtype)
    if u.shape[0] > u.shape[1]:
        x = x.T
    for _ in range(iterations):
        gram = x @ x.T
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.T if u.shape[0] > u.shape[1] else x


def reference(t, p):
    m = np.float64(p["momentum"]) * t["momentum"] + t["gradient"]
    u = t["gradient"] + p["momentum"] * m if p["nesterov"] else m
    scale = np.sqrt(max(1.0, t["parameters"].shape[0] / t["parameters"].shape[1]))
    return m, scale, orthogonalised(u, p["epsilon"], p["iterations"]), orthogonalised(u, p["epsilon"], p["iterations"], np.float32), (1 - p["alpha"] * p["weight_decay"]) * t["parameters"]


def settings(**changes):
    return dict(dict(alpha=1 / 32, momentum=61 / 64, weight_decay=1 / 8, epsilon=2.0 ** -23, nesterov=1, iterations=5), **changes)


def tensors_of(seed, shapes):
    rng = np.random.default_rng(seed)
    n = lambda s, k: (k * rng.standard_normal(s)).astype(np.float32)
    return [dict(parameters=n(s, 1.0), gradient=n(s, 1e-3), momentum=n(s, 1e-2)) for s in shapes]


def workspace(rocm, table, n):
    size = rocm.device.lib.rlt_rocm_muon_workspace_bytes(table, n)
    return rocm.device.empty((max(int(size), 16),), np.uint8), size


def run(rocm, tensors, p, in_place=False):
    arrays = [{n: rocm.array(a) for n, a in t.items()} for t in tensors]
    for t, a in zip(tensors, arrays):
        a["next_parameters"] = a["parameters"] if in_place else rocm.array(np.full(t["parameters"].shape, 7.0, np.float32))
        a["next_momentum"] = a["momentum"] if in_place else rocm.array(np.full(t["parameters"].shape, 7.0, np.float32))
    table = (capi.MuonTensor * len(tensors))(*[capi.MuonTensor(*[a[n].ptr for n in ("parameters", "gradient", "momentum", "next_parameters", "next_momentum")], *t["parameters"].shape) for t, a in zip(tensors, arrays)])
    w, size = workspace(rocm, table, len(tensors))
    w.upload(np.full(w.shape, 255, np.uint8))      # (no call counts on what its workspace holds)
    rocm.call("muon_step", table, len(tensors), C.byref(capi.MuonParameters(**p)), w.ptr, size)
    rocm.sync()
    return [{n: a[n].numpy() for n in ("next_parameters", "next_momentum")} for a in arrays]


def check(tensors, p, got):
    for t, r in zip(tensors, got):
        m, scale, x, x32, kept = reference(t, p)
        rows, cols = x.shape
        assert np.all(np.abs(r["next_momentum"] - m) <= 2 * U * (np.abs(p["momentum"] * t["momentum"]) + np.abs(m)) + 1e-45)
        off = (r["next_parameters"].astype(np.float64) - (kept - p["alpha"] * scale * x)) / (p["alpha"] * scale)
        own = 3 * U * (np.abs(kept) + p["alpha"] * scale * np.abs(x)) / (p["alpha"] * scale)      # the update's own roundings
        error = np.sign(off) * np.maximum(np.abs(off) - own, 0.0)
        d = 960 * U * (np.sqrt(rows) + np.sqrt(cols))
        bound = d * sum(3.4445 ** k for k in range(p["iterations"]))
        assert np.linalg.norm(error, 2) <= bound, (x.shape, np.linalg.norm(error, 2), bound)
        size, plain = np.sqrt((error ** 2).mean()), np.sqrt(((x32 - x) ** 2).mean())
        assert size <= 4 * plain + U * np.sqrt((x ** 2).mean()), (x.shape, size, plain)


SHAPES = [[(1, 1)], [(1, 7)], [(7, 1)], [(64, 64)], [(63, 65), (65, 63)], [(17, 256), (256, 17), (256, 256), (6, 256)], [(128, 130)], [(300, 100)], [(511, 600)], [(512, 512)], [(600, 513), (513, 600), (20, 33)], [(40, 1000)], [(1100, 515)]]


@gpu
@pytest.mark.parametrize("shapes", SHAPES)
def test_a_step(rocm, shapes):
    print("case", shapes, flush=True)
    tensors, p = tensors_of(len(shapes) + shapes[0][0], shapes), settings()
    check(tensors, p, run(rocm, tensors, p))


@gpu
@pytest.mark.parametrize("changes", [dict(nesterov=0), dict(iterations=1), dict(iterations=2), dict(iterations=6), dict(weight_decay=0.0), dict(momentum=0.0), dict(epsilon=0.0)])
def test_settings(rocm, changes):
    tensors, p = tensors_of(3, [(70, 90), (520, 530)]), settings(**changes)
    check(tensors, p, run(rocm, tensors, p))


@gpu
def test_more_matrices_than_a_launch_takes(rocm):
    shapes = [(20 + i, 50 - i) for i in range(30)] + [(512 + i, 512) for i in range(2)]
    tensors, p = tensors_of(5, shapes), settings()
    check(tensors, p, run(rocm, tensors, p))


@gpu
@pytest.mark.parametrize("shapes", [[(100, 200), (200, 64)], [(520, 700)]])
def test_in_place_and_again_bit_for_bit(rocm, shapes):
    tensors, p = tensors_of(7, shapes), settings()
    first, second = run(rocm, tensors, p), run(rocm, tensors, p, in_place=True)
    for a, b in zip(first, second):
        assert all(np.array_equal(a[n], b[n]) for n in a)


# matrices that a workgroup holds (sides of up to 64 and 256), by themselves; just beyond; and beside larger ones
HELD = [[(64, 256)], [(256, 64)], [(64, 192)], [(1, 256), (256, 1)], [(17, 200), (200, 17), (64, 64), (1, 1), (63, 255), (255, 63), (33, 129)], [(64, 257)], [(257, 64)], [(65, 64)], [(64, 256), (65, 256)]]


@gpu
@pytest.mark.parametrize("shapes", HELD)
def test_matrices_that_a_workgroup_holds(rocm, shapes):
    print("case", shapes, flush=True)
    tensors, p = tensors_of(21, shapes), settings()
    first, second = run(rocm, tensors, p), run(rocm, tensors, p, in_place=True)
    check(tensors, p, first)
    for a, b in zip(first, second):
        assert all(np.array_equal(a[n], b[n]) for n in a)


@gpu
@pytest.mark.parametrize("changes", [dict(nesterov=0), dict(iterations=1), dict(iterations=2), dict(iterations=6), dict(weight_decay=0.0), dict(momentum=0.0), dict(epsilon=0.0)])
def test_settings_of_matrices_that_a_workgroup_holds(rocm, changes):
    tensors, p = tensors_of(23, [(60, 64), (250, 30), (40, 100)]), settings(**changes)
    check(tensors, p, run(rocm, tensors, p))


@gpu
@pytest.mark.parametrize("size", [1e-30, 1e30])
def test_small_matrices_of_any_size_of_none_and_of_what_is_not_finite(rocm, size):
    tensors, p = tensors_of(25, [(60, 64), (64, 200), (200, 10), (30, 30)] * 8), settings(epsilon=2.0 ** -149)
    for t in tensors:
        t["gradient"], t["momentum"] = (t["gradient"] * np.float32(size)).astype(np.float32), (t["momentum"] * np.float32(size)).astype(np.float32)
    clean = run(rocm, tensors, p)
    check(tensors, p, clean)
    tensors[1]["gradient"][3, 4] = np.nan
    tensors[2]["gradient"][:] = tensors[2]["momentum"][:] = 0
    got = run(rocm, tensors, p)
    assert np.isnan(got[1]["next_parameters"]).any() and np.isnan(got[1]["next_momentum"]).sum() == 1
    assert np.allclose(got[2]["next_parameters"], (1 - p["alpha"] * p["weight_decay"]) * tensors[2]["parameters"], rtol=2e-7, atol=0)
    for i in range(3, len(got)):
        assert all(np.array_equal(got[i][n], clean[i][n]) for n in got[i])


# tiles of 128, 192 and 256, and lengths of k that workgroups share: by the sizes that come to them
@gpu
@pytest.mark.parametrize("shapes", [[(2048, 512), (64, 1024), (1024, 32), (512, 1024)] * 4, [(64, 8192)], [(1000, 1030)], [(2880, 2870)], [(2048, 8190)], [(8190, 2048)], [(5600, 5632)]])
def test_large_matrices(rocm, shapes):
    """no element is further off than the bound on the spectral norm of the errors, and their root mean square is as in check"""
    print("case", shapes, flush=True)
    tensors, p = tensors_of(27, shapes), settings(iterations=2)
    for t, r in zip(tensors, run(rocm, tensors, p)):
        m, scale, x, x32, kept = reference(t, p)
        assert np.all(np.abs(r["next_momentum"] - m) <= 2 * U * (np.abs(p["momentum"] * t["momentum"]) + np.abs(m)) + 1e-45)
        off = (r["next_parameters"].astype(np.float64) - (kept - p["alpha"] * scale * x)) / (p["alpha"] * scale)
        own = 3 * U * (np.abs(kept) + p["alpha"] * scale * np.abs(x)) / (p["alpha"] * scale)
        error = np.maximum(np.abs(off) - own, 0.0)
        assert error.max() <= 960 * U * (np.sqrt(x.shape[0]) + np.sqrt(x.shape[1])) * (1 + 3.4445)
        assert np.sqrt((error ** 2).mean()) <= 4 * np.sqrt(((x32 - x) ** 2).mean()) + U * np.sqrt((x ** 2).mean()), x.shape


# Rows or columns far below the others. What is held, two parts of 16 bits, has a quantum of 2^-47 of the update's norm where the low part leaves its normal range: a root mean square of 2^-49 an element, sqrt(n) 2^-49 of a row of n. In tiles of 128
# and more a product takes a factor's high part times 2^-9 with the other's low part, of at most 2^-11: 2^-15 (times 0.29) of 2^-14 there, by 2^-11 times 0.29 of the other factor: 2^-44 of that one's norm, which is as large as X's or, for A and
# b A + c A A, ten times that with their coefficients. Both relative to the row as it is at the start (it grows as fast as the errors do); four as a factor of safety, and on top of four times what the same products in fp32 are off.
WEAK = [((40, 200), 5), ((128, 256), 5), ((256, 128), 5), ((512, 1024), 5), ((1030, 1000), 5), ((2048, 2050), 2), ((8190, 2048), 2), ((2048, 8190), 2)]


@gpu
@pytest.mark.parametrize("shape,iterations", WEAK)
@pytest.mark.parametrize("size", [2.0 ** -17, 2.0 ** -27])
@pytest.mark.parametrize("side", [0, 1])
def test_rows_and_columns_far_below_the_others(rocm, shape, iterations, size, side):
    print("case", shape, size, side, flush=True)
    t, p = tensors_of(29, [shape])[0], settings(alpha=1.0, momentum=0.0, weight_decay=0.0, nesterov=0, iterations=iterations, epsilon=0.0)
    weak = (slice(None),) * side + (slice(shape[side] // 2, None),)
    t["parameters"][:] = t["momentum"][:] = 0
    t["gradient"][weak] *= np.float32(size)
    got = run(rocm, [t], p)[0]
    _, scale, x, x32, _ = reference(t, p)
    error = np.linalg.norm((got["next_parameters"].astype(np.float64) / -scale - x)[weak]) / np.linalg.norm(x[weak])
    plain = np.linalg.norm((x32 - x)[weak]) / np.linalg.norm(x[weak])
    start = size / np.sqrt(shape[side] / 2)      # the norm of a weak row (or column) at the start
    assert error <= 4 * plain + U + 4 * (np.sqrt(shape[1 - side]) * 2.0 ** -49 + 10 * 2.0 ** -44) / start, (error, plain)


@gpu
@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e12, 1e30])
def test_gradients_of_any_size(rocm, size):
    """the norm's squares leave the range of fp32, the orthogonalised update does not depend on the size"""
    tensors, p = tensors_of(9, [(60, 80)]), settings(epsilon=0.0)
    for t in tensors:
        t["gradient"], t["momentum"] = (t["gradient"] * np.float32(size)).astype(np.float32), (t["momentum"] * np.float32(size)).astype(np.float32)
    check(tensors, p, run(rocm, tensors, p))


@gpu
def test_matrices_of_few_directions_and_of_none(rocm):
    """a matrix of rank one, one of zeros (its update is zero: epsilon), one with a single large element"""
    tensors, p = tensors_of(11, [(80, 100), (70, 70), (90, 60)]), settings()
    rng = np.random.default_rng(1)
    tensors[0]["gradient"] = np.outer(rng.standard_normal(80), rng.standard_normal(100)).astype(np.float32)
    tensors[0]["momentum"] = 3 * tensors[0]["gradient"]
    for n in ("gradient", "momentum"):
        tensors[1][n][:] = 0
        tensors[2][n][:] = 0
        tensors[2][n][5, 7] = 4.0
    got = run(rocm, tensors, p)
    for t, r in zip(tensors, got):
        m, scale, x, _, kept = reference(t, p)
        error = (r["next_parameters"] - (kept - p["alpha"] * scale * x)) / (p["alpha"] * scale)
        d = 960 * U * (np.sqrt(x.shape[0]) + np.sqrt(x.shape[1])) * 200
        assert np.linalg.norm(error, 2) <= d + 3 * U * np.linalg.norm(kept) / p["alpha"]
    assert np.allclose(got[1]["next_parameters"], (1 - p["alpha"] * p["weight_decay"]) * tensors[1]["parameters"], rtol=2e-7, atol=0)


@gpu
def test_a_value_that_is_not_finite_stays_in_its_matrix(rocm):
    tensors, p = tensors_of(13, [(60, 70), (70, 60), (64, 64)]), settings()
    clean = run(rocm, tensors, p)
    tensors[1]["gradient"][3, 4] = np.nan
    got = run(rocm, tensors, p)
    for i in (0, 2):
        assert all(np.array_equal(got[i][n], clean[i][n]) for n in got[i])
    assert np.isnan(got[1]["next_parameters"]).any() and np.isnan(got[1]["next_momentum"]).sum() == 1


@gpu
def test_a_graph_replays_steps(rocm):
    lib, h = rocm.device.lib, rocm.device.handle
    tensors, p = tensors_of(15, [(100, 140), (520, 512)]), settings()
    want = tensors
    for _ in range(3):
        want = [dict(t, parameters=r["next_parameters"], momentum=r["next_momentum"]) for t, r in zip(want, run(rocm, want, p))]
    arrays = [{n: rocm.array(a) for n, a in t.items()} for t in tensors]
    table = (capi.MuonTensor * 2)(*[capi.MuonTensor(a["parameters"].ptr, a["gradient"].ptr, a["momentum"].ptr, a["parameters"].ptr, a["momentum"].ptr, *t["parameters"].shape) for t, a in zip(tensors, arrays)])
    w, size = workspace(rocm, table, 2)
    rocm.sync()
    assert lib.rlt_rocm_graph_begin_capture(h) == 0
    rocm.call("muon_step", table, 2, C.byref(capi.MuonParameters(**p)), w.ptr, size)
    graph = C.c_void_p()
    assert lib.rlt_rocm_graph_end_capture(h, C.byref(graph)) == 0
    for _ in range(3):
        w.upload(np.zeros(w.shape, np.uint8))      # eager work between the replays
        assert lib.rlt_rocm_graph_launch(h, graph) == 0
        rocm.sync()
    for a, t in zip(arrays, want):
        assert np.array_equal(a["parameters"].numpy(), t["parameters"]) and np.array_equal(a["momentum"].numpy(), t["momentum"])
    lib.rlt_rocm_graph_destroy(h, graph)


def test_refusals_without_a_device():
    lib = package().load_library()
    size = lambda *shapes: lib.rlt_rocm_muon_workspace_bytes((capi.MuonTensor * len(shapes))(*[capi.MuonTensor(0, 0, 0, 0, 0, *s) for s in shapes]), len(shapes))
    assert size((4, 5)) > 0 and size((4, 5), (6, 7)) > size((4, 5))
    assert size((0, 5)) == size((4, -1)) == size((4, 5), (3, 2 ** 16 + 1)) == size((2 ** 16, 2 ** 15)) == lib.rlt_rocm_muon_workspace_bytes(None, 1) == 0
    assert lib.rlt_rocm_muon_step(None, None, 0, None, None, 0) == capi.RLT_E_NOT_INITIALISED


@gpu
def test_refusals(rocm):
    lib, h = rocm.device.lib, rocm.device.handle
    buffers = [rocm.zeros((8, 8)) for _ in range(10)]
    ptr = [b.ptr for b in buffers]

    def step(entries=(tuple(ptr[:5]) + (8, 8),), n=None, p=settings(), offset=0, short=0):
        table = (capi.MuonTensor * len(entries))(*[capi.MuonTensor(*e) for e in entries])
        w, size = workspace(rocm, (capi.MuonTensor * 2)(*[capi.MuonTensor(0, 0, 0, 0, 0, 8, 8)] * 2), 2)
        size = lib.rlt_rocm_muon_workspace_bytes(table, len(entries)) if short else size
        return lib.rlt_rocm_muon_step(h, table, len(entries) if n is None else n, C.byref(capi.MuonParameters(**p)) if p else None, w.ptr + offset, size - short)
    first, second = tuple(ptr[:5]) + (8, 8), tuple(ptr[5:]) + (8, 8)
    assert step() == step((first, second)) == 0
    bad = capi.RLT_E_INVALID_ARGUMENT
    for i in range(5):
        assert step((first[:i] + (None,) + first[i + 1:],)) == bad
    assert step((first[:5] + (0, 8),)) == step((first[:5] + (8, -1),)) == step(n=0) == step(p=None) == step(offset=8) == step(short=1) == bad
    assert step(p=settings(iterations=0)) == step(p=settings(iterations=33)) == step(p=settings(epsilon=-1.0)) == step(p=settings(epsilon=float("nan"))) == bad
    assert step((first, first)) == step((first, second[:3] + (first[3], second[4], 8, 8))) == step((first, second[:4] + (first[4], 8, 8))) == bad      # a matrix twice
    assert step((first[:3] + (first[1], first[4], 8, 8),)) == step((first[:4] + (first[3], 8, 8),)) == step((first[:4] + (first[0], 8, 8),)) == bad      # buffers that overlap
    for i in range(5):      # what one matrix writes and another reads
        for written in (3, 4):
            assert step((first, second[:i] + (first[written],) + second[i + 1:])) == bad
    assert step((first, second[:1] + (first[1],) + second[2:])) == 0      # a gradient that two read
    assert step((first[:5] + (2 ** 16 + 1, 1),)) == step((first[:5] + (2 ** 16, 2 ** 15),)) == capi.RLT_E_UNSUPPORTED
    rocm.sync()

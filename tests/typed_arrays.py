"""Arrays of either element type of the C ABI (float32, bfloat16) for tests: bfloat16 travels as uint16, rounded to nearest, ties to even."""
import numpy as np

UNIT = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8}      # half a unit in the last place, relative


def to_bits(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return np.where(np.isnan(x), 0x7FC0, (u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def rounded(x, dtype):
    """x as the type holds it, in float64"""
    x = np.asarray(x, np.float32)
    return (x if dtype == "float32" else (to_bits(x).astype(np.uint32) << 16).view(np.float32)).astype(np.float64)


def upload(rocm, x, dtype):
    return rocm.array(np.asarray(x, np.float32) if dtype == "float32" else to_bits(np.asarray(x, np.float32)))


def download(array, dtype):
    a = array.numpy()
    return (a if dtype == "float32" else (a.astype(np.uint32) << 16).view(np.float32)).astype(np.float64)


def filled(rocm, shape, dtype, value=7.0):
    """an output buffer whose old content a test would notice"""
    return upload(rocm, np.full(shape, value, np.float32), dtype)

"""The operators around a transformer's blocks at the ends of their ranges: 8-bit values next to a border between two of them, masks and maxima of any
finite size, rows of many millions of elements, positions beyond 2^29, weights and epsilons next to the ends of f32.

Tolerances count roundings, as beside the other tests of these operators."""
import ctypes as C

import numpy as np
import pytest

from block_util import F32_STEP, Guarded, Kind, near, up

pytestmark = pytest.mark.gpu
TYPES = ["f32", "f16", "bf16"]
P = C.c_void_p


# ---- 8 bits: the f32 quotient by the scale, to nearest, ties to even ---------------------------------------

def borders(fmt):
    """Half way between each two neighbouring values of the format that are not negative."""
    v = np.arange(128.0) if fmt == "i8" else np.array([(b & 7) * 2.0 ** -9 if b < 8 else (8 + (b & 7)) * 2.0 ** ((b >> 3) - 10) for b in range(127)])
    return (v[1:] + v[:-1]) / 2


def beside_borders(rng, fmt, n, most):
    """n numbers up to `most`, which is the first: borders times the scale, and a few places to both sides."""
    top = np.float32(127 if fmt == "i8" else 448)
    s = np.float32(most) / top
    y = (rng.choice(borders(fmt), n) * np.float64(s)).astype(np.float32)
    for _ in range(3):
        y = np.where(rng.uniform(size=n) < 0.5, np.nextafter(y, rng.choice([0, np.inf], n).astype(np.float32)), y)
    y = np.minimum(y, np.float32(most)) * rng.choice([-1, 1], n).astype(np.float32)
    y[0] = most
    return y.astype(np.float32)


def codes(fmt, quotient):
    if fmt == "i8":
        return np.rint(quotient).astype(np.int8)
    at, b = np.abs(quotient).astype(np.float64), borders(fmt)
    code = np.searchsorted(b, at)  # (the lower code on a border, which is right where it is even)
    code += (code < len(b)) & (code % 2 == 1) & (at == b[np.minimum(code, len(b) - 1)])
    return (code + 128 * np.signbit(quotient)).astype(np.uint8)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("cols,group", [(64, 0), (77, 0), (5120, 0), (1001, 0), (1024, 128), (4096, 64), (1001, 7), (5000, 1000), (70000, 0), (70000, 1000)])
def test_8_bit_values_are_the_quotients(hpt, dev, fmt, name, cols, group):
    """Rows of ones and of their negatives: the norm is +-gamma, exactly."""
    k, rng = Kind(hpt, name), np.random.default_rng(cols + group)
    each = group or cols
    mosts = rng.uniform(0.5, 3, cols // each) * 2.0 ** rng.integers(-14, 14, cols // each)
    g, gamma = k.up(np.concatenate([beside_borders(rng, fmt, each, k.round(m)) for m in mosts]))
    x, h = k.up(np.array([1, -1, 1, -1, -1])[:, None] * np.ones(cols))
    y = (h * gamma).astype(np.float32).reshape(5, -1, each)
    scale = np.abs(y).max(-1, keepdims=True) / np.float32(127 if fmt == "i8" else 448)
    want = codes(fmt, y / scale)
    if name == "f32" and each >= 1000:
        assert (codes(fmt, y * (1 / scale)) != want).any(), "these numbers tell a quotient from a product with the reciprocal"
    q, s = Guarded(hpt, [5, cols], hpt.i8 if fmt == "i8" else hpt.u8), Guarded(hpt, [5, cols // each], hpt.f32)
    x.rms_norm_quant([cols], g, 1e-30, format=fmt, group=group, out=q.t, scale_out=s.t)
    assert np.array_equal(s.numpy(), scale[..., 0])
    assert np.array_equal(q.numpy(), want.reshape(5, cols))
    half, _ = k.up(h / 2)
    a, b, _ = half.rms_norm_quant([cols], g, 1e-30, residual=half, format=fmt, group=group)
    assert np.array_equal(a.numpy(), q.numpy()) and np.array_equal(b.numpy().reshape(-1), s.numpy().reshape(-1))


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("power", [-124, -112, -90, 90, 110])
def test_8_bit_values_of_tiny_and_huge_norms(hpt, dev, fmt, power):
    cols, rng = 2048, np.random.default_rng(3)
    gamma = beside_borders(rng, fmt, cols, 1.3 * 2.0 ** power)
    x = hpt.Tensor.ones([2, cols], hpt.f32)
    scale = np.maximum(np.abs(gamma).max() / np.float32(127 if fmt == "i8" else 448), np.float32(2.0 ** -120))
    q, s = x.rms_norm_quant([cols], up(hpt, gamma), 1e-30, format=fmt)
    assert (s.numpy() == scale).all()
    assert np.array_equal(q.numpy(), np.broadcast_to(codes(fmt, gamma / scale), (2, cols)))

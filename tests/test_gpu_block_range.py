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


# ---- logits of any finite size --------------------------------------------------------------------------------

LSE = 128 * F32_STEP  # absolute, of the log of the sum
MASKS = [-1e4, -65504.0, -9e4, -1.2e5, -2e5, -1e6, -1e9, -1e10, -1e12, -1e20, -1e30, -1e37, -1.6e38, -3e38]


def logsumexp(x):
    m = x.max(-1, keepdims=True)
    return (m + np.log(np.exp(x - m).sum(-1, keepdims=True)))[..., 0]


def masked_rows(x, v):
    """Rows of which all, a stretch, or all but a few logits are v."""
    n = x.shape[-1]
    stretches = [slice(0, n), slice(0, n // 2), slice(n // 2, n), slice(n // 3, 2 * n // 3), slice(1, n), slice(0, n - 1), slice(0, n, 2), slice(0, 0)]
    for i in range(len(x)):
        x[i, stretches[i % len(stretches)]] = v
    x[-1] = v
    x[-1, n // 2] = 0.5
    return x


def check_rows(hpt, k, x, what):
    """Log-probabilities of both ends of each row's range, and the loss with its gradient, against 64 bits."""
    t, x = k.up(x)
    rows = len(x)
    lse = logsumexp(x)
    for token in (x.argmax(-1), x.argmin(-1)):
        logp = (x[np.arange(rows), token] - x.max(-1)) - (lse - x.max(-1) if np.abs(x).max() < 1e3 else logsumexp(x - x.max(-1, keepdims=True)))
        a, b = t.token_logp(up(hpt, token))
        near(a.numpy(), logp, LSE + F32_STEP * np.abs(logp), f"logp {what}")
        near(b.numpy(), lse, LSE + F32_STEP * np.abs(lse), f"lse {what}")
    token = x.argmax(-1)
    logp = -logsumexp(x - x.max(-1, keepdims=True))
    old = (logp + 0.05).astype(np.float32)
    adv = np.where(np.arange(rows) % 2, 1, -1).astype(np.float32)
    r = t.policy_loss(up(hpt, token), up(hpt, old), up(hpt, adv))
    ratio = np.exp(logp - old.astype(np.float64))
    near(r.weight.numpy(), -ratio * adv / rows, (LSE * ratio + 4 * F32_STEP) / rows, f"weight {what}")
    near(r.loss.numpy()[0], (-ratio * adv).mean(), (LSE * ratio + 4 * F32_STEP).mean(), f"loss {what}")
    d = k.down(t.policy_loss_backward(up(hpt, token), r.lse, r.weight, 64.0))
    assert np.isfinite(d).all(), what


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,cols", [(9, 50), (9, 5000), (9, 40000), (2100, 70)])
def test_finite_masks_of_any_size(hpt, dev, name, rows, cols):
    """Whole rows, stretches that whole threads, wavefronts and parts of a split row meet nothing else of, and all but one."""
    k, rng = Kind(hpt, name), np.random.default_rng(cols)
    for v in MASKS:
        if name != "f16" or v >= -65504:
            check_rows(hpt, k, masked_rows(rng.standard_normal((rows, cols)) * 3, v), f"mask {v}")


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("cols", [50, 5000, 40000])
def test_maxima_of_any_size(hpt, dev, name, cols):
    """One logit far above the others, and rows that lie far from zero as a whole."""
    k, rng = Kind(hpt, name), np.random.default_rng(cols)
    for v in [-m for m in MASKS]:
        if name == "f16" and v > 65504:
            continue
        x = rng.standard_normal((9, cols)) * 3
        x[np.arange(9), rng.integers(0, cols, 9)] = v
        x[0] = v
        x[1, ::2] = v
        check_rows(hpt, k, x, f"maximum {v}")
    for c in (1e3, 3e4, 6e4, 8.9e4, 9.2e4, 1e5, 1.7e5, 1.9e5, 1e6, 1e7):
        for sign in (1, -1):
            if name == "f16" and c > 6e4:
                continue
            # of both sides of a stretch, a few apart, in either order
            x = sign * c + rng.standard_normal((6, cols)) * 3
            x[1, : cols // 2] += 4
            x[2, cols // 2:] += 4
            x[3, cols // 3: cols // 2] -= 5000
            x[4, : cols // 2] -= 90000 if name != "f16" else 5000
            x[5, cols // 2:] -= 90000 if name != "f16" else 5000
            if name == "f16":
                x = np.clip(x, -65504, 65504)
            check_rows(hpt, k, x, f"around {sign * c}")


# ---- scores of any finite size --------------------------------------------------------------------------------

def softmax(s):
    e = np.exp(s - s.max(-1, keepdims=True))
    return e / e.sum(-1, keepdims=True)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("n,queries", [(40, 24), (1000, 24), (2056, 24), (9000, 24), (70000, 24), (1500, 1)])
def test_masks_and_maxima_of_any_size(hpt, dev, name, n, queries):
    """Queries all of whose keys a caller has masked with one finite number, part of them, or one key far above the others. The scores that the
    probabilities are taken of are scale * x + bias in f32: what they say is computed from those."""
    k, rng = Kind(hpt, name), np.random.default_rng(n)
    low = {"f32": np.finfo(np.float32).min, "f16": -65504.0, "bf16": -3.3895313892515355e38}[name]
    values = [v for v in (-1e4, -6e4, -9e5, -1.3e6, -1e9, -1e10, -1e12, -1e15, -1e20, -1e30, -1e37, low) if name != "f16" or v >= -65504]
    values += [-v for v in values]
    tab, table = k.up(np.array([0, 1, -1, 2, 0.5, -0.5, 1.5, 3])[:, None])
    q, j = np.arange(queries)[:, None], np.arange(n)
    d = q + (n - queries) - j
    bias = table[:, 0][np.where(d < 4, np.maximum(d, 0), np.minimum(7, 4 + np.floor(np.log2(np.maximum(d, 1) / 4) / 2 * 4 + 1e-9).astype(int)))]
    for scale in (1.0, 0.125, 0.0884):
        sc = np.float64(np.float32(scale))
        for first in range(0, len(values), queries):
            some = values[first:first + queries]
            for pattern in ("all", "part", "one"):
                x = rng.standard_normal((queries, n)) * 4
                for i, v in enumerate(some):
                    if pattern == "all":
                        x[i] = v
                    elif pattern == "part":
                        x[i, n // 3: n - 5] = v
                    else:
                        x[i, rng.integers(0, n)] = v
                t, x = k.up(x[None, None])
                s = (sc * x[0, 0] + bias).astype(np.float32).astype(np.float64)
                want = softmax(s)
                got = k.down(t.softmax_bias(tab, scale, bidirectional=False, max_distance=16, query_offset=n - queries))[0, 0]
                # a difference of two scores is rounded once, and twice on its way to a power of two: it is weighted with e^-difference <= 1 / difference
                near(got, want, want * (k.step + (100 + 3 * np.minimum(s.max(-1, keepdims=True) - s, 200)) * F32_STEP) + k.least, f"{pattern} {some[:2]} scale {scale}")


# ---- rows of many millions of elements --------------------------------------------------------------------------

@pytest.fixture()
def hip():
    h = C.CDLL("libamdhip64.so")
    h.hipStreamCreateWithFlags.argtypes = [C.POINTER(P), C.c_uint]
    h.hipStreamBeginCapture.argtypes = [P, C.c_int]
    h.hipStreamEndCapture.argtypes = [P, C.POINTER(P)]
    h.hipGraphInstantiate.argtypes = [C.POINTER(P), P, P, P, C.c_size_t]
    h.hipGraphLaunch.argtypes = [P, P]
    for f in (h.hipStreamSynchronize, h.hipGraphExecDestroy, h.hipGraphDestroy, h.hipStreamDestroy):
        f.argtypes = [P]
    return h


def captured(hip, call):
    """The call recorded without a workspace, so in the form without scratch, and replayed once."""
    s, g, e = P(), P(), P()
    assert hip.hipStreamCreateWithFlags(C.byref(s), 1) == 0
    try:
        assert hip.hipStreamBeginCapture(s, 0) == 0
        try:
            call(s)
        finally:
            rc = hip.hipStreamEndCapture(s, C.byref(g))
        assert rc == 0 and g.value and hip.hipGraphInstantiate(C.byref(e), g, None, None, 0) == 0
        assert hip.hipGraphLaunch(e, s) == 0 and hip.hipStreamSynchronize(s) == 0
        hip.hipGraphExecDestroy(e)
        hip.hipGraphDestroy(g)
    finally:
        hip.hipStreamDestroy(s)


def part(hpt, t, first, n):
    """n elements of a tensor's memory."""
    return hpt.Tensor.from_raw(t.ptr + first * t.dtype.size, [n], t.dtype)


LONG = 1 << 26  # elements of a row: 65536 of a thread, whose sum in f32, term by term, would be off by 1e-4 and more
# A vector's sum in f32 (up to 16 terms, or 32 logits with their exponentials), the rest in 64 bits, a rounding, a root, a reciprocal and products: below 64 half steps.
SUM = 64 * F32_STEP


@pytest.mark.parametrize("residual", [False, True])
def test_norm_of_a_long_row(hpt, dev, residual):
    x = hpt.Tensor.full(1.1, [1, LONG], hpt.f32)
    v = np.float64(np.float32(1.1))
    if residual:
        r = hpt.Tensor.full(0.2, [1, LONG], hpt.f32)
        v = np.float64(np.float32(1.1) + np.float32(0.2))
        y, _ = x.add_rms_norm(r, [LONG], None, 0.25, sum_out=r)
    else:
        y = x.rms_norm([LONG], None, 0.25)
    want = v / np.sqrt(v * v + 0.25)
    for first in (0, LONG - 100):
        near(part(hpt, y, first, 100).numpy(), np.full(100, want), (SUM + F32_STEP) * want)


@pytest.mark.parametrize("name", TYPES)
def test_8_bit_norm_of_a_long_row(hpt, dev, name):
    k = Kind(hpt, name)
    v = float(k.round([1.1])[0])
    _, s = hpt.Tensor.full(1.1, [1, LONG], k.dtype).rms_norm_quant([LONG], None, 0.25)
    want = v / np.sqrt(v * v + 0.25) / 127
    near(s.numpy(), [want], (SUM + 2 * F32_STEP) * want)


def test_norm_gradient_of_a_long_row(hpt, dev):
    x, gy = hpt.Tensor.full(1.1, [1, LONG], hpt.f32), hpt.Tensor.full(0.7, [1, LONG], hpt.f32)
    a, b = np.float64(np.float32(1.1)), np.float64(np.float32(0.7))
    r = 1 / np.sqrt(a * a + 0.25)
    gx, gg = x.rms_norm_backward(gy, [LONG], None, 0.25)
    size = r * (b + a * r * r * a * b)
    for first in (0, LONG - 100):
        near(part(hpt, gx, first, 100).numpy(), np.full(100, r * (b - a * r * r * a * b)), (2 * SUM + F32_STEP) * size)
        near(part(hpt, gg, first, 100).numpy(), np.full(100, a * b * r), (SUM + F32_STEP) * a * b * r)


def test_softmax_of_a_long_row(hpt, dev, hip):
    """One score of 0, all others -0.1: split, and as a whole."""
    x = hpt.Tensor.full(-0.1, [1, 1, LONG], hpt.f32)
    assert hpt.lib().hpt_hip_memcpy_h2d_sync(0, P(x.ptr + 4 * 5), np.zeros(1, np.float32).ctypes.data_as(P), 4) == 0
    tab = hpt.Tensor.zeros([8, 1], hpt.f32)
    e = np.exp(np.float64(np.float32(-0.1)))
    total = 1 + (LONG - 1) * e
    out = hpt.Tensor.zeros([1, 1, LONG], hpt.f32)

    def check(y):
        for first in (6, LONG - 100):
            near(part(hpt, y, first, 100).numpy(), np.full(100, e / total), (F32_STEP + SUM) * e / total)
        near(part(hpt, y, 5, 1).numpy(), [1 / total], (F32_STEP + SUM) / total)

    check(x.softmax_bias(tab, max_distance=16))
    captured(hip, lambda s: x.softmax_bias(tab, max_distance=16, out=out, stream=s))
    check(out)


def test_softmax_gradient_of_a_long_row(hpt, dev):
    """All gradients alike: those of the scores are zeros, but for roundings of what cancels."""
    p, g = hpt.Tensor.full(2.0 ** -26, [1, 1, LONG], hpt.f32), hpt.Tensor.full(1.1, [1, 1, LONG], hpt.f32)
    gx, gt = p.softmax_bias_backward(g, 8, max_distance=16)
    for first in (0, LONG - 100):
        near(part(hpt, gx, first, 100).numpy(), np.zeros(100), (SUM + 4 * F32_STEP) * 1.1 * 2.0 ** -26)
    near(gt.numpy(), np.zeros((8, 1)), (SUM + 64 * F32_STEP) * 1.1)


@pytest.mark.parametrize("top", [0.0, 2.0 ** 18, 2.0 ** 20])
def test_log_probability_of_a_long_row(hpt, dev, hip, top):
    """One logit of `top`, all others an eighth below: split, and as a whole."""
    x = hpt.Tensor.full(top - 0.125, [1, LONG], hpt.f32)
    assert hpt.lib().hpt_hip_memcpy_h2d_sync(0, P(x.ptr + 4 * 7), np.full(1, top, np.float32).ctypes.data_as(P), 4) == 0
    token = up(hpt, np.array([7]))
    rest = np.log(1 + (LONG - 1) * np.exp(-0.125))
    logp, lse = hpt.Tensor.zeros([1], hpt.f32), hpt.Tensor.zeros([1], hpt.f32)

    def check(logp, lse):
        near(logp.numpy(), [-rest], (SUM + 32 * F32_STEP))
        near(lse.numpy(), [top + rest], SUM + 32 * F32_STEP + F32_STEP * top)

    check(*x.token_logp(token))
    captured(hip, lambda s: x.token_logp(token, logp_out=logp, lse_out=lse, stream=s))
    check(logp, lse)


# ---- positions beyond 2^29 ---------------------------------------------------------------------------------------

def test_a_query_beyond_two_to_the_29(hpt, dev):
    """A query some places behind the last of nearly 2^29 keys: the buckets of their distances, forward and backward."""
    k = Kind(hpt, "bf16")
    n, tail = (1 << 29) - 2, 256
    offset = (1 << 29) + 5
    begin = [0, 1, 2, 3, 4, 8, 16, 32]  # 8 buckets, distances up to 64
    d = offset - np.arange(n - tail, n)
    which = np.array([max(b for b in range(8) if begin[b] <= v) for v in d])
    x = hpt.Tensor.zeros([1, 1, n], hpt.bf16)
    tab, table = k.up(np.array([0, 1, 2, 3, 4, 5, 6, 0.5])[:, None])
    p = x.softmax_bias(tab, bidirectional=False, max_distance=64, query_offset=offset, out=x)
    near_ones = np.exp(table[which, 0])
    total = (n - tail) * np.exp(0.5) + near_ones.sum()
    assert sorted(set(which)) == [5, 6, 7], "the last keys are in the buckets before the last one"
    # (scores up to 6: 4 * 6 + 72 half steps as for any probabilities, and as much again for each of the steps between the parts of a row; 400 covers them)
    near(k.down(part(hpt, p, n - tail, tail)), near_ones / total, near_ones / total * (k.step + 400 * F32_STEP))
    g = hpt.Tensor.zeros([1, 1, n], hpt.bf16)
    ones, last = k.up(np.ones(tail))
    assert hpt.lib().hpt_hip_memcpy_d2d_sync(0, P(g.ptr + 2 * (n - tail)), P(ones.ptr), 2 * tail) == 0
    p_tail = k.down(part(hpt, p, n - tail, tail))
    gt = p.softmax_bias_backward(g, 8, bidirectional=False, max_distance=64, query_offset=offset, out=p)[1].numpy()[:, 0]
    s = p_tail.sum()
    want = np.array([(p_tail * (1 - s))[which == b].sum() for b in range(8)])
    assert not gt[:5].any()
    near(gt[5:7], want[5:7], 400 * F32_STEP * want[5:7])


# ---- weights of the mask next to the ends of f32 -----------------------------------------------------------------

@pytest.mark.parametrize("size", [1e-38, 1e-30, 1.0, 1e30, 1e37])
@pytest.mark.parametrize("rows,cols", [(2100, 40), (9, 40)])
def test_a_mask_of_any_size(hpt, dev, rows, cols, size):
    """The mask's weights are relative: all of them 1e-38 or 1e37 are the same as all of them 1."""
    k, rng = Kind(hpt, "f32"), np.random.default_rng(rows)
    t, x = k.up(rng.standard_normal((rows, cols)) * 3)
    token = rng.integers(0, cols, rows)
    logp = x[np.arange(rows), token] - logsumexp(x)
    old, adv = (logp + 0.05).astype(np.float32), (rng.standard_normal(rows) * 30).astype(np.float32)
    mask = np.full(rows, size, np.float32)
    r = t.policy_loss(up(hpt, token), up(hpt, old), up(hpt, adv), mask=up(hpt, mask))
    each = -np.exp(logp - old.astype(np.float64)) * adv
    near(r.weight.numpy(), each / rows, (LSE + 4 * F32_STEP) * np.abs(each) / rows)
    near(r.loss.numpy()[0], each.mean(), (LSE + 4 * F32_STEP) * np.abs(each).mean())


@pytest.mark.parametrize("cols", [1, 3])
def test_norm_gradient_of_millions_of_rows_shorter_than_a_vector(hpt, dev, cols):
    """The gradient of gamma, thousands of rows for each workgroup."""
    rows = 1 << 22
    x, gy = hpt.Tensor.full(1.1, [rows, cols], hpt.f32), hpt.Tensor.full(0.7, [rows, cols], hpt.f32)
    a, b = np.float64(np.float32(1.1)), np.float64(np.float32(0.7))
    want = rows * a * b / np.sqrt(a * a + 0.25)
    near(x.rms_norm_backward(gy, [cols], None, 0.25)[1].numpy(), np.full(cols, want), SUM * want)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("grad", [float("inf"), float("-inf"), float("nan"), 1e300, 2.0])
def test_a_row_of_weight_0_has_no_gradient(hpt, dev, name, grad):
    """Whatever the logits and the loss's gradient are (a loss scale that has overflowed)."""
    k, rng = Kind(hpt, name), np.random.default_rng(1)
    x = rng.standard_normal((3, 5003))
    x[1] = np.nan
    t, x = k.up(x)
    zero = hpt.Tensor.zeros([3], hpt.f32)
    weight = up(hpt, np.array([1, 0, -0.0], np.float32))
    got = k.down(t.policy_loss_backward(up(hpt, np.array([3, -100, 4])), zero, weight, grad))
    assert not got[1:].any()
    if grad == 2.0:
        assert np.isfinite(got[0]).all() and got[0].any()


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [5, 64, 1001, 4096, 40000])
@pytest.mark.parametrize("eps", [1e-12, 1e-38, 1e-40])
def test_gradient_of_rows_of_zeros(hpt, dev, name, cols, eps):
    """1 / sqrt(eps) times the gradient, also where 1 / eps is beyond f32."""
    k, rng = Kind(hpt, name), np.random.default_rng(cols)
    x = rng.standard_normal((5, cols))
    x[::2] = 0
    t, x = k.up(x)
    gy, grad = k.up(rng.standard_normal((5, cols)))
    gx, gg = t.rms_norm_backward(gy, [cols], None, eps)
    e = np.float64(np.float32(eps))
    want = grad[::2] / np.sqrt(e)
    near(k.down(gx)[::2], want, (k.step + 64 * F32_STEP) * np.abs(want))
    assert np.isfinite(k.down(gx)).all() and np.isfinite(gg.numpy()).all()

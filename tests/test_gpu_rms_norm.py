"""RMS norm on the device against the definition in 64 bits: with the residual's addition, in 8 bits with scales, backward.

Tolerances count roundings. A result is off by half a step of its type, and by what the f32 arithmetic before it adds: a row's
sum of squares is a tree over threads that add up to ROW_TERMS terms each, so 1 / sqrt of it is off by (ROW_TERMS + 20) / 2 + 2
half steps of f32 at most, and two products follow; F32 = 64 half steps covers rows of up to 80 terms a thread."""
import numpy as np
import pytest

from block_util import F32_STEP, Guarded, Kind, near, shifted, up

pytestmark = pytest.mark.gpu
F32 = 64 * F32_STEP
EPS = 1e-6
TYPES = ["f32", "f16", "bf16"]


def rms(h, gamma, eps=EPS):
    r = 1 / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    return h * r * (1 if gamma is None else gamma)


def hidden(rng, rows, cols):
    """Rows of different size, a few channels that stand out."""
    return rng.standard_normal((rows, cols)) * rng.uniform(0.3, 3, (rows, 1)) * (0.5 + 10 * rng.uniform(0, 1, cols) ** 8)


def total(hpt, k, x, r):
    return k.round(x.astype(np.float32) + r.astype(np.float32))


SHAPES = [(1, 1), (3, 2), (5, 7), (2, 8), (700, 9), (33, 64), (1000, 96), (17, 127), (300, 128), (65, 257), (9, 512), (130, 1000), (3, 1001), (40, 2048),
          (7, 4099), (33, 5120), (4, 8200), (2, 16384), (3, 20001), (2, 32768), (2, 65536), (1, 70001)]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_norm(hpt, dev, name, rows, cols):
    k, rng = Kind(hpt, name), np.random.default_rng(rows * 7 + cols)
    t, x = k.up(hidden(rng, rows, cols))
    g, gamma = k.up(rng.normal(1, 0.2, cols))
    out = Guarded(hpt, [rows, cols], k.dtype)
    t.rms_norm([cols], g, EPS, out=out.t)
    want = rms(x, gamma)
    near(k.load(out.numpy()), want, (k.step + F32) * np.abs(want) + k.least, "rms_norm")
    plain = t.rms_norm([cols])
    want = rms(x, None)
    near(k.down(plain), want, (k.step + F32) * np.abs(want) + k.least, "without gamma")
    # with a residual: the sum as an addition of its own stores it
    r, res = k.up(rng.standard_normal((rows, cols)))
    out, added = Guarded(hpt, [rows, cols], k.dtype), Guarded(hpt, [rows, cols], k.dtype)
    t.add_rms_norm(r, [cols], g, EPS, out=out.t, sum_out=added.t)
    h = total(hpt, k, x, res)
    assert np.array_equal(k.load(added.numpy()), h)
    want = rms(h, gamma)
    near(k.load(out.numpy()), want, (k.step + F32) * np.abs(want) + k.least, "add_rms_norm")
    y, s = t.add_rms_norm(r, [cols], g, EPS)
    assert np.array_equal(y.numpy(), out.numpy()) and np.array_equal(s.numpy(), added.numpy())
    assert np.array_equal(s.numpy(), t.add(r).numpy()), "the sum is the framework's own"


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("shift", [(0, 0, 1), (1, 0, 0), (3, 2, 1), (0, 1, 0)])
@pytest.mark.parametrize("cols", [64, 520, 4096, 9, 40000])
def test_norm_off_the_grid(hpt, dev, name, shift, cols):
    """Operands and results that start anywhere."""
    k, rng = Kind(hpt, name), np.random.default_rng(cols)
    rows = 5
    t, x, b1 = shifted(hpt, k, hidden(rng, rows, cols), shift[0])
    g, gamma, b2 = shifted(hpt, k, rng.normal(1, 0.2, cols), shift[1])
    r, res, b3 = shifted(hpt, k, rng.standard_normal((rows, cols)), shift[1])
    out, added = Guarded(hpt, [rows, cols], k.dtype, shift[2]), Guarded(hpt, [rows, cols], k.dtype, shift[1])
    t.add_rms_norm(r, [cols], g, EPS, out=out.t, sum_out=added.t)
    h = total(hpt, k, x, res)
    assert np.array_equal(k.load(added.numpy()), h)
    want = rms(h, gamma)
    near(k.load(out.numpy()), want, (k.step + F32) * np.abs(want) + k.least)
    gx, gg = Guarded(hpt, [rows, cols], k.dtype, shift[2]), Guarded(hpt, [cols], hpt.f32, shift[1])
    t.rms_norm_backward(r, [cols], g, EPS, out=gx.t, gamma_out=gg.t)
    check_grad(k, x, res, gamma, None, k.load(gx.numpy()), gg.numpy(), rows)


@pytest.mark.parametrize("name", TYPES)
def test_strided_rows(hpt, dev, name):
    """Rows that lie apart: a slice of wider ones, heads of a packed product, reversed, broadcast."""
    k, rng = Kind(hpt, name), np.random.default_rng(3)
    t, x = k.up(hidden(rng, 40, 640).reshape(8, 5, 10, 64))
    g, gamma = k.up(rng.normal(1, 0.2, 64))
    views = [("heads 2 to 7", t[:, :, 2:7], x[:, :, 2:7]), ("every second token", t[::2], x[::2]), ("turned", t.permute([1, 0, 2, 3]), x.transpose(1, 0, 2, 3)),
             ("backwards", t[:, ::-1], x[:, ::-1]), ("a part of each row", t[:, :, :, 8:40], x[:, :, :, 8:40]), ("an odd part", t[:, :, :, 3:40], x[:, :, :, 3:40])]
    row, one = k.up(hidden(rng, 1, 64))
    views.append(("broadcast", row.expand([6, 64]), np.broadcast_to(one, (6, 64))))
    for what, v, a in views:
        c = a.shape[-1]
        gv, ga = (g, gamma) if c == 64 else (None, None)
        want = rms(a, ga)
        near(k.down(v.rms_norm([c], gv)), want, (k.step + F32) * np.abs(want) + k.least, what)
        gy, grad = k.up(rng.standard_normal(a.shape))
        gx, gg = v.rms_norm_backward(gy, [c], gv, EPS)
        check_grad(k, a.reshape(-1, c), grad.reshape(-1, c), ga, None, k.down(gx).reshape(-1, c), gg.numpy(), a.size // c)
    # two normalised dims
    want = rms(x.reshape(8, 5, 640), None).reshape(x.shape)
    near(k.down(t.rms_norm([10, 64])), want, (k.step + F32) * np.abs(want) + k.least, "two dims")


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("cols", [63, 256, 4096, 5001, 70000])
def test_in_place(hpt, dev, name, cols):
    """Each result in the place of each operand that it may take."""
    k, rng = Kind(hpt, name), np.random.default_rng(cols)
    rows = 6
    x, res, gamma = hidden(rng, rows, cols), rng.standard_normal((rows, cols)), rng.normal(1, 0.2, cols)
    up3 = lambda: (k.up(x)[0], k.up(res)[0], k.up(gamma)[0])  # noqa: E731
    t, r, g = up3()
    y, s = (v.numpy() for v in t.add_rms_norm(r, [cols], g, EPS))
    n = t.rms_norm([cols], g, EPS).numpy()
    for where in ("sum in the residual", "sum in the input", "output in the input", "output in the residual", "both"):
        t, r, g = up3()
        out, added = {"sum in the residual": (None, r), "sum in the input": (None, t), "output in the input": (t, None), "output in the residual": (r, None),
                      "both": (t, r)}[where]
        a, b = t.add_rms_norm(r, [cols], g, EPS, out=out, sum_out=added)
        assert np.array_equal(a.numpy(), y) and np.array_equal(b.numpy(), s), where
    t, r, g = up3()
    assert np.array_equal(t.rms_norm([cols], g, EPS, out=t).numpy(), n)
    # backward
    t, r, g = up3()
    m, _ = k.up(x[::-1])
    gx, gg = (v.numpy() for v in t.rms_norm_backward(r, [cols], g, EPS, grad_sum=m))
    for which in range(3):
        t, r, g = up3()
        m, _ = k.up(x[::-1])
        a, b = t.rms_norm_backward(r, [cols], g, EPS, grad_sum=m, out=(t, r, m)[which])
        assert np.array_equal(a.numpy(), gx) and np.array_equal(b.numpy(), gg), which


# ---- 8 bits ------------------------------------------------------------------------------------------

E4M3 = np.array([(-1) ** (b >> 7) * (np.nan if b & 127 == 127 else (b & 7) * 2.0 ** -9 if not b & 120 else (8 + (b & 7)) * 2.0 ** ((b >> 3 & 15) - 10)) for b in range(256)])


def check_quant(q, s, y, group, fmt, slack):
    """Every value within half a step of y / scale, the scale that of the group's largest |y|."""
    rows, cols = y.shape
    most = np.abs(y.reshape(rows, cols // group, group)).max(-1)
    top = 127.0 if fmt == "i8" else 448.0
    want = np.maximum(most / top, 2.0 ** -120)
    s = s.reshape(want.shape).astype(np.float64)
    near(s, want, want * (slack + 2 * F32_STEP), "scales")
    each = np.repeat(s, group, 1)
    v = q.astype(np.float64) if fmt == "i8" else E4M3[q]
    assert np.isfinite(v).all() and np.abs(v).max() <= top
    off = np.abs(y) / each * (slack + 2 * F32_STEP)  # what y and the scale may be off, in steps of 1
    half = 0.5 if fmt == "i8" else np.maximum(2.0 ** np.floor(np.log2(np.maximum(np.abs(y) / each * (1 + 1e-4), 2.0 ** -6))) / 16, 2.0 ** -10)
    near(v, y / each, half + off + 1e-12, "values")


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,cols,group", [(1, 1, 0), (7, 5, 0), (4, 9, 3), (33, 64, 0), (33, 64, 32), (5, 96, 8), (17, 256, 64), (300, 1000, 0), (9, 1000, 8), (9, 1024, 256), (4, 1024, 512),
                                             (3, 1001, 7), (12, 4096, 128), (33, 5120, 0), (3, 5120, 64), (2, 20000, 0), (2, 70000, 0), (2, 70016, 128), (2, 70000, 1000), (1, 49, 49)])
def test_quant(hpt, dev, fmt, name, rows, cols, group):
    k, rng = Kind(hpt, name), np.random.default_rng(rows + cols + group)
    t, x = k.up(hidden(rng, rows, cols))
    g, gamma = k.up(rng.normal(1, 0.2, cols))
    r, res = k.up(rng.standard_normal((rows, cols)))
    out = Guarded(hpt, [rows, cols], hpt.i8 if fmt == "i8" else hpt.u8)
    sc = Guarded(hpt, [rows, cols // (group or cols)], hpt.f32)
    t.rms_norm_quant([cols], g, EPS, format=fmt, group=group, out=out.t, scale_out=sc.t)
    check_quant(out.numpy(), sc.numpy(), rms(x, gamma), group or cols, fmt, F32)
    q, s, h = t.rms_norm_quant([cols], None, EPS, residual=r, format=fmt, group=group)
    assert s.shape == ([rows, cols // group] if group else [rows])
    want = total(hpt, k, x, res)
    assert np.array_equal(k.down(h), want)
    check_quant(q.numpy(), s.numpy(), rms(want, None), group or cols, fmt, F32)
    # the sum in the residual's place
    q2, s2, h2 = t.rms_norm_quant([cols], None, EPS, residual=r, format=fmt, group=group, sum_out=r)
    assert np.array_equal(q2.numpy(), q.numpy()) and np.array_equal(s2.numpy(), s.numpy()) and np.array_equal(k.down(r), want)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("shift", [1, 2, 8])
def test_quant_off_the_grid(hpt, dev, fmt, shift):
    k, rng = Kind(hpt, "bf16"), np.random.default_rng(5)
    for cols, group in ((256, 0), (256, 64), (77, 11)):
        t, x, base = shifted(hpt, k, hidden(rng, 5, cols), shift)
        out = Guarded(hpt, [5, cols], hpt.i8 if fmt == "i8" else hpt.u8, shift)
        sc = Guarded(hpt, [5, cols // (group or cols)], hpt.f32, shift)
        t.rms_norm_quant([cols], format=fmt, group=group, out=out.t, scale_out=sc.t)
        check_quant(out.numpy(), sc.numpy(), rms(x, None), group or cols, fmt, F32)


@pytest.mark.parametrize("cols", [64, 96, 1001, 70000])
@pytest.mark.parametrize("name", TYPES)
def test_zeros_infinities_and_nan(hpt, dev, name, cols):
    k, rng = Kind(hpt, name), np.random.default_rng(1)
    x = hidden(rng, 6, cols)
    x[1], x[2, 3], x[3, cols - 1], x[4] = 0, np.nan, np.inf, 1e-30
    t, x = k.up(x)
    with np.errstate(invalid="ignore"):
        want = rms(x, None)
    want[3] = 0  # (an infinite sum of squares: everything finite is 0, the infinity NaN)
    want[3, cols - 1] = np.nan
    got = k.down(t.rms_norm([cols]))
    near(got, want, (k.step + F32) * np.abs(np.nan_to_num(want)) + 2 * k.least)
    for fmt, dt in (("i8", np.int8), ("e4m3", np.uint8)):
        for group in (0, cols // 7 if cols % 7 == 0 else 32 if cols % 32 == 0 else 0):
            q, s = (v.numpy() for v in t.rms_norm_quant([cols], format=fmt, group=group))
            assert q.dtype == dt
            s = s.reshape(6, -1)
            assert (s[1] == np.float32(2.0 ** -120)).all() and not q[1].any()
            assert np.isnan(s[2]).all()
            assert (q[2] == 0).all() if fmt == "i8" else np.isnan(E4M3[q[2]]).all()
            assert np.isnan(s[3, -1]) and (s[3, :-1] == np.float32(2.0 ** -120)).all()


# ---- backward ----------------------------------------------------------------------------------------

def grads(x, gy, gamma, more, eps=EPS):
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    gg = gy if gamma is None else gy * gamma
    c = r * r * (gg * x).mean(-1, keepdims=True)
    gx = r * (gg - x * c)
    ca = r * r * np.abs(gg * x).mean(-1, keepdims=True)
    size = r * (np.abs(gg) + np.abs(x) * ca)  # what the terms are before they cancel
    if more is not None:
        gx, size = gx + more, size + np.abs(more)
    return gx, size, (gy * x * r).sum(0), np.abs(gy * x * r).sum(0)


def check_grad(k, x, gy, gamma, more, gx, ggamma, rows):
    want, size, wg, sg = grads(x, gy, gamma, more)
    near(gx, want, k.step * np.abs(want) + 2 * F32 * size + k.least, "gradient of the input")
    # (a workgroup adds up to rows / 512 rows one after the other, and up to 64 that it holds side by side)
    near(np.asarray(ggamma).reshape(-1), wg, (rows / 512 + 64 + 64) * F32_STEP * sg + 1e-40, "gradient of gamma")


def test_the_formula_against_differences():
    rng = np.random.default_rng(0)
    x, gy, gamma = rng.standard_normal((3, 11)), rng.standard_normal((3, 11)), rng.normal(1, 0.3, 11)
    gx, _, gg, _ = grads(x, gy, gamma, None, 1e-3)
    f = lambda x, gamma: (rms(x, gamma, 1e-3) * gy).sum()  # noqa: E731
    d = 1e-6
    for i in np.ndindex(x.shape):
        e = np.zeros_like(x)
        e[i] = d
        assert abs((f(x + e, gamma) - f(x - e, gamma)) / (2 * d) - gx[i]) < 1e-8
    for i in range(11):
        e = np.zeros_like(gamma)
        e[i] = d
        assert abs((f(x, gamma + e) - f(x, gamma - e)) / (2 * d) - gg[i]) < 1e-8


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES + [(5000, 64), (3001, 100), (1200, 1001), (2000, 4096)])
def test_backward(hpt, dev, name, rows, cols):
    k, rng = Kind(hpt, name), np.random.default_rng(rows * 7 + cols)
    t, x = k.up(hidden(rng, rows, cols))
    g, gamma = k.up(rng.normal(1, 0.2, cols))
    gy, grad = k.up(rng.standard_normal((rows, cols)) * 0.1)
    m, more = k.up(rng.standard_normal((rows, cols)) * 0.1)
    gx, gg = Guarded(hpt, [rows, cols], k.dtype), Guarded(hpt, [cols], hpt.f32)
    need = hpt.rms_norm_backward_workspace(t, 1)
    ws = Guarded(hpt, [need], hpt.u8)
    t.rms_norm_backward(gy, [cols], g, EPS, grad_sum=m, out=gx.t, gamma_out=gg.t, workspace=ws.t)
    ws.numpy()
    check_grad(k, x, grad, gamma, more, k.load(gx.numpy()), gg.numpy(), rows)
    a, b = t.rms_norm_backward(gy, [cols], g, EPS, grad_sum=m)
    assert np.array_equal(a.numpy(), gx.numpy()) and np.array_equal(b.numpy(), gg.numpy()), "with and without a workspace"
    a, b = t.rms_norm_backward(gy, [cols])
    check_grad(k, x, grad, None, None, k.down(a), b.numpy(), rows)


def test_backward_without_rows_or_gamma(hpt, dev):
    x = hpt.Tensor.empty([0, 24], hpt.f32)
    gx, gg = x.rms_norm_backward(hpt.Tensor.empty([0, 24], hpt.f32), [24])
    assert gx.shape == [0, 24] and not gg.numpy().any() and gg.shape == [24]
    # through the ABI: no gradient of gamma is wanted
    import ctypes as C
    k, rng = Kind(hpt, "f32"), np.random.default_rng(4)
    t, x = k.up(hidden(rng, 20, 40))
    g, grad = k.up(rng.standard_normal((20, 40)))
    out = hpt.Tensor.empty([20, 40], hpt.f32)
    (vx, k1), (vg, k2), (vo, k3) = t._c_view(), g._c_view(), out._c_view()
    from hpt_amd import _ffi
    _ffi.check(hpt.lib().hpt_hip_rms_norm_backward(0, None, C.byref(vx), C.byref(vg), None, 1, None, EPS, None, C.byref(vo), None))
    assert np.array_equal(out.numpy(), t.rms_norm_backward(g, [40])[0].numpy())


def test_a_workspace_too_small(hpt, dev):
    t = hpt.Tensor.zeros([64, 64], hpt.f32)
    need = hpt.rms_norm_backward_workspace(t, 1)
    with pytest.raises(hpt.HptError, match=f"{need} are needed"):
        t.rms_norm_backward(t, [64], out=hpt.Tensor.empty([64, 64], hpt.f32), workspace=hpt.Tensor.empty([need - 1], hpt.u8))
    with pytest.raises(hpt.ParamError, match="16 bytes"):
        w = hpt.Tensor.empty([need + 64], hpt.u8)
        t.rms_norm_backward(t, [64], out=hpt.Tensor.empty([64, 64], hpt.f32), workspace=w[1:need + 1])

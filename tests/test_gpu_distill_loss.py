"""The divergence from a teacher's top logits and the logits' gradient on the device, against 64 bits.

Tolerances count roundings. The sum of exponentials is off by 2 D + 4 half steps of f32 for terms at distance D below the maximum (weighted with their shares, so D = 4 + log V
on average at most) and by what a thread adds one after the other in f32 (31 half steps): below 128 together, which is what a log of a sum is off by. kl has up to three of
them (of all tokens twice, of the unnamed ones once, each with a weight of 1 at most) and is rounded once. A probability of the gradient has that of its sum, 2 D + 16 half steps of
its exponential, and the results' own rounding."""
import numpy as np
import pytest

from block_util import F32_STEP, Guarded, Kind, near, shifted, up
from vocab_util import distilled, logsumexp, order

pytestmark = pytest.mark.gpu
TYPES = ["f32", "f16", "bf16"]
LSE = 128 * F32_STEP


def make(rng, k, rows, cols, n, tau):
    """A student, a teacher's n largest logits with their tokens, and its log of the sum."""
    teacher = rng.standard_normal((rows, cols)) * 3
    x = k.round(0.6 * teacher + rng.standard_normal((rows, cols)))
    teacher = k.round(teacher)
    index = order(teacher)[:, :n]
    return x, np.take_along_axis(teacher, index, -1), index, logsumexp(teacher / tau).astype(np.float32)


def tolerance_of_gradient(k, x, tau, kl_grad, w, scale, lse_t, rest):
    z = x / tau
    lse = logsumexp(z)[:, None]
    p = np.exp(z - lse)
    d = np.abs(w * scale)[:, None]
    # (p's own errors; with the rest, mass - r / s has those of s; q and the difference are rounded)
    return (k.step * np.abs(kl_grad) * d + d * (p * (3 * LSE + (3 * np.abs(z - lse) + 16) * F32_STEP) + np.abs(kl_grad) * (2 * LSE + (3 * np.abs(z - lse) + 24) * F32_STEP)
            + 8 * F32_STEP * np.abs(p - kl_grad)) + k.least)


SHAPES = [(1, 1, 1), (4, 2, 2), (3, 7, 3), (5, 31, 31), (70, 100, 8), (3, 1001, 64), (33, 5000, 17), (1, 50257, 64), (9, 50257, 300), (2100, 40, 5), (600, 2000, 20),
          (2, 152001, 1024), (1, 300000, 50)]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("rows,cols,n", SHAPES)
def test_loss_and_gradient(hpt, dev, name, rest, rows, cols, n):
    k, rng = Kind(hpt, name), np.random.default_rng(rows + cols + n)
    tau = float(rng.choice([1.0, 1.7, 2.0]))
    x, t, index, lse_t = make(rng, k, rows, cols, n, tau)
    mask = (rng.uniform(size=rows) < 0.7) * rng.uniform(0.5, 2, rows)
    mask[0] = 1
    mask = mask.astype(np.float32)
    stored, st, si = x.copy(), t.copy(), index.copy()
    stored[mask == 0] = np.nan  # what does not count is not read
    st[mask == 0] = np.nan
    si[mask == 0] = cols + 5
    # entries that are missing, in some rows all
    gone = rng.uniform(size=index.shape) < 0.2
    gone[:, 0] &= rng.uniform(size=rows) < 0.5
    si[gone] = -1
    index = np.where(gone, -1, index)
    s = shifted(hpt, k, stored, 1)
    ts = k.up(st)[0]
    loss, kl, terms = Guarded(hpt, [1], hpt.f32, 3), Guarded(hpt, [rows], hpt.f32, 1), Guarded(hpt, [rows, 8], hpt.f32, 1)
    ws = Guarded(hpt, [hpt.distill_loss_workspace(s[0])], hpt.u8)
    args = (ts, up(hpt, si.astype(np.int64)))
    kw = dict(teacher_lse=up(hpt, lse_t) if rest else None, temperature=tau)
    s[0].distill_loss(*args, mask=up(hpt, mask), loss_out=loss.t, kl_out=kl.t, terms_out=terms.t, workspace=ws.t, **kw)
    ws.numpy()
    on = mask > 0
    want, grad = distilled(x, t, index, tau, lse_t.astype(np.float64) if rest else None)
    want = np.where(on, want, 0)
    near(kl.numpy(), want, 3 * LSE + F32_STEP * np.abs(want))
    m = mask.astype(np.float64)
    near(loss.numpy()[0], tau * tau * (want * m).sum() / m.sum(), tau * tau * 3 * LSE + 4 * F32_STEP * tau * tau * (np.abs(want) * m).sum() / m.sum())
    # 32-bit tokens, a teacher of another type, the library's scratch: the same bits
    again = s[0].distill_loss(hpt.Tensor.from_numpy(k.load(ts.numpy()).astype(np.float32)).to_hip(dev), up(hpt, si.astype(np.int32)), mask=up(hpt, mask), **kw)
    for a, b in zip(again, (loss, kl, terms)):
        assert np.array_equal(a.numpy(), b.numpy())
    out = Guarded(hpt, [rows, cols], k.dtype, 1)
    scale = 64.0
    s[0].distill_loss_backward(*args, terms.t, temperature=tau, grad=scale, out=out.t)
    w = m * tau / m.sum()
    got = k.load(out.numpy())
    assert not got[~on].any()
    empty = (index < 0).all(-1) if not rest else np.zeros(rows, bool)
    assert not got[empty].any()
    d = grad * (w * scale)[:, None]
    near(got[on], d[on], tolerance_of_gradient(k, x, tau, grad, w, scale, lse_t, rest)[on], "gradient")
    # in the logits' place
    assert np.array_equal(s[0].distill_loss_backward(*args, terms.t, temperature=tau, grad=scale, out=s[0]).numpy(), out.numpy())


@pytest.mark.parametrize("rest", [False, True])
def test_the_formulas_against_differences(rest):
    rng = np.random.default_rng(0)
    rows, cols, n, tau = 4, 9, 4, 1.7
    teacher, x = rng.standard_normal((rows, cols)) * 2, rng.standard_normal((rows, cols))
    index = order(teacher)[:, :n]
    t = np.take_along_axis(teacher, index, -1)
    index[1, 2] = -1
    index[2, 3] = index[2, 0]  # a token named twice
    lse = logsumexp(teacher / tau) if rest else None
    grad = distilled(x, t, index, tau, lse)[1]
    for i in np.ndindex(x.shape):
        h = 1e-6
        a, b = x.copy(), x.copy()
        a[i] += h
        b[i] -= h
        diff = (distilled(a, t, index, tau, lse)[0][i[0]] - distilled(b, t, index, tau, lse)[0][i[0]]) / (2 * h)
        assert abs(diff - grad[i] / tau) < 1e-8


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("cols,n", [(50, 6), (5000, 300), (140000, 1024)])
def test_tokens_named_twice(hpt, dev, name, rest, cols, n):
    """Both entries count, in every order, and the same call gives the same bits."""
    k, rng = Kind(hpt, name), np.random.default_rng(cols)
    x, t, index, _ = make(rng, k, 3, cols, n, 1.0)
    index[:, 3:6] = index[:, :1]
    index[1] = rng.integers(0, min(cols, 40), n)
    index[2, 1] = index[2, 2]
    lse_t = (logsumexp(t) + 0.3).astype(np.float32)
    args = (k.up(t)[0], up(hpt, index))
    kw = dict(teacher_lse=up(hpt, lse_t)) if rest else {}
    tx = k.up(x)[0]
    got = tx.distill_loss(*args, **kw)
    want, grad = distilled(x, t, index, 1.0, lse_t.astype(np.float64) if rest else None)
    near(got.kl.numpy(), want, 3 * LSE + F32_STEP * np.abs(want))
    d = tx.distill_loss_backward(*args, got.terms, grad=3.0)
    w = np.full(3, 1 / 3)
    # (a sum of up to n probabilities of f32)
    near(k.down(d), grad, tolerance_of_gradient(k, x, 1.0, grad, w, 3.0, lse_t, rest) + n * F32_STEP * np.abs(grad))
    for _ in range(3):
        again = tx.distill_loss(*args, **kw)
        assert all(np.array_equal(a.numpy(), b.numpy()) for a, b in zip(again, got))
        assert np.array_equal(tx.distill_loss_backward(*args, again.terms, grad=3.0).numpy(), d.numpy())


@pytest.mark.parametrize("name", TYPES)
def test_masks_within_rows(hpt, dev, name):
    """Masked logits of the student and entries of the teacher that are -inf; what makes a row NaN or infinite."""
    k, rng = Kind(hpt, name), np.random.default_rng(1)
    low = {"f32": -3.4028235e38, "f16": -65504.0, "bf16": -3.3895314e38}[name]
    rows, cols, n = 8, 700, 6
    x, t, index, _ = make(rng, k, rows, cols, n, 1.0)
    x[0, 100:] = -np.inf
    index[0] = [3, 5, 7, 9, 11, -1]
    x[1, 100:] = low
    index[1] = [3, 5, 7, 9, 11, 50]
    t[2, 2:] = -np.inf
    t[3] = -np.inf
    x[4, 5] = -np.inf
    index[4, 0] = 5  # the teacher's likeliest token is impossible to the student
    x[5, 300] = np.nan
    index[6, 1] = cols  # outside the vocabulary
    x[7] = np.where(np.isin(np.arange(cols), index[7]), x[7], -np.inf)  # nothing left to the rest
    lse_t = (logsumexp(np.where(np.isfinite(t), t, -1e30)) + 0.2).astype(np.float32)
    lse_t[3] = 0.5
    tx, args = k.up(x)[0], (k.up(t)[0], up(hpt, index))
    with np.errstate(all="ignore"):
        for kw, lse in ((dict(), None), (dict(teacher_lse=up(hpt, lse_t)), lse_t.astype(np.float64))):
            got = tx.distill_loss(*args, **kw)
            kl = got.kl.numpy().astype(np.float64)
            good = [0, 1, 2, 3, 7]
            want, grad = distilled(x[good], t[good], index[good], 1.0, None if lse is None else lse[good])
            near(kl[good], want, 3 * LSE + F32_STEP * np.abs(want))
            assert kl[4] == np.inf and np.isnan(kl[5]) and np.isnan(kl[6])
            d = k.down(tx.distill_loss_backward(*args, got.terms, grad=float(rows)))
            near(d[good], grad, tolerance_of_gradient(k, np.where(np.isfinite(x), x, -1e3)[good], 1.0, grad, np.full(len(good), 1 / rows), rows, None, lse is not None))
            assert np.isfinite(d[4]).all() or lse is not None
            if lse is None:
                assert not d[3].any(), "a row without an entry that counts"


def test_no_row_counts(hpt, dev):
    k = Kind(hpt, "bf16")
    t = k.up(np.full((4, 9), np.nan))[0]
    args = (k.up(np.zeros((4, 2)))[0], up(hpt, np.full((4, 2), 77)))
    r = t.distill_loss(*args, mask=up(hpt, np.zeros(4, bool)))
    assert r.loss.numpy()[0] == 0 and not r.kl.numpy().any()
    assert not t.distill_loss_backward(*args, r.terms, grad=float("inf")).numpy().any()
    e = hpt.Tensor.empty([0, 9], hpt.f32)
    r = e.distill_loss(hpt.Tensor.empty([0, 2], hpt.f32), hpt.Tensor.empty([0, 2], hpt.i64))
    assert r.loss.numpy()[0] == 0 and r.kl.shape == [0] and r.terms.shape == [0, 8]
    assert e.distill_loss_backward(hpt.Tensor.empty([0, 2], hpt.f32), hpt.Tensor.empty([0, 2], hpt.i64), r.terms).shape == [0, 9]


def test_a_teacher_like_the_student(hpt, dev):
    """Its own top logits and its own log of the sum: no divergence, no gradient."""
    k, rng = Kind(hpt, "f32"), np.random.default_rng(3)
    t, x = k.up(rng.standard_normal((5, 3000)) * 3)
    v, i, lse = t.topk(100, temperature=2.0, lse=True)
    got = t.distill_loss(v, i, teacher_lse=lse, temperature=2.0)
    # (lse is rounded: r is off by |lse| half steps)
    near(got.kl.numpy(), np.zeros(5), 3 * LSE + 16 * F32_STEP)
    p = np.exp(x / 2 - logsumexp(x / 2)[:, None])
    near(k.down(t.distill_loss_backward(v, i, got.terms, temperature=2.0, grad=2.5)), np.zeros((5, 3000)), p * 6 * LSE)


def test_rows_anywhere(hpt, dev):
    rng = np.random.default_rng(4)
    k = Kind(hpt, "bf16")
    wide, x = k.up(rng.standard_normal((6, 3, 1003)) * 2)
    v = wide.permute([1, 0, 2])[:, ::2]
    part = np.ascontiguousarray(np.transpose(x, (1, 0, 2))[:, ::2]).reshape(9, -1)
    t, index = rng.standard_normal((9, 4)).astype(np.float32), order(part)[:, :4]
    args = (up(hpt, t.reshape(3, 3, 4)), up(hpt, index.reshape(3, 3, 4)))
    got = v.distill_loss(*args)
    want, grad = distilled(part, t.astype(np.float64), index)
    assert got.kl.shape == [3, 3] and got.terms.shape == [3, 3, 8]
    near(got.kl.numpy().reshape(-1), want, 3 * LSE + F32_STEP * np.abs(want))
    d = v.distill_loss_backward(*args, got.terms, grad=9.0)
    near(k.down(d).reshape(9, -1), grad, tolerance_of_gradient(k, part, 1.0, grad, np.full(9, 1 / 9), 9.0, None, False))

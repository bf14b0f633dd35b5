"""Token log-probabilities, the clipped policy loss with its KL term and the logits' gradient on the device, against 64 bits.

Tolerances count roundings: the sum of exponentials is off by 2 D + 4 half steps of f32 for terms at distance D below the maximum
(weighted with their shares, so D = 4 + log V on average at most) and by what a thread adds one after the other (a quarter of V / 256
terms in f32, whose errors are below 64 half steps here); logp and lse are rounded to f32 once. A weight moves with its ratio."""
import numpy as np
import pytest

from block_util import F32_STEP, Guarded, Kind, near, shifted, up

pytestmark = pytest.mark.gpu
TYPES = ["f32", "f16", "bf16"]
LSE = 128 * F32_STEP  # absolute, of the log of the sum


def logsumexp(x):
    m = x.max(-1, keepdims=True)
    return (m + np.log(np.exp(x - m).sum(-1, keepdims=True)))[..., 0]


def losses(logp, old, adv, ref, low, high, kl):
    ratio = np.exp(logp - old)
    free, held = ratio * adv, np.clip(ratio, 1 - low, 1 + high) * adv
    loss, slope = -np.minimum(free, held), np.where(free <= held, -free, 0)
    if ref is not None and kl:
        k = ref - logp
        loss, slope = loss + kl * (np.exp(k) - k - 1), slope + kl * (1 - np.exp(k))
    return loss, slope


def sample(rng, k, rows, cols):
    x = k.round(rng.standard_normal((rows, cols)) * 3)
    token = (x + rng.gumbel(size=x.shape)).argmax(-1)
    logp = x[np.arange(rows), token] - logsumexp(x)
    # away from the borders of the clipping, where the derivative jumps
    d = rng.normal(0, 0.15, rows)
    for border in (np.log(0.8), np.log(1.28)):
        d = np.where(np.abs(d + border) < 1e-3, d + 4e-3, d)
    f = lambda a: a.astype(np.float32)  # noqa: E731
    return x, token, logp, f(logp + d), f(rng.standard_normal(rows)), f(logp + rng.normal(0, 0.3, rows))


SHAPES = [(1, 1), (4, 2), (3, 7), (6, 8), (5, 31), (70, 100), (3, 1001), (33, 5000), (1, 50257), (9, 50257), (2100, 40), (600, 2000), (2, 152001), (1, 300000)]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_loss_and_gradient(hpt, dev, name, rows, cols):
    k, rng = Kind(hpt, name), np.random.default_rng(rows + cols)
    x, token, logp, old, adv, ref = sample(rng, k, rows, cols)
    mask = (rng.uniform(size=rows) < 0.7).astype(np.float32)
    mask[0] = 1
    stored = x.copy()
    stored[mask == 0] = np.nan  # what does not count is not read
    t = k.up(stored)[0]
    tok = np.where(mask > 0, token, -100)
    f32s = {n: Guarded(hpt, [rows], hpt.f32, 1) for n in ("logp", "lse", "weight")}
    loss = Guarded(hpt, [1], hpt.f32, 3)
    need = hpt.policy_loss_workspace(t)
    ws = Guarded(hpt, [need], hpt.u8)
    args = (up(hpt, tok.astype(np.int64)), up(hpt, old), up(hpt, adv))
    kw = dict(reference=up(hpt, ref), clip_low=0.2, clip_high=0.28, kl_weight=0.04)
    got = t.policy_loss(*args, mask=up(hpt, mask), loss_out=loss.t, logp_out=f32s["logp"].t, lse_out=f32s["lse"].t, weight_out=f32s["weight"].t, workspace=ws.t, **kw)
    ws.numpy()
    on = mask > 0
    each, slope = losses(logp, old.astype(np.float64), adv.astype(np.float64), ref.astype(np.float64), 0.2, 0.28, 0.04)
    lse = logsumexp(x)
    near(f32s["logp"].numpy(), np.where(on, logp, 0), LSE + F32_STEP * np.abs(logp))
    near(f32s["lse"].numpy(), np.where(on, lse, 0), LSE + F32_STEP * np.abs(lse))
    n = mask.sum()
    moves = LSE * (np.abs(np.exp(logp - old) * adv) + 0.04 * np.exp(ref - logp))  # by what a wrong logp moves a slope
    near(f32s["weight"].numpy(), np.where(on, slope, 0) / n, (moves + 4 * F32_STEP * np.abs(slope)) / n)
    near(loss.numpy()[0], each[on].sum() / n, (LSE * (np.abs(slope) + np.abs(np.exp(logp - old) * adv))[on].sum() + 4 * F32_STEP * np.abs(each[on]).sum()) / n)
    # a mask of truth values and 32-bit tokens, the library's scratch: the same bits
    again = t.policy_loss(up(hpt, tok.astype(np.int32)), *args[1:], mask=up(hpt, on), **kw)
    for a, b in zip(again, got):
        assert np.array_equal(a.numpy(), b.numpy())
    # the gradient from the stored values
    w, l = f32s["weight"].numpy().astype(np.float64), f32s["lse"].numpy().astype(np.float64)
    out = Guarded(hpt, [rows, cols], k.dtype, 1)
    scale = 512.0
    t.policy_loss_backward(args[0], got.lse, got.weight, scale, out=out.t)
    p = np.exp(x - l[:, None])
    d = -p
    d[np.arange(rows), token] += 1
    d *= (w * scale)[:, None]
    d[w == 0] = 0
    tol = k.step * np.abs(d) + np.abs(w * scale)[:, None] * (p * (4 * np.abs(x - l[:, None]) + 16) * F32_STEP + 4 * F32_STEP * np.abs(d / np.where(w == 0, 1, w * scale)[:, None])) + k.least
    near(k.load(out.numpy()), d, tol, "gradient")
    # in the logits' place
    assert np.array_equal(t.policy_loss_backward(args[0], got.lse, got.weight, scale, out=t).numpy(), out.numpy())


def test_the_formulas_against_differences():
    rng = np.random.default_rng(0)
    rows, cols = 5, 9
    x, token = rng.standard_normal((rows, cols)), rng.integers(0, cols, rows)
    old, adv, ref = rng.normal(-2, 0.3, rows), rng.standard_normal(rows), rng.normal(-2, 0.3, rows)
    mask = np.array([1, 0, 0.5, 1, 1])

    def f(x):
        logp = x[np.arange(rows), token] - logsumexp(x)
        return (losses(logp, old, adv, ref, 0.2, 0.3, 0.1)[0] * mask).sum() / mask.sum()

    logp = x[np.arange(rows), token] - logsumexp(x)
    w = losses(logp, old, adv, ref, 0.2, 0.3, 0.1)[1] * mask / mask.sum()
    d = -np.exp(x - logsumexp(x)[:, None])
    d[np.arange(rows), token] += 1
    d *= w[:, None]
    for i in np.ndindex(x.shape):
        e = np.zeros_like(x)
        e[i] = 1e-6
        assert abs((f(x + e) - f(x - e)) / 2e-6 - d[i]) < 1e-8


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (7, 33), (5, 4000), (2, 100001), (2200, 50)])
def test_token_logp(hpt, dev, name, rows, cols):
    k, rng = Kind(hpt, name), np.random.default_rng(cols)
    x, token, logp, *_ = sample(rng, k, rows, cols)
    t, _, base = shifted(hpt, k, x, 1)
    a, b = t.token_logp(up(hpt, token.astype(np.int64)))
    near(a.numpy(), logp, LSE + F32_STEP * np.abs(logp))
    lse = logsumexp(x)
    near(b.numpy(), lse, LSE + F32_STEP * np.abs(lse))
    assert a.shape == [rows]
    # tokens that are none
    for bad in (-1, cols, -100, 2 ** 40):
        a, b = t.token_logp(up(hpt, np.full(rows, bad, np.int64)))
        assert np.isnan(a.numpy()).all()
        near(b.numpy(), lse, LSE + F32_STEP * np.abs(lse))


def test_strided_logits(hpt, dev):
    """Positions of a padded batch: the last one of each sequence is left out, and so is part of the vocabulary."""
    k, rng = Kind(hpt, "bf16"), np.random.default_rng(8)
    t, x = k.up(rng.standard_normal((3, 6, 120)) * 3)
    v, a = t[:, :5, :101], x[:, :5, :101]
    token = rng.integers(0, 101, (3, 5))
    lse = logsumexp(a)
    want = np.take_along_axis(a, token[..., None], -1)[..., 0] - lse
    logp, got = v.token_logp(up(hpt, token))
    assert logp.shape == [3, 5]
    near(logp.numpy(), want, LSE + F32_STEP * np.abs(want))
    w = rng.standard_normal((3, 5)).astype(np.float32)
    d = k.down(v.policy_loss_backward(up(hpt, token), got, up(hpt, w)))
    p = np.exp(a - got.numpy()[..., None])
    e = -p
    np.put_along_axis(e, token[..., None], np.take_along_axis(e, token[..., None], -1) + 1, -1)
    e *= w[..., None]
    near(d, e, k.step * np.abs(e) + np.abs(w[..., None]) * p * 100 * F32_STEP + 8 * F32_STEP * np.abs(w[..., None]))
    # one row, no leading dims
    one = hpt.Tensor.from_raw(t.ptr, [120], hpt.bf16)
    assert abs(one.token_logp(up(hpt, np.array([7])))[0].numpy()[0] - (x[0, 0, 7] - logsumexp(x[0, 0]))) < LSE + 1e-6


def test_nothing_counts(hpt, dev):
    k, rng = Kind(hpt, "f32"), np.random.default_rng(8)
    t, _ = k.up(np.full((6, 30), np.nan))
    z = up(hpt, np.zeros(6, np.float32))
    r = t.policy_loss(up(hpt, np.full(6, -100)), z, z, mask=z)
    assert all(not v.numpy().any() for v in r)
    assert not t.policy_loss_backward(up(hpt, np.full(6, -100)), r.lse, r.weight).numpy().any()
    e = hpt.Tensor.empty([0, 30], hpt.f32)
    n = hpt.Tensor.empty([0], hpt.f32)
    r = e.policy_loss(hpt.Tensor.empty([0], hpt.i64), n, n)
    assert r.loss.numpy()[0] == 0 and r.logp.shape == [0]
    # a token outside the vocabulary in a row that counts
    t, x = k.up(rng.standard_normal((3, 30)))
    one = up(hpt, np.ones(3, np.float32))
    r = t.policy_loss(up(hpt, np.array([1, 30, 2])), one, one)
    assert np.isnan(r.loss.numpy()[0]) and np.isnan(r.weight.numpy()[1]) and np.isfinite(r.weight.numpy()[[0, 2]]).all()
    assert np.isnan(t.policy_loss_backward(up(hpt, np.array([1, 30, 2])), r.lse, r.weight).numpy()[1]).all()


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("cols", [3, 50, 40000])
def test_the_lowest_value_as_a_mask(hpt, dev, name, cols):
    """Logits that a caller has masked with the type's lowest value, all of a row among them, and their mirror."""
    k, rng = Kind(hpt, name), np.random.default_rng(3)
    low = {"f32": np.finfo(np.float32).min, "f16": -65504.0, "bf16": -3.3895313892515355e38}[name]
    x = rng.standard_normal((5, cols))
    x[0] = low
    x[1, 1:] = low
    x[2] = -low
    x[3, 1] = low / 1.3
    x[3, 2:] = low
    x[3, 0] = low
    t, x = k.up(x)
    token = np.array([1, 0, 2, 1, 2])
    logp, lse = (v.numpy().astype(np.float64) for v in t.token_logp(up(hpt, token)))
    near(logp, [-np.log(cols), 0, -np.log(cols), 0, x[4, 2] - logsumexp(x[4])], LSE + F32_STEP * 12)
    near(lse, logsumexp(x), LSE + F32_STEP * np.abs(logsumexp(x)))


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("cols", [50, 40000])
def test_infinities_and_nan(hpt, dev, name, cols):
    k, rng = Kind(hpt, name), np.random.default_rng(3)
    x = rng.standard_normal((5, cols))
    x[0, 5:] = -np.inf
    x[1, 4] = np.nan
    x[2, 4] = np.inf
    x[3] = -np.inf
    t, x = k.up(x)
    with np.errstate(invalid="ignore"):
        logp, lse = (v.numpy().astype(np.float64) for v in t.token_logp(up(hpt, np.array([2, 2, 2, 2, 2]))))
    near(lse[0], logsumexp(x[0, :5]), LSE + 1e-6)
    near(logp[0], x[0, 2] - logsumexp(x[0, :5]), LSE + 1e-6)
    assert np.isnan(logp[1]) and np.isnan(lse[1])
    assert logp[2] == -np.inf and lse[2] == np.inf
    assert np.isnan(logp[3]) and lse[3] == -np.inf
    near(lse[4], logsumexp(x[4]), LSE + F32_STEP * 12)
    # a token without any probability
    assert t.token_logp(up(hpt, np.array([7, 0, 0, 0, 0])))[0].numpy()[0] == -np.inf


def test_the_free_side_where_both_are_equal(hpt, dev):
    """A ratio of exactly 1 within no clipping at all: the minimum's sides are equal and the gradient is the unclipped one's."""
    t = up(hpt, np.array([[0.0, -np.inf], [0.0, -np.inf]], np.float32))
    z, a = up(hpt, np.zeros(2, np.float32)), up(hpt, np.array([2.0, -2.0], np.float32))
    r = t.policy_loss(up(hpt, np.zeros(2, np.int64)), z, a, clip_low=0.0, clip_high=0.0)
    assert np.array_equal(r.weight.numpy(), np.array([-1.0, 1.0], np.float32)) and r.loss.numpy()[0] == 0

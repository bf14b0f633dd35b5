"""Top-k, sampling and distillation at the ends of their ranges: workspaces of exactly the size that is asked for, borders within a rounding of what decides,
logits that lie anywhere, rows by many millions.

Tolerances count half steps of f32, as beside each test."""
import ctypes as C

import numpy as np
import pytest

from block_util import F32_STEP, Guarded, Kind, near, up
from test_gpu_block_calls import P, hip, stream  # noqa: F401
from vocab_util import logsumexp, order, sampled

pytestmark = pytest.mark.gpu
TYPES = ["f32", "f16", "bf16"]


# ---- scratch ------------------------------------------------------------------------------------


@pytest.mark.parametrize("name,rows,cols", [("bf16", 8192, 128256), ("f32", 4096, 128256), ("f32", 4096, 152000), ("f32", 16384, 50257), ("bf16", 32768, 32000),
                                            ("bf16", 4096, 256000), ("f32", 16384, 32000)])
def test_a_workspace_of_the_size_that_is_asked_for(hpt, dev, name, rows, cols):
    """Rows beyond one run, with the sum and without it. The same eight rows again and again."""
    kind, rng, k = Kind(hpt, name), np.random.default_rng(cols), 3
    t, x = kind.up(rng.standard_normal((8, cols)))
    v = hpt.Tensor.from_raw(t.ptr, [rows // 8, 8, cols], kind.dtype, 0, [0, cols, 1])
    ws = Guarded(hpt, [hpt.topk_workspace(v, k)], hpt.u8)
    want = np.broadcast_to(order(x)[:, :k], (rows // 8, 8, k))
    for lse in (False, True):
        got = v.topk(k, lse=lse, workspace=ws.t)
        ws.numpy()
        assert np.array_equal(got[1].numpy(), want)


def test_rows_that_registers_hold_take_no_scratch(hpt, dev, hip, stream):  # noqa: F811
    """They are captured without a workspace."""
    kind, rng, k = Kind(hpt, "f32"), np.random.default_rng(1), 8
    t, x = kind.up(rng.standard_normal((600, 64)))
    v, i, lse = hpt.Tensor.empty([600, k], hpt.f32), hpt.Tensor.empty([600, k], hpt.i64), hpt.Tensor.empty([600], hpt.f32)
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    try:
        t.topk(k, lse=True, stream=stream, values_out=v, index_out=i, lse_out=lse)
    finally:
        g = P()
        rc = hip.hipStreamEndCapture(stream, C.byref(g))
    assert rc == 0 and g.value
    e = P()
    assert hip.hipGraphInstantiate(C.byref(e), g, None, None, 0) == 0
    try:
        for scale in (1.0, 0.5, -2.0):
            a = (x * scale).astype(np.float32)
            assert hpt.lib().hpt_hip_memcpy_h2d_sync(0, P(t.ptr), a.ctypes.data_as(P), a.nbytes) == 0
            assert hip.hipGraphLaunch(e, stream) == 0 and hip.hipStreamSynchronize(stream) == 0
            assert np.array_equal(i.numpy(), order(a)[:, :k])
            want = [r.numpy() for r in t.topk(k, lse=True)]
            assert all(np.array_equal(r.numpy(), w) for r, w in zip((v, i, lse), want))
    finally:
        hip.hipGraphExecDestroy(e)
        hip.hipGraphDestroy(g)


# ---- sampling: borders within a rounding of what decides ---------------------------------------------------

OCTAVE = 1.4426950408889634  # the temperature at which logits are octaves


def test_halves_of_the_same_sum(hpt, dev):
    """Twice the same weights, each time with a stretch of nothing behind them, and u in the middle of the row's sum: where the sums in 64 bits put the border between the halves depends on their
    order, but the token is the last of the first half or the first of the second, and its probability is its own."""
    rows, n = 1200, 2048
    x = np.full((rows, 2 * n), -np.inf)
    for r in range(rows):
        rng = np.random.default_rng(r)
        a = -rng.integers(0, 24, 1536).astype(float)
        a[0] = 0
        x[r, :1536], x[r, n:n + 1536] = a, rng.permutation(a)
    t, x = Kind(hpt, "f32").up(x)
    for part in (slice(0, 200), slice(0, rows)):  # (forms for few rows and for many)
        count = part.stop
        u = up(hpt, np.full(count, 0.5, np.float32))
        v = hpt.Tensor.from_raw(t.ptr, [count, 2 * n], hpt.f32, 0)
        each = dict(temperature=up(hpt, np.full(count, OCTAVE, np.float32)))
        for settings in (dict(temperature=OCTAVE), each, dict(temperature=OCTAVE, min_p=1e-30)):
            token, logp = (a.numpy() for a in v.sample(u, **settings))
            assert np.isin(token, [1535, n]).all(), (settings, token[~np.isin(token, [1535, n])][:4])
            w = np.exp2(x[:count])
            near(logp, np.log(w[np.arange(count), token] / w.sum(-1)), 30 * F32_STEP)


# (temperature, numbers of logits 200, 199, ..., how far below 200 1500 and 2500 more lie, top_p): with the sums of the kernels top_p's border lies in a bucket of which rounding
# makes something though it is empty, and in which no bf16 number lies
BETWEEN = [
    (6.53, [67, 221, 131, 264, 243, 34, 81, 59, 53, 20, 252, 248], 17, 0.7570882010828001),
    (6.45, [135, 298, 217, 230, 88, 29, 108], 10, 0.5078388538921861),
    (6.26, [23, 172, 268, 218, 16, 186, 153, 42, 194, 252, 292, 246], 16, 0.7572712300091017),
    (6.31, [190, 133, 209, 67, 272, 32, 114], 14, 0.6392513511158395),
    (6.74, [165, 115, 192, 84, 102, 141, 212], 10, 0.4474014156237754),
    (6.86, [99, 293, 289, 102, 77, 50, 10, 256, 173, 230], 13, 0.6240515076129396),
]


@pytest.mark.parametrize("case", range(len(BETWEEN)))
def test_a_border_in_an_empty_bucket(hpt, dev, case):
    temperature, counts, low, top_p = BETWEEN[case]
    x = np.full((1, 8192), -np.inf)
    many = sum(counts)
    x[0, :many] = 200.0 - np.repeat(np.arange(len(counts)), counts)
    x[0, many:many + 4000] = 200.0 - low - np.repeat([0, 1], [1500, 2500])
    t = Kind(hpt, "bf16").up(x)[0]
    w = np.exp((x[0] - 200) / temperature)
    assert abs(w[:many].sum() / w.sum() - top_p) < 2.0 ** -40
    for u in (0.0, 0.3, 0.9, 0.9999):
        token, logp = (a.numpy()[0] for a in t.sample(up(hpt, np.array([u], np.float32)), temperature=temperature, top_p=top_p))
        # (the first of those below may or may not be needed to reach top_p)
        upto = w[:many + 1].cumsum()
        wants = {int((upto[:n] <= np.float32(u) * upto[n - 1]).sum()) for n in (many, many + 1)}
        assert token in wants, (token, wants, many)
        near(logp, np.log(w[token] / upto[many - 1]), 20 * F32_STEP + w[many] / upto[many])


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("settings", [dict(top_k=1500, top_p=0.9003), dict(top_k=4000, top_p=0.3001), dict(top_p=0.65037), dict(temperature=1e12, top_p=0.30003), dict(top_k=777, top_p=0.5003)], ids=str)
def test_tied_rows_that_decide_clearly(hpt, dev, name, settings):
    """Rows of equal logits, of few values, and of masks, with a border and a u that no part of them equals."""
    kind, rng, cols = Kind(hpt, name), np.random.default_rng(11), 20001
    low = {"f32": -3.4028235e38, "f16": -65504.0, "bf16": -3.3895314e38}[name]
    x = np.zeros((8, cols))
    x[1] = -7.25
    x[2] = low
    x[3, cols // 2:] = -np.inf
    x[4, :cols // 3] = low
    x[5] = np.where(np.arange(cols) % 2, 3.0, 3.5)
    x[6] = rng.integers(0, 3, cols) / 8
    x[7] = np.where(np.arange(cols) % 5, low, 1.0)
    t, x = kind.up(x)
    u = np.array([0.30103, 0.61803, 0.14159, 0.71828, 0.57721, 0.41421, 0.73205, 0.23606], np.float32)
    with np.errstate(over="ignore"):
        want = [sampled(x[r], u[r], **settings) for r in range(8)]
    clear = np.array([w[2] > 2.0 ** -36 for w in want])
    assert clear.all(), [w[2] for w in want]
    for rep in (1, 40, 200):
        v = hpt.Tensor.from_raw(t.ptr, [rep, 8, cols], kind.dtype, 0, [0, cols, 1])
        token, logp = v.sample(up(hpt, np.tile(u, rep)), **settings)
        assert np.array_equal(token.numpy(), np.broadcast_to([w[0] for w in want], (rep, 8)))
        logs = np.array([w[1] for w in want])
        near(logp.numpy(), np.broadcast_to(logs, (rep, 8)), F32_STEP * np.abs(logs) + 1e-11)


# ---- top-k and sampling: logits anywhere -------------------------------------------------------------------


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("reps,cols,k", [(1, 5000, 50), (1, 50257, 600), (20, 5000, 64), (60, 20001, 33), (260, 9000, 20), (260, 9000, 300)])
def test_first_places_anywhere(hpt, dev, name, reps, cols, k):
    """A number added to all logits: the first places of either sign, on both sides of zero, and far from it. Five rows again and again."""
    kind, rng = Kind(hpt, name), np.random.default_rng(cols + k)
    base = rng.standard_normal((5, cols)) * np.array([[0.5], [1], [2], [4], [8]])
    u = rng.uniform(size=5).astype(np.float32)
    for offset in (-4.0, -8.0, -30.0, 100.0, -100.0, 6e4, -1e9, 1e20, -1e34):
        if abs(offset) > 6e4 and name == "f16":
            continue
        t, x = kind.up(base * max(1.0, abs(offset) / 2e4) + offset)
        v = hpt.Tensor.from_raw(t.ptr, [reps, 5, cols], kind.dtype, 0, [0, cols, 1])
        want = order(x)[:, :k]
        values, index = v.topk(k)
        assert np.array_equal(index.numpy(), np.broadcast_to(want, (reps, 5, k))), offset
        assert np.array_equal(kind.load(values.numpy()), np.broadcast_to(np.take_along_axis(x, want, -1), (reps, 5, k)))
        for settings in (dict(top_k=k), dict(top_k=k, top_p=0.7), dict(top_p=0.9), dict(min_p=0.02), dict()):
            settings["temperature"] = max(1.0, abs(offset) / 2e4)
            chosen = [sampled(x[r], u[r], **settings) for r in range(5)]
            clear = np.array([c[2] > 2.0 ** -36 for c in chosen])
            token, logp = v.sample(up(hpt, np.tile(u, reps)), **settings)
            tokens, logs = np.array([c[0] for c in chosen]), np.array([c[1] for c in chosen])
            assert np.array_equal(token.numpy()[:, clear], np.broadcast_to(tokens, (reps, 5))[:, clear]), (offset, settings)
            near(logp.numpy()[:, clear], np.broadcast_to(logs, (reps, 5))[:, clear], (F32_STEP * np.abs(logs) + 1e-11)[clear], f"{offset} {settings}")


# ---- top-k: the log of the sum -----------------------------------------------------------------------------


def lse_tolerance(z):
    """A term at distance D below the largest is off by 2 D (its distance and its exponent are rounded) + 2 (the exponential) half steps, and by 3 of the sum of eight of them; the join of
    wavefronts' parts is another exponential's 2 of what is not next to the largest, and the result is rounded once. Terms at distance 0 are 1."""
    d = z.max(-1, keepdims=True) - z
    p = np.exp(z - logsumexp(z)[:, None])
    return F32_STEP * ((p * np.where(d > 0, 2 * d + 4, 0)).sum(-1) + np.where((d > 0).any(-1), 3, 0) + np.abs(logsumexp(z))) + 1e-13


LENGTHS = [(3, 6), (3, 64), (700, 256), (5, 1000), (700, 2000), (3, 5000), (300, 20001), (1100, 20001), (2, 152000), (40003, 70)]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,cols", LENGTHS)
def test_the_sum_of_equal_logits(hpt, dev, name, rows, cols):
    """Every term is 1: only the result is rounded, also where the logits are about the negative log of their number and the result is next to 0."""
    kind = Kind(hpt, name)
    x = np.array([0.0, -np.log(cols), 1.25, -100.0, 300.0, -3e4, -np.log(cols) + 1e-3])
    for tau in (1.0, 2.0, 0.7):
        for value in x:
            t, v = kind.up(np.full((1, cols), value * tau))
            b = hpt.Tensor.from_raw(t.ptr, [rows, cols], kind.dtype, 0, [0, 1])
            want = logsumexp(v / tau)
            near(b.topk(3, lse=True, temperature=tau)[2].numpy(), np.broadcast_to(want, rows), F32_STEP * np.abs(want) + 1e-12 * (1 + np.abs(v[0, 0] / tau)), f"{value} at {tau}")


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,cols", LENGTHS)
@pytest.mark.parametrize("sd", [0.3, 3.0, 8.0])
def test_the_sum_to_a_few_roundings(hpt, dev, name, rows, cols, sd):
    """Logits, and log-probabilities, whose sum is 1."""
    kind, rng = Kind(hpt, name), np.random.default_rng(cols)
    x = rng.standard_normal((3, cols)) * sd
    x[1] -= logsumexp(x[1:2])
    x[2, 0] = x[2].max() + 6 * sd + 5
    x[2] -= logsumexp(x[2:3])
    for tau in (1.0, 1.7):
        t, v = kind.up(x * tau)
        n = max(1, rows // 3)
        b = hpt.Tensor.from_raw(t.ptr, [n, 3, cols], kind.dtype, 0, [0, cols, 1])
        near(b.topk(5, lse=True, temperature=tau)[2].numpy(), np.broadcast_to(logsumexp(v / tau), (n, 3)), lse_tolerance(v / tau))


# ---- distillation: logits anywhere -------------------------------------------------------------------------


def diverged(x, t, index, tau, teacher_lse=None):
    """(kl, its gradient by x / tau) of each row, every entry a token of its own, from distances alone: what lies so far below that its probability is no number of 64 bits still has a logarithm."""
    rows = len(x)
    kl, grad = np.zeros(rows), np.zeros(x.shape)
    for r in range(rows):
        z = (x[r] - x[r].max()) / tau
        e = (t[r] - t[r].max()) / tau
        lse = logsumexp(z)
        logq = e - logsumexp(e) if teacher_lse is None else t[r] / tau - teacher_lse[r]
        q = np.exp(logq)
        rest = 0.0 if teacher_lse is None else max(0.0, 1 - q.sum())
        on = q > 0
        kl[r] = (q[on] * (logq[on] - (z[index[r]][on] - lse))).sum()
        grad[r] = (q.sum() + rest) * np.exp(z - lse)
        grad[r, index[r]] -= q
        if rest:
            out = np.ones(len(z), bool)
            out[index[r]] = False
            logs = logsumexp(z[out])
            kl[r] += rest * (np.log(rest) - (logs - lse))
            grad[r][out] -= rest * np.exp(z[out] - logs)
    return kl, grad


def kl_tolerance(x, tau, kl, rest=True):
    """The student's log of the sum, as above (a rescaled sum in 64 bits), and the result's own rounding; of the rest the sum over the unnamed counts too, at most as much."""
    z = (x - x.max(-1, keepdims=True)) / tau
    return (1 + rest) * (lse_tolerance(z) - F32_STEP * np.abs(logsumexp(z))) + F32_STEP * np.abs(kl) + 1e-12


def gradient_tolerance(k, x, t, tau, grad, w, lse_part):
    """A probability p at distance D is off by 2 D + 2 half steps as above, by its sum's, and by one each of the reciprocal of the sum, its weight, two products and the difference; q by 8, or as p where it is r / s times p; the result by half a step of its
    type. An exponential below f32's normal numbers may be 0, which loses 2^-126 of p at most."""
    z = (x - x.max(-1, keepdims=True)) / tau
    lse = logsumexp(z)[:, None]
    p = np.exp(z - lse)
    q = np.abs(p - grad)
    w = np.abs(w)[:, None]
    return w * (p + q) * (F32_STEP * (2 * -z + 8) + 2 * lse_part[:, None]) + k.step * np.abs(grad) * w + k.least + 2.0 ** -126 * (1 + w)


OFFSETS = [0.0, -1e4, 6e4, -9e4, 1e6, -1e9, 1e12, -1e20, 1e30, -1e37, 1.6e38, "low"]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("rows,cols,n", [(6, 50, 5), (6, 5000, 60), (6, 40001, 300), (2100, 70, 8)])
def test_students_that_lie_anywhere(hpt, dev, name, rest, rows, cols, n):
    """The divergence does not change with a number added to all logits of a row, whatever is left of their differences; rows that a mask has left nothing but the type's lowest value."""
    k, rng = Kind(hpt, name), np.random.default_rng(cols)
    low = {"f32": -3.4028235e38, "f16": -65504.0, "bf16": -3.3895314e38}[name]
    for offset in OFFSETS if rows < 100 else OFFSETS[::3] + OFFSETS[-1:]:
        value = low if offset == "low" else offset
        if abs(value) > 65504 and name == "f16":
            continue
        for tau in (1.0, 2.0, 0.6):
            teacher = k.round(rng.standard_normal((rows, cols)) * 3)
            index = order(teacher)[:, :n]
            tt = np.take_along_axis(teacher, index, -1)
            lse_t = logsumexp(teacher / tau).astype(np.float32)
            x = np.full((rows, cols), value)
            if offset != "low":
                with np.errstate(over="ignore"):
                    x = k.round(x + rng.standard_normal((rows, cols)) * max(3.0, abs(value) * 2.0 ** -9))
                x = np.clip(x, low, -low)
            x[-1] = value
            tx, x = k.up(x)
            args = (k.up(tt)[0], up(hpt, index))
            kw = dict(teacher_lse=up(hpt, lse_t)) if rest else {}
            got = tx.distill_loss(*args, temperature=tau, **kw)
            shifted = x - x.max(-1, keepdims=True)
            with np.errstate(all="ignore"):
                want, grad = diverged(x, tt, index, tau, lse_t.astype(np.float64) if rest else None)
            # (a divergence beyond f32 is an infinity)
            fits = np.abs(want) < 3.4e38
            part = lse_tolerance(shifted / tau)
            near(got.kl.numpy()[fits], want[fits], kl_tolerance(x, tau, want)[fits] + np.abs(want[fits]) * 1e-12, f"kl at {value}, {tau}")
            scale = float(rows)
            d = tx.distill_loss_backward(*args, got.terms, temperature=tau, grad=scale)
            w = np.full(rows, tau)
            near(k.down(d), grad * tau, gradient_tolerance(k, x, tt, tau, grad, w, part), f"gradient at {value}, {tau}")


@pytest.mark.parametrize("name", TYPES)
def test_teachers_that_lie_anywhere(hpt, dev, name):
    """Without the rest, a number added to all of a teacher's entries changes nothing."""
    k, rng = Kind(hpt, name), np.random.default_rng(3)
    low = {"f32": -3.4028235e38, "f16": -65504.0, "bf16": -3.3895314e38}[name]
    rows, cols, n = 5, 3000, 40
    x = rng.standard_normal((rows, cols)) * 2
    index = order(rng.standard_normal((rows, cols)))[:, :n]
    tx, x = k.up(x)
    for value in (-1e4, 6e4, -1e9, 1e20, -1e37, low):
        if abs(value) > 65504 and name == "f16":
            continue
        t = k.round(value + (rng.standard_normal((rows, n)) * max(2.0, abs(value) * 2.0 ** -9) if value != low else 0.0 * index))
        for tau in (1.0, 0.6):
            got = tx.distill_loss(k.up(t)[0], up(hpt, index), temperature=tau)
            want, grad = diverged(x, t, index, tau)
            near(got.kl.numpy(), want, kl_tolerance(x, tau, want))
            d = tx.distill_loss_backward(k.up(t)[0], up(hpt, index), got.terms, temperature=tau, grad=float(rows))
            near(k.down(d), grad * tau, gradient_tolerance(k, x, t, tau, grad, np.full(rows, tau), lse_tolerance((x - x.max(-1, keepdims=True)) / tau)))


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("cols", [300, 5000, 50257])
def test_sums_of_equal_terms(hpt, dev, name, rest, cols):
    """One largest logit and all others at one distance below it: as many equal terms, whose sum would be off by a rounding for each were they added in f32 one after the other. Without the largest, terms of 1, which
    are not off at all."""
    k = Kind(hpt, name)
    rows = 400
    x = np.repeat(-np.linspace(0.003, 1.7, rows)[:, None], cols, 1)
    x[:, cols // 3] = 0
    tx, x = k.up(x)
    index = np.broadcast_to(np.array([[cols // 3, 1]]), (rows, 2))
    tt = np.broadcast_to(k.round(np.array([[0.5, 0.25]])), (rows, 2))
    lse_t = np.full(rows, 1.7, np.float32)
    got = tx.distill_loss(k.up(tt)[0], up(hpt, index), **(dict(teacher_lse=up(hpt, lse_t)) if rest else {}))
    want, _ = diverged(x, tt, index, 1.0, lse_t.astype(np.float64) if rest else None)
    near(got.kl.numpy(), want, kl_tolerance(x, 1.0, want, rest))


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("rows,cols", [(2100, 1 << 20), (2100, 50257), (300, 50257), (1, 300000), (2100, 300)])
def test_rising_rows(hpt, dev, name, rest, rows, cols):
    """Every vector of a thread has a new largest logit: the sum is rescaled each time. One row again and again."""
    k, rng = Kind(hpt, name), np.random.default_rng(4)
    for span in (4.0, 30.0):
        t, x = k.up(np.linspace(-span, 0, cols)[None])
        v = hpt.Tensor.from_raw(t.ptr, [rows, cols], k.dtype, 0, [0, 1])
        index = np.broadcast_to(np.array([[1, cols // 2, cols - 2]]), (rows, 3))
        tt = np.broadcast_to(k.round(rng.standard_normal((1, 3))), (rows, 3))
        lse_t = np.full(rows, logsumexp(tt[:1])[0] + 0.7, np.float32)
        got = v.distill_loss(k.up(tt)[0], up(hpt, index), **(dict(teacher_lse=up(hpt, lse_t)) if rest else {}))
        want, _ = diverged(x, tt[:1], index[:1], 1.0, lse_t[:1].astype(np.float64) if rest else None)
        near(got.kl.numpy(), np.broadcast_to(want, rows), kl_tolerance(x, 1.0, want)[0], f"span {span}")


def test_more_than_2_26_rows(hpt, dev):
    """One row of logits and its entries, so often that a workgroup of 1024 threads for each 16 rows would be more work items than a launch has."""
    rows = (1 << 26) + 21
    base = Kind(hpt, "f32").up(np.array([0.25, -1.5, 0.75]))[0]
    v = hpt.Tensor.from_raw(base.ptr, [rows, 3], hpt.f32, 0, [0, 1])
    teacher, index = hpt.Tensor.empty([rows, 1], hpt.f32), hpt.Tensor.empty([rows, 1], hpt.i32)
    for t, a in ((teacher, np.ones(rows, np.float32)), (index, (np.arange(rows) % 3).astype(np.int32))):
        assert hpt.lib().hpt_hip_memcpy_h2d_sync(0, P(t.ptr), a.ctypes.data_as(P), a.nbytes) == 0
    got = v.distill_loss(teacher, index)
    want = (logsumexp(np.array([[0.25, -1.5, 0.75]])) - np.array([0.25, -1.5, 0.75])).astype(np.float32)
    kl = got.kl.numpy()
    assert np.abs(kl.reshape(-1)[:rows // 3 * 3].reshape(-1, 3) - want).max() < 16 * F32_STEP
    assert np.abs(kl[-3:] - want[np.arange(rows - 3, rows) % 3]).max() < 16 * F32_STEP
    near(got.loss.numpy()[0], want.astype(np.float64).mean(), 16 * F32_STEP)

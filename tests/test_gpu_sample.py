"""Sampled tokens on the device, against the definition in 64 bits.

Tokens are exact wherever no border (of the probability mass, of min_p, or between two tokens) lies within 2^-36 of the row's sum of what decides: weights have
half a step of 2^-40 of the largest at most, and a row's sum is off by less than 2^-38 of itself. logp is rounded once."""
import ctypes as C

import numpy as np
import pytest

from block_util import F32_STEP, Guarded, Kind, near, shifted, up
from vocab_util import sampled

pytestmark = pytest.mark.gpu
TYPES = ["f32", "f16", "bf16"]
NEAR = 2.0 ** -36
SETTINGS = [dict(), dict(temperature=0.7), dict(temperature=0.0), dict(top_k=1), dict(top_k=20, top_p=0.8, temperature=0.7), dict(top_k=50), dict(top_k=1024, min_p=0.02),
            dict(top_p=0.9), dict(top_p=0.5, temperature=2.0), dict(top_p=0.0), dict(min_p=0.1), dict(min_p=1.0), dict(top_p=0.95, min_p=0.01), dict(top_k=3000, top_p=0.9),
            dict(top_k=4000), dict(top_p=0.999999), dict(temperature=0.01, top_p=0.99), dict(temperature=50.0, top_p=0.7), dict(temperature=50.0, top_k=2500, min_p=0.5),
            dict(temperature=1e-12), dict(temperature=1e12, top_p=0.3)]


def check(hpt, t, x, u, settings, dev=0, **kw):
    rows = x.shape[0]
    token, logp = Guarded(hpt, [rows], hpt.i64, 1), Guarded(hpt, [rows], hpt.f32, 1)
    ws = Guarded(hpt, [hpt.sample_workspace(t)], hpt.u8)
    t.sample(up(hpt, u), token_out=token.t, logp_out=logp.t, workspace=ws.t, **settings)
    ws.numpy()
    got, lp = token.numpy(), logp.numpy().astype(np.float64)
    each = [{n: v.numpy()[r] if hasattr(v, "numpy") else v for n, v in settings.items()} for r in range(rows)]
    want = [sampled(x[r], u[r], **{n: float(v) if n != "top_k" else int(v) for n, v in each[r].items()}) for r in range(rows)]
    clear = np.array([w[2] > NEAR for w in want])
    tokens, logs = np.array([w[0] for w in want]), np.array([w[1] for w in want])
    # (at 1e12 all weights are the same but for 1e-12, and 0.3 of 5000 is the very border)
    assert clear.sum() * 100 >= 90 * rows or rows < 20 or settings.get("temperature") == 1e12, "most rows decide clearly"
    assert np.array_equal(got[clear], tokens[clear]), [(r, got[r], tokens[r], each[r], u[r]) for r in np.flatnonzero(clear & (got != tokens))[:3]]
    # (1e-11: what a row's sum may be off by, of which the logarithm shows as much)
    near(lp[clear], logs[clear], F32_STEP * np.abs(logs[clear]) + 1e-11)
    return got, lp


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("settings", SETTINGS, ids=lambda s: "-".join(f"{k}{v}" for k, v in s.items()) or "plain")
def test_settings(hpt, dev, name, settings):
    kind = Kind(hpt, name)
    for rows, cols, sd in ((40, 5000, 3), (3, 50257, 2), (1, 152001, 1), (2, 8192, 4), (2, 8193, 4)):
        rng = np.random.default_rng(rows + cols)
        t, x, _ = shifted(hpt, kind, rng.standard_normal((rows, cols)) * sd, 1)
        u = rng.uniform(size=rows).astype(np.float32)
        got, lp = check(hpt, t, x, u, settings)
        # the library's scratch, 32-bit tokens: the same
        i32 = hpt.Tensor.empty([rows], hpt.i32)
        again = t.sample(up(hpt, u), token_out=i32, **settings)
        assert np.array_equal(i32.numpy(), got) and np.array_equal(again[1].numpy().astype(np.float64), lp, equal_nan=True)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 1), (4, 2), (3, 7), (70, 31), (1100, 40), (600, 1000), (64, 9000)])
def test_settings_of_each_row(hpt, dev, name, rows, cols):
    kind, rng = Kind(hpt, name), np.random.default_rng(rows * 7 + cols)
    t, x = kind.up(rng.standard_normal((rows, cols)) * 3)
    u = rng.uniform(size=rows).astype(np.float32)
    some = lambda off, a: np.where(rng.uniform(size=rows) < 0.3, off, a)  # noqa: E731
    f = lambda a: up(hpt, a.astype(np.float32))  # noqa: E731
    settings = dict(temperature=f(some(0.0, rng.uniform(0.3, 2, rows))), top_p=f(some(1.0, rng.uniform(0.1, 1, rows))), min_p=f(some(0.0, rng.uniform(0, 0.5, rows))),
                    top_k=up(hpt, some(0, rng.integers(-1, 2 * cols + 2, rows)).astype(np.int32)))
    got, lp = check(hpt, t, x, u, settings)
    wide = dict(settings, top_k=up(hpt, settings["top_k"].numpy().astype(np.int64)))
    token, logp = t.sample(up(hpt, u), **wide)
    assert np.array_equal(token.numpy(), got) and np.array_equal(logp.numpy(), lp.astype(np.float32))
    # one setting of each row beside three numbers
    check(hpt, t, x, u, dict(temperature=0.8, top_k=settings["top_k"], top_p=0.9))


def test_bad_settings_of_a_row(hpt, dev):
    rng = np.random.default_rng(1)
    t, x = Kind(hpt, "f32").up(rng.standard_normal((6, 3000)))
    nan, inf = np.nan, np.inf
    u = up(hpt, np.full(6, 0.5, np.float32))
    f = lambda a: up(hpt, np.array(a, np.float32))  # noqa: E731
    for kw in (dict(temperature=f([1, -1, nan, inf, 1, 0])), dict(top_p=f([0.5, nan, nan, nan, 0.5, 1])), dict(min_p=f([0.1, nan, nan, nan, 0.1, 0]))):
        token, logp = (a.numpy() for a in t.sample(u, **kw))
        assert (token[1:4] == -1).all() and np.isnan(logp[1:4]).all()
        assert (token[[0, 4, 5]] >= 0).all() and not np.isnan(logp[[0, 4, 5]]).any()


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("cols", [5, 1000, 20001])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=3), dict(top_p=0.5), dict(min_p=0.5), dict(temperature=0.0), dict(top_k=1500, top_p=0.9)], ids=str)
def test_rows_that_tie_and_masked_rows(hpt, dev, name, cols, settings):
    """Few values, masks down to the type's lowest value, rows without a distribution."""
    kind, rng = Kind(hpt, name), np.random.default_rng(cols)
    low = {"f32": -3.4028235e38, "f16": -65504.0, "bf16": -3.3895314e38}[name]
    x = rng.integers(-2, 3, (12, cols)).astype(np.float64)
    x[1] = 0
    x[2] = -7.25
    x[3, 1:] = -np.inf
    x[4, :-1] = low
    x[5, : cols // 2] = -np.inf
    x[6] = low
    x[7] = -np.inf
    x[8, cols // 2] = np.nan
    x[9, cols - 1] = np.inf
    x[10] = np.where(np.arange(cols) % 3, -1e4, 30.0)
    t, x = kind.up(x)
    u = np.array([0.3, 0.49, 0.7, 0.2, 0.9, 0.999, 0.51, 0.5, 0.5, 0.5, 0.123, 0.77], np.float32)
    got, lp = check(hpt, t, x, u, settings)
    assert (got[7:10] == -1).all() and np.isnan(lp[7:10]).all()


def test_half_of_equal_logits(hpt, dev):
    """Of equal logits the first half reaches a half of their sum, whatever their value."""
    for value in (0.0, 1.0, -7.25, 11.3, 0.7):
        for n in (2, 4, 64, 4096):
            t = Kind(hpt, "f32").up(np.full((1, n), value))[0]
            for u, want in ((0.0, 0), (0.9999999, n // 2 - 1)):
                token, logp = t.sample(up(hpt, np.array([u], np.float32)), top_p=0.5)
                assert token.numpy()[0] == want, (value, n, u)
                near(logp.numpy(), [-np.log(n // 2)], F32_STEP * np.log(n) + 1e-11)


def test_numbers_outside(hpt, dev):
    rng = np.random.default_rng(2)
    kind = Kind(hpt, "bf16")
    t, x = kind.up(rng.standard_normal((5, 9000)) * 2)
    u = np.array([-1, 1.0, 7.0, np.nan, 0.0], np.float32)
    for settings in (dict(), dict(top_k=10), dict(top_p=0.7)):
        check(hpt, t, x, u, settings)


def test_frequencies(hpt, dev):
    """Numbers spread evenly give every token its probability: with n of them, to 1 / n."""
    x = np.log(np.array([[0.05, 0.4, 0.01, 0.3, 0.24]]))
    n = 4000
    row = Kind(hpt, "f32").up(x)[0]
    t = hpt.Tensor.from_raw(row.ptr, [n, 5], hpt.f32, 0, [0, 1])
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    for settings, p in ((dict(), [0.05, 0.4, 0.01, 0.3, 0.24]), (dict(top_k=3), [0, 0.4, 0, 0.3, 0.24]), (dict(top_p=0.6), [0, 0.4, 0, 0.3, 0]),
                        (dict(min_p=0.1), [0.05, 0.4, 0, 0.3, 0.24]), (dict(temperature=0.5), [0.05 ** 2, 0.16, 1e-4, 0.09, 0.24 ** 2])):
        p = np.array(p) / np.sum(p)
        token = t.sample(up(hpt, u), **settings)[0].numpy()
        near(np.bincount(token, minlength=5) / n, p, 1.5 / n)


def test_rows_anywhere(hpt, dev):
    rng = np.random.default_rng(3)
    kind = Kind(hpt, "f16")
    wide, x = kind.up(rng.standard_normal((6, 3, 1003)) * 2)
    v = wide.permute([1, 0, 2])[:, ::2]
    part = np.ascontiguousarray(np.transpose(x, (1, 0, 2))[:, ::2]).reshape(9, -1)
    u = rng.uniform(size=9).astype(np.float32)
    for settings in (dict(), dict(top_k=10), dict(top_p=0.7)):
        token, logp = v.sample(up(hpt, u.reshape(3, 3)), **settings)
        want = [sampled(part[r], u[r], **settings) for r in range(9)]
        assert token.shape == logp.shape == [3, 3] and np.array_equal(token.numpy().reshape(-1), [w[0] for w in want])
    # rows more than 2^31 elements apart
    apart = (1 << 31) + 24
    big = hpt.Tensor.empty([apart + 1003], hpt.f16)
    for r in range(2):
        row = kind.store(part[r])
        assert hpt.lib().hpt_hip_memcpy_h2d_sync(0, C.c_void_p(big.ptr + r * apart * 2), row.ctypes.data_as(C.c_void_p), row.nbytes) == 0
    t = hpt.Tensor.from_raw(big.ptr, [2, 1003], hpt.f16, 0, [apart, 1])
    for settings in (dict(), dict(top_k=10), dict(top_p=0.7)):
        check(hpt, t, part[:2], u[:2], settings)


def test_the_largest_vocabulary(hpt, dev):
    cols = 1 << 22
    rng = np.random.default_rng(6)
    t, x = Kind(hpt, "bf16").up(rng.standard_normal((1, cols)) * 3)
    for settings in (dict(), dict(top_k=100), dict(top_p=0.9), dict(top_k=100000, top_p=0.8), dict(temperature=40.0, top_p=0.5)):
        check(hpt, t, x, np.array([0.618], np.float32), settings)


def test_more_rows_than_a_run(hpt, dev):
    rng = np.random.default_rng(5)
    kind, cols = Kind(hpt, "bf16"), 40
    t, x = kind.up(rng.standard_normal((7, cols)) * 2)
    rep = (64 << 20) // hpt.sample_workspace(hpt.Tensor.from_raw(t.ptr, [1, cols], hpt.bf16, 0)) // 7 + 2
    v = hpt.Tensor.from_raw(t.ptr, [rep, 7, cols], hpt.bf16, 0, [0, cols, 1])
    u = rng.uniform(size=7).astype(np.float32)
    token = v.sample(up(hpt, np.tile(u, rep)), top_p=0.8)[0].numpy()
    assert np.array_equal(token, np.broadcast_to([sampled(x[r], u[r], top_p=0.8)[0] for r in range(7)], (rep, 7)))


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("each", [False, True])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=20, top_p=0.8), dict(top_k=600, min_p=0.01), dict(top_p=0.9), dict(min_p=0.05), dict(top_k=3000, top_p=0.9), dict(temperature=0.0)], ids=str)
def test_many_rows(hpt, dev, name, each, settings):
    """More rows than the forms for few rows take: the same twenty again and again, of which some have few values or masks."""
    kind, rng, cols, rep = Kind(hpt, name), np.random.default_rng(8), 20001, 40
    x = rng.standard_normal((20, cols)) * 3
    x[3] = rng.integers(-2, 3, cols)
    x[7] = 1.5
    x[9, cols // 9:] = -np.inf
    x[11, :-3] = -65504.0
    x[13, cols // 2] = np.nan
    x[17] = -np.inf
    t, x = kind.up(x)
    u = rng.uniform(size=20).astype(np.float32)
    want = [sampled(x[r], u[r], **settings) for r in range(20)]
    clear = np.array([w[2] > NEAR for w in want])
    assert clear.sum() >= 18
    v = hpt.Tensor.from_raw(t.ptr, [rep, 20, cols], kind.dtype, 0, [0, cols, 1])
    if each:
        full = dict(dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **settings)
        settings = {n: up(hpt, np.full(rep * 20, a, np.int64 if n == "top_k" else np.float32)) for n, a in full.items()}
        # (a setting of f32 is not quite the number in 64 bits: what it is decides)
        want = [sampled(x[r], u[r], **{n: int(a) if n == "top_k" else float(np.float32(a)) for n, a in full.items()}) for r in range(20)]
        clear = np.array([w[2] > NEAR for w in want])
    token, logp = v.sample(up(hpt, np.tile(u, rep)), **settings)
    token, logp = token.numpy().reshape(rep, 20), logp.numpy().reshape(rep, 20).astype(np.float64)
    assert (token == token[:1]).all() and np.array_equal(logp, np.broadcast_to(logp[:1], logp.shape), equal_nan=True)
    tokens, logs = np.array([w[0] for w in want]), np.array([w[1] for w in want])
    assert np.array_equal(token[0][clear], tokens[clear])
    near(logp[0][clear], logs[clear], F32_STEP * np.abs(logs[clear]) + 1e-11)


def test_a_bucket_of_many(hpt, dev):
    """More logits within an eighth of a power of two of the weights than a list holds, none like another, at the border."""
    rng, cols = np.random.default_rng(9), 120000
    x = np.concatenate([rng.uniform(0, 0.08, (2, 40000)), rng.uniform(-9, -3, (2, cols - 40000))], 1)
    t, x = Kind(hpt, "f32").up(np.stack([rng.permutation(r) for r in x]))
    for settings in (dict(top_p=0.5), dict(top_k=20000), dict(top_k=20000, top_p=0.3), dict(min_p=0.97)):
        check(hpt, t, x, np.array([0.4, 0.9], np.float32), settings)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("settings", [dict(top_k=20, top_p=0.8), dict(top_k=64, min_p=0.01, temperature=1.5), dict(top_k=1), dict(top_p=0.9), dict()], ids=str)
def test_very_many_rows(hpt, dev, name, settings):
    """More rows than a workgroup each is for, of few values and masks among others."""
    kind, rng, cols, rep, n = Kind(hpt, name), np.random.default_rng(10), 20001, 100, 12
    x = rng.standard_normal((n, cols)) * 3
    x[2] = rng.integers(-2, 3, cols)
    x[4] = 1.5
    x[6, cols // 9:] = -np.inf
    x[8, cols // 2] = np.nan
    x[10] = -np.inf
    t, x = kind.up(x)
    u = rng.uniform(size=n).astype(np.float32)
    want = [sampled(x[r], u[r], **settings) for r in range(n)]
    clear = np.array([w[2] > NEAR for w in want])
    assert clear.sum() >= n - 2 and rep * n > 1024
    v = hpt.Tensor.from_raw(t.ptr, [rep, n, cols], kind.dtype, 0, [0, cols, 1])
    token, logp = v.sample(up(hpt, np.tile(u, rep)), **settings)
    token, logp = token.numpy().reshape(rep, n), logp.numpy().reshape(rep, n).astype(np.float64)
    assert (token == token[:1]).all() and np.array_equal(logp, np.broadcast_to(logp[:1], logp.shape), equal_nan=True)
    assert np.array_equal(token[0][clear], np.array([w[0] for w in want])[clear])
    logs = np.array([w[1] for w in want])
    near(logp[0][clear], logs[clear], F32_STEP * np.abs(logs[clear]) + 1e-11)

"""The k largest of each row on the device, against a stable sort, and the rows' log of the sum of exponentials against 64 bits.

Values and indices are exact. The sum's tolerance counts roundings: a thread adds 32 terms in f32 (31 half steps), a term at distance D below
its tile's largest is off by 2 D + 4, with D = 4 + log V on average at most: below 128 half steps together, and lse is rounded once."""
import ctypes as C

import numpy as np
import pytest

from block_util import F32_STEP, Guarded, Kind, near, shifted, up
from vocab_util import logsumexp, order

pytestmark = pytest.mark.gpu
TYPES = ["f32", "f16", "bf16"]
LSE = 128 * F32_STEP

SHAPES = [(1, 1, 1), (4, 2, 2), (3, 7, 7), (5, 31, 8), (70, 100, 33), (3, 1001, 64), (33, 5000, 50), (1, 8192, 1024), (2, 8193, 1000), (1, 1500, 1024), (9, 50257, 64),
          (600, 2000, 20), (1100, 40, 7), (1, 152001, 512), (2, 300000, 20), (530, 9000, 3), (2, 16384, 513)]


def check(hpt, t, x, k, dtype, lse=True, tau=1.0):
    rows = x.shape[0]
    values, index = Guarded(hpt, [rows, k], dtype, 1), Guarded(hpt, [rows, k], hpt.i64, 1)
    total = Guarded(hpt, [rows], hpt.f32, 1)
    ws = Guarded(hpt, [hpt.topk_workspace(t, k)], hpt.u8)
    t.topk(k, lse=lse, temperature=tau, values_out=values.t, index_out=index.t, lse_out=total.t if lse else None, workspace=ws.t)
    ws.numpy()
    want = order(x)[:, :k]
    got = index.numpy()
    assert np.array_equal(got, want), np.argwhere(got != want)[:3]
    return values.numpy(), want, total.numpy().astype(np.float64)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,cols,k", SHAPES)
def test_largest(hpt, dev, name, rows, cols, k):
    kind, rng = Kind(hpt, name), np.random.default_rng(rows + cols)
    t, x, _ = shifted(hpt, kind, rng.standard_normal((rows, cols)) * 3, 1)
    tau = 1.7
    values, at, lse = check(hpt, t, x, k, kind.dtype, True, tau)
    assert np.array_equal(kind.load(values), np.take_along_axis(x, at, -1))
    want = logsumexp(x / tau)
    near(lse, want, LSE + F32_STEP * np.abs(want))
    # fresh results, 32-bit indices, the library's scratch, without the sum
    v, i = t.topk(k)
    assert np.array_equal(v.numpy(), values) and np.array_equal(i.numpy(), at) and i.shape == [rows, k]
    i32 = hpt.Tensor.empty([rows, k], hpt.i32)
    t.topk(k, index_out=i32)
    assert np.array_equal(i32.numpy(), at)


def rows_that_tie(rng, cols):
    """Rows of few different values, masks, and what is no number."""
    few = rng.integers(-3, 4, (2, cols)).astype(np.float64)
    same = np.full((1, cols), 1.5)
    steps = np.repeat(np.arange(-(-cols // 700)), 700)[None, :cols] * 0.5
    one = np.full((1, cols), -np.inf)
    one[0, cols // 3] = 2
    none = np.full((1, cols), -np.inf)
    zeros = np.where(rng.uniform(size=(1, cols)) < 0.5, -0.0, 0.0)
    least = rng.standard_normal((1, cols))
    least[0, cols // 4:] = -65504.0
    nan = rng.standard_normal((3, cols))
    nan[0, ::97] = np.nan
    nan[1, cols // 2] = -np.nan
    nan[2, [1, cols - 1]] = np.inf, np.nan
    return np.concatenate([few, same, steps, one, none, zeros, least, nan])


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("cols,k", [(9, 9), (1000, 64), (5001, 1024), (50257, 100), (33333, 513)])
def test_rows_that_tie(hpt, dev, name, cols, k):
    kind, rng = Kind(hpt, name), np.random.default_rng(cols)
    s = kind.store(rows_that_tie(rng, cols))
    if name != "f32":  # NaNs of both signs and of any payload
        bits = s.view(np.uint16)
        bits[-2, cols // 2] = 0xFFFF if name == "bf16" else 0xFC01
    else:
        s.view(np.uint32)[-2, cols // 2] = 0xFFFFFFFF
    t = hpt.Tensor.from_numpy(s, kind.dtype).to_hip(dev)
    x = kind.load(s)
    values, at, lse = check(hpt, t, x, k, kind.dtype)
    assert np.array_equal(values.view(np.uint8), np.take_along_axis(s, at, -1).view(np.uint8)), "the very bits of the logits"
    nan = np.isnan(x).any(-1)
    want = np.where(nan, np.nan, logsumexp(np.where(np.isnan(x), 0, x)))
    near(lse, want, LSE + F32_STEP * np.abs(np.where(np.isfinite(want), want, 0)))
    inf = np.zeros((1, cols))
    inf[0, cols // 2] = np.inf
    assert kind.up(inf)[0].topk(1, lse=True)[2].numpy()[0] == np.inf


def test_rows_anywhere(hpt, dev):
    """Rows of a wider buffer, broadcast rows, and a leading shape."""
    rng = np.random.default_rng(3)
    kind = Kind(hpt, "bf16")
    wide, x = kind.up(rng.standard_normal((6, 3, 1003)))
    v = wide.permute([1, 0, 2])[:, ::2]
    part = np.transpose(x, (1, 0, 2))[:, ::2]
    values, index = v.topk(5)
    assert index.shape == [3, 3, 5]
    want = order(part.reshape(9, -1))[:, :5].reshape(3, 3, 5)
    assert np.array_equal(index.numpy(), want) and np.array_equal(kind.load(values.numpy()), np.take_along_axis(part, want, -1))
    rep = hpt.Tensor.from_raw(wide.ptr, [4, 1003], kind.dtype, 0, [0, 1])
    assert np.array_equal(rep.topk(3)[1].numpy(), np.repeat(order(x[0, :1])[:, :3], 4, 0))
    row = hpt.Tensor.from_raw(wide.ptr, [1003], kind.dtype, 0)
    values, index, lse = row.topk(3, lse=True)
    assert index.shape == [3] and lse.shape == [1] and np.array_equal(index.numpy(), order(x[0, :1])[0, :3])


def test_offsets_beyond_32_bits(hpt, dev):
    """Rows that lie more than 2^31 elements apart."""
    rng = np.random.default_rng(4)
    kind, cols, apart = Kind(hpt, "bf16"), 9001, (1 << 31) + 24
    big = hpt.Tensor.empty([apart + cols], hpt.bf16)
    s = kind.store(rng.standard_normal((2, cols)))
    for r in range(2):
        row = np.ascontiguousarray(s[r])
        assert hpt.lib().hpt_hip_memcpy_h2d_sync(0, C.c_void_p(big.ptr + r * apart * 2), row.ctypes.data_as(C.c_void_p), row.nbytes) == 0
    t = hpt.Tensor.from_raw(big.ptr, [2, cols], hpt.bf16, 0, [apart, 1])
    check(hpt, t, kind.load(s), 40, hpt.bf16)


@pytest.mark.parametrize("cols", [40, 50257])
def test_more_rows_than_a_run(hpt, dev, cols):
    """Rows are taken in runs of as many as their scratch allows."""
    kind, rng = Kind(hpt, "f32"), np.random.default_rng(5)
    row = hpt.topk_workspace(hpt.Tensor.from_raw(1 << 40, [1, cols], hpt.f32, 0), 5)
    rows = (64 << 20) // row + 3
    base = rng.standard_normal((7, cols))
    t, x = kind.up(base)
    # the same seven rows again and again, and nothing is copied: a broadcast leading dim
    rep = -(-rows // 7)
    v = hpt.Tensor.from_raw(t.ptr, [rep, 7, cols], hpt.f32, 0, [0, cols, 1])
    assert hpt.topk_workspace(v, 5) < rep * 7 * row
    index = v.topk(5)[1].numpy()
    assert np.array_equal(index, np.broadcast_to(order(x)[:, :5], (rep, 7, 5)))


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("k", [3, 64, 128, 200, 513, 1024])
def test_many_rows(hpt, dev, name, k):
    """More rows than the form for few rows takes: rows of few values and masks among others, again and again."""
    kind, rng, cols, rep = Kind(hpt, name), np.random.default_rng(k), 20001, 30
    ties = rows_that_tie(rng, cols)
    # (places that differ by their index alone but for a few: more than the digits of a key can tell apart)
    near_same = 1.0 + (rng.uniform(size=(2, cols)) < 0.02) * 2.0 ** -7 * np.array([[1.0], [2.0]])
    t, x = kind.up(np.concatenate([ties, near_same, rng.standard_normal((12, cols)) * 3]))
    n = x.shape[0]
    v = hpt.Tensor.from_raw(t.ptr, [rep, n, cols], kind.dtype, 0, [0, cols, 1])
    values, index, lse = v.topk(k, lse=True)
    want = order(x)[:, :k]
    assert np.array_equal(index.numpy(), np.broadcast_to(want, (rep, n, k)))
    assert np.array_equal(values.numpy(), np.broadcast_to(kind.store(np.take_along_axis(x, want, -1)), (rep, n, k)), equal_nan=name != "bf16")
    few = t.topk(k, lse=True)
    assert np.array_equal(few[1].numpy(), want)
    got, nan = lse.numpy().astype(np.float64), np.isnan(x).any(-1)
    exact = np.where(nan, np.nan, logsumexp(np.where(np.isnan(x), 0, x)))
    near(got[0], exact, LSE + F32_STEP * np.abs(np.where(np.isfinite(exact), exact, 0)))
    assert np.array_equal(got, np.broadcast_to(got[:1], got.shape), equal_nan=True)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("cols,k", [(9, 9), (40, 8), (64, 64), (65, 33), (256, 64), (257, 1), (1000, 20), (1024, 64), (2048, 64), (2048, 3), (2049, 64)])
def test_small_rows(hpt, dev, name, cols, k):
    """A router's rows and others that a wavefront holds: few and many of them, of few values, off the vectors' grid, every k-th of a wider buffer."""
    kind, rng = Kind(hpt, name), np.random.default_rng(cols * 3 + k)
    x = np.concatenate([rows_that_tie(rng, cols), rng.standard_normal((13, cols))])
    t, x, _ = shifted(hpt, kind, x, 1)
    values, at, lse = check(hpt, t, x, k, kind.dtype, True, 0.8)
    assert np.array_equal(kind.load(values), np.take_along_axis(x, at, -1), equal_nan=True)
    nan = np.isnan(x).any(-1)
    exact = np.where(nan, np.nan, logsumexp(np.where(np.isnan(x), 0, x) / 0.8))
    near(lse, exact, LSE + F32_STEP * np.abs(np.where(np.isfinite(exact), exact, 0)))
    n = len(x)
    v = hpt.Tensor.from_raw(t.ptr, [50, n, cols], kind.dtype, 0, [0, cols, 1])
    i32 = hpt.Tensor.empty([50, n, k], hpt.i32)
    many = v.topk(k, index_out=i32)
    assert np.array_equal(i32.numpy(), np.broadcast_to(at, (50, n, k)))
    assert np.array_equal(kind.load(many[0].numpy()), np.broadcast_to(np.take_along_axis(x, at, -1), (50, n, k)), equal_nan=True)
    apart = v[:, ::2]
    assert np.array_equal(apart.topk(k)[1].numpy(), np.broadcast_to(at[::2], (50, len(at[::2]), k)))


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("cols,k", [(20001, 1), (20001, 20), (20001, 64), (40003, 50)])
def test_very_many_rows(hpt, dev, name, cols, k):
    """More rows than a workgroup each is for, of few values and masks among others."""
    kind, rng, rep = Kind(hpt, name), np.random.default_rng(cols + k), 50
    x = np.concatenate([rows_that_tie(rng, cols), rng.standard_normal((11, cols)) * 3, np.sort(rng.standard_normal((3, cols)))])
    t, x = kind.up(x)
    n = len(x)
    v = hpt.Tensor.from_raw(t.ptr, [rep, n, cols], kind.dtype, 0, [0, cols, 1])
    assert rep * n > 1024
    values, index, lse = v.topk(k, lse=True)
    want = order(x)[:, :k]
    assert np.array_equal(index.numpy(), np.broadcast_to(want, (rep, n, k)))
    assert np.array_equal(kind.load(values.numpy()), np.broadcast_to(np.take_along_axis(x, want, -1), (rep, n, k)), equal_nan=True)
    got, nan = lse.numpy().astype(np.float64), np.isnan(x).any(-1)
    exact = np.where(nan, np.nan, logsumexp(np.where(np.isnan(x), 0, x)))
    near(got[-1], exact, LSE + F32_STEP * np.abs(np.where(np.isfinite(exact), exact, 0)))
    assert np.array_equal(got, np.broadcast_to(got[:1], got.shape), equal_nan=True)

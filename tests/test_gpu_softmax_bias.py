"""softmax(scale * scores + table[bucket(key - query), head]) on the device against the definition in 64 bits, and its backward pass.

Tolerances count roundings: a result is off by half a step of its type; a score of size S (scaled, biased) by 2 half steps of f32, which
its exponential turns into 2 S relative; the exponential of a distance D below the maximum by 2 D + 4 half steps (the hardware's
form; the argument is rounded once in the change of base); sums by 64 (32 terms a thread, a tree above). So 4 S + 72, S the largest score."""
import numpy as np
import pytest

from block_util import F32_STEP, Guarded, Kind, near, shifted, up

pytestmark = pytest.mark.gpu
TYPES = ["f32", "f16", "bf16"]


def bucket(rel, total, both, most):
    """By whole numbers: bucket half + j begins where (d / half)^(n - half) >= (most / half)^j."""
    n = total // 2 if both else total
    half = n // 2
    first = n if both and rel > 0 else 0
    d = abs(rel) if both else max(-rel, 0)
    if d < half:
        return first + d
    j = 0
    while half + j + 1 < n and d ** (n - half) * half ** (j + 1) >= most ** (j + 1) * half ** (n - half):
        j += 1
    return first + half + j


def buckets_of(q, k, offset, total, both, most):
    each = np.array([bucket(r, total, both, most) for r in range(-most - 1, most + 2)])  # beyond: the last ones
    rel = np.arange(k) - np.arange(q)[:, None] - offset
    return each[np.clip(rel, -most - 1, most + 1) + most + 1]


def live_of(batch, q, k, offset, causal, lengths):
    live = np.ones((batch, 1, q, k), bool)
    if causal:
        live &= np.arange(k) <= np.arange(q)[:, None] + offset
    if lengths is not None:
        live &= np.arange(k) < np.asarray(lengths).reshape(-1, 1, 1, 1)
    return live


def forward(x, table, which, live, scale):
    t = scale * x + np.moveaxis(table[which], -1, 0)
    t = np.where(live, t, -np.inf)
    any_ = live.any(-1, keepdims=True)
    m = np.where(any_, t.max(-1, keepdims=True), 0)
    with np.errstate(invalid="ignore"):
        e = np.where(live, np.exp(t - m), 0)
        s = e.sum(-1, keepdims=True)
        return np.where(live, e / np.where(any_, s, 1), 0), np.abs(np.where(np.isfinite(t), t, 0)).max()


CASES = [
    # batch, heads, queries, keys, buckets, both, most, offset, causal, lengths
    (1, 1, 1, 1, 8, True, 16, 0, False, None),
    (2, 3, 5, 7, 8, True, 16, 0, False, None),
    (2, 3, 7, 5, 8, False, 16, 0, True, None),
    (2, 2, 9, 64, 32, True, 128, 55, True, [64, 30]),
    (3, 2, 33, 65, 32, True, 128, 0, False, [0, 1, 65]),
    (1, 2, 20, 300, 32, False, 128, 280, True, None),
    (2, 2, 300, 300, 32, True, 64, 0, False, [299, 17]),
    (1, 1, 130, 513, 64, False, 256, 383, True, None),
    (2, 4, 1, 1000, 32, False, 128, 999, True, [1000, 400]),
    (1, 2, 3, 1024, 16, True, 512, 500, False, None),
    (1, 2, 40, 24, 16, True, 20, -30, True, None),      # the first queries stand before every key
    (2, 1, 4, 100, 3, False, 9, 96, True, [100, -5]),
    (1, 1, 6, 2051, 2, False, 4096, 2045, True, None),
    (1, 1, 3, 9000, 256, True, 4096, 4000, False, None),
    (1, 2, 2, 17000, 32, True, 128, 9000, False, None),
    (1, 1, 2, 33000, 32, False, 128, 32998, True, None),
    (1, 2, 2, 70001, 32, True, 128, 60000, False, [69000]),
]


def ids(c):
    return "x".join(map(str, c[:4])) + f"-b{c[4]}{'both' if c[5] else ''}" + ("-causal" if c[8] else "") + ("-lengths" if c[9] else "")


def args_of(c):
    return dict(bidirectional=c[5], max_distance=c[6], query_offset=c[7], causal=c[8])


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("c", CASES, ids=ids)
def test_forward(hpt, dev, name, c):
    batch, heads, q, n, total, both, most, offset, causal, lengths = c
    k, rng = Kind(hpt, name), np.random.default_rng(q * n)
    shape = [batch, heads, q, n]
    x = rng.standard_normal(shape) * 16
    live = live_of(batch, q, n, offset, causal, lengths)
    x[~np.broadcast_to(live, shape)] = np.nan  # what is hidden is not read
    t, x = k.up(x)
    tab, table = k.up(rng.standard_normal((total, heads)))
    ln = None if lengths is None else up(hpt, np.array(lengths, np.int64))
    out = Guarded(hpt, shape, k.dtype)
    t.softmax_bias(tab, 0.125, lengths=ln, out=out.t, **args_of(c))
    which = buckets_of(q, n, offset, total, both, most)
    want, size = forward(np.where(live, x, 0), table, which, live, 0.125)
    got = k.load(out.numpy())
    assert not got[~np.broadcast_to(live, shape)].any()
    near(got, want, want * (k.step + (4 * size + 72) * F32_STEP) + k.least)
    # 32-bit lengths, a table that lies the other way round, in place
    ln32 = None if lengths is None else up(hpt, np.array(lengths, np.int32))
    turned, _ = k.up(table.T)
    again = t.softmax_bias(turned.t(), 0.125, lengths=ln32, out=t, **args_of(c))
    assert np.array_equal(again.numpy(), out.numpy())


# Where the deal of a row to threads changes: one row of few, one of many, and whole matrices, one vector to both sides.
EDGES = [(1, 2, q, n, 32, True, 64, q // 2 + n // 2, False, None) for n in (1016, 1025, 1031, 2047, 2049, 3079, 4105, 6145, 8200, 9217, 16391, 18440) for q in (1, 5)] + [
    (8, 130, 1, n, 16, False, 32, n - 1, True, None) for n in (130, 513, 1030, 2056, 3085)]


# Fewer queries and keys than distances, in front of one another, apart by less and by more than the last bucket begins at.
NEAR = [(2, 2, 6, 10, 32, both, 256, offset, causal, None) for both, causal in ((True, False), (False, True), (False, False)) for offset in (0, -5, 9, -50, 300, -300, 1 << 40, -(1 << 40))]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("c", NEAR, ids=lambda c: f"{'both' if c[5] else ''}{c[7]}{'-causal' if c[8] else ''}")
def test_distances_out_of_reach(hpt, dev, name, c):
    test_forward(hpt, dev, name, c)
    test_backward(hpt, dev, name, c)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("c", EDGES, ids=ids)
def test_edges_of_the_deal(hpt, dev, name, c):
    test_forward(hpt, dev, name, c)


@pytest.mark.parametrize("total,both,most", [(32, True, 128), (32, False, 128), (16, True, 64), (2, False, 2), (4, True, 2), (256, True, 4096), (256, False, 4096), (6, True, 1000),
                                             (7, False, 33), (64, True, 17)])
def test_every_distance_is_in_its_bucket(hpt, dev, total, both, most):
    """All buckets but one at -1e30: the keys that keep a share are exactly that bucket's."""
    n = min(2 * most + 40, 8300)
    pos = n // 2
    which = np.array([bucket(j - pos, total, both, most) for j in range(n)])
    x = hpt.Tensor.zeros([total, 1, 1, n], hpt.f32)
    # one batch entry for each bucket: through the heads, each with a table of its own
    x = hpt.Tensor.zeros([1, total, 1, n], hpt.f32)
    table = np.full((total, total), -1e30, np.float32)
    np.fill_diagonal(table, 0)
    p = x.softmax_bias(up(hpt, table), 1.0, bidirectional=both, max_distance=most, query_offset=pos).numpy()[0, :, 0]
    for b in range(total):
        has = which == b
        if has.any():
            assert np.array_equal(p[b] > 0, has), b


@pytest.mark.parametrize("name", TYPES)
def test_strided_scores(hpt, dev, name):
    k, rng = Kind(hpt, name), np.random.default_rng(9)
    t, x = k.up(rng.standard_normal((3, 20, 4, 48)) * 8)
    tab, table = k.up(rng.standard_normal((8, 4)))
    for what, v, a in (("queries before heads", t.permute([0, 2, 1, 3]), x.transpose(0, 2, 1, 3)), ("part of the keys", t.permute([0, 2, 1, 3])[:, :, :, 5:40], x.transpose(0, 2, 1, 3)[..., 5:40]),
                       ("every second query", t.permute([0, 2, 1, 3])[:, :, ::2], x.transpose(0, 2, 1, 3)[:, :, ::2])):
        q, n = a.shape[-2:]
        want, size = forward(a, table, buckets_of(q, n, 3, 8, True, 16), live_of(3, q, n, 3, True, None), 1.0)
        near(k.down(v.softmax_bias(tab, 1.0, max_distance=16, query_offset=3, causal=True)), want, want * (k.step + (4 * size + 72) * F32_STEP) + k.least, what)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("shift", [1, 3])
@pytest.mark.parametrize("n", [64, 77, 1030, 40000])
def test_off_the_grid(hpt, dev, name, shift, n):
    k, rng = Kind(hpt, name), np.random.default_rng(n)
    t, x, base = shifted(hpt, k, rng.standard_normal((2, 5, n)) * 8, shift)
    tab, table = k.up(rng.standard_normal((8, 2)))
    out = Guarded(hpt, [2, 5, n], k.dtype, 4 - shift)
    t.softmax_bias(tab, 0.5, max_distance=16, query_offset=7, out=out.t)
    which, live = buckets_of(5, n, 7, 8, True, 16), live_of(1, 5, n, 7, False, None)
    want, size = forward(x[None], table, which, live, 0.5)
    got = k.load(out.numpy())
    near(got, want[0], want[0] * (k.step + (4 * size + 72) * F32_STEP) + k.least)
    g, grad, b2 = shifted(hpt, k, rng.standard_normal((2, 5, n)), shift)
    gx, gt = Guarded(hpt, [2, 5, n], k.dtype, 4 - shift), Guarded(hpt, [8, 2], hpt.f32, shift)
    out.t.softmax_bias_backward(g, 8, 0.5, max_distance=16, query_offset=7, out=gx.t, table_out=gt.t)
    check_grad(k, got[None], grad[None], which, live, 0.5, 8, k.load(gx.numpy())[None], gt.numpy())


@pytest.mark.parametrize("n", [40, 1000, 70000])
@pytest.mark.parametrize("name", TYPES)
def test_infinities_and_nan(hpt, dev, name, n):
    k, rng = Kind(hpt, name), np.random.default_rng(2)
    x = rng.standard_normal((1, 7, n))
    x[0, 1] = -np.inf                      # nothing but masked by the caller
    x[0, 2, 3:] = -np.inf
    x[0, 3, 5] = np.nan
    x[0, 4, 6] = np.inf
    low = {"f32": np.finfo(np.float32).min, "f16": -65504.0, "bf16": -3.3895313892515355e38}[name]
    x[0, 5, 4:] = low                      # the type's lowest value as a mask
    x[0, 6] = low
    t, x = k.up(x)
    tab, table = k.up(np.zeros((8, 1)))
    live = live_of(1, 7, n, n - 9, True, None)
    got = k.down(t.softmax_bias(tab, 1.0, max_distance=16, query_offset=n - 9, causal=True))[0]
    hidden = ~live[0, 0]
    assert not got[hidden].any()
    seen = live[0, 0]
    for row in (1, 3, 4):
        assert np.isnan(got[row][seen[row]]).all(), row
    for row, keys in ((2, 3), (5, 4)):
        e = np.exp(x[0, row, :keys] - x[0, row, :keys].max())
        near(got[row, :keys], e / e.sum(), e * (k.step + 100 * F32_STEP))
        assert not got[row, keys:].any()
    near(got[6][seen[6]], np.full(seen[6].sum(), 1 / seen[6].sum()), (k.step + 100 * F32_STEP) / seen[6].sum() + k.least)
    near(got[0].sum(), 1, k.step * 4 + 1e-5)


# ---- backward ------------------------------------------------------------------------------------------

def backward(p, g, which, live, scale, total):
    g = np.where(live, g, 0)
    p = np.where(live, p, 0)
    s, sa = (p * g).sum(-1, keepdims=True), (p * np.abs(g)).sum(-1, keepdims=True)
    d, size = p * (g - s), p * (np.abs(g) + sa)
    heads = p.shape[1]
    table, ts = np.zeros((total, heads)), np.zeros((total, heads))
    d0, s0 = d.sum(0), size.sum(0)
    for b in range(total):
        on = which == b
        table[b], ts[b] = d0[:, on].sum(-1), s0[:, on].sum(-1)
    return scale * d, abs(scale) * size, table, ts


def check_grad(k, p, g, which, live, scale, total, gx, gtable):
    want, size, wt, st = backward(p, g, which, live, scale, total)
    near(gx, want, k.step * np.abs(want) + 100 * F32_STEP * size + k.least, "gradient of the scores")
    # (each d is off by 100 half steps of its terms; a thread adds what it has of a row, 32 at most, and of the rows of its workgroup)
    near(gtable, wt, (100 + 32 + 64) * F32_STEP * st + 1e-40, "gradient of the table")


def test_the_formula_against_differences():
    rng = np.random.default_rng(0)
    which = buckets_of(4, 6, 1, 8, True, 8)
    live = live_of(2, 4, 6, 1, True, [6, 3])
    x, table, g = rng.standard_normal((2, 3, 4, 6)), rng.standard_normal((8, 3)), rng.standard_normal((2, 3, 4, 6))
    f = lambda x, table: (forward(x, table, which, live, 0.7)[0] * g).sum()  # noqa: E731
    gx, _, gt, _ = backward(forward(x, table, which, live, 0.7)[0], g, which, live, 0.7, 8)
    d = 1e-6
    for a, grad in ((x, gx), (table, gt)):
        for i in np.ndindex(a.shape):
            keep = a[i]
            a[i] = keep + d
            hi = f(x, table)
            a[i] = keep - d
            lo = f(x, table)
            a[i] = keep
            assert abs((hi - lo) / (2 * d) - grad[i]) < 1e-8


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("c", CASES + [(2, 2, 700, 90, 32, True, 128, 0, False, [90, 50]), (1, 3, 1100, 140, 16, False, 64, 0, True, None), (1, 1, 2100, 600, 32, False, 128, 0, True, None)], ids=ids)
def test_backward(hpt, dev, name, c):
    batch, heads, q, n, total, both, most, offset, causal, lengths = c
    k, rng = Kind(hpt, name), np.random.default_rng(q * n + 1)
    shape = [batch, heads, q, n]
    live = live_of(batch, q, n, offset, causal, lengths)
    e = np.where(live, np.exp(rng.standard_normal(shape)), 0)
    p = e / np.maximum(e.sum(-1, keepdims=True), 1e-30)
    g = rng.standard_normal(shape)
    g[~np.broadcast_to(live, shape)] = np.inf
    t, p = k.up(p)
    gr, g = k.up(g)
    ln = None if lengths is None else up(hpt, np.array(lengths, np.int64))
    out, tg = Guarded(hpt, shape, k.dtype), Guarded(hpt, [total, heads], hpt.f32)
    need = hpt.softmax_bias_backward_workspace(t, total)
    ws = Guarded(hpt, [need], hpt.u8)
    t.softmax_bias_backward(gr, total, 0.3, lengths=ln, out=out.t, table_out=tg.t, workspace=ws.t, **args_of(c))
    ws.numpy()
    gx = k.load(out.numpy())
    assert not gx[~np.broadcast_to(live, shape)].any()
    check_grad(k, p, g, buckets_of(q, n, offset, total, both, most), live, 0.3, total, gx, tg.numpy())
    # the library's own scratch; in the gradient's place
    a, b = t.softmax_bias_backward(gr, total, 0.3, lengths=ln, out=gr, **args_of(c))
    assert np.array_equal(a.numpy(), out.numpy()) and np.array_equal(b.numpy(), tg.numpy())
    # in the probabilities' place, the gradient as before
    gr, _ = k.up(np.where(live, g, 0))
    a, b = t.softmax_bias_backward(gr, total, 0.3, lengths=ln, out=t, **args_of(c))
    assert np.array_equal(a.numpy(), out.numpy()) and np.array_equal(b.numpy(), tg.numpy())


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("n", [510, 520, 1033, 2047, 2056, 4104, 6160, 9000])
def test_edges_of_the_backward_deal(hpt, dev, name, n):
    test_backward(hpt, dev, name, (1, 2, 37, n, 32, True, 64, n // 2, False, None))


def test_backward_without_rows_or_table(hpt, dev):
    p = hpt.Tensor.empty([2, 3, 0, 5], hpt.f32)
    gx, gt = p.softmax_bias_backward(hpt.Tensor.empty([2, 3, 0, 5], hpt.f32), 8)
    assert gx.shape == [2, 3, 0, 5] and gt.shape == [8, 3] and not gt.numpy().any()
    p = hpt.Tensor.empty([0, 3, 4, 5], hpt.f32)
    assert not p.softmax_bias_backward(hpt.Tensor.empty([0, 3, 4, 5], hpt.f32), 8)[1].numpy().any()
    import ctypes as C
    from hpt_amd import _ffi
    k, rng = Kind(hpt, "f32"), np.random.default_rng(4)
    t, _ = k.up(rng.uniform(0, 0.1, (2, 6, 40)))
    g, _ = k.up(rng.standard_normal((2, 6, 40)))
    out = hpt.Tensor.empty([2, 6, 40], hpt.f32)
    (vx, k1), (vg, k2), (vo, k3) = t._c_view(), g._c_view(), out._c_view()
    _ffi.check(hpt.lib().hpt_hip_softmax_bias_backward(0, None, C.byref(vx), C.byref(vg), 0.5, 1, 128, 0, 1, None, None, C.byref(vo), None))
    assert np.array_equal(out.numpy(), t.softmax_bias_backward(g, 32, 0.5, causal=True)[0].numpy())


@pytest.mark.parametrize("name", TYPES)
def test_a_workspace_gives_the_same(hpt, dev, name):
    """Few, long rows with a workspace, with the library's scratch, and unevenly divided."""
    k, rng = Kind(hpt, name), np.random.default_rng(6)
    tab, table = k.up(rng.standard_normal((8, 2)))
    for n in (40000, 65537, 131072):
        t, x = k.up(rng.standard_normal((2, 1, n)) * 4)
        need = hpt.softmax_bias_workspace(t)
        ws = Guarded(hpt, [max(need, 1)], hpt.u8)
        a = t.softmax_bias(tab, max_distance=16, query_offset=n - 1, workspace=ws.t)
        ws.numpy()
        assert np.array_equal(a.numpy(), t.softmax_bias(tab, max_distance=16, query_offset=n - 1).numpy())
        d = np.clip(np.arange(n) - (n - 1), -16, 16)
        near_ones = np.array([bucket(i, 8, True, 16) for i in range(-16, 17)])
        want, size = forward(x[None], table, near_ones[d + 16][None], np.ones((1, 1, 1, n), bool), 1.0)
        near(k.down(a), want[0], want[0] * (k.step + (4 * size + 72 + n / 8192) * F32_STEP) + k.least)

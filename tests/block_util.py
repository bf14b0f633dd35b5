"""Shared by the tests of the operators around a transformer's blocks: the three dtypes as numpy carries them, and tensors that live
inside a larger buffer, so that a byte written beside a result shows."""
import numpy as np

F32_STEP = 2.0 ** -24  # half a step of f32, relative


class Kind:
    """A dtype: numbers -> its values, and back; `step`: half a step, relative; `least`: half the smallest subnormal."""

    def __init__(self, hpt, name):
        self.name, self.hpt = name, hpt
        self.dtype = getattr(hpt, name)
        self.step, self.least = {"f32": (2.0 ** -24, 2.0 ** -150), "f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 2.0 ** -134)}[name]

    def store(self, x):
        x = np.asarray(x, np.float32)
        if self.name == "f32":
            return x.copy()
        return self.hpt.f32_to_bf16_bits(x) if self.name == "bf16" else x.astype(np.float16)

    def load(self, a):
        return (self.hpt.bf16_bits_to_f32(a) if self.name == "bf16" else a).astype(np.float64)

    def round(self, x):
        return self.load(self.store(x))

    def up(self, x, dev=0):
        """A device tensor of these numbers, and the numbers that it holds."""
        s = self.store(x)
        return self.hpt.Tensor.from_numpy(s, self.dtype).to_hip(dev), self.load(s)

    def down(self, t):
        return self.load(t.numpy())


def up(hpt, a, dev=0):
    return hpt.Tensor.from_numpy(np.ascontiguousarray(a)).to_hip(dev)


GUARD = 96  # bytes on both sides


class Guarded:
    """A contiguous result that starts `shift` elements behind a 64-byte boundary of a buffer filled with a pattern."""

    def __init__(self, hpt, shape, dtype, shift=0, dev=0):
        n = int(np.prod(shape))
        self.hpt, self.dtype, self.n, self.shape = hpt, dtype, n, list(shape)
        self.at = GUARD * 2 // dtype.size + shift
        self.pattern = np.random.default_rng(n + 17).integers(0, 256, (self.at + n) * dtype.size + 2 * GUARD, dtype=np.uint8)
        self.base = up(hpt, self.pattern, dev)
        self.t = hpt.Tensor.from_raw(self.base.ptr + self.at * dtype.size, shape, dtype, dev)

    def numpy(self):
        """The result, after a look at what lies around it."""
        self.hpt.synchronize(self.t.device)
        b = self.base.numpy()
        lo, hi = self.at * self.dtype.size, (self.at + self.n) * self.dtype.size
        assert np.array_equal(b[:lo], self.pattern[:lo]), "written in front of the result"
        assert np.array_equal(b[hi:], self.pattern[hi:]), "written behind the result"
        return b[lo:hi].view(self.dtype.np_dtype).reshape(self.shape)


def shifted(hpt, kind, x, shift, dev=0):
    """The numbers of `x` in a device tensor that starts `shift` elements behind a boundary; (tensor, numbers, owner)."""
    s = kind.store(x)
    flat = np.concatenate([np.zeros(shift, s.dtype), s.reshape(-1)])
    base = hpt.Tensor.from_numpy(flat, kind.dtype).to_hip(dev)
    return hpt.Tensor.from_raw(base.ptr + shift * kind.dtype.size, s.shape, kind.dtype, dev), kind.load(s), base


def near(got, want, tol, what=""):
    """|got - want| <= tol, element by element; NaN and infinities in the same places."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, f"{what}: {got.shape} != {want.shape}"
    tol = np.broadcast_to(tol, want.shape)
    with np.errstate(invalid="ignore"):
        ok = (np.abs(got - want) <= tol) | (np.isnan(got) & np.isnan(want)) | (got == want)
    if not ok.all():
        at = tuple(np.argwhere(~ok)[0])
        raise AssertionError(f"{what}: {(~ok).sum()} of {ok.size} are off; first at {at}: got {got[at]!r}, want {want[at]!r}, tolerance {tol[at]!r}")

"""How top-k, sampling and distillation are called: captured into graphs and replayed, on streams of the caller, from several threads, through
ctypes, and all of them together as a teacher, a student and a server use them."""
import threading

import numpy as np
import pytest

from block_util import F32_STEP, Kind, near, up
from test_gpu_block_calls import P, hip, stream  # noqa: F401
from vocab_util import distilled, logsumexp, order, sampled

pytestmark = pytest.mark.gpu


class Calls:
    """One call of every operator into results of its own, on inputs that can be written anew. Long rows, so that all of them are split."""

    def __init__(self, hpt, name, rows=12, cols=40009, seed=0):
        self.hpt, self.k, rng = hpt, Kind(hpt, name), np.random.default_rng(seed)
        k, e = self.k, hpt.Tensor.empty
        self.host = {"x": rng.standard_normal((rows, cols)) * 3, "t": rng.standard_normal((rows, cols)) * 3}
        self.dev = {n: k.up(a)[0] for n, a in self.host.items()}
        self.u = up(hpt, rng.uniform(size=rows).astype(np.float32))
        f = lambda a: up(hpt, np.asarray(a, np.float32))  # noqa: E731
        some = lambda off, a: np.where(np.arange(rows) % 3 == 0, off, a)  # noqa: E731
        self.each = dict(temperature=f(some(0, rng.uniform(0.5, 2, rows))), top_k=up(hpt, some(0, rng.integers(1, 3000, rows)).astype(np.int32)),
                         top_p=f(rng.uniform(0.3, 1, rows)), min_p=f(rng.uniform(0, 0.2, rows)))
        i64, f32 = hpt.i64, hpt.f32
        self.out = {"v": e([rows, 50], k.dtype), "i": e([rows, 50], i64), "tl": e([rows], f32), "loss": e([1], f32), "kl": e([rows], f32), "terms": e([rows, 8], f32),
                    "loss2": e([1], f32), "kl2": e([rows], f32), "terms2": e([rows, 8], f32), "g": e([rows, cols], k.dtype), "g2": e([rows, cols], k.dtype)}
        for n in range(4):
            self.out.update({f"token{n}": e([rows], i64), f"logp{n}": e([rows], f32)})
        d = self.dev
        self.ws = {"topk": e([hpt.topk_workspace(d["t"], 50)], hpt.u8), "sample": e([hpt.sample_workspace(d["x"])], hpt.u8),
                   "distill": e([hpt.distill_loss_workspace(d["x"])], hpt.u8)}

    def write(self, seed):
        rng = np.random.default_rng(seed)
        for n in ("x", "t"):
            a = self.k.store(self.host[n] * rng.uniform(0.5, 1.5, self.host[n].shape))
            assert self.hpt.lib().hpt_hip_memcpy_h2d_sync(0, P(self.dev[n].ptr), a.ctypes.data_as(P), a.nbytes) == 0

    def run(self, stream=None, ws=True):  # noqa: F811
        x, t, o, w = self.dev["x"], self.dev["t"], self.out, self.ws if ws else {}
        kw = dict(temperature=2.0, stream=stream)
        t.topk(50, lse=True, values_out=o["v"], index_out=o["i"], lse_out=o["tl"], workspace=w.get("topk"), **kw)
        x.distill_loss(o["v"], o["i"], loss_out=o["loss"], kl_out=o["kl"], terms_out=o["terms"], workspace=w.get("distill"), **kw)
        x.distill_loss_backward(o["v"], o["i"], o["terms"], grad=100.0, out=o["g"], **kw)
        x.distill_loss(o["v"], o["i"], teacher_lse=o["tl"], loss_out=o["loss2"], kl_out=o["kl2"], terms_out=o["terms2"], workspace=w.get("distill"), **kw)
        x.distill_loss_backward(o["v"], o["i"], o["terms2"], grad=100.0, out=o["g2"], **kw)
        for n, s in enumerate((dict(), dict(top_k=40, top_p=0.9), dict(top_p=0.9, temperature=0.8), self.each)):
            x.sample(self.u, stream=stream, token_out=o[f"token{n}"], logp_out=o[f"logp{n}"], workspace=w.get("sample"), **s)

    def clear(self):
        for n, t in self.out.items():
            # (indices that are read before they are written anew stay within the vocabulary)
            a = np.full(t.size() * t.dtype.size, 0 if n == "i" else 0xA5, np.uint8)
            assert self.hpt.lib().hpt_hip_memcpy_h2d_sync(0, P(t.ptr), a.ctypes.data_as(P), a.nbytes) == 0

    def bits(self):
        return {n: t.numpy().tobytes() for n, t in self.out.items()}


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_captured_and_replayed(hpt, dev, hip, stream, name):  # noqa: F811
    """Every operator in one graph, replayed on new inputs with eager work and synchronisation in between; a second graph of the same
    calls with its own results and workspaces lives beside it."""
    import ctypes as C
    graphs = []
    for c in (Calls(hpt, name), Calls(hpt, name, seed=1)):
        c.run(stream)
        assert hip.hipStreamSynchronize(stream) == 0
        assert hip.hipStreamBeginCapture(stream, 0) == 0
        try:
            c.run(stream)
        finally:
            g = P()
            rc = hip.hipStreamEndCapture(stream, C.byref(g))
        assert rc == 0 and g.value
        e = P()
        assert hip.hipGraphInstantiate(C.byref(e), g, None, None, 0) == 0
        graphs.append((c, g, e))
    try:
        for seed in range(5, 9):
            for c, _, e in graphs:
                c.write(seed)
                c.clear()
                hpt.synchronize(dev)
                assert hip.hipGraphLaunch(e, stream) == 0
                assert hip.hipStreamSynchronize(stream) == 0
                got = c.bits()
                c.clear()
                c.run()  # eagerly, on the default stream
                hpt.synchronize(dev)
                want = c.bits()
                assert want == got, (seed, [n for n in want if want[n] != got[n]])
    finally:
        for _, g, e in graphs:
            hip.hipGraphExecDestroy(e)
            hip.hipGraphDestroy(g)


def test_without_a_workspace_a_capture_is_refused(hpt, dev, hip, stream):  # noqa: F811
    import ctypes as C
    c = Calls(hpt, "f32")
    x, o = c.dev["x"], c.out
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    try:
        with pytest.raises(hpt.MemoryError_, match="workspace"):
            x.topk(50, stream=stream, values_out=o["v"], index_out=o["i"])
        with pytest.raises(hpt.MemoryError_, match="workspace"):
            x.sample(c.u, stream=stream, token_out=o["token0"], logp_out=o["logp0"])
        with pytest.raises(hpt.MemoryError_, match="workspace"):
            x.distill_loss(o["v"], o["i"], stream=stream, loss_out=o["loss"], kl_out=o["kl"], terms_out=o["terms"])
        small = hpt.Tensor.from_raw(c.ws["sample"].ptr, [16], hpt.u8)
        with pytest.raises(hpt.MemoryError_, match="holds 16 bytes"):
            x.sample(c.u, stream=stream, token_out=o["token0"], logp_out=o["logp0"], workspace=small)
        with pytest.raises(hpt.ParamError, match="aligned to 16"):
            x.sample(c.u, stream=stream, token_out=o["token0"], logp_out=o["logp0"],
                     workspace=hpt.Tensor.from_raw(c.ws["sample"].ptr + 8, [hpt.sample_workspace(x)], hpt.u8))
    finally:
        g = P()
        assert hip.hipStreamEndCapture(stream, C.byref(g)) == 0
    if g.value:
        hip.hipGraphDestroy(g)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_streams_scratch_and_ctypes_give_the_same_bits(hpt, dev, hip, stream, name):  # noqa: F811
    c = Calls(hpt, name)
    c.run()
    hpt.synchronize(dev)
    want = c.bits()
    for what, call in (("again", c.run), ("the library's scratch", lambda: c.run(ws=False)), ("a stream of the caller", lambda: c.run(int(stream.value))),
                       ("that stream, the library's scratch", lambda: c.run(int(stream.value), ws=False)), ("through ctypes", lambda: c.run(P(0))),
                       ("through ctypes, the stream and scratch", lambda: c.run(stream, ws=False))):
        c.clear()
        hpt.synchronize(dev)
        call()
        assert hip.hipStreamSynchronize(stream) == 0
        hpt.synchronize(dev)
        got = c.bits()
        assert got == want, (what, [n for n in want if want[n] != got[n]])


def test_threads(hpt, dev, hip):  # noqa: F811
    """Calls from several threads at once, on streams of their own and on the default one, with the library's scratch."""
    import ctypes as C
    made, errors = [], []
    for _ in range(3):
        s = P()
        assert hip.hipStreamCreateWithFlags(C.byref(s), 1) == 0
        made.append(s)
    calls = [Calls(hpt, "bf16", seed=i) for i in range(5)]
    want = []
    for c in calls:
        c.run()
        hpt.synchronize(dev)
        want.append(c.bits())
        c.clear()
    hpt.synchronize(dev)

    def work(i):
        try:
            s = int(made[i].value) if i < 3 else None
            for _ in range(8):
                calls[i].run(s, ws=False)
                hpt.synchronize(dev, P(s) if s else None)
                assert calls[i].bits() == want[i]
        except Exception as e:  # noqa: BLE001 - reported below
            errors.append((i, e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(5)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for s in made:
        hip.hipStreamDestroy(s)
    assert not errors, errors


def test_the_cpp_host_side():
    """The prebuilt program hpt_amd/lib/vocab_api_test (source tests/cpp/vocab_api_test.cpp)."""
    import subprocess

    from hpt_amd import build
    assert build.VOCAB_TEST_BIN.exists(), f"{build.VOCAB_TEST_BIN} is missing: run `python -m hpt_amd.build`"
    r = subprocess.run([str(build.VOCAB_TEST_BIN)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and " 0 failures" in r.stdout, f"{r.stdout}\n{r.stderr}"


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_a_teacher_a_student_and_a_server(hpt, dev, name):
    """A teacher hands on its top logits, a student takes a step along the gradient, and answers are sampled from it and scored; against the same in 64 bits.
    The student's stored logits are the same on both sides of each comparison, so only each operator's own roundings count (as in its own tests)."""
    k, rng = Kind(hpt, name), np.random.default_rng(9)
    rows, cols, tau = 7, 6007, 2.0
    teacher, t = k.up(rng.standard_normal((rows, cols)) * 3)
    student, x = k.up(rng.standard_normal((rows, cols)) * 2)
    value, index, lse = teacher.topk(40, lse=True, temperature=tau)
    at = order(t)[:, :40]
    assert np.array_equal(index.numpy(), at)
    near(lse.numpy(), logsumexp(t / tau), 128 * F32_STEP + F32_STEP * 16)
    mask = np.array([1, 1, 0, 1, 1, 1, 0], np.float32)
    before = student.distill_loss(value, index, teacher_lse=lse, mask=up(hpt, mask), temperature=tau)
    kl, grad = distilled(x, np.take_along_axis(t, at, -1), at, tau, lse.numpy().astype(np.float64))
    near(before.loss.numpy()[0], tau * tau * (kl * mask).sum() / 5, tau * tau * 400 * F32_STEP + 4 * F32_STEP * tau * tau * kl.max())
    step = student.distill_loss_backward(value, index, before.terms, temperature=tau, grad=-20.0)
    moved, y = k.up(x + k.down(step))
    after = moved.distill_loss(value, index, teacher_lse=lse, mask=up(hpt, mask), temperature=tau)
    near(after.kl.numpy(), np.where(mask, distilled(y, np.take_along_axis(t, at, -1), at, tau, lse.numpy().astype(np.float64))[0], 0), 400 * F32_STEP + F32_STEP * 40)
    u = rng.uniform(size=rows).astype(np.float32)
    token, logp = moved.sample(up(hpt, u))
    want = [sampled(y[r], u[r]) for r in range(rows)]
    assert all(w[2] > 2.0 ** -36 for w in want) and np.array_equal(token.numpy(), [w[0] for w in want])
    # without filters it is the model's own log-probability, which a policy's loss takes as the old one
    scored, _ = moved.token_logp(token)
    near(scored.numpy(), logp.numpy(), 128 * F32_STEP + F32_STEP * 2 * 20)
    greedy = moved.sample(up(hpt, u), temperature=0.0)[0]
    assert np.array_equal(greedy.numpy(), moved.argmax(-1).numpy())
    assert np.array_equal(greedy.numpy(), moved.topk(1)[1].numpy()[:, 0])

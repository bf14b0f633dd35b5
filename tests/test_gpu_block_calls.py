"""How the operators around a transformer's blocks are called: captured into graphs and replayed, on streams of the caller, from several
threads, through ctypes, over tensors of more than 2^31 elements, and all of them together as a training step and as a step of
decoding use them."""
import ctypes as C
import threading

import numpy as np
import pytest

from block_util import F32_STEP, Kind, near, up

pytestmark = pytest.mark.gpu
P = C.c_void_p


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


@pytest.fixture()
def stream(hip):
    s = P()
    assert hip.hipStreamCreateWithFlags(C.byref(s), 1) == 0
    yield s
    hip.hipStreamDestroy(s)


class Calls:
    """One call of every operator into results of its own, on inputs that can be written anew. `kind`: a dtype."""

    def __init__(self, hpt, name, rows=200, cols=328, vocabulary=5003, seed=0):
        self.hpt, self.k, rng = hpt, Kind(hpt, name), np.random.default_rng(seed)
        k, e = self.k, hpt.Tensor.empty
        self.host = {"x": rng.standard_normal((rows, cols)), "r": rng.standard_normal((rows, cols)), "g": rng.normal(1, 0.2, cols),
                     "s": rng.standard_normal((2, 3, 40, 104)) * 4, "t": rng.standard_normal((16, 3)), "v": rng.standard_normal((rows // 4, vocabulary)) * 3,
                     "long": rng.standard_normal((2, 1, 70001)) * 3, "tl": rng.standard_normal((16, 2))}
        self.dev = {n: k.up(a)[0] for n, a in self.host.items()}
        n = rows // 4
        self.token = up(hpt, rng.integers(0, vocabulary, n))
        self.old, self.adv = (up(hpt, a.astype(np.float32)) for a in (rng.normal(-9, 0.1, n), rng.standard_normal(n)))
        self.lengths = up(hpt, np.array([104, 60]))
        like = lambda t, d=None: e(t.shape, d or t.dtype)  # noqa: E731
        d = self.dev
        self.out = {"norm": like(d["x"]), "add": like(d["x"]), "sum": like(d["x"]), "q": like(d["x"], hpt.u8), "scale": e([rows], hpt.f32), "gx": like(d["x"]),
                    "gg": e([cols], hpt.f32), "p": like(d["s"]), "gs": like(d["s"]), "gt": e([16, 3], hpt.f32), "pl": like(d["long"]), "loss": e([1], hpt.f32),
                    "logp": e([n], hpt.f32), "lse": e([n], hpt.f32), "weight": e([n], hpt.f32), "gv": like(d["v"]), "tlogp": e([n], hpt.f32), "tlse": e([n], hpt.f32)}
        need = {"norm": hpt.rms_norm_backward_workspace(d["x"], 1), "bias": hpt.softmax_bias_backward_workspace(d["s"], 16),
                "long": hpt.softmax_bias_workspace(d["long"]), "policy": hpt.policy_loss_workspace(d["v"])}
        assert all(need.values()), "every one of these needs some"
        self.ws = {n: e([b], hpt.u8) for n, b in need.items()}

    def write(self, seed):
        """New inputs in the same memory."""
        rng = np.random.default_rng(seed)
        l = self.hpt.lib()
        for n in ("x", "r", "s", "v", "long"):
            a = self.k.store(self.host[n] * rng.uniform(0.5, 1.5, self.host[n].shape))
            assert l.hpt_hip_memcpy_h2d_sync(0, P(self.dev[n].ptr), a.ctypes.data_as(P), a.nbytes) == 0

    def run(self, stream=None, ws=True):
        d, o, w = self.dev, self.out, self.ws if ws else {}
        c = [d["x"].shape[1]]
        d["x"].rms_norm(c, d["g"], stream=stream, out=o["norm"])
        d["x"].add_rms_norm(d["r"], c, d["g"], stream=stream, out=o["add"], sum_out=o["sum"])
        d["x"].rms_norm_quant(c, d["g"], format="e4m3", stream=stream, out=o["q"], scale_out=o["scale"])
        o["sum"].rms_norm_backward(d["r"], c, d["g"], grad_sum=o["norm"], stream=stream, out=o["gx"], gamma_out=o["gg"], workspace=w.get("norm"))
        kw = dict(max_distance=40, query_offset=64, causal=True, lengths=self.lengths, stream=stream)
        d["s"].softmax_bias(d["t"], 0.5, out=o["p"], **kw)
        o["p"].softmax_bias_backward(d["s"], 16, 0.5, out=o["gs"], table_out=o["gt"], workspace=w.get("bias"), **kw)
        d["long"].softmax_bias(d["tl"], 0.5, max_distance=40, query_offset=70000, stream=stream, out=o["pl"], workspace=w.get("long"))
        d["v"].policy_loss(self.token, self.old, self.adv, stream=stream, loss_out=o["loss"], logp_out=o["logp"], lse_out=o["lse"], weight_out=o["weight"],
                           workspace=w.get("policy"))
        d["v"].policy_loss_backward(self.token, o["lse"], o["weight"], 100.0, stream=stream, out=o["gv"])
        d["v"].token_logp(self.token, stream=stream, logp_out=o["tlogp"], lse_out=o["tlse"], workspace=w.get("policy"))

    def clear(self):
        for t in self.out.values():
            a = np.full(t.size() * t.dtype.size, 0xA5, np.uint8)
            assert self.hpt.lib().hpt_hip_memcpy_h2d_sync(0, P(t.ptr), a.ctypes.data_as(P), a.nbytes) == 0

    def bits(self):
        return {n: t.numpy().tobytes() for n, t in self.out.items()}


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_captured_and_replayed(hpt, dev, hip, stream, name):
    """Every operator in one graph, replayed on new inputs with eager work and synchronisation in between; a second graph of the same
    calls with its own results and workspaces lives beside it."""
    first, second = Calls(hpt, name), Calls(hpt, name, seed=1)
    graphs = []
    for c in (first, second):
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
                assert c.bits() == got, f"replay and eager call differ, input {seed}"
    finally:
        for _, g, e in graphs:
            hip.hipGraphExecDestroy(e)
            hip.hipGraphDestroy(g)


def test_without_a_workspace_a_capture_is_refused_or_goes_without(hpt, dev, hip, stream):
    c = Calls(hpt, "f32")
    c.run()
    hpt.synchronize(dev)
    want = c.bits()
    d, o = c.dev, c.out
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    try:
        with pytest.raises(hpt.MemoryError_, match="workspace"):
            o["sum"].rms_norm_backward(d["r"], [328], d["g"], stream=stream, out=o["gx"], gamma_out=o["gg"])
        with pytest.raises(hpt.MemoryError_, match="workspace"):
            o["p"].softmax_bias_backward(d["s"], 16, 0.5, max_distance=40, stream=stream, out=o["gs"], table_out=o["gt"])
        with pytest.raises(hpt.MemoryError_, match="workspace"):
            d["v"].policy_loss(c.token, c.old, c.adv, stream=stream, loss_out=o["loss"], logp_out=o["logp"], lse_out=o["lse"], weight_out=o["weight"])
        d["long"].softmax_bias(d["tl"], 0.5, max_distance=40, query_offset=70000, stream=stream, out=o["pl"])
        d["v"].token_logp(c.token, stream=stream, logp_out=o["tlogp"], lse_out=o["tlse"])
    finally:
        g = P()
        rc = hip.hipStreamEndCapture(stream, C.byref(g))
    assert rc == 0 and g.value
    e = P()
    assert hip.hipGraphInstantiate(C.byref(e), g, None, None, 0) == 0
    c.clear()
    for _ in range(3):
        assert hip.hipGraphLaunch(e, stream) == 0
        assert hip.hipStreamSynchronize(stream) == 0
        hpt.synchronize(dev)
        # another order of summing: the same numbers but for roundings
        for n, tol in (("pl", 64 * F32_STEP), ("tlogp", 128 * F32_STEP), ("tlse", 128 * F32_STEP)):
            w = np.frombuffer(want[n], np.float32).astype(np.float64)
            near(o[n].numpy().reshape(-1), w, tol * (np.abs(w) + (n != "pl")), n)
    hip.hipGraphExecDestroy(e)
    hip.hipGraphDestroy(g)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_streams_scratch_and_ctypes_give_the_same_bits(hpt, dev, hip, stream, name):
    c = Calls(hpt, name)
    c.run()
    hpt.synchronize(dev)
    want = c.bits()
    for what, call in (("the library's scratch", lambda: c.run(ws=False)), ("a stream of the caller", lambda: c.run(int(stream.value))),
                       ("that stream, the library's scratch", lambda: c.run(int(stream.value), ws=False)), ("through ctypes", lambda: c.run(P(0))),
                       ("through ctypes, the stream and scratch", lambda: c.run(stream, ws=False))):
        c.clear()
        hpt.synchronize(dev)
        call()
        assert hip.hipStreamSynchronize(stream) == 0
        hpt.synchronize(dev)
        assert c.bits() == want, what


def test_threads(hpt, dev, hip):
    """Calls from several threads at once, on streams of their own and on the default one, with the library's scratch."""
    made, errors = [], []
    for _ in range(4):
        s = P()
        assert hip.hipStreamCreateWithFlags(C.byref(s), 1) == 0
        made.append(s)
    calls = [Calls(hpt, "bf16", seed=i) for i in range(6)]
    want = []
    for c in calls:
        c.run()
        hpt.synchronize(dev)
        want.append(c.bits())
        c.clear()

    def work(i):
        try:
            s = int(made[i].value) if i < 4 else None
            for _ in range(10):
                calls[i].run(s, ws=False)
                hpt.synchronize(dev, P(s) if s else None)
                assert calls[i].bits() == want[i]
        except Exception as e:  # noqa: BLE001 - reported below
            errors.append((i, e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for s in made:
        hip.hipStreamDestroy(s)
    assert not errors, errors


def test_the_cpp_host_side():
    """The prebuilt program hpt_amd/lib/block_api_test (source tests/cpp/block_api_test.cpp)."""
    import subprocess

    from hpt_amd import build
    assert build.BLOCK_TEST_BIN.exists(), f"{build.BLOCK_TEST_BIN} is missing: run `python -m hpt_amd.build`"
    r = subprocess.run([str(build.BLOCK_TEST_BIN)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and " 0 failures" in r.stdout, f"{r.stdout}\n{r.stderr}"


# ---- more than 2^31 elements ---------------------------------------------------------------------------

def test_rows_beyond_two_to_the_31(hpt, dev):
    """The last rows of large tensors are what a small call makes of them."""
    k, rng = Kind(hpt, "bf16"), np.random.default_rng(1)
    rows, cols = 70000, 32768
    x, r = hpt.Tensor.zeros([rows, cols], hpt.bf16), hpt.Tensor.zeros([rows, cols], hpt.bf16)
    tail = lambda t: hpt.Tensor.from_raw(t.ptr + (t.size() - 3 * cols) * 2, [3, cols], hpt.bf16)  # noqa: E731
    a, _ = k.up(rng.standard_normal((3, cols)))
    b, _ = k.up(rng.standard_normal((3, cols)))
    for big, small in ((x, a), (r, b)):
        assert hpt.lib().hpt_hip_memcpy_d2d_sync(0, P(tail(big).ptr), P(small.ptr), 3 * cols * 2) == 0
    y, _ = x.add_rms_norm(r, [cols], sum_out=r)
    assert np.array_equal(tail(y).numpy(), a.add_rms_norm(b, [cols])[0].numpy())
    del y
    gx, gg = x.rms_norm_backward(r, [cols], out=r)
    added = hpt.Tensor.from_numpy(k.store(k.down(a).astype(np.float32) + k.down(b).astype(np.float32)), hpt.bf16).to_hip()
    w, wg = a.rms_norm_backward(added, [cols])
    assert np.array_equal(tail(gx).numpy(), w.numpy())
    near(gg.numpy(), wg.numpy(), 64 * F32_STEP * (np.abs(wg.numpy()) + 1))  # (all other rows are zeros)
    del gx, gg, r
    # the same memory as scores: one head of 70000 queries
    t, _ = k.up(rng.standard_normal((8, 1)))
    s = hpt.Tensor.from_raw(x.ptr, [1, rows, cols], hpt.bf16)
    p = s.softmax_bias(t, max_distance=16, query_offset=-rows + 100)
    small = hpt.Tensor.from_raw(a.ptr, [1, 3, cols], hpt.bf16).softmax_bias(t, max_distance=16, query_offset=97)
    assert np.array_equal(tail(p).numpy(), small.numpy()[0])
    del p
    # and as logits
    token = up(hpt, np.full(rows, 7))
    logp, lse = x.token_logp(token)
    wl, we = a.token_logp(up(hpt, np.full(3, 7)))
    near(logp.numpy()[-3:], wl.numpy(), 256 * F32_STEP * 12)
    w = hpt.Tensor.ones([rows], hpt.f32)
    g = x.policy_loss_backward(token, lse, w, out=x)
    e = hpt.Tensor.from_raw(lse.ptr + (rows - 3) * 4, [3], hpt.f32)
    assert np.array_equal(tail(g).numpy(), a.policy_loss_backward(up(hpt, np.full(3, 7)), e, hpt.Tensor.ones([3], hpt.f32)).numpy())


# ---- together ------------------------------------------------------------------------------------------

def test_a_training_step(hpt, dev):
    """One block and its loss, forward and backward, with the products on the host, against the derivative that torch takes of the whole
    in 64 bits. Each device result is off by 128 half steps of f32 of its terms at most; six of them follow each other and amplify what came
    before by no more than ten: 6 * 128 * 10 half steps of the largest entry."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(0)
    B, T, H, D, E, V, N = 2, 9, 3, 8, 24, 50, 16
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    h0, g1, g2 = f(B * T, E), (1 + 0.2 * f(E)).astype(np.float32), (1 + 0.2 * f(E)).astype(np.float32)
    wq, wk, wv, wo, wl = (0.2 * f(E, H * D) for _ in range(3)), None, None, None, None
    wq, wk, wv = wq
    wo, wl = 0.3 * f(H * D, E), 0.3 * f(E, V)
    table = f(N, H)
    lengths = np.array([T, 6])
    token = rng.integers(0, V, B * T)
    mask = (np.arange(T) < lengths[:, None]).astype(np.float32).reshape(-1)
    adv, scale = f(B * T), np.float32(D ** -0.5)

    def heads(a):
        return a.reshape(B, T, H, D).transpose(0, 2, 1, 3)

    def rows(a):
        return a.transpose(0, 2, 1, 3).reshape(B * T, H * D)

    # the oracle
    t = {n: torch.tensor(a.astype(np.float64), requires_grad=True) for n, a in dict(h0=h0, g1=g1, g2=g2, table=table, wq=wq).items()}
    c = {n: torch.tensor(a.astype(np.float64)) for n, a in dict(wk=wk, wv=wv, wo=wo, wl=wl).items()}
    rms = lambda x, g: x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * g  # noqa: E731
    y1 = rms(t["h0"], t["g1"])
    split = lambda a: a.reshape(B, T, H, D).transpose(1, 2)  # noqa: E731
    q, kk, v = split(y1 @ t["wq"]), split(y1 @ c["wk"]), split(y1 @ c["wv"])
    half = N // 4
    rel = np.arange(T)[None] - np.arange(T)[:, None]
    n = N // 2
    d = np.abs(rel)
    which = (rel > 0) * n + np.where(d < half, d, np.minimum(n - 1, half + np.floor(np.log(np.maximum(d, 1) / half) / np.log(7 / half) * (n - half) + 1e-9)).astype(int))
    s = scale.astype(np.float64) * (q @ kk.transpose(-1, -2)) + t["table"][torch.tensor(which)].permute(2, 0, 1)
    live = torch.tensor((np.arange(T)[None, :] <= np.arange(T)[:, None])[None, None] & (np.arange(T) < lengths[:, None])[:, None, None])
    p = torch.softmax(s.masked_fill(~live, -np.inf), -1)
    a = (p @ v).transpose(1, 2).reshape(B * T, H * D) @ c["wo"]
    h1 = a + t["h0"]
    logits = rms(h1, t["g2"]) @ c["wl"]
    logp = torch.log_softmax(logits, -1)[torch.arange(B * T), torch.tensor(token)]
    old = (logp.detach() + 0.1 * torch.tensor(f(B * T).astype(np.float64))).float().double()
    ref = (logp.detach() + 0.2 * torch.tensor(f(B * T).astype(np.float64))).float().double()
    ratio = torch.exp(logp - old)
    ad, m = torch.tensor(adv.astype(np.float64)), torch.tensor(mask.astype(np.float64))
    k = ref - logp
    each = -torch.minimum(ratio * ad, ratio.clamp(0.8, 1.2) * ad) + 0.1 * (torch.exp(k) - k - 1)
    loss = (each * m).sum() / m.sum()
    want = dict(zip(t, torch.autograd.grad(loss, list(t.values()))))

    # the device
    x, G1, G2, TB = (up(hpt, z) for z in (h0, g1, g2, table))
    L = up(hpt, lengths)
    bias = dict(max_distance=7, causal=True, lengths=L)
    Y1 = x.rms_norm([E], G1)
    y = Y1.numpy()
    Q, K, Vv = heads(y @ wq), heads(y @ wk), heads(y @ wv)
    probs = up(hpt, Q @ K.transpose(0, 1, 3, 2)).softmax_bias(TB, scale, **bias)
    att = rows(probs.numpy() @ Vv)
    Y2, H1 = up(hpt, att @ wo).add_rms_norm(x, [E], G2)
    lg = up(hpt, Y2.numpy() @ wl)
    tok = up(hpt, token)
    got = lg.policy_loss(tok, up(hpt, old.float().numpy()), up(hpt, adv), reference=up(hpt, ref.float().numpy()), mask=up(hpt, mask), kl_weight=0.1)
    assert abs(got.loss.numpy()[0] - loss.item()) < 6 * 128 * 10 * F32_STEP
    dlg = lg.policy_loss_backward(tok, got.lse, got.weight).numpy()
    dh1, dg2 = H1.rms_norm_backward(up(hpt, dlg @ wl.T), [E], G2)
    datt = heads(dh1.numpy() @ wo.T)
    dprobs = up(hpt, datt @ Vv.transpose(0, 1, 3, 2))
    ds, dtable = probs.softmax_bias_backward(dprobs, N, scale, **bias)
    dS = ds.numpy()
    dq, dk, dv = rows(dS @ K), rows(dS.transpose(0, 1, 3, 2) @ Q), rows(probs.numpy().transpose(0, 1, 3, 2) @ datt)
    dy1 = dq @ wq.T + dk @ wk.T + dv @ wv.T
    dh0, dg1 = x.rms_norm_backward(up(hpt, dy1), [E], G1, grad_sum=dh1)
    for n, g in dict(h0=dh0.numpy(), g1=dg1.numpy(), g2=dg2.numpy(), table=dtable.numpy(), wq=y.T @ dq).items():
        w = want[n].numpy()
        near(g, w, 6 * 128 * 10 * F32_STEP * np.abs(w).max(), n)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_a_step_of_decoding(hpt, dev, name):
    """The last query alone, against the whole prompt: the same norm, the same 8-bit values, the same probabilities, the same log-probability,
    but for the order of sums."""
    k, rng = Kind(hpt, name), np.random.default_rng(5)
    T, E, H, V = 200, 512, 4, 3001
    x, _ = k.up(rng.standard_normal((T, E)))
    r, _ = k.up(rng.standard_normal((T, E)))
    g, _ = k.up(rng.normal(1, 0.2, E))
    y, h = x.add_rms_norm(r, [E], g)
    y1, h1 = x[T - 1:T].add_rms_norm(hpt.Tensor.from_raw(r.ptr + (T - 1) * E * k.dtype.size, [1, E], k.dtype), [E], g)
    assert np.array_equal(h.numpy()[-1:], h1.numpy())
    a, b = k.down(y)[-1:], k.down(y1)
    near(b, a, 2 * k.step * np.abs(a) + 64 * F32_STEP * np.abs(a))
    q, s = h.rms_norm_quant([E], g, format="i8")
    q1, s1 = h1.rms_norm_quant([E], g, format="i8")
    near(s1.numpy(), s.numpy()[-1:], 64 * F32_STEP * s.numpy()[-1:])
    assert np.abs(q.numpy()[-1:].astype(int) - q1.numpy()).max() <= 1
    table, _ = k.up(rng.standard_normal((32, H)))
    sc, _ = k.up(rng.standard_normal((1, H, T, T)) * 8)
    p = k.down(sc.softmax_bias(table, 0.3, bidirectional=False, causal=True))[0, :, -1]
    one = k.down(sc[:, :, T - 1:T].softmax_bias(table, 0.3, bidirectional=False, causal=True, query_offset=T - 1))[0, :, 0]
    near(one, p, 2 * (k.step + 64 * F32_STEP) * p + k.least)
    lg, _ = k.up(rng.standard_normal((T, V)) * 3)
    tok = rng.integers(0, V, T)
    whole, single = lg.token_logp(up(hpt, tok))[0].numpy(), lg[T - 1:T].token_logp(up(hpt, tok[-1:]))[0].numpy()
    near(single, whole[-1:], 128 * F32_STEP * (1 + np.abs(whole[-1:])))

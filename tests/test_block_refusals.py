"""What the operators around a transformer's blocks refuse, before anything touches a device: dtypes, shapes, strides, overlaps,
parameters, workspaces. No GPU: the tensors only carry addresses."""
import ctypes as C

import numpy as np
import pytest


@pytest.fixture
def at(hpt):
    """Tensors at addresses of their own, never read."""
    place = [1 << 40]

    def make(shape, dtype=None, strides=None, ptr=None, device=0):
        if ptr is None:
            ptr = place[0]
            place[0] += 1 << 32
        return hpt.Tensor.from_raw(ptr, list(shape), dtype or hpt.f32, device, strides)
    return make


def refused(hpt, error, match, call):
    with pytest.raises(getattr(hpt, error), match=match):
        call()


# ---- RMS norm ------------------------------------------------------------------------------------

def norm(at, hpt, x=None, dims=(8,), gamma=None, eps=1e-6, out=None):
    x = x if x is not None else at([4, 8])
    return lambda: x.rms_norm(list(dims), gamma, eps, out=out if out is not None else at(x.shape, x.dtype))


def test_rms_norm_dtypes_and_shapes(hpt, at):
    refused(hpt, "DTypeError", "expected f16, bf16 or f32", norm(at, hpt, at([4, 8], hpt.f64)))
    refused(hpt, "DTypeError", "expected f16, bf16 or f32", norm(at, hpt, at([4, 8], hpt.i32)))
    refused(hpt, "ShapeError", "normalized dims must match", norm(at, hpt, dims=(9,)))
    refused(hpt, "ShapeError", "normalized dims must match", norm(at, hpt, dims=()))
    refused(hpt, "ShapeError", "neighbours in memory", norm(at, hpt, at([4, 8], strides=[1, 4])))
    refused(hpt, "ShapeError", "neighbours in memory", norm(at, hpt, at([4, 8], strides=[16, 2])))
    refused(hpt, "ShapeError", "Size mismatch", norm(at, hpt, gamma=at([7])))
    refused(hpt, "DTypeError", "gamma", norm(at, hpt, gamma=at([8], hpt.f16)))
    refused(hpt, "ShapeError", "must be contiguous", norm(at, hpt, gamma=at([8], strides=[2])))
    refused(hpt, "ShapeError", "Size mismatch", norm(at, hpt, out=at([4, 9])))
    refused(hpt, "DTypeError", "output", norm(at, hpt, out=at([4, 8], hpt.bf16)))
    refused(hpt, "ShapeError", "must be contiguous", norm(at, hpt, out=at([4, 8], strides=[9, 1])))
    refused(hpt, "ShapeError", "rows of", norm(at, hpt, at([1, 1 << 29]), dims=(1 << 29,)))
    # nine dims of rows that cannot be walked as fewer
    shape = [2] * 9 + [4]
    refused(hpt, "ShapeError", "separate dims", norm(at, hpt, at(shape, strides=[5 * 3 ** i for i in range(8, -1, -1)] + [1]), dims=(4,)))


@pytest.mark.parametrize("eps", [0.0, -1e-6, float("nan"), float("inf"), 1e-60])
def test_rms_norm_eps(hpt, at, eps):
    refused(hpt, "ParamError", "eps", norm(at, hpt, eps=eps))
    x = at([4, 8])
    refused(hpt, "ParamError", "eps", lambda: x.rms_norm_backward(at([4, 8]), [8], None, eps, out=at([4, 8]), gamma_out=at([8])))


def test_rms_norm_residual(hpt, at):
    x, out, total = at([4, 8]), at([4, 8]), at([4, 8])
    refused(hpt, "ShapeError", "shape differs", lambda: x.add_rms_norm(at([8, 4]), [8], out=out, sum_out=total))
    refused(hpt, "DTypeError", "residual", lambda: x.add_rms_norm(at([4, 8], hpt.f16), [8], out=out, sum_out=total))
    refused(hpt, "ShapeError", "must be contiguous", lambda: x.add_rms_norm(at([4, 8], strides=[16, 1]), [8], out=out, sum_out=total))
    refused(hpt, "ParamError", "no residual", lambda: x.rms_norm_quant([8], out=at([4, 8], hpt.i8), scale_out=at([4]), sum_out=total))


def test_rms_norm_overlaps(hpt, at):
    x, res = at([4, 8]), at([4, 8])
    over = at([4, 8], ptr=x.ptr + 32)
    refused(hpt, "ParamError", "overlaps the input", lambda: x.rms_norm([8], out=over))
    refused(hpt, "ParamError", "overlaps gamma", lambda: x.rms_norm([8], at([8], ptr=res.ptr), out=res))
    refused(hpt, "ParamError", "overlaps another result", lambda: x.add_rms_norm(res, [8], out=x, sum_out=x))
    refused(hpt, "ParamError", "overlaps the residual", lambda: x.add_rms_norm(res, [8], out=at([4, 8], ptr=res.ptr + 4), sum_out=at([4, 8])))
    # a strided view of the buffer that the result takes
    view = at([4, 8], strides=[16, 1], ptr=x.ptr)
    refused(hpt, "ParamError", "overlaps the input", lambda: view.rms_norm([8], out=x))
    refused(hpt, "ParamError", "overlaps the input", lambda: x.rms_norm_quant([8], out=at([4, 8], hpt.i8, ptr=x.ptr), scale_out=at([4])))
    refused(hpt, "ParamError", "overlaps another result", lambda: x.rms_norm_quant([8], out=at([4, 8], hpt.i8, ptr=res.ptr), scale_out=at([4], ptr=res.ptr + 16)))


def test_rms_norm_quant(hpt, at):
    x = at([4, 8], hpt.bf16)
    q, s = at([4, 8], hpt.i8), at([4])
    refused(hpt, "ParamError", "unknown format", lambda: x.rms_norm_quant([8], format="e5m2", out=q, scale_out=s))
    refused(hpt, "ShapeError", "do not divide", lambda: x.rms_norm_quant([8], group=3, out=q, scale_out=s))
    refused(hpt, "ShapeError", "do not divide", lambda: x.rms_norm_quant([8], group=-1, out=q, scale_out=s))
    refused(hpt, "ShapeError", "do not divide", lambda: x.rms_norm_quant([8], group=16, out=q, scale_out=s))
    refused(hpt, "ShapeError", "Size mismatch", lambda: x.rms_norm_quant([8], group=4, out=q, scale_out=s))
    refused(hpt, "DTypeError", "expected u8", lambda: x.rms_norm_quant([8], format="e4m3", out=q, scale_out=s))
    refused(hpt, "DTypeError", "scale", lambda: x.rms_norm_quant([8], out=q, scale_out=at([4], hpt.bf16)))


def test_rms_norm_backward(hpt, at):
    x, g, out, gg = at([40, 8]), at([40, 8]), at([40, 8]), at([8])
    call = lambda **k: x.rms_norm_backward(**{"grad": g, "normalized_shape": [8], "out": out, "gamma_out": gg, **k})  # noqa: E731
    refused(hpt, "ShapeError", "shape differs", lambda: call(grad=at([8, 40])))
    refused(hpt, "DTypeError", "grad_sum", lambda: call(grad_sum=at([40, 8], hpt.f16)))
    refused(hpt, "DTypeError", "grad_gamma", lambda: call(gamma_out=at([8], hpt.f16)))
    refused(hpt, "ShapeError", "Size mismatch", lambda: call(gamma_out=at([9])))
    refused(hpt, "ParamError", "overlaps grad", lambda: call(gamma_out=at([8], ptr=g.ptr)))
    refused(hpt, "ParamError", "overlaps the input", lambda: call(out=at([40, 8], ptr=x.ptr + 4)))
    need = hpt.rms_norm_backward_workspace(x, 1)
    assert need > 0 and need % 4 == 0
    refused(hpt, "ParamError", "overlaps another result", lambda: call(workspace=at([need], hpt.u8, ptr=out.ptr)))


# ---- softmax with a position bias ------------------------------------------------------------------

def bias_of(hpt, at, shape=(2, 3, 4, 5), table=(8, 3), x=None, **k):
    x = x if x is not None else at(shape)
    kw = {"table": at(table, x.dtype) if isinstance(table, tuple) else table, "out": at(x.shape, x.dtype), **k}
    return lambda: x.softmax_bias(**kw)


def test_bias_shapes_and_parameters(hpt, at):
    refused(hpt, "ShapeError", "at least 3 dims", bias_of(hpt, at, (4, 5)))
    refused(hpt, "DTypeError", "expected f16, bf16 or f32", bias_of(hpt, at, x=at([2, 3, 4, 5], hpt.f64)))
    refused(hpt, "ShapeError", "buckets x 3 heads", bias_of(hpt, at, table=(8, 4)))
    refused(hpt, "ShapeError", "buckets x 3 heads", bias_of(hpt, at, table=(24,)))
    refused(hpt, "DTypeError", "table", bias_of(hpt, at, table=at([8, 3], hpt.f16)))
    refused(hpt, "ParamError", "odd number", bias_of(hpt, at, table=(9, 3)))
    refused(hpt, "ParamError", "buckets", bias_of(hpt, at, table=(1, 3), bidirectional=False))
    refused(hpt, "ParamError", "two buckets", bias_of(hpt, at, table=(2, 3)))
    refused(hpt, "ParamError", "buckets", bias_of(hpt, at, table=(258, 3)))
    refused(hpt, "ParamError", "max_distance 2", bias_of(hpt, at, max_distance=2))
    refused(hpt, "ParamError", "max_distance 4097", bias_of(hpt, at, max_distance=4097))
    refused(hpt, "ParamError", "scale", bias_of(hpt, at, scale=float("nan")))
    refused(hpt, "ParamError", "scale", bias_of(hpt, at, scale=1e300))
    refused(hpt, "ParamError", "query_offset", bias_of(hpt, at, query_offset=1 << 41))
    refused(hpt, "ShapeError", "neighbours in memory", bias_of(hpt, at, x=at([2, 3, 4, 5], strides=[60, 20, 1, 4])))
    refused(hpt, "DTypeError", "lengths", bias_of(hpt, at, lengths=at([2], hpt.f32)))
    refused(hpt, "ShapeError", "Size mismatch", bias_of(hpt, at, lengths=at([3], hpt.i64)))
    refused(hpt, "ShapeError", "Size mismatch", bias_of(hpt, at, out=at([2, 3, 4, 6])))


def test_bias_overlaps(hpt, at):
    x = at([2, 3, 4, 5])
    refused(hpt, "ParamError", "overlaps the input", bias_of(hpt, at, x=x, out=at([2, 3, 4, 5], ptr=x.ptr + 4)))
    out = at([2, 3, 4, 5])
    refused(hpt, "ParamError", "overlaps the table", bias_of(hpt, at, x=x, table=at([8, 3], ptr=out.ptr), out=out))
    refused(hpt, "ParamError", "overlaps the lengths", bias_of(hpt, at, x=x, lengths=at([2], hpt.i64, ptr=out.ptr), out=out))


def test_bias_backward(hpt, at):
    p = at([2, 3, 4, 5])
    call = lambda **k: p.softmax_bias_backward(**{"grad": at([2, 3, 4, 5]), "buckets": 8, "out": at([2, 3, 4, 5]), "table_out": at([8, 3]), **k})  # noqa: E731
    refused(hpt, "ShapeError", "shape differs", lambda: call(grad=at([2, 3, 5, 4])))
    refused(hpt, "DTypeError", "grad", lambda: call(grad=at([2, 3, 4, 5], hpt.f16)))
    refused(hpt, "ShapeError", "buckets x 3 heads", lambda: call(table_out=at([3, 8])))
    refused(hpt, "DTypeError", "grad_table", lambda: call(table_out=at([8, 3], hpt.f16)))
    refused(hpt, "ParamError", "odd number", lambda: call(buckets=9, table_out=at([9, 3])))
    q = at([2, 3, 4, 5], strides=[120, 40, 10, 1])
    refused(hpt, "ShapeError", "must be contiguous", lambda: q.softmax_bias_backward(at([2, 3, 4, 5]), 8, out=at([2, 3, 4, 5]), table_out=at([8, 3])))
    assert hpt.softmax_bias_backward_workspace(p, 8) > 0
    refused(hpt, "ParamError", "buckets", lambda: hpt.softmax_bias_backward_workspace(p, 300))


# ---- policy loss -----------------------------------------------------------------------------------

def policy(hpt, at, x=None, **k):
    x = x if x is not None else at([6, 50])
    rows = [6]
    kw = {"token": at(rows, hpt.i64), "old_logp": at(rows), "advantage": at(rows), "loss_out": at([1]), "logp_out": at(rows), "lse_out": at(rows),
          "weight_out": at(rows), **k}
    return lambda: x.policy_loss(**kw)


def test_policy_refusals(hpt, at):
    refused(hpt, "DTypeError", "expected f16, bf16 or f32", policy(hpt, at, at([6, 50], hpt.f64)))
    refused(hpt, "ShapeError", "neighbours in memory", policy(hpt, at, at([6, 50], strides=[1, 6])))
    refused(hpt, "ShapeError", "no tokens", policy(hpt, at, at([6, 0])))
    refused(hpt, "DTypeError", "token", policy(hpt, at, token=at([6])))
    refused(hpt, "ShapeError", "Size mismatch", policy(hpt, at, token=at([5], hpt.i64)))
    refused(hpt, "DTypeError", "old_logp", policy(hpt, at, old_logp=at([6], hpt.f16)))
    refused(hpt, "ShapeError", "must be contiguous", policy(hpt, at, advantage=at([6], strides=[2])))
    refused(hpt, "DTypeError", "mask", policy(hpt, at, mask=at([6], hpt.i32)))
    refused(hpt, "ParamError", "clip_low", policy(hpt, at, clip_low=-0.1))
    refused(hpt, "ParamError", "clip_low", policy(hpt, at, clip_low=1.5))
    refused(hpt, "ParamError", "clip_low", policy(hpt, at, clip_high=float("nan")))
    refused(hpt, "ParamError", "kl_weight", policy(hpt, at, kl_weight=float("inf"), reference=at([6])))
    refused(hpt, "ParamError", "reference", policy(hpt, at, kl_weight=0.1))
    old = at([6])
    refused(hpt, "ParamError", "overlaps old_logp", policy(hpt, at, old_logp=old, logp_out=at([6], ptr=old.ptr)))
    lse = at([6])
    refused(hpt, "ParamError", "overlaps another result", policy(hpt, at, lse_out=lse, weight_out=at([6], ptr=lse.ptr + 4)))
    need = hpt.policy_loss_workspace(at([6, 50]))
    assert need > 0
    x = at([6, 50])
    back = lambda **k: x.policy_loss_backward(**{"token": at([6], hpt.i64), "lse": at([6]), "weight": at([6]), "out": at([6, 50]), **k})  # noqa: E731
    refused(hpt, "DTypeError", "weight", lambda: back(weight=at([6], hpt.f64)))
    refused(hpt, "ShapeError", "Size mismatch", lambda: back(out=at([6, 51])))
    refused(hpt, "ParamError", "overlaps the logits", lambda: back(out=at([6, 50], ptr=x.ptr + 4)))
    refused(hpt, "ShapeError", "Size mismatch", lambda: x.token_logp(at([7], hpt.i64), logp_out=at([6]), lse_out=at([6])))


# ---- all of them -----------------------------------------------------------------------------------

def test_operands_on_two_devices(hpt, at):
    x = at([4, 8])
    refused(hpt, "ParamError", "device 0 and on device 1", lambda: x.rms_norm([8], at([8], device=1), out=at([4, 8])))
    refused(hpt, "ParamError", "device 0 and on device 1", lambda: x.add_rms_norm(at([4, 8]), [8], out=at([4, 8]), sum_out=at([4, 8], device=1)))


def test_host_tensors(hpt, at):
    h = hpt.Tensor.from_numpy(np.zeros((4, 8), np.float32))
    with pytest.raises(NotImplementedError):
        h.rms_norm([8])
    with pytest.raises(NotImplementedError):
        at([4, 8]).rms_norm([8], hpt.Tensor.from_numpy(np.zeros(8, np.float32)), out=at([4, 8]))


def test_refusals_come_through_ctypes_too(hpt, at):
    # (a stream given as a ctypes pointer takes that way)
    x = at([4, 8])
    refused(hpt, "ShapeError", "Size mismatch", lambda: x.rms_norm([8], at([7]), out=at([4, 8]), stream=C.c_void_p(0)))
    refused(hpt, "ShapeError", "Size mismatch", lambda: x.token_logp(at([5], hpt.i64), logp_out=at([4]), lse_out=at([4]), stream=C.c_void_p(0)))


def test_null_arguments(hpt):
    l = hpt.lib()
    assert l.hpt_hip_rms_norm(0, None, None, None, 1, None, 1e-6, None, None) == 1
    assert l.hpt_hip_rms_norm_quant(0, None, None, None, 1, None, 1e-6, 1, 0, None, None, None) == 1
    assert l.hpt_hip_rms_norm_backward(0, None, None, None, None, 1, None, 1e-6, None, None, None) == 1
    assert l.hpt_hip_softmax_bias(0, None, None, 1.0, None, 0, 128, 0, 0, None, None, None) == 1
    assert l.hpt_hip_softmax_bias_backward(0, None, None, None, 1.0, 0, 128, 0, 0, None, None, None, None) == 1
    assert l.hpt_hip_token_logp(0, None, None, None, None, None, None) == 1
    assert l.hpt_hip_policy_loss(0, None, None, None, None, None, None, None, 0.2, 0.2, 0.0, None, None, None, None, None) == 1
    assert l.hpt_hip_policy_loss_backward(0, None, None, None, None, None, 1.0, None) == 1
    for name, args in (("rms_norm_backward", (None, 1)), ("softmax_bias", (None,)), ("softmax_bias_backward", (None, 8)), ("policy_loss", (None,))):
        n = C.c_size_t()
        assert getattr(l, f"hpt_hip_{name}_workspace")(*args, C.byref(n)) == 1
        assert getattr(l, f"hpt_hip_{name}_workspace")(*args, None) == 1


def test_nothing_to_do(hpt, at):
    """Empty tensors: no launch, so no device is needed."""
    x = at([0, 8])
    assert x.rms_norm([8], out=at([0, 8])).shape == [0, 8]
    e = at([2, 3, 0, 5])
    assert e.softmax_bias(at([8, 3]), out=at([2, 3, 0, 5])).shape == [2, 3, 0, 5]
    assert hpt.softmax_bias_workspace(e) == 0 and hpt.rms_norm_backward_workspace(x, 1) == 0

"""What top-k, sampling and distillation refuse, before anything touches a device. No GPU: the tensors only carry addresses."""
import ctypes as C

import numpy as np
import pytest

from test_block_refusals import at, refused  # noqa: F401


def topk(at, hpt, x=None, k=4, **kw):
    x = x if x is not None else at([6, 50])
    rows = int(np.prod(x.shape[:-1]))
    kw = {"values_out": at([rows, max(k, 0)], x.dtype), "index_out": at([rows, max(k, 0)], hpt.i64), "workspace": at([1 << 20], hpt.u8), **kw}
    return lambda: x.topk(k, **kw)


def test_topk(hpt, at):  # noqa: F811
    refused(hpt, "DTypeError", "expected f16, bf16 or f32", topk(at, hpt, at([6, 50], hpt.f64)))
    refused(hpt, "DTypeError", "expected f16, bf16 or f32", topk(at, hpt, at([6, 50], hpt.i32)))
    refused(hpt, "ShapeError", "neighbours in memory", topk(at, hpt, at([6, 50], strides=[1, 6])))
    refused(hpt, "ShapeError", "neighbours in memory", topk(at, hpt, at([6, 50], strides=[100, 2])))
    refused(hpt, "ShapeError", "no tokens", topk(at, hpt, at([6, 0])))
    refused(hpt, "ShapeError", "no dimensions", topk(at, hpt, at([])))
    refused(hpt, "ShapeError", "rows of", topk(at, hpt, at([1, 1 << 29])))
    for k in (0, -1, 51, 1025):
        refused(hpt, "ParamError", "expected 1 to 50", topk(at, hpt, k=k))
    refused(hpt, "ParamError", "expected 1 to 1024", topk(at, hpt, at([2, 5000]), k=1025))
    refused(hpt, "DTypeError", "values", topk(at, hpt, values_out=at([6, 4], hpt.f16)))
    refused(hpt, "ShapeError", "Size mismatch", topk(at, hpt, values_out=at([6, 5])))
    refused(hpt, "DTypeError", "index", topk(at, hpt, index_out=at([6, 4], hpt.u32)))
    refused(hpt, "ShapeError", "must be contiguous", topk(at, hpt, index_out=at([6, 4], hpt.i64, strides=[8, 1])))
    refused(hpt, "DTypeError", "lse", topk(at, hpt, lse_out=at([6], hpt.bf16)))
    refused(hpt, "ShapeError", "Size mismatch", topk(at, hpt, lse_out=at([5])))
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-31):
        refused(hpt, "ParamError", "temperature", topk(at, hpt, lse_out=at([6]), temperature=t))
    x = at([6, 50])
    refused(hpt, "ParamError", "overlaps the input", topk(at, hpt, x, values_out=at([6, 4], ptr=x.ptr)))
    v = at([6, 4])
    refused(hpt, "ParamError", "overlaps another result", topk(at, hpt, values_out=v, index_out=at([6, 4], hpt.i64, ptr=v.ptr)))
    refused(hpt, "ParamError", "overlaps another result", topk(at, hpt, values_out=v, workspace=at([1 << 20], hpt.u8, ptr=v.ptr)))
    need = hpt.topk_workspace(x, 4)
    refused(hpt, "ShapeError", "must be contiguous", topk(at, hpt, workspace=at([2, need], hpt.u8, strides=[need + 1, 1])))


def sample(at, hpt, x=None, **kw):
    x = x if x is not None else at([6, 50])
    rows = int(np.prod(x.shape[:-1]))
    kw = {"u": at([rows]), "token_out": at([rows], hpt.i64), "logp_out": at([rows]), **kw}
    return lambda: x.sample(**kw)


def test_sample(hpt, at):  # noqa: F811
    refused(hpt, "DTypeError", "expected f16, bf16 or f32", sample(at, hpt, at([6, 50], hpt.f64)))
    refused(hpt, "ShapeError", "neighbours in memory", sample(at, hpt, at([6, 50], strides=[1, 6])))
    refused(hpt, "ShapeError", "no tokens", sample(at, hpt, at([6, 0])))
    refused(hpt, "ShapeError", "vocabulary of 4194305 tokens", sample(at, hpt, at([1, (1 << 22) + 1])))
    refused(hpt, "DTypeError", "sample u", sample(at, hpt, u=at([6], hpt.f16)))
    refused(hpt, "ShapeError", "Size mismatch", sample(at, hpt, u=at([5])))
    for t in (-0.5, float("nan"), float("inf"), 1e-31):
        refused(hpt, "ParamError", "temperature", sample(at, hpt, temperature=t))
    refused(hpt, "ParamError", "top_p", sample(at, hpt, top_p=float("nan")))
    refused(hpt, "ParamError", "min_p", sample(at, hpt, min_p=float("nan")))
    for name in ("temperature", "top_p", "min_p"):
        refused(hpt, "DTypeError", name, sample(at, hpt, **{name: at([6], hpt.f64)}))
        refused(hpt, "ShapeError", "Size mismatch", sample(at, hpt, **{name: at([7])}))
        refused(hpt, "ShapeError", "must be contiguous", sample(at, hpt, **{name: at([6], strides=[2])}))
    refused(hpt, "DTypeError", "top_k", sample(at, hpt, top_k=at([6])))
    refused(hpt, "ShapeError", "Size mismatch", sample(at, hpt, top_k=at([7], hpt.i32)))
    refused(hpt, "DTypeError", "token", sample(at, hpt, token_out=at([6])))
    refused(hpt, "ShapeError", "Size mismatch", sample(at, hpt, token_out=at([5], hpt.i64)))
    refused(hpt, "DTypeError", "logp", sample(at, hpt, logp_out=at([6], hpt.i32)))
    t = at([6])
    refused(hpt, "ParamError", "overlaps the temperatures", sample(at, hpt, temperature=t, logp_out=at([6], ptr=t.ptr)))
    u = at([6])
    refused(hpt, "ParamError", "overlaps u", sample(at, hpt, u=u, logp_out=at([6], ptr=u.ptr)))
    refused(hpt, "ParamError", "device 0 and on device 1", sample(at, hpt, top_p=at([6], device=1)))


def distill(at, hpt, x=None, k=4, **kw):
    x = x if x is not None else at([6, 50])
    rows = int(np.prod(x.shape[:-1]))
    kw = {"teacher": at([rows, k]), "index": at([rows, k], hpt.i64), "loss_out": at([1]), "kl_out": at([rows]), "terms_out": at([rows, 8]), **kw}
    return lambda: x.distill_loss(**kw)


def test_distill(hpt, at):  # noqa: F811
    refused(hpt, "DTypeError", "expected f16, bf16 or f32", distill(at, hpt, at([6, 50], hpt.f64)))
    refused(hpt, "ShapeError", "neighbours in memory", distill(at, hpt, at([6, 50], strides=[1, 6])))
    refused(hpt, "ShapeError", "no tokens", distill(at, hpt, at([6, 0])))
    refused(hpt, "DTypeError", "teacher", distill(at, hpt, teacher=at([6, 4], hpt.i32)))
    refused(hpt, "ShapeError", "Size mismatch", distill(at, hpt, teacher=at([5, 4])))
    refused(hpt, "ShapeError", "must be contiguous", distill(at, hpt, teacher=at([6, 4], strides=[8, 1])))
    refused(hpt, "ShapeError", "1 to 1024", distill(at, hpt, k=1025))
    refused(hpt, "ShapeError", "1 to 1024", distill(at, hpt, k=0))
    refused(hpt, "DTypeError", "index", distill(at, hpt, index=at([6, 4])))
    refused(hpt, "ShapeError", "Size mismatch", distill(at, hpt, index=at([6, 5], hpt.i64)))
    refused(hpt, "ShapeError", "as many entries", distill(at, hpt, index=at([4, 6], hpt.i64)))
    refused(hpt, "DTypeError", "teacher_lse", distill(at, hpt, teacher_lse=at([6], hpt.bf16)))
    refused(hpt, "ShapeError", "Size mismatch", distill(at, hpt, teacher_lse=at([7])))
    refused(hpt, "DTypeError", "mask", distill(at, hpt, mask=at([6], hpt.i32)))
    refused(hpt, "ShapeError", "Size mismatch", distill(at, hpt, mask=at([7])))
    for t in (0.0, -1.0, float("nan"), float("inf")):
        refused(hpt, "ParamError", "temperature", distill(at, hpt, temperature=t))
    refused(hpt, "ShapeError", "Size mismatch", distill(at, hpt, terms_out=at([6, 7])))
    refused(hpt, "ShapeError", "Size mismatch", distill(at, hpt, loss_out=at([2])))
    kl = at([6])
    refused(hpt, "ParamError", "overlaps another result", distill(at, hpt, kl_out=kl, loss_out=at([1], ptr=kl.ptr)))
    x = at([6, 50])
    back = lambda **k: x.distill_loss_backward(**{"teacher": at([6, 4]), "index": at([6, 4], hpt.i32), "terms": at([6, 8]), "out": at([6, 50]), **k})  # noqa: E731
    refused(hpt, "ShapeError", "Size mismatch", lambda: back(terms=at([6, 4])))
    refused(hpt, "ParamError", "temperature", lambda: back(temperature=0.0))
    refused(hpt, "DTypeError", "grad_logits", lambda: back(out=at([6, 50], hpt.f16)))
    refused(hpt, "ParamError", "overlaps the logits", lambda: back(out=at([6, 50], ptr=x.ptr + 4)))
    terms = at([6, 8])
    refused(hpt, "ParamError", "overlaps the terms", lambda: back(terms=terms, out=at([6, 50], ptr=terms.ptr)))


def test_null_arguments(hpt):
    l = hpt.lib()
    assert l.hpt_hip_topk(0, None, None, 1, 1.0, None, None, None, None) == 1
    assert l.hpt_hip_sample(0, None, None, None, 1.0, None, 0, None, 1.0, None, 0.0, None, None, None, None) == 1
    assert l.hpt_hip_distill_loss(0, None, None, None, None, None, None, 1.0, None, None, None, None) == 1
    assert l.hpt_hip_distill_loss_backward(0, None, None, None, None, None, 1.0, 1.0, None) == 1
    n = C.c_size_t()
    for name, args in (("topk", (None, 1)), ("sample", (None,)), ("distill_loss", (None,))):
        assert getattr(l, f"hpt_hip_{name}_workspace")(*args, C.byref(n)) == 1
        assert getattr(l, f"hpt_hip_{name}_workspace")(*args, None) == 1


def test_results_that_are_missing(hpt, at):  # noqa: F811
    """A view for every result but one, through the C ABI."""
    l = hpt.lib()
    x, one, ints = at([6, 50]), at([6]), at([6], hpt.i64)
    v, o, i = x._c_view(), one._c_view(), ints._c_view()
    r = C.byref
    assert l.hpt_hip_topk(0, None, r(v[0]), 1, 1.0, None, None, r(i[0]), None) == 1
    assert l.hpt_hip_topk(0, None, r(v[0]), 1, 1.0, None, r(o[0]), None, None) == 1
    assert l.hpt_hip_sample(0, None, r(v[0]), r(o[0]), 1.0, None, 0, None, 1.0, None, 0.0, None, None, None, r(o[0])) == 1


def test_nothing_to_do(hpt, at):  # noqa: F811
    """No rows: no launch, so no device is needed."""
    x = at([0, 50])
    values, index = x.topk(4, values_out=at([0, 4]), index_out=at([0, 4], hpt.i64))
    assert values.shape == index.shape == [0, 4]
    token, logp = x.sample(at([0]), token_out=at([0], hpt.i64), logp_out=at([0]))
    assert token.shape == logp.shape == [0]
    assert hpt.topk_workspace(x, 4) == hpt.sample_workspace(x) == hpt.distill_loss_workspace(x) == 0


def test_workspaces_are_bounded(hpt, at):  # noqa: F811
    """Rows are taken in runs, so that a large batch needs no more scratch than a part of it."""
    most = 64 << 20
    for rows in (1, 64, 4096, 1 << 20):
        x = at([rows, 152000], hpt.bf16)
        assert 0 < hpt.topk_workspace(x, 64) <= most and 0 < hpt.sample_workspace(x) <= most
    assert hpt.sample_workspace(at([1 << 20, 7])) <= most

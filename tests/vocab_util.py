"""What top-k, sampling and distillation compute, from their definitions in 64 bits."""
import numpy as np


def order(x):
    """The indices of each row in order: NaN first, then the larger value, equal ones by index."""
    nan = np.isnan(x)
    v = np.where(nan, np.inf, x) + 0.0
    return np.lexsort((np.broadcast_to(np.arange(x.shape[-1]), x.shape), -v, ~nan), axis=-1)


def logsumexp(x, axis=-1):
    with np.errstate(invalid="ignore", divide="ignore"):
        m = x.max(axis, keepdims=True)
        m = np.where(np.isfinite(m), m, 0.0)
        return np.take(m + np.log(np.exp(x - m).sum(axis, keepdims=True)), 0, axis)


def sampled(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, logp, how far, as a part of the row's sum, the nearest border is from what decides) of one row."""
    cols = len(x)
    if not np.isfinite(x.max()):  # (NaN among them)
        return -1, np.nan, 1.0
    if temperature == 0:
        temperature, top_k = 1.0, 1
    at = order(x[None])[0]
    w = np.exp((x - x.max()) / temperature)
    k = top_k if 1 <= top_k < cols else cols
    kept, margin = at[:k], 1.0
    if top_p < 1:
        upto = w[kept].cumsum()
        reach = upto / upto[-1] - top_p
        margin = min(margin, np.abs(reach).min())
        kept = kept[:int((reach < 0).sum()) + 1]
    if min_p > 0:
        margin = min(margin, np.abs(w - min(min_p, 1.0))[w != 1].min(initial=1.0))
        kept = kept[w[kept] >= min(min_p, 1.0)]
    kept = np.sort(kept)
    upto = w[kept].cumsum()
    part = upto / upto[-1]
    u = min(max(float(u), 0.0), 1.0) if u == u else 0.0
    if 0 < u < 1:
        margin = min(margin, np.abs(part - u).min())
    where = int((part <= u).sum())
    if where == len(kept):
        where = int(np.flatnonzero(w[kept] > 0)[-1])
    return kept[where], np.log(w[kept[where]] / upto[-1]), margin


def distilled(x, t, index, tau=1.0, teacher_lse=None):
    """(kl, its gradient by x / tau) of each row; entries with a negative index are none."""
    rows, cols = x.shape
    kl, grad = np.zeros(rows), np.zeros(x.shape)
    z = x / tau
    for r in range(rows):
        named = index[r] >= 0
        i, e = index[r][named], t[r][named] / tau
        lse = logsumexp(z[r])
        logp = z[r] - lse
        p = np.exp(logp)
        if teacher_lse is None:
            if not len(i) or e.max() == -np.inf:
                continue
            logq = e - logsumexp(e)
            rest, out = 0.0, None
        else:
            logq = e - teacher_lse[r]
            rest = max(0.0, 1 - np.exp(logq).sum())
            out = np.ones(cols, bool)
            out[i] = False
            out &= p > 0
            rest = rest if out.any() else 0.0
        q = np.exp(logq)
        on = q > 0
        kl[r] = (q[on] * (logq[on] - logp[i[on]])).sum()
        mass = q.sum() + rest
        grad[r] = mass * p
        np.add.at(grad[r], i, -q)
        if rest:
            logs = logsumexp(logp[out])
            kl[r] += rest * (np.log(rest) - logs)
            grad[r][out] -= rest * np.exp(logp[out] - logs)
    return kl, grad

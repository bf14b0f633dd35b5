"""Operators over a vocabulary of logits: what a model answers with and what it learns from a teacher, case by case, for timing
and for comparing outputs.

  topk      the k largest logits of each row with their indices, largest first, equal ones by index; where asked for, the log of
            the sum of exponentials of the row over a temperature (what a teacher hands on)
  sample    one token for each row, from a given random number: softmax(logits / temperature), cut to the k likeliest tokens, then to
            the fewest of these that hold `top_p` of their probability, then to those with at least `min_p` of the likeliest
            one's; the number picks a token from what is left, in the order of the indices
  distill   the divergence of the student's distribution from a teacher's, of which the top logits are known, and the gradient
            of the student's logits; with the teacher's log of the sum, what it gives to all other tokens counts as one token

A case is a dict of plain values. `own` false: elementary torch operations in 32 bits (64 for long sums and next to the borders
that a token's choice depends on), rounded once at the end. `own` true: the calls of the framework, on the same device memory.
`exact` gives the same results from the definitions in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # The likeliest tokens shown beside an answer's next token: all latency.
        {"name": "topk_step_bf16", "kind": "topk", "dtype": "bf16", "rows": 1, "cols": 152000, "k": 20, "lse": True, "temperature": 1.0},
        # Candidates of a beam search, full precision, an odd vocabulary.
        {"name": "topk_beam_f32_odd", "kind": "topk", "dtype": "f32", "rows": 37, "cols": 50257, "k": 33, "lse": False, "temperature": 1.0},
        # A teacher's top logits over a micro-batch of positions.
        {"name": "topk_teacher_bf16", "kind": "topk", "dtype": "bf16", "rows": 4096, "cols": 50257, "k": 64, "lse": True, "temperature": 2.0},
        # Many candidates of a large vocabulary, to be scored again by something else.
        {"name": "topk_wide_f16", "kind": "topk", "dtype": "f16", "rows": 256, "cols": 152000, "k": 512, "lse": False, "temperature": 1.0},
        # A single conversation's next token with the usual three settings: all latency.
        {"name": "sample_step_bf16", "kind": "sample", "dtype": "bf16", "rows": 1, "cols": 152000, "temperature": 0.7, "top_k": 20,
         "top_p": 0.8, "min_p": 0.0, "each": False},
        # A serving batch, in which every request has settings of its own (greedy ones and unfiltered ones among them).
        {"name": "sample_serving_bf16", "kind": "sample", "dtype": "bf16", "rows": 64, "cols": 152000, "temperature": 0.8, "top_k": 50,
         "top_p": 0.9, "min_p": 0.05, "each": True},
        # A small batch in full precision, an odd vocabulary, cut by probability alone.
        {"name": "sample_nucleus_f32_odd", "kind": "sample", "dtype": "f32", "rows": 33, "cols": 50257, "temperature": 1.0, "top_k": 0,
         "top_p": 0.95, "min_p": 0.0, "each": False},
        # Answers to train on, sampled from the model's own distribution by thousands.
        {"name": "sample_rollout_bf16", "kind": "sample", "dtype": "bf16", "rows": 2048, "cols": 50257, "temperature": 1.0, "top_k": 0,
         "top_p": 1.0, "min_p": 0.0, "each": False},
        # A small student in full precision, odd sizes, rows for which the teacher has fewer entries.
        {"name": "distill_f32_odd", "kind": "distill", "dtype": "f32", "rows": 301, "cols": 32000, "k": 17, "rest": False,
         "temperature": 1.0, "ragged": True},
        # Half precision, a large vocabulary, more entries.
        {"name": "distill_f16", "kind": "distill", "dtype": "f16", "rows": 1000, "cols": 152000, "k": 128, "rest": False,
         "temperature": 1.5, "ragged": False},
        # A training step's micro-batch with the rest of the teacher's distribution as one token; the largest case.
        {"name": "distill_rest_bf16", "kind": "distill", "dtype": "bf16", "rows": 8192, "cols": 50257, "k": 64, "rest": True,
         "temperature": 2.0, "ragged": False},
    ]


# ---- drawn cases --------------------------------------------------------------------------------

_MOST = 1 << 26  # elements of a drawn case's logits


def _spread(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm; half of them rounded to what sizes mostly are."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        step = 64 if n >= 512 else 8 if n >= 32 else 1
        n = n // step * step
    return max(lo, min(hi, n))


def _dtype(rng):
    return rng.choice(["bf16", "bf16", "f16", "f32"])


def _draw_topk(rng):
    cols = _spread(rng, 16384, 152000)
    return {"kind": "topk", "dtype": _dtype(rng), "rows": _spread(rng, 1, _MOST // cols), "cols": cols, "k": _spread(rng, 1, 512),
            "lse": rng.random() < 0.5, "temperature": rng.choice([1.0, 1.0, 2.0])}


def _draw_sample(rng):
    cols = _spread(rng, 16384, 152000)
    return {"kind": "sample", "dtype": _dtype(rng), "rows": _spread(rng, 1, _MOST // cols), "cols": cols,
            "temperature": round(rng.uniform(0.5, 1.3), 2), "top_k": rng.choice([0, 0, _spread(rng, 1, 500)]),
            "top_p": rng.choice([1.0, round(rng.uniform(0.5, 0.99), 3)]), "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.2), 3)]),
            "each": rng.random() < 0.4}


def _draw_distill(rng):
    cols = _spread(rng, 16384, 152000)
    return {"kind": "distill", "dtype": _dtype(rng), "rows": _spread(rng, 1, _MOST // cols), "cols": cols, "k": _spread(rng, 8, 512),
            "rest": rng.random() < 0.5, "temperature": rng.choice([1.0, 1.5, 2.0, 4.0]), "ragged": rng.random() < 0.3}


def draw(rng):
    return rng.choice([_draw_topk, _draw_sample, _draw_distill])(rng)


# ---- inputs -------------------------------------------------------------------------------------


def _logits(gen, rows, cols):
    """Logits in 32 bits as a language model has them: a wide floor of tokens that do not fit, a few hundred that might, and in
    some rows one or a few that stand out."""
    x = torch.empty([rows, cols], device="cuda", dtype=torch.float32).normal_(0, 2, generator=gen)
    many = min(200, cols)
    place = torch.randint(0, cols, [rows, many], device="cuda", generator=gen)
    sure = torch.empty([rows, 1], device="cuda").uniform_(0, 9, generator=gen)
    rank = torch.arange(1, many + 1, device="cuda", dtype=torch.float32)
    return x.scatter_reduce_(1, place, 6 + sure - 1.6 * torch.log(rank), "amax")


def _prepare_topk(c, gen, dtype):
    x = _logits(gen, c["rows"], c["cols"]).to(dtype)
    s = {"x": x, "values_out": torch.empty([c["rows"], c["k"]], device="cuda", dtype=dtype),
         "index_out": torch.empty([c["rows"], c["k"]], device="cuda", dtype=torch.int64)}
    if c["lse"]:
        s["lse_out"] = torch.empty([c["rows"]], device="cuda", dtype=torch.float32)
    return s


def _prepare_sample(c, gen, dtype):
    rows = c["rows"]
    uniform = lambda lo, hi: torch.empty([rows], device="cuda", dtype=torch.float32).uniform_(lo, hi, generator=gen)  # noqa: E731
    s = {"x": _logits(gen, rows, c["cols"]).to(dtype), "u": uniform(0, 1)}
    if c["each"]:
        # a fifth of the requests leaves a setting off, a tenth is greedy
        s["temperature"] = torch.where(uniform(0, 1) < 0.1, 0.0, c["temperature"] * uniform(0.8, 1.2))
        s["top_k"] = torch.where(uniform(0, 1) < 0.2, 0.0, (c["top_k"] * uniform(0.5, 2)).ceil()).to(torch.int32)
        s["top_p"] = torch.where(uniform(0, 1) < 0.2, 1.0, (c["top_p"] * uniform(0.8, 1.1)).clamp_(max=1))
        s["min_p"] = torch.where(uniform(0, 1) < 0.2, 0.0, c["min_p"] * uniform(0.5, 2))
    s["token_out"] = torch.empty([rows], device="cuda", dtype=torch.int64)
    s["logp_out"] = torch.empty([rows], device="cuda", dtype=torch.float32)
    return s


def _prepare_distill(c, gen, dtype):
    rows, cols, k = c["rows"], c["cols"], c["k"]
    teacher = _logits(gen, rows, cols)
    # a student that is on its way: half of what the teacher says, and its own opinion
    x = torch.empty([rows, cols], device="cuda", dtype=torch.float32).normal_(0, 1.5, generator=gen).add_(teacher, alpha=0.6).to(dtype)
    teacher = teacher.to(dtype).float()
    value, index = torch.topk(teacher, k, -1)
    s = {"x": x, "teacher": value.to(dtype)}
    if c["rest"]:
        s["teacher_lse"] = torch.logsumexp(teacher.div_(c["temperature"]), -1)
    if c["ragged"]:
        left = torch.randint(1, k + 1, [rows, 1], device="cuda", generator=gen)
        index = torch.where(torch.arange(k, device="cuda") < left, index, -1)
    s["index"] = index.contiguous()
    # a sixth of the places is padding
    s["mask"] = (torch.empty([rows], device="cuda").uniform_(0, 1, generator=gen) < 5 / 6).float()
    s["mask"][0] = 1
    s["out"] = torch.empty_like(x)
    s["loss_out"] = torch.empty([1], device="cuda", dtype=torch.float32)
    s["kl_out"] = torch.empty([rows], device="cuda", dtype=torch.float32)
    s["terms_out"] = torch.empty([rows, 8], device="cuda", dtype=torch.float32)
    s["upstream"] = 65536.0 if c["dtype"] == "f16" else 1.0  # a loss scale, so that f16 gradients do not vanish
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    make = {"topk": _prepare_topk, "sample": _prepare_sample, "distill": _prepare_distill}[case["kind"]]
    return {"case": dict(case), **make(case, gen, _DTYPES[case["dtype"]])}


# ---- the plain forms ----------------------------------------------------------------------------


def _plain_topk(c, s):
    x = s["x"]
    value, index = torch.sort(x, dim=-1, descending=True, stable=True)
    answer = [value[:, : c["k"]].contiguous(), index[:, : c["k"]].contiguous()]
    if c["lse"]:
        z = x.float() / c["temperature"]
        most = z.amax(-1, keepdim=True)
        answer.append((most[:, 0].double() + torch.log(torch.exp(z - most).sum(-1, dtype=torch.float64))).float())
    return answer


def _settings(c, s):
    """Each row's temperature, number of tokens, probability and part of the likeliest one's, as columns in 64 bits."""
    if c["each"]:
        return [s[n].double()[:, None] for n in ("temperature", "top_k", "top_p", "min_p")]
    return [torch.full([c["rows"], 1], float(c[n]), device="cuda", dtype=torch.float64) for n in ("temperature", "top_k", "top_p", "min_p")]


def _plain_sample(c, s):
    # (which token a number picks depends on sums over the whole row: in 64 bits)
    x = s["x"]
    temperature, k, p, least = _settings(c, s)
    greedy = temperature == 0
    k = torch.where(greedy, 1.0, k)
    k = torch.where(k <= 0, float(c["cols"]), k)
    weight = torch.exp((x.double() - x.amax(-1, keepdim=True).double()) / torch.where(greedy, 1.0, temperature))
    if c["each"] or c["top_k"] > 0 or c["top_p"] < 1 or c["min_p"] > 0:
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices
        ranked = weight.gather(1, order)
        keep = torch.arange(c["cols"], device="cuda") < k
        ranked = torch.where(keep, ranked, 0.0)
        before = ranked.cumsum(-1)
        keep &= (p >= 1) | (before - ranked < p * before[:, -1:])
        keep[:, 0] = True
        keep &= ranked >= least
        weight = torch.zeros_like(weight).scatter_(1, order, torch.where(keep, ranked, 0.0))
    upto = weight.cumsum(-1)
    last = (weight > 0).long().mul_(torch.arange(c["cols"], device="cuda")).amax(-1)
    token = torch.minimum((upto <= s["u"].double()[:, None] * upto[:, -1:]).sum(-1), last)
    logp = torch.log(weight.gather(1, token[:, None])[:, 0] / upto[:, -1])
    return [token, logp.float()]


def _known(c, index):
    """[rows, cols]: the tokens that the teacher names."""
    named = torch.zeros([len(index), c["cols"] + 1], device="cuda", dtype=torch.bool)
    return named.scatter_(1, torch.where(index >= 0, index, c["cols"]), True)[:, : c["cols"]]


def _plain_distill(c, s):
    tau = c["temperature"]
    x = s["x"].float() / tau
    index = s["index"].clamp_min(0)
    known = s["index"] >= 0
    t = torch.where(known, s["teacher"].double() / tau, -math.inf)
    most = x.amax(-1, keepdim=True)
    lse = most[:, 0].double() + torch.log(torch.exp(x - most).sum(-1, dtype=torch.float64))
    mine = x.gather(1, index).double() - lse[:, None]
    logq = t - (s["teacher_lse"].double()[:, None] if c["rest"] else torch.logsumexp(t, -1, keepdim=True))
    q = torch.exp(logq)
    kl = torch.where(known, q * (logq - mine), 0.0).sum(-1)
    p = torch.exp(x - lse.float()[:, None])
    live = s["mask"] > 0
    count = s["mask"].double().sum()
    weight = (s["mask"].double() * tau / count * s["upstream"]).float()[:, None]
    if c["rest"]:
        known_to = _known(c, s["index"])
        others = x.masked_fill(known_to, -math.inf)
        top = others.amax(-1, keepdim=True)
        lse_rest = top[:, 0].double() + torch.log(torch.exp(others - top).sum(-1, dtype=torch.float64))
        rest = (1 - q.sum(-1)).clamp_min(0)
        kl = kl + torch.where(rest > 0, rest * (torch.log(rest) - (lse_rest - lse)), 0.0)
        mass = q.sum(-1) + rest
        p *= torch.where(known_to, mass.float()[:, None], (mass - rest * torch.exp(lse - lse_rest)).float()[:, None])
    d = p.scatter_add_(1, index, torch.where(known, -q, 0.0).float())
    kl = torch.where(live, kl, 0.0)
    loss = tau * tau * (kl * s["mask"].double()).sum() / count
    return [loss.float().reshape(1), kl.float(), (d * weight).to(s["x"].dtype)]


_PLAIN = {"topk": _plain_topk, "sample": _plain_sample, "distill": _plain_distill}


# ---- the framework's calls ----------------------------------------------------------------------


def _tensors(s):
    """The state's device memory as tensors of the framework; nothing is copied. A program has them in hand, so they are
    made on the first pass and kept."""
    if "tensors" not in s:
        import hpt_amd as hpt

        names = {torch.float32: hpt.f32, torch.float16: hpt.f16, torch.bfloat16: hpt.bf16, torch.int32: hpt.i32, torch.int64: hpt.i64}
        t = {k: hpt.Tensor.from_raw(v.data_ptr(), list(v.shape), names[v.dtype]) for k, v in s.items() if isinstance(v, torch.Tensor)}
        # what a program keeps: the workspace
        c = s["case"]
        need = (hpt.topk_workspace(t["x"], c["k"]) if c["kind"] == "topk" else hpt.sample_workspace(t["x"]) if c["kind"] == "sample"
                else hpt.distill_loss_workspace(t["x"]))
        t["workspace"] = hpt.Tensor.empty([need], hpt.u8) if need else None
        s["tensors"] = t
    return s["tensors"]


def _own_topk(c, s):
    t = _tensors(s)
    t["x"].topk(c["k"], lse=c["lse"], temperature=c["temperature"], values_out=t["values_out"], index_out=t["index_out"],
                lse_out=t.get("lse_out"), workspace=t["workspace"])
    return [s["values_out"], s["index_out"]] + ([s["lse_out"]] if c["lse"] else [])


def _own_sample(c, s):
    t = _tensors(s)
    temperature, k, p, least = (t[n] if c["each"] else c[n] for n in ("temperature", "top_k", "top_p", "min_p"))
    t["x"].sample(t["u"], temperature=temperature, top_k=k, top_p=p, min_p=least, token_out=t["token_out"], logp_out=t["logp_out"],
                  workspace=t["workspace"])
    return [s["token_out"], s["logp_out"]]


def _own_distill(c, s):
    t = _tensors(s)
    t["x"].distill_loss(t["teacher"], t["index"], teacher_lse=t.get("teacher_lse"), mask=t["mask"], temperature=c["temperature"],
                        loss_out=t["loss_out"], kl_out=t["kl_out"], terms_out=t["terms_out"], workspace=t["workspace"])
    t["x"].distill_loss_backward(t["teacher"], t["index"], t["terms_out"], temperature=c["temperature"], grad=s["upstream"], out=t["out"])
    return [s["loss_out"], s["kl_out"], s["out"]]


_OWN = {"topk": _own_topk, "sample": _own_sample, "distill": _own_distill}


def run(state):
    c = state["case"]
    return (_OWN if own else _PLAIN)[c["kind"]](c, state)


# ---- what a pass cannot do without --------------------------------------------------------------


def work(case):
    """Every input is read once and every result written once; of the distillation's logits what is no padding (read by the loss,
    and again by its gradient, which needs the whole row's sum)."""
    kind, size = case["kind"], _SIZE[case["dtype"]]
    rows, n = case["rows"], case["rows"] * case["cols"]
    if kind == "topk":
        return {"bytes": n * size + rows * case["k"] * (size + 8) + (4 * rows if case["lse"] else 0), "flops": (4 if case["lse"] else 1) * n}
    if kind == "sample":
        return {"bytes": n * size + rows * (4 + 12 + (16 if case["each"] else 0)), "flops": 4 * n}
    live = 5 / 6
    return {"bytes": int(n * size * (2 * live + 1) + rows * (case["k"] * (size + 8) * live + 12)), "flops": int(9 * n * live)}


# ---- from the definitions -----------------------------------------------------------------------


def _exact_topk(c, s):
    x = s["x"].double()
    # the order by (larger value, smaller index), from the k largest values and all that equal the last of them
    values, indices = [], []
    for row in x:
        least = row.topk(c["k"]).values[-1]
        place = (row >= least).nonzero()[:, 0]
        place = place[torch.argsort(row[place], descending=True, stable=True)][: c["k"]]
        values.append(row[place])
        indices.append(place)
    answer = [torch.stack(values), torch.stack(indices)]
    if c["lse"]:
        answer.append(torch.logsumexp(x / c["temperature"], -1))
    return answer


def _exact_sample(c, s):
    tokens, logps = [], []
    settings = torch.cat(_settings(c, s), 1).tolist()
    numbers = s["u"].tolist()
    for row, u, (temperature, k, p, least) in zip(s["x"].double(), numbers, settings):
        if temperature == 0:
            tokens.append((row == row.max()).nonzero()[0, 0])
            logps.append(torch.zeros([], device="cuda", dtype=torch.float64))
            continue
        prob = torch.softmax(row / temperature, -1)
        left = torch.argsort(row, descending=True, stable=True)
        if k > 0:
            left = left[: int(k)]
        if p < 1:
            part = prob[left].cumsum(0)
            left = left[: int(torch.searchsorted(part, part[-1] * p)) + 1]
        left = left[prob[left] >= least * prob.max()].sort().values
        part = prob[left].cumsum(0)
        at = min(int(torch.searchsorted(part, part[-1] * u, right=True)), len(left) - 1)
        tokens.append(left[at])
        logps.append(torch.log(prob[left[at]] / part[-1]))
    return [torch.stack(tokens), torch.stack(logps)]


def _exact_distill(c, s):
    tau = c["temperature"]
    losses, grads = [], []
    # some rows at a time: 64 bits of the whole would be many times the state
    for at in range(0, c["rows"], 256):
        part = slice(at, at + 256)
        x = (s["x"][part].double() / tau).requires_grad_()
        known = s["index"][part] >= 0
        index = s["index"][part].clamp_min(0)
        t = s["teacher"][part].double() / tau
        logp = torch.log_softmax(x, -1)
        mine = logp.gather(1, index)
        if c["rest"]:
            logq = t - s["teacher_lse"][part].double()[:, None]
            q = torch.where(known, logq.exp(), 0.0)
            r = (1 - q.sum(-1)).clamp_min(0)
            inside = torch.zeros_like(x)
            for j in range(c["k"]):
                inside[torch.arange(len(x), device="cuda"), index[:, j]] += known[:, j]
            other = torch.logsumexp(logp.masked_fill(inside > 0, -math.inf), -1)
            kl = (q * (logq - mine)).sum(-1) + torch.where(r > 0, r * (r.clamp_min(1e-300).log() - other), 0.0)
        else:
            logq = torch.log_softmax(t.masked_fill(~known, -math.inf), -1)
            kl = torch.where(known, logq.exp() * (torch.where(known, logq, 0.0) - mine), 0.0).sum(-1)
        mask = s["mask"][part].double()
        (d,) = torch.autograd.grad((kl * mask).sum() * tau * tau, [x])
        losses.append(kl.detach() * (mask > 0))
        grads.append(d.mul_(s["upstream"] / tau / s["mask"].double().sum()))
    kl = torch.cat(losses)
    loss = tau * tau * (kl * s["mask"].double()).sum() / s["mask"].double().sum()
    return [loss.reshape(1), kl, torch.cat(grads)]


def exact(case, seed):
    s = prepare(case, seed)
    return {"topk": _exact_topk, "sample": _exact_sample, "distill": _exact_distill}[case["kind"]](case, s)

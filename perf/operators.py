"""The row operators around a transformer's blocks, forward and backward, case by case, for timing and for comparing outputs.

  norm         h = x + residual, y = h / sqrt(mean(h^2) + eps) * gamma, rows of hidden states
  norm_8bit    the same with y in 8 bits (e4m3), a scale for each row or for each group of a row
  norm_grad    its backward pass: the gradient of h (with what arrives at h from elsewhere added) and of gamma
  bias         attention's softmax(scale * scores + table[bucket(key - query), head]) over the keys, with a causal mask,
               with the lengths of a padded batch, or with neither
  bias_grad    its backward pass: the gradient of the scores and of the table
  policy       the clipped policy loss with a KL term over a vocabulary of logits, and the gradient of the logits

A case is a dict of plain values. `own` false: elementary torch operations in 32 bits (64 for long sums and next to the
clipping borders), rounded once at the end. `own` true: the calls of the framework, on the same device memory.
`exact` gives the same results from the definitions in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = 1e-6
_E4M3_MOST = 448.0
_LEAST_SCALE = 2.0 ** -120  # of a row of zeros
_CLIP_LOW, _CLIP_HIGH, _KL = 0.2, 0.28, 0.04


def listed():
    return [
        # One step of decoding for a batch of eight: all latency.
        {"name": "norm_decode_bf16", "kind": "norm", "dtype": "bf16", "rows": 8, "cols": 4096, "residual": True},
        # Prefill in half precision at a hidden size that is no power of two: the norm of a block with the residual's addition.
        {"name": "norm_prefill_f16", "kind": "norm", "dtype": "f16", "rows": 13107, "cols": 5120, "residual": True},
        # Decoding for a batch of 33, the input of an 8-bit product, a scale for each token.
        {"name": "norm_8bit_decode_bf16", "kind": "norm_8bit", "dtype": "bf16", "rows": 33, "cols": 5120, "residual": True, "group": 0},
        # Prefill, a scale for each group of 128 elements.
        {"name": "norm_8bit_prefill_bf16", "kind": "norm_8bit", "dtype": "bf16", "rows": 8192, "cols": 4096, "residual": True, "group": 128},
        # Training: the norm's backward pass with the gradient of the residual stream.
        {"name": "norm_grad_bf16", "kind": "norm_grad", "dtype": "bf16", "rows": 16384, "cols": 4096, "stream": True},
        # The same in full precision for short rows of odd length.
        {"name": "norm_grad_f32_odd", "kind": "norm_grad", "dtype": "f32", "rows": 1237, "cols": 1001, "stream": False},
        # An encoder's attention in training: a padded batch, positions in both directions.
        {"name": "bias_encoder_bf16", "kind": "bias", "dtype": "bf16", "batch": 8, "heads": 16, "queries": 1024, "keys": 1024,
         "buckets": 32, "distance": 128, "both": True, "causal": False, "lengths": True},
        # A decoder's step for a batch of 16: one query against a cache of 4097 keys.
        {"name": "bias_decode_f16", "kind": "bias", "dtype": "f16", "batch": 16, "heads": 32, "queries": 1, "keys": 4097,
         "buckets": 32, "distance": 128, "both": False, "causal": True, "lengths": False},
        # A decoder's attention in training, backward.
        {"name": "bias_grad_causal_bf16", "kind": "bias_grad", "dtype": "bf16", "batch": 4, "heads": 16, "queries": 1024, "keys": 1024,
         "buckets": 32, "distance": 128, "both": False, "causal": True, "lengths": False},
        # A small encoder in full precision, odd lengths, backward.
        {"name": "bias_grad_f32_odd", "kind": "bias_grad", "dtype": "f32", "batch": 3, "heads": 12, "queries": 197, "keys": 211,
         "buckets": 32, "distance": 64, "both": True, "causal": False, "lengths": True},
        # A small batch of answers over an odd vocabulary, full-precision logits.
        {"name": "policy_f32", "kind": "policy", "dtype": "f32", "rows": 640, "cols": 50257, "reference": True},
        # A training step's micro-batch over the same vocabulary; the largest case.
        {"name": "policy_bf16", "kind": "policy", "dtype": "bf16", "rows": 8192, "cols": 50257, "reference": True},
    ]


# ---- drawn cases --------------------------------------------------------------------------------

_MOST = 1 << 26  # elements of a drawn case's largest tensor


def _spread(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm; half of them rounded to what sizes mostly are."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        step = 64 if n >= 512 else 8 if n >= 32 else 1
        n = n // step * step
    return max(lo, min(hi, n))


def _dtype(rng):
    return rng.choice(["bf16", "bf16", "f16", "f32"])


def _draw_norm(rng):
    cols = _spread(rng, 64, 16384)
    rows = _spread(rng, 1, max(1, min(131072, _MOST // cols)))
    return {"kind": "norm", "dtype": _dtype(rng), "rows": rows, "cols": cols, "residual": rng.random() < 0.6}


def _draw_norm_8bit(rng):
    group = rng.choice([0, 0, 64, 128])
    cols = _spread(rng, 64, 16384)
    if group:
        cols = max(group, cols // group * group)
    rows = _spread(rng, 1, max(1, min(131072, _MOST // cols)))
    return {"kind": "norm_8bit", "dtype": _dtype(rng), "rows": rows, "cols": cols, "residual": rng.random() < 0.6, "group": group}


def _draw_norm_grad(rng):
    cols = _spread(rng, 64, 16384)
    rows = _spread(rng, 16, max(16, min(131072, _MOST // 2 // cols)))
    return {"kind": "norm_grad", "dtype": _dtype(rng), "rows": rows, "cols": cols, "stream": rng.random() < 0.5}


def _draw_scores(rng, kind, most):
    keys = _spread(rng, 16, 4096)
    # as many queries as keys, a chunk of a longer context, or one step of decoding
    queries = rng.choice([keys, keys, _spread(rng, 1, keys)] + ([1] if kind == "bias" else []))
    heads = rng.choice([4, 6, 8, 12, 16, 32])
    batch = _spread(rng, 1, max(1, min(64, most // (keys * queries * heads))))
    if batch * heads * queries * keys > most:
        heads, batch = max(1, most // (keys * queries)), 1
    both = rng.random() < 0.5
    return {"kind": kind, "dtype": _dtype(rng), "batch": batch, "heads": heads, "queries": queries, "keys": keys,
            "buckets": rng.choice([16, 32, 32, 64]), "distance": rng.choice([64, 128, 128, 256]), "both": both,
            "causal": not both, "lengths": rng.random() < 0.5}


def _draw_bias(rng):
    return _draw_scores(rng, "bias", _MOST)


def _draw_bias_grad(rng):
    return _draw_scores(rng, "bias_grad", _MOST // 2)


def _draw_policy(rng):
    cols = _spread(rng, 16384, 152000)
    return {"kind": "policy", "dtype": _dtype(rng), "rows": _spread(rng, 1, _MOST // cols), "cols": cols,
            "reference": rng.random() < 0.7}


def draw(rng):
    return rng.choice([_draw_norm, _draw_norm_8bit, _draw_norm_grad, _draw_bias, _draw_bias_grad, _draw_policy])(rng)


# ---- inputs -------------------------------------------------------------------------------------


def _normal(gen, shape, dtype, std=1.0, mean=0.0):
    return torch.empty(shape, device="cuda", dtype=dtype).normal_(mean, std, generator=gen)


def _prepare_norm(case, gen, dtype):
    rows, cols = case["rows"], case["cols"]
    # hidden states: tokens of different size, a few channels that stand out
    size = torch.empty([rows, 1], device="cuda").uniform_(0.3, 3, generator=gen)
    channel = torch.empty([cols], device="cuda").uniform_(0, 1, generator=gen).pow_(8).mul_(10).add_(0.5)
    x = _normal(gen, [rows, cols], torch.float32).mul_(size).mul_(channel).to(dtype)
    s = {"x": x, "gamma": _normal(gen, [cols], dtype, 0.2, 1.0)}
    if case["kind"] == "norm_grad":
        s["grad"] = _normal(gen, [rows, cols], dtype, 0.1)
        if case["stream"]:
            s["grad_sum"] = _normal(gen, [rows, cols], dtype, 0.1)
        s["out"] = torch.empty_like(x)
        s["gamma_out"] = torch.empty([cols], device="cuda", dtype=torch.float32)
        return s
    if case["residual"]:
        s["residual"] = _normal(gen, [rows, cols], dtype)
        s["sum_out"] = torch.empty_like(x)
    if case["kind"] == "norm":
        s["out"] = torch.empty_like(x)
    else:
        s["out"] = torch.empty([rows, cols], device="cuda", dtype=torch.uint8)
        s["scale_out"] = torch.empty([rows, cols // case["group"]] if case["group"] else [rows], device="cuda", dtype=torch.float32)
    return s


def _offset(case):
    """The position of the first query: the last one sees every key."""
    return case["keys"] - case["queries"]


def _live(case, lengths):
    """[batch or 1, queries, keys]: which keys a query sees."""
    key = torch.arange(case["keys"], device="cuda")
    live = torch.ones([1, case["queries"], case["keys"]], device="cuda", dtype=torch.bool)
    if case["causal"]:
        live = live & (key <= torch.arange(case["queries"], device="cuda")[:, None] + _offset(case))
    if lengths is not None:
        live = live & (key < lengths[:, None, None])
    return live


def _prepare_scores(case, gen, dtype):
    shape = [case["batch"], case["heads"], case["queries"], case["keys"]]
    s = {"scale": 0.125}
    if case["lengths"]:
        # a padded batch: most sequences reach over half the keys
        part = torch.empty([case["batch"]], device="cuda").uniform_(0.4, 1, generator=gen)
        s["lengths"] = (part * case["keys"]).ceil().to(torch.int64).clamp_(1, case["keys"])
    if case["kind"] == "bias":
        s["x"] = _normal(gen, shape, dtype, 16.0)
        s["table"] = _normal(gen, [case["buckets"], case["heads"]], dtype, 0.5)
    else:
        # the probabilities that the forward pass has returned, and the gradient that the values' product sends back
        p = _normal(gen, shape, torch.float32, 2.0)
        p.masked_fill_(~_live(case, s.get("lengths"))[:, None], -math.inf)
        s["probs"] = torch.nan_to_num_(torch.softmax(p, -1)).to(dtype)
        s["grad"] = _normal(gen, shape, dtype, 0.1)
        s["table_out"] = torch.empty([case["buckets"], case["heads"]], device="cuda", dtype=torch.float32)
    s["out"] = torch.empty(shape, device="cuda", dtype=dtype)
    return s


def _prepare_policy(case, gen, dtype):
    rows, cols = case["rows"], case["cols"]
    x = _normal(gen, [rows, cols], dtype, 3.0)
    s = {"x": x, "out": torch.empty_like(x)}
    # tokens as a model samples them; what the policy that sampled them and the reference said of them
    noise = torch.empty([rows, cols], device="cuda", dtype=torch.float32).exponential_(generator=gen).log_()
    token = (x.float() - noise).argmax(-1)
    del noise
    logp = x.float().gather(1, token[:, None])[:, 0] - torch.logsumexp(x.float(), -1)
    s["old"] = logp + _normal(gen, [rows], torch.float32, 0.15)
    if case["reference"]:
        s["reference"] = logp + _normal(gen, [rows], torch.float32, 0.3)
    s["advantage"] = _normal(gen, [rows], torch.float32)
    # a sixth of the places is padding, without a token
    s["mask"] = (torch.empty([rows], device="cuda").uniform_(0, 1, generator=gen) < 5 / 6).float()
    s["mask"][0] = 1
    s["token"] = torch.where(s["mask"] > 0, token, -100)
    for name in ("logp", "lse", "weight"):
        s[name + "_out"] = torch.empty([rows], device="cuda", dtype=torch.float32)
    s["loss_out"] = torch.empty([1], device="cuda", dtype=torch.float32)
    s["upstream"] = 4096.0 if case["dtype"] == "f16" else 1.0  # a loss scale, so that f16 gradients do not vanish
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    make = {"norm": _prepare_norm, "bias": _prepare_scores, "policy": _prepare_policy}[case["kind"].partition("_")[0]]
    return {"case": dict(case), **make(case, gen, _DTYPES[case["dtype"]])}


# ---- the plain forms ----------------------------------------------------------------------------


def _plain_norm(c, s):
    x = s["x"]
    answer = []
    if c["residual"]:
        h = (x.float() + s["residual"].float()).to(x.dtype)
        answer = [h]
    else:
        h = x
    h = h.float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + _EPS) * s["gamma"].float()
    if c["kind"] == "norm":
        return [y.to(x.dtype)] + answer
    groups = y.view(c["rows"], -1, c["group"] or c["cols"])
    scale = (groups.abs().amax(-1, keepdim=True) / _E4M3_MOST).clamp_min(_LEAST_SCALE)
    q = (groups / scale).to(torch.float8_e4m3fn)
    return [q.view(c["rows"], c["cols"]), scale.view(s["scale_out"].shape)] + answer


def _plain_norm_grad(c, s):
    x, gy = s["x"].float(), s["grad"].float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS)
    n = x * r
    g = gy * s["gamma"].float()
    d = r * (g - n * (g * n).mean(-1, keepdim=True))
    if c["stream"]:
        d = d + s["grad_sum"].float()
    return [d.to(s["x"].dtype), (gy * n).sum(0)]


def _bucket(c, rel):
    """The bucket of key - query. Half of the buckets (of each direction) hold one distance each, the
    others grow with the logarithm up to the largest distance. (The logarithm decides at whole distances: in 64 bits.)"""
    n = c["buckets"] // 2 if c["both"] else c["buckets"]
    first = (rel > 0) * n if c["both"] else torch.zeros_like(rel)
    far = rel.abs() if c["both"] else (-rel).clamp_min(0)
    exact_ones = n // 2
    grown = torch.log2(far.clamp_min(1).double() / exact_ones) / math.log2(c["distance"] / exact_ones) * (n - exact_ones)
    grown = exact_ones + torch.floor(grown + 1e-9).long()
    return first + torch.where(far < exact_ones, far, grown.clamp_max(n - 1))


def _plain_bias(c, s):
    x = s["x"]
    rel = torch.arange(c["keys"], device="cuda") - (torch.arange(c["queries"], device="cuda")[:, None] + _offset(c))
    bias = s["table"].float()[_bucket(c, rel)].permute(2, 0, 1)
    live = _live(c, s.get("lengths"))[:, None]
    t = (s["scale"] * x.float() + bias).masked_fill(~live, -math.inf)
    most = t.amax(-1, keepdim=True)
    e = torch.exp(t - torch.where(live.any(-1, keepdim=True), most, 0.0))
    return [(e / e.sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).tiny)).to(x.dtype)]


def _plain_bias_grad(c, s):
    p = s["probs"].float()
    g = s["grad"].float().masked_fill(~_live(c, s.get("lengths"))[:, None], 0.0)
    d = p * (g - (p * g).sum(-1, keepdim=True))
    # the sums of equal distances: every row moved on by one place less than the one before, so that they are columns
    q, k = c["queries"], c["keys"]
    total = torch.nn.functional.pad(d.sum(0, dtype=torch.float64).flip(1), (0, q))
    total = total.reshape(c["heads"], -1)[:, : q * (k + q - 1)].view(c["heads"], q, k + q - 1).sum(1)
    rel = torch.arange(1 - q, k, device="cuda") - _offset(c)
    table = total @ torch.nn.functional.one_hot(_bucket(c, rel), c["buckets"]).double()
    return [(s["scale"] * d).to(s["probs"].dtype), table.t().float().contiguous()]


def _plain_policy(c, s):
    x = s["x"].float()
    live = s["mask"] > 0
    token = s["token"].clamp_min(0)[:, None]
    most = x.amax(-1, keepdim=True)
    total = torch.exp(x - most).sum(-1, dtype=torch.float64)
    lse = most[:, 0].double() + torch.log(total)
    logp = x.gather(1, token)[:, 0].double() - lse
    mask, a = s["mask"].double(), s["advantage"].double()
    ratio = torch.exp(logp - s["old"].double())
    free, held = ratio * a, ratio.clamp(1 - _CLIP_LOW, 1 + _CLIP_HIGH) * a
    each = -torch.minimum(free, held)
    slope = torch.where(free <= held, -free, 0.0)
    if c["reference"]:
        k = s["reference"].double() - logp
        each = each + _KL * (torch.exp(k) - k - 1)
        slope = slope + _KL * (1 - torch.exp(k))
    count = mask.sum()
    loss = torch.where(live, each * mask, 0.0).sum() / count
    weight = (torch.where(live, slope * mask, 0.0) / count).float()
    lse = torch.where(live, lse, 0.0).float()
    d = -torch.exp(x - lse[:, None])
    d.scatter_add_(1, token, torch.ones_like(token, dtype=torch.float32))
    d = d * (weight * s["upstream"])[:, None]
    return [loss.float().reshape(1), torch.where(live, logp, 0.0).float(), lse, weight, d.to(s["x"].dtype)]


_PLAIN = {"norm": _plain_norm, "norm_8bit": _plain_norm, "norm_grad": _plain_norm_grad, "bias": _plain_bias, "bias_grad": _plain_bias_grad,
          "policy": _plain_policy}


# ---- the framework's calls ----------------------------------------------------------------------


def _tensors(s):
    """The state's device memory as tensors of the framework; nothing is copied. A program has them in hand, so they are
    made on the first pass and kept."""
    if "tensors" not in s:
        import hpt_amd as hpt

        names = {torch.float32: hpt.f32, torch.float16: hpt.f16, torch.bfloat16: hpt.bf16, torch.uint8: hpt.u8, torch.int64: hpt.i64}
        s["tensors"] = {k: hpt.Tensor.from_raw(v.data_ptr(), list(v.shape), names[v.dtype]) for k, v in s.items() if isinstance(v, torch.Tensor)}
        # what a program keeps for its backward passes: their workspaces
        c = s["case"]
        need = 0
        if c["kind"] == "norm_grad":
            need = hpt.rms_norm_backward_workspace(s["tensors"]["x"], 1)
        elif c["kind"] == "bias_grad":
            need = hpt.softmax_bias_backward_workspace(s["tensors"]["probs"], c["buckets"])
        elif c["kind"] == "bias":
            need = hpt.softmax_bias_workspace(s["tensors"]["x"])
        elif c["kind"] == "policy":
            need = hpt.policy_loss_workspace(s["tensors"]["x"])
        s["tensors"]["workspace"] = hpt.Tensor.empty([need], hpt.u8) if need else None
    return s["tensors"]


def _own_norm(c, s):
    t = _tensors(s)
    if c["kind"] == "norm_8bit":
        t["x"].rms_norm_quant([c["cols"]], t["gamma"], _EPS, residual=t.get("residual"), format="e4m3", group=c["group"], out=t["out"],
                              scale_out=t["scale_out"], sum_out=t.get("sum_out"))
        answer = [s["out"].view(torch.float8_e4m3fn), s["scale_out"]]
    elif c["residual"]:
        t["x"].add_rms_norm(t["residual"], [c["cols"]], t["gamma"], _EPS, out=t["out"], sum_out=t["sum_out"])
        answer = [s["out"]]
    else:
        t["x"].rms_norm([c["cols"]], t["gamma"], _EPS, out=t["out"])
        answer = [s["out"]]
    return answer + ([s["sum_out"]] if c["residual"] else [])


def _own_norm_grad(c, s):
    t = _tensors(s)
    t["x"].rms_norm_backward(t["grad"], [c["cols"]], t["gamma"], _EPS, grad_sum=t.get("grad_sum"), out=t["out"], gamma_out=t["gamma_out"],
                             workspace=t["workspace"])
    return [s["out"], s["gamma_out"]]


def _own_bias(c, s):
    t = _tensors(s)
    t["x"].softmax_bias(t["table"], s["scale"], bidirectional=c["both"], max_distance=c["distance"], query_offset=_offset(c), causal=c["causal"],
                        lengths=t.get("lengths"), out=t["out"], workspace=t["workspace"])
    return [s["out"]]


def _own_bias_grad(c, s):
    t = _tensors(s)
    t["probs"].softmax_bias_backward(t["grad"], c["buckets"], s["scale"], bidirectional=c["both"], max_distance=c["distance"],
                                     query_offset=_offset(c), causal=c["causal"], lengths=t.get("lengths"), out=t["out"],
                                     table_out=t["table_out"], workspace=t["workspace"])
    return [s["out"], s["table_out"]]


def _own_policy(c, s):
    t = _tensors(s)
    t["x"].policy_loss(t["token"], t["old"], t["advantage"], reference=t.get("reference"), mask=t["mask"], clip_low=_CLIP_LOW,
                       clip_high=_CLIP_HIGH, kl_weight=_KL if c["reference"] else 0.0, loss_out=t["loss_out"], logp_out=t["logp_out"],
                       lse_out=t["lse_out"], weight_out=t["weight_out"], workspace=t["workspace"])
    t["x"].policy_loss_backward(t["token"], t["lse_out"], t["weight_out"], s["upstream"], out=t["out"])
    return [s["loss_out"], s["logp_out"], s["lse_out"], s["weight_out"], s["out"]]


_OWN = {"norm": _own_norm, "norm_8bit": _own_norm, "norm_grad": _own_norm_grad, "bias": _own_bias, "bias_grad": _own_bias_grad,
        "policy": _own_policy}


def run(state):
    c = state["case"]
    return (_OWN if own else _PLAIN)[c["kind"]](c, state)


# ---- what a pass cannot do without --------------------------------------------------------------


def _live_keys(case):
    """How many keys a matrix of the batch's queries sees, on average."""
    q, k = case["queries"], case["keys"]
    part = 0.7 if case["lengths"] else 1.0
    if not case["causal"]:
        return q * k * part
    return sum(min(k * part, i + k - q + 1) for i in range(q))


def work(case):
    """Every input is read once and every result written once; of the scores what the masks leave, of the logits (read
    by the loss, and again by its gradient, which needs the whole row's sum) what is no padding."""
    kind, size = case["kind"], _SIZE[case["dtype"]]
    if kind.startswith("norm"):
        n, cols = case["rows"] * case["cols"], case["cols"]
        if kind == "norm_grad":
            return {"bytes": n * size * (4 if case["stream"] else 3) + cols * (size + 4), "flops": 14 * n}
        moved = n * size * (3 if case["residual"] else 1) + cols * size
        if kind == "norm":
            return {"bytes": moved + n * size, "flops": 5 * n}
        return {"bytes": moved + n + 4 * (n // case["group"] if case["group"] else case["rows"]), "flops": 8 * n}
    if kind.startswith("bias"):
        whole = case["batch"] * case["heads"] * case["queries"] * case["keys"]
        live = case["batch"] * case["heads"] * _live_keys(case)
        table = case["buckets"] * case["heads"]
        if kind == "bias":
            return {"bytes": (live + whole + table) * size, "flops": 8 * live}
        return {"bytes": (2 * live + whole) * size + 4 * table, "flops": 6 * live}
    n = case["rows"] * case["cols"]
    return {"bytes": n * size * (5 / 6 * 2 + 1) + case["rows"] * 40, "flops": 5 / 6 * 9 * n}


# ---- the results in 64 bits ---------------------------------------------------------------------


def _exact_norm(c, s):
    x, gamma = s["x"].double(), s["gamma"].double()
    if c["kind"] == "norm_grad":
        # the definition's own derivative
        x.requires_grad_(True)
        gamma.requires_grad_(True)
        y = x / (x.pow(2).sum(-1, keepdim=True) / c["cols"] + _EPS).sqrt() * gamma
        dx, dgamma = torch.autograd.grad(y, [x, gamma], s["grad"].double())
        return [dx + s["grad_sum"].double() if c["stream"] else dx, dgamma]
    h = x
    if c["residual"]:
        h = (x + s["residual"].double()).to(s["x"].dtype).double()  # the sum is stored in the inputs' type
    y = h / (h.pow(2).sum(-1, keepdim=True) / c["cols"] + _EPS).sqrt() * gamma
    more = [h] if c["residual"] else []
    if c["kind"] == "norm":
        return [y] + more
    width = c["group"] or c["cols"]
    most = torch.linalg.vector_norm(y.unflatten(1, (-1, width)), math.inf, -1)
    scale = torch.maximum(most / _E4M3_MOST, torch.full_like(most, _LEAST_SCALE))
    return [y / scale.repeat_interleave(width, 1), scale.reshape(s["scale_out"].shape)] + more


def _exact_buckets(c):
    """The buckets by the distances at which they begin."""
    n = c["buckets"] // 2 if c["both"] else c["buckets"]
    half = n // 2
    grow = [half * (c["distance"] / half) ** (j / (n - half)) for j in range(1, n - half)]
    begins = list(range(1, half + 1)) + [math.ceil(g * (1 - 1e-12)) for g in grow]
    place = torch.arange(c["keys"], device="cuda") - torch.arange(c["queries"], device="cuda")[:, None] - _offset(c)
    begins = torch.tensor(begins, device="cuda")
    back = torch.searchsorted(begins, (-place).clamp_min(0), right=True)
    if not c["both"]:
        return back
    return torch.where(place > 0, n + torch.searchsorted(begins, place.clamp_min(0), right=True), back)


def _exact_scores(c, s):
    live = _live(c, s.get("lengths"))[:, None]
    which = _exact_buckets(c)
    if c["kind"] == "bias":
        t = s["x"].double() * s["scale"] + torch.nn.functional.embedding(which, s["table"].double()).movedim(-1, 0)
        return [torch.softmax(t.masked_fill(~live, -math.inf), -1).masked_fill(~live, 0.0)]
    p, g = s["probs"].double(), s["grad"].double() * live
    d = p * g - p * (p * g).sum(-1, keepdim=True)
    total = d.sum(0)
    # the sums of the diagonals of equal distance, bucket by bucket
    table = torch.stack([(total * (which == b)).sum((1, 2)) for b in range(c["buckets"])])
    return [s["scale"] * d, table]


def _exact_policy(c, s):
    # the loss as a function of the chosen tokens' log-probabilities and its derivative, then the log-softmax's
    x = s["x"].double()
    live = s["mask"] > 0
    token = torch.where(live, s["token"], 0)
    lse = torch.logsumexp(x, -1)
    logp = (x[torch.arange(c["rows"], device="cuda"), token] - lse).requires_grad_(True)
    ratio = torch.exp(logp - s["old"].double())
    a = s["advantage"].double()
    inside = torch.where(a >= 0, ratio <= 1 + _CLIP_HIGH, ratio >= 1 - _CLIP_LOW)
    held = torch.where(a >= 0, 1 + _CLIP_HIGH, 1 - _CLIP_LOW)
    each = -a * torch.where(inside, ratio, held)
    if c["reference"]:
        k = s["reference"].double() - logp
        each = each + _KL * (torch.expm1(k) - k)
    loss = (each * s["mask"].double()).sum() / s["mask"].double().sum()
    (weight,) = torch.autograd.grad(loss, [logp])
    d = torch.softmax(x, -1).neg_()
    d[torch.arange(c["rows"], device="cuda"), token] += 1
    d *= (weight * s["upstream"])[:, None]
    return [loss.detach().reshape(1), (logp.detach() * live), lse * live, weight, d]


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "bias": _exact_scores, "policy": _exact_policy}[case["kind"].partition("_")[0]](case, s)

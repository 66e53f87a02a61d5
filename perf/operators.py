"""Operators on rows of candidate logits: what they compute, in plain form, and how long they take.

A row holds the logits of one node's candidate window (or any other row of logits); its first ``counts[r]`` places are
valid.  Four operators work on such rows:

  sample   draws positions without replacement, with temperature, top-k, top-p and min-p, from given random numbers
  top      a teacher's largest logits with their positions, and the row's log-sum-exp
  distill  the loss of a student's rows against a teacher's top logits, and its gradient
  scores   logits looked up in a table over (kind of row, class of candidate), and the gradient of that table

``own`` False computes them out of elementary torch operations; True calls ``gan_amd.logits``.
"""
import math

import numpy as np
import torch

own = False

UNIT = 2.0 ** 36          # weights of a row are whole multiples of 1 / UNIT of its largest
DEV = "cuda"
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


# ------------------------------------------------------------------ cases
def listed():
    f32 = "float32"
    return [
        # one slot of the default window: what a single choice costs
        dict(name="sample_one_row", op="sample", rows=1, width=512, draws=2, dtype=f32, temperature=0.8, top_k=0, top_p=0.95,
             min_p=0.0, per_row=False, counts="full", ties=False),
        # every slot of a 100k-node template at k = 64: two fan-ins each, all filters
        dict(name="sample_100k_k64", op="sample", rows=100000, width=64, draws=2, dtype=f32, temperature=0.8, top_k=32,
             top_p=0.9, min_p=0.02, per_row=False, counts="ramp", ties=True),
        # a block of 64 draws of the c7552-sized template at k = 256 (bulk sampling)
        dict(name="sample_bulk_k256", op="sample", rows=152896, width=256, draws=2, dtype=f32, temperature=1.0, top_k=0,
             top_p=0.9, min_p=0.0, per_row=False, counts="full", ties=False),
        # requests with settings of their own over long rows in half precision
        dict(name="sample_wide_bf16", op="sample", rows=48, width=50001, draws=1, dtype="bfloat16", temperature=0.9, top_k=50,
             top_p=0.95, min_p=0.0, per_row=True, counts="full", ties=False),
        # a teacher's answers kept for a 100k-node template
        dict(name="top_100k_k64", op="top", rows=100000, width=64, m=16, dtype=f32, temperature=2.0, counts="ramp", ties=True),
        # ... and from long rows
        dict(name="top_wide_f16", op="top", rows=96, width=32771, m=64, dtype="float16", temperature=1.0, counts="full", ties=False),
        # the loss alone on a small graph (validation): latency
        dict(name="distill_loss_243", op="distill", way="loss", rows=243, width=16, m=4, dtype=f32, temperature=2.0, tail=True,
             counts="ramp", weighted=False),
        # a training step on a million-node graph: loss and gradient in one call
        dict(name="distill_step_1m_k64", op="distill", way="step", rows=1000000, width=64, m=8, dtype=f32, temperature=2.0,
             tail=True, counts="full", weighted=True),
        # the minibatch of all eleven ISCAS85-sized graphs at the default window, through autograd, half precision
        dict(name="distill_k512_bf16", op="distill", way="autograd", rows=26279, width=512, m=32, dtype="bfloat16",
             temperature=1.0, tail=False, counts="ragged", weighted=False),
        # long rows through autograd
        dict(name="distill_wide_bf16", op="distill", way="autograd", rows=512, width=32001, m=64, dtype="bfloat16",
             temperature=1.5, tail=True, counts="full", weighted=False),
        # the generator's candidate logits of a 100k-node template and the gradient of its score table
        dict(name="scores_100k_k64", op="scores", rows=100000, width=64, kinds=9, classes=9, counts="ramp"),
        # ... of eleven graphs of a minibatch at the default window (a table per graph)
        dict(name="scores_11x2389_k512", op="scores", rows=26279, width=512, kinds=99, classes=9, counts="full"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["sample", "sample", "top", "distill", "distill", "scores"])
    dtype = rng.choice(["float32", "float32", "bfloat16", "float16"])
    counts = rng.choice(["full", "ramp", "ragged"])
    if op != "scores" and rng.random() < 0.35:
        width = _log_int(rng, 1025, 131072)
        rows = _log_int(rng, 1, max(1, min(512, 20_000_000 // width)))
    else:
        width = _log_int(rng, 1, 1024)
        rows = _log_int(rng, 1, max(1, min(1_000_000, 20_000_000 // width)))
    if op == "sample":
        return dict(op=op, rows=rows, width=width, draws=rng.randint(1, 4), dtype=dtype,
                    temperature=round(rng.uniform(0.3, 2.0), 3), top_k=rng.choice([0, 0, _log_int(rng, 1, 200)]),
                    top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]), min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.3), 4)]),
                    per_row=rng.random() < 0.3, counts=counts, ties=rng.random() < 0.4)
    if op == "top":
        return dict(op=op, rows=rows, width=width, m=_log_int(rng, 1, min(256, width)), dtype=dtype,
                    temperature=round(rng.uniform(0.5, 4.0), 3), counts=counts, ties=rng.random() < 0.4)
    if op == "distill":              # (a loss that is zero but for rounding says nothing: rows with some choice in them)
        width = max(width, 8)
        counts = counts if rows >= 16 else "full"
        return dict(op=op, way=rng.choice(["loss", "step", "autograd"]), rows=rows, width=width, m=_log_int(rng, 1, min(128, width // 2)),
                    dtype=dtype, temperature=round(rng.uniform(0.5, 4.0), 3), tail=rng.random() < 0.5, counts=counts,
                    weighted=rng.random() < 0.5)
    return dict(op=op, rows=rows, width=width, kinds=_log_int(rng, 1, 200), classes=_log_int(rng, 1, 40), counts=counts)


def _places(case):
    """Valid places of all rows (on average for ragged counts)."""
    rows, width = case["rows"], case["width"]
    if case["counts"] == "full":
        return rows * width
    if case["counts"] == "ramp":
        k = min(rows, width + 1)
        return k * (k - 1) // 2 + (rows - k) * width
    return rows * (width + 1) // 2


def work(case):
    rows, places = case["rows"], _places(case)
    size = 2 if case.get("dtype") in ("float16", "bfloat16") else 4
    counts = 0 if case["counts"] == "full" else 4 * rows
    if case["op"] == "sample":       # logits, random numbers, counts, settings; picks.  An exp and a few additions a place
        return {"bytes": places * size + 8 * rows * case["draws"] + counts + (16 * rows if case["per_row"] else 0), "flops": 24 * places}
    if case["op"] == "top":          # logits, counts; values, positions, log-sum-exp
        return {"bytes": places * size + counts + 8 * rows * case["m"] + 4 * rows, "flops": 8 * places}
    if case["op"] == "distill":      # logits once, the teacher's part; the losses, and the gradient once (whole rows: zeros too)
        teacher = 8 * rows * case["m"] + (4 * rows if case["tail"] else 0) + (4 * rows if case["weighted"] else 0)
        grad = 0 if case["way"] == "loss" else rows * case["width"] * size
        loss = 4 * rows if case["way"] != "autograd" else 4
        return {"bytes": places * size + counts + teacher + grad + loss, "flops": (8 if case["way"] == "loss" else 12) * places}
    # candidates and upstream gradient once, logits once (whole rows), classes, kinds, order of the rows, both tables
    return {"bytes": 8 * places + 4 * rows * case["width"] + counts + 12 * rows + 8 * case["kinds"] * case["classes"], "flops": places}


# ------------------------------------------------------------------ inputs
def _counts(case, g):
    rows, width = case["rows"], case["width"]
    if case["counts"] == "full":
        return None
    if case["counts"] == "ramp":     # the r-th node of a template has at most r candidates
        return torch.arange(rows, device=DEV).clamp(max=width).to(torch.int32)
    return torch.randint(0, width + 1, (rows,), device=DEV, generator=g, dtype=torch.int32)


def _logits(rows, width, dtype, g, ties=False):
    if ties:      # scores of a template: a handful of distinct values a row
        table = torch.randn(9, 9, device=DEV, generator=g)
        a = torch.randint(0, 9, (rows, width), device=DEV, generator=g)
        b = torch.randint(0, 9, (rows, 1), device=DEV, generator=g)
        return table[b, a].to(dtype)
    return (2.0 * torch.randn(rows, width, device=DEV, generator=g)).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    rows, width = case["rows"], case["width"]
    s = dict(case, counts=_counts(case, g))
    if case["op"] == "sample":
        s["logits"] = _logits(rows, width, DTYPES[case["dtype"]], g, case["ties"])
        s["u"] = torch.rand(rows, case["draws"], device=DEV, generator=g)
        if case["per_row"]:
            def spread(v, lo, hi):
                return (v * (0.6 + 0.8 * torch.rand(rows, device=DEV, generator=g))).clamp(lo, hi)
            s["temperature"] = spread(case["temperature"], 0.1, 10.0)
            s["top_k"] = (spread(float(case["top_k"]), 0.0, 1e6)).round().to(torch.int32)
            s["top_p"] = spread(case["top_p"], 0.05, 1.0)
            s["min_p"] = spread(case["min_p"], 0.0, 1.0)
    elif case["op"] == "top":
        s["logits"] = _logits(rows, width, DTYPES[case["dtype"]], g, case["ties"])
    elif case["op"] == "distill":
        # the teacher's rows are near the student's, as they are once a student has begun to learn
        student = 2.0 * torch.randn(rows, width, device=DEV, generator=g)
        teacher = student + 0.7 * torch.randn(rows, width, device=DEV, generator=g)
        if s["counts"] is not None:
            teacher.masked_fill_(torch.arange(width, device=DEV) >= s["counts"][:, None], -math.inf)
        v, i = teacher.topk(case["m"], dim=1)
        s["values"], s["index"] = v, torch.where(v > -math.inf, i, -1).to(torch.int32)
        s["lse"] = torch.logsumexp(teacher / case["temperature"], dim=1) if case["tail"] else None
        s["weight"] = torch.rand(rows, device=DEV, generator=g) if case["weighted"] else None
        s["logits"] = student.to(DTYPES[case["dtype"]]).requires_grad_(case["way"] == "autograd")
    else:
        kinds, classes = case["kinds"], case["classes"]
        s["table"] = torch.randn(kinds, classes, device=DEV, generator=g).requires_grad_(True)
        s["classes_of"] = torch.randint(0, classes, (rows,), device=DEV, generator=g, dtype=torch.int32)
        s["row_kind"] = torch.randint(0, kinds, (rows,), device=DEV, generator=g, dtype=torch.int32)
        # windows of nearby nodes, as a template's are
        start = (torch.arange(rows, device=DEV) - width).clamp(min=0)[:, None]
        s["cand"] = (start + torch.arange(width, device=DEV)).clamp(max=rows - 1).to(torch.int32)
        s["grad"] = torch.randn(rows, width, device=DEV, generator=g)
        # kept with a template's plan: its rows in the order of their kinds
        s["by_kind"] = torch.argsort(s["row_kind"], stable=True).to(torch.int32)
        s["kind_start"] = torch.searchsorted(s["row_kind"][s["by_kind"].long()].contiguous(),
                                             torch.arange(kinds + 1, device=DEV, dtype=torch.int32)).to(torch.int32)
    return s


# ------------------------------------------------------------------ plain forms
def _valid(s, x):
    ok = x > -math.inf                       # neither masked nor NaN
    if s["counts"] is not None:
        ok &= torch.arange(x.size(1), device=x.device) < s["counts"][:, None]
    return ok


def _setting(v, rows):
    """A setting of all rows or of each, in the 32 bits that it is taken in, as a column in 64."""
    if torch.is_tensor(v):
        return v.float().double()[:, None]
    return torch.full((rows, 1), float(np.float32(v)), dtype=torch.float64, device=DEV)


def _plain_sample(s):
    rows, width, draws = s["rows"], s["width"], s["draws"]
    temperature, top_k, top_p, min_p = (_setting(s[k], rows) for k in ("temperature", "top_k", "top_p", "min_p"))
    x = s["logits"].double()
    ok = _valid(s, x)
    x = x.masked_fill(~ok, -math.inf)
    top = x.amax(1, keepdim=True)
    q = torch.where(x == top, torch.zeros_like(x), x - top).div_(temperature).exp_().mul_(UNIT).round_()
    q.masked_fill_(~ok, 0.0)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    q = q.gather(1, order)
    rank = torch.arange(width, device=DEV)
    q *= (rank < top_k) | (top_k <= 0)
    upto = q.cumsum(1)
    q *= (rank == 0) | (top_p >= 1) | (upto - q < top_p * upto[:, -1:])
    q *= q >= min_p.clamp(max=1.0) * UNIT
    kept = torch.zeros_like(q).scatter_(1, order, q)
    picks = torch.empty(rows, draws, dtype=torch.int32, device=DEV)
    u = s["u"].double().clamp(0.0, 1.0 - 2.0 ** -24)
    for d in range(draws):
        upto = kept.cumsum(1)
        total = upto[:, -1]
        pick = (upto <= (u[:, d] * total)[:, None]).sum(1)
        picks[:, d] = torch.where(total > 0, pick, -1)
        kept.scatter_(1, pick.clamp(max=width - 1)[:, None], 0.0)
    return picks


def _plain_top(s):
    x = s["logits"].float()
    x = x.masked_fill(~_valid(s, x), -math.inf)
    v, i = torch.sort(x, dim=1, descending=True, stable=True)
    v, i = v[:, :s["m"]], i[:, :s["m"]]
    index = torch.where(v > -math.inf, i, -1).to(torch.int32)
    y = x / s["temperature"]
    top = y.amax(1, keepdim=True)
    lse = torch.log(torch.exp(y - torch.where(top > -math.inf, top, 0.0)).sum(1)) + torch.where(top > -math.inf, top, 0.0)[:, 0]
    return v.contiguous(), index, lse


def _plain_distill(s, with_grad):
    """The loss of each row, times its weight, and its gradient: temperature^2 times the divergence of the student's
    probabilities from the teacher's over the listed places (and, with ``tail``, all others as one)."""
    rows, width, t = s["rows"], s["width"], s["temperature"]
    x = s["logits"].detach().float()
    ok = _valid(s, x)
    y = (x / t).masked_fill(~ok, -math.inf)
    e = torch.exp(y - y.amax(1, keepdim=True))
    total = e.double().sum(1, keepdim=True)
    p = (e / total).float()
    logp = y - y.amax(1, keepdim=True) - torch.log(total).float()
    idx = s["index"].long()
    listed_ = idx >= 0
    idx = idx.clamp(min=0)
    tv = (s["values"] / t).masked_fill(~listed_, -math.inf)
    lse = s["lse"][:, None] if s["tail"] else torch.logsumexp(tv, 1, keepdim=True)
    q = torch.exp(tv - lse).masked_fill(~listed_, 0.0)
    loss = torch.where(q > 0, q * (tv - lse - logp.gather(1, idx)), torch.zeros_like(q)).sum(1)
    inside = torch.zeros_like(ok).scatter_(1, torch.where(listed_, idx, idx[:, :1]), True) & ok
    rest_q = (1.0 - q.double().sum(1)).clamp(min=0.0).float() if s["tail"] else torch.zeros(rows, device=DEV)
    rest_p = (e.double() * ~inside).sum(1) / total[:, 0]
    rest = torch.where(rest_q > 0, rest_q * (torch.log(rest_q) - torch.log(rest_p)).float(), torch.zeros_like(rest_q))
    live = ok.any(1) & listed_.any(1)
    scale = t * t * (torch.ones(rows, device=DEV) if s["weight"] is None else s["weight"])
    # a student without a place outside the listed ones has no rest to learn
    has_rest = rest_p > 0
    loss = torch.where(live, scale * (loss + torch.where(has_rest, rest, torch.zeros_like(rest))), torch.zeros_like(loss))
    if not with_grad:
        return loss, None
    full = q.sum(1, keepdim=True) + torch.where(has_rest, rest_q, torch.zeros_like(rest_q))[:, None]
    outside = torch.where(has_rest, rest_q / rest_p.float().clamp(min=1e-38), torch.zeros_like(rest_q))[:, None]
    grad = p * (full - torch.where(inside, torch.zeros_like(p), outside))
    grad = grad.scatter_add(1, idx, -q)
    grad = torch.where(live[:, None] & ok, grad, torch.zeros_like(grad)) * (scale / t)[:, None]
    return loss, grad.to(s["logits"].dtype)


def _plain_scores(s):
    rows, width = s["rows"], s["width"]
    kind = s["row_kind"].long()[:, None].expand(rows, width)
    cls = s["classes_of"].long()[s["cand"].long()]
    out = s["table"].detach()[kind, cls]
    g = s["grad"].double()
    if s["counts"] is not None:
        off = torch.arange(width, device=DEV) >= s["counts"][:, None]
        out = out.masked_fill(off, -math.inf)
        g = g.masked_fill(off, 0.0)
    # per row first (rows have few classes), then per kind: no addition of millions of values to one address
    per_row = torch.stack([(g * (cls == c)).sum(1) for c in range(s["classes"])], dim=1)
    per_kind = torch.zeros(s["kinds"] + 1, s["classes"], dtype=torch.float64, device=DEV)
    upto = torch.cat([torch.zeros_like(per_row[:1]), per_row[s["by_kind"].long()].cumsum(0)])
    per_kind = upto[s["kind_start"].long()].diff(dim=0)
    return out, per_kind.float()


def run(s):
    if not own:
        if s["op"] == "sample":
            return _plain_sample(s)
        if s["op"] == "top":
            return _plain_top(s)
        if s["op"] == "distill":
            loss, grad = _plain_distill(s, s["way"] != "loss")
            return loss if s["way"] == "loss" else (loss, grad) if s["way"] == "step" else (loss.sum(), grad)
        return _plain_scores(s)
    from gan_amd import logits as L
    if s["op"] == "sample":
        return L.sample_rows(s["logits"], s["u"], counts=s["counts"], temperature=s["temperature"], top_k=s["top_k"],
                             top_p=s["top_p"], min_p=s["min_p"])
    if s["op"] == "top":
        return tuple(L.top_rows(s["logits"], s["m"], counts=s["counts"], temperature=s["temperature"]))
    if s["op"] == "distill":
        top = L.TopRows(s["values"], s["index"], s["lse"])
        kw = dict(counts=s["counts"], weight=s["weight"], temperature=s["temperature"], tail=s["tail"])
        if s["way"] == "loss":
            return L.distill_loss(s["logits"], top, reduction="none", **kw)
        if s["way"] == "step":
            return L.distill_loss_and_grad(s["logits"], top, **kw)
        s["logits"].grad = None
        loss = L.distill_loss(s["logits"], top, reduction="sum", **kw)
        loss.backward()
        return loss.detach(), s["logits"].grad
    s["table"].grad = None
    windows = L.ScoreWindows(s["cand"], s["counts"], s["classes_of"], s["row_kind"], s["by_kind"], s["kind_start"])
    out = L.class_scores(s["table"], windows)
    out.backward(s["grad"])
    return out.detach(), s["table"].grad


# ------------------------------------------------------------------ from the definitions, in 64 bits
def _exact_sample(s):
    """Row by row, as one would by hand."""
    rows, width, draws = s["rows"], s["width"], s["draws"]
    x = s["logits"].float().cpu().numpy().astype(np.float64)
    u = s["u"].cpu().numpy().astype(np.float64)
    counts = np.full(rows, width) if s["counts"] is None else s["counts"].cpu().numpy()
    sets = [s[k].float().cpu().numpy().astype(np.float64) if torch.is_tensor(s[k]) else np.full(rows, np.float64(np.float32(s[k])))
            for k in ("temperature", "top_k", "top_p", "min_p")]
    picks = np.full((rows, draws), -1, dtype=np.int32)
    for r in range(rows):
        temperature, top_k, top_p, min_p = (float(v[r]) for v in sets)
        at = np.arange(int(counts[r]))
        at = at[x[r, :counts[r]] > -np.inf]
        if not len(at):
            continue
        at = at[np.lexsort((at, -x[r, at]))]
        q = np.rint(np.exp((x[r, at] - x[r, at[0]]) / temperature) * UNIT)
        if top_k > 0:
            at, q = at[:int(top_k)], q[:int(top_k)]
        if top_p < 1:
            before = np.concatenate([[0.0], np.cumsum(q)[:-1]])
            n = max(1, int(np.searchsorted(before, top_p * q.sum(), side="left")))
            at, q = at[:n], q[:n]
        keep = q >= max(min(min_p, 1.0) * UNIT, 1.0)
        at, q = at[keep], q[keep]
        by_place = np.argsort(at)
        at, q = at[by_place], q[by_place]
        for d in range(min(draws, len(at))):
            j = int(np.searchsorted(np.cumsum(q), u[r, d] * q.sum(), side="right"))
            picks[r, d] = at[j]
            at, q = np.delete(at, j), np.delete(q, j)
    return torch.from_numpy(picks)


def _exact_top(s):
    rows, width, m = s["rows"], s["width"], s["m"]
    x = s["logits"].float().cpu().numpy().astype(np.float64)
    if s["counts"] is not None:
        x[np.arange(width)[None, :] >= s["counts"].cpu().numpy()[:, None]] = -np.inf
    at = np.argsort(-x, axis=1, kind="stable")[:, :m]
    v = np.take_along_axis(x, at, axis=1)
    top = x.max(axis=1)
    with np.errstate(divide="ignore"):
        lse = np.log(np.exp((x - np.where(np.isfinite(top), top, 0.0)[:, None]) / s["temperature"]).sum(axis=1)) + np.where(
            np.isfinite(top), top, 0.0) / s["temperature"]
    return torch.from_numpy(v), torch.from_numpy(np.where(np.isfinite(v), at, -1).astype(np.int32)), torch.from_numpy(lse)


def _exact_distill(s):
    """The loss as a function of the student's logits, and its gradient by differentiating that."""
    t, rows, width = s["temperature"], s["rows"], s["width"]
    x = s["logits"].detach().double().requires_grad_(True)
    place = torch.arange(width, device=DEV)
    count = torch.full((rows,), width, device=DEV) if s["counts"] is None else s["counts"].long()
    logp = torch.log_softmax((x / t).masked_fill(place >= count.clamp(min=1)[:, None], -math.inf), dim=1)
    has = (s["index"] >= 0)
    idx = s["index"].long().clamp(min=0)
    tv = torch.where(has, s["values"].double(), torch.zeros((), dtype=torch.float64, device=DEV)) / t
    tv = tv.masked_fill(~has, -1e300)
    logq = tv - (s["lse"].double()[:, None] if s["tail"] else torch.logsumexp(tv, 1, keepdim=True))
    q = torch.exp(logq) * has
    picked = torch.where(has, logp.gather(1, idx), torch.zeros_like(q))
    loss = torch.where(has, q * (logq - picked), torch.zeros_like(q)).sum(1)
    if s["tail"]:
        taken = torch.zeros(rows, width + 1, dtype=torch.bool, device=DEV)
        taken.scatter_(1, torch.where(has, idx, width), True)
        others = logp.masked_fill(taken[:, :width], -math.inf)
        alone = torch.isinf(others).all(1)
        rest_p = torch.logsumexp(torch.where(alone[:, None], torch.zeros_like(others), others), 1)
        rest_q = (1.0 - q.sum(1)).clamp(min=0.0)
        use = (rest_q > 0) & ~alone
        loss = loss + torch.where(use, rest_q * (torch.log(rest_q.clamp(min=1e-300)) - rest_p), torch.zeros_like(rest_q))
    scale = t * t * (1.0 if s["weight"] is None else s["weight"].double())
    loss = torch.where((count > 0) & has.any(1), scale * loss, torch.zeros_like(loss))
    if s["way"] == "loss":
        return loss.detach()
    grad, = torch.autograd.grad(loss.sum(), x)
    return (loss.detach(), grad) if s["way"] == "step" else (loss.detach().sum(), grad)


def _exact_scores(s):
    rows, width = s["rows"], s["width"]
    kind = s["row_kind"].cpu().numpy().astype(np.int64)
    cls = s["classes_of"].cpu().numpy()[s["cand"].cpu().numpy()].astype(np.int64)
    out = s["table"].detach().cpu().numpy().astype(np.float64)[kind[:, None], cls]
    pair = kind[:, None] * s["classes"] + cls
    g = s["grad"].cpu().numpy().astype(np.float64)
    if s["counts"] is not None:
        off = np.arange(width)[None, :] >= s["counts"].cpu().numpy()[:, None]
        out[off], g[off] = -np.inf, 0.0
    grad = np.bincount(pair.reshape(-1), weights=g.reshape(-1), minlength=s["kinds"] * s["classes"])
    return torch.from_numpy(out), torch.from_numpy(grad.reshape(s["kinds"], s["classes"]))


def exact(case, seed):
    if case["op"] == "sample" and (case["rows"] > 120000 or case["rows"] * case["width"] > 30_000_000):
        return None
    s = prepare(case, seed)
    return {"sample": _exact_sample, "top": _exact_top, "distill": _exact_distill, "scores": _exact_scores}[case["op"]](s)

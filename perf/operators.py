"""What the loss operators are measured on: log-probabilities of chosen classes with their backward pass, the
clipped policy loss, and the preference loss, over the range of sizes that tree ensembles (few classes, many rows)
and token models (many classes, fewer rows) give them.

A case is a dict of plain values:
  op        "log_prob" | "log_prob_grad" | "policy" | "preference" (consecutive segments) | "pairs" (any pairs of
            rows) | "preference_step" (log_prob, preference, log_prob_grad in turn: one training step on the margins)
  dtype     the margins' type: "float32", "float16", "bfloat16"
  rows, classes, pad   margins [rows][classes] whose rows are classes + pad apart
  ignored   share of the rows that have no label (prompt or padding positions)
  hess      whether the diagonal curvature is asked for, as a boosting round does
  pairs     number of pairs; for segments the rows are split over 2 * pairs of them by random lengths
  ref, weight, smoothing   whether there is a reference model / a weight per pair or row; the label smoothing
"""
import math

import numpy as np
import torch

own = False

CLIP = (0.2, 0.3)
KL = 0.05
BETA = 0.3
TYPES = {"float32": 4, "float16": 2, "bfloat16": 2}


def _case(name, op, dtype="float32", rows=1, classes=1, pad=0, ignored=0.0, hess=False, pairs=0, ref=True, weight=False,
          smoothing=0.0):
    c = {"op": op, "dtype": dtype, "rows": rows, "classes": classes, "pad": pad, "ignored": ignored, "hess": hess,
         "pairs": pairs, "ref": ref, "weight": weight, "smoothing": smoothing}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # scoring one decision of a token model: latency, one long row
        _case("log_prob one row", "log_prob", "bfloat16", 1, 50000),
        # scoring every row of a ten-class table (60,000 x 10 is the framework's multi-class configuration)
        _case("log_prob 60k x 10", "log_prob", "float32", 60000, 10),
        # scoring a packed batch of sequences; odd class count, so no row but the first starts on 16 bytes
        _case("log_prob 4096 x 65537", "log_prob", "bfloat16", 4096, 65537, ignored=0.1),
        # backward of the score for a boosting round on a ten-class table
        _case("grad 60k x 10 + hess", "log_prob_grad", "float32", 60000, 10, hess=True),
        # backward of a packed batch, a quarter of it prompt
        _case("grad 4096 x 65536", "log_prob_grad", "bfloat16", 4096, 65536, ignored=0.25),
        # one policy step of a handful of decisions: latency
        _case("policy 64 x 1000", "policy", "float16", 64, 1000, pad=8, ignored=0.1),
        # policy round of a tree ensemble over 10M rows (the framework's largest table) with four actions
        _case("policy 10M x 4 + hess", "policy", "float32", 10_000_000, 4, hess=True),
        # policy step of a token model over a packed batch
        _case("policy 8192 x 65536", "policy", "bfloat16", 8192, 65536, ignored=0.25, weight=True),
        # a small batch of paired sequences: latency
        _case("preference 16 pairs", "preference", rows=9001, pairs=16, smoothing=0.1),
        # paired single rows: a reward model on 1M comparisons
        _case("preference 1M pairs", "preference", rows=2_000_000, pairs=1_000_000, ref=False, hess=True),
        # ranking: rows compared with many others
        _case("pairs 8M over 1M rows", "pairs", rows=1_000_000, pairs=8_000_000, ref=False, weight=True, hess=True),
        # one whole training step on paired sequences
        _case("preference step", "preference_step", "bfloat16", 3000, 100_003, ignored=0.3, pairs=24),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["log_prob", "log_prob_grad", "policy", "preference", "pairs", "preference_step"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    ref, weight = rng.random() < 0.5, rng.random() < 0.5
    smoothing = rng.choice([0.0, 0.1])
    if op == "preference":
        pairs = _log(rng, 1, 1_000_000)
        return _case(None, op, "float32", 2 * pairs if rng.random() < 0.3 else _log(rng, pairs, 4_000_000) + 1, 1,
                     hess=rng.random() < 0.5, pairs=pairs, ref=ref, weight=weight, smoothing=smoothing)
    if op == "pairs":
        return _case(None, op, "float32", _log(rng, 2, 4_000_000), 1, hess=rng.random() < 0.5,
                     pairs=_log(rng, 1, 8_000_000), ref=ref, weight=weight, smoothing=smoothing)
    classes = _log(rng, 2, 131072)
    hess = op != "preference_step" and dtype == "float32" and rng.random() < 0.5
    most = (1 << 27) // (2 if dtype == "float32" else 1) // (2 if hess else 1)
    rows = _log(rng, 1, min(10_000_000, max(1, most // classes)))
    if op == "preference_step":
        rows, ref = max(rows, 8), True
    return _case(None, op, dtype, rows, classes, pad=rng.choice([0, 0, 1, 8]), ignored=rng.choice([0.0, 0.1, 0.3]),
                 hess=hess, pairs=rng.randint(1, max(1, min(64, rows // 2))) if op == "preference_step" else 0, ref=ref,
                 weight=weight, smoothing=smoothing)


# ---------------------------------------------------------------- inputs

def _segments(rows, pairs, gen):
    """Offsets of 2 * pairs segments over all rows; single rows where there are just as many."""
    if rows == 2 * pairs:
        return torch.arange(rows + 1, dtype=torch.int64, device="cuda")
    cut = torch.randint(0, rows + 1, (2 * pairs - 1,), generator=gen, device="cuda").sort().values
    zero = torch.zeros(1, dtype=torch.int64, device="cuda")
    return torch.cat([zero, cut, zero + rows])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, classes, pairs = case["rows"], case["classes"], case["pairs"]
    normal = lambda *n, sd=1.0: torch.randn(*n, generator=gen, device="cuda") * sd  # noqa: E731
    s = dict(case)
    if case["op"] in ("preference", "pairs"):
        # log-probabilities of short answers, or scores of single rows, and those of the model it started from
        s["score"] = normal(rows, sd=2.0)
        s["ref_score"] = s["score"] + normal(rows, sd=0.5) if case["ref"] else None
    else:
        z = torch.randn(rows, classes + case["pad"], generator=gen, device="cuda", dtype=getattr(torch, case["dtype"]))
        z *= 2.0
        s["margin"] = z[:, :classes]
        label = torch.randint(0, classes, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        s["label"] = torch.where(torch.rand(rows, generator=gen, device="cuda") < case["ignored"], -1, label).int()
        if case["op"] != "log_prob":
            logp, s["norm"] = _log_prob(s["margin"], s["label"])
        if case["op"] == "log_prob_grad":
            s["weight"] = normal(rows)
        if case["op"] == "policy":
            s["old"] = logp + normal(rows, sd=0.2)
            s["ref_logp"] = logp + normal(rows, sd=0.5) if case["ref"] else None
            s["advantage"] = normal(rows)
            s["weight"] = torch.rand(rows, generator=gen, device="cuda") if case["weight"] else None
        if case["op"] == "preference_step":
            s["ref_score"] = logp + normal(rows, sd=0.05) if case["ref"] else None
    if case["op"] in ("preference", "preference_step"):
        s["begin"] = None if rows == 2 * pairs else _segments(rows, pairs, gen)
        s["offsets"] = _segments(rows, pairs, gen) if s["begin"] is None else s["begin"]
    if case["op"] == "pairs":
        a = torch.randint(0, rows, (pairs,), generator=gen, device="cuda")
        b = (a + torch.randint(1, rows, (pairs,), generator=gen, device="cuda")) % rows
        s["pairs_list"] = torch.stack([a, b], 1).int()
    if case["op"] in ("preference", "pairs", "preference_step"):
        s["pair_weight"] = torch.rand(pairs, generator=gen, device="cuda") + 0.5 if case["weight"] else None
    if own and case["op"] == "pairs":
        # the pairs of a training set stay the same from round to round: the program keeps their plan
        s["plan"] = _dp().PreferencePairs(s["pairs_list"], rows)
    return s


# ---------------------------------------------------------------- one pass

def _dp():
    import pathlib
    import sys
    at = str(pathlib.Path(__file__).resolve().parents[1] / "decision-programs_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import dp_gbdt
    return dp_gbdt


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    dp, op = _dp(), s["op"]
    if op == "log_prob":
        logp, norm = dp.log_prob(s["margin"], s["label"])
        return {"log_prob": logp, "norm": norm}
    if op == "log_prob_grad":
        grad, hess = dp.log_prob_grad(s["margin"], s["label"], s["norm"], s["weight"], hess=s["hess"])
        return {"grad": grad, "hess": hess}
    if op == "policy":
        r = dp.policy_loss(s["margin"], s["label"], s["old"], s["advantage"], ref_log_prob=s["ref_logp"],
                           weight=s["weight"], clip=CLIP, kl=KL, hess=s["hess"])
        return {"loss": r.loss, "log_prob": r.log_prob, "grad": r.grad, "hess": r.hess}
    if op == "pairs":
        r = s["plan"].loss(s["score"], ref_score=s["ref_score"], weight=s["pair_weight"], beta=BETA,
                           smoothing=s["smoothing"], hess=s["hess"])
        return {"loss": r.loss, "grad": r.grad, "hess": r.hess}
    if op == "preference":
        r = dp.preference_loss(s["score"], ref_score=s["ref_score"], item_begin=s["begin"], weight=s["pair_weight"],
                               beta=BETA, smoothing=s["smoothing"], hess=s["hess"])
        return {"loss": r.loss, "grad": r.grad, "hess": r.hess}
    logp, norm = dp.log_prob(s["margin"], s["label"])
    r = dp.preference_loss(logp, ref_score=s["ref_score"], item_begin=s["begin"], weight=s["pair_weight"], beta=BETA,
                           smoothing=s["smoothing"])
    grad, _ = dp.log_prob_grad(s["margin"], s["label"], norm, r.grad)
    return {"log_prob": logp, "loss": r.loss, "grad": grad}


def _run_plain(s):
    op = s["op"]
    if op == "log_prob":
        logp, norm = _log_prob(s["margin"], s["label"])
        return {"log_prob": logp, "norm": norm}
    if op == "log_prob_grad":
        grad, hess = _log_prob_grad(s["margin"], s["label"], s["norm"], s["weight"], s["hess"])
        return {"grad": grad, "hess": hess}
    if op == "policy":
        return _policy(s)
    if op in ("preference", "pairs"):
        return _preference(s, s["score"])
    logp, norm = _log_prob(s["margin"], s["label"])
    r = _preference(s, logp)
    grad, _ = _log_prob_grad(s["margin"], s["label"], norm, r["grad"], False)
    return {"log_prob": logp, "loss": r["loss"], "grad": grad}


# ---------------------------------------------------------------- plain forms, in 32 bits

def _log_prob(margin, label):
    z = margin.float()
    kept = (label >= 0) & (label < z.shape[1])
    top = z.max(1).values
    log_sum = (z - top[:, None]).exp().sum(1).log()
    chosen = z.gather(1, torch.where(kept, label, 0).long()[:, None])[:, 0]
    logp = torch.where(kept, (chosen - top) - log_sum, 0.0)
    return logp, torch.where(kept[:, None], torch.stack([top, log_sum], 1), 0.0)


def _log_prob_grad(margin, label, norm, weight, hess):
    z = margin.float()
    kept = (label >= 0) & (label < z.shape[1])
    c = torch.where(kept, weight, 0.0)
    p = ((z - norm[:, :1]) - norm[:, 1:]).exp()
    del z
    h = c.abs()[:, None] * (2.0 * p * (1.0 - p)).clamp_min(1e-16) if hess else None
    g = p.mul_(-c[:, None])
    g.scatter_add_(1, torch.where(kept, label, 0).long()[:, None], c[:, None])
    g = torch.where(kept[:, None], g, 0.0)
    return g.to(margin.dtype), h


def _policy(s):
    label = s["label"]
    logp, norm = _log_prob(s["margin"], label)
    kept = label >= 0
    w = torch.where(kept, 1.0 if s["weight"] is None else s["weight"], 0.0)
    ratio = (logp - s["old"]).exp()
    free = ratio * s["advantage"]
    held = ratio.clamp(1.0 - CLIP[0], 1.0 + CLIP[1]) * s["advantage"]
    loss = -torch.minimum(free, held)
    c = torch.where(free <= held, -free, 0.0)
    if s["ref_logp"] is not None:
        d = s["ref_logp"] - logp
        loss = loss + KL * (d.exp() - d - 1.0)
        c = c + KL * (1.0 - d.exp())
    grad, hess = _log_prob_grad(s["margin"], label, norm, c * w, s["hess"])
    return {"loss": loss * w, "log_prob": logp, "grad": grad, "hess": hess}


def _preference(s, score):
    eps = s["smoothing"]
    gap = score if s["ref_score"] is None else score - s["ref_score"]
    if s["op"] == "pairs":
        a, b = s["pairs_list"][:, 0].long(), s["pairs_list"][:, 1].long()
        total = gap
    else:
        at = s["offsets"]
        item = torch.repeat_interleave(torch.arange(at.numel() - 1, device=gap.device), at.diff(), output_size=gap.numel())
        total = torch.zeros(at.numel() - 1, device=gap.device).index_add_(0, item, gap)
        a = torch.arange(0, at.numel() - 1, 2, device=gap.device)
        b = a + 1
    x = BETA * (total[a] - total[b])
    small = (-x.abs()).exp().log1p()
    loss = (1.0 - eps) * ((-x).clamp_min(0.0) + small) + eps * (x.clamp_min(0.0) + small)
    up, down = 1.0 / (1.0 + (-x).exp()), 1.0 / (1.0 + x.exp())
    slope = BETA * (eps * up - (1.0 - eps) * down)
    bend = BETA * BETA * up * down
    if s["pair_weight"] is not None:
        loss, slope, bend = loss * s["pair_weight"], slope * s["pair_weight"], bend * s["pair_weight"]
    spread = lambda u, v: torch.zeros_like(total).index_add_(0, a, u).index_add_(0, b, v)  # noqa: E731
    grad = spread(slope, -slope)
    hess = spread(bend, bend).clamp_min(1e-16) if s["hess"] else None
    if s["op"] != "pairs":
        grad, hess = grad[item], None if hess is None else hess[item]
    return {"loss": loss, "grad": grad, "hess": hess}


# ---------------------------------------------------------------- cost

def work(case):
    """Rows without a label are not read; their gradient is written all the same."""
    size, rows, classes, pairs = TYPES[case["dtype"]], case["rows"], case["classes"], case["pairs"]
    read = rows * (1.0 - case["ignored"]) * classes * size
    made = rows * classes * (size + (4 if case["hess"] else 0))
    ref, weight = 4 * case["ref"], 4 * case["weight"]
    each = rows * classes
    if case["op"] == "log_prob":
        return {"bytes": read + 16 * rows, "flops": 4 * each}
    if case["op"] == "log_prob_grad":
        return {"bytes": read + 16 * rows + made, "flops": 5 * each}
    if case["op"] == "policy":
        return {"bytes": read + made + rows * (20 + ref + weight), "flops": 8 * each}
    scores = rows * (4 + ref + 4 + 4 * case["hess"]) + pairs * (4 + weight)
    if case["op"] == "preference":
        return {"bytes": scores + (0 if rows == 2 * pairs else 16 * pairs), "flops": 2 * rows + 20 * pairs}
    if case["op"] == "pairs":
        return {"bytes": scores + 8 * pairs, "flops": 24 * pairs}
    # the margins are read for the scores, and again for the gradient once the whole segment's sum is known
    return {"bytes": 2 * read + made + rows * (24 + ref) + pairs * (20 + weight), "flops": 10 * each}


# ---------------------------------------------------------------- the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op, eps = case["op"], case["smoothing"]

    def softmax_rows(coefficient=None):
        """log p of each row's label and (max, log sum); with a coefficient per row, the gradient and curvature of
        its product with log p, a slab of rows at a time."""
        z16, y = s["margin"], s["label"].long()
        rows, classes = z16.shape
        step = max(1, (1 << 26) // classes)
        lp, nm, gr, hs = [], [], [], []
        for r in range(0, rows, step):
            z, lab = z16[r:r + step].double(), y[r:r + step]
            live = (lab >= 0).double()
            top = z.amax(1)
            lse = torch.logsumexp(z, 1)
            hit = torch.nn.functional.one_hot(lab.clamp_min(0), classes).bool() if classes <= 64 else None
            picked = z[torch.arange(len(z), device=z.device), lab.clamp_min(0)]
            lp.append((picked - lse) * live)
            nm.append(torch.stack([top, lse - top], 1) * live[:, None])
            if coefficient is not None:
                c = (coefficient[r:r + step].double() * live)[:, None]
                p = torch.softmax(z, 1)
                if hess:
                    hs.append(c.abs() * torch.clamp(2 * p * (1 - p), min=1e-16))
                g = -c * p
                if hit is not None:
                    g = g + c * hit
                else:
                    g[torch.arange(len(z), device=z.device), lab.clamp_min(0)] += c[:, 0]
                gr.append(g)
        whole = lambda v: torch.cat(v) if v else None  # noqa: E731
        return whole(lp), whole(nm), whole(gr), whole(hs)

    def preferred(score):
        f64 = lambda t: t.double().cpu().numpy()  # noqa: E731
        v = f64(score) - (f64(s["ref_score"]) if s["ref_score"] is not None else 0.0)
        if op == "pairs":
            left, right = s["pairs_list"].long().cpu().numpy().T
        else:
            at = s["offsets"].cpu().numpy()
            run = np.concatenate([[0.0], np.cumsum(v)])
            lengths = np.diff(at)
            v = run[at[1:]] - run[at[:-1]]
            left, right = np.arange(0, len(v), 2), np.arange(1, len(v), 2)
        w = f64(s["pair_weight"]) if s["pair_weight"] is not None else np.ones(len(left))
        x = BETA * (v[left] - v[right])
        loss = w * ((1 - eps) * np.logaddexp(0, -x) + eps * np.logaddexp(0, x))
        sig = 0.5 * (1 + np.tanh(x / 2))
        q = w * BETA * ((sig - 1) + eps)
        q = np.where(x > 30, w * BETA * (eps - np.exp(-x)), q)
        k = w * BETA ** 2 / (4 * np.cosh(np.clip(x / 2, -300, 300)) ** 2)
        g = np.bincount(left, q, len(v)) - np.bincount(right, q, len(v))
        h = np.maximum(np.bincount(left, k, len(v)) + np.bincount(right, k, len(v)), 1e-16)
        if op != "pairs":
            g, h = np.repeat(g, lengths), np.repeat(h, lengths)
        give = lambda t: torch.from_numpy(t).cuda()  # noqa: E731
        return give(loss), give(g), give(h) if case["hess"] else None

    hess = case["hess"]
    if op == "log_prob":
        lp, nm, _, _ = softmax_rows()
        return {"log_prob": lp, "norm": nm}
    if op == "log_prob_grad":
        # the norm is an input here: its own rounding is not the operator's
        _, _, g, h = softmax_rows(s["weight"])
        return {"grad": g, "hess": h}
    if op == "policy":
        lp, _, _, _ = softmax_rows()
        live = (s["label"] >= 0).double()
        w = live if s["weight"] is None else live * s["weight"].double()
        r, adv = torch.exp(lp - s["old"].double()), s["advantage"].double()
        bounded = torch.clamp(r, 1 - CLIP[0], 1 + CLIP[1])
        through = torch.where(adv >= 0, r <= 1 + CLIP[1], r >= 1 - CLIP[0])
        loss, c = -torch.minimum(r * adv, bounded * adv), -(r * adv) * through
        if s["ref_logp"] is not None:
            d = s["ref_logp"].double() - lp
            loss, c = loss + KL * (torch.expm1(d) - d), c - KL * torch.expm1(d)
        _, _, g, h = softmax_rows(c * w)
        return {"loss": loss * w, "log_prob": lp, "grad": g, "hess": h}
    if op in ("preference", "pairs"):
        loss, g, h = preferred(s["score"])
        return {"loss": loss, "grad": g, "hess": h}
    lp, _, _, _ = softmax_rows()
    loss, q, _ = preferred(lp)
    _, _, g, _ = softmax_rows(q)
    return {"log_prob": lp, "loss": loss, "grad": g}

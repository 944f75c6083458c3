"""Alternatives of class scores and distillation from them, as measurable cases.

Four kinds of call:

* ``alternatives``       log-probability of each row's label, the entropy, and the best k classes
                         with their log-probabilities (``class_alternatives``);
* ``alternatives_grad``  the gradient of what a training step makes of these
                         (``class_alternatives_grad``);
* ``distill``            divergence of the scores from a teacher's listed classes, with the
                         gradient (``distill_loss``);
* ``teach``              one after the other, as a student learns: the teacher's alternatives, the
                         divergence from them, and the labels' own log-probabilities, whose
                         gradient is added.

``own`` chooses between the plain forms (torch, elementary operations) and the package's entry
points; ``exact`` computes the same outputs from the definitions in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
F32, F64 = torch.float32, torch.float64
TYPES = dict(float32=torch.float32, bfloat16=torch.bfloat16, float16=torch.float16)
SIZES = dict(float32=4, bfloat16=2, float16=2)
LABEL = 0.3                 # weight of the labels next to the teacher
LEAST = 2.0 ** -20          # a teacher's rest below this is rounding of its log-probabilities


# --------------------------------------------------------------------------- the cases
def listed():
    return [
        # one decision answered, with its twenty best alternatives
        dict(name="alternatives one row", kind="alternatives", rows=1, classes=50_001, top=20,
             dtype="float32", major="row", masked=0.0, temperature=1.0),
        # the decisions logged with a class forest's table, scores class by class as the engine
        # keeps them, the three best classes of ten
        dict(name="alternatives class forest", kind="alternatives", rows=1_000_000, classes=10,
             top=3, dtype="float32", major="class", masked=0.0, temperature=1.0),
        # few hundred classes, odd sizes, half precision
        dict(name="alternatives odd", kind="alternatives", rows=20_047, classes=257, top=8,
             dtype="float16", major="row", masked=0.1, temperature=1.0),
        # a teacher's lists over a large set of classes, softened
        dict(name="alternatives many classes", kind="alternatives", rows=8_191, classes=16_001,
             top=64, dtype="bfloat16", major="row", masked=0.0, temperature=2.0),
        # an entropy bonus for a gate's scores
        dict(name="alternatives grad gate", kind="alternatives_grad", rows=65_536, classes=64,
             top=0, dtype="bfloat16", major="row", masked=0.0, temperature=1.0),
        # a training step on log-probabilities of twenty alternatives, the label and the entropy
        dict(name="alternatives grad many classes", kind="alternatives_grad", rows=4_099,
             classes=32_000, top=20, dtype="bfloat16", major="row", masked=0.0, temperature=1.0),
        # a small batch: launches and the call count
        dict(name="distill small batch", kind="distill", rows=256, classes=1_000, top=10,
             dtype="float32", major="row", masked=0.0, temperature=1.0, rest=False),
        # a student forest's round: every row's four best classes of ten, and the rest
        dict(name="distill class forest", kind="distill", rows=1_000_000, classes=10, top=4,
             dtype="float32", major="class", masked=0.0, temperature=1.0, rest=True),
        # the largest: a forest of a hundred classes, sixteen of them listed, softened
        dict(name="distill hundred classes", kind="distill", rows=1_000_000, classes=100, top=16,
             dtype="float32", major="class", masked=0.0, temperature=2.0, rest=True),
        # long lists over a large set of classes
        dict(name="distill many classes", kind="distill", rows=8_191, classes=16_001, top=64,
             dtype="bfloat16", major="row", masked=0.0, temperature=1.0, rest=True),
        # few hundred classes, some not allowed to the student, lists without their rest
        dict(name="distill odd", kind="distill", rows=20_047, classes=257, top=8,
             dtype="float16", major="row", masked=0.1, temperature=3.0, rest=False),
        # a small table's round with its labels
        dict(name="teach small", kind="teach", rows=10_000, classes=33, top=5, dtype="float32",
             major="class", masked=0.0, temperature=2.0),
    ]


BYTES = 780_000_000  # of the scores and gradients of the largest drawn case
MATRICES = dict(alternatives=1, alternatives_grad=2, distill=2, teach=5)


def _log(rng, lo, hi):
    """A whole number whose logarithm is uniform between those of lo and hi."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["alternatives", "alternatives", "alternatives_grad", "distill", "distill",
                       "distill", "teach"])
    dtype = rng.choice(["float32", "float32", "bfloat16", "float16"])
    major = rng.choice(["row", "class"])
    classes = _log(rng, 2, 65_537)
    cells = min(131_000_000, BYTES // MATRICES[kind] // SIZES[dtype])
    # (a single confident row's gradient is a difference of nearly equal numbers in any form)
    rows = _log(rng, 1 if kind == "alternatives" else 20, max(20, min(1_000_000, cells // classes)))
    # (a list of all classes and rows of one say nothing of a teacher)
    top = _log(rng, 1, max(1, min(64, classes // 2)))
    if kind == "alternatives_grad" and rng.random() < 0.3:
        top = 0
    case = dict(kind=kind, rows=rows, classes=classes, top=top, dtype=dtype, major=major,
                masked=rng.choice([0.0, 0.0, 0.2]), temperature=rng.choice([1.0, 1.0, 0.7, 2.0, 4.0]))
    if kind == "distill":
        case["rest"] = rng.random() < 0.5
    return case


# --------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1_000_003 * int(seed) + 31)
    return g


def _normal(shape, g):
    return torch.randn(shape, generator=g, device=DEV)


def _scale(case):
    """Gradients in float16 need a loss scale, or they fall below its smallest normal number."""
    return 1024.0 if case["dtype"] == "float16" else 1.0


def _inputs(case, seed):
    """Scores [rows, classes] as a forest or a gate gives them (a spread of a few units, some
    classes liked more), and what the kind of call takes beside them."""
    g = _gen(seed)
    kind, n, K, k = case["kind"], case["rows"], case["classes"], case["top"]
    by_class = case["major"] == "class"
    shape = (K, n) if by_class else (n, K)
    dim = 0 if by_class else 1
    lean = _normal((K, 1) if by_class else (1, K), g)
    scores = 1.5 * _normal(shape, g) + lean
    teacher = None
    if kind in ("distill", "teach"):
        # (a student at the start of its training)
        teacher = 0.8 * scores + _normal(shape, g)
    if case["masked"]:
        # classes that a row may not take; its best class always stays
        shut = torch.rand(shape, generator=g, device=DEV) < case["masked"]
        best = scores.argmax(dim, keepdim=True)
        shut.scatter_(dim, best, False)
        scores.masked_fill_(shut, -math.inf)
        del shut
    scores = scores.to(TYPES[case["dtype"]])
    noise = torch.rand(shape, generator=g, device=DEV).clamp_(1e-7, 1 - 1e-7).log_().neg_().log_()
    taken = noise.neg_().add_(scores).argmax(dim).to(torch.int32)
    del noise
    d = dict(scores=scores.t() if by_class else scores)
    if kind != "distill":
        d["labels"] = taken
    live = (torch.rand(n, generator=g, device=DEV) >= 0.1).to(F32)
    weight = live * (0.5 + torch.rand(n, generator=g, device=DEV)) * _scale(case)
    if kind == "alternatives_grad":
        d["grad_label"] = weight * _normal((n,), g)
        d["grad_entropy"] = weight * _normal((n,), g)
        if k:
            best = _ordered(d["scores"], k)
            d["classes"] = best[1]
            d["grad_top"] = weight[:, None] * _normal((n, k), g)
    if kind in ("distill", "teach"):
        d["weight"] = weight
    if kind == "distill":
        # what a teacher left: its best classes, a fifth of the rows with fewer of them (-1)
        logits, classes = torch.topk(teacher, k, dim=dim)
        if by_class:
            logits, classes = logits.t(), classes.t()
        cut = torch.where(torch.rand(n, generator=g, device=DEV) < 0.2,
                          torch.randint(1, k + 1, (n,), generator=g, device=DEV), k)
        gone = torch.arange(k, device=DEV)[None, :] >= cut[:, None]
        d["classes"] = classes.masked_fill(gone, -1).to(torch.int32).contiguous()
        d["logits"] = logits.masked_fill(gone, 0.0).contiguous()
        if case["rest"]:
            d["log_norm"] = torch.logsumexp(teacher / case["temperature"], dim)
    if kind == "teach":
        d["teacher"] = teacher.to(scores.dtype)
        if by_class:
            d["teacher"] = d["teacher"].t()
        d["grad_label"] = -LABEL * weight
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    d["case"] = case
    if case["kind"] == "alternatives_grad":
        # what the forward pass left
        d["norm"] = _norm(d["scores"], case["temperature"], F64).to(F32)
    return d


# --------------------------------------------------------------------------- the plain forms
def _norm(scores, tau, dtype=F32):
    """Per row: the largest score, log(sum exp((s - max) / tau)), mean of (max - s) / tau."""
    s = scores.to(dtype)
    top = s.amax(1)
    x = (s - top[:, None]) / tau
    e = torch.exp(x)
    z = e.sum(1)
    down = torch.where(e > 0, -x * e, 0.0).sum(1) / z
    return torch.stack([top, z.log(), down], 1)


def _ordered(scores, k):
    """The k best scores of each row and their classes, the lower class first among equals; -1
    where a row has fewer classes."""
    best, at = torch.sort(scores.float(), dim=1, descending=True, stable=True)
    best, at = best[:, :k], at[:, :k]
    return best, torch.where(best > -math.inf, at, -1).to(torch.int32)


def _alternatives(scores, labels, k, tau):
    norm = _norm(scores, tau)
    best, classes = _ordered(scores, k)
    log_prob = (best - norm[:, :1]) / tau - norm[:, 1:2]
    label = scores.float().gather(1, labels.long()[:, None])[:, 0]
    return dict(classes=classes, log_prob=log_prob, entropy=norm[:, 1] + norm[:, 2],
                label_log_prob=(label - norm[:, 0]) / tau - norm[:, 1], norm=norm)


def _alternatives_grad(d, norm, tau):
    s = d["scores"].float()
    x = (s - norm[:, :1]) / tau
    p = torch.exp(x - norm[:, 1:2])
    whole = d["grad_label"]
    if "grad_top" in d:
        whole = whole + d["grad_top"].sum(1)
    slope = whole[:, None]
    if "grad_entropy" in d:
        slope = slope + d["grad_entropy"][:, None] * torch.where(p > 0, x + norm[:, 2:], 0.0)
    out = -p * slope
    out.scatter_add_(1, d["labels"].long()[:, None], d["grad_label"][:, None])
    if "grad_top" in d:
        out.scatter_add_(1, d["classes"].clamp(min=0).long(),
                         torch.where(d["classes"] >= 0, d["grad_top"], 0.0))
    return out / tau


def _distill(scores, classes, logits, log_norm, weight, tau):
    # the divergence is a small difference of large logarithms: in 64 bits
    x = scores.double() / tau
    n, K = x.shape
    used = (classes >= 0) & (classes < K)
    at = torch.where(used, classes, 0).long()
    top = x.amax(1, keepdim=True)
    logp = x - top - torch.exp(x - top).sum(1, keepdim=True).log()
    del x
    # the classes that are not listed, together
    seen = torch.zeros((n, K + 1), dtype=torch.bool, device=logp.device)
    seen.scatter_(1, torch.where(used, classes, K).long(), True)
    others = logp.masked_fill(seen[:, :K], -math.inf)
    most = others.amax(1, keepdim=True).clamp(min=-1e30)
    spread = torch.exp(others - most).sum(1, keepdim=True)
    log_rest = most[:, 0] + spread[:, 0].log()
    lp = logp.gather(1, at)
    counts = used & (lp > -math.inf)
    lq = logits.double() / tau
    if log_norm is None:
        rest = torch.zeros(n, dtype=F64, device=logp.device)
        lq = lq - lq.masked_fill(~counts, -math.inf).amax(1, keepdim=True)
    else:
        lq = lq - log_norm.double()[:, None]
        rest = 1.0 - torch.where(used, torch.exp(lq), 0.0).sum(1)
        rest = torch.where((rest >= LEAST) & (log_rest > -math.inf), rest, 0.0)
    mass = torch.where(counts, torch.exp(lq), 0.0).sum(1) + rest
    live = (weight != 0) & (mass > 0)
    mass = torch.where(live, mass, 1.0)
    lq, rest = lq - mass.log()[:, None], rest / mass
    q = torch.where(counts, torch.exp(lq), 0.0)
    loss = torch.where(q > 0, q * (lq - lp), 0.0).sum(1)
    loss = loss + torch.where(rest > 0, rest * (rest.log() - log_rest), 0.0)
    part = torch.where(rest > 0, rest / spread[:, 0], 0.0)
    grad = (torch.exp(logp) - torch.exp(others - most) * part[:, None]).float()
    grad.scatter_add_(1, at, -q.float())
    grad = torch.where(live[:, None], grad * (weight * tau)[:, None], 0.0)
    return torch.where(live, loss * weight * tau * tau, 0.0).float(), grad


def _run_plain(d):
    case = d["case"]
    kind, tau, dtype = case["kind"], case["temperature"], d["scores"].dtype
    if kind == "alternatives":
        return _alternatives(d["scores"], d["labels"], case["top"], tau)
    if kind == "alternatives_grad":
        return dict(grad=_alternatives_grad(d, d["norm"], tau).to(dtype))
    if kind == "distill":
        loss, grad = _distill(d["scores"], d["classes"], d["logits"], d.get("log_norm"),
                              d["weight"], tau)
        return dict(loss=loss, grad=grad.to(dtype))
    t = _alternatives(d["teacher"], d["labels"], case["top"], tau)
    loss, grad = _distill(d["scores"], t["classes"], t["log_prob"] * tau,
                          torch.zeros_like(t["entropy"]), d["weight"], tau)
    norm = _norm(d["scores"], 1.0)
    label = d["scores"].float().gather(1, d["labels"].long()[:, None])[:, 0]
    grad = grad + _alternatives_grad(dict(scores=d["scores"], labels=d["labels"],
                                          grad_label=d["grad_label"]), norm, 1.0)
    return dict(classes=t["classes"], log_prob=t["log_prob"], entropy=t["entropy"], loss=loss,
                label_log_prob=label - norm[:, 0] - norm[:, 1], grad=grad.to(dtype))


# --------------------------------------------------------------------------- the package's calls
def _run_own(d):
    from warpgbm_amd import losses

    case = d["case"]
    kind, tau = case["kind"], case["temperature"]
    if kind == "alternatives":
        r = losses.class_alternatives(d["scores"], case["top"], labels=d["labels"], temperature=tau)
        return dict(classes=r.classes, log_prob=r.log_prob, entropy=r.entropy,
                    label_log_prob=r.label_log_prob, norm=r.norm)
    if kind == "alternatives_grad":
        return dict(grad=losses.class_alternatives_grad(
            d["scores"], d["norm"], labels=d["labels"], grad_label_log_prob=d["grad_label"],
            classes=d.get("classes"), grad_log_prob=d.get("grad_top"),
            grad_entropy=d["grad_entropy"], temperature=tau))
    if kind == "distill":
        r = losses.distill_loss(d["scores"], d["classes"], d["logits"], log_norm=d.get("log_norm"),
                                weight=d["weight"], temperature=tau)
        return dict(loss=r.loss, grad=r.grad)
    t = losses.class_alternatives(d["teacher"], case["top"], temperature=tau)
    r = losses.distill_loss(d["scores"], t.classes, t.log_prob * tau if tau != 1.0 else t.log_prob,
                            log_norm=0.0, weight=d["weight"], temperature=tau)
    f = losses.class_alternatives(d["scores"], 0, labels=d["labels"])
    grad = losses.class_alternatives_grad(d["scores"], f.norm, labels=d["labels"],
                                          grad_label_log_prob=d["grad_label"], grad=r.grad)
    return dict(classes=t.classes, log_prob=t.log_prob, entropy=t.entropy, loss=r.loss,
                label_log_prob=f.label_log_prob, grad=grad)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# --------------------------------------------------------------------------- work
def work(case):
    """Bytes: scores read once, gradients written once, the rows' and lists' numbers; operations:
    an exponential counted as one."""
    kind, n, K, k = case["kind"], case["rows"], case["classes"], case["top"]
    cells, es = n * K, SIZES[case["dtype"]]
    if kind == "alternatives":
        return dict(bytes=es * cells + 24 * n + 8 * n * k, flops=7 * cells)
    if kind == "alternatives_grad":
        return dict(bytes=2 * es * cells + 24 * n + 8 * n * k, flops=6 * cells)
    if kind == "distill":
        return dict(bytes=2 * es * cells + 8 * n + (4 * n if case["rest"] else 0) + 8 * n * k,
                    flops=7 * cells + 12 * n * k)
    return dict(bytes=3 * es * cells + 24 * n + 8 * n * k, flops=20 * cells + 12 * n * k)


# --------------------------------------------------------------------------- in 64 bits
def _logs64(scores, tau):
    return torch.log_softmax(scores.to(F64) / tau, 1)


def _exact_alternatives(scores, labels, k, tau):
    L = _logs64(scores, tau)
    rows = torch.arange(L.shape[0], device=DEV)
    order = torch.argsort(scores.to(F64), dim=1, descending=True, stable=True)[:, :k]
    top = L.gather(1, order)
    H = -torch.special.xlogy(L.exp(), L.exp()).sum(1)
    high = scores.to(F64).max(1).values
    lse = torch.logsumexp(scores.to(F64) / tau, 1) - high / tau
    return dict(classes=order.masked_fill(top == -math.inf, -1).to(torch.int32), log_prob=top,
                entropy=H, label_log_prob=L[rows, labels.long()],
                norm=torch.stack([high, lse, H - lse], 1))


def _exact_alternatives_grad(d, tau):
    """By automatic differentiation of what the upstream gradients weigh."""
    s = d["scores"].to(F64).requires_grad_(True)
    shut = d["scores"] == -math.inf
    L = torch.log_softmax(s / tau, 1)
    rows = torch.arange(s.shape[0], device=DEV)
    total = (d["grad_label"].to(F64) * L[rows, d["labels"].long()]).sum()
    safe = L.masked_fill(shut, 0.0)
    if "grad_entropy" in d:
        total = total - (d["grad_entropy"].to(F64) * (L.exp() * safe).sum(1)).sum()
    if "grad_top" in d:
        c = d["classes"].long()
        there = c >= 0
        total = total + (safe.gather(1, c.clamp(min=0)) * there * d["grad_top"].to(F64)).sum()
    (grad,) = torch.autograd.grad(total, s)
    return grad


def _exact_distill(d, classes, logits, log_norm, tau):
    """The teacher as a row of shares of every class and of the rest; the gradient by automatic
    differentiation."""
    K = d["scores"].shape[1]
    s = d["scores"].to(F64).requires_grad_(True)
    shut = d["scores"] == -math.inf
    L = torch.log_softmax(s / tau, 1)
    slot = classes.long().masked_fill((classes < 0) | (classes >= K), K)
    t = torch.full((s.shape[0], K + 1), -math.inf, dtype=F64, device=DEV)
    t.scatter_(1, slot, logits.to(F64) / tau)
    t, in_list = t[:, :K], torch.zeros_like(t, dtype=torch.bool).scatter_(1, slot, True)[:, :K]
    free = ~in_list & ~shut
    if log_norm is None:
        R = torch.zeros(s.shape[0], dtype=F64, device=DEV)
    else:
        t = t - log_norm.to(F64)[:, None]
        R = 1 - t.exp().sum(1)
        R = R.masked_fill((R < LEAST) | ~free.any(1), 0.0)
    t = t.masked_fill(shut, -math.inf)
    if log_norm is None:
        t = t - t.max(1, keepdim=True).values.clamp(min=-1e300)
    share = t.exp()
    whole = share.sum(1) + R
    on = (d["weight"] != 0) & (whole > 0)
    whole = whole.masked_fill(~on, 1.0)
    share, R = share / whole[:, None], R / whole
    logs = L.masked_fill(shut, 0.0)
    loss = torch.special.xlogy(share, share).sum(1) - (share * logs).sum(1)
    both = R > 0
    gather = torch.logsumexp(L.masked_fill(~free, -1e300), 1).masked_fill(~both, 0.0)
    loss = loss + torch.special.xlogy(R, R) - R * gather
    loss = (loss * d["weight"].to(F64) * tau * tau).masked_fill(~on, 0.0)
    (grad,) = torch.autograd.grad(loss.sum(), s)
    return loss.detach(), grad


def exact(case, seed):
    d = _inputs(case, seed)
    kind, tau, k = case["kind"], case["temperature"], case["top"]
    if kind == "alternatives":
        return _exact_alternatives(d["scores"], d["labels"], k, tau)
    if kind == "alternatives_grad":
        return dict(grad=_exact_alternatives_grad(d, tau))
    if kind == "distill":
        loss, grad = _exact_distill(d, d["classes"], d["logits"], d.get("log_norm"), tau)
        return dict(loss=loss, grad=grad)
    t = _exact_alternatives(d["teacher"], d["labels"], k, tau)
    # (a teacher's lists are handed on in 32 bits)
    loss, grad = _exact_distill(d, t["classes"], t["log_prob"].to(F32).to(F64) * tau,
                                torch.zeros_like(t["entropy"]), tau)
    L = _logs64(d["scores"], 1.0)
    label = L[torch.arange(L.shape[0], device=DEV), d["labels"].long()]
    more = _exact_alternatives_grad(dict(scores=d["scores"], labels=d["labels"],
                                         grad_label=d["grad_label"]), 1.0)
    return dict(classes=t["classes"], log_prob=t["log_prob"], entropy=t["entropy"], loss=loss,
                label_log_prob=label, grad=grad + more)

"""The losses of class scores and of paired scores, as measurable cases.

Seven kinds of call:

* ``log_probs``       log-probability of each row's class (``class_log_probs``);
* ``log_probs_grad``  its gradient (``class_log_probs_grad``);
* ``policy``          clipped policy loss with a KL term and its gradient (``policy_loss``);
* ``balance``         per-class counts, mean probabilities, the balance loss and its gradient
                      (``balance_loss``);
* ``preference``      paired log ratios of rows or of sequences of rows, with the gradient
                      (``preference_loss``);
* ``step``            what a policy round computes: the policy loss, then the balance loss, whose
                      gradient is added to the policy's;
* ``sequence``        what a preference round of a class policy computes: log-probabilities, their
                      paired log ratios, and the gradient with respect to the scores.

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
BETA, SMOOTH = 0.5, 0.1          # of the preference losses
CLIP = (0.2, 0.25)               # below and above 1
KL = 0.1                         # weight of the KL term


# --------------------------------------------------------------------------- the cases
def listed():
    return [
        # one decision answered: a single row over a large set of classes
        dict(name="log probs one row", kind="log_probs", rows=1, classes=50_001, dtype="float32",
             major="row", masked=0.0),
        # the decisions logged with a class forest's training table, scores class by class as
        # the engine keeps them
        dict(name="log probs class forest", kind="log_probs", rows=1_000_000, classes=10,
             dtype="float32", major="class", masked=0.0),
        # few hundred classes, odd sizes, half precision
        dict(name="log probs grad odd", kind="log_probs_grad", rows=20_047, classes=257,
             dtype="float16", major="row", masked=0.1),
        # a large set of classes for each of some thousand rows
        dict(name="log probs grad many classes", kind="log_probs_grad", rows=4_099, classes=32_000,
             dtype="bfloat16", major="row", masked=0.0),
        # a policy's whole training table against a reference model's scores, some classes
        # not allowed in some rows
        dict(name="policy class forest", kind="policy", rows=1_000_000, classes=10,
             dtype="float32", major="class", kl="exact", masked=0.2),
        # the widest: a large set of classes, the reference known by its log-probabilities
        dict(name="policy many classes", kind="policy", rows=8_191, classes=16_001,
             dtype="bfloat16", major="row", kl="sampled", masked=0.0),
        # load of a hundred classes over the headline number of rows, a tenth of them left out
        dict(name="balance class forest", kind="balance", rows=1_000_000, classes=100,
             dtype="float32", major="class", top_k=1, masked=0.0),
        # a gate's scores: two of 64 for each row
        dict(name="balance gate", kind="balance", rows=65_536, classes=64, dtype="bfloat16",
             major="row", top_k=2, masked=0.0),
        # ranking: items drawn again and again, some far more often than others
        dict(name="preference items", kind="preference", rows=1_000_000, segments=0,
             pairs=2_000_000, length=1, reference=False),
        # sequences of very different lengths, empty ones among them, each in one pair
        dict(name="preference sequences", kind="preference", rows=0, segments=100_000,
             pairs=50_000, length=200, reference=True),
        # a small table's round: launches count, not bytes
        dict(name="step small", kind="step", rows=10_000, classes=3, dtype="float32",
             major="class", kl="sampled", top_k=1, masked=0.0),
        # a preference round of a class policy
        dict(name="sequence class forest", kind="sequence", rows=0, segments=20_001, pairs=30_000,
             length=25, classes=32, dtype="float32", major="class", masked=0.0),
    ]


CELLS = 1 << 27  # rows * classes of the largest case


def _log(rng, lo, hi):
    """A whole number whose logarithm is uniform between those of lo and hi."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["log_probs", "log_probs_grad", "policy", "policy", "balance", "balance",
                       "preference", "preference", "step", "sequence"])
    if kind == "preference":
        reference = rng.random() < 0.5
        if rng.random() < 0.5:
            rows = _log(rng, 2, 1_000_000)
            return dict(kind=kind, rows=rows, segments=0, pairs=_log(rng, 1, 2_000_000), length=1,
                        reference=reference)
        segments = _log(rng, 2, 100_000)
        return dict(kind=kind, rows=0, segments=segments, pairs=_log(rng, 1, 2 * segments),
                    length=_log(rng, 1, max(2, min(200_000, 20_000_000 // segments))),
                    reference=reference)
    # (a round's scores are the engine's: 32 bits)
    dtype = "float32" if kind == "step" else rng.choice(["float32", "float32", "bfloat16",
                                                         "float16"])
    major = rng.choice(["row", "class"])
    masked = rng.choice([0.0, 0.0, 0.2])
    if kind == "sequence":
        classes = _log(rng, 2, 512)
        segments = _log(rng, 50, 20_000)
        most = max(2, min(10_000, CELLS // 4 // classes // segments))
        return dict(kind=kind, rows=0, segments=segments, pairs=_log(rng, 50, 2 * segments),
                    length=_log(rng, 1, most), classes=classes, dtype=dtype, major=major,
                    masked=masked)
    most = 4_096 if kind in ("balance", "step") else 65_537
    classes = _log(rng, 2, most)
    cells = CELLS if kind != "step" else CELLS // 8
    # (a single confident row's gradient is a difference of nearly equal numbers in any form)
    rows = _log(rng, 1 if kind == "log_probs" else 20, min(1_000_000, cells // classes))
    case = dict(kind=kind, rows=rows, classes=classes, dtype=dtype, major=major, masked=masked)
    if kind in ("policy", "step"):
        case["kl"] = rng.choice(["none", "sampled", "exact"])
        if case["kl"] == "exact":
            case["rows"] = max(20, rows // 2)
    if kind in ("balance", "step"):
        # (a gradient of zero where every class is taken says nothing)
        case["top_k"] = rng.choice([k for k in (1, 1, 2, 8) if k == 1 or 2 * k <= classes])
    return case


# --------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1_000_003 * int(seed) + 29)
    return g


def _normal(shape, g):
    return torch.randn(shape, generator=g, device=DEV)


def _class_inputs(case, seed, rows):
    """Scores [rows, classes] as a forest or a gate gives them (a spread of a few units, some
    classes liked more), a behaviour policy near them, and the classes that it took."""
    g = _gen(seed)
    n, K = rows, case["classes"]
    by_class = case["major"] == "class"
    shape = (K, n) if by_class else (n, K)
    lean = _normal((K, 1) if by_class else (1, K), g)
    scores = 1.5 * _normal(shape, g) + lean
    away = 0.3 * _normal(shape, g)
    if case["masked"]:
        # classes that a row may not take; its best class always stays
        shut = torch.rand(shape, generator=g, device=DEV) < case["masked"]
        best = scores.argmax(0 if by_class else 1, keepdim=True)
        shut.scatter_(0 if by_class else 1, best, False)
        scores.masked_fill_(shut, -math.inf)
        del shut
    scores = scores.to(TYPES[case["dtype"]])
    if by_class:
        scores, away = scores.t(), away.t()
    behave = scores.float() + away
    noise = torch.rand(shape, generator=g, device=DEV).clamp_(1e-7, 1 - 1e-7).log_().neg_().log_()
    noise = noise.t() if by_class else noise
    taken = (behave - noise).argmax(1)
    del noise
    old = behave.gather(1, taken[:, None])[:, 0] - torch.logsumexp(behave, 1)
    d = dict(scores=scores, taken=taken.to(torch.int32))
    kind = case["kind"]
    if kind in ("policy", "step"):
        adv = _normal((n,), g)
        d["advantage"] = torch.where(torch.rand(n, generator=g, device=DEV) < 0.1, 0.0, adv)
        d["old"] = old
        # rows of no weight: padding at the end of a batch, rows held out
        live = (torch.rand(n, generator=g, device=DEV) >= 0.1).to(F32)
        d["weight"] = live * (0.5 + torch.rand(n, generator=g, device=DEV))
        if case["kl"] == "sampled":
            d["ref"] = old + 0.2 * _normal((n,), g)
        elif case["kl"] == "exact":
            d["ref_scores"] = (0.9 * scores.float() + away).to(scores.dtype)
    if kind in ("balance", "step"):
        d["mask"] = torch.rand(n, generator=g, device=DEV) >= 0.1
    return d


def _segment_rows(case):
    return case["segments"] * case["length"] + 3


def _pair_inputs(case, seed):
    """Pairs (preferred, other) of rows or sequences, the sequences' offsets, weights."""
    g = _gen(seed + 7919)
    S, P = case["segments"], case["pairs"]
    d = {}
    if S:
        # cuts at random places: lengths spread like an exponential's, one sequence in twenty
        # empty; padding rows behind the last sequence
        n, ends = _segment_rows(case), S
        cuts = torch.randint(0, n - 2, (S + 1,), generator=g, device=DEV).sort().values
        again = torch.rand(S, generator=g, device=DEV) < 0.05
        cuts[1:] = torch.where(again, cuts[:-1], cuts[1:])
        cuts[0], cuts[-1] = 0, n - 3
        d["segments"] = cuts
    else:
        n = ends = case["rows"]
    if S and 2 * P <= S:
        pairs = torch.randperm(S, generator=g, device=DEV)[:2 * P].reshape(P, 2)
    else:
        # the square of a uniform number: items with low numbers come more often
        u = torch.rand((P, 2), generator=g, device=DEV)
        pairs = (u * u * ends).long().clamp_(max=ends - 1)
    d["pairs"] = pairs.to(torch.int32)
    d["pair_weight"] = 0.5 + torch.rand(P, generator=g, device=DEV)
    if case["kind"] == "preference":
        d["log_prob"] = -2.0 * torch.rand(n, generator=g, device=DEV)
        if case["reference"]:
            d["reference"] = d["log_prob"] + 0.1 * _normal((n,), g)
    return d, n


def _inputs(case, seed):
    kind = case["kind"]
    if kind == "preference":
        return _pair_inputs(case, seed)[0]
    if kind == "sequence":
        d, n = _pair_inputs(case, seed)
        d.update(_class_inputs(case, seed, n))
        d["reference"] = _log_probs(d["scores"], d["taken"])[0] + 0.5 * _normal((n,), _gen(seed + 1))
        return d
    d = _class_inputs(case, seed, case["rows"])
    if kind == "log_probs_grad":
        # what the forward pass left: log-probabilities' norms, and a gradient for them
        d["norm"] = _log_probs(d["scores"], d["taken"])[1]
        d["grad_log_prob"] = _normal((case["rows"],), _gen(seed + 1))
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    d["case"] = case
    if own and "pairs" in d:
        from warpgbm_amd import losses

        # laid out once for all rounds of a fit
        n = d["log_prob"].shape[0] if "log_prob" in d else d["scores"].shape[0]
        d["plan"] = losses.PreferencePlan(d["pairs"], n, segments=d.get("segments"))
    return d


# --------------------------------------------------------------------------- the plain forms
def _coef(case):
    """Weight of the balance term next to losses summed over the rows; gradients in float16 need
    a loss scale, or they fall below its smallest normal number."""
    return 0.01 * case["rows"] * (1024 if case["dtype"] == "float16" else 1)


def _log_probs(scores, taken):
    s = scores.float()
    top = s.amax(1)
    spread = torch.exp(s - top[:, None]).sum(1).log()
    logp = s.gather(1, taken.long()[:, None])[:, 0] - top - spread
    return logp, torch.stack([top, spread], 1)


def _log_probs_grad(scores, taken, norm, grad):
    p = torch.exp(scores.float() - norm[:, :1] - norm[:, 1:])
    out = -p * grad[:, None]
    out.scatter_add_(1, taken.long()[:, None], grad[:, None])
    return out


def _policy(d):
    scores, taken, w = d["scores"], d["taken"].long()[:, None], d["weight"]
    s = scores.float()
    logs = torch.log_softmax(s, 1)
    p = torch.exp(logs)
    # the ratio is compared with the clip's borders: in 64 bits
    wide = scores.double()
    logp = wide.gather(1, taken)[:, 0] - torch.logsumexp(wide, 1)
    del wide
    A = d["advantage"].double()
    ratio = torch.exp(logp - d["old"].double())
    free, held = ratio * A, ratio.clamp(1 - CLIP[0], 1 + CLIP[1]) * A
    loss = -torch.minimum(free, held)
    slope = torch.where(free <= held, -free, torch.zeros_like(free))  # d loss / d log-probability
    out = {}
    if "ref" in d:
        gap = d["ref"].double() - logp
        out["kl"] = torch.exp(gap) - gap - 1
        slope = slope + KL * (1 - torch.exp(gap))
        loss = loss + KL * out["kl"]
    grad = -p * slope.float()[:, None]
    # 1 - p of the taken class from its logarithm: no difference of nearly equal numbers
    grad.scatter_(1, taken, (-torch.expm1(logp) * slope).float()[:, None])
    if "ref_scores" in d:
        gap = torch.where(p > 0, logs - torch.log_softmax(d["ref_scores"].float(), 1), 0.0)
        kl = (p * gap).sum(1)
        grad += KL * p * (gap - kl[:, None])
        loss = loss + KL * kl
        out["kl"] = kl
    live = w != 0
    grad = torch.where(live[:, None], grad * w[:, None], 0.0)
    out["loss"] = torch.where(live, loss * w, 0.0).float()
    out["log_prob"] = torch.where(live, logp, 0.0).float()
    if "kl" in out:
        out["kl"] = torch.where(live, out["kl"], 0.0).float()
    return out, grad


def _balance(d, k):
    s = d["scores"].float()
    live = d["mask"]
    n, K = s.shape
    p = torch.where(live[:, None], torch.softmax(s, 1), 0.0)
    rows = live.sum().clamp(min=1)
    # the k best classes, the lowest number first among equals
    left, counts = s.clone(), torch.zeros(K, dtype=torch.int64, device=s.device)
    for _ in range(k):
        top, best = left.max(1)
        best = (left == top[:, None]).to(torch.int8).argmax(1)
        counts.index_add_(0, best, (live & (top > -math.inf)).long())
        left.scatter_(1, best[:, None], -math.inf)
    mean = (p.sum(0, dtype=F64) / rows).float()
    share = (counts.double() / (rows * k)).float()
    coef = _coef(d["case"])
    loss = coef * K * (share * mean).sum()
    grad = (coef * K / rows.float()) * p * (share - (p @ share)[:, None])
    return dict(loss=loss, counts=counts, prob=mean), grad


def _preference(d, logp):
    u = logp.double()
    if "reference" in d:
        u = u - d["reference"].double()
    n, seg = u.shape[0], d.get("segments")
    if seg is not None:
        sums = torch.zeros(n + 1, dtype=F64, device=u.device)
        torch.cumsum(u, 0, out=sums[1:])
        total = sums[seg[1:]] - sums[seg[:-1]]
    else:
        total = u
    a, b = d["pairs"][:, 0].long(), d["pairs"][:, 1].long()
    margin = total[a] - total[b]
    z, w = BETA * margin, d["pair_weight"].double()
    up = torch.log1p(torch.exp(-z.abs()))
    loss = w * ((1 - SMOOTH) * (up + (-z).clamp(min=0)) + SMOOTH * (up + z.clamp(min=0)))
    slope = w * BETA * (torch.sigmoid(z) - (1 - SMOOTH))
    per = torch.zeros_like(total).index_add_(0, a, slope).index_add_(0, b, -slope)
    if seg is not None:
        at = torch.searchsorted(seg, torch.arange(n, device=u.device), right=True) - 1
        per = torch.where(at < per.shape[0], per[at.clamp(max=per.shape[0] - 1)], 0.0)
    return dict(loss=loss.float(), margin=margin.float()), per.float()


def _run_plain(d):
    case = d["case"]
    kind = case["kind"]
    if kind == "log_probs":
        logp, norm = _log_probs(d["scores"], d["taken"])
        return dict(log_prob=logp, norm=norm)
    if kind == "log_probs_grad":
        g = _log_probs_grad(d["scores"], d["taken"], d["norm"], d["grad_log_prob"])
        return dict(grad=g.to(d["scores"].dtype))
    if kind == "policy":
        out, grad = _policy(d)
        return dict(out, grad=grad.to(d["scores"].dtype))
    if kind == "balance":
        out, grad = _balance(d, case["top_k"])
        return dict(out, grad=grad.to(d["scores"].dtype))
    if kind == "step":
        out, grad = _policy(d)
        even, more = _balance(d, case["top_k"])
        out.update(balance=even["loss"], counts=even["counts"], prob=even["prob"])
        return dict(out, grad=(grad + more).to(d["scores"].dtype))
    if kind == "preference":
        out, grad = _preference(d, d["log_prob"])
        return dict(out, grad=grad)
    logp, norm = _log_probs(d["scores"], d["taken"])
    out, back = _preference(d, logp)
    grad = _log_probs_grad(d["scores"], d["taken"], norm, back)
    return dict(out, log_prob=logp, grad=grad.to(d["scores"].dtype))


# --------------------------------------------------------------------------- the package's calls
def _run_own(d):
    from warpgbm_amd import losses

    case = d["case"]
    kind = case["kind"]

    def policy():
        return losses.policy_loss(d["scores"], d["taken"], d["old"], d["advantage"],
                                  weight=d["weight"], ref_log_prob=d.get("ref"),
                                  ref_scores=d.get("ref_scores"), clip=CLIP,
                                  kl_coef=KL if case["kl"] != "none" else 0.0)

    def preference(logp):
        return losses.preference_loss(logp, d["plan"], ref_log_prob=d.get("reference"),
                                      weight=d["pair_weight"], beta=BETA, label_smoothing=SMOOTH)

    if kind == "log_probs":
        r = losses.class_log_probs(d["scores"], d["taken"])
        return dict(log_prob=r.log_prob, norm=r.norm)
    if kind == "log_probs_grad":
        return dict(grad=losses.class_log_probs_grad(d["scores"], d["taken"], d["norm"],
                                                     d["grad_log_prob"]))
    if kind == "policy":
        r = policy()
        out = dict(loss=r.loss, log_prob=r.log_prob, grad=r.grad)
        return dict(out, kl=r.kl) if case["kl"] != "none" else out
    if kind == "balance":
        r = losses.balance_loss(d["scores"], top_k=case["top_k"], mask=d["mask"], coef=_coef(case))
        return dict(loss=r.loss, counts=r.counts, prob=r.prob, grad=r.grad)
    if kind == "step":
        r = policy()
        e = losses.balance_loss(d["scores"], top_k=case["top_k"], mask=d["mask"], coef=_coef(case),
                                grad=r.grad)
        out = dict(loss=r.loss, log_prob=r.log_prob, balance=e.loss, counts=e.counts, prob=e.prob,
                   grad=e.grad)
        return dict(out, kl=r.kl) if case["kl"] != "none" else out
    if kind == "preference":
        r = preference(d["log_prob"])
        return dict(loss=r.loss, margin=r.margin, grad=r.grad)
    f = losses.class_log_probs(d["scores"], d["taken"])
    r = preference(f.log_prob)
    return dict(loss=r.loss, margin=r.margin, log_prob=f.log_prob,
                grad=losses.class_log_probs_grad(d["scores"], d["taken"], f.norm, r.grad))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# --------------------------------------------------------------------------- work
def work(case):
    """Bytes: scores (and reference scores) read once, gradients written once, the rows' and
    pairs' numbers; operations: an exponential counted as one."""
    kind = case["kind"]
    n, P = case["rows"], case.get("pairs", 0)
    if case.get("segments", 0):
        n = _segment_rows(case)
    pairs = 8 * P + 4 * P + 8 * P + 8 * (case.get("segments", 0) + 1) if P else 0
    if kind == "preference":
        per_row = 8 + (4 if case["reference"] else 0)
        return dict(bytes=per_row * n + pairs, flops=2 * n + 12 * P)
    K, es = case["classes"], 4 if case["dtype"] == "float32" else 2
    cells = n * K
    if kind == "log_probs":
        return dict(bytes=es * cells + 16 * n, flops=4 * cells)
    if kind == "log_probs_grad":
        return dict(bytes=2 * es * cells + 16 * n, flops=4 * cells)
    if kind == "sequence":
        return dict(bytes=2 * es * cells + 4 * n + 4 * n + 4 * n + pairs, flops=8 * cells)
    matrices = 2 + (1 if case.get("kl") == "exact" else 0)
    nbytes, flops = matrices * es * cells, 8 * cells
    if kind in ("policy", "step"):
        nbytes += 24 * n + (8 * n if case["kl"] == "sampled" else 4 * n)
        flops += 10 * cells if case["kl"] == "exact" else 0
    if kind in ("balance", "step"):
        nbytes += n + 16 * K
        flops += 6 * cells
    return dict(bytes=nbytes, flops=flops)


# --------------------------------------------------------------------------- in 64 bits
def _log_softmax64(scores):
    x = scores.to(F64)
    return x - torch.logsumexp(x, dim=1, keepdim=True)


def _onehot_rows(like, cls, value):
    """A matrix of zeros with value[i] at (i, cls[i])."""
    m = torch.zeros_like(like)
    m[torch.arange(cls.shape[0], device=cls.device), cls.long()] = value
    return m


def _exact_policy(d):
    L = _log_softmax64(d["scores"])
    P = L.exp()
    rows = torch.arange(L.shape[0], device=DEV)
    lp = L[rows, d["taken"].long()]
    A, w = d["advantage"].to(F64), d["weight"].to(F64)
    r = (lp - d["old"].to(F64)).exp()
    lo, hi = 1 - CLIP[0], 1 + CLIP[1]
    # positive advantages stop at the upper border, negative ones at the lower
    stopped = ((A > 0) & (r > hi)) | ((A < 0) & (r < lo))
    value = -A * torch.where(stopped, torch.where(A > 0, hi, lo), r)
    dlp = torch.where(stopped, 0.0, -A * r)
    kl = None
    if "ref" in d:
        x = d["ref"].to(F64) - lp
        kl = torch.expm1(x) - x
        dlp = dlp - KL * torch.expm1(x)
    G = _onehot_rows(L, d["taken"], dlp) - P * dlp[:, None]
    if "ref_scores" in d:
        diff = (L - _log_softmax64(d["ref_scores"])).masked_fill(P == 0, 0.0)
        kl = (P * diff).sum(1)
        G = G + KL * P * (diff - kl[:, None])
    if kl is not None:
        value = value + KL * kl
    off = w == 0
    out = dict(loss=(w * value).masked_fill(off, 0.0), log_prob=lp.masked_fill(off, 0.0))
    if kl is not None:
        out["kl"] = kl.masked_fill(off, 0.0)
    return out, (G * w[:, None]).masked_fill(off[:, None], 0.0)


def _exact_balance(d, k):
    live, coef = d["mask"], _coef(d["case"])
    x = d["scores"].to(F64)[live]
    K = x.shape[1]
    P = torch.softmax(x, 1)
    n = max(1, x.shape[0])
    # a stable sort keeps the lower class first among equals
    order = torch.sort(x, dim=1, descending=True, stable=True)
    first = order.indices[:, :k][order.values[:, :k] > -math.inf]
    counts = torch.bincount(first, minlength=K)
    mean, f = P.sum(0) / n, counts.to(F64) / (n * k)
    G = torch.zeros(d["scores"].shape, dtype=F64, device=DEV)
    G[live] = coef * K / n * P * (f[None, :] - (P * f).sum(1, keepdim=True))
    return dict(loss=coef * K * torch.dot(f, mean), counts=counts, prob=mean), G


def _exact_preference(d, logp):
    u = logp.to(F64) - (d["reference"].to(F64) if "reference" in d else 0.0)
    n = u.shape[0]
    if "segments" in d:
        S = d["segments"].shape[0] - 1
        of = torch.full((n,), S, dtype=torch.int64, device=DEV)
        lengths = d["segments"].diff()
        of[:int(lengths.sum())] = torch.repeat_interleave(torch.arange(S, device=DEV), lengths)
    else:
        S, of = n, torch.arange(n, device=DEV)
    U = torch.zeros(S + 1, dtype=F64, device=DEV).scatter_add_(0, of, u)
    win, lose = d["pairs"].long().unbind(1)
    m, w = U[win] - U[lose], d["pair_weight"].to(F64)
    ls = torch.nn.functional.logsigmoid
    loss = -w * ((1 - SMOOTH) * ls(BETA * m) + SMOOTH * ls(-BETA * m))
    dm = w * BETA * (SMOOTH * torch.sigmoid(BETA * m) - (1 - SMOOTH) * torch.sigmoid(-BETA * m))
    g = torch.zeros(S + 1, dtype=F64, device=DEV)
    g.scatter_add_(0, win, dm)
    g.scatter_add_(0, lose, -dm)
    g[S:] = 0
    if "segments" not in d:
        return dict(loss=loss, margin=m), g[:S]
    return dict(loss=loss, margin=m), g[of]


def exact(case, seed):
    d = _inputs(case, seed)
    d["case"] = case
    kind = case["kind"]
    if kind == "preference":
        out, grad = _exact_preference(d, d["log_prob"])
        return dict(out, grad=grad)
    rows = torch.arange(d["scores"].shape[0], device=DEV)
    if kind == "log_probs":
        L = _log_softmax64(d["scores"])
        top = d["scores"].max(1).values.to(F64)
        lse = torch.logsumexp(d["scores"].to(F64), 1)
        return dict(log_prob=L[rows, d["taken"].long()], norm=torch.stack([top, lse - top], 1))
    if kind == "log_probs_grad":
        g, P = d["grad_log_prob"].to(F64), _log_softmax64(d["scores"]).exp_()
        return dict(grad=_onehot_rows(P, d["taken"], g) - P * g[:, None])
    if kind == "policy":
        out, grad = _exact_policy(d)
        return dict(out, grad=grad)
    if kind == "balance":
        out, grad = _exact_balance(d, case["top_k"])
        return dict(out, grad=grad)
    if kind == "step":
        out, grad = _exact_policy(d)
        even, more = _exact_balance(d, case["top_k"])
        return dict(out, balance=even["loss"], counts=even["counts"], prob=even["prob"],
                    grad=grad + more)
    L = _log_softmax64(d["scores"])
    lp = L[rows, d["taken"].long()]
    out, back = _exact_preference(d, lp)
    P = L.exp()
    return dict(out, log_prob=lp, grad=_onehot_rows(P, d["taken"], back) - P * back[:, None])

"""Alternatives of class scores, their gradient, and distillation from listed
classes, against plain float64 forms.

The float64 forms follow the definitions (dense shares of every class); their
gradients come from autograd.  Tolerances count roundings as in test_losses: 2^-24
of each float32 step, half a step of the gradient's type, and STEPS roundings
for a sum over a row's classes.
"""
import ctypes as C
import math

import pytest
import torch

from conftest import print_case
from test_losses import (DTYPES, F64, ORDERS, SHAPES, STEPS, U, check, live_rows, make_scores,
                         to_gpu)

INF = math.inf


# --------------------------------------------------------------------- float64 forms
def logs64(s, tau):
    """x = (s - max) / tau and log softmax(s / tau); rows without a class: 0, not used.
    The sum's logarithm is log1p of the sum without its largest term, 1: in float64
    too, a row sure of its class would keep few digits of a logarithm near 0."""
    s = s.to(F64)
    has = (s > -INF).any(1) | torch.isnan(s).any(1)
    s = torch.where(has[:, None], s, torch.zeros((), dtype=F64))
    best = s.detach().max(1, keepdim=True)
    x = (s - best.values) / tau
    rest = torch.exp(x).scatter(1, best.indices, 0.0).sum(1, keepdim=True)
    return x, x - torch.log1p(rest), has


def alternatives64(s, label, k, tau):
    x, L, has = logs64(s, tau)
    p = L.exp()
    best = torch.sort(s.to(F64), dim=1, descending=True, stable=True)
    cls = torch.where(best.values[:, :k] > -INF, best.indices[:, :k], -1)
    lp = torch.where(cls >= 0, L.gather(1, cls.clamp(min=0)), -INF)
    down = torch.where(p > 0, -x * p, torch.zeros((), dtype=F64)).sum(1)
    square = torch.where(p > 0, x * x * p, torch.zeros((), dtype=F64)).sum(1)
    lse = -(L.max(1).values)
    K = s.shape[1]
    at = label.long().clamp(0, K - 1)[:, None]
    use = has & (label >= 0) & (label < K)
    lab = torch.where(use, L.gather(1, at)[:, 0], torch.zeros((), dtype=F64))
    zero = torch.zeros((), dtype=F64)
    return dict(classes=torch.where(has[:, None], cls, -1),
                log_prob=torch.where(has[:, None], lp, -INF),
                entropy=torch.where(has, lse + down, zero), label=lab, lse=lse, down=down,
                square=square, has=has, top=s.to(F64).max(1).values)


def check_alternatives(r, want, k, label=True):
    has, n = want["has"], want["has"].shape[0]
    assert r.classes.dtype == torch.int32 and tuple(r.classes.shape) == (n, k)
    assert torch.equal(r.classes.cpu().long(), want["classes"]), "classes"
    lse, down = want["lse"], want["down"]
    # the sum without its largest term is a share 1 - e^-lse of the sum
    t_lse = U * (STEPS * (1 - torch.exp(-lse)) + 4 * down + 8 * lse)
    t_down = U * (STEPS * down + 4 * want["square"])

    def lp_tol(L):
        return t_lse + U * (2 * L.abs() + 2 * lse)

    w = want["log_prob"]
    fin = w > -INF
    assert (r.log_prob.cpu()[~fin] == -INF).all()
    tol = t_lse[:, None] + U * 4 * w.abs()
    # (numbers below the smallest normal one of float32 may be 0)
    check(torch.where(fin, r.log_prob.cpu().to(F64), 0.0), torch.where(fin, w, 0.0), tol + 1e-37,
          "log_prob")
    check(r.entropy, want["entropy"], t_lse + t_down + U * want["entropy"] + 1e-37, "entropy")
    if label:
        w = want["label"]
        fin = w > -INF
        assert (r.label_log_prob.cpu()[~fin] == -INF).all()
        check(r.label_log_prob[fin.cuda()], w[fin], (t_lse + U * 4 * w.abs())[fin] + 1e-37, "label")
    norm = r.norm.cpu()
    assert (norm[~has] == torch.tensor([-INF, 0.0, 0.0])).all()
    check(norm[has, 0], want["top"][has], 0.0, "maximum")
    check(norm[has, 1], lse[has], t_lse[has] + 1e-37, "log of the sum")
    check(norm[has, 2], down[has], t_down[has] + U * down[has] + 1e-37, "mean distance")


def first_listed(classes, K):
    """Per entry: whether it counts (in range, not named before by the row)."""
    n, k = classes.shape
    seen = torch.zeros((n, K + 1), dtype=torch.bool)
    ok = torch.zeros((n, k), dtype=torch.bool)
    rows = torch.arange(n)
    for j in range(k):
        c = classes[:, j].long()
        c = torch.where((c >= 0) & (c < K), c, K)
        ok[:, j] = (c < K) & ~seen[rows, c]
        seen[rows, c] = True
    return ok, seen[:, :K]


def distill64(s, classes, logits, log_norm, w, tau):
    """Losses and gradient of the rows that count, and the ingredients of their
    tolerances."""
    n, K = s.shape
    ok, listed = first_listed(classes, K)
    shut = s == -INF
    live = live_rows(s, weight=w)
    slot = torch.where(ok, classes.long(), K)
    t = torch.full((n, K + 1), -INF, dtype=F64)
    t.scatter_(1, slot, logits.to(F64) / tau)
    t = t[:, :K]
    # (an unused slot's logit was written behind the classes)
    t = torch.where(listed, t, -INF)
    Q = torch.zeros(n, dtype=F64)
    if log_norm is not None:
        t = t - torch.as_tensor(log_norm, dtype=F64).reshape(-1, 1)
        Q = 1 - t.exp().sum(1)
        Q = torch.where((Q >= 2.0 ** -20) & (~listed & ~shut).any(1), Q, torch.zeros((), dtype=F64))
    t = torch.where(shut, -INF, t)
    if log_norm is None:
        t = t - t.max(1, keepdim=True).values.clamp(min=-1e300)
    q = t.exp()
    mass = q.sum(1) + Q
    live &= mass > 0
    mass = torch.where(live, mass, torch.ones((), dtype=F64))
    q, Q = q / mass[:, None], Q / mass
    x = torch.where(live[:, None], s.to(F64), torch.zeros((), dtype=F64)).requires_grad_(True)
    L = torch.log_softmax(x / tau, 1)
    safe = torch.where(shut & live[:, None], torch.zeros((), dtype=F64), L)
    loss = torch.special.xlogy(q, q).sum(1) - (q * safe).sum(1)
    others = torch.where(listed | (shut & live[:, None]), -1e300, L)
    rest = torch.where(Q > 0, torch.logsumexp(others, 1), torch.zeros((), dtype=F64))
    loss = loss + torch.special.xlogy(Q, Q) - Q * rest
    loss = torch.where(live, loss * w.to(F64) * tau * tau, torch.zeros((), dtype=F64))
    (grad,) = torch.autograd.grad(loss.sum(), x)
    p = L.detach().exp()
    r = torch.where(listed | shut, torch.zeros((), dtype=F64), torch.exp(others - torch.logsumexp(
        others, 1, keepdim=True))).detach()
    P = torch.where(listed, torch.zeros((), dtype=F64), p).sum(1)
    far = torch.where(torch.isfinite(safe), safe, torch.zeros((), dtype=F64)).detach().abs()
    lost = (p - q).abs().sum(1)
    return dict(loss=loss.detach(), grad=grad.detach(), live=live, p=p, q=q, Q=Q, P=P, r=r, far=far,
                lost=lost, k=classes.shape[1], rest=rest.detach())


def check_distill(got, want, w, tau, dtype, old=None):
    d = want
    value = (w.to(F64) * tau * tau).abs()
    one = d["k"] + 8
    # first order: |p - q| times the sums' roundings; each bucket's own arithmetic; Q
    gap = torch.where(d["q"] > 0, (d["q"].log() + d["far"]).abs(), torch.zeros((), dtype=F64))
    own = (d["p"] + d["q"] * (1 + gap)).sum(1) + 2
    far_rest = torch.where(d["Q"] > 0, (d["Q"].clamp(min=1e-30).log() - d["rest"]).abs(),
                           torch.zeros((), dtype=F64))
    tol = value * U * (STEPS * d["lost"] + 16 * own + one * (2 + far_rest))
    check(got.loss, d["loss"], tol + U * d["loss"].abs() + 1e-37, "loss")
    assert (got.loss.cpu()[~d["live"]] == 0).all()
    if got.grad is None:
        return
    scale = (w.to(F64) * tau).abs()[:, None]
    p, q, r, P, Q = d["p"], d["q"], d["r"], d["P"][:, None], d["Q"][:, None]
    t = scale * U * ((STEPS + 4 * d["far"] + 64) * (p + q + r * (P + Q)) + one * (q + r))
    grad = d["grad"] if old is None else d["grad"] + old.to(F64)
    half = 0.0 if dtype == "f32" else torch.finfo(DTYPES[dtype]).eps / 2
    t = t + (U if dtype == "f32" else half * (1 + 1e-3)) * grad.abs()
    t = t + (2.0 ** -25 if dtype == "f16" else 1e-37)
    check(got.grad, grad, t, "gradient")


# --------------------------------------------------------------------- inputs
def lists_for(s, k, seed, tau, spare=True):
    """A teacher's lists for scores s: its best classes of noisy scores, some rows
    with fewer, and (spare) rows that name a class twice, out of range, or nothing."""
    g = torch.Generator().manual_seed(seed)
    n, K = s.shape
    base = torch.where(s == -INF, torch.zeros(()), s.float())
    t = 0.7 * base + torch.randn((n, K), generator=g)
    best = torch.sort(t, dim=1, descending=True)
    logits, cls = best.values[:, :k], best.indices[:, :k].to(torch.int32)
    if k > K:  # lists longer than the row
        more = k - K
        logits = torch.cat([logits, torch.zeros(n, more)], 1)
        cls = torch.cat([cls, torch.full((n, more), -1, dtype=torch.int32)], 1)
    log_norm = torch.logsumexp(t.double() / tau, 1).float()
    logits, cls = logits.clone(), cls.clone()
    cut = torch.randint(1, k + 1, (n,), generator=g)
    gone = (torch.arange(k)[None, :] >= cut[:, None]) & (torch.rand(n, 1, generator=g) < 0.3)
    cls[gone] = -1
    if spare and n >= 9:
        cls[3] = -7
        cls[5, 0] = K
        if k > 1:
            cls[7, k - 1] = cls[7, 0]
            logits[7, k - 1] += 1.0
            cls[8] = cls[8, 0]
    # (entries that are not used may hold anything)
    logits[(cls < 0) | (cls >= K)] = float("nan")
    return cls.contiguous(), logits.contiguous(), log_norm


LENGTHS = [1, 3, 8, 20, 64]


def lengths(K, j):
    return min(K, LENGTHS[j % len(LENGTHS)])


# --------------------------------------------------------------------- alternatives
@pytest.mark.gpu
@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_alternatives(gpu, dtype, order):
    from warpgbm_amd import losses

    for j, (n, K) in enumerate(SHAPES + [(5, 40_001), (70, 600), (3, 70_000), (2, 140_003)]):
        for k in sorted({0, lengths(K, j), lengths(K, j + 2)}):
            tau = [1.0, 0.5, 3.0][(j + k) % 3]
            print_case("alternatives", dtype, order, n, K, k, tau)
            s = make_scores(n, K, dtype, order, 300 + j, masked=0.3 if j % 2 else 0.0)
            a = torch.randint(0, K, (n,), generator=torch.Generator().manual_seed(j),
                              dtype=torch.int32)
            if n > 4:
                a[1], a[3] = -1, K
                s[2] = -INF
                s[4] = -INF
                s[4, K // 2] = 1.5  # a single class
            r = losses.class_alternatives(to_gpu(s), k, labels=a.cuda(), temperature=tau)
            check_alternatives(r, alternatives64(s, a, k, tau), k)


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_alternatives_of_equal_scores(gpu, dtype, order):
    """The lower class first: constant rows, few values, signed zeros, and rows whose
    best classes lie next to each other."""
    from warpgbm_amd import losses

    for K in (2, 10, 16, 40, 100, 300, 513, 1000, 2500, 9000, 33_000, 70_001):
        n, k = 5, min(K, 64)
        print_case("equal", dtype, order, K)
        g = torch.Generator().manual_seed(K)
        s = torch.zeros((n, K))
        s[1] = torch.randint(0, 3, (K,), generator=g).float()
        s[2, ::2] = -0.0
        s[3] = torch.linspace(3, -3, K)
        s[4] = torch.randn(K, generator=g)
        s[4, K // 3:K // 3 + 70] += 20.0
        s = s.to(DTYPES[dtype])
        if order == "class":
            s = s.t().contiguous().t()
        a = torch.zeros(n, dtype=torch.int32)
        r = losses.class_alternatives(to_gpu(s), k, labels=a.cuda())
        check_alternatives(r, alternatives64(s, a, k, 1.0), k)


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
def test_alternatives_of_sure_and_far_rows(gpu, order):
    """Rows sure of a class keep the digits of what is left; offsets, lowest finite
    masks, and rows of NaN."""
    from warpgbm_amd import losses

    for K in (3, 12, 50, 400, 2000, 20_000):
        print_case("sure", order, K)
        g = torch.Generator().manual_seed(K)
        s = torch.randn((7, K), generator=g)
        s[0, K // 2] = 30.0
        s[1] += 1e5
        s[2] = torch.finfo(torch.float32).min
        s[2, 1] = 0.25
        s[3] = torch.finfo(torch.float32).min
        s[4] = 0.125
        s[5, 0] = 80.0
        if order == "class":
            s = s.t().contiguous().t()
        k = min(K, 5)
        a = torch.full((7,), K // 2, dtype=torch.int32)
        r = losses.class_alternatives(to_gpu(s), k, labels=a.cuda())
        check_alternatives(r, alternatives64(s, a, k, 1.0), k)
        s[6, 1] = float("nan")
        r = losses.class_alternatives(to_gpu(s), k, labels=a.cuda())
        assert torch.isnan(r.entropy[6]) and torch.isnan(r.label_log_prob[6])
        assert not torch.isnan(r.entropy[:6]).any()
        c = r.classes[6].cpu()
        assert (c != 1).all() and (c < K).all() and (c >= -1).all()


@pytest.mark.gpu
def test_alternatives_without_labels_and_rows(gpu):
    from warpgbm_amd import losses

    s = make_scores(40, 11, "f32", "row", 1).cuda()
    with_labels = losses.class_alternatives(s, 4, labels=torch.zeros(40, dtype=torch.int32).cuda())
    r = losses.class_alternatives(s, 4)
    assert r.label_log_prob is None and torch.equal(r.classes, with_labels.classes)
    assert torch.equal(r.log_prob, with_labels.log_prob) and torch.equal(r.norm, with_labels.norm)
    e = losses.class_alternatives(s[:0], 4)
    assert tuple(e.classes.shape) == (0, 4) and tuple(e.norm.shape) == (0, 3)
    g = losses.class_alternatives_grad(s[:0], e.norm, grad_entropy=e.entropy)
    assert tuple(g.shape) == (0, 11)
    d = losses.distill_loss(s[:0], e.classes, e.log_prob)
    assert tuple(d.loss.shape) == (0,) and tuple(d.grad.shape) == (0, 11)


# --------------------------------------------------------------------- their gradient
def alternatives_grad64(s, label, g_label, cls, g_list, g_entropy, tau):
    """Gradient by autograd, and its tolerance before the rounding to a type."""
    n, K = s.shape
    zero = torch.zeros((), dtype=F64)
    has = live_rows(s)
    x = torch.where(has[:, None], s.to(F64), zero).requires_grad_(True)
    shut = (s == -INF) & has[:, None]
    L = torch.log_softmax(x / tau, 1)
    p = L.exp()
    # log p of class k is x_k / tau - log sum
    lse = torch.logsumexp(x / tau, 1, keepdim=True)
    flat = torch.where(shut, zero, x) / tau - lse
    total, own = zero, torch.zeros((n, K), dtype=F64)
    mass = torch.zeros(n, dtype=F64)
    rows = torch.arange(n)

    def add(c, g):
        nonlocal total, mass
        use = has & (c >= 0) & (c < K)
        g = torch.where(use, g.to(F64), zero)
        total = total + (g * flat.gather(1, c.long().clamp(0, K - 1)[:, None])[:, 0]).sum()
        own.index_put_((rows, c.long().clamp(0, K - 1)), g, accumulate=True)
        mass = mass + g.abs()

    if label is not None:
        add(label, g_label)
    if cls is not None:
        for j in range(cls.shape[1]):
            add(cls[:, j], g_list[:, j])
    if g_entropy is not None:
        safe = torch.where(shut, zero, L)
        total = total - (torch.where(has, g_entropy.to(F64), zero) * (p * safe).sum(1)).sum()
    (grad,) = torch.autograd.grad(total, x)
    # (a listed class of score -inf: autograd has no slope through the constant)
    grad = grad + torch.where(shut, own / tau, zero)
    d = torch.where(p > 0, (x.detach() - x.detach().max(1, keepdim=True).values) / tau, zero).detach()
    down = -(p.detach() * d).sum(1, keepdim=True)
    h = g_entropy.to(F64).abs()[:, None] if g_entropy is not None else 0.0
    per = (mass[:, None] + h * (d.abs() + down + 1)) * p.detach()
    tol = U / tau * (per * (STEPS + 6 * d.abs() + 64) + 16 * own.abs())
    return grad.detach(), torch.where(has[:, None], tol, zero)


def round_tol(tol, want, dtype):
    if dtype == "f32":
        return tol + U * want.abs() + 1e-37
    return tol + torch.finfo(DTYPES[dtype]).eps / 2 * (1 + 1e-3) * want.abs() + (
        2.0 ** -25 if dtype == "f16" else 1e-37)


@pytest.mark.gpu
@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_alternatives_gradient(gpu, dtype, order):
    from warpgbm_amd import losses

    for j, (n, K) in enumerate(SHAPES + [(5, 40_001), (70, 600), (3, 70_000), (2, 140_003)]):
        for what in ("all", "label", "entropy", "list"):
            k = lengths(K, j + len(what)) if what != "entropy" else 0
            tau = [1.0, 0.5, 3.0][(j + k) % 3]
            add = (j + k) % 2 == 1
            print_case("alternatives grad", dtype, order, n, K, k, what, tau, add)
            s = make_scores(n, K, dtype, order, 400 + j, masked=0.2 if j % 3 == 1 else 0.0)
            g = torch.Generator().manual_seed(j)
            a = torch.randint(0, K, (n,), generator=g, dtype=torch.int32)
            cls = torch.argsort(torch.rand((n, K), generator=g), 1)[:, :k].to(torch.int32)
            gl, ge = torch.randn(n, generator=g), torch.randn(n, generator=g)
            gt = torch.randn((n, k), generator=g)
            if n > 4:
                a[1], a[3] = -1, K
                s[2] = -INF
                gl[0] = ge[0] = 0.0
                gt[0] = 0.0
            if k and n > 8:
                cls[4, 0], cls[5, k - 1] = -1, K + 3
                cls[6] = cls[6, 0]           # one class only, again and again
                cls[7, k - 1] = a[7]
                a[8] = cls[8, 0]
            sd = to_gpu(s)
            f = losses.class_alternatives(sd, 0, temperature=tau)
            want_label = what in ("all", "label")
            want_list = what in ("all", "list") and k > 0
            want_ent = what in ("all", "entropy")
            grad, tol = alternatives_grad64(s, a if want_label else None, gl,
                                            cls if want_list else None, gt,
                                            ge if want_ent else None, tau)
            kw = {}
            if want_label:
                kw.update(labels=a.cuda(), grad_label_log_prob=gl.cuda())
            if want_list:
                kw.update(classes=cls.cuda(), grad_log_prob=gt.cuda())
            if want_ent:
                kw.update(grad_entropy=ge.cuda())
            old = None
            if add:
                old = make_scores(n, K, dtype, order, 900 + j)
                kw.update(grad=to_gpu(old))
                grad = grad + old.to(F64)
            got = losses.class_alternatives_grad(sd, f.norm, temperature=tau, **kw)
            assert got.dtype == s.dtype and got.shape == s.shape
            check(got, grad, round_tol(tol, grad, dtype), "gradient")
            if add:
                untouched(got, n, K, order)


def untouched(got, n, K, order):
    """The NaNs around a matrix with strides stay."""
    if order not in ("row+", "class+"):
        return
    whole = got.untyped_storage().nbytes() // got.element_size()
    flat = torch.as_strided(got, (whole,), (1,), 0).float().cpu()
    keep = torch.isnan(flat)
    inside = torch.as_strided(torch.zeros(whole, dtype=torch.bool), got.shape, got.stride(),
                              got.storage_offset())
    inside[:] = True
    flat_in = torch.as_strided(inside, (whole,), (1,), 0)
    assert keep[~flat_in].all()


# --------------------------------------------------------------------- distillation
@pytest.mark.gpu
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_distill(gpu, dtype, order, rest):
    from warpgbm_amd import losses

    for j, (n, K) in enumerate(SHAPES + [(5, 40_001), (70, 600), (3, 70_000), (2, 140_003)]):
        for k in sorted({lengths(K, j), lengths(K, j + 3), 64 if j % 4 == 0 else 2}):
            tau = [1.0, 0.5, 3.0][(j + k) % 3]
            add = (j + k) % 2 == 1
            print_case("distill", dtype, order, n, K, k, tau, rest, add)
            s = make_scores(n, K, dtype, order, 500 + j, masked=0.2 if j % 2 else 0.0)
            cls, logits, ln = lists_for(s, k, 600 + j, tau)
            g = torch.Generator().manual_seed(j)
            w = 0.5 + torch.rand(n, generator=g)
            if n > 4:
                w[1] = 0.0
                s[2] = -INF
            want = distill64(s, cls, logits, ln if rest else None, w, tau)
            s[w == 0] = float("nan")
            old, kw = None, {}
            if add:
                old = make_scores(n, K, dtype, order, 700 + j)
                kw.update(grad=to_gpu(old))
            got = losses.distill_loss(to_gpu(s), cls.cuda(), logits.cuda(),
                                      log_norm=ln.cuda() if rest else None, weight=w.cuda(),
                                      temperature=tau, **kw)
            assert got.grad.dtype == s.dtype and got.grad.shape == s.shape
            check_distill(got, want, w, tau, dtype, old)
            if add:
                untouched(got.grad, n, K, order)
            none = losses.distill_loss(to_gpu(s), cls.cuda(), logits.cuda(),
                                       log_norm=ln.cuda() if rest else None, weight=w.cuda(),
                                       temperature=tau, with_grad=False)
            assert none.grad is None
            check_distill(none, want, w, tau, dtype)


# --------------------------------------------------------------------- distillation, edges
def place(s, order):
    return s.t().contiguous().t() if order == "class" else s


EDGE_CLASSES = [2, 3, 11, 40, 300, 1500, 9000, 70_001]


@pytest.mark.gpu
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("order", ["row", "class"])
def test_distill_lists_that_leave_little(gpu, order, rest):
    """Rows whose list the row may not take, whose other classes it may not take, with
    one class, without a list; a list of all classes; a teacher sure of a class."""
    from warpgbm_amd import losses

    for K in EDGE_CLASSES:
        print_case("edges", order, K, rest)
        n, k = 9, min(K, 12)
        g = torch.Generator().manual_seed(K)
        s = torch.randn((n, K), generator=g)
        cls = torch.argsort(torch.rand((n, K), generator=g), 1)[:, :k].to(torch.int32).contiguous()
        t = torch.randn((n, K), generator=g)
        logits = t.gather(1, cls.long())
        ln = torch.logsumexp(t.double(), 1).float()
        rows = torch.arange(k)
        s[0, cls[0].long()] = -INF                      # nothing of the list
        keep = s[1, cls[1].long()].clone()
        s[1] = -INF
        s[1, cls[1].long()] = keep                      # nothing but the list
        s[2] = -INF
        s[2, cls[2, 0].long()] = 0.5                    # one class, listed
        s[3] = -INF
        s[3, (set(range(K)) - set(cls[3].tolist()) or {0}).__iter__().__next__()] = 0.5
        cls[4] = -1                                     # no list
        logits[5] = logits[5, 0]                        # an even teacher
        logits[6] = -50.0
        logits[6, 0] = float(ln[6])                     # a sure one
        s[7, cls[7, : max(1, k // 2)].long()] = -INF    # a part of the list
        w = 0.5 + torch.rand(n, generator=g)
        s = place(s, order)
        norms = ln if rest else None
        want = distill64(s, cls, logits, norms, w, 1.0)
        got = losses.distill_loss(to_gpu(s), cls.cuda(), logits.cuda(), weight=w.cuda(),
                                  log_norm=norms.cuda() if rest else None)
        check_distill(got, want, w, 1.0, "f32")
        assert bool(want["live"][0]) == (rest and k < K)
        assert bool(want["live"][4]) == rest


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
def test_distill_sure_rows_keep_their_digits(gpu, order):
    """Student and teacher both sure of a class: the gradient there is a difference
    of numbers next to 1, the rest a difference of small ones."""
    from warpgbm_amd import losses

    for K in EDGE_CLASSES[1:]:
        print_case("sure", order, K)
        s = torch.zeros((4, K))
        s[:, 0] = torch.tensor([14.0, 12.0, 9.0, 16.0])
        s[:, 1] = 1.0
        cls = torch.tensor([[0, 1]] * 4, dtype=torch.int32)
        left = torch.tensor([4e-5, 1e-4, 3e-3, 8e-6], dtype=F64)  # of the teacher beside class 0
        logits = torch.stack([torch.log1p(-left), torch.log(0.4 * left)], 1).float()
        w = torch.ones(4)
        sp = place(s, order)
        got = losses.distill_loss(to_gpu(sp), cls.cuda(), logits.cuda(), log_norm=0.0)
        # shares and probabilities beside class 0, without differences of numbers near 1
        x = s.to(F64) - s.to(F64)[:, :1]
        z = torch.exp(x[:, 1:]).sum(1)
        dp = z / (1 + z)
        q = logits.to(F64).exp()
        dq = -torch.expm1(logits[:, 0].to(F64))
        Q = dq - q[:, 1]
        p1 = torch.exp(x[:, 1]) / (1 + z)
        P = dp - p1
        tol = U * (STEPS + 64) * (dp + dq)
        check(got.grad[:, 0], dq - dp, tol, "sure class")
        check(got.grad[:, 1], p1 - q[:, 1], tol, "listed class")
        r = torch.exp(x[:, 2]) / torch.exp(x[:, 2:]).sum(1)
        check(got.grad[:, 2], r * (P - Q), tol * r, "other class")
        # terms q (e^x - 1 - x), a second-order difference
        want = (torch.special.xlogy(q[:, 1], q[:, 1] / p1) + torch.special.xlogy(Q, Q / P)
                + q[:, 0] * (torch.log1p(-dq) - torch.log1p(-dp)))
        gap = (dp - dq).abs() + (p1 - q[:, 1]).abs() + (P - Q).abs()
        check(got.loss, want, U * ((STEPS + 64) * gap + 64 * (dp + dq)), "loss")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("order", ["row", "class"])
def test_distill_far_scores_and_lowest_masks(gpu, order, dtype):
    """Offsets far from 0, and classes masked by the type's lowest number, which
    count as scores: masked like -inf where the teacher's rest is none."""
    from warpgbm_amd import losses

    low = torch.finfo(DTYPES[dtype]).min
    for K in EDGE_CLASSES[1:]:
        print_case("far", dtype, order, K)
        g = torch.Generator().manual_seed(K)
        n, k = 6, 2
        s = torch.randn((n, K), generator=g)
        s[0] += 3e4
        s[1] -= 3e4
        s = s.to(DTYPES[dtype])
        cls = torch.argsort(torch.rand((n, K), generator=g), 1)[:, :k].to(torch.int32).contiguous()
        t = torch.randn((n, k), generator=g)
        t = (t - torch.logsumexp(t, 1, keepdim=True)).contiguous()  # a teacher of these alone
        others = torch.ones((n, K), dtype=torch.bool).scatter_(1, cls.long(), False)
        others[:2] = False
        w = torch.ones(n)
        a = losses.distill_loss(to_gpu(place(s.masked_fill(others, low), order)), cls.cuda(),
                                t.cuda(), log_norm=0.0)
        b = distill64(place(s.masked_fill(others, -INF), order), cls, t, 0.0, w, 1.0)
        check_distill(a, b, w, 1.0, dtype)
        c = losses.distill_loss(to_gpu(place(s.masked_fill(others, low), order)), cls.cuda(),
                                t.cuda())
        check_distill(c, distill64(place(s.masked_fill(others, -INF), order), cls, t, None, w, 1.0),
                      w, 1.0, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
def test_lists_with_strides(gpu, order):
    """The first entries of longer lists, lists inside of other tensors, and lists whose
    rows are next to each other."""
    from warpgbm_amd import losses

    for n, K in ((37, 12), (37, 90), (20, 700)):
        s = make_scores(n, K, "f32", order, 3)
        cls, logits, ln = lists_for(s, 8, 4, 1.0, spare=False)
        big = torch.full((n, 19), 77, dtype=torch.int32)
        big[:, 5:13] = cls
        far = torch.full((n, 11), float("nan"))
        far[:, 3:11] = logits
        sd, w = to_gpu(s), torch.ones(n)
        a = losses.distill_loss(sd, big.cuda()[:, 5:9], far.cuda()[:, 3:7], log_norm=ln.cuda())
        check_distill(a, distill64(s, cls[:, :4], logits[:, :4], ln, w, 1.0), w, 1.0, "f32")
        b = losses.distill_loss(sd, cls[:, :4].contiguous().cuda(), logits[:, :4].contiguous().cuda(),
                                log_norm=ln.cuda())
        assert torch.equal(a.loss, b.loss) and torch.equal(a.grad, b.grad)
        b = losses.distill_loss(sd, cls.cuda().t().contiguous().t()[:, :4],
                                far.cuda().t().contiguous().t()[:, 3:7], log_norm=ln.cuda())
        assert torch.equal(a.loss, b.loss) and torch.equal(a.grad, b.grad)
        f = losses.class_alternatives(sd, 0)
        up = torch.randn((n, 30), generator=torch.Generator().manual_seed(1)).cuda()
        x = losses.class_alternatives_grad(sd, f.norm, classes=big.cuda()[:, 5:9],
                                           grad_log_prob=up[:, 7:11])
        y = losses.class_alternatives_grad(sd, f.norm, classes=cls[:, :4].contiguous().cuda(),
                                           grad_log_prob=up[:, 7:11].contiguous())
        assert torch.equal(x, y)
        y = losses.class_alternatives_grad(
            sd, f.norm, classes=cls.cuda().t().contiguous().t()[:, :4],
            grad_log_prob=up.t().contiguous().t()[:, 7:11])
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_distill_against_differences(gpu):
    """The gradient against central differences of the kernel's own losses."""
    from warpgbm_amd import losses

    n, h = 64, 2.0 ** -6
    for K in (6, 50, 600):
        s = make_scores(n, K, "f32", "row", 9, spread=1.0)
        cls, logits, ln = lists_for(s, 4, 10, 2.0, spare=False)
        way = torch.randn((n, K), generator=torch.Generator().manual_seed(3))

        def run(x, grad=False):
            return losses.distill_loss(x.cuda(), cls.cuda(), logits.cuda(), log_norm=ln.cuda(),
                                       temperature=2.0, with_grad=grad)

        slope = (run(s + h * way).loss.double() - run(s - h * way).loss.double()).cpu() / (2 * h)
        along = (run(s, True).grad.cpu().double() * way.double()).sum(1)
        # third derivatives of a log-sum-exp of scores / T are at most 1 / T^3 of the cube of
        # the direction; two of them, T^2; the losses' own rounding
        cube = way.abs().max(1).values.double() ** 3
        assert ((slope - along).abs() <= 2 * cube * h * h / 6 + 64 * 60 * U / h).all()


# --------------------------------------------------------------------- together
def teach(s, t, a, w, k, tau, coef):
    """A student's step: the teacher's lists, the divergence, the labels."""
    from warpgbm_amd import losses

    f = losses.class_alternatives(t, k, temperature=tau)
    r = losses.distill_loss(s, f.classes, f.log_prob * tau, log_norm=0.0, weight=w, temperature=tau)
    e = losses.class_alternatives(s, 0, labels=a)
    up = -coef * w
    g = losses.class_alternatives_grad(s, e.norm, labels=a, grad_label_log_prob=up, grad=r.grad)
    return f, r, e, g


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_a_student_learns_from_a_teacher(gpu, dtype, order):
    for n, K, k in ((200, 12, 4), (100, 90, 8), (50, 700, 20), (9, 20_001, 64)):
        print_case("teach", dtype, order, n, K, k)
        tau, coef = 2.0, 0.25
        s = make_scores(n, K, dtype, order, 21, masked=0.1)
        t = make_scores(n, K, dtype, order, 22)
        g = torch.Generator().manual_seed(2)
        a = torch.randint(0, K, (n,), generator=g, dtype=torch.int32)
        w = 0.5 + torch.rand(n, generator=g)
        f, r, e, got = teach(to_gpu(s), to_gpu(t), a.cuda(), w.cuda(), k, tau, coef)
        check_alternatives(f, alternatives64(t, a, k, tau), k, label=False)
        want = distill64(s, f.classes.cpu(), f.log_prob.cpu() * tau, 0.0, w, tau)
        assert got.data_ptr() == r.grad.data_ptr()
        more, tol = alternatives_grad64(s, a, -coef * w, None, None, None, 1.0)
        # the divergence's gradient was rounded to the type before the labels' came
        first = want["grad"]
        total = first + more
        scale = (w.to(F64) * tau)[:, None]
        p, q, rr, P, Q = want["p"], want["q"], want["r"], want["P"][:, None], want["Q"][:, None]
        tol = tol + scale * U * ((STEPS + 4 * want["far"] + 64) * (p + q + rr * (P + Q))
                                 + (k + 8) * (q + rr))
        half = U if dtype == "f32" else torch.finfo(DTYPES[dtype]).eps / 2 * (1 + 1e-3)
        tol = tol + half * (first.abs() + total.abs()) + (2.0 ** -24 if dtype == "f16" else 1e-37)
        check(got, total, tol, "gradient")


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
@pytest.mark.parametrize("K", [12, 90, 700, 20_001])
def test_graphs_streams_and_same_bits(gpu, K, order):
    """Two captured steps replayed in turn with eager work between, each replay
    against the eager result on the same inputs; another stream."""
    n, k = 64, 8
    inputs = [[make_scores(n, K, "f32", order, 30 + 2 * j).cuda() for j in range(2)] for _ in "ab"]
    a = torch.randint(0, K, (n,), dtype=torch.int32).cuda()
    w = torch.ones(n).cuda()
    side = torch.cuda.Stream()
    graphs, outs = [], []
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s, t in inputs:
            teach(s, t, a, w, k, 2.0, 0.5)
    side.synchronize()
    for s, t in inputs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(teach(s, t, a, w, k, 2.0, 0.5))
        graphs.append(gr)
    for turn in range(4):
        which = turn % 2
        s, t = inputs[which]
        s.copy_(make_scores(n, K, "f32", order, 50 + turn))
        t.copy_(make_scores(n, K, "f32", order, 60 + turn))
        graphs[which].replay()
        torch.cuda.synchronize()
        f, r, e, g = teach(s, t, a, w, k, 2.0, 0.5)
        F, R, E, G = outs[which]
        for x, y in ((f.classes, F.classes), (f.log_prob, F.log_prob), (f.norm, F.norm),
                     (r.loss, R.loss), (e.entropy, E.entropy), (g, G)):
            assert torch.equal(x, y)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = teach(s, t, a, w, k, 2.0, 0.5)
        side.synchronize()
        assert torch.equal(other[3], g) and torch.equal(other[1].loss, r.loss)


# --------------------------------------------------------------------- refusals
def test_float64_forms_against_differences():
    s = make_scores(9, 7, "f32", "row", 1, masked=0.2).to(F64)
    cls, logits, ln = lists_for(s, 3, 2, 1.5, spare=False)
    w, h = torch.ones(9), 1e-5
    way = torch.randn((9, 7), generator=torch.Generator().manual_seed(1), dtype=F64)
    for norm in (None, ln):
        d = distill64(s, cls, logits, norm, w, 1.5)
        up = distill64(s + h * way, cls, logits, norm, w, 1.5)["loss"]
        down = distill64(s - h * way, cls, logits, norm, w, 1.5)["loss"]
        finite = torch.where(s > -INF, way, torch.zeros((), dtype=F64))
        assert torch.allclose((up - down) / (2 * h), (d["grad"] * finite).sum(1), atol=1e-7)


def test_refusals_without_a_gpu():
    from warpgbm_amd import losses

    s = torch.zeros((4, 8))
    c, x = torch.zeros((4, 2), dtype=torch.int32), torch.zeros((4, 2))
    for call in (lambda: losses.class_alternatives(s, 2),
                 lambda: losses.class_alternatives_grad(s, torch.zeros((4, 3))),
                 lambda: losses.distill_loss(s, c, x)):
        with pytest.raises(RuntimeError, match="GPU tensor"):
            call()
    cpu = torch.device("cpu")
    with pytest.raises(RuntimeError, match="dtype"):
        losses._list(c.long(), "classes", torch.int32, 4, 2, cpu)
    with pytest.raises(RuntimeError, match="shape"):
        losses._list(c, "classes", torch.int32, 4, 3, cpu)
    wide = torch.zeros((8, 18), dtype=torch.int32)
    for bad in (wide[::2, ::9], c[:1].expand(4, 2), c[:, :1].expand(4, 2)):
        with pytest.raises(RuntimeError, match="next to each other"):
            losses._list(bad, "classes", torch.int32, 4, 2, cpu)
    assert losses._list(c.t().contiguous().t(), "classes", torch.int32, 4, 2, cpu)[1:] == (1, 4)
    assert losses._list(c[:1], "classes", torch.int32, 1, 2, cpu)[1:] == (2, 1)
    assert losses._list(wide[:4, :1], "c", torch.int32, 4, 1, cpu)[1:] == (18, 1)
    assert losses._list(wide[:4, 3:5], "c", torch.int32, 4, 2, cpu)[1:] == (18, 1)
    assert losses._list(wide.t()[:4, :2], "c", torch.int32, 4, 2, cpu)[1:] == (1, 18)
    for t in (0.0, -1.0, INF, float("nan")):
        with pytest.raises(RuntimeError, match="temperature"):
            losses._temperature(t)


def test_c_entries_refuse_before_any_launch():
    from warpgbm_amd import _lib

    lib = _lib.load()
    one = 16  # never dereferenced

    def scores(**kw):
        f = dict(data=one, dtype=0, n_rows=4, n_classes=8, row_stride=8, class_stride=1)
        f.update(kw)
        return _lib.Scores(*f.values())

    def refused(rc, text):
        msg = lib.wgbm_last_error().decode()
        assert rc == 1000 and text in msg, (rc, msg)

    def alternatives(s=None, k=2, tau=1.0, labels=None, label=one, out=one, ws=0):
        return lib.wgbm_class_alternatives(C.byref(s or scores()), labels, k, tau, out, out, one,
                                           label, one, None if ws == 0 else one, ws, None)

    refused(alternatives(k=-1), "length")
    refused(alternatives(k=65, s=scores(n_classes=100, row_stride=100)), "length")
    refused(alternatives(k=9), "top_k")
    refused(alternatives(tau=0.0), "temperature")
    refused(alternatives(tau=float("nan")), "temperature")
    refused(alternatives(labels=one, label=None), "null pointer")
    refused(alternatives(out=None), "null pointer")
    refused(alternatives(s=scores(dtype=9)), "type code")
    wide = dict(n_classes=600, row_stride=1, class_stride=4)
    refused(alternatives(s=scores(**wide)), "workspace too small")
    refused(alternatives(s=scores(**wide), ws=4 * 600 * 4 - 1), "workspace too small")
    assert lib.wgbm_class_alternatives_workspace(C.byref(scores(**wide))) == 4 * 600 * 4
    assert lib.wgbm_class_alternatives_workspace(C.byref(scores(**wide, dtype=1))) == 4 * 600 * 2
    assert lib.wgbm_distill_loss_workspace(C.byref(scores(**wide, dtype=1))) == 4 * 600 * 4
    assert lib.wgbm_class_alternatives_grad_workspace(C.byref(scores())) == 0
    assert lib.wgbm_distill_loss_workspace(C.byref(scores(dtype=7))) == -1
    assert alternatives(s=scores(n_rows=0)) == 0

    def grad(out=None, **kw):
        f = dict(norm=one, labels=None, grad_label_log_prob=None, classes=one, classes_stride=2,
                 classes_step=1, grad_log_prob=one, grad_stride=2, grad_step=1, list_length=2, grad_entropy=None,
                 temperature=1.0)
        f.update(kw)
        args = _lib.AlternativesGradArgs(*f.values())
        return lib.wgbm_class_alternatives_grad(C.byref(scores()), C.byref(args),
                                                C.byref(out or scores()), 0, None, 0, None)

    refused(grad(list_length=65, classes_stride=65, grad_stride=65), "length")
    refused(grad(classes_stride=1), "stride")
    refused(grad(grad_stride=1), "stride")
    refused(grad(temperature=-1.0), "temperature")
    refused(grad(norm=None), "null pointer")
    refused(grad(labels=one), "null pointer")
    refused(grad(classes=None), "null pointer")
    refused(grad(out=scores(dtype=1)), "shape and type")
    refused(grad(out=scores(row_stride=1, class_stride=8)), "order")

    def distill(out=None, **kw):
        f = dict(classes=one, classes_stride=2, classes_step=1, logits=one, logits_stride=2,
                 logits_step=1, list_length=2, rest=0,
                 log_norm=None, log_norm_all=0.0, weight=None, temperature=1.0)
        f.update(kw)
        args = _lib.DistillArgs(*f.values())
        return lib.wgbm_distill_loss(C.byref(scores()), C.byref(args), one,
                                     C.byref(out) if out else None, 0, None, 0, None)

    refused(distill(list_length=0), "length")
    refused(distill(list_length=65), "length")
    refused(distill(classes_stride=1), "stride")
    refused(distill(classes_stride=1, classes_step=3), "stride")
    refused(distill(classes_stride=4, classes_step=2), "stride")
    refused(distill(logits_stride=1 << 41), "stride")
    refused(distill(temperature=0.0), "temperature")
    refused(distill(rest=1, log_norm_all=INF), "log_norm")
    refused(distill(classes=None), "null pointer")
    refused(distill(logits=None), "null pointer")
    refused(distill(out=scores(n_classes=7)), "shape and type")


@pytest.mark.gpu
def test_refusals_on_the_gpu(gpu):
    from warpgbm_amd import losses

    s = torch.zeros((4, 8)).cuda()
    c, x = torch.zeros((4, 2), dtype=torch.int32).cuda(), torch.zeros((4, 2)).cuda()
    v = torch.zeros(4).cuda()
    f = losses.class_alternatives(s, 2)

    def no(text, call):
        with pytest.raises(RuntimeError, match=text):
            call()

    for k in (-1, 9, 2.0, True, None):
        no("top_k", lambda: losses.class_alternatives(s, k))
    no("labels must have dtype", lambda: losses.class_alternatives(s, 2, labels=v))
    no("come together", lambda: losses.class_alternatives_grad(s, f.norm, labels=c[:, 0]))
    no("come together", lambda: losses.class_alternatives_grad(s, f.norm, classes=c))
    no("norm must be", lambda: losses.class_alternatives_grad(s, f.norm[:, :2], grad_entropy=v))
    no("must have shape", lambda: losses.class_alternatives_grad(
        s, f.norm, classes=c, grad_log_prob=x[:, :1]))
    no("at most 64", lambda: losses.class_alternatives_grad(
        s, f.norm, classes=torch.zeros((4, 65), dtype=torch.int32).cuda(),
        grad_log_prob=torch.zeros((4, 65)).cuda()))
    no("share", lambda: losses.class_alternatives_grad(s, f.norm, grad_entropy=v, grad=s))
    whole = torch.zeros(64).cuda()
    no("share", lambda: losses.class_alternatives_grad(
        s, whole[:12].view(4, 3), grad_entropy=v, grad=whole[:32].view(4, 8)))
    no("share", lambda: losses.distill_loss(s, c, whole[10:18].view(4, 2),
                                            grad=whole[:32].view(4, 8)))
    no("1 to 64", lambda: losses.distill_loss(s, c[:, :0], x[:, :0]))
    no("must have dtype", lambda: losses.distill_loss(s, c.long(), x))
    no("must have dtype", lambda: losses.distill_loss(s, c, x.double()))
    no("must be on", lambda: losses.distill_loss(s, c.cpu(), x))
    no("must have shape", lambda: losses.distill_loss(s, c, x[:3]))
    no("must have shape", lambda: losses.distill_loss(s, c, x, weight=v[:3]))
    no("must have shape", lambda: losses.distill_loss(s, c, x, log_norm=v[:3]))
    no("log_norm", lambda: losses.distill_loss(s, c, x, log_norm=INF))
    no("with_grad", lambda: losses.distill_loss(s, c, x, grad=torch.zeros_like(s), with_grad=False))
    no("temperature", lambda: losses.distill_loss(s, c, x, temperature=0))


# --------------------------------------------------------------------- edges of frames
def run_all(s, k, dtype, tau, seed):
    """Every operator on s with lists of k, against the float64 forms."""
    from warpgbm_amd import losses

    n, K = s.shape
    g = torch.Generator().manual_seed(seed)
    a = torch.randint(0, K, (n,), generator=g, dtype=torch.int32)
    w = 0.5 + torch.rand(n, generator=g)
    sd = to_gpu(s)
    f = losses.class_alternatives(sd, min(k, K), labels=a.cuda(), temperature=tau)
    check_alternatives(f, alternatives64(s, a, min(k, K), tau), min(k, K))
    cls, logits, ln = lists_for(s, k, seed, tau, spare=False)
    for norms in (None, ln):
        got = losses.distill_loss(sd, cls.cuda(), logits.cuda(), weight=w.cuda(), temperature=tau,
                                  log_norm=None if norms is None else norms.cuda())
        check_distill(got, distill64(s, cls, logits, norms, w, tau), w, tau, dtype)
    up = torch.randn((n, k), generator=g)
    ge = torch.randn(n, generator=g)
    got = losses.class_alternatives_grad(
        sd, f.norm, labels=a.cuda(), grad_label_log_prob=w.cuda(), classes=cls.cuda(),
        grad_log_prob=up.cuda(), grad_entropy=ge.cuda(), temperature=tau)
    grad, tol = alternatives_grad64(s, a, w, cls, up, ge, tau)
    check(got, grad, round_tol(tol, grad, dtype), "gradient")


CLASS_EDGES = [4, 5, 8, 9, 12, 13, 16, 17, 32, 33, 40, 41, 52, 53, 64, 65, 80, 81, 104, 105, 128,
               129, 160, 208, 209, 256, 257, 312, 313, 432, 433, 500, 512, 513]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_edges_of_class_major_frames(gpu, dtype):
    for K in CLASS_EDGES:
        for n, k in ((67, 64), (130, 7)):
            print_case("class edges", dtype, n, K, k)
            run_all(make_scores(n, K, dtype, "class", K, masked=0.1), k, dtype, 1.0, K + k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_edges_of_row_major_frames(gpu, dtype):
    """One class less and more than what a number of 16-byte chunks holds, up to rows that
    go in tiles."""
    VE = 4 if dtype == "f32" else 8
    for chunks in (1, 2, 3, 4, 8, 16, 32, 64, 128, 256, 512, 1024, 2048, 4096, 8192, 16384):
        for K in (chunks * VE - 1, chunks * VE, chunks * VE + 1):
            n, k = (35, 17) if chunks <= 512 else (3, 64 if K % 2 else 5)
            print_case("row edges", dtype, n, K, k)
            run_all(make_scores(n, K, dtype, "row+" if K % 2 else "row", K, masked=0.1), k, dtype,
                    2.0, K + k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_many_short_rows(gpu, dtype):
    """Rows enough for fewer threads each, a part of a workgroup left over."""
    for K, chunks in ((30, 8), (60, 16), (100, 32), (13, 4), (6, 2)):
        if dtype != "f32" and K > 8:
            K *= 2
        n = (1 << 19) // chunks + 37
        print_case("many", dtype, n, K)
        run_all(make_scores(n, K, dtype, "row", K), 5, dtype, 1.0, K)


@pytest.mark.gpu
def test_lists_past_32_bits(gpu):
    """The first and last rows of matrices of more than 2^31 elements against the same
    rows alone."""
    from warpgbm_amd import losses

    for n, K, k in ((66_000, 33_000, 9), (2_200_000, 1000, 5)):
        print_case("past 32 bits", n, K)
        s = torch.empty((n, K), dtype=torch.bfloat16, device="cuda")
        s.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
        rows = torch.cat([torch.arange(3), torch.arange(n - 5, n)]).cuda()
        a = torch.arange(n, dtype=torch.int32, device="cuda") % K
        f = losses.class_alternatives(s, k, labels=a, temperature=1.5)
        r = losses.distill_loss(s, f.classes, f.log_prob, log_norm=0.125)
        few = s[rows].contiguous()
        F = losses.class_alternatives(few, k, labels=a[rows].contiguous(), temperature=1.5)
        R = losses.distill_loss(few, F.classes, F.log_prob, log_norm=0.125)
        up = torch.ones(n, device="cuda")
        G = losses.class_alternatives_grad(few, F.norm, grad_entropy=up[:8], classes=F.classes,
                                           grad_log_prob=F.log_prob, temperature=1.5)
        for x, y in ((f.classes, F.classes), (f.log_prob, F.log_prob), (f.norm, F.norm),
                     (f.label_log_prob, F.label_log_prob), (r.loss, R.loss), (r.grad, R.grad)):
            assert torch.equal(x[rows], y)
        del r
        g = losses.class_alternatives_grad(s, f.norm, grad_entropy=up, classes=f.classes,
                                           grad_log_prob=f.log_prob, temperature=1.5)
        assert torch.equal(g[rows], G)
        del s, g, f
        torch.cuda.empty_cache()


@pytest.mark.gpu
def test_temperatures_at_their_limits(gpu):
    from warpgbm_amd import losses

    for order in ("row", "class"):
        for K in (6, 60, 700):
            s = make_scores(20, K, "f32", order, 4)
            a = torch.zeros(20, dtype=torch.int32)
            for tau in (1e-6, 1e-3, 1e3, 1e6):
                print_case("temperature", order, K, tau)
                r = losses.class_alternatives(to_gpu(s), 3, labels=a.cuda(), temperature=tau)
                check_alternatives(r, alternatives64(s, a, 3, tau), 3)
                d = losses.distill_loss(to_gpu(s), r.classes, r.log_prob.clamp(min=-1e30) * tau,
                                        log_norm=0.0, temperature=tau)
                assert torch.isfinite(d.loss).all() and torch.isfinite(d.grad).all()


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
def test_a_rest_next_to_its_border(gpu, order):
    """Whether the teacher's rest is one (2^-20 or more) is decided as in float64."""
    from warpgbm_amd import losses

    for K, k in ((6, 5), (40, 12), (300, 20), (9000, 64)):
        print_case("border", order, K, k)
        n = 400
        g = torch.Generator().manual_seed(K)
        s = torch.randn((n, K), generator=g)
        cls = torch.argsort(torch.rand((n, K), generator=g), 1)[:, :k].to(torch.int32).contiguous()
        t = torch.log_softmax(torch.randn((n, k), generator=g, dtype=F64), 1)
        # rests from 0.9 to 1.1 times the border
        rest = 2.0 ** -20 * torch.linspace(0.9, 1.1, n, dtype=F64)
        logits = (t + torch.log1p(-rest)[:, None]).float()
        w = torch.ones(n)
        left = 1 - logits.to(F64).exp().sum(1)
        # (the sum's own rounding in float64)
        assert ((left - 2.0 ** -20).abs() > 1e-13).all()
        want = distill64(place(s, order), cls, logits, 0.0, w, 1.0)
        got = losses.distill_loss(to_gpu(place(s, order)), cls.cuda(), logits.cuda(), log_norm=0.0)
        check_distill(got, want, w, 1.0, "f32")
        # the others' share of the gradient: P of them without a rest, P - Q with one
        others = torch.ones((n, K), dtype=torch.bool).scatter_(1, cls.long(), False)
        share = torch.where(others, got.grad.cpu().to(F64), 0.0).sum(1)
        assert ((share - (want["P"] - want["Q"])).abs() <= U * (STEPS + 64) * want["P"] + 2e-8).all()


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
def test_distill_of_a_small_listed_share(gpu, order):
    """A softened teacher whose list is a small part of it: the others' gradient is a
    difference of shares next to 1, which the listed shares' digits give."""
    from warpgbm_amd import losses

    for n, K in ((40, 400), (12, 3000), (5, 30_000)):
        print_case("small share", order, n, K)
        g = torch.Generator().manual_seed(K)
        s = place(torch.randn((n, K), generator=g), order)
        t = 0.8 * s + 0.5 * torch.randn((n, K), generator=g)
        logits, cls = (x[:, :2].contiguous() for x in torch.sort(t, dim=1, descending=True))
        cls = cls.to(torch.int32)
        ln = torch.logsumexp(t.double() / 4.0, 1).float()
        got = losses.distill_loss(to_gpu(s), cls.cuda(), logits.cuda(), log_norm=ln.cuda(),
                                  temperature=4.0)
        want = distill64(s, cls, logits, ln, torch.ones(n), 4.0)
        check_distill(got, want, torch.ones(n), 4.0, "f32")
        # listed: p_k and q_k of a few roundings each (and log norm's, which all share);
        # others: (listed q - listed p) r_k, the same
        p, q, r = want["p"], want["q"], want["r"]
        small = (torch.where(q > 0, p, 0.0).sum(1, keepdim=True) + q.sum(1, keepdim=True))
        tol = 4.0 * U * (STEPS + 128) * torch.where(q > 0, p + q, small * r)
        check(got.grad, want["grad"], tol + U * want["grad"].abs(), "gradient")


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
def test_distill_where_the_teacher_s_best_class_is_closed(gpu, order):
    """The row may not take the class that has almost all of the teacher's share: what is
    left, scaled to sum 1, keeps its digits."""
    from warpgbm_amd import losses

    for n, K in ((64, 4), (64, 40), (16, 900)):
        print_case("closed", order, n, K)
        g = torch.Generator().manual_seed(K)
        s = torch.randn((n, K), generator=g)
        t = torch.randn((n, K), generator=g)
        t[torch.arange(n), torch.arange(n) % K] += torch.linspace(2.0, 11.0, n)
        best = torch.sort(t, dim=1, descending=True)
        logits = best.values[:, :3].contiguous()
        cls = best.indices[:, :3].to(torch.int32).contiguous()
        s[torch.arange(n), cls[:, 0].long()] = -INF
        tau = 0.7  # (not a float32)
        ln = torch.logsumexp(t.double() / tau, 1).float()
        got = losses.distill_loss(to_gpu(place(s, order)), cls.cuda(), logits.cuda(),
                                  log_norm=ln.cuda(), temperature=tau)
        w = torch.ones(n)
        want = distill64(place(s, order), cls, logits, ln, w, tau)
        check_distill(got, want, w, tau, "f32")
        # sums of what is left: a few roundings of each share, not of the closed one (log_norm's
        # own rounding is an input)
        gap = torch.where(want["q"] > 0, (want["q"].log() + want["far"]).abs(), 0.0)
        far_rest = torch.where(want["Q"] > 0, (want["Q"].clamp(min=1e-30).log() - want["rest"]).abs(),
                               0.0)
        tol = tau * tau * U * (STEPS * want["lost"] + 24 * (2 + (want["q"] * gap).sum(1) + far_rest))
        check(got.loss, want["loss"], tol + U * want["loss"], "loss")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,order,n", [("f16", "class", 2), ("f32", "row", 1)])
def test_rows_of_the_most_classes(gpu, dtype, order, n):
    """2^24 classes: rows in the most tiles, and their copy where they are class-major."""
    K = 1 << 24
    print_case("most classes", dtype, order, n, K)
    run_all(make_scores(n, K, dtype, order, 77), 64, dtype, 1.0, 78)


@pytest.mark.gpu
@pytest.mark.parametrize("K,order", [(90, "class"), (700, "class"), (20_001, "row")])
def test_two_streams_at_once(gpu, K, order):
    """Steps that run beside each other have the bits of steps that run alone."""
    n, k = 3000, 8
    a = torch.randint(0, K, (n,), dtype=torch.int32).cuda()
    w = torch.ones(n).cuda()
    inputs = [[to_gpu(make_scores(n, K, "f32", order, 80 + 2 * j + i)) for i in range(2)]
              for j in range(2)]
    alone = [teach(s, t, a, w, k, 2.0, 0.5) for s, t in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    got = [[], []]
    for _ in range(5):
        for j, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[j].append(teach(*inputs[j], a, w, k, 2.0, 0.5))
    torch.cuda.synchronize()
    for j in range(2):
        f, r, e, g = alone[j]
        for F, R, E, G in got[j]:
            for x, y in ((f.classes, F.classes), (f.log_prob, F.log_prob), (r.loss, R.loss),
                         (e.entropy, E.entropy), (g, G)):
                assert torch.equal(x, y)

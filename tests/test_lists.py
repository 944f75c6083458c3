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
    check(torch.where(fin, r.log_prob.cpu().to(F64), 0.0), torch.where(fin, w, 0.0), tol + 1e-300,
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

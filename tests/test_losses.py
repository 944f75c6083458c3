"""Losses of class scores and of paired scores against plain float64 forms.

The float64 forms define the losses; their gradients come from autograd, which
shares nothing with the kernels' formulas.  Tolerances count roundings: 2^-24
of each float32 step, half a step of the gradient's type (torch.finfo(t).eps /
2 of the value, and half of float16's smallest subnormal number).
"""
import math
import sys

import numpy as np
import pytest
import torch

from conftest import print_case

F64 = torch.float64
U = 2.0 ** -24
# roundings of a row's statistics: 256 classes added one after the other by a
# thread at most, joins, exponentials and logarithms
STEPS = 320


# --------------------------------------------------------------------- float64 forms
def log_softmax64(s):
    """log softmax over classes; rows without a class give 0 everywhere."""
    s = s.to(F64)
    empty = (s == -math.inf).all(1, keepdim=True)
    s = torch.where(empty, torch.zeros_like(s), s)
    m = s.max(1, keepdim=True).values.detach()
    return s - m - torch.log(torch.exp(s - m).sum(1, keepdim=True))


def live_rows(s, label=None, weight=None):
    live = ~(s == -math.inf).all(1)
    if label is not None:
        live &= (label >= 0) & (label < s.shape[1])
    if weight is not None:
        live &= weight != 0
    return live


def policy64(s, a, old, adv, w, ref_lp, ref_s, clip, kl_coef):
    """(weighted losses, log-probs, kl) per row, differentiable in s (rows left
    out must have been replaced by finite scores)."""
    L = log_softmax64(s)
    lp = L.gather(1, a.long()[:, None])[:, 0]
    r = torch.exp(lp - old.to(F64))
    A = adv.to(F64)
    free, held = r * A, r.clamp(1 - clip[0], 1 + clip[1]) * A
    loss = -torch.minimum(free, held)
    kl = None
    if ref_lp is not None:
        x = ref_lp.to(F64) - lp
        kl = torch.exp(x) - x - 1
    elif ref_s is not None:
        P = L.exp()
        d = torch.where(P > 0, L - log_softmax64(ref_s), torch.zeros_like(L))
        kl = (P * d).sum(1)
    if kl is not None:
        loss = loss + kl_coef * kl
    return loss * w.to(F64), lp, kl


def preference64(lp, pairs, n_seq, seg, ref, w, beta, smooth):
    """(losses, margins), differentiable in lp."""
    u = lp.to(F64) - (ref.to(F64) if ref is not None else 0.0)
    if seg is None:
        Us = u
    else:
        Us = torch.stack([u[int(seg[k]):int(seg[k + 1])].sum() for k in range(n_seq)]) \
            if n_seq else u[:0]
    m = Us[pairs[:, 0].long()] - Us[pairs[:, 1].long()]
    z = beta * m
    ls = torch.nn.functional.logsigmoid
    loss = -((1 - smooth) * ls(z) + smooth * ls(-z))
    return loss * (w.to(F64) if w is not None else 1.0), m


# --------------------------------------------------------------------- inputs
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def make_scores(n, K, dtype, order, seed, masked=0.0, spread=2.0):
    """[n, K] scores on the CPU as they sit in memory: "row", "class", and both
    with strides and a start that is aligned to the element only."""
    g = torch.Generator().manual_seed(seed)
    v = spread * torch.randn((n, K), generator=g)
    if masked:
        shut = torch.rand((n, K), generator=g) < masked
        if n and K:
            shut[torch.arange(n), torch.randint(0, K, (n,), generator=g)] = False
        v[shut] = -math.inf
    v = v.to(DTYPES[dtype])
    if order == "row":
        return v
    if order == "class":
        return v.t().contiguous().t()
    if order == "row+":
        big = torch.full((n, K + 5), float("nan"), dtype=v.dtype)
        big[:, 3:3 + K] = v
        return big[:, 3:3 + K]
    big = torch.full((K, n + 7), float("nan"), dtype=v.dtype)
    big[:, 1:1 + n] = v.t()
    return big[:, 1:1 + n].t()


def to_gpu(t):
    """A copy on the GPU that keeps strides and the start's offset."""
    whole = t.untyped_storage().nbytes() // t.element_size()
    flat = torch.as_strided(t, (whole,), (1,), 0).cuda()
    return torch.as_strided(flat, t.shape, t.stride(), t.storage_offset())


def grad_tol(want, scale, dtype):
    """Per-element bound: the row's scale times the float32 steps, and the
    rounding to the gradient's type."""
    fin = torch.finfo(DTYPES[dtype])
    tiny = 2.0 ** -25 if dtype == "f16" else 0.0
    half = 0.0 if dtype == "f32" else fin.eps / 2
    return STEPS * U * scale[:, None] + (half * (1 + 1e-3)) * want.abs() + tiny


def check(got, want, tol, what):
    got = got.detach().cpu().to(F64)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), (got - want).abs().max().item(),
                           got[bad][:4], want[bad][:4])


SHAPES = [(1, 1), (5, 1), (1, 2), (1, 3), (3, 2), (64, 10), (65, 7), (257, 10), (1000, 3),
          (63, 31), (130, 32), (70, 33), (33, 64), (9, 65), (300, 100), (21, 257), (50, 513),
          (7, 1000), (3, 4097), (2, 20001)]
# rows enough for a workgroup to take several a thread group, a part of a
# workgroup left over
MANY_ROWS = [(262_147, 10), (131_075, 33), (66_000, 65), (33_001, 130), (17_003, 257),
             (8_300, 700)]
ORDERS = ["row", "class", "row+", "class+"]


def norm_tol(L):
    """Log-probabilities: the sum's relative error, and the roundings of two
    differences."""
    return U * (STEPS + 4 * (L.abs() + 12))


# --------------------------------------------------------------------- log-probabilities
@pytest.mark.gpu
@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_log_probs_and_gradient(gpu, dtype, order):
    from warpgbm_amd import losses

    for j, (n, K) in enumerate(SHAPES):
        print_case("log_probs", dtype, order, n, K)
        s = make_scores(n, K, dtype, order, 100 + j, masked=0.2 if j % 2 else 0.0)
        g = torch.Generator().manual_seed(j)
        a = torch.randint(0, K, (n,), generator=g, dtype=torch.int32)
        if n > 4:
            a[1], a[3] = -1, K
            s[2] = -math.inf
        up = torch.randn(n, generator=g)
        up[n // 2] = 0.0
        sd = to_gpu(s)
        assert sd.stride() == s.stride()
        r = losses.class_log_probs(sd, a.cuda())
        live = live_rows(s, a)
        safe = torch.where(live[:, None], s.to(F64), torch.zeros((), dtype=F64))
        safe.requires_grad_(True)
        L = log_softmax64(safe)
        lp = L.gather(1, a.long().clamp(0, K - 1)[:, None])[:, 0]
        taken = live & (lp > -math.inf)
        want = torch.where(live, lp, torch.zeros_like(lp)).detach()
        fin = want > -math.inf
        check(r.log_prob[fin.cuda()], want[fin], norm_tol(want[fin]), "log_prob")
        assert (r.log_prob.cpu()[~fin] == -math.inf).all()
        has = live_rows(s)
        check(r.norm[has.cuda(), 0], s[has].to(F64).max(1).values, 0.0, "maximum")
        assert (r.norm.cpu()[~has] == torch.tensor([-math.inf, 0.0])).all()
        got = losses.class_log_probs_grad(sd, a.cuda(), r.norm, up.cuda())
        assert got.dtype == s.dtype and got.shape == s.shape
        (lp[taken] * up.to(F64)[taken]).sum().backward()
        # (a label at -inf: the formula's gradient, with p of the label 0)
        P = torch.softmax(torch.where(has[:, None], s.to(F64), torch.zeros((), dtype=F64)), 1)
        grad = safe.grad.clone()
        odd = live & ~taken
        grad[odd] = -P[odd] * up.to(F64)[odd, None]
        grad[odd, a[odd].long()] += up.to(F64)[odd]
        check(got, grad, grad_tol(grad, up.abs().to(F64), dtype), "gradient")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_many_rows(gpu, dtype):
    """The first, some middle and the last rows of large matrices against the
    same rows alone, which float64 forms check above (a row's results may differ
    by the order of its sums)."""
    from warpgbm_amd import losses

    for n, K in MANY_ROWS:
        print_case("many rows", dtype, n, K)
        g = torch.Generator(device="cuda").manual_seed(K)
        s = (2 * torch.randn((n, K), generator=g, device="cuda")).to(DTYPES[dtype])
        a = torch.randint(-1, K, (n,), generator=g, device="cuda", dtype=torch.int32)
        old = -2 - torch.rand(n, generator=g, device="cuda")
        adv = torch.randn(n, generator=g, device="cuda")
        w = (torch.rand(n, generator=g, device="cuda") < 0.9).float()
        f = losses.class_log_probs(s, a)
        p = losses.policy_loss(s, a, old, adv, weight=w, ref_log_prob=old, kl_coef=0.1)
        one = torch.ones(n, device="cuda")
        b = losses.class_log_probs_grad(s, a, f.norm, one)
        for at in (0, n // 2 + 1, n - 301):
            r = slice(at, at + 301)
            f1 = losses.class_log_probs(s[r], a[r])
            p1 = losses.policy_loss(s[r], a[r], old[r], adv[r], weight=w[r], ref_log_prob=old[r],
                                    kl_coef=0.1)
            # log-probabilities down to some -20: 2 STEPS of rounding
            assert torch.allclose(f.log_prob[r], f1.log_prob, rtol=0, atol=2 * STEPS * U)
            assert torch.allclose(p.log_prob[r], p1.log_prob, rtol=0, atol=2 * STEPS * U)
            size = (1 + adv[r].abs()) * (1 + torch.exp(p1.log_prob - old[r]))
            assert ((p.loss[r] - p1.loss).abs() <= 60 * STEPS * U * size).all()
            fin = torch.finfo(s.dtype)
            step = (0.0 if dtype == "f32" else fin.eps) + 1e-30
            tol = 60 * STEPS * U * size[:, None] + step * p1.grad[:].float().abs() + 2.0 ** -24
            assert ((p.grad[r].float() - p1.grad.float()).abs() <= tol).all()
            b1 = losses.class_log_probs_grad(s[r], a[r], f1.norm, one[r])
            tol = STEPS * U + step * b1.float().abs() + 2.0 ** -24
            assert ((b[r].float() - b1.float()).abs() <= tol).all()


# --------------------------------------------------------------------- policy
def policy_inputs(n, K, dtype, order, seed, masked=0.0):
    s = make_scores(n, K, dtype, order, seed, masked)
    g = torch.Generator().manual_seed(seed + 1)
    p = torch.softmax(s.float(), 1)
    a = torch.multinomial(p, 1, generator=g)[:, 0].to(torch.int32)
    lp = log_softmax64(s).gather(1, a.long()[:, None])[:, 0].float()
    d = dict(s=s, a=a, old=lp + 0.3 * torch.randn(n, generator=g),
             adv=torch.randn(n, generator=g), w=0.5 + torch.rand(n, generator=g),
             ref=lp + 0.4 * torch.randn(n, generator=g))
    shift = (0.5 * torch.randn((n, K), generator=g)).to(s.dtype)
    rs = make_scores(n, K, dtype, order, seed, masked)
    rs += shift
    d["ref_s"] = rs
    if n > 4:
        d["w"][1] = 0.0
        d["adv"][2] = 0.0
        d["a"][3] = -1
        s[1], s[3] = float("nan"), float("nan")
        s[4], rs[4] = -math.inf, -math.inf
    return d


def policy_want(d, kl, clip, c):
    s, a, w = d["s"], d["a"], d["w"]
    live = live_rows(s, a, w)
    safe = torch.where(live[:, None], s.to(F64), torch.zeros((), dtype=F64)).requires_grad_(True)
    ref_s = None
    if kl == "exact":
        ref_s = torch.where(live[:, None], d["ref_s"].to(F64), torch.zeros((), dtype=F64))
    a0 = torch.where(live, a, torch.zeros_like(a))
    loss, lp, k = policy64(safe, a0, d["old"], d["adv"], w, d["ref"] if kl == "sampled" else None,
                           ref_s, clip, c)
    zero = torch.zeros((), dtype=F64)
    loss = torch.where(live, loss, zero)
    loss.sum().backward()
    keep = torch.isfinite(safe.grad)
    assert keep.all()
    k = torch.where(live, k, zero).detach() if k is not None else None
    return loss.detach(), torch.where(live, lp, zero).detach(), k, safe.grad, live


def policy_scales(d, kl, c, want_kl, live):
    """Sizes that roundings are relative to: of the row's loss, and of its
    gradient's coefficients."""
    lp = log_softmax64(torch.where(live[:, None], d["s"].to(F64), torch.zeros((), dtype=F64)))
    lpa = lp.gather(1, d["a"].long().clamp(0, lp.shape[1] - 1)[:, None])[:, 0]
    reach = 1 + lpa.abs() + d["old"].abs().to(F64)
    ratio = torch.exp(lpa - d["old"].to(F64))
    scale = d["adv"].abs().to(F64) * ratio * reach
    if kl == "sampled":
        scale = scale + c * torch.exp(d["ref"].to(F64) - lpa) * (reach + d["ref"].abs().to(F64))
        scale = scale + c * (1 + (d["ref"].to(F64) - lpa).abs())
    if kl == "exact":
        # the divergence's terms: p |log p - log q| with logarithms of up to
        # some tens
        scale = scale + c * (30.0 + want_kl)
    return torch.where(live, scale * d["w"].to(F64), torch.zeros((), dtype=F64))


def run_policy(d, kl, clip, c, **kw):
    from warpgbm_amd import losses

    return losses.policy_loss(
        to_gpu(d["s"]), d["a"].cuda(), d["old"].cuda(), d["adv"].cuda(), weight=d["w"].cuda(),
        ref_log_prob=d["ref"].cuda() if kl == "sampled" else None,
        ref_scores=to_gpu(d["ref_s"]) if kl == "exact" else None, clip=clip, kl_coef=c, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("kl", ["none", "sampled", "exact"])
@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_policy_loss(gpu, dtype, order, kl):
    clip, c = (0.2, 0.3), 0.25
    for j, (n, K) in enumerate(SHAPES):
        print_case("policy", dtype, order, kl, n, K)
        d = policy_inputs(n, K, dtype, order, 200 + j, masked=0.2 if j % 2 else 0.0)
        loss, lp, k, grad, live = policy_want(d, kl, clip, c)
        scale = policy_scales(d, kl, c, k, live)
        r = run_policy(d, kl, clip, c)
        check(r.log_prob, lp, norm_tol(lp), "log_prob")
        check(r.loss, loss, STEPS * U * (scale + d["w"].to(F64)), "loss")
        if kl == "none":
            assert r.kl is None
        else:
            unit = torch.where(live, scale / d["w"].to(F64) / c, torch.zeros((), dtype=F64))
            check(r.kl, k, STEPS * U * (unit + 1), "kl")
        check(r.grad, grad, grad_tol(grad, scale, dtype), "gradient")
        # the losses alone; and added to a gradient that is there
        alone = run_policy(d, kl, clip, c, with_grad=False)
        assert alone.grad is None and torch.equal(alone.loss, r.loss)
        before = make_scores(n, K, dtype, order, 900 + j)
        base = to_gpu(before)
        again = run_policy(d, kl, clip, c, grad=base)
        assert again.grad is base
        both = before.to(F64) + grad
        tol = grad_tol(both, scale + before.abs().to(F64).amax(1), dtype)
        check(base, both, tol, "added gradient")
        keep = ~live
        assert torch.equal(base.cpu()[keep], before[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
@pytest.mark.parametrize("side", ["high", "low"])
def test_policy_ratio_next_to_the_border(gpu, order, side):
    """Ratios within float32's error of a border are clipped as in float64."""
    clip = (0.2, 0.25)
    for n, K in ((4096, 5), (256, 700), (64, 5000)):
        print_case("border", order, side, n, K)
        d = policy_inputs(n, K, "f32", order, 31)
        live = live_rows(d["s"], d["a"], d["w"])
        safe = torch.where(live[:, None], d["s"].to(F64), torch.zeros((), dtype=F64))
        lp = log_softmax64(safe).gather(1, d["a"].long().clamp(min=0)[:, None])[:, 0]
        edge = math.log(1 + clip[1]) if side == "high" else math.log(1 - clip[0])
        d["old"] = (lp - edge).float()  # off the border by the rounding of old alone
        d["adv"] = d["adv"].abs() + 0.1
        if side == "low":
            d["adv"] = -d["adv"]
        loss, lp, _, grad, live = policy_want(d, "none", clip, 0.0)
        r = run_policy(d, "none", clip, 0.0)
        scale = policy_scales(d, "none", 0.0, None, live)
        stopped = (grad == 0).all(1) & live
        assert 0.2 * n < int(stopped.sum()) < 0.8 * n  # both outcomes are met
        check(r.grad, grad, grad_tol(grad, scale, "f32"), "gradient")


@pytest.mark.gpu
def test_policy_extreme_rows(gpu):
    """Ratios that overflow, labels of probability 0, the type's lowest values
    as masks, NaN and infinite scores."""
    from warpgbm_amd import losses

    low = torch.finfo(torch.float32).min
    s = torch.tensor([[0.0, 1.0, 2.0], [0.0, -math.inf, 1.0], [low, low, low], [low, 3.0, low],
                      [float("nan"), 0.0, 0.0], [math.inf, 0.0, 0.0], [-math.inf] * 3])
    a = torch.tensor([0, 1, 2, 1, 1, 1, 0], dtype=torch.int32)
    old = torch.tensor([-200.0, -1.0, math.log(1 / 3), 0.0, -1.0, -1.0, -1.0])
    adv = torch.tensor([1.0, 1.0, 2.0, 1.0, 1.0, 1.0, 1.0])
    for order in ("row", "class"):
        sd = s.cuda() if order == "row" else s.t().contiguous().cuda().t()
        r = losses.policy_loss(sd, a.cuda(), old.cuda(), adv.cuda(), clip=(0.2, 0.2))
        loss, lp, g = r.loss.cpu(), r.log_prob.cpu(), r.grad.cpu()
        assert loss[0] == pytest.approx(-1.2, rel=1e-6) and (g[0] == 0).all()
        assert lp[1] == -math.inf and loss[1] == 0 and (g[1] == 0).all()
        assert lp[2] == pytest.approx(math.log(1 / 3), rel=1e-6)
        assert np.allclose(g[2], [2 / 3, 2 / 3, -4 / 3], rtol=1e-5)
        assert lp[3] == 0 and loss[3] == pytest.approx(-1.0) and (g[3] == 0).all()
        assert torch.isnan(loss[4]) and torch.isnan(g[4]).all()
        assert torch.isnan(loss[5]) and torch.isnan(lp[5])
        assert loss[6] == 0 and lp[6] == 0 and (g[6] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("K", [3, 40, 700, 6000])
def test_policy_against_a_reference_that_excludes_a_class(gpu, K):
    """The divergence is infinite then; it does no harm where it does not count,
    nor does a class of probability 0 that the reference allows."""
    from warpgbm_amd import losses

    g = torch.Generator().manual_seed(K)
    for order in ("row", "class"):
        s = torch.randn((4, K), generator=g)
        r = s + 0.1
        r[0, 1] = -math.inf
        s[1, 2] = -math.inf
        a = torch.zeros(4, dtype=torch.int32)
        old, adv = torch.full((4,), -2.0), torch.ones(4)
        put = (lambda t: t.cuda()) if order == "row" else (lambda t: t.t().contiguous().cuda().t())
        plain = losses.policy_loss(put(s), a.cuda(), old.cuda(), adv.cuda())
        zero = losses.policy_loss(put(s), a.cuda(), old.cuda(), adv.cuda(), ref_scores=put(r))
        assert torch.equal(zero.loss, plain.loss)
        assert torch.allclose(zero.grad, plain.grad, rtol=1e-5, atol=1e-7)
        assert zero.kl[0] == math.inf and torch.isfinite(zero.kl[1:]).all()
        some = losses.policy_loss(put(s), a.cuda(), old.cuda(), adv.cuda(), ref_scores=put(r),
                                  kl_coef=0.5)
        assert some.loss[0] == math.inf
        assert torch.isfinite(some.loss[1:]).all() and torch.isfinite(some.grad[1:]).all()
        far = losses.policy_loss(put(s), a.cuda(), old.cuda(), adv.cuda(), kl_coef=0.0,
                                 ref_log_prob=torch.full((4,), math.inf).cuda())
        assert torch.equal(far.loss, plain.loss) and (far.kl == math.inf).all()


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
def test_very_long_rows(gpu, order):
    """Rows past every frame: ranges, joined."""
    for dtype, n, K in (("f32", 3, 300_001), ("bf16", 2, 140_003), ("f16", 70, 131_080)):
        for kl in ("sampled", "exact"):
            print_case("long rows", order, dtype, n, K, kl)
            d = policy_inputs(n, K, dtype, order, 61)
            loss, lp, k, grad, live = policy_want(d, kl, (0.2, 0.2), 0.1)
            scale = policy_scales(d, kl, 0.1, k, live)
            r = run_policy(d, kl, (0.2, 0.2), 0.1)
            check(r.log_prob, lp, norm_tol(lp), "log_prob")
            check(r.loss, loss, STEPS * U * (scale + d["w"].to(F64)), "loss")
            check(r.grad, grad, grad_tol(grad, scale, dtype), "gradient")


# --------------------------------------------------------------------- balance
def balance_want(s, mask, k, coef):
    live = live_rows(s)
    if mask is not None:
        live &= mask
    n = int(live.sum())
    x = s.to(F64)[live].requires_grad_(True)
    K = s.shape[1]
    P = log_softmax64(x).exp()
    order = torch.sort(s[live].to(F64), dim=1, descending=True, stable=True)
    counts = torch.bincount(order.indices[:, :k][order.values[:, :k] > -math.inf], minlength=K)
    f = counts.to(F64) / max(n * k, 1)
    prob = P.sum(0) / max(n, 1)
    loss = coef * K * (f * prob).sum()
    grad = torch.zeros(s.shape, dtype=F64)
    if n:
        loss.backward()
        grad[live] = x.grad
    return loss.detach(), counts, prob.detach(), grad, live


BALANCE_SHAPES = [s for s in SHAPES if s[1] <= 4096] + [(5, 4096), (2000, 16), (129, 2048),
                                                        (5000, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_balance_loss(gpu, dtype, order):
    from warpgbm_amd import losses

    for j, (n, K) in enumerate(BALANCE_SHAPES):
        top_k = [1, 2, 8, 3][j % 4]
        top_k = min(top_k, K)
        print_case("balance", dtype, order, n, K, top_k)
        s = make_scores(n, K, dtype, order, 300 + j, masked=0.2 if j % 2 else 0.0)
        mask = torch.rand(n, generator=torch.Generator().manual_seed(j)) < 0.8
        if n > 4:
            s[2] = -math.inf
            mask[1] = False
            s[1] = float("nan")
        else:
            mask = None
        coef = 3.0 * n
        loss, counts, prob, grad, live = balance_want(s, mask, top_k, coef)
        sd = to_gpu(s)
        md = mask.cuda() if mask is not None else None
        r = losses.balance_loss(sd, top_k=top_k, mask=md, coef=coef)
        assert torch.equal(r.counts.cpu(), counts)
        # each probability STEPS roundings, a partial sum over rows as many again
        check(r.prob, prob, 2 * STEPS * U * prob + 1e-12, "prob")
        check(r.loss, loss, 2 * STEPS * U * loss.abs() + 1e-12, "loss")
        nl = max(int(live.sum()), 1)
        f = counts.to(F64) / (nl * top_k)
        P = torch.zeros(s.shape, dtype=F64)
        P[live] = torch.softmax(s[live].to(F64), 1)
        unit = coef * K / nl * (P * (f + (P @ f)[:, None]))
        tol = STEPS * U * unit.amax(1) + 1e-12
        check(r.grad, grad, grad_tol(grad, torch.zeros(n, dtype=F64), dtype) + tol[:, None], "grad")
        alone = losses.balance_loss(sd, top_k=top_k, mask=md, coef=coef, with_grad=False)
        assert alone.grad is None and torch.equal(alone.loss, r.loss)
        assert torch.equal(alone.prob, r.prob)
        before = make_scores(n, K, dtype, order, 700 + j)
        base = to_gpu(before)
        losses.balance_loss(sd, top_k=top_k, mask=md, coef=coef, grad=base)
        both = before.to(F64) + grad
        check(base, both, grad_tol(both, U * before.abs().to(F64).amax(1) / U, dtype)
              + tol[:, None], "added gradient")
        keep = ~live
        assert torch.equal(base.cpu()[keep], before[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
def test_balance_ties_and_nothing_left(gpu, order):
    from warpgbm_amd import losses

    for K in (4, 40, 600):
        s = torch.zeros((6, K))
        s[1, 1] = s[1, 3] = 2.0
        s[3, 2:] = -math.inf  # two classes left, three asked for
        sd = s.cuda() if order == "row" else s.t().contiguous().cuda().t()
        r = losses.balance_loss(sd, top_k=3)
        want = torch.zeros(K, dtype=torch.int64)
        for row in ([0, 1, 2], [1, 3, 0], [0, 1, 2], [0, 1], [0, 1, 2], [0, 1, 2]):
            want[row] += 1
        assert torch.equal(r.counts.cpu(), want)
        none = losses.balance_loss(sd, mask=torch.zeros(6, dtype=torch.bool, device="cuda"))
        assert none.loss.item() == 0 and not none.counts.any() and not none.prob.any()
        assert not none.grad.any()


# --------------------------------------------------------------------- preferences
def pref_case(kind, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "hub":
        # one item in more pairs than a piece holds, some in a few hundred
        n = S = 3000
        seg = None
        pairs = torch.randint(0, n, (40_000, 2), generator=g)
        pairs[::2, 0] = 5
        pairs[1::100, 1] = 2999
        pairs[:, 1] = torch.where(torch.arange(40_000) % 50 == 0, 700, pairs[:, 1])
    elif kind == "items":
        n = S = 1000
        seg = None
        pairs = torch.randint(0, n, (3000, 2), generator=g)
        pairs[5, 1] = pairs[5, 0]           # an item against itself
        pairs[7] = pairs[6]                 # the same pair twice
        pairs[1000:1900, 0] = 17            # one item in very many pairs
    elif kind == "two":
        n = S = 2
        seg, pairs = None, torch.tensor([[1, 0]])
    else:
        S = {"sequences": 400, "disjoint": 400, "long": 5, "empty": 6, "tail": 50}[kind]
        top = {"sequences": 60, "disjoint": 60, "long": 30_000, "empty": 1, "tail": 4}[kind]
        length = torch.randint(0, top, (S,), generator=g)
        if kind == "tail":
            length[:] = 3
        length[S // 2] = 0
        if kind == "long":
            length[1] = 1
        seg = torch.zeros(S + 1, dtype=torch.int64)
        seg[1:] = length.cumsum(0)
        n = int(seg[-1]) + (11 if kind != "tail" else 9000)
        if kind in ("disjoint", "tail"):
            # (some sequences in no pair)
            pairs = torch.randperm(S, generator=g).reshape(-1, 2)[3:]
        else:
            pairs = torch.randint(0, S, (700, 2), generator=g)
    P = pairs.shape[0]
    d = dict(n=n, S=S, seg=seg, pairs=pairs.to(torch.int32),
             lp=-2 * torch.rand(n, generator=g), w=0.5 + torch.rand(P, generator=g))
    d["ref"] = d["lp"] + 0.2 * torch.randn(n, generator=g)
    if P > 20:
        d["w"][11] = 0.0
    return d


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["plain", "reference", "weights"])
@pytest.mark.parametrize("kind", ["items", "hub", "two", "sequences", "disjoint", "tail", "long",
                                  "empty"])
def test_preference_loss(gpu, kind, how):
    from warpgbm_amd import losses

    print_case("preference", kind, how)
    d = pref_case(kind, 41)
    beta, smooth = (0.7, 0.0) if how == "plain" else (0.25, 0.1)
    ref = d["ref"] if how == "reference" else None
    w = d["w"] if how == "weights" else None
    lp = d["lp"].to(F64).requires_grad_(True)
    loss, margin = preference64(lp, d["pairs"], d["S"], d["seg"], ref, w, beta, smooth)
    loss.sum().backward()
    margin, loss = margin.detach(), loss.detach()
    if w is not None:
        margin = torch.where(w == 0, torch.zeros_like(margin), margin)
    plan = losses.PreferencePlan(d["pairs"].cuda(), d["n"],
                                 segments=d["seg"].cuda() if d["seg"] is not None else None)
    kw = dict(ref_log_prob=ref.cuda() if ref is not None else None,
              weight=w.cuda() if w is not None else None, beta=beta, label_smoothing=smooth)
    r = losses.preference_loss(d["lp"].cuda(), plan, **kw)
    # margins: float64 sums, one rounding; z = beta m rounded to float32, then
    # some float32 steps of numbers no larger than 1 + |z|
    z = (beta * margin).abs()
    unit = w.to(F64) if w is not None else torch.ones_like(z)
    check(r.margin, margin, 1.01 * U * margin.abs() + 1e-12, "margin")
    check(r.loss, loss, 16 * U * unit * (1 + z), "loss")
    slope = unit * beta * 16 * U * (1 + z.clamp(max=20))
    per = torch.zeros(max(d["S"], 1), dtype=F64)
    per.index_add_(0, d["pairs"][:, 0].long(), slope)
    per.index_add_(0, d["pairs"][:, 1].long(), slope)
    if d["seg"] is None:
        tol = per
    else:
        tol = torch.zeros(d["n"], dtype=F64)
        tol[:int(d["seg"][-1])] = per.repeat_interleave(d["seg"].diff())
    check(r.grad, lp.grad, tol + 1.01 * U * lp.grad.abs(), "gradient")
    alone = losses.preference_loss(d["lp"].cuda(), plan, with_grad=False, **kw)
    assert alone.grad is None and torch.equal(alone.loss, r.loss)
    # host arrays make the same plan; the same call gives the same bits
    host = losses.PreferencePlan(d["pairs"].numpy(), d["n"], device="cuda",
                                 segments=d["seg"].numpy() if d["seg"] is not None else None)
    again = losses.preference_loss(d["lp"].cuda(), host, **kw)
    assert torch.equal(again.grad, r.grad) and torch.equal(again.margin, r.margin)


@pytest.mark.gpu
def test_preference_left_out_and_extreme(gpu):
    """Pairs of weight 0 are not read; infinite and large margins keep losses
    and gradients finite where they are."""
    from warpgbm_amd import losses

    lp = torch.tensor([0.0, 500.0, -500.0, float("nan"), 1e-3])
    pairs = torch.tensor([[1, 2], [2, 1], [3, 0], [4, 0]], dtype=torch.int32)
    w = torch.tensor([1.0, 1.0, 0.0, 1.0])
    plan = losses.PreferencePlan(pairs.cuda(), 5)
    r = losses.preference_loss(lp.cuda(), plan, weight=w.cuda(), beta=1.0)
    assert r.loss.cpu().tolist()[:3] == [0.0, 1000.0, 0.0]
    assert r.margin.cpu().tolist()[2] == 0.0
    g = r.grad.cpu()
    assert g[3] == 0 and g[1] == 1.0 and g[2] == -1.0
    p = 1 / (1 + math.exp(1e-3))
    assert g[4].item() == pytest.approx(-p, rel=1e-6) and g[0].item() == pytest.approx(p, rel=1e-6)
    # sequences that cannot be (log-probability -inf)
    lp = torch.tensor([0.0, -math.inf, -1.0, -2.0])
    for seg in (None, np.asarray([0, 1, 2, 3, 4])):
        plan = losses.PreferencePlan(np.asarray([[0, 1], [2, 3]]), 4, segments=seg, device="cuda")
        r = losses.preference_loss(lp.cuda(), plan)
        assert r.margin.tolist() == [math.inf, 1.0] and r.loss[0] == 0.0
        assert r.grad.tolist()[:2] == [0.0, 0.0] and r.grad[2] < 0
        plan = losses.PreferencePlan(np.asarray([[1, 0], [2, 3]]), 4, segments=seg, device="cuda")
        r = losses.preference_loss(lp.cuda(), plan)
        assert r.loss[0] == math.inf and r.grad.tolist()[:2] == [1.0, -1.0]
        assert r.margin[1] == 1.0
    for P, n, seg in ((0, 4, None), (0, 4, [0, 2, 4]), (0, 0, [0])):
        plan = losses.PreferencePlan(np.zeros((P, 2), np.int32), n, device="cuda",
                                     segments=np.asarray(seg) if seg is not None else None)
        r = losses.preference_loss(torch.ones(n, device="cuda"), plan)
        assert r.loss.shape == (0,) and not r.grad.any() and r.grad.shape == (n,)


# --------------------------------------------------------------------- together
@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
def test_policy_and_balance_in_one_gradient(gpu, order):
    from warpgbm_amd import losses

    d = policy_inputs(777, 12, "f32", order, 5)
    loss, lp, kl, grad, live = policy_want(d, "sampled", (0.2, 0.2), 0.1)
    mask = live.clone()
    even = balance_want(d["s"], mask, 2, 50.0)
    r = run_policy(d, "sampled", (0.2, 0.2), 0.1)
    e = losses.balance_loss(to_gpu(d["s"]), top_k=2, mask=mask.cuda(), coef=50.0, grad=r.grad)
    scale = policy_scales(d, "sampled", 0.1, kl, live) + 50.0 * 12 / int(live.sum())
    check(e.grad, grad + even[3], STEPS * U * (scale[:, None] + 1e-6), "gradient")
    assert torch.equal(e.counts.cpu(), even[1])


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
def test_sequence_preference_of_a_class_policy(gpu, order):
    """Log-probabilities, their paired log ratios, the gradient of the scores."""
    from warpgbm_amd import losses

    d = pref_case("sequences", 77)
    n, K = d["n"], 9
    s = make_scores(n, K, "f32", order, 78)
    a = torch.randint(0, K, (n,), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    x = s.to(F64).requires_grad_(True)
    lp = log_softmax64(x).gather(1, a.long()[:, None])[:, 0]
    ref = lp.detach().float() + 0.3
    ref[::3] -= 0.8
    loss, margin = preference64(lp, d["pairs"], d["S"], d["seg"], ref, None, 0.5, 0.0)
    loss.sum().backward()
    sd = to_gpu(s)
    f = losses.class_log_probs(sd, a.cuda())
    plan = losses.PreferencePlan(d["pairs"].cuda(), n, segments=d["seg"].cuda())
    r = losses.preference_loss(f.log_prob, plan, ref_log_prob=ref.cuda(), beta=0.5)
    got = losses.class_log_probs_grad(sd, a.cuda(), f.norm, r.grad)
    # a margin's error: its rows' log-probabilities; every pair of a sequence
    # moves its rows' gradient by at most that times beta^2 / 4
    rows = torch.zeros(d["S"], dtype=F64)
    rows.copy_(d["seg"].diff().to(F64))
    lp_err = U * (STEPS + 100)
    pair_err = (rows[d["pairs"][:, 0].long()] + rows[d["pairs"][:, 1].long()]) * lp_err
    check(r.margin, margin.detach(), pair_err + U * margin.detach().abs(), "margin")
    per = torch.zeros(d["S"], dtype=F64)
    for side in (0, 1):
        per.index_add_(0, d["pairs"][:, side].long(), 0.25 * 0.25 * pair_err + 32 * U)
    tol = torch.zeros(n, dtype=F64)
    tol[:int(d["seg"][-1])] = per.repeat_interleave(d["seg"].diff())
    check(got, x.grad, (tol + STEPS * U * r.grad.abs().cpu().to(F64))[:, None], "gradient")


@pytest.mark.gpu
def test_gradient_against_differences(gpu):
    """The policy's, the balance's and the preferences' gradients against
    central differences of the kernels' own losses (float32 losses summed in
    float64; the step makes the differences' rounding 2^-24 * loss / h)."""
    from warpgbm_amd import losses

    n, K, h = 64, 6, 2.0 ** -6
    d = policy_inputs(n, K, "f32", "row", 9)
    d["old"] += 0.01
    live = live_rows(d["s"], d["a"], d["w"])
    way = torch.randn((n, K), generator=torch.Generator().manual_seed(3))
    # a power of two times the direction keeps s + h * way within a rounding

    def total(s):
        r = run_policy(dict(d, s=s), "exact", (10.0 / 11, 10.0), 0.3)
        e = losses.balance_loss(s.cuda(), mask=live.cuda(), coef=5.0, top_k=6)
        return r.loss.double().cpu()[live].sum() + e.loss.double().cpu()

    s = torch.where(live[:, None], d["s"], torch.zeros(()))
    d["s"] = s
    d["w"][~live] = 0.0
    slope = (total(s + h * way) - total(s - h * way)) / (2 * h)
    r = run_policy(d, "exact", (10.0 / 11, 10.0), 0.3)
    e = losses.balance_loss(s.cuda(), mask=live.cuda(), coef=5.0, top_k=6, grad=r.grad)
    along = (e.grad.cpu().double() * way.double()).sum()
    # third derivatives of softmax-like losses are below 2 of their size
    size = (r.loss.abs().sum().cpu().double() + 5.0) * way.abs().max().double() ** 3
    assert abs(slope - along) < 2 * size * h * h + n * 1e-6 / h


# --------------------------------------------------------------------- streams, graphs
@pytest.mark.gpu
def test_other_stream_and_same_bits(gpu):
    from warpgbm_amd import losses

    d = policy_inputs(3000, 50, "bf16", "row", 55)
    one = run_policy(d, "exact", (0.2, 0.2), 0.1)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        two = run_policy(d, "exact", (0.2, 0.2), 0.1)
        e2 = losses.balance_loss(to_gpu(d["ref_s"]), top_k=2)
    st.synchronize()
    e1 = losses.balance_loss(to_gpu(d["ref_s"]), top_k=2)
    nan = torch.isnan(one.grad)
    assert torch.equal(nan, torch.isnan(two.grad))
    assert torch.equal(one.grad[~nan], two.grad[~nan]) and torch.equal(one.loss, two.loss)
    assert torch.equal(e1.grad, e2.grad) and torch.equal(e1.loss, e2.loss)


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
def test_captured_graph_replays(gpu, order):
    """Two captured graphs, replayed in turn with eager calls between, on
    inputs that change."""
    from warpgbm_amd import losses

    d = pref_case("sequences", 91)
    n, K = d["n"], 20
    plan = losses.PreferencePlan(d["pairs"].cuda(), n, segments=d["seg"].cuda())
    s = to_gpu(make_scores(n, K, "f32", order, 1))
    a = torch.randint(0, K, (n,), dtype=torch.int32).cuda()
    old, adv = torch.full((n,), -3.0).cuda(), torch.randn(n).cuda()

    def sequence():
        f = losses.class_log_probs(s, a)
        r = losses.preference_loss(f.log_prob, plan, beta=0.3)
        return [f.log_prob, r.loss, r.grad, losses.class_log_probs_grad(s, a, f.norm, r.grad)]

    def step():
        r = losses.policy_loss(s, a, old, adv)
        e = losses.balance_loss(s, top_k=2, coef=100.0, grad=r.grad)
        return [r.loss, e.loss, e.counts, e.prob, e.grad]

    graphs = []
    for fn in (sequence, step):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fn()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = fn()
        graphs.append((g, out, fn))
    for turn in range(4):
        s.copy_(to_gpu(make_scores(n, K, "f32", order, 50 + turn)))
        for g, out, fn in graphs:
            g.replay()
            torch.cuda.synchronize()
            for x, y in zip(out, fn()):
                assert torch.equal(x, y)


@pytest.mark.gpu
def test_offsets_past_32_bits(gpu):
    """A matrix of more than 2^32 bytes and 2^31 elements, both orders: the
    last rows are the small matrix's."""
    from warpgbm_amd import losses

    n, K = 2_200_000, 1000
    tail = 5
    for order in ("row", "class"):
        print_case("large", order, n, K)
        small = make_scores(tail, K, "bf16", order, 4)
        a = torch.arange(tail, dtype=torch.int32)
        adv = torch.ones(tail)
        want = losses.policy_loss(small.cuda() if order == "row" else small.t().contiguous().cuda().t(),
                                  a.cuda(), -7 * adv.cuda(), adv.cuda())
        big = torch.zeros((n, K) if order == "row" else (K, n), dtype=torch.bfloat16, device="cuda")
        big = big if order == "row" else big.t()
        big[-tail:] = small.cuda()
        labels = torch.zeros(n, dtype=torch.int32, device="cuda")
        labels[-tail:] = a.cuda()
        w = torch.zeros(n, device="cuda")
        w[-tail:] = 1.0
        one = torch.ones(n, device="cuda")
        r = losses.policy_loss(big, labels, -7 * one, one, weight=w)
        # (the classes may be added in another order: other sizes)
        assert torch.allclose(r.loss[-tail:], want.loss, rtol=1e-5)
        g, wg = r.grad[-tail:].float(), want.grad.float()
        assert torch.allclose(g, wg, rtol=2.0 ** -7, atol=1e-6)
        assert not r.grad[:4].any()
        f = losses.class_log_probs(big, labels)
        assert torch.allclose(f.log_prob[-tail:], want.log_prob, rtol=1e-5)
        del big, r, f
        torch.cuda.empty_cache()


# --------------------------------------------------------------------- CPU: forms and refusals
def test_float64_forms_against_differences():
    """The forms that the kernels are held to, against central differences."""
    g = torch.Generator().manual_seed(2)
    s = torch.randn((4, 5), generator=g, dtype=F64)
    r = s + 0.3 * torch.randn((4, 5), generator=g, dtype=F64)
    a = torch.tensor([0, 3, 2, 4])
    old = log_softmax64(s).gather(1, a[:, None])[:, 0] + torch.tensor([0.05, -0.6, 0.6, 0.01])
    adv, w = torch.tensor([1.0, 2.0, -1.0, -0.5]), torch.tensor([1.0, 0.5, 2.0, 1.0])
    for ref_lp, ref_s in ((None, None), (old + 0.2, None), (None, r)):
        x = s.clone().requires_grad_(True)
        policy64(x, a, old, adv, w, ref_lp, ref_s, (0.2, 0.2), 0.5)[0].sum().backward()
        for i in range(4):
            for k in range(5):
                d = torch.zeros_like(s)
                d[i, k] = 1e-6
                f = [policy64(s + e, a, old, adv, w, ref_lp, ref_s, (0.2, 0.2), 0.5)[0].sum()
                     for e in (d, -d)]
                assert abs((f[0] - f[1]) / 2e-6 - x.grad[i, k]) < 1e-7


def test_refusals_without_a_gpu():
    from warpgbm_amd import losses

    s, a = torch.zeros((3, 4)), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        losses.class_log_probs(s, a)
    with pytest.raises(RuntimeError, match="torch.Tensor"):
        losses.policy_loss(s.numpy(), a, a, a)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        losses.balance_loss(s.double())
    with pytest.raises(RuntimeError, match="shape"):
        losses.PreferencePlan(np.zeros((3, 3), np.int64), 4, device="cpu")
    with pytest.raises(RuntimeError, match="int32 or int64"):
        losses.PreferencePlan(np.zeros((3, 2), np.float32), 4, device="cpu")
    for pairs, n, seg, text in (
            ([[0, 4]], 4, None, "sequence numbers"), ([[-1, 0]], 4, None, "sequence numbers"),
            ([[0, 2]], 4, [0, 2, 4], "sequence numbers"), ([[0, 1]], 4, [0, 3, 2], "ascend"),
            ([[0, 1]], 4, [1, 3, 4], "ascend"), ([[0, 1]], 4, [0, 3, 5], "ascend"),
            ([[0, 1]], 4, [[0, 3]], "offsets"), ([[0, 0]], -1, None, "negative")):
        with pytest.raises(RuntimeError, match=text):
            losses.PreferencePlan(np.asarray(pairs), n, device="cpu",
                                  segments=np.asarray(seg) if seg is not None else None)
    with pytest.raises(RuntimeError, match="PreferencePlan"):
        losses.preference_loss(s[0], None)


def test_strides_of_single_rows_and_classes():
    """The strides of [n, K] scores: that of a dimension of one element does not
    count, a repeated row or class is refused (the library would read past its
    end)."""
    from warpgbm_amd.losses import _strides

    assert _strides(0, 4, 0, 0, "s") == (4, 1)
    assert _strides(1, 1, 0, 7, "s") == (1, 1)
    assert _strides(5, 1, 1, 9, "s") == (1, 1) and _strides(5, 1, 8, 0, "s") == (8, 1)
    assert _strides(1, 4, 0, 1, "s") == (4, 1) and _strides(1, 4, 0, 3, "s") == (1, 3)
    assert _strides(5, 4, 6, 1, "s") == (6, 1) and _strides(5, 4, 1, 5, "s") == (1, 5)
    for n, K, rs, ks in ((5, 1, 0, 1), (5, 1, 0, 0), (1, 4, 4, 0), (5, 4, 3, 1), (5, 4, 1, 4),
                         (5, 4, 0, 1), (5, 4, 1, 0), (5, 4, 8, 2)):
        with pytest.raises(RuntimeError, match="next to each other"):
            _strides(n, K, rs, ks, "s")


def test_plan_without_a_gpu_is_not_evaluated():
    from warpgbm_amd import losses

    plan = losses.PreferencePlan(np.asarray([[0, 1]]), 2, device="cpu")
    with pytest.raises(RuntimeError, match="on a GPU"):
        losses.preference_loss(torch.zeros(2), plan)


def test_plan_layout():
    """The tables of a plan (on the CPU): incidences grouped by sequence in pair
    order, tasks that cover every row once, in order, sequences in many pairs in
    pieces."""
    from warpgbm_amd import losses

    p = losses.PreferencePlan(np.asarray([[2, 0], [0, 1], [0, 0]]), 3, device="cpu")
    assert p.incidence.tolist() == [1, 2, 4, 5, 3, 0]
    assert p.incidence_start.tolist() == [0, 4, 5, 6]
    assert p.task is None and p.piece is None and not p.disjoint
    seg = np.asarray([0, 5, 5, 4106, 14000, 14002])
    p = losses.PreferencePlan(np.asarray([[0, 1], [0, 2], [3, 4]]), 18100, segments=seg,
                              device="cpu")
    rows = p.task.tolist()
    assert [r[0] for r in rows] == [0, 1, 2, 2, 3, 3, 3, 4, -1, -1]
    assert p.task_start.tolist() == [0, 1, 2, 4, 7, 8]
    assert rows[1] == [1, 5, 5] and rows[3] == [2, 4101, 4106]
    assert rows[0][1] == 0 and rows[-1][2] == 18100
    assert all(a[2] == b[1] and a[2] - a[1] <= 4096 for a, b in zip(rows, rows[1:]))
    p = losses.PreferencePlan(np.asarray([[3, 1]]), 9, segments=np.asarray([0, 2, 3, 3, 5, 8]),
                              device="cpu")
    assert p.disjoint and p.idle.tolist() == [[0, 2], [5, 8], [8, 9]]
    # a sequence of 17,000 incidences, one of 300, others of few
    pairs = np.asarray([[7, k % 5] if k < 17_000 else [8, 7 - k % 3] for k in range(17_300)])
    p = losses.PreferencePlan(pairs, 10, device="cpu")
    inc, start = p.incidence.numpy(), p.incidence_start.tolist()
    assert sorted(inc.tolist()) == list(range(2 * len(pairs)))
    ends = pairs.reshape(-1)[inc]
    for s in range(10):
        assert (ends[start[s]:start[s + 1]] == s).all()
    share = p.share.tolist()
    assert share[0] == 0 and share[-1] == 10 and share == sorted(share)
    assert p.is_long.tolist() == [int(start[s] == start[s + 1] and s != 9) for s in range(10)]
    covered = start[-1]
    whole = {s: f for s, f, e in p.multi.tolist() for s in [s]}
    assert 7 in whole
    owner = {}
    for s, f, e in p.multi.tolist():
        owner.update({q: s for q in range(f, e)})
    for q, (s, f, e) in enumerate(p.piece.tolist()):
        assert f == covered and 0 < e - f <= 8192
        covered = e
        assert (ends[f:e] == (s if s >= 0 else owner[q])).all()
    assert covered == 2 * len(pairs)


def test_c_entries_refuse_before_any_launch():
    import ctypes as C

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

    def lp(s, ws=1 << 30):
        return lib.wgbm_class_log_probs(C.byref(s), one, one, one, one, ws, None)

    refused(lp(scores(dtype=3)), "type code")
    refused(lp(scores(n_rows=-1)), "n_rows")
    refused(lp(scores(n_classes=0)), "n_classes")
    refused(lp(scores(row_stride=7)), "strides")
    refused(lp(scores(row_stride=1, class_stride=3)), "strides")
    refused(lp(scores(row_stride=16, class_stride=2)), "strides")
    refused(lp(scores(data=18)), "aligned")
    refused(lp(scores(data=None)), "null data")
    # (rows of 100,000 classes go through the workspace)
    refused(lp(scores(n_classes=100_000, row_stride=100_000), ws=8), "workspace too small")
    empty = scores(n_rows=0)
    for fn in (lib.wgbm_class_log_probs_workspace, lib.wgbm_policy_loss_workspace,
               lib.wgbm_balance_loss_workspace):
        assert fn(C.byref(empty)) >= 0
    assert lib.wgbm_class_log_probs_workspace(C.byref(scores(dtype=3))) == -1
    assert lp(scores(n_rows=0)) == 0

    def policy(a=None, grad=None, **kw):
        f = dict(actions=one, old_log_prob=one, advantage=one, weight=None, ref_log_prob=None,
                 ref_scores=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0)
        f.update(kw)
        args = _lib.PolicyArgs(*f.values())
        return lib.wgbm_policy_loss(C.byref(a or scores()), C.byref(args), one, one, None,
                                    C.byref(grad) if grad else None, 0, one, 1 << 30, None)

    refused(policy(clip_low=1.5), "clip_low")
    refused(policy(clip_low=float("nan")), "clip_low")
    refused(policy(clip_high=-0.1), "clip_high")
    refused(policy(clip_high=float("inf")), "clip_high")
    refused(policy(kl_coef=-1.0), "kl_coef")
    refused(policy(actions=None), "null pointer")
    refused(policy(grad=scores(dtype=1)), "grad must have the shape and type")
    refused(policy(grad=scores(row_stride=1, class_stride=8)), "order")
    refused(policy(ref_scores=C.pointer(scores(n_classes=7))), "ref_scores")
    refused(policy(ref_scores=C.pointer(scores()), ref_log_prob=one), "exclude")

    def balance(s, k, coef=1.0):
        return lib.wgbm_balance_loss(C.byref(s), None, k, coef, one, one, one, None, 0, one,
                                     1 << 30, None)

    refused(balance(scores(), 0), "top_k")
    refused(balance(scores(), 9), "top_k")
    refused(balance(scores(n_classes=4), 5), "top_k")
    refused(balance(scores(n_classes=4097, row_stride=4097), 1), "4096")
    refused(balance(scores(), 1, float("inf")), "coef")

    def pref(**kw):
        f = dict(log_prob=one, ref_log_prob=None, n_rows=4, sequence_start=None, n_sequences=4,
                 pairs=one, n_pairs=2, incidence=one, incidence_start=one, share=one, n_shares=1,
                 is_long=None, task=None, n_tasks=0,
                 task_start=None, piece=None, n_pieces=0, multi=None, n_multi=0, idle=None,
                 n_idle=0, disjoint=0, weight=None, beta=1.0, label_smoothing=0.0)
        f.update(kw)
        args = _lib.PreferenceArgs(*f.values())
        return lib.wgbm_preference_loss(C.byref(args), one, one, one, one, 1 << 30, None)

    refused(pref(beta=0.0), "beta")
    refused(pref(beta=float("nan")), "beta")
    refused(pref(label_smoothing=0.6), "label_smoothing")
    refused(pref(n_sequences=3), "every row is a sequence")
    refused(pref(n_pairs=1 << 30), "n_pairs")
    refused(pref(lanes=5), "lanes")
    refused(pref(lanes=128), "lanes")
    refused(pref(incidence=None), "gradient needs")
    refused(pref(sequence_start=one), "tasks")
    refused(pref(share=None), "gradient needs")
    refused(pref(n_pieces=1), "gradient needs")
    refused(pref(n_pieces=1, is_long=one), "null table")
    refused(pref(n_multi=-1), "table sizes")
    refused(pref(disjoint=1), "every row is a sequence")


@pytest.mark.gpu
def test_refusals_on_the_gpu(gpu):
    from warpgbm_amd import losses

    s = torch.zeros((6, 4), device="cuda")
    a, f = torch.zeros(6, dtype=torch.int32, device="cuda"), torch.zeros(6, device="cuda")

    def no(text, fn, *args, **kw):
        with pytest.raises(RuntimeError, match=text):
            fn(*args, **kw)

    no("labels must have dtype", losses.class_log_probs, s, a.long())
    no("labels must have shape", losses.class_log_probs, s, a[:5])
    no("labels must be contiguous", losses.class_log_probs, s,
       torch.zeros(12, dtype=torch.int32, device="cuda")[::2])
    no("labels must be on", losses.class_log_probs, s, a.cpu())
    no("next to each other", losses.class_log_probs, s.repeat(2, 2)[::2, ::2], a)
    no("next to each other", losses.class_log_probs, s[:, :1].expand(6, 4), a)
    no("next to each other", losses.class_log_probs, s[:1].expand(6, 4), a)
    no("next to each other", losses.class_log_probs, s[:1, :1].expand(6, 1), a)
    no("at least one class", losses.class_log_probs, s[:, :0], a)
    no("2-D", losses.class_log_probs, s[0], a)
    no("norm", losses.class_log_probs_grad, s, a, f, f)
    no("exclude", losses.policy_loss, s, a, f, f, ref_log_prob=f, ref_scores=s)
    no("clip", losses.policy_loss, s, a, f, f, clip=0.2)
    no("clip_low", losses.policy_loss, s, a, f, f, clip=(2.0, 0.2))
    no("ref_scores", losses.policy_loss, s, a, f, f, ref_scores=s.bfloat16())
    no("ref_scores", losses.policy_loss, s, a, f, f, ref_scores=s.t().contiguous().t())
    no("scores' memory", losses.policy_loss, s, a, f, f, grad=s)
    no("next to each other as scores", losses.policy_loss, s, a, f, f,
       grad=torch.zeros((4, 6), device="cuda").t())
    no("shape, dtype and device", losses.policy_loss, s, a, f, f, grad=s.half())
    no("with_grad", losses.policy_loss, s, a, f, f, grad=s.clone(), with_grad=False)
    no("top_k", losses.balance_loss, s, top_k=5)
    no("mask must have dtype", losses.balance_loss, s, mask=f)
    no("at most 4096", losses.balance_loss, torch.zeros((2, 4097), device="cuda"))
    plan = losses.PreferencePlan(np.asarray([[0, 1]]), 6, device="cuda")
    no("log_prob must have shape", losses.preference_loss, f[:5], plan)
    no("weight must have shape", losses.preference_loss, f, plan, weight=f)
    no("beta", losses.preference_loss, f, plan, beta=0.0)
    # nothing to do
    e = losses.policy_loss(s[:0], a[:0], f[:0], f[:0], ref_log_prob=f[:0])
    assert e.grad.shape == (0, 4) and e.loss.shape == (0,) and e.kl.shape == (0,)
    b = losses.balance_loss(s[:0])
    assert b.loss.item() == 0 and not b.counts.any() and not b.prob.any()
    assert losses.class_log_probs(s[:0], a[:0]).norm.shape == (0, 2)


@pytest.mark.gpu
def test_more_threads_than_a_grid_counts(gpu):
    """Rows of 64 threads each whose launch would have some 2^32 threads: the
    last rows as in a call of their own, the first ones too."""
    from warpgbm_amd import losses

    n, K, m = 16_900_000, 257, 3000
    s = torch.zeros((n, K), dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(3)
    parts = [slice(0, m), slice(n - 500_000, n - 500_000 + m), slice(n - m, n)]
    for p in parts:
        s[p] = torch.randn((m, K), generator=gen, device="cuda").to(torch.bfloat16)
    a = torch.randint(0, K, (n,), generator=gen, device="cuda", dtype=torch.int32)
    old = torch.full((n,), -5.5, device="cuda")
    adv = torch.randn(n, generator=gen, device="cuda")
    f = losses.class_log_probs(s, a)
    g = losses.class_log_probs_grad(s, a, f.norm, adv)
    want = []
    for p in parts:
        x = losses.class_log_probs(s[p], a[p])
        assert torch.equal(f.log_prob[p], x.log_prob) and torch.equal(f.norm[p], x.norm)
        assert torch.equal(g[p], losses.class_log_probs_grad(s[p], a[p], x.norm, adv[p]))
        want.append(losses.policy_loss(s[p], a[p], old[p], adv[p], weight=adv[p].abs(),
                                       ref_log_prob=old[p], kl_coef=0.1))
    del f, g
    r = losses.policy_loss(s, a, old, adv, weight=adv.abs(), ref_log_prob=old, kl_coef=0.1)
    for p, x in zip(parts, want):
        assert torch.equal(r.loss[p], x.loss) and torch.equal(r.log_prob[p], x.log_prob)
        assert torch.equal(r.kl[p], x.kl) and torch.equal(r.grad[p], x.grad)


@pytest.mark.gpu
@pytest.mark.parametrize("twice", [False, True])
def test_more_sequences_than_a_grid_counts(gpu, twice):
    """A wave a sequence, more than 2^26 of them; with a pair's sequence in
    another pair, the steps apart."""
    from warpgbm_amd import losses

    n = (1 << 26) + 5000
    pairs = [[0, n - 2], [n - 1, 5]] + ([[0, n - 1]] if twice else [])
    plan = losses.PreferencePlan(np.asarray(pairs), n,
                                 segments=torch.arange(n + 1, device="cuda"))
    assert plan.disjoint != twice
    lp = torch.zeros(n, device="cuda")
    lp[n - 1], lp[0], lp[n - 2] = 1.5, -0.5, 2.0
    r = losses.preference_loss(lp, plan)
    margin = [-2.5, 1.5] + ([-2.0] if twice else [])
    assert r.margin.tolist() == margin
    # -sigmoid(-margin), float32's expf, sum, reciprocal and product: 6 roundings
    slope = [-1 / (1 + np.exp(v)) for v in margin]
    want = {0: slope[0], n - 2: -slope[0], n - 1: slope[1], 5: -slope[1]}
    if twice:
        want[0] += slope[2]
        want[n - 1] -= slope[2]
    at = sorted(want)
    got = r.grad[torch.tensor(at, device="cuda")].cpu().double().numpy()
    assert np.abs(got - [want[i] for i in at]).max() <= 8 * 2.0 ** -24
    r.grad[torch.tensor(at, device="cuda")] = 0
    assert not r.grad.any()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["pairs", "mixed"])
@pytest.mark.parametrize("lanes", [0, 4, 8, 16, 32, 64])
def test_threads_of_a_sequence(gpu, kind, lanes):
    """Sequences of 0 to 700 rows and rows behind the last one, by as many threads
    as a plan may choose; one pair a sequence, or several."""
    from warpgbm_amd import losses

    g = torch.Generator().manual_seed(31)
    S = 120
    length = torch.randint(0, 12, (S,), generator=g)
    length[7], length[50], length[119] = 700, 257, 64
    seg = torch.cat([torch.zeros(1, dtype=torch.int64), length.cumsum(0)])
    n = int(seg[-1]) + 333
    if kind == "pairs":
        pairs = torch.randperm(S, generator=g)[:80].reshape(-1, 2)
    else:
        pairs = torch.randint(0, S, (200, 2), generator=g)
    lp, ref = -torch.rand(n, generator=g), -torch.rand(n, generator=g)
    plan = losses.PreferencePlan(pairs, n, segments=seg, device="cuda")
    assert plan.disjoint == (kind == "pairs")
    plan.lanes = lanes
    r = losses.preference_loss(lp.cuda(), plan, ref_log_prob=ref.cuda(), beta=0.5,
                               label_smoothing=0.1)
    x = lp.to(F64).requires_grad_()
    loss, margin = preference64(x, pairs, S, seg, ref, None, 0.5, 0.1)
    loss.sum().backward()
    # sums in float64; the margin, its product with beta, and the few operations
    # of a loss or slope round to float32: 2^-24 of each, eight at most
    # relative to 1 + |margin|; a gradient adds its pairs' slopes (at most 0.5)
    scale = 1 + margin.detach().abs()
    assert ((r.margin.cpu() - margin.detach()).abs() <= 2 ** -24 * scale).all()
    assert ((r.loss.cpu() - loss.detach()).abs() <= 8 * 2 ** -24 * scale).all()
    many = torch.bincount(pairs.reshape(-1), minlength=S).max()
    tol = float(many) * 0.5 * 8 * 2 ** -24 * float(scale.max())
    assert (r.grad.cpu() - x.grad).abs().max() <= tol
    assert not r.grad[int(seg[-1]):].any()


# classes at which rows take another number of threads, chunks or slices
EDGES = [(70, K) for K in (16, 17, 32, 33, 36, 40, 41, 52, 53, 64, 65, 80, 81, 104, 105, 128, 129,
                           156, 157, 192, 193, 208, 209, 256, 257)] + \
        [(11, K) for K in (511, 512, 513, 1024, 1025, 2047, 2048, 2049, 4095, 4096, 4097)]
# rows enough for the balance loss to take two chunks a thread
BALANCE_ROWS = [(44_000, 49), (42_003, 99), (21_001, 201), (11_000, 403), (1_500, 2500)]


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_edges_of_frames(gpu, monkeypatch, dtype, order):
    here = sys.modules[__name__]
    monkeypatch.setattr(here, "SHAPES", EDGES)
    test_log_probs_and_gradient(gpu, dtype, order)
    for kl in ("none", "sampled", "exact"):
        test_policy_loss(gpu, dtype, order, kl)
    monkeypatch.setattr(here, "BALANCE_SHAPES", [e for e in EDGES if e[1] <= 4096])
    test_balance_loss(gpu, dtype, order)


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "row+"])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_balance_loss_of_many_rows(gpu, monkeypatch, dtype, order):
    monkeypatch.setattr(sys.modules[__name__], "BALANCE_SHAPES", BALANCE_ROWS)
    test_balance_loss(gpu, dtype, order)

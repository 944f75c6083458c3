"""Losses with lists of classes at lengths, scores and arguments next to their limits:
tiles of very long rows, NaN among scores, log norms far from 0,
logits of -inf, lowest masks at low temperatures, rows
and teachers far from 0, shares below float32's range, launches in parts."""
import ctypes as C
import math

import pytest
import torch

from conftest import print_case
from test_lists import alternatives_grad64, check_distill, distill64, round_tol
from test_losses import DTYPES, STEPS, U, check, make_scores, to_gpu

INF = math.inf
MOST = {False: {0: 16_384, 1: 32_768}, True: {0: 4096, 1: 8192}}  # classes of a tile


def tiles_of(K, code, grad):
    from warpgbm_amd import _lib

    span = C.c_int32()
    v = _lib.Scores(16, code, 1, K, K, 1)
    return _lib.load().wgbm_lists_tiles(C.byref(v), int(grad), C.byref(span)), span.value


# --------------------------------------------------------------------- tiles of long rows
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("code", [0, 1, 2])
def test_tiles_hold_a_chunk_and_fit_their_frame(code, grad):
    """Every class in one tile, none longer than the frame, none shorter than 8 classes:
    the lengths next to every multiple of a tile, and some between."""
    most = MOST[grad][min(code, 1)]
    whole = most if grad else 4 * most
    g = torch.Generator().manual_seed(code)
    lengths = torch.randint(13, (1 << 24) + 1, (20_000,), generator=g).tolist()
    for step in (most, most - 8, most - 16):
        for at in range(0, 1 << 24, step):
            lengths += range(max(13, at - 1), at + 9)
    for K in lengths:
        if K > 1 << 24:
            continue
        tiles, span = tiles_of(K, code, grad)
        if K <= whole:
            assert (tiles, span) == (1, K)
            continue
        last = K - (tiles - 1) * span
        assert span % 8 == 0 and 8 <= last <= span <= most, (K, tiles, span)


def test_tiles_of_other_scores():
    from warpgbm_amd import _lib

    entry = _lib.load().wgbm_lists_tiles
    assert entry(C.byref(_lib.Scores(16, 0, 4, 90_000, 1, 4)), 1, None) == 1  # class-major
    assert entry(C.byref(_lib.Scores(16, 0, 4, 90_000, 90_000, 1)), 1, None) == 22
    assert entry(C.byref(_lib.Scores(16, 5, 4, 90_000, 90_000, 1)), 1, None) == -1
    assert entry(None, 0, None) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,order,n,K", [
    ("f32", "row", 2, 2_093_057), ("f32", "row+", 2, 2_093_058), ("f32", "class", 2, 2_093_059),
    ("bf16", "row", 1, 8_380_417), ("f16", "row+", 1, 8_380_423), ("bf16", "class", 2, 2_093_057)])
def test_gradient_of_rows_that_leave_a_few_classes_over(gpu, dtype, order, n, K):
    """Lengths a few classes over a multiple of the tile's, with the label and an entry
    among these."""
    from warpgbm_amd import losses

    s = make_scores(n, K, dtype, order, 7)
    g = torch.Generator().manual_seed(K)
    a = torch.full((n,), K - 1, dtype=torch.int32)
    cls = torch.randint(0, K, (n, 20), generator=g, dtype=torch.int32)
    cls[:, 3], cls[:, 4], cls[:, 5] = K - 2, K - 9, 0
    gl, ge = torch.randn(n, generator=g), torch.randn(n, generator=g)
    gt = torch.randn((n, 20), generator=g)
    old = make_scores(n, K, dtype, order, 8)
    sd = to_gpu(s)
    f = losses.class_alternatives(sd, 0)
    for what in ("label", "list", "added"):
        print_case("over", dtype, order, n, K, what)
        lists = what != "label"
        want, tol = alternatives_grad64(s, a, gl, cls if lists else None, gt, ge, 1.0)
        kw = dict(classes=cls.cuda(), grad_log_prob=gt.cuda()) if lists else {}
        if what == "added":
            kw["grad"] = to_gpu(old)
            want = want + old.double()
        got = losses.class_alternatives_grad(sd, f.norm, labels=a.cuda(),
                                             grad_label_log_prob=gl.cuda(),
                                             grad_entropy=ge.cuda(), **kw)
        assert got.dtype == DTYPES[dtype]
        check(got, want, round_tol(tol, want, dtype), what)


# --------------------------------------------------------------------- NaN among scores
def rows_with_nan(K, dtype, order, seed):
    """Rows with one NaN, one of either sign first and last, a run of them, every other
    class, all but one, all; with classes that the row may not take; among equal scores."""
    g = torch.Generator().manual_seed(seed)
    s = torch.randn((13, K), generator=g)
    nan = float("nan")
    s[0, K // 2] = nan
    s[1, 0], s[1, K - 1] = nan, -nan
    s[2, K // 3:K // 3 + 40] = nan
    s[3, ::2] = nan
    one = s[4, K // 2].clone()
    s[4] = nan
    s[4, K // 2] = one
    s[5] = nan
    s[6, 1::2] = -INF
    s[6, K // 2 // 2 * 2] = nan
    s[7] = 0.5
    s[7, K // 4] = nan
    s[8] = -s[8].abs() - 1e3
    s[8, K // 5] = nan
    s = s.to(DTYPES[dtype])
    # (NaN of a type's own, of either sign: a conversion may choose another sign)
    bits = s.view(torch.int32 if dtype == "f32" else torch.int16)
    quiet = {"f32": 0x7fc00000, "bf16": 0x7fc0, "f16": 0x7e00}[dtype]
    sign = torch.iinfo(bits.dtype).min
    bits[10, K // 2] = bits[11, K - 1] = quiet
    bits[11, 0] = quiet + sign
    bits[12, K // 3:K // 3 + 40] = quiet
    return s if order == "row" else s.t().contiguous().t()


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_nan_takes_no_place_among_the_alternatives(gpu, dtype, order):
    """The other classes in their order; -1 only where a row has fewer of them."""
    from warpgbm_amd import losses

    for K in (3, 10, 14, 40, 130, 200, 257, 400, 512, 600, 1000, 1500, 3000, 5000, 12_000, 20_000,
              70_001, 140_003):
        if order == "class" and K > 3000:
            continue
        s = rows_with_nan(K, dtype, order, K)
        there = ~torch.isnan(s) & (s > -INF)
        at = torch.sort(torch.where(there, s.double(), -INF), dim=1, descending=True, stable=True)
        for k in sorted({1, min(5, K), min(64, K)}):
            print_case("nan", dtype, order, K, k)
            want = torch.where(at.values[:, :k] > -INF, at.indices[:, :k], -1).to(torch.int32)
            r = losses.class_alternatives(to_gpu(s), k)
            assert torch.equal(r.classes.cpu(), want), (K, k)
            lp = r.log_prob.cpu()
            assert (lp[want < 0] == -INF).all()
            has = torch.isnan(s).any(1)
            assert torch.isnan(lp[has][want[has] >= 0]).all()
            assert not torch.isnan(lp[~has]).any()


# --------------------------------------------------------------------- log norms as numbers
@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
def test_a_log_norm_for_all_rows_keeps_its_digits(gpu, order):
    """A number is taken in float64, as temperatures are: rounded to float32, one of some
    thousand would move every share by up to 2.4e-4 of it."""
    from warpgbm_amd import losses

    for K, k, tau, norm in ((6, 3, 1.0, 4096.3), (40, 8, 0.7, -3000.1), (300, 12, 2.0, 777.77),
                            (900, 20, 1.0, 2049.1), (70_001, 64, 1.0, 5000.1)):
        print_case("log norm", order, K, k, tau, norm)
        n = 12
        g = torch.Generator().manual_seed(K)
        s = torch.randn((n, K), generator=g)
        s = s if order == "row" else s.t().contiguous().t()
        cls = torch.argsort(torch.rand((n, K), generator=g), 1)[:, :k].to(torch.int32).contiguous()
        t = torch.log_softmax(torch.randn((n, K), generator=g, dtype=torch.float64), 1)
        logits = (tau * (t.gather(1, cls.long()) + norm)).float()
        w = torch.ones(n)
        got = losses.distill_loss(to_gpu(s), cls.cuda(), logits.cuda(), log_norm=norm,
                                  temperature=tau)
        check_distill(got, distill64(s, cls, logits, norm, w, tau), w, tau, "f32")


# --------------------------------------------------------------------- logits of -inf
@pytest.mark.gpu
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("order", ["row", "class"])
def test_listed_classes_that_the_teacher_rules_out(gpu, order, rest):
    """Entries of logit -inf: a share of 0, of some, of all, of closed classes; the scores'
    probability there is to go."""
    from warpgbm_amd import losses

    for K, k in ((5, 3), (12, 5), (40, 8), (300, 20), (900, 20), (9000, 64), (70_001, 64)):
        print_case("ruled out", order, K, k, rest)
        n = 8
        g = torch.Generator().manual_seed(K)
        s = torch.randn((n, K), generator=g)
        cls = torch.argsort(torch.rand((n, K), generator=g), 1)[:, :k].to(torch.int32).contiguous()
        t = torch.log_softmax(torch.randn((n, K), generator=g), 1)
        logits = t.gather(1, cls.long())
        logits[0, 0] = logits[1, k - 1] = -INF
        logits[2, 1:] = -INF
        logits[3] = -INF
        logits[4, 0] = -INF
        s[4, cls[4, 0].long()] = -INF
        s[5, cls[5, 0].long()] = -INF
        logits[5, 1:] = -INF
        w = 0.5 + torch.rand(n, generator=g)
        s = s if order == "row" else s.t().contiguous().t()
        norm = 0.0 if rest else None
        got = losses.distill_loss(to_gpu(s), cls.cuda(), logits.cuda(), log_norm=norm,
                                  weight=w.cuda())
        want = distill64(s, cls, logits, norm, w, 1.0)
        assert bool(want["live"][3]) == rest and bool(want["live"][5]) == rest
        check_distill(got, want, w, 1.0, "f32")


# --------------------------------------------------------------------- lowest masks
@pytest.mark.gpu
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("order", ["row", "class"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_lowest_masks_at_low_temperatures(gpu, dtype, order, rest):
    """A class masked by the type's lowest number that the teacher takes: a divergence of
    some 10^37, which fits, though log(q / p) at the temperature does not."""
    from warpgbm_amd import losses

    low = torch.finfo(DTYPES[dtype]).min
    for K, k in ((4, 2), (12, 5), (40, 8), (300, 20), (900, 20), (9000, 64), (140_003, 64)):
        for tau in (0.7, 0.05):
            print_case("lowest", dtype, order, K, k, tau, rest)
            n = 6
            g = torch.Generator().manual_seed(K)
            s = torch.randn((n, K), generator=g).to(DTYPES[dtype])
            cls = torch.argsort(torch.rand((n, K), generator=g), 1)[:, :k].to(torch.int32).contiguous()
            t = torch.log_softmax(torch.randn((n, K), generator=g) / tau, 1)
            t[0] = -math.log(K)
            logits = tau * t.gather(1, cls.long())
            others = torch.ones((n, K), dtype=torch.bool).scatter_(1, cls.long(), False)
            s[0, cls[0, 1].long()] = low             # an entry
            s[1, cls[1].long()] = low                # the whole list
            s[2, others[2]] = low                    # what is not listed
            s[3, others[3]] = low
            s[3, cls[3, 0].long()] = low
            w = 0.5 + torch.rand(n, generator=g)
            s = s if order == "row" else s.t().contiguous().t()
            norm = 0.0 if rest else None
            got = losses.distill_loss(to_gpu(s), cls.cuda(), logits.cuda(), log_norm=norm,
                                      weight=w.cuda(), temperature=tau)
            want = distill64(s, cls, logits, norm, w, tau)
            assert 1e35 < want["loss"].max() < torch.finfo(torch.float32).max
            # the other classes' parts of their sum from their own maximum: the log of a sum
            # of e^(-10^39) keeps no number of them, in float64 either
            x = s.double() / tau
            x = torch.where(others, x, -INF)
            r = torch.exp(x - x.max(1, keepdim=True).values)
            r = r / r.sum(1, keepdim=True)
            p, q, Q = want["p"], want["q"], want["Q"][:, None]
            # A share q = e^y, y = log q, has the power of two of a float32 product: the
            # difference's, the product's and log2(e) / tau's roundings are 2.3 |y| 2^-24 of
            # it. Elsewhere that is a rounding of the largest share (|y| e^-|y| < 1 / e);
            # here q multiplies log(q / p) of any size, and so does its rounding.
            value = w.double() * tau * tau
            y = torch.where(q > 0, q.log().abs(), 0.0)
            gap = torch.where(q > 0, y + want["far"], 0.0)
            gap_rest = torch.where(want["Q"] > 0, want["rest"].abs() + 30.0, 0.0)
            tol = value * U * (STEPS * want["lost"] + (k + 16) * 4
                               + (q * gap * (16 + 2.3 * y)).sum(1) + (k + 8) * gap_rest)
            check(got.loss, want["loss"], tol + U * want["loss"], "loss")
            scale = (w.double() * tau)[:, None]
            grad = scale * (p - q - Q * r)
            tol = scale * U * ((STEPS + 64) * (p + q + r * (want["P"][:, None] + Q))
                               + (k + 8) * (q + r))
            half = U if dtype == "f32" else 2.0 ** -8 * (1 + 1e-3)
            check(got.grad, grad, tol + half * grad.abs() + 1e-37, "gradient")


# --------------------------------------------------------------------- far from 0
FAR = [1e6, -1e10, 1e20, -1e30, torch.finfo(torch.float32).max, torch.finfo(torch.float32).min]


@pytest.mark.gpu
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("order", ["row", "class"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_distillation_of_rows_and_teachers_far_from_0(gpu, dtype, order, rest):
    """Rows masked as a whole by the lowest number, and others of equal scores of any size:
    even probabilities; lists of logits of any size, whose differences count."""
    from warpgbm_amd import losses

    for K, k in ((4, 2), (12, 5), (40, 8), (300, 20), (900, 20), (9000, 64), (140_003, 64)):
        print_case("far", dtype, order, K, k, rest)
        n = 2 * len(FAR)
        g = torch.Generator().manual_seed(K)
        s = torch.randn((n, K), generator=g)
        t = torch.log_softmax(torch.randn((n, K), generator=g), 1)
        cls = torch.argsort(torch.rand((n, K), generator=g), 1)[:, :k].to(torch.int32).contiguous()
        logits = t.gather(1, cls.long())
        for i, far in enumerate(FAR):
            s[i] = far
            if not rest:
                logits[len(FAR) + i] = far
        s = s.to(DTYPES[dtype]).clamp(torch.finfo(DTYPES[dtype]).min, torch.finfo(DTYPES[dtype]).max)
        s = s if order == "row" else s.t().contiguous().t()
        w = 0.5 + torch.rand(n, generator=g)
        norm = 0.0 if rest else None
        got = losses.distill_loss(to_gpu(s), cls.cuda(), logits.cuda(), log_norm=norm,
                                  weight=w.cuda())
        check_distill(got, distill64(s, cls, logits, norm, w, 1.0), w, 1.0, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
def test_alternatives_of_rows_far_from_0(gpu, order):
    """Differences of scores count: rows of few values at any distance from 0 have the bits
    of the same rows at 0."""
    from warpgbm_amd import losses

    for K, k in ((4, 2), (12, 5), (40, 8), (300, 20), (900, 20), (9000, 64), (140_003, 64)):
        print_case("far alternatives", order, K, k)
        n = len(FAR)
        g = torch.Generator().manual_seed(K)
        near = torch.zeros((n, K))
        far = torch.tensor(FAR)[:, None].expand(n, K).clone()
        for i in range(n):
            gone = torch.rand(K, generator=g) < 0.3
            gone[i % K] = False
            near[i, gone] = far[i, gone] = -INF
        cls = torch.argsort(torch.rand((n, K), generator=g), 1)[:, :k].to(torch.int32).contiguous()
        up, ge = torch.randn((n, k), generator=g).cuda(), torch.randn(n, generator=g).cuda()
        a = torch.randint(0, K, (n,), generator=g, dtype=torch.int32).cuda()
        got = []
        for s in (near, far):
            s = to_gpu(s if order == "row" else s.t().contiguous().t())
            f = losses.class_alternatives(s, k, labels=a, temperature=0.7)
            d = losses.class_alternatives_grad(s, f.norm, labels=a, grad_label_log_prob=ge,
                                               classes=cls.cuda(), grad_log_prob=up,
                                               grad_entropy=ge, temperature=0.7)
            got.append((f.classes, f.log_prob, f.entropy, f.label_log_prob, f.norm[:, 1:], d))
        for x, y in zip(*got):
            assert torch.equal(x, y) and not torch.isnan(y).any()


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
def test_shares_below_and_above_float32_s_range(gpu, order):
    """A row that may take only classes to which the teacher gives e^-100 and less: they
    are scaled to sum 1, whatever is left of the teacher. Logits with a log norm far below
    theirs, the same."""
    from warpgbm_amd import losses

    for K, k in ((4, 3), (12, 5), (40, 8), (300, 20), (900, 20), (9000, 64), (70_001, 64)):
        print_case("range", order, K, k)
        n = 6
        g = torch.Generator().manual_seed(K)
        s = torch.randn((n, K), generator=g)
        cls = torch.argsort(torch.rand((n, K), generator=g), 1)[:, :k].to(torch.int32).contiguous()
        logits = torch.randn((n, k), generator=g)
        others = torch.ones((n, K), dtype=torch.bool).scatter_(1, cls.long(), False)
        logits[:4, 0] = torch.tensor([100.0, 200.0, 600.0, 100.0])
        ln = torch.logsumexp(logits.double(), 1).float()
        for i in range(4):                          # the teacher's class is closed
            s[i, cls[i, 0].long()] = -INF
        s[3, others[3]] = -INF                      # and all that it does not list
        s[4, others[4]] = -INF
        logits[4:] += torch.tensor([[100.0], [300.0]])  # shares of e^100 and e^300
        ln[4:] = 0.0
        w = 0.5 + torch.rand(n, generator=g)
        s = s if order == "row" else s.t().contiguous().t()
        got = losses.distill_loss(to_gpu(s), cls.cuda(), logits.cuda(), log_norm=ln.cuda(),
                                  weight=w.cuda())
        want = distill64(s, cls, logits, ln, w, 1.0)
        assert want["live"].all()
        check_distill(got, want, w, 1.0, "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
def test_nan_shows_in_its_row_of_a_distillation(gpu, order):
    """In a score, a logit, a log norm, a weight; not in entries that are not used or rows
    that are left out, and in no other row."""
    from warpgbm_amd import losses

    nan = float("nan")
    for K, k in ((4, 2), (12, 5), (40, 8), (300, 20), (900, 20), (9000, 64), (70_001, 64)):
        print_case("nan row", order, K, k)
        n = 16
        g = torch.Generator().manual_seed(K)
        s = torch.randn((n, K), generator=g)
        cls = torch.argsort(torch.rand((n, K), generator=g), 1)[:, :k].to(torch.int32).contiguous()
        t = torch.log_softmax(torch.randn((n, K), generator=g), 1)
        logits, ln, w = t.gather(1, cls.long()), torch.zeros(n), torch.ones(n)
        others = torch.ones((n, K), dtype=torch.bool).scatter_(1, cls.long(), False)
        s[1, cls[1, 0].long()] = nan
        s[2, int(others[2].nonzero()[0])] = nan
        logits[3, 0] = nan
        ln[4] = nan                       # (counts with log norms only)
        ln[5] = nan
        s[5, others[5]] = -INF            # (no rest, whatever the log norm)
        w[6] = nan
        s[8], logits[8], ln[8], w[8] = nan, nan, nan, 0.0
        cls[9, 1], logits[9, 1] = -1, nan
        s[10, cls[10, 0].long()], logits[10, 0] = -INF, nan   # (a closed class: of the rest)
        s[11, cls[11, 0].long()], logits[11, 0] = -INF, nan
        s[11, others[11]] = -INF                              # (no rest)
        s = s if order == "row" else s.t().contiguous().t()
        for norms, rows in ((None, {1, 2, 3, 6}), (ln, {1, 2, 3, 4, 5, 6, 10})):
            r = losses.distill_loss(to_gpu(s), cls.cuda(), logits.cuda(), weight=w.cuda(),
                                    log_norm=None if norms is None else norms.cuda())
            assert set(torch.isnan(r.loss).nonzero()[:, 0].tolist()) == rows
            assert set(torch.isnan(r.grad).any(1).nonzero()[:, 0].tolist()) == rows
            assert r.loss[8] == 0 and (r.grad[8] == 0).all()


# --------------------------------------------------------------------- launches in parts
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,order,K", [("bf16", "row", 257), ("f32", "class", 40)])
def test_lists_of_rows_that_go_in_parts(gpu, dtype, order, K):
    """More rows than a launch's threads are counted for: rows at both sides of the part's
    end and the last ones against the same rows alone, with every argument of a row."""
    from warpgbm_amd import losses

    part = ((1 << 32) - 1) // (K + 3) // 1024 * 1024
    n, k = part + 77_777, 3
    print_case("parts", dtype, order, n, K)
    s = torch.empty((n, K) if order == "row" else (K, n), dtype=DTYPES[dtype], device="cuda")
    s.normal_(generator=torch.Generator(device="cuda").manual_seed(5))
    s = s if order == "row" else s.t()
    at = torch.cat([torch.arange(3), torch.arange(part - 5, part + 5), torch.arange(n - 5, n)]).cuda()
    i = torch.arange(n, device="cuda")
    a = (i % K).to(torch.int32)
    w, ln = 0.5 + (i % 7).float(), 2.0 + (i % 5).float()
    few = s[at].contiguous() if order == "row" else s.t()[:, at].contiguous().t()
    A, W, N = a[at], w[at], ln[at]
    f = losses.class_alternatives(s, k, labels=a, temperature=1.5)
    F = losses.class_alternatives(few, k, labels=A, temperature=1.5)
    for x, y in zip(f, F):
        assert torch.equal(x[at], y)
    # (lists of either order)
    cls = f.classes if order == "row" else f.classes.t().contiguous().t()
    r = losses.distill_loss(s, cls, f.log_prob, log_norm=ln, weight=w)
    R = losses.distill_loss(few, F.classes, F.log_prob, log_norm=N, weight=W)
    assert torch.equal(r.loss[at], R.loss) and torch.equal(r.grad[at], R.grad)
    del r
    g = losses.class_alternatives_grad(s, f.norm, labels=a, grad_label_log_prob=w, classes=cls,
                                       grad_log_prob=f.log_prob, grad_entropy=ln, temperature=1.5)
    G = losses.class_alternatives_grad(few, F.norm, labels=A, grad_label_log_prob=W,
                                       classes=F.classes, grad_log_prob=F.log_prob, grad_entropy=N,
                                       temperature=1.5)
    assert torch.equal(g[at], G)
    del s, g, f
    torch.cuda.empty_cache()


# --------------------------------------------------------------------- refusals
def test_what_is_no_number_is_refused_as_other_arguments_are():
    from warpgbm_amd import losses

    for x in (None, "warm", [1.0], (2.0, 3.0), 1j):
        with pytest.raises(RuntimeError, match="temperature must be a number"):
            losses._temperature(x)
    assert losses._temperature(torch.tensor(2.0)) == 2.0 == losses._temperature(2)


@pytest.mark.gpu
def test_lists_refuse_what_is_no_number(gpu):
    from warpgbm_amd import losses

    s = torch.zeros((4, 8)).cuda()
    c, x = torch.zeros((4, 2), dtype=torch.int32).cuda(), torch.zeros((4, 2)).cuda()
    for bad in ("zero", [0.0] * 4, 1j):
        with pytest.raises(RuntimeError, match="log_norm must be a number"):
            losses.distill_loss(s, c, x, log_norm=bad)
    for call in (lambda t: losses.class_alternatives(s, 2, temperature=t),
                 lambda t: losses.class_alternatives_grad(s, torch.zeros((4, 3)).cuda(), temperature=t),
                 lambda t: losses.distill_loss(s, c, x, temperature=t)):
        with pytest.raises(RuntimeError, match="temperature must be a number"):
            call(None)

"""The losses at scores of any finite size: rows far from zero, classes masked
by finite numbers, whole ranges of them, and sums of very many rows, against
float64 forms."""
import math

import numpy as np
import pytest
import torch

from conftest import print_case
from test_losses import (DTYPES, F64, STEPS, U, balance_want, check, grad_tol, log_softmax64,
                         norm_tol, policy_scales, policy_want, run_policy, to_gpu)

# every frame, and rows in ranges: class-major of more than 512 classes, row-major
# of more than 65536 float32 or 131072 16-bit classes
SHAPES = [(40, 3), (70, 10), (65, 40), (33, 100), (24, 257), (18, 700), (9, 5000), (9, 70_001)]
LONG = {"f32": (9, 70_001), "bf16": (9, 140_003), "f16": (9, 140_003)}
OFFSETS = [0.0, 1e3, -1e3, 1e5, -1e6, 1e10, -1e10, 1e30, -3e38]
OFFSETS_F16 = [0.0, 1e3, -1e3, 3e4, -6e4, 6e4]
MASKS = [-1e4, -1e9, -1e10, -1e30, float(torch.finfo(torch.float32).min)]
MASKS_F16 = [-1e4, -6e4, float(torch.finfo(torch.float16).min)]


def place(v, order):
    return v if order == "row" else v.t().contiguous().t()


def far_rows(n, K, dtype, order, seed, roll=0):
    """Rows of a few units' spread about offsets of many sizes."""
    g = torch.Generator().manual_seed(seed)
    off = OFFSETS_F16 if dtype == "f16" else OFFSETS
    at = torch.tensor([off[(i + roll) % len(off)] for i in range(n)], dtype=F64)
    v = at[:, None] + 2 * torch.randn((n, K), generator=g, dtype=F64)
    return place(v.to(DTYPES[dtype]), order)


def masked_rows(n, K, dtype, order, seed):
    """Rows with blocks of classes masked by finite numbers: the first half, the
    second, all but one class, every other class; the open classes."""
    g = torch.Generator().manual_seed(seed)
    low = MASKS_F16 if dtype == "f16" else MASKS
    v = 2 * torch.randn((n, K), generator=g)
    shut = torch.zeros((n, K), dtype=torch.bool)
    for i in range(n):
        one = int(torch.randint(0, K, (1,), generator=g))
        way = i % 4
        if way == 0:
            shut[i, :K // 2] = True
        elif way == 1:
            shut[i, (K + 1) // 2:] = True
        elif way == 2:
            shut[i] = True
            shut[i, one] = False
        else:
            shut[i, ::2] = True
        v[i, shut[i]] = max(low[(i // 4) % len(low)], float(torch.finfo(DTYPES[dtype]).min))
    return place(v.to(DTYPES[dtype]), order), ~shut


def labels_of(s, allowed, seed):
    g = torch.Generator().manual_seed(seed)
    p = torch.softmax(s.to(F64), 1) if allowed is None else allowed.to(F64)
    return torch.multinomial(p, 1, generator=g)[:, 0].to(torch.int32)


def check_log_probs(s, a, dtype):
    """class_log_probs and its gradient (finite scores only)."""
    from warpgbm_amd import losses

    n = s.shape[0]
    up = torch.randn(n, generator=torch.Generator().manual_seed(n))
    sd = to_gpu(s)
    r = losses.class_log_probs(sd, a.cuda())
    L = log_softmax64(s)
    lp = L.gather(1, a.long()[:, None])[:, 0]
    check(r.log_prob, lp, norm_tol(lp), "log_prob")
    top = s.to(F64).max(1).values
    check(r.norm[:, 0], top, 0.0, "maximum")
    spread = torch.exp(s.to(F64) - top[:, None]).sum(1).log()
    check(r.norm[:, 1], spread, norm_tol(spread), "log of the sum")
    got = losses.class_log_probs_grad(sd, a.cuda(), r.norm, up.cuda())
    grad = -L.exp() * up.to(F64)[:, None]
    at = torch.arange(n)
    grad[at, a.long()] = -torch.expm1(lp) * up.to(F64)
    check(got, grad, grad_tol(grad, up.abs().to(F64), dtype), "gradient")


def policy_dict(s, rs, a, seed):
    n = s.shape[0]
    g = torch.Generator().manual_seed(seed)
    lp = log_softmax64(s).gather(1, a.long()[:, None])[:, 0].float()
    return dict(s=s, ref_s=rs, a=a, old=lp + 0.3 * torch.randn(n, generator=g),
                adv=torch.randn(n, generator=g), w=0.5 + torch.rand(n, generator=g),
                ref=lp + 0.4 * torch.randn(n, generator=g))


def check_policy(d, dtype):
    clip, c = (0.2, 0.3), 0.25
    for kl in ("none", "sampled", "exact"):
        loss, lp, k, grad, live = policy_want(d, kl, clip, c)
        scale = policy_scales(d, kl, c, k, live)
        r = run_policy(d, kl, clip, c)
        check(r.log_prob, lp, norm_tol(lp), "log_prob")
        check(r.loss, loss, STEPS * U * (scale + d["w"].to(F64)), "loss")
        if kl != "none":
            check(r.kl, k, STEPS * U * (scale / d["w"].to(F64) / c + 1), "kl")
        check(r.grad, grad, grad_tol(grad, scale, dtype), "gradient")


def check_balance(s, dtype, top_k):
    from warpgbm_amd import losses

    n, K = s.shape
    coef = 3.0 * n
    loss, counts, prob, grad, live = balance_want(s, None, top_k, coef)
    r = losses.balance_loss(to_gpu(s), top_k=top_k, coef=coef)
    assert torch.equal(r.counts.cpu(), counts)
    check(r.prob, prob, 2 * STEPS * U * prob + 1e-12, "prob")
    check(r.loss, loss, 2 * STEPS * U * loss.abs() + 1e-12, "loss")
    f = counts.to(F64) / (n * top_k)
    P = torch.softmax(s.to(F64), 1)
    tol = STEPS * U * (coef * K / n * (P * (f + (P @ f)[:, None]))).amax(1) + 1e-12
    check(r.grad, grad, grad_tol(grad, torch.zeros(n, dtype=F64), dtype) + tol[:, None], "grad")


def shapes_of(dtype):
    return SHAPES + ([LONG[dtype]] if LONG[dtype] not in SHAPES else [])


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_rows_far_from_zero(gpu, dtype, order):
    """A row's offset, however large, changes nothing but the scores' own
    rounding."""
    for j, (n, K) in enumerate(shapes_of(dtype)):
        print_case("far rows", dtype, order, n, K)
        s = far_rows(n, K, dtype, order, 400 + j)
        a = labels_of(s, None, j)
        check_log_probs(s, a, dtype)
        rs = far_rows(n, K, dtype, order, 500 + j, roll=2)
        check_policy(policy_dict(s, rs, a, 600 + j), dtype)
        if K <= 4096:
            check_balance(s, dtype, min(K, 1 + j % 3))


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_classes_masked_by_finite_numbers(gpu, dtype, order):
    """Blocks of -1e4 to the type's lowest value count as far less likely classes,
    also where a range or a thread's part of a row holds nothing else."""
    for j, (n, K) in enumerate(shapes_of(dtype)):
        print_case("finite masks", dtype, order, n, K)
        n = max(n, 20)
        s, allowed = masked_rows(n, K, dtype, order, 700 + j)
        any_label = torch.randint(0, K, (n,), generator=torch.Generator().manual_seed(j),
                                  dtype=torch.int32)
        check_log_probs(s, any_label, dtype)
        a = labels_of(s, allowed, j)
        g = torch.Generator().manual_seed(800 + j)
        noise = torch.where(allowed, 0.5 * torch.randn((n, K), generator=g), torch.zeros(()))
        rs = place((s.float() + noise).to(s.dtype), order)
        check_policy(policy_dict(s, rs, a, 900 + j), dtype)
        if K <= 4096:
            check_balance(s, dtype, min(K, 1 + j % 3))


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
def test_divergence_from_a_reference_masked_by_finite_numbers(gpu, order):
    """Classes that only the reference masks: the divergence is as large as the
    mask times their probability, and finite."""
    for j, (n, K) in enumerate(SHAPES):
        print_case("reference masked", order, n, K)
        n = max(n, 20)
        rs, allowed = masked_rows(n, K, "f32", order, 1000 + j)
        rs.clamp_(min=-1e30)
        g = torch.Generator().manual_seed(j)
        s = place(2 * torch.randn((n, K), generator=g), order)
        check_policy(policy_dict(s, rs, labels_of(s, None, j), 1100 + j), "f32")


# (type, order, rows, classes): some 4096, 2048 and 1950 rows for each thread of the
# first pass
CHAINS = [("f32", "row", (1 << 30) - 5, 2), ("bf16", "class", (1 << 30) + 77, 2),
          ("bf16", "class", (1 << 29) + 77, 17), ("f32", "row", 1_000_003, 4096)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,order,n,K", CHAINS)
def test_balance_of_very_many_equal_rows(gpu, dtype, order, n, K):
    """Equal rows: one after the other in float32 their probabilities would round
    the same way each time, thousands of times."""
    from warpgbm_amd import losses

    print_case("very many rows", dtype, order, n, K)
    torch.cuda.empty_cache()
    row = torch.randn(K, generator=torch.Generator().manual_seed(K)).to(DTYPES[dtype])
    if K == 2:
        row = torch.tensor([0.0, 1.3]).to(DTYPES[dtype])
    if order == "row":
        s = torch.empty((n, K), dtype=row.dtype, device="cuda")
        s[:] = row.cuda()
    else:
        s = torch.empty((K, n), dtype=row.dtype, device="cuda").t()
        for k in range(K):
            s[:, k] = float(row[k])
    r = losses.balance_loss(s, with_grad=False)
    del s
    prob = torch.softmax(row.to(F64), 0)
    counts = torch.zeros(K, dtype=torch.int64)
    counts[row.argmax()] = n
    assert torch.equal(r.counts.cpu(), counts)
    # 256 additions one after the other, ten more in a workgroup; 70 roundings of a
    # row's exponentials (their powers: 2.3 * 8 * 1.44 ln 2, at most 19), of its sum and
    # of the quotient
    check(r.prob, prob, (256 + 10 + 70) * U * prob, "prob")
    want = K * prob[row.argmax()]
    check(r.loss, want, (256 + 10 + 70 + 1) * U * want, "loss")
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_large_and_small_ratios(gpu):
    """Ratios from e^-80 to e^85 that no border holds, of rows of one class, whose
    log-probability is 0: the loss is the ratio."""
    from warpgbm_amd import losses

    n = 200_000
    g = torch.Generator().manual_seed(12)
    old = 80 - 165 * torch.rand(n, generator=g)
    s = torch.randn((n, 1), generator=g)
    r = losses.policy_loss(s.cuda(), torch.zeros(n, dtype=torch.int32, device="cuda"), old.cuda(),
                           -torch.ones(n, device="cuda"), clip=(1.0, 0.2))
    assert not r.log_prob.any()
    want = torch.exp(-old.to(F64))
    # v_exp_f32: one ulp (2 * 2^-24 of the value at most); the correction's product and
    # sum round once more
    check(r.loss, want, 4 * U * want, "loss")


def test_refused_sizes_keep_their_message():
    """A refusal says why each time, whatever was refused in between."""
    from warpgbm_amd import losses

    for _ in range(2):
        with pytest.raises(RuntimeError, match="at most 4096 classes"):
            losses._bytes_of("wgbm_balance_loss_workspace", 0, 6, 5000, False)
        with pytest.raises(RuntimeError, match="n_classes must be in"):
            losses._bytes_of("wgbm_class_log_probs_workspace", 0, 6, (1 << 24) + 1, False)


def test_shared_memory_is_found():
    """Views of one buffer: whether they share an element, for rows between rows,
    columns, single rows and vectors."""
    from warpgbm_amd import losses

    rng = np.random.default_rng(5)
    buf = torch.arange(400, dtype=torch.int16)

    def view():
        at, way = int(rng.integers(0, 120)), int(rng.integers(0, 4))
        n, K, gap = (int(x) for x in rng.integers(1, 6, 3))
        if way == 0:
            return torch.as_strided(buf, (n * K,), (1,), at)
        if way == 1:
            return torch.as_strided(buf, (n, K), (K + gap * 5, 1), at)
        if way == 2:
            return torch.as_strided(buf, (n, K), (1, n + gap * 5), at)
        # (a stride that two views often have in common)
        return torch.as_strided(buf, (n, K), (20, 1), at)

    seen = [0, 0]
    for _ in range(4000):
        a, b = view(), view()
        share = bool(set(a.reshape(-1).tolist()) & set(b.reshape(-1).tolist()))
        assert losses._meet(a, b) == share, (a, b)
        seen[share] += 1
    assert min(seen) > 500
    assert not losses._meet(buf[:0], buf) and not losses._meet(buf[:0].view(0, 3), buf)


@pytest.mark.gpu
def test_a_gradient_that_shares_memory_is_refused(gpu):
    from warpgbm_amd import losses

    both = torch.zeros((6, 9), device="cuda")
    s, a = both[:, :4], torch.zeros(6, dtype=torch.int32, device="cuda")
    f = torch.zeros(6, device="cuda")
    for grad in (both[:, 1:5], both[:, 3:7], both[:, :4]):
        with pytest.raises(RuntimeError, match="scores' memory"):
            losses.balance_loss(s, grad=grad)
        with pytest.raises(RuntimeError, match="share memory with an input"):
            losses.policy_loss(torch.zeros((6, 4), device="cuda"), a, f, f, ref_scores=s,
                               grad=grad)
    flat = torch.zeros(48, device="cuda")
    with pytest.raises(RuntimeError, match="share memory with an input"):
        losses.policy_loss(s.clone(), a, flat[20:26], f, grad=flat[:24].view(6, 4))
    # rows between the scores' rows are not the scores'
    want = losses.balance_loss(s.clone())
    got = losses.balance_loss(s, grad=both[:, 5:])
    assert torch.equal(got.grad, want.grad) and not both[:, :5].any()


@pytest.mark.gpu
@pytest.mark.parametrize("K", [40_001, 131_072, 131_081])
def test_policy_workspace_without_a_reference(gpu, K):
    """Rows that fit registers without a reference's take no working memory then,
    by torch or by the C entry."""
    import ctypes as C

    from warpgbm_amd import _lib, losses

    n = 6
    s = far_rows(n, K, "bf16", "row", 3).cuda()
    a = torch.zeros(n, dtype=torch.int32, device="cuda")
    f = torch.ones(n, device="cuda")
    old = -12 * f

    def allocations(**kw):
        before = torch.cuda.memory_stats()["allocation.all.allocated"]
        r = losses.policy_loss(s, a, old, f, **kw)
        return torch.cuda.memory_stats()["allocation.all.allocated"] - before, r

    long = K > 131_072
    count, r = allocations()
    assert count == 3 + long  # the gradient, the loss, the log-probabilities
    count, with_ref = allocations(ref_scores=s)
    assert count == 5  # the divergence and the working memory too
    assert torch.allclose(r.log_prob, with_ref.log_prob, rtol=1e-5, atol=1e-5)
    if long:
        return
    v = losses._matrix(s, "scores")
    assert gpu.wgbm_policy_loss_workspace(C.byref(v)) > 0
    args = _lib.PolicyArgs(a.data_ptr(), old.data_ptr(), f.data_ptr(), None, None, None, 0.2, 0.2,
                           0.0)
    loss, lp = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    rc = gpu.wgbm_policy_loss(C.byref(v), C.byref(args), loss.data_ptr(), lp.data_ptr(), None, None,
                              0, None, 0, _lib.current_stream_ptr())
    assert rc == 0 and torch.equal(loss, r.loss) and torch.equal(lp, r.log_prob)
    rv = losses._matrix(s, "scores")
    args.ref_scores = C.pointer(rv)
    rc = gpu.wgbm_policy_loss(C.byref(v), C.byref(args), loss.data_ptr(), lp.data_ptr(), None, None,
                              0, None, 0, _lib.current_stream_ptr())
    assert rc == 1000 and "workspace too small" in gpu.wgbm_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["row", "class"])
@pytest.mark.parametrize("K", [3, 40, 700, 70_001])
def test_divergence_from_a_reference_without_a_class(gpu, K, order):
    """It excludes every class: the divergence is infinite, and does no harm where
    it does not count."""
    from warpgbm_amd import losses

    n = 5
    g = torch.Generator().manual_seed(K)
    s = place(torch.randn((n, K), generator=g), order)
    rs = place(s.clone(memory_format=torch.contiguous_format) + 0.1, order)
    rs[2] = -math.inf
    a, old = torch.zeros(n, dtype=torch.int32).cuda(), torch.full((n,), -2.0).cuda()
    adv = torch.ones(n).cuda()
    r = losses.policy_loss(to_gpu(s), a, old, adv, ref_scores=to_gpu(rs), kl_coef=0.5)
    rest = [0, 1, 3, 4]
    assert r.kl[2] == math.inf and r.loss[2] == math.inf
    assert torch.isfinite(r.kl[rest]).all() and torch.isfinite(r.grad[rest]).all()
    zero = losses.policy_loss(to_gpu(s), a, old, adv, ref_scores=to_gpu(rs))
    plain = losses.policy_loss(to_gpu(s), a, old, adv)
    assert zero.kl[2] == math.inf and torch.isfinite(zero.grad).all()
    # (the frames may differ: the classes are added in another order)
    assert torch.allclose(zero.loss, plain.loss, rtol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [2056, 4104])
def test_launches_of_more_than_2_to_the_32_threads(gpu, K):
    """Rows of 256 threads each, more than 2^24 of them: the gradient's of 257 to 512
    chunks of 16 bytes, the log-probabilities' of 513 to 1024."""
    from warpgbm_amd import losses

    n, m = (1 << 24) + 9000, 60
    matrices = 1 if K > 4096 else 2
    print_case("threads", n, K)
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < matrices * 2 * n * K + (4 << 30):
        pytest.skip("the card's memory is in use")
    s = torch.zeros((n, K), dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(3)
    # the ends, and rows by where 2^32 threads are and by where parts of 4095 * 1024
    # rows end
    at = [0, 4095 * 1024 - m // 2, 4 * 4095 * 1024 - m // 2, (1 << 24) - m // 2, n - m]
    for i in at:
        s[i:i + m] = 2 * torch.randn((m, K), generator=gen, device="cuda")
    a = torch.randint(0, K, (n,), generator=gen, device="cuda", dtype=torch.int32)
    up = torch.randn(n, generator=gen, device="cuda")
    f = losses.class_log_probs(s, a)
    even = torch.ones(n, dtype=torch.bool, device="cuda")
    for i in at:
        even[i:i + m] = False
    flat = f.log_prob[even]
    assert ((flat + math.log(K)).abs() <= norm_tol(torch.tensor(math.log(K))).item()).all()
    grad = losses.class_log_probs_grad(s, a, f.norm, up) if matrices == 2 else None
    for i in at:
        x, b = s[i:i + m].cpu(), a[i:i + m].cpu().long()
        L = log_softmax64(x)
        lp = L.gather(1, b[:, None])[:, 0]
        check(f.log_prob[i:i + m], lp, norm_tol(lp), "log_prob")
        if grad is None:
            continue
        u = up[i:i + m].cpu().to(F64)
        want = -L.exp() * u[:, None]
        want[torch.arange(m), b] = -torch.expm1(lp) * u
        check(grad[i:i + m], want, grad_tol(want, u.abs(), "bf16"), "gradient")
    if grad is not None:
        # (a row of equal scores; every 1009th, so that a part left out shows)
        some = torch.arange(0, n, 1009, device="cuda")
        some = some[even[some]]
        want = -up[some] / K
        other = (a[some] + 1) % K
        got = grad[some, other.long()].float()
        assert ((got - want).abs() <= (2.0 ** -8 + STEPS * U) * want.abs()).all()
    del s, grad
    torch.cuda.empty_cache()

"""The estimator's objectives of warpgbm_amd.losses, and the engine's given
gradients."""
import numpy as np
import pytest
import torch

from conftest import print_case
from test_losses import log_softmax64, policy64, preference64

def table(n, F, seed, informative=4):
    rng = np.random.default_rng(seed)
    X = rng.standard_normal((n, F), dtype=np.float32)
    u = X[:, :informative].sum(1) + 0.5 * X[:, 0] * X[:, 1]
    return X, u.astype(np.float32), rng


def engine_rounds(codes, order, start, eras, B, depth, trees, objective, targets, pred, rounds,
                  tuning=()):
    """Rounds of the native engine; targets(pred) gives each round's target."""
    from warpgbm_amd import device as D

    n, F = codes.n, codes.n_feats
    eng = D.Engine(codes, order, start, B, eras, depth, trees, objective, 5.0, 0.0, 1e-6, 0.3)
    for key, value in tuning:
        eng.set_tuning(key, value)
    H = (1 << (depth + 1)) - 1
    sel = torch.arange(F, dtype=torch.int32, device="cuda")
    out = []
    for _ in range(rounds):
        rec = dict(feat=torch.empty((trees, H), dtype=torch.int32, device="cuda"),
                   bin=torch.zeros((trees, H), dtype=torch.int32, device="cuda"),
                   leaf=torch.zeros((trees, H), dtype=torch.float32, device="cuda"),
                   count=torch.zeros((trees, H), dtype=torch.int64, device="cuda"),
                   gain=torch.zeros((trees, H, eras), dtype=torch.float32, device="cuda"))
        eng.round(targets(pred), pred, sel, rec)
        feat = rec["feat"].cpu()
        out.append((feat, rec["bin"].cpu() * (feat >= 0), rec["leaf"].cpu() * (feat == -1)))
    eng.close()
    return out, pred


@pytest.mark.gpu
@pytest.mark.parametrize("n,eras", [(900, 1), (30_000, 1), (6_000, 7)])
def test_engine_gradients_of_squared_error(gpu, n, eras):
    """Objective 2 with the gradient pred - y grows regression's trees."""
    from warpgbm_amd import device as D

    print_case("engine gradients", n, eras)
    X, u, rng = table(n, 12, n)
    y = torch.from_numpy(u).cuda()
    Xd = torch.from_numpy(X).cuda()
    codes = D.bin_matrix(Xd, D.quantile_edges(Xd, 16), with_cm=True)
    uniq, _, order, start = D.era_layout(rng.integers(0, eras, n))
    order, start = torch.from_numpy(order).cuda(), torch.from_numpy(start).cuda()
    args = (codes, order, start, len(uniq), 16, 4, 1)
    a, pa = engine_rounds(*args, 0, lambda p: y, torch.zeros(n, device="cuda"), 3)
    b, pb = engine_rounds(*args, 2, lambda p: p - y, torch.zeros(n, device="cuda"), 3)
    for x, z in zip(a, b):
        assert all(torch.equal(s, t) for s, t in zip(x, z))
    assert torch.equal(pa, pb)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [700, 25_000])
def test_engine_gradients_of_softmax(gpu, n):
    """Objective 2 with p - onehot (the library's row softmax) grows softmax's
    trees, class-major scores."""
    from warpgbm_amd import device as D

    print_case("engine softmax gradients", n)
    K = 4
    X, u, rng = table(n, 9, n + 1)
    label = torch.from_numpy(np.digitize(u, [-2.0, 0.0, 2.0]).astype(np.int32)).cuda()
    Xd = torch.from_numpy(X).cuda()
    codes = D.bin_matrix(Xd, D.quantile_edges(Xd, 10), with_cm=True)
    order = torch.arange(n, dtype=torch.int32, device="cuda")
    start = torch.tensor([0, n], dtype=torch.int64, device="cuda")
    hot = torch.nn.functional.one_hot(label.long(), K).float()

    def grad(pred):
        p = pred.t().contiguous()
        D.softmax_rows(p)
        return (p - hot).t().contiguous()

    args = (codes, order, start, 1, 10, 3, K)
    a, pa = engine_rounds(*args, 1, lambda p: label, torch.zeros((K, n), device="cuda"), 3)
    b, pb = engine_rounds(*args, 2, grad, torch.zeros((K, n), device="cuda"), 3)
    for x, z in zip(a, b):
        assert all(torch.equal(s, t) for s, t in zip(x, z))
    assert torch.equal(pa, pb)


# --------------------------------------------------------------------- fits
def ranking_data(n, seed, sequences):
    X, u, rng = table(n, 8, seed)
    if sequences:
        length = rng.integers(0, 9, n // 4)
        seg = np.concatenate([[0], np.cumsum(length)])
        seg = seg[seg <= n].astype(np.int64)
        S = len(seg) - 1
        value = np.array([u[seg[k]:seg[k + 1]].sum() for k in range(S)])
    else:
        seg, S, value = None, n, u
    pairs = rng.integers(0, S, (2 * S, 2))
    flip = value[pairs[:, 0]] + rng.logistic(size=2 * S) < value[pairs[:, 1]]
    pairs[flip] = pairs[flip, ::-1]
    return X, u, pairs, seg, rng


def policy_data(n, K, seed):
    X, u, rng = table(n, 8, seed)
    best = np.digitize(u, np.quantile(u, np.arange(1, K) / K))
    y = rng.integers(0, K, n)
    adv = np.where(y == best, 1.0, -0.3) + 0.2 * rng.standard_normal(n)
    return X, y, adv.astype(np.float32), best, rng


KW = dict(num_bins=16, max_depth=3, learning_rate=0.3, min_child_weight=5, device="cuda")


def fits(kind, n=3000, K=3, seed=5):
    """(constructor arguments, fit arguments, float64 mean loss of scores)."""
    if kind == "policy":
        X, y, adv, best, rng = policy_data(n, K, seed)
        names = np.array(["left", "middle", "right"])[:K]
        w = (rng.random(n) < 0.9) * rng.random(n).astype(np.float32)
        old = np.full(n, -np.log(K), np.float32) + 0.1 * rng.standard_normal(n).astype(np.float32)
        ref = rng.standard_normal((n, K)).astype(np.float32)

        def loss(scores):
            s = torch.from_numpy(scores)
            a = torch.from_numpy(y)
            rows = policy64(s, a, torch.from_numpy(old), torch.from_numpy(adv),
                            torch.from_numpy(w), None, torch.from_numpy(ref), (0.2, 0.3), 0.1)[0]
            return rows.sum().item() / w.astype(np.float64).sum()

        return (dict(objective="policy", clip=(0.2, 0.3), kl_coef=0.1),
                dict(X=X, y=names[y], advantage=adv, behavior_log_prob=old, reference=ref,
                     sample_weight=w), loss)
    X, u, pairs, seg, rng = ranking_data(n, seed, kind != "items")
    w = (0.5 + rng.random(len(pairs))).astype(np.float32)
    pt = torch.from_numpy(pairs)
    S = n if seg is None else len(seg) - 1
    if kind == "policy_preference":
        y = np.digitize(u, [0.0]) ^ (rng.random(n) < 0.2)
        ref = (-0.7 + 0.1 * rng.standard_normal(n)).astype(np.float32)

        def loss(scores):
            lp = log_softmax64(torch.from_numpy(scores))[torch.arange(n), torch.from_numpy(y)]
            rows = preference64(lp, pt, S, seg, torch.from_numpy(ref), torch.from_numpy(w), 0.5, 0.1)
            return rows[0].sum().item() / w.astype(np.float64).sum()

        return (dict(objective="policy_preference", beta=0.5, label_smoothing=0.1),
                dict(X=X, y=y, pairs=pairs, segments=seg, pair_weight=w, reference=ref), loss)
    y = 0.1 * rng.standard_normal(n).astype(np.float32)

    def loss(scores):
        rows = preference64(torch.from_numpy(scores[:, 0]), pt, S, seg, torch.from_numpy(y),
                            torch.from_numpy(w), 0.5, 0.1)
        return rows[0].sum().item() / w.astype(np.float64).sum()

    return (dict(objective="preference", beta=0.5, label_smoothing=0.1),
            dict(X=X, y=y, pairs=pairs, segments=seg, pair_weight=w), loss)


KINDS = ["items", "sequences", "policy", "policy_preference"]


def scores_of(m, X):
    if m.objective == "preference":
        return m.predict(X)[:, None].astype(np.float64)
    return np.log(m.predict_proba(X).astype(np.float64))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_training_loss_is_that_of_the_predictions(gpu, kind):
    """Round j's training loss is the float64 loss of the predictions of a
    forest of j rounds."""
    from warpgbm_amd import WarpGBM

    print_case("fit", kind)
    new, given, loss = fits(kind)
    full = WarpGBM(n_estimators=5, **new, **KW).fit(**given)
    assert len(full.training_loss) == 5
    for rounds in (1, 3):
        m = WarpGBM(n_estimators=rounds, **new, **KW).fit(**given)
        want = loss(scores_of(m, given["X"]))
        # float32 sums of some thousand losses of about one
        assert full.training_loss[rounds] == pytest.approx(want, abs=2e-5)
        assert m.forest == full.forest[:rounds]
        assert m.training_loss == full.training_loss[:rounds]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_leaves_are_mean_negative_gradients(gpu, kind):
    """The first tree's leaves against the float64 gradient at the start."""
    from warpgbm_amd import WarpGBM

    print_case("leaves", kind)
    new, given, loss = fits(kind, seed=8)
    m = WarpGBM(n_estimators=1, **new, **KW).fit(**given)
    K = 1 if kind in ("items", "sequences") else m.num_classes
    n = given["X"].shape[0]
    # (the loss functions take arrays: differences of their total)
    trees = [m.forest[0]] if K == 1 else m.forest[0]
    codes = m.bin_inference_data(given["X"]).rm.cpu().numpy()
    total = given["sample_weight" if kind == "policy" else "pair_weight"]
    total = total.astype(np.float64).sum()

    def leaves(node, rows):
        if "leaf_value" in node:
            return [(node["leaf_value"], rows)]
        left = codes[rows, int(node["feature"])] <= int(node["bin"])
        return leaves(node["left"], rows[left]) + leaves(node["right"], rows[~left])

    for k, tree in enumerate(trees):
        for value, rows in leaves(tree, np.arange(n)):
            h = 1e-5
            up, down = np.zeros((n, K)), np.zeros((n, K))
            up[rows, k], down[rows, k] = h, -h
            slope = total * (loss(up) - loss(down)) / (2 * h)
            assert value == pytest.approx(-slope / len(rows), rel=2e-4, abs=2e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_warm_start_and_persistence(gpu, kind, tmp_path):
    from warpgbm_amd import WarpGBM

    print_case("warm start", kind)
    new, given, _ = fits(kind, seed=9)
    full = WarpGBM(n_estimators=6, **new, **KW).fit(**given)
    m = WarpGBM(n_estimators=4, warm_start=True, **new, **KW).fit(**given)
    m.n_estimators = 6
    m.fit(**given)
    assert m.forest == full.forest and m.training_loss == full.training_loss
    path = str(tmp_path / "m.pkl")
    full.save_model(path)
    back = WarpGBM().load_model(path)
    assert back.clip == full.clip and back.beta == full.beta
    X = given["X"]
    assert np.array_equal(back.predict(X), full.predict(X))
    if kind.startswith("policy"):
        lp = back.log_prob(X, given["y"])
        p = full.predict_proba(X)
        at = full.label_encoder.transform(given["y"])
        want = np.log(p.astype(np.float64)[np.arange(len(at)), at])
        assert np.allclose(lp, want, rtol=1e-5, atol=2e-6)
    else:
        with pytest.raises(ValueError, match="log_prob"):
            back.log_prob(X, given["y"])


@pytest.mark.gpu
def test_policy_with_balance_and_eras(gpu):
    """The balance term joins the gradient; eras and column subsets as for the
    other objectives."""
    from warpgbm_amd import WarpGBM

    n, K = 4000, 5
    X, y, adv, best, rng = policy_data(n, K, 3)
    eras = rng.integers(0, 3, n)
    losses = []
    for coef in (0.0, 0.5):
        m = WarpGBM(objective="policy", n_estimators=3, balance_coef=coef, balance_top_k=2,
                    colsample_bytree=0.7, random_state=1, **KW)
        m.fit(X, y, era_id=eras, advantage=adv)
        assert m.predict_proba(X).shape == (n, K)
        assert m.get_per_era_feature_importance().shape == (3, X.shape[1])
        losses.append(m.training_loss)
    # at uniform scores every class has probability 1/K and the two lowest
    # classes take all places: the balance loss is its coefficient
    assert losses[1][0] - losses[0][0] == pytest.approx(0.5, rel=1e-5)


# --------------------------------------------------------------------- refusals (CPU)
@pytest.mark.parametrize("kw,exc", [
    ({"beta": 0.0}, ValueError), ({"beta": "1"}, TypeError), ({"label_smoothing": 0.7}, ValueError),
    ({"clip": 0.2}, TypeError), ({"clip": (1.2, 0.2)}, ValueError), ({"clip": (0.2, -1)}, ValueError),
    ({"kl_coef": -0.1}, ValueError), ({"balance_coef": float("inf")}, ValueError),
    ({"balance_top_k": 0}, ValueError), ({"balance_top_k": 1.5}, TypeError),
])
def test_loss_parameters(kw, exc):
    from warpgbm_amd import WarpGBM

    with pytest.raises(exc):
        WarpGBM(objective="policy", **kw)


def test_fit_argument_refusals():
    from warpgbm_amd import WarpGBM

    X, y = np.zeros((6, 2), np.float32), np.zeros(6, np.float32)
    pairs = np.array([[0, 1], [2, 3]])

    def no(exc, text, objective, **kw):
        with pytest.raises(exc, match=text):
            WarpGBM(objective=objective).fit(X, y, **kw)

    no(ValueError, "needs pairs", "preference")
    no(ValueError, "needs advantage", "policy")
    no(ValueError, "not an argument", "regression", pairs=pairs)
    no(ValueError, "not an argument", "preference", pairs=pairs, advantage=y)
    no(TypeError, "numpy array", "preference", pairs=[[0, 1]])
    no(TypeError, "integers", "preference", pairs=pairs.astype(float))
    no(ValueError, r"shape \(P, 2\)", "preference", pairs=pairs[:, :1])
    no(ValueError, r"in \[0, 6\)", "preference", pairs=pairs + 3)
    no(ValueError, "ascend", "preference", pairs=pairs, segments=np.array([0, 4, 2, 3, 5]))
    no(ValueError, r"in \[0, 2\)", "preference", pairs=pairs, segments=np.array([0, 4, 6]))
    no(ValueError, "pair_weight", "preference", pairs=pairs, pair_weight=y)
    no(ValueError, "advantage must have shape", "policy", advantage=y[:3])
    no(ValueError, "one entry per row", "policy", advantage=y, reference=y[:2])
    no(ValueError, "eval set", "preference", pairs=pairs, X_eval=X, y_eval=y, eval_every_n_trees=1)
    no(ValueError, "at least 2 classes", "policy", advantage=y)
    with pytest.raises(ValueError, match="log_prob"):
        WarpGBM().log_prob(X, y)

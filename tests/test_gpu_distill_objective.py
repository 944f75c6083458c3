"""The objective "distill", the policy's entropy term, and a forest's alternatives."""
import numpy as np
import pytest
import torch

from conftest import print_case
from test_gpu_loss_objectives import KW, policy_data, scores_of
from test_lists import F64, distill64, lists_for
from test_losses import log_softmax64, policy64


def distill_data(n, K, seed, rest, coef, tau):
    """(constructor arguments, fit arguments, float64 mean loss of scores)."""
    X, y, _, best, rng = policy_data(n, K, seed)
    names = np.array(["left", "middle", "right", "up", "down"])[:K]
    order = np.argsort(names)
    t = torch.from_numpy(np.eye(K, dtype=np.float32)[best] * 2.0)
    cls, logits, ln = lists_for(t, 3, seed, tau)
    # (columns of classes_, the sorted names)
    back = np.argsort(order)
    cls_cols = np.where((cls >= 0) & (cls < K), back[np.clip(cls, 0, K - 1)], cls.numpy())
    w = ((rng.random(n) < 0.9) * (0.5 + rng.random(n))).astype(np.float32)

    def loss(scores):
        s = torch.from_numpy(np.asarray(scores, np.float64))
        c = torch.from_numpy(cls_cols.astype(np.int32))
        d = distill64(s, c, torch.nan_to_num(logits), ln if rest else None,
                      torch.from_numpy((w * np.float32(1 - coef))), tau)
        lp = log_softmax64(s)[torch.arange(n), torch.from_numpy(back[y])]
        total = d["loss"].sum() - coef * (torch.from_numpy(w).to(F64) * lp).sum()
        return total.item() / w.astype(np.float64).sum()

    fit = dict(X=X, y=names[y], teacher_classes=cls_cols.astype(np.int64),
               teacher_logits=logits.numpy(), sample_weight=w)
    if rest:
        fit["teacher_log_norm"] = ln.numpy()
    return dict(objective="distill", temperature=tau, label_coef=coef), fit, loss


WAYS = [(False, 0.0, 1.0), (True, 0.0, 2.0), (True, 0.25, 1.5)]


@pytest.mark.gpu
@pytest.mark.parametrize("rest,coef,tau", WAYS)
def test_training_loss_is_that_of_the_predictions(gpu, rest, coef, tau):
    from warpgbm_amd import WarpGBM

    print_case("distill fit", rest, coef, tau)
    new, given, loss = distill_data(3000, 5, 5, rest, coef, tau)
    full = WarpGBM(n_estimators=5, **new, **KW).fit(**given)
    assert len(full.training_loss) == 5
    for rounds in (1, 3):
        m = WarpGBM(n_estimators=rounds, **new, **KW).fit(**given)
        # float32 sums of some thousand losses of about one
        assert full.training_loss[rounds] == pytest.approx(loss(scores_of(m, given["X"])), abs=2e-5)
        assert m.forest == full.forest[:rounds]


@pytest.mark.gpu
@pytest.mark.parametrize("rest,coef,tau", WAYS)
def test_leaves_are_mean_negative_gradients(gpu, rest, coef, tau):
    """The first trees' leaves against differences of the float64 loss at the start."""
    from warpgbm_amd import WarpGBM

    new, given, loss = distill_data(1500, 3, 8, rest, coef, tau)
    m = WarpGBM(n_estimators=1, **new, **KW).fit(**given)
    n, K = given["X"].shape[0], m.num_classes
    codes = m.bin_inference_data(given["X"]).rm.cpu().numpy()
    total = given["sample_weight"].astype(np.float64).sum()

    def leaves(node, rows):
        if "leaf_value" in node:
            return [(node["leaf_value"], rows)]
        left = codes[rows, int(node["feature"])] <= int(node["bin"])
        return leaves(node["left"], rows[left]) + leaves(node["right"], rows[~left])

    for k, tree in enumerate(m.forest[0]):
        for value, rows in leaves(tree, np.arange(n)):
            h = 1e-4
            up, down = np.zeros((n, K)), np.zeros((n, K))
            up[rows, k], down[rows, k] = h, -h
            slope = total * (loss(up) - loss(down)) / (2 * h)
            assert value == pytest.approx(-slope / len(rows), rel=2e-4, abs=2e-5)


@pytest.mark.gpu
def test_warm_start_persistence_and_alternatives(gpu, tmp_path):
    from warpgbm_amd import WarpGBM

    new, given, _ = distill_data(2500, 5, 9, True, 0.3, 2.0)
    full = WarpGBM(n_estimators=6, **new, **KW).fit(**given)
    m = WarpGBM(n_estimators=4, warm_start=True, **new, **KW).fit(**given)
    m.n_estimators = 6
    m.fit(**given)
    assert m.forest == full.forest and m.training_loss == full.training_loss
    path = str(tmp_path / "m.pkl")
    full.save_model(path)
    back = WarpGBM().load_model(path)
    assert (back.temperature, back.label_coef, back.entropy_coef) == (2.0, 0.3, 0.0)
    X = given["X"]
    r = back.alternatives(X, 3, y=given["y"])
    p = full.predict_proba(X).astype(np.float64)
    at = np.argsort(-p, axis=1, kind="stable")[:, :3]
    best = np.take_along_axis(p, at, 1)
    # (probabilities in float32 may tie where scores differ)
    assert np.allclose(np.exp(r.log_prob), best, rtol=1e-5)
    assert np.allclose(np.take_along_axis(p, r.classes.astype(np.int64), 1), best, rtol=1e-6)
    assert np.allclose(r.entropy, -(p * np.log(p)).sum(1), rtol=1e-5, atol=1e-6)
    assert np.allclose(r.label_log_prob, back.log_prob(X, given["y"]), rtol=1e-6, atol=1e-6)
    # more alternatives than classes: all of them; its own lists teach it nothing
    all_of = back.alternatives(X, 20, temperature=2.0)
    assert all_of.classes.shape == (len(X), 5) and all_of.label_log_prob is None
    own = WarpGBM(n_estimators=8, warm_start=True, objective="distill", temperature=2.0, **KW)
    own.fit(X, given["y"], teacher_classes=all_of.classes,
            teacher_logits=all_of.log_prob * 2.0,
            teacher_log_norm=np.zeros(len(X), np.float32))
    with pytest.raises(ValueError, match="alternatives"):
        WarpGBM(objective="regression").alternatives(X)


@pytest.mark.gpu
@pytest.mark.parametrize("weighted", [False, True])
def test_policy_with_an_entropy_term(gpu, weighted):
    from warpgbm_amd import WarpGBM

    n, K = 3000, 4
    X, y, adv, best, rng = policy_data(n, K, 3)
    w = (rng.random(n) < 0.9).astype(np.float32) if weighted else None
    full = WarpGBM(objective="policy", n_estimators=4, entropy_coef=0.2, **KW)
    full.fit(X, y, advantage=adv, sample_weight=w)
    m = WarpGBM(objective="policy", n_estimators=3, entropy_coef=0.2, **KW)
    m.fit(X, y, advantage=adv, sample_weight=w)
    assert m.forest == full.forest[:3]
    s = torch.from_numpy(scores_of(m, X))
    ww = torch.ones(n) if w is None else torch.from_numpy(w)
    rows = policy64(s, torch.from_numpy(y), torch.full((n,), -np.log(K)), torch.from_numpy(adv),
                    ww, None, None, (0.2, 0.2), 0.0)[0]
    L = log_softmax64(s)
    H = -(L.exp() * L).sum(1)
    want = (rows - 0.2 * ww.to(F64) * H).sum().item() / ww.to(F64).sum().item()
    assert full.training_loss[3] == pytest.approx(want, abs=2e-5)
    plain = WarpGBM(objective="policy", n_estimators=1, **KW).fit(X, y, advantage=adv,
                                                                  sample_weight=w)
    # policies start uniform: the entropy there is log K
    assert plain.training_loss[0] - full.training_loss[0] == pytest.approx(0.2 * np.log(K), rel=1e-5)


@pytest.mark.parametrize("kw,exc", [
    ({"entropy_coef": -0.1}, ValueError), ({"entropy_coef": "1"}, TypeError),
    ({"temperature": 0.0}, ValueError), ({"temperature": None}, TypeError),
    ({"label_coef": 1.5}, ValueError), ({"label_coef": float("nan")}, ValueError),
])
def test_parameters(kw, exc):
    from warpgbm_amd import WarpGBM

    with pytest.raises(exc):
        WarpGBM(objective="distill", **kw)


def test_fit_argument_refusals():
    from warpgbm_amd import WarpGBM

    X, y = np.zeros((6, 2), np.float32), np.zeros(6, np.float32)
    c, t = np.zeros((6, 2), np.int64), np.zeros((6, 2), np.float32)

    def no(exc, text, objective="distill", **kw):
        with pytest.raises(exc, match=text):
            WarpGBM(objective=objective).fit(X, y, **kw)

    no(ValueError, "needs teacher_classes", teacher_logits=t)
    no(ValueError, "needs teacher_logits", teacher_classes=c)
    no(TypeError, "integers", teacher_classes=t, teacher_logits=t)
    no(ValueError, "teacher_classes must have shape", teacher_classes=c[:3], teacher_logits=t)
    no(ValueError, "teacher_classes must have shape", teacher_classes=c[:, 0], teacher_logits=t)
    no(ValueError, "teacher_classes must have shape", teacher_classes=np.zeros((6, 65), np.int64),
       teacher_logits=np.zeros((6, 65), np.float32))
    no(ValueError, "teacher_logits must have shape", teacher_classes=c, teacher_logits=t[:, :1])
    no(ValueError, "teacher_log_norm must have shape", teacher_classes=c, teacher_logits=t,
       teacher_log_norm=y[:2])
    no(ValueError, "not an argument", teacher_classes=c, teacher_logits=t, advantage=y)
    no(ValueError, "not an argument", "policy", advantage=y, teacher_classes=c)
    no(ValueError, "eval set", teacher_classes=c, teacher_logits=t, X_eval=X, y_eval=y,
       eval_every_n_trees=1)


@pytest.mark.gpu
def test_a_teacher_of_more_classes_is_not_taken_in_silence(gpu):
    """Numbers past the student's columns name none of its classes: they are left out, and
    the fit says so."""
    import warnings

    from warpgbm_amd import WarpGBM

    new, given, _ = distill_data(600, 4, 11, True, 0.0, 1.0)
    tc = given["teacher_classes"]
    inside = dict(given, teacher_classes=np.where(tc < 4, tc, -1))
    beyond = dict(given, teacher_classes=tc.copy())
    beyond["teacher_classes"][7, 0] = 4
    inside["teacher_classes"][7, 0] = -1
    fits = []
    with warnings.catch_warnings():
        warnings.simplefilter("error", UserWarning)
        fits.append(WarpGBM(n_estimators=2, **new, **KW).fit(**inside))
    with pytest.warns(UserWarning, match="past the last of the 4 classes"):
        fits.append(WarpGBM(n_estimators=2, **new, **KW).fit(**beyond))
    assert fits[0].forest == fits[1].forest
    assert fits[0].training_loss == fits[1].training_loss


@pytest.mark.gpu
def test_a_forest_s_own_lists_teach_it_nothing(gpu):
    """A forest that goes on from where its lists were taken: losses and leaves of the
    next round are roundings."""
    from warpgbm_amd import WarpGBM

    tau, K = 2.0, 5
    new, given, _ = distill_data(2500, K, 9, True, 0.0, tau)
    m = WarpGBM(n_estimators=4, warm_start=True, **new, **KW).fit(**given)
    X = given["X"]
    lists = m.alternatives(X, K, temperature=tau)
    assert (lists.classes >= 0).all()
    s = scores_of(m, X)
    m.n_estimators = 5
    m.fit(X, given["y"], teacher_classes=lists.classes, teacher_logits=lists.log_prob * tau,
          teacher_log_norm=np.zeros(len(X), np.float32))
    # log p - log q of a class: the lists' rounding to float32 and, of the student, the
    # scores' sums over four rounds and a few more steps; a gradient is at most T of it, a
    # loss T^2 of its square
    far = np.abs(s).max()
    x = 2.0 ** -24 * (2 * np.abs(lists.log_prob).max() + 16 * far + 64)
    assert len(m.training_loss) == 5
    assert m.training_loss[3] > 1e-3 and 0 <= m.training_loss[4] <= (tau * x) ** 2

    def leaves(node):
        if "leaf_value" in node:
            return [abs(node["leaf_value"])]
        return leaves(node["left"]) + leaves(node["right"])

    before = max(max(leaves(t)) for t in m.forest[3])
    assert before > 1e-3
    for tree in m.forest[4]:
        assert max(leaves(tree)) <= tau * x

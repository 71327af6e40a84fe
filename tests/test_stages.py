"""Staged prediction and joint refitting of leaf values: the CPU path against predict() and the formulas, the GPU path
(lookup, recurrence and their gradients) against the CPU path.

Tolerances: a staged score is an fp64 sum of at most 60 leaf values of magnitude below 10, in another order than predict()
takes: 60 * 60 * 10 * 2^-53 < 1e-11 absolute; link functions do not amplify that here (slopes up to 10).
"""
import numpy as np
import pytest

import lightgbm_amd as lgb
from lightgbm_amd import LightGBMError

gpu = pytest.mark.gpu
TOL = 1e-10


def make(kind, rows=700, seed=0, **params):
    rng = np.random.default_rng(seed)
    X = rng.normal(size=(rows, 6))
    X[rng.random(X.shape) < 0.05] = np.nan
    X[:, 5] = rng.integers(0, 7, rows)
    signal = np.nan_to_num(X[:, 0]) + np.sin(2 * np.nan_to_num(X[:, 1])) + (X[:, 5] > 3)
    p = {"objective": kind, "num_leaves": 9, "learning_rate": 0.2, "verbose": -1, "device_type": "cpu", "min_data_in_leaf": 5, **params}
    if kind == "binary":
        y = (signal + rng.normal(size=rows) > 0.5).astype(float)
    elif kind == "multiclass":
        y = np.clip(np.floor(signal + 1), 0, 2)
        p["num_class"] = 3
    elif kind in ("poisson", "gamma"):
        y = np.exp(0.3 * signal) + 0.01
    else:
        y = signal + 0.1 * rng.normal(size=rows)
    w = rng.random(rows) + 0.5
    booster = lgb.train(p, lgb.Dataset(X, label=y, params=p, categorical_feature=[5] if kind == "regression" else "auto"), num_boost_round=20)
    return booster, X, y, w


MODELS = {"regression": {}, "binary": {}, "multiclass": {}, "poisson": {}, "cross_entropy": {}, "gamma": {}, "multiclassova": {"num_class": 3},
          "forest": {"boosting": "rf", "bagging_fraction": 0.6, "bagging_freq": 1, "feature_fraction": 0.8}, "dart": {"boosting": "dart"}}


def model(name):
    kind = {"forest": "regression", "dart": "binary", "multiclassova": "multiclass", "cross_entropy": "binary"}.get(name, name)
    params = dict(MODELS[name])
    if name in ("multiclassova", "cross_entropy"):
        params["objective"] = name
    return make(kind, **params)


def check_stages(booster, X, got, raw, start=0):
    n = got.shape[0]
    assert n == booster.current_iteration() - start
    for k in (0, 1, 6, n - 1):
        want = booster.predict(X, start_iteration=start, num_iteration=k + 1, raw_score=raw, device="cpu")
        assert got[k].shape == want.shape
        assert np.abs(got[k] - want).max() <= TOL


@pytest.mark.parametrize("name", MODELS)
@pytest.mark.parametrize("raw", [False, True])
def test_staged_predictions_are_the_predictions_of_every_stage(name, raw):
    booster, X, _, _ = model(name)
    check_stages(booster, X, booster.staged_predict(X, raw_score=raw, device="cpu"), raw)
    check_stages(booster, X[:1], booster.staged_predict(X[:1], start_iteration=3, raw_score=raw, device="cpu"), raw, start=3)
    few = booster.staged_predict(X, num_iteration=4, raw_score=raw, device="cpu")
    assert few.shape[0] == 4 and np.array_equal(few, booster.staged_predict(X, raw_score=raw, device="cpu")[:4])


def test_staged_prediction_follows_best_iteration_and_empty_matrices():
    booster, X, _, _ = make("regression")
    booster.best_iteration = 5
    assert booster.staged_predict(X).shape == (5, len(X))
    assert booster.staged_predict(X, num_iteration=-1).shape == (20, len(X))
    assert booster.staged_predict(X[:0], num_iteration=-1).shape == (20, 0)
    assert booster.staged_predict(X, start_iteration=20, num_iteration=3).shape == (0, len(X))
    with pytest.raises(TypeError):
        booster.staged_predict(lgb.Dataset(X))
    with pytest.raises(LightGBMError):
        booster.staged_predict(X, device="tpu")


def test_blocks_of_rows_change_nothing(monkeypatch):
    from lightgbm_amd import stages
    booster, X, y, w = make("multiclass")
    whole = booster.staged_predict(X, device="cpu")
    refitted = booster.refit_stages(X, y, w, num_steps=3, device="cpu")
    monkeypatch.setattr(stages, "_BLOCK_VALUES", 20 * 3 * 100)
    assert np.array_equal(booster.staged_predict(X, device="cpu"), whole)
    again = booster.refit_stages(X, y, w, num_steps=3, device="cpu")
    # sums of the blocks' gradients instead of one sum
    assert np.abs(again.predict(X, raw_score=True) - refitted.predict(X, raw_score=True)).max() <= TOL


def loss(kind, raw, y, w):
    """Weighted mean loss of one stage."""
    if kind == "regression":
        l = 0.5 * (raw - y) ** 2
    elif kind == "binary":
        l = np.logaddexp(0, raw) - y * raw
    else:
        top = raw.max(1)
        l = top + np.log(np.exp(raw - top[:, None]).sum(1)) - raw[np.arange(len(y)), y.astype(int)]
    return (l * w).sum() / w.sum()


@pytest.mark.parametrize("kind", ["regression", "binary", "multiclass"])
@pytest.mark.parametrize("stages", ["all", "last"])
def test_refitted_leaves_step_along_the_gradient(kind, stages):
    """A step moves every leaf by -rate * gradient / bound: the gradient against differences of the loss."""
    booster, X, y, w = make(kind, rows=200)
    rate = 1e-3
    after = booster.refit_stages(X, y, w, num_steps=1, learning_rate=rate, stages=stages, device="cpu")
    n, K = booster.current_iteration(), booster.num_model_per_iteration()
    leaves = booster.predict(X, pred_leaf=True)

    def total(b):
        raw = b.staged_predict(X, raw_score=True, device="cpu")
        return np.mean([loss(kind, r, y, w) for r in raw]) if stages == "all" else loss(kind, raw[-1], y, w)
    q = {"regression": 1.0, "binary": 0.25, "multiclass": 0.5}[kind]
    old, new = booster._tree_arrays(), after._tree_arrays()
    for tree in (0, 5 * K + K - 1, n * K - 1):
        k = np.arange(tree // K + 1, n + 1)
        per_row = q * (np.mean(np.where(np.arange(1, n + 1) > tree // K, np.arange(1, n + 1), 0)) if stages == "all" else n)
        for leaf in (0, len(old[tree]["leaf_value"]) - 1):
            bound = (w / w.sum())[leaves[:, tree] == leaf].sum() * per_row
            step = 1e-4
            value = old[tree]["leaf_value"][leaf]
            booster.set_leaf_output(tree, leaf, value + step)
            up = total(booster)
            booster.set_leaf_output(tree, leaf, value - step)
            down = total(booster)
            booster.set_leaf_output(tree, leaf, value)
            moved = new[tree]["leaf_value"][leaf] - value
            # differences: third derivatives below 1 times step^2, and roundings of a loss near 1 over 2 step
            assert abs(moved - -rate * (up - down) / (2 * step) / bound) <= rate / bound * (step ** 2 + 1e-15 / step)


def test_refit_leaves_structures_and_unreached_leaves_alone():
    booster, X, y, w = make("regression")
    some = X[:40]
    after = booster.refit_stages(some, y[:40], num_steps=5, device="cpu")
    assert np.array_equal(after.predict(X, pred_leaf=True), booster.predict(X, pred_leaf=True))
    leaves = booster.predict(some, pred_leaf=True)
    changed = 0
    for tree, (a, b) in enumerate(zip(booster._tree_arrays(), after._tree_arrays())):
        for leaf, (p, q) in enumerate(zip(a["leaf_value"], b["leaf_value"])):
            if leaf not in leaves[:, tree]:
                assert p == q
            changed += p != q
    assert changed
    same = booster.refit_stages(X, y, num_steps=0)
    assert np.array_equal(same.predict(X), booster.predict(X))


def test_refit_stages_refusals():
    booster, X, y, w = make("regression", rows=200)
    forest, *_ = model("forest")
    poisson, *_ = model("poisson")
    multi, Xm, ym, _ = make("multiclass", rows=200)
    for b, kw in ((forest, {}), (poisson, {}), (booster, {"stages": "some"}), (booster, {"num_steps": -1}), (booster, {"num_steps": 1.5}),
                  (booster, {"learning_rate": 0.0}), (booster, {"learning_rate": 2.5}), (booster, {"lambda_l2": -1.0}), (booster, {"device": "tpu"}),
                  (booster, {"weight": np.ones(3)}), (booster, {"weight": -np.ones(200)}), (booster, {"weight": np.zeros(200)})):
        with pytest.raises(LightGBMError):
            b.refit_stages(X[:200], y[:200], **kw)
    with pytest.raises(LightGBMError):
        booster.refit_stages(X, y[:-1])
    with pytest.raises(LightGBMError):
        multi.refit_stages(Xm, ym + 0.5)
    with pytest.raises(LightGBMError):
        multi.refit_stages(Xm, ym + 3)


@pytest.mark.parametrize("kind", ["regression", "binary", "multiclass"])
@pytest.mark.parametrize("odd", [np.nan, np.inf, -np.inf])
def test_refit_stages_refuses_what_is_not_finite(kind, odd):
    booster, X, y, w = make(kind, rows=200)
    label, weight = y.copy(), w.copy()
    label[3], weight[3] = odd, odd
    for kw in ({"label": label}, {"label": label, "num_steps": 0}, {"label": label, "weight": np.where(np.arange(200) == 3, 0.0, 1.0)},
               {"label": y, "weight": weight}, {"label": y, "weight": np.full(200, 1e308)}, {"label": y, "lambda_l2": odd}):
        with pytest.raises(LightGBMError):
            booster.refit_stages(X, device="cpu", **kw)


def test_the_gpu_is_refused_where_there_is_none():
    from lightgbm_amd import _lib
    if _lib.load()[1]:
        pytest.skip("a GPU is visible")
    booster, X, y, _ = make("regression", rows=200)
    with pytest.raises(LightGBMError):
        booster.staged_predict(X, device="gpu")
    with pytest.raises(LightGBMError):
        booster.refit_stages(X, y, device="gpu")


@gpu
@pytest.mark.parametrize("name", MODELS)
def test_gpu_stages_are_the_cpu_stages(name):
    booster, X, _, _ = model(name)
    for raw in (False, True):
        for rows in (1, 65, len(X)):
            a, b = booster.staged_predict(X[:rows], raw_score=raw, device="gpu"), booster.staged_predict(X[:rows], raw_score=raw, device="cpu")
            assert a.shape == b.shape and np.abs(a - b).max() <= TOL
    check_stages(booster, X, booster.staged_predict(X, start_iteration=2, device="gpu"), False, start=2)


@gpu
@pytest.mark.parametrize("kind", ["regression", "binary", "multiclass"])
@pytest.mark.parametrize("stages", ["all", "last"])
def test_gpu_refit_is_the_cpu_refit(kind, stages, monkeypatch):
    from lightgbm_amd import stages as module
    booster, X, y, w = make(kind, rows=3000)
    kw = dict(weight=w, num_steps=6, learning_rate=1.5, lambda_l2=1e-3, stages=stages)
    a = booster.refit_stages(X, y, device="gpu", **kw)
    b = booster.refit_stages(X, y, device="cpu", **kw)
    # steps contract differences: six steps of gradients that differ by the order of sums of 60000 fp64 terms
    for p, q, o in zip(a._tree_arrays(), b._tree_arrays(), booster._tree_arrays()):
        assert np.abs(p["leaf_value"] - q["leaf_value"]).max() <= 1e-8
    assert np.abs(a.predict(X, raw_score=True) - booster.predict(X, raw_score=True)).max() > 1e-4
    monkeypatch.setattr(module, "_BLOCK_VALUES", 20 * 3 * 6 * 500)
    c = booster.refit_stages(X, y, device="gpu", **kw)
    for p, q in zip(a._tree_arrays(), c._tree_arrays()):
        assert np.abs(p["leaf_value"] - q["leaf_value"]).max() <= 1e-8

"""Targets, bias and refusals of the losses distill, policy and preference (no GPU needed)."""
import numpy as np
import pytest


def test_learners(pkg):
    c = pkg.EvoTreeClassifier(loss="distill", tau=2.0)
    assert c.metric == "distill" and pkg.EvoTreeClassifier(loss="policy").metric == "policy"
    assert pkg.EvoTreeRegressor(loss="preference").metric == "preference"
    for bad in (dict(loss="distill", tau=0.0), dict(loss="distill", tail=True, tau=2.0), dict(loss="policy", clip=(1.5, 0.2)), dict(loss="policy", clip=(0.2,)),
                dict(loss="policy", beta=-1.0), dict(loss="distill", metric="mlogloss"), dict(loss="mlogloss", metric="distill"), dict(loss="distill", nclasses=40),
                dict(loss="preference")):
        with pytest.raises(ValueError):
            pkg.EvoTreeClassifier(**bad)
    for bad in (dict(loss="preference", smooth=1.5), dict(loss="preference", metric="mse"), dict(loss="distill")):
        with pytest.raises(ValueError):
            pkg.EvoTreeRegressor(**bad)


def test_pack_distill(pkg):
    from evotrees_b200.fit import init_objective, pack_objective
    p = pkg.EvoTreeClassifier(loss="distill")
    ids, t = np.array([[3, 1], [2, 0], [1, 4]]), np.array([[0.5, -1.0], [2.0, 9.0], [0.0, 0.0]])
    K, y, ycols = pack_objective(p, (ids, t), 3)
    assert (K, ycols, y.dtype, y.shape) == (4, 4, np.uint32, (3, 4))
    assert np.array_equal(y[:, :2], ids) and np.array_equal(y[:, 2:].view(np.float32), t.astype(np.float32))
    assert pack_objective(pkg.EvoTreeClassifier(loss="distill", nclasses=7), (ids, t), 3)[0] == 7
    K, y, ycols, mu, levels, off = init_objective(p, (ids, t), None, 3)
    q0 = np.exp([0.5, -1.0]) / np.exp([0.5, -1.0]).sum()
    want = np.array([q0[1] + 0.5, 1.0, q0[0], 0.5]) / 3
    np.testing.assert_allclose(np.exp(mu) / np.exp(mu).sum(), want, rtol=1e-5)
    assert mu.max() == 0 and levels.tolist() == [1, 2, 3, 4]
    # a tail is shared by all classes
    tail = pkg.EvoTreeClassifier(loss="distill", tail=True)
    mu = init_objective(tail, (np.array([[1], [2]]), np.log(np.array([[0.5], [0.8]])), ), None, 2)[3]
    np.testing.assert_allclose(np.exp(mu) / np.exp(mu).sum(), np.array([0.5 + 0.35, 0.8 + 0.35]) / 2, rtol=1e-5)
    bad = [(ids, t[:2]), (ids.astype(float), t), (ids[:2], t[:2]), (ids - 1, t), (ids,), ids, (ids[:, 0], t[:, 0]), (ids * 20, t), (np.ones((3, 2), int), t),
           (ids, np.where(t > 1, np.nan, t)), (np.ones((3, 1025), int) * 2, np.ones((3, 1025)))]
    for y in bad:
        with pytest.raises(ValueError):
            pack_objective(p, y, 3)
    with pytest.raises(ValueError):
        pack_objective(p, (ids, t), 3, K=3)


def test_pack_policy_and_preference(pkg):
    from evotrees_b200.fit import init_objective, objective_parameters, pack_objective
    p = pkg.EvoTreeClassifier(loss="policy", beta=0.0, tau=0.5, clip=(0.1, 0.3))
    a, old, adv = np.array([1, 0, 3]), np.array([-1.0, -2.0, -3.0]), np.array([0.5, 1.5, -2.5])
    K, y, ycols = pack_objective(p, (a, old, adv), 3)
    assert (K, ycols) == (3, 4) and np.array_equal(y[:, 0], a) and np.array_equal(y[:, 2].view(np.float32), adv.astype(np.float32)) and (y[:, 3] == 0).all()
    assert (init_objective(p, (a, old, adv), None, 3)[3] == 0).all() and objective_parameters(p) == (0.5, 0.1, 0.3, 0.0)
    kl = pkg.EvoTreeClassifier(loss="policy", beta=0.2)
    assert np.array_equal(pack_objective(kl, (a, old, adv, old), 3)[1][:, 3].view(np.float32), old.astype(np.float32))
    for cfg, y in ((kl, (a, old, adv)), (p, (a, old)), (p, (a[:, None], old, adv)), (p, (a, old[:2], adv)), (p, (np.array([1, 1, 1]), old, adv))):
        with pytest.raises(ValueError):
            pack_objective(cfg, y, 3)
    r = pkg.EvoTreeRegressor(loss="preference")
    assert pack_objective(r, None, 4)[1].tolist() == [0.0] * 4 and pack_objective(r, [1, 2], 2)[2] == 1
    assert objective_parameters(r) == (0.1, 0.0) and objective_parameters(pkg.EvoTreeRegressor()) is None
    for y, n in ((None, 3), ([1, 2, 3], 4), ([1, np.nan], 2)):
        with pytest.raises(ValueError):
            pack_objective(r, y, n)


def test_refusals_before_any_device(pkg):
    x = np.zeros((4, 2), np.float32)
    with pytest.raises(ValueError, match="y_train"):
        pkg.fit(pkg.EvoTreeRegressor(nrounds=1), x_train=x)
    class Comm:
        rank = 0
    with pytest.raises(ValueError, match="one GPU"):
        pkg.fit(pkg.EvoTreeRegressor(loss="preference", nrounds=1), x_train=x, comm=Comm())

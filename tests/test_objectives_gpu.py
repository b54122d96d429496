"""The losses distill, policy and preference as losses of `fit`: gradients and hessians of every round against the definitions in 64 bits at the
predictions that the handle holds, metrics, inference, and the three one after the other."""
import numpy as np
import pytest
import torch

from tests import losses_ref as R

pytestmark = pytest.mark.gpu
F8 = torch.float64


def table(rng, n, f=6):
    return rng.normal(size=(n, f)).astype(np.float32)


def distill_target(rng, x, K, T, tail=False):
    t = x @ rng.normal(size=(x.shape[1], K)) * 0.7
    if tail:
        t = t - np.log(np.exp(t).sum(1, keepdims=True))
    ids = np.argsort(-t, axis=1, kind="stable")[:, :T]
    vals = np.take_along_axis(t, ids, 1).astype(np.float32)
    ids = ids + 1
    ids[rng.random(ids.shape) < 0.1] = 0
    return ids, vals


def policy_target(rng, n, K, ref):
    a = rng.integers(0, K + 1, n)
    old = np.log(0.5 + rng.random(n)) - np.log(K)
    out = (a, old.astype(np.float32), rng.normal(size=n).astype(np.float32))
    return out + ((old + 0.2).astype(np.float32),) if ref else out


def check_grads(params, cache, y, w, K, first=0):
    """Gradient records of the handle against the formulas at its predictions (the ones that the next tree is grown on)."""
    rec, z = torch.from_numpy(cache.grads()).to(F8), torch.from_numpy(cache.pred())
    wt = None if w is None else torch.from_numpy(w)
    if params.loss == "preference":
        s = z[:, 0].to(F8) - torch.from_numpy(np.zeros(z.shape[0]) if y is None else np.asarray(y)).to(F8)
        m = params.beta * (s[0::2] - s[1::2])
        wp = torch.ones_like(m) if wt is None else wt[0::2].to(F8)
        g = params.beta * wp * (params.smooth * torch.sigmoid(m) - (1 - params.smooth) * torch.sigmoid(-m))
        h = params.beta ** 2 * wp * torch.sigmoid(m) * torch.sigmoid(-m)
        # differences of scores are off by a step of them, sigmoids by 32 steps
        tol = 64 * R.U * (1 + params.beta * z[:, 0].abs().max().to(F8)) * params.beta
        R.close(rec[:, 0], torch.stack([g, -g], 1).reshape(-1), tol, "grad")
        R.close(rec[:, 1], torch.stack([h, h], 1).reshape(-1), tol * max(params.beta, 1.0), "hess")
        return
    t = [torch.from_numpy(np.asarray(v)) for v in y]
    if params.loss == "distill":
        loss, grad, hess, scale = R.distill(z, t[0], t[1], wt, params.tau, params.tail)
        rel = R.part(z, params.tau) + R.slots_part(t[1], params.tau)
        size = params.tau * (1.0 + grad.abs())
        if params.tail:       # 1 - sum q is off by `rel`, whatever probability of the student stands against it
            size = size + params.tau / torch.softmax(z.to(F8), 1).amin(1, keepdim=True).clamp(min=1e-6) * torch.softmax(z.to(F8), 1)
    else:
        ref = t[3] if params.beta > 0 else None
        loss, logp, grad, hess, scale = R.policy(z, t[0], t[1], t[2], ref, wt, params.tau, params.clip, params.beta)
        rel = 4 * (R.part(z, params.tau) + 4 * R.U * logp.abs())
        size = (scale / params.tau)[:, None] + torch.zeros_like(grad)
        # rows on the border of the clip: 32 bits decide for them
        r = torch.exp(logp - t[1].to(F8))
        edge = ((r - 1 - params.clip[1]).abs() < 1e-5) | ((r - 1 + params.clip[0]).abs() < 1e-5)
        rec[:, :K] = torch.where(edge[:, None], grad, rec[:, :K])
    wmax = 1.0 if wt is None else wt.to(F8)[:, None]
    R.close(rec[:, :K], grad, R.rounded(grad, torch.float32, 2 * rel[:, None], wmax * size), "grad")
    R.close(rec[:, K:2 * K], hess, R.rounded(hess, torch.float32, 2 * rel[:, None], wmax * 2 / min(1.0, params.tau ** 2)), "hess")


CASES = [("distill", dict(tau=2.0), 5, 3), ("distill", dict(tail=True), 4, 2), ("distill", {}, 2, 2), ("distill", {}, 12, 5), ("distill", dict(nclasses=32), 20, 20),
         ("policy", dict(beta=0.0), 3, 0), ("policy", dict(beta=0.1, tau=0.7), 18, 0), ("policy", dict(beta=0.05), 8, 0), ("preference", dict(beta=0.5), 1, 0),
         ("preference", dict(beta=1.0, smooth=0.1), 1, 0)]


def make(pkg, loss, kw, K, T, n, rng, **more):
    cls = pkg.EvoTreeRegressor if loss == "preference" else pkg.EvoTreeClassifier
    params = cls(loss=loss, **{**dict(nrounds=6, max_depth=4, nbins=32, eta=0.3, min_weight=1.0, seed=5), **kw, **more})
    x = table(rng, n)
    if loss == "distill":
        y = distill_target(rng, x, K, T, kw.get("tail", False))
    elif loss == "policy":
        y = policy_target(rng, n, K, kw.get("beta", 0.1) > 0)
    else:
        y = (rng.normal(size=n) * 0.3).astype(np.float32)
    return params, x, y, params.nclasses or K


@pytest.mark.parametrize("loss,kw,K,T", CASES)
@pytest.mark.parametrize("weights", [False, True])
def test_gradients_of_every_round(pkg, loss, kw, K, T, weights):
    rng = np.random.default_rng(K + T)
    n = 602
    params, x, y, Km = make(pkg, loss, kw, K, T, n, rng)
    w = np.repeat(0.5 + rng.random(n // 2), 2).astype(np.float32) if weights else None
    m, cache = pkg.init_core(params, x, y, w)
    js = np.arange(1, x.shape[1] + 1, dtype=np.uint32)
    for r in range(4):           # the first round launches directly, later ones replay a graph
        tree = pkg.grow_tree(cache, params, None, js, True)
        check_grads(params, cache, y, w, Km)
        m.trees.append(tree)
    assert any(t.split.any() for t in m.trees)
    # the model's predictions are those of the handle
    pred, out = cache.pred(), m(x)
    want = pred[:, 0] if loss == "preference" else np.exp(pred.astype(np.float64)) / np.exp(pred.astype(np.float64)).sum(1, keepdims=True)
    np.testing.assert_allclose(out, want, rtol=2e-5, atol=2e-6)
    cache.close()


@pytest.mark.parametrize("loss,kw,K,T", [CASES[0], CASES[1], CASES[6], CASES[9]])
def test_metric_and_samples(pkg, loss, kw, K, T):
    """Rows and columns sampled, evaluation data tracked: the metric of every round is the mean loss at the predictions tracked."""
    rng = np.random.default_rng(17)
    params, x, y, Km = make(pkg, loss, kw, K, T, 800, rng, rowsample=0.6, colsample=0.7)
    _, xe, ye, _ = make(pkg, loss, kw, K, T, 300, rng)
    we = np.repeat(0.5 + rng.random(150), 2).astype(np.float32)
    m, cache = pkg.init_core(params, x, y)
    cb = pkg.CallBack(params, m, cache, xe, ye, we)
    for r in range(4):
        value = cb.initial if r == 0 else cb.last()
        z = torch.from_numpy(cb.pred())
        if loss == "preference":
            s = z[:, 0].to(F8) - torch.from_numpy(ye).to(F8)
            mg, wp = params.beta * (s[0::2] - s[1::2]), torch.from_numpy(we[0::2]).to(F8)
            sp = torch.nn.functional.softplus
            want = float((wp * ((1 - params.smooth) * sp(-mg) + params.smooth * sp(mg))).sum() / wp.sum())
        else:
            t = [torch.from_numpy(np.asarray(v)) for v in ye]
            ws = torch.from_numpy(we)
            loss_rows = R.distill(z, t[0], t[1], ws, params.tau, params.tail)[0] if loss == "distill" else R.policy(z, *t[:3], t[3], ws, params.tau, params.clip, params.beta)[0]
            want = float(loss_rows.sum() / ws.to(F8).sum())
        assert abs(value - want) < 1e-4 * (1 + abs(want))
        pkg.grow_evotree(m, cache, params)
    cache.close()
    # `fit` with the same data logs the same way, and stops
    m = pkg.fit(params, x_train=x, y_train=y, x_eval=xe, y_eval=ye, w_eval=we)
    assert len(m.info["logger"]["metrics"]) == params.nrounds + 1 and all(np.isfinite(m.info["logger"]["metrics"]))


def test_hard_labels_are_mlogloss(pkg):
    """One slot a row is a class: gradients and hessians of mlogloss, to the rounding of two exponentials."""
    rng = np.random.default_rng(2)
    x = table(rng, 500)
    lab = rng.integers(1, 5, 500)
    p1 = pkg.EvoTreeClassifier(loss="distill", nrounds=1, max_depth=3, nbins=16, eta=0.3)
    p2 = pkg.EvoTreeClassifier(loss="mlogloss", nrounds=1, max_depth=3, nbins=16, eta=0.3)
    m1, c1 = pkg.init_core(p1, x, (lab[:, None], np.zeros((500, 1))))
    m2, c2 = pkg.init_core(p2, x, lab)
    np.testing.assert_allclose(m1.trees[0].pred, m2.trees[0].pred, rtol=1e-5, atol=1e-6)
    js = np.arange(1, 7, dtype=np.uint32)
    pkg.grow_tree(c1, p1, None, js, True), pkg.grow_tree(c2, p2, None, js, True)
    z1, z2 = c1.pred(), c2.pred()
    if np.abs(z1 - z2).max() < 1e-4:
        np.testing.assert_allclose(c1.grads(), c2.grads(), rtol=1e-3, atol=1e-4)
    c1.close(), c2.close()


def test_oblivious_trees_bagging_and_many_slots(pkg):
    rng = np.random.default_rng(9)
    for kw, K, T in ((dict(tree_type="oblivious"), 4, 3), (dict(bagging_size=2, rowsample=0.7), 4, 3)):
        params, x, y, Km = make(pkg, "distill", kw, K, T, 400, rng)
        m, cache = pkg.init_core(params, x, y)
        for _ in range(3):
            pkg.grow_evotree(m, cache, params)
        check_grads(params, cache, y, None, Km)
        cache.close()
    # more slots than classes, most of them empty or again
    params = pkg.EvoTreeClassifier(loss="distill", nrounds=2, max_depth=3, nbins=16, nclasses=6)
    x = table(rng, 200)
    ids = rng.integers(0, 7, (200, 50))
    vals = rng.normal(size=(200, 50)).astype(np.float32)
    m, cache = pkg.init_core(params, x, (ids, vals))
    pkg.grow_evotree(m, cache, params)
    check_grads(params, cache, (ids, vals), None, 6)
    cache.close()


def test_refusals(pkg):
    rng = np.random.default_rng(1)
    x = table(rng, 40)
    p = pkg.EvoTreeRegressor(loss="preference", nrounds=1)
    with pytest.raises(ValueError, match="pair"):
        pkg.fit(p, x_train=x, w_train=np.arange(1, 41).astype(np.float32))
    m, cache = pkg.init_core(p, x, None)
    with pytest.raises(ValueError, match="even"):
        pkg.CallBack(p, m, cache, x[:5], None)
    with pytest.raises(ValueError, match="pair"):
        pkg.CallBack(p, m, cache, x, None, np.arange(1, 41))
    cache.close()
    d = pkg.EvoTreeClassifier(loss="distill", nrounds=1, nclasses=3)
    ids, vals = np.ones((40, 2), int), np.zeros((40, 2))
    m, cache = pkg.init_core(d, x, (ids, vals))
    with pytest.raises(ValueError, match="slots"):
        pkg.CallBack(d, m, cache, x, (ids[:, :1], vals[:, :1]))
    cache.close()


def test_distilled_then_preferred_then_rewarded(pkg):
    """A student is distilled from a teacher's best classes, a score is learned from preferences between its choices, and the policy that starts at the
    student is moved by that score: every step takes what the one before it gave, and every gradient is the formula's."""
    rng = np.random.default_rng(4)
    n, K = 400, 4
    x = table(rng, n)
    ids, vals = distill_target(rng, x, K, 3)
    student = pkg.fit(pkg.EvoTreeClassifier(loss="distill", nclasses=K, nrounds=8, max_depth=4, nbins=32, eta=0.3), x_train=x, y_train=(ids, vals))
    prob = student(x)
    assert prob.shape == (n, K) and np.allclose(prob.sum(1), 1.0, atol=1e-5)
    # preferences between two choices for the same row: features and the choice
    good, other = prob.argmax(1), (prob.argmax(1) + rng.integers(1, K, n)) % K
    pairs = np.empty((2 * n, x.shape[1] + 1), np.float32)
    pairs[0::2], pairs[1::2] = np.column_stack([x, good]), np.column_stack([x, other])
    ref = np.log(np.maximum(np.stack([prob[np.arange(n), good], prob[np.arange(n), other]], 1).reshape(-1), 1e-6)).astype(np.float32)
    cfg = pkg.EvoTreeRegressor(loss="preference", nrounds=5, max_depth=4, nbins=32, eta=0.3, beta=0.5)
    score, cache = pkg.fit(cfg, x_train=pairs, y_train=ref, return_cache=True)
    check_grads(cfg, cache, ref, None, 1)
    cache.close()
    # what was sampled from the student, scored; the policy begins at the student's probabilities
    action = np.array([rng.choice(K, p=p / p.sum()) for p in prob.astype(np.float64)])
    reward = score(np.column_stack([x, action]).astype(np.float32))
    adv = ((reward - reward.mean()) / (reward.std() + 1e-6)).astype(np.float32)
    logp = np.log(prob[np.arange(n), action]).astype(np.float32)
    y = (action + 1, logp, adv, logp)
    cfg = pkg.EvoTreeClassifier(loss="policy", nclasses=K, nrounds=5, max_depth=4, nbins=32, eta=0.3, beta=0.1)
    policy, cache = pkg.fit(cfg, x_train=x, y_train=y, offset_train=prob, return_cache=True)
    check_grads(cfg, cache, y, None, K)
    # the same from the device: the predictions of the handle, the operator on them
    z = torch.from_numpy(cache.pred()).cuda()
    out = pkg.policy_grads(z, torch.from_numpy((action + 1).astype(np.int32)).cuda(), torch.from_numpy(logp).cuda(), torch.from_numpy(adv).cuda(),
                           ref_logp=torch.from_numpy(logp).cuda(), beta=0.1, hess=True)
    rec = cache.grads()
    assert np.array_equal(out[2].cpu().numpy(), rec[:, :K]) and np.array_equal(out[3].cpu().numpy(), rec[:, K:2 * K])
    cache.close()

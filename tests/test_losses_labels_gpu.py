"""Codes of rows that do not count, and more slots than classes."""
import numpy as np
import pytest
import torch

from tests import losses_ref as R
from tests.test_losses_gpu import F8, check_distill, log_probs, logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K", [5, 20, 300, 33000, 300001])
def test_preference_labels_that_no_pair_counts(pkg, K):
    """A label above the classes outside of all sequences, or in a pair of weight 0: its row has a gradient of zeros and a log-probability of NaN, the pair a
    margin of NaN and a loss of 0.  All else is as without it."""
    rng = np.random.default_rng(K)
    n = 9
    z, zd = logits(rng, n, K, torch.float32)
    label = torch.from_numpy(rng.integers(1, K + 1, size=n).astype(np.int32))
    seq, w = torch.tensor([1, 3, 5, 6, 8], dtype=torch.int32), torch.tensor([1.0, 0.0])
    good = pkg.preference_grads(zd, label.cuda(), seq.cuda(), w=w.cuda())
    label[[0, 6, 8]] = torch.tensor([K + 1, K + 2, -1], dtype=torch.int32)
    loss, margin, logp, grad = pkg.preference_grads(zd, label.cuda(), seq.cuda(), w=w.cuda())
    assert torch.equal(loss, good[0]) and loss[1] == 0
    assert margin[0] == good[1][0] and torch.isnan(margin[1])
    assert torch.isnan(logp[[0, 6, 8]]).all() and torch.equal(logp[[1, 2, 3, 4, 5, 7]], good[2][[1, 2, 3, 4, 5, 7]])
    assert torch.equal(grad, good[3]) and (grad[[0, 5, 6, 7, 8]] == 0).all()


@pytest.mark.parametrize("K,T", [(3, 40), (9, 33), (20, 50), (20, 200), (32, 1024), (200, 1000)])
@pytest.mark.parametrize("n", [6, 700])
@pytest.mark.parametrize("tail", [False, True])
def test_more_slots_than_classes(pkg, K, T, n, tail):
    """Most of them empty or of a class that other slots name too."""
    rng = np.random.default_rng(T)
    z, zd = logits(rng, n, K, torch.float32)
    ids = torch.from_numpy((rng.integers(0, K, (n, T)) * (rng.random((n, T)) < 0.5)).astype(np.int32))      # one class is never named
    t = torch.from_numpy(rng.normal(size=(n, T)).astype(np.float32))
    t = log_probs(t, 0.9) if tail else t
    out = pkg.distill_grads(zd, ids.cuda(), t.cuda(), tail=tail, hess=True)
    keep = [0, 1, n // 2, n - 2, n - 1]
    check_distill([o[keep] for o in out], z[keep], ids[keep], t[keep], None, 1.0, tail, True)


@pytest.mark.parametrize("K,T", [(12, 40), (31, 100)])
@pytest.mark.parametrize("weights", [False, True])
def test_more_slots_than_classes_in_fit(pkg, K, T, weights):
    from tests.test_objectives_gpu import check_grads, table
    rng = np.random.default_rng(K)
    n = 500
    params = pkg.EvoTreeClassifier(loss="distill", nrounds=3, max_depth=3, nbins=16, nclasses=K)
    x = table(rng, n)
    y = rng.integers(0, K + 1, (n, T)), rng.normal(size=(n, T)).astype(np.float32)
    w = (0.5 + rng.random(n)).astype(np.float32) if weights else None
    m, cache = pkg.init_core(params, x, y, w)
    cb = pkg.CallBack(params, m, cache, x, y, w)
    for _ in range(2):
        pkg.grow_evotree(m, cache, params)
        check_grads(params, cache, y, w, K)
    t = [torch.from_numpy(np.asarray(v)) for v in y]
    wt = torch.ones(n) if w is None else torch.from_numpy(w)
    want = float(R.distill(torch.from_numpy(cb.pred()), t[0], t[1], wt)[0].sum() / wt.to(F8).sum())
    assert abs(cb.last() - want) < 1e-4 * (1 + abs(want))
    cache.close()

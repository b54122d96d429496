"""Distillation with a tail where the classes without a slot lie far from the named ones, or all of them far from zero."""
import numpy as np
import pytest
import torch

from tests import losses_ref as R
from tests.test_losses_gpu import DTYPES, F8, NINF, log_probs, logits, slots

pytestmark = pytest.mark.gpu
CLASSES = [5, 9, 32, 40, 1000, 9000, 70001, 200003]      # every kernel


def check(out, z, ids, t, w=None, hess=False):
    """Against the definition.  A probability p_k is off by `rel` of itself, and so is p_k / p_T of a class without a slot (both are terms over a sum of
    terms, at most 120 below their own maximum where they are not zero in 32 bits), q_T by `rel` of 1, whatever is left of it."""
    n, K = z.shape
    loss, grad, h, scale = R.distill(z, ids, t, w, 1.0, True)
    wt = torch.ones(n, dtype=F8) if w is None else w.to(F8)
    named = torch.zeros((n, K + 1), dtype=torch.bool).scatter_(1, torch.where(t > NINF, ids.long(), 0), True)[:, 1:]
    rest = z.to(F8).masked_fill(named, NINF)
    rel = torch.maximum(R.part(z), R.part(rest)) + R.slots_part(t)
    p, share = torch.softmax(z.to(F8), 1), torch.softmax(rest, 1).nan_to_num()
    q = torch.zeros((n, K + 1), dtype=F8).scatter_add_(1, ids.long(), t.to(F8).exp())[:, 1:]
    R.close(out[0], loss, 2 * rel * scale + R.U * loss.abs(), "loss")
    R.close(out[1], grad, R.rounded(grad, z.dtype, 2 * rel[:, None], wt[:, None] * (p + q + 2 * share)), "grad")
    if hess:
        R.close(out[2], h, R.rounded(h, z.dtype, 2 * rel[:, None], wt[:, None] * (p + p * p)), "hess")


@pytest.mark.parametrize("offset", [100.0, 1.0e4, 1.0e6])
@pytest.mark.parametrize("K", CLASSES)
def test_offsets(pkg, K, offset):
    """Softmax does not see what is added to all classes of a row; the predictions are rounded before they are compared."""
    rng = np.random.default_rng(K)
    n = 5
    z = (logits(rng, n, K, torch.float32)[0].to(F8) + offset).float()
    ids, t = slots(rng, n, K, min(64, K - 2), empty=0.0)
    t = log_probs(t, 0.7)
    check(pkg.distill_grads(z.cuda(), ids.cuda(), t.cuda(), tail=True, hess=True), z, ids, t, hess=True)


@pytest.mark.parametrize("above", [100.0, 1.0e4])
@pytest.mark.parametrize("K,dtype", [(1000, "f32"), (9000, "f32"), (70001, "f32"), (131073, "f32"), (200003, "f32"), (270001, "bf16")])
def test_named_classes_above_all_others(pkg, K, dtype, above):
    """The classes that the teacher names lie further above the others than 32-bit exponents reach."""
    rng = np.random.default_rng(K)
    n = 4
    z, _ = logits(rng, n, K, DTYPES[dtype])
    ids, t = slots(rng, n, K, 40, empty=0.0)
    z.scatter_(1, ids.long() - 1, (above + torch.from_numpy(rng.normal(size=(n, 40)))).to(z.dtype))
    t = log_probs(t, 0.9)
    check(pkg.distill_grads(z.cuda(), ids.cuda(), t.cuda(), tail=True, hess=True), z, ids, t, hess=True)

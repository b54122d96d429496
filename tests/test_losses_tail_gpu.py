"""Distillation with a tail where the classes without a slot lie far from the named ones, or all of them far from zero."""
import numpy as np
import pytest
import torch

from tests import losses_ref as R
from tests.test_losses_gpu import DTYPES, F8, NINF, check_distill, log_probs, logits, slots

pytestmark = pytest.mark.gpu
CLASSES = [5, 9, 32, 40, 1000, 9000, 70001, 200003]      # every kernel


def check(out, z, ids, t, w=None, hess=False):
    """Against the definition.  A probability p_k is off by `rel` of itself, and so is p_k / p_T of a class without a slot (both are terms over a sum of
    terms, at most 120 below their own maximum where they are not zero in 32 bits), q_T by `rel` of 1, whatever is left of it.  Gradients are the formula's:
    differentiation goes through log p_T, which in 64 bits no longer holds the logarithm of the number of classes beside a mask of 1e38."""
    n, K = z.shape
    loss, _, h, scale = R.distill(z, ids, t, w, 1.0, True)
    wt = torch.ones(n, dtype=F8) if w is None else w.to(F8)
    named = torch.zeros((n, K + 1), dtype=torch.bool).scatter_(1, torch.where(t > NINF, ids.long(), 0), True)[:, 1:]
    rest = z.to(F8).masked_fill(named, NINF)
    rel = torch.maximum(R.part(z), R.part(rest)) + R.slots_part(t)
    p, share = torch.softmax(z.to(F8), 1), torch.softmax(rest, 1).nan_to_num()
    q = torch.zeros((n, K + 1), dtype=F8).scatter_add_(1, ids.long(), t.to(F8).exp())[:, 1:]
    left = torch.where((rest > NINF).any(1), (1 - q.sum(1)).clamp(min=0), 0)[:, None]
    grad = wt[:, None] * ((q.sum(1, keepdim=True) + left) * p - q - left * share)
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


def masked_rows(rng, K, dtype, mask):
    """Rows of which only the named classes are allowed, or nearly so."""
    n, T = 6, 4
    z = torch.full((n, K), mask, dtype=DTYPES[dtype])
    ids, t = slots(rng, n, K, T, empty=0.0)
    t = log_probs(t, 0.9)
    t[0] = float(np.log(0.25 * 0.96))
    t[1] += float(np.log(1.2))                              # more than 1: nothing is left for the tail
    z[2, ::2] = mask / 2                                    # masks of two kinds ..
    z[3, 1::3] = NINF                                       # .. and classes that are ruled out
    if -mask > 1.0e5:
        z[5] = torch.from_numpy(rng.normal(size=K)).to(z.dtype)
    z.scatter_(1, ids.long() - 1, torch.tensor([2.0, 1.0, 0.0, -1.0], dtype=z.dtype).expand(n, T))
    if -mask > 1.0e5:                                       # the named ones are far away, the others are not
        z[5, ids[5].long() - 1] = torch.tensor([-mask, -mask, -mask / 2, 0.0], dtype=z.dtype)
    ids[4, 2] = ids[4, 0]                                   # a class in two slots; another one is allowed and has none
    return z, ids, t, torch.from_numpy((0.5 + rng.random(n)).astype(np.float32))


@pytest.mark.parametrize("dtype,mask", [("f32", -1.0e4), ("f32", -1.0e8), ("f32", -1.0e9), ("f32", "lowest"), ("bf16", -1.0e4), ("bf16", -1.0e8), ("bf16", -1.0e9),
                                        ("bf16", "lowest"), ("f16", -1.0e4), ("f16", "lowest")])
@pytest.mark.parametrize("K", CLASSES)
def test_all_other_classes_masked(pkg, K, dtype, mask):
    from evotrees_b200 import _lib
    rng = np.random.default_rng(K)
    # of the type's lowest value half: sums of losses stay within 32 bits
    z, ids, t, w = masked_rows(rng, K, dtype, torch.finfo(DTYPES[dtype]).min / (1 if dtype == "f16" else 2) if mask == "lowest" else mask)
    check(pkg.distill_grads(z.cuda(), ids.cuda(), t.cuda(), w=w.cuda(), tail=True, hess=True), z, ids, t, w, hess=True)
    # many rows: kernels of other shapes, with and without work memory
    n, r = z.shape[0], 56
    many = [v.cuda().repeat(r, *([1] * (v.dim() - 1))) for v in (z, ids, t, w)]
    loss, g = pkg.distill_grads(many[0], many[1], many[2], w=many[3], tail=True)
    loss2, g2 = torch.empty_like(loss), torch.empty_like(g)
    _lib.check(_lib.lib().evb_distill_grads(0, 0, many[0].data_ptr(), {"f32": _lib.EVB_F32, "bf16": _lib.EVB_BF16, "f16": _lib.EVB_F16}[dtype], n * r, K, K, many[1].data_ptr(),
                                            many[2].data_ptr(), _lib.EVB_F32, ids.shape[1], 1, many[3].data_ptr(), 1.0, loss2.data_ptr(), g2.data_ptr(), K, None, 0, None))
    torch.cuda.synchronize()
    for a, b in ((loss, g), (loss2, g2)):
        check((a[:n], b[:n]), z, ids, t, w)
        check((a[-n:], b[-n:]), z, ids, t, w)               # the same rows beginning elsewhere


@pytest.mark.parametrize("K", CLASSES)
def test_other_classes_at_the_lowest_value(pkg, K):
    """The lowest value itself, the teacher leaves a twentieth of its mass to it: a loss of 1.7e37."""
    for dtype in ("f32", "bf16"):
        low = torch.finfo(DTYPES[dtype]).min
        z = torch.full((2, K), low, dtype=DTYPES[dtype])
        ids = torch.tensor([[1, 2, 3], [K, K - 1, 1]], dtype=torch.int32)
        z.scatter_(1, ids.long() - 1, torch.tensor([[3.0, 1.0, -1.0]], dtype=z.dtype).expand(2, 3))
        t = torch.log(torch.tensor([[0.57, 0.285, 0.095], [0.6, 0.4, 0.1]]))
        check(pkg.distill_grads(z.cuda(), ids.cuda(), t.cuda(), tail=True, hess=True), z, ids, t, hess=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("K", CLASSES + [270001])
def test_class_named_or_taken_near_the_lowest_value(pkg, K, dtype):
    """Its log-probability is a number: the loss is a share of that, not infinite."""
    rng = np.random.default_rng(K)
    z, _ = logits(rng, 3, K, DTYPES[dtype])
    ids, t = slots(rng, 3, K, 3, empty=0.0)
    low = 0.8 * torch.finfo(z.dtype).min                    # its product with log2(e) is beyond 32 bits
    z[0, ids[0, 1].long() - 1] = low
    z[1, ids[1].long() - 1] = low                           # nothing else is named
    z[2, ids[2, 0].long() - 1] = low / 2
    lt = log_probs(t, 0.6)
    check(pkg.distill_grads(z.cuda(), ids.cuda(), lt.cuda(), tail=True, hess=True), z, ids, lt, hess=True)
    check_distill(pkg.distill_grads(z.cuda(), ids.cuda(), t.cuda(), hess=True), z, ids, t, None, 1.0, False, True)
    a, old, adv = ids[torch.arange(3), torch.tensor([1, 0, 0])].contiguous(), torch.tensor([-1.0, -2.0, -3.0]), torch.tensor([1.0, -1.0, 0.5])
    out = pkg.policy_grads(z.cuda(), a.cuda(), old.cuda(), adv.cuda(), hess=True)
    loss, logp, grad, h, scale = R.policy(z, a, old, adv)
    rel = R.part(z)
    R.close(out[1], logp, 8 * R.U * logp.abs() + rel, "logp")
    R.close(out[0], loss, 4 * rel * scale + R.U * loss.abs(), "loss")
    R.close(out[2], grad, R.rounded(grad, z.dtype, 4 * rel[:, None], scale[:, None]), "grad")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("K", CLASSES[1:])
@pytest.mark.parametrize("tau", [0.5, 1.0, 2.0])
def test_many_named_classes_near_the_lowest_value(pkg, K, dtype, tau):
    """What the slots add up to before they are divided by their sum, and what a temperature divides, may be beyond 32 bits where the loss is not."""
    rng = np.random.default_rng(K)
    z, _ = logits(rng, 2, K, DTYPES[dtype])
    ids, _ = slots(rng, 2, K, 7, empty=0.0)
    z.scatter_(1, ids[:, 1:].long() - 1, 0.8 * torch.finfo(z.dtype).min)
    t = torch.zeros((2, 7))
    t[:, 1:] = tau * float(np.log(0.25))                    # the masked six have 0.6 together
    check_distill(pkg.distill_grads(z.cuda(), ids.cuda(), t.cuda(), tau=tau, hess=True), z, ids, t, None, tau, False, True)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("K", CLASSES)
@pytest.mark.parametrize("tail", [False, True])
def test_rows_with_a_prediction_that_is_no_number(pkg, K, tail, value):
    """Wherever it is, in a slot or not, the only one named or not: NaN in all that the row gives."""
    for dtype in DTYPES.values():
        z = torch.zeros((4, K), dtype=dtype)
        z[0, 1], z[1, 2], z[2, K - 1] = value, value, value
        ids = torch.tensor([[2, 0], [1, 3], [1, 2], [1, 2]], dtype=torch.int32)
        out = pkg.distill_grads(z.cuda(), ids.cuda(), torch.full((4, 2), -0.8).cuda(), tail=tail, hess=True)
        assert all(torch.isnan(o[:3]).all() and torch.isfinite(o[3]).all() for o in out)
        a, v = torch.tensor([2, 1, 1, 1], dtype=torch.int32).cuda(), torch.ones(4, device="cuda")
        out = pkg.policy_grads(z.cuda(), a, -v, v, hess=True)
        assert all(torch.isnan(o[:3]).all() and torch.isfinite(o[3]).all() for o in out)

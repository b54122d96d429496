"""Losses on rows of raw predictions that live on the GPU, with their gradients (and hessians, for boosting): distillation from a
teacher's top logits, the clipped policy loss with a KL term, the preference loss of paired log ratios.  The formulas are in
include/evb.h (`evb_distill_grads`, `evb_policy_grads`, `evb_preference_grads`).

Arrays are torch tensors on one CUDA device.  `pred` is [rows, classes] float32, bfloat16 or float16, a row's classes side by side, rows at
any stride; class codes are int32, 1..classes, 0 = none.  Per-row vectors are contiguous float32.  Calls run on the device's current
stream, wait for nothing, and can be captured into a CUDA graph; they take no part in autograd: gradients are returned.
"""
from __future__ import annotations

import torch

from . import _lib

# a call on a few rows is as long as its way through here: one attribute look-up each, no objects that are not needed
_F32, _I32 = torch.float32, torch.int32
_DTYPES = {torch.float32: _lib.EVB_F32, torch.bfloat16: _lib.EVB_BF16, torch.float16: _lib.EVB_F16}


def _rows(pred):
    """Type code, rows, classes, row stride and device of `pred`."""
    if not isinstance(pred, torch.Tensor) or pred.dim() != 2:
        raise ValueError("`pred` must be a torch tensor of shape [rows, classes]")
    code = _DTYPES.get(pred.dtype)
    if code is None:
        raise ValueError(f"`pred` must be float32, bfloat16 or float16, not {pred.dtype}")
    if not pred.is_cuda:
        raise _lib.EvbError(-2, "`pred` is not on a CUDA device: this library has no CPU fallback")
    n, K = pred.shape
    if K < 1:
        raise ValueError("`pred` has no classes")
    ld, one = pred.stride()
    if n <= 1:
        ld = K
    if (K > 1 and one != 1) or ld < K:
        raise ValueError("the classes of a row of `pred` must lie side by side, rows behind one another")
    return code, n, K, ld, pred.device


def _vec(name, v, shape, dtype, dev):
    """Address of an array that goes with `pred`."""
    try:
        if v.dtype is dtype and v.shape == shape and v.is_contiguous() and v.device == dev:
            return v.data_ptr()
    except AttributeError:
        pass
    raise ValueError(f"`{name}` must be a contiguous {dtype} tensor of shape {list(shape)} on {dev}")


def _outputs(pred, n, K, grads, hess):
    if not grads:
        return None, 0, None, 0
    g = pred.new_empty((n, K))
    if not hess:
        return g, g.data_ptr(), None, 0
    h = pred.new_empty((n, K))
    return g, g.data_ptr(), h, h.data_ptr()


def distill_grads(pred, ids, teacher, *, w=None, tau: float = 1.0, tail: bool = False, hess: bool = False, grads: bool = True):
    """Divergence from a teacher of whom the top classes of every row were kept: `ids` int32 [rows, slots] (0 = empty) with `teacher`
    [rows, slots], its logits, or with `tail=True` its log-probabilities, the probability of all other classes then being one class
    more.  Returns (loss [rows], gradient [rows, classes][, hessian]); the loss alone with `grads=False`."""
    code, n, K, ld, dev = _rows(pred)
    if not isinstance(ids, torch.Tensor) or ids.dim() != 2 or ids.shape[1] < 1:
        raise ValueError("`ids` must be a torch tensor of shape [rows, slots] with at least one slot")
    T = ids.shape[1]
    pi = _vec("ids", ids, (n, T), _I32, dev)
    tcode = _DTYPES.get(getattr(teacher, "dtype", None))
    if tcode is None:
        raise ValueError("`teacher` must be a float32, bfloat16 or float16 tensor")
    pt = _vec("teacher", teacher, (n, T), teacher.dtype, dev)
    pw = None if w is None else _vec("w", w, (n,), _F32, dev)
    loss = torch.empty(n, dtype=_F32, device=dev)
    g, pg, h, ph = _outputs(pred, n, K, grads, hess)
    work = torch.empty(8 * n, dtype=_F32, device=dev) if K > 1000 else None
    rc = _lib.lib().evb_distill_grads(dev.index, _lib.raw_stream(dev.index), pred.data_ptr(), code, n, K, ld, pi, pt, tcode, T, bool(tail), pw, tau,
                                      loss.data_ptr(), pg, K, ph, K, None if work is None else work.data_ptr())
    if rc:
        _lib.check(rc)
    return (loss,) if g is None else (loss, g) if h is None else (loss, g, h)


def policy_grads(pred, action, old_logp, adv, *, ref_logp=None, w=None, tau: float = 1.0, clip=(0.2, 0.2), beta: float = 0.0,
                 hess: bool = False, grads: bool = True):
    """Clipped policy loss of the class `action` (int32 [rows], 0 = the row does not count) that was taken with log-probability `old_logp`
    and turned out with advantage `adv`, plus `beta` times an estimate of the divergence from a reference policy (`ref_logp`).
    Returns (loss [rows], logp [rows], gradient [rows, classes][, hessian]); (loss, logp) with `grads=False`."""
    code, n, K, ld, dev = _rows(pred)
    row = (n,)
    pa = _vec("action", action, row, _I32, dev)
    po, pv = _vec("old_logp", old_logp, row, _F32, dev), _vec("adv", adv, row, _F32, dev)
    pr = None if ref_logp is None else _vec("ref_logp", ref_logp, row, _F32, dev)
    pw = None if w is None else _vec("w", w, row, _F32, dev)
    low, high = clip
    loss, logp = torch.empty(n, dtype=_F32, device=dev), torch.empty(n, dtype=_F32, device=dev)
    g, pg, h, ph = _outputs(pred, n, K, grads, hess)
    rc = _lib.lib().evb_policy_grads(dev.index, _lib.raw_stream(dev.index), pred.data_ptr(), code, n, K, ld, pa, po, pv, pr, pw, tau, low, high, beta,
                                     loss.data_ptr(), logp.data_ptr(), pg, K, ph, K)
    if rc:
        _lib.check(rc)
    return (loss, logp) if g is None else (loss, logp, g) if h is None else (loss, logp, g, h)


def preference_grads(pred, label, seq, *, ref_logp=None, w=None, beta: float = 0.1, smooth: float = 0.0, mean: bool = False, grads: bool = True):
    """Preference loss of pairs of sequences of rows.  `label` int32 [rows] is the class of every row (0 = not counted), `seq` int32
    [2 pairs + 1] where the sequences begin and end: sequence 2 p is preferred to sequence 2 p + 1.  The margin of a pair is `beta` times
    the difference of the sequences' sums (`mean=True`: means) of log p - `ref_logp`.
    Returns (loss [pairs], margin [pairs], logp [rows], gradient [rows, classes]); without the last with `grads=False`."""
    code, n, K, ld, dev = _rows(pred)
    row = (n,)
    pl = _vec("label", label, row, _I32, dev)
    if not isinstance(seq, torch.Tensor) or seq.dim() != 1 or seq.shape[0] % 2 != 1:
        raise ValueError("`seq` must be a torch tensor of 2 pairs + 1 row numbers")
    P = seq.shape[0] // 2
    ps = _vec("seq", seq, seq.shape, _I32, dev)
    pr = None if ref_logp is None else _vec("ref_logp", ref_logp, row, _F32, dev)
    pw = None if w is None else _vec("w", w, (P,), _F32, dev)
    loss, margin = torch.empty(P, dtype=_F32, device=dev), torch.empty(P, dtype=_F32, device=dev)
    logp, work = torch.empty(n, dtype=_F32, device=dev), torch.empty(3 * n, dtype=_F32, device=dev)
    g, pg, _, _ = _outputs(pred, n, K, grads, False)
    rc = _lib.lib().evb_preference_grads(dev.index, _lib.raw_stream(dev.index), pred.data_ptr(), code, n, K, ld, pl, ps, P, pr, pw, beta, smooth, bool(mean),
                                         loss.data_ptr(), margin.data_ptr(), logp.data_ptr(), pg, K, work.data_ptr())
    if rc:
        _lib.check(rc)
    return (loss, margin, logp) if g is None else (loss, margin, logp, g)

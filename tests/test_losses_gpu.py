"""Losses on rows of raw predictions against their definitions in 64 bits: sizes that take every path, masks, strides, extremes."""
import numpy as np
import pytest
import torch

from tests import losses_ref as R

pytestmark = pytest.mark.gpu
F8 = torch.float64
NINF = float("-inf")
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# around the borders of what a thread, a warp, a block and several blocks hold, and odd sizes
CLASSES = [1, 2, 3, 5, 8, 17, 31, 32, 33, 64, 65, 127, 200, 255, 256, 257, 511, 1000, 1024, 1025, 2047, 2049, 4096, 8191, 16385, 32768, 50021, 65536, 65537, 131072]
WIDE = [131073, 270001, 600000]      # beyond what a cluster holds, for the wider types first


def logits(rng, n, K, dtype, pad=0, shift=0):
    """[n, K] on the CPU and a view of it on the GPU, `pad` elements between rows, the first one `shift` elements into its buffer."""
    z = torch.from_numpy((rng.normal(size=(n, K)) * 2.0).astype(np.float32))
    for i in range(n):
        z[i, rng.integers(0, K)] += 6.0
    z = z.to(dtype)
    buf = torch.full((n * (K + pad) + shift,), float("nan"), dtype=dtype, device="cuda")
    view = buf[shift:].view(n, K + pad)[:, :K]
    view.copy_(z)
    return z, view


def slots(rng, n, K, T, dtype=torch.float32, empty=0.2):
    ids = np.stack([rng.choice(K, size=T, replace=False) + 1 for _ in range(n)]).astype(np.int32)
    ids[rng.random((n, T)) < empty] = 0
    t = torch.from_numpy((rng.normal(size=(n, T)) * 2.0).astype(np.float32))
    return torch.from_numpy(ids), t.to(dtype)


def log_probs(t, share):
    """Slots' log-probabilities that sum up to `share`."""
    return (torch.log_softmax(t.to(F8), 1) + np.log(share)).float()


def check_distill(out, z, ids, t, w, tau, tail, hess):
    loss, grad, h, scale = R.distill(z, ids, t, w, tau, tail)
    rel = R.part(z, tau) + R.slots_part(t, tau)
    wt = torch.ones(z.shape[0], dtype=F8) if w is None else torch.nan_to_num(w.to(F8)).abs()
    R.close(out[0], loss, 2 * rel * scale + R.U * loss.abs(), "loss")
    p = torch.softmax(z.to(F8) / tau, 1).nan_to_num()
    # a gradient is a difference of probabilities: what each of them may be off; with a tail also of p_k / p_T
    size = p + torch.zeros_like(p).scatter_add_(1, (ids.long() - 1).clamp(min=0), torch.where(ids > 0, (t.to(F8) if tail else torch.log_softmax(
        torch.where(ids > 0, t.to(F8) / tau, torch.full_like(t, -1e300, dtype=F8)), 1)).exp().nan_to_num(), torch.zeros((), dtype=F8)))
    if tail:
        size = size + grad.abs().nan_to_num() / wt.clamp(min=1e-300)[:, None]
        # 1 - sum q is off by `rel`, whatever is left of it
        named = torch.zeros((z.shape[0], z.shape[1] + 1), dtype=torch.bool).scatter_(1, ids.long().clamp(0, z.shape[1]), True)[:, 1:]
        rest = torch.where(named, torch.zeros_like(p), p)
        size = size + rest / rest.sum(1, keepdim=True).clamp(min=1e-300)
    R.close(out[1], grad, R.rounded(grad, z.dtype, 2 * rel[:, None], wt[:, None] * tau * size), "grad")
    if hess:
        R.close(out[2], h, R.rounded(h, z.dtype, 2 * rel[:, None], wt[:, None] * (p + p * p)), "hess")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("K", CLASSES)
def test_distill_sizes(pkg, K, dtype):
    rng = np.random.default_rng(K)
    n, T = (5, min(K, 1 + K % 37)) if K > 300 else (int(rng.integers(1, 400)), min(K, 6))
    z, zd = logits(rng, n, K, DTYPES[dtype])
    ids, t = slots(rng, n, K, T, DTYPES[dtype])
    hess = K % 2 == 0
    out = pkg.distill_grads(zd, ids.cuda(), t.cuda(), tau=1.5, hess=hess)
    check_distill(out, z, ids, t, None, 1.5, False, hess)
    lt = log_probs(t, 0.9)
    out = pkg.distill_grads(zd, ids.cuda(), lt.cuda(), tail=True, hess=hess)
    check_distill(out, z, ids, lt, None, 1.0, True, hess)


@pytest.mark.parametrize("K", [2500, 20011, 70001, 200003])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_with_and_without_work_memory(pkg, K, tail):
    """Enough rows for a launch of its own for the teacher's side, which the C entry leaves out without work memory."""
    from evotrees_b200 import _lib
    rng = np.random.default_rng(K)
    n, T = 320, 70
    z, zd = logits(rng, n, K, torch.bfloat16)
    ids, t = slots(rng, n, K, T)
    ids[5] = 0
    ids[7, 3] = K + 1
    ids[9, :6] = ids[9, 0].clamp(min=1)                            # a class again and again
    w = torch.ones(n)
    w[11] = 0.0
    t = log_probs(t, 0.9) if tail else t
    idd, td, wd = ids.cuda(), t.cuda(), w.cuda()
    loss, g = pkg.distill_grads(zd, idd, td, w=wd, tail=tail)
    loss2, g2 = torch.empty(n, device="cuda"), torch.empty_like(g)
    _lib.check(_lib.lib().evb_distill_grads(0, 0, zd.data_ptr(), _lib.EVB_BF16, n, K, K, idd.data_ptr(), td.data_ptr(), _lib.EVB_F32, T, int(tail), wd.data_ptr(),
                                            1.0, loss2.data_ptr(), g2.data_ptr(), K, None, 0, None))
    torch.cuda.synchronize()
    keep = [0, 1, 5, 9, 11, n - 1]
    for out in ((loss, g), (loss2, g2)):
        assert torch.isnan(out[0][7]) and torch.isnan(out[1][7]).all()
        check_distill([o[keep] for o in out], z[keep], ids[keep], t[keep], w[keep], 1.0, tail, False)


def test_distill_most_slots_of_many_rows_in_a_graph(pkg):
    rng = np.random.default_rng(8)
    n, K, T = 300, 5000, 1024
    z, zd = logits(rng, n, K, torch.float32)
    ids, t = slots(rng, n, K, T)
    lt = log_probs(t, 0.9)
    idd, td = ids.cuda(), lt.cuda()
    plain = pkg.distill_grads(zd, idd, td, tail=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = pkg.distill_grads(zd, idd, td, tail=True)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(plain, out))
    keep = [0, 150, n - 1]
    check_distill([o[keep] for o in out], z[keep], ids[keep], lt[keep], None, 1.0, True, False)


def test_calls_of_several_threads(pkg):
    """Calls of different sizes at the same time, each thread on its own stream: the bits of calls one by one."""
    import threading
    rng = np.random.default_rng(12)
    jobs = []
    for n, K, T in ((300, 5, 3), (200, 300, 40), (320, 9000, 70), (12, 40000, 5)):
        z, zd = logits(rng, n, K, torch.float32)
        ids, t = slots(rng, n, K, T) if T <= K else None
        jobs.append((zd, ids.cuda(), t.cuda()))
    torch.cuda.synchronize()
    want = [pkg.distill_grads(*j) for j in jobs]
    torch.cuda.synchronize()
    wrong = []

    def work(j, w):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                out = pkg.distill_grads(*j)
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(x, y) for x, y in zip(out, w)):
                    wrong.append(j[0].shape)

    threads = [threading.Thread(target=work, args=a) for a in zip(jobs, want)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong


@pytest.mark.parametrize("K,T", [(40, 40), (40, 39), (1500, 1024), (9000, 700), (131072, 1024), (7, 1)])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_many_slots(pkg, K, T, tail):
    """Up to the most slots, up to a slot for every class: with a tail no class is left then."""
    rng = np.random.default_rng(T)
    z, zd = logits(rng, 4, K, torch.float32)
    ids, t = slots(rng, 4, K, T, empty=0.0)
    if tail:
        t = log_probs(t, 0.8)
    out = pkg.distill_grads(zd, ids.cuda(), t.cuda(), tail=tail, hess=True)
    check_distill(out, z, ids, t, None, 1.0, tail, True)


@pytest.mark.parametrize("K", [6, 50, 300, 5000, 131071])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_class_in_several_slots(pkg, K, tail):
    rng = np.random.default_rng(K)
    z, zd = logits(rng, 6, K, torch.float32)
    ids = torch.from_numpy(rng.integers(1, min(K, 4) + 1, size=(6, 9)).astype(np.int32))
    t = torch.from_numpy(rng.normal(size=(6, 9)).astype(np.float32))
    if tail:
        t = log_probs(t, 0.7)
    out = pkg.distill_grads(zd, ids.cuda(), t.cuda(), tail=tail, hess=True)
    check_distill(out, z, ids, t, None, 1.0, tail, True)


@pytest.mark.parametrize("K", [9, 70, 700, 9000, 70001])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_masks_and_extremes(pkg, K, tail):
    """Rows without slots, of weight 0 with NaN in them, slots of -inf, classes of -inf and of the type's lowest value, a class that is certain."""
    rng = np.random.default_rng(K)
    n, T = 10, 5
    z, _ = logits(rng, n, K, torch.float32)
    ids, t = slots(rng, n, K, T, empty=0.0)
    t = log_probs(t, 0.9) if tail else t
    w = torch.from_numpy((0.5 + rng.random(n)).astype(np.float32))
    ids[0] = 0                                                     # no slot at all
    t[1] = NINF                                                    # slots that hold nothing
    w[2], z[2], t[2] = 0.0, float("nan"), float("nan")             # masked: whatever is there
    z[3, torch.randperm(K)[: K // 2]] = NINF                       # classes that are ruled out ..
    z[3, ids[3].long() - 1] = 0.0                                  # .. the named ones are not
    low = torch.randperm(K)[: K // 3]
    z[4, low] = torch.finfo(torch.float32).min
    z[4, ids[4].long() - 1] = 1.0
    z[5, ids[5, 0].long() - 1] = 90.0                              # certain
    z[6, :] = NINF
    z[6, ids[6].long() - 1] = 0.5                                  # only the named classes are possible: no class is left for a tail
    t[7, 1:] = NINF                                                # one slot
    z[8] = 0.0
    ids[9, 2] = K + 1 if K % 2 else -3                             # a class that there is not
    out = pkg.distill_grads(z.cuda(), ids.cuda(), t.cuda(), w=w.cuda(), tail=tail, hess=True)
    assert (out[0][:3] == 0).all() and (out[1][:3] == 0).all() and (out[2][:3] == 0).all()
    assert torch.isnan(out[0][9]) and torch.isnan(out[1][9]).all() and torch.isnan(out[2][9]).all()
    keep = [3, 4, 5, 6, 7, 8]
    check_distill([o[keep] for o in out], z[keep], ids[keep], t[keep], w[keep], 1.0, tail, True)


def test_distill_named_class_ruled_out(pkg):
    """A class that the teacher wants and the student rules out: an infinite loss, a finite gradient."""
    z = torch.zeros((2, 100)); z[:, 7] = NINF
    ids = torch.tensor([[8, 3], [3, 8]], dtype=torch.int32)
    t = torch.tensor([[0.0, 0.0], [0.0, -200.0]])                  # in the second row its probability is zero in 32 bits
    loss, g = pkg.distill_grads(z.cuda(), ids.cuda(), t.cuda())
    assert loss[0].item() == float("inf") and torch.isfinite(loss[1]) and torch.isfinite(g).all()
    assert abs(g[0, 7].item() + 0.5) < 1e-6 and g[1, 7].item() == 0.0
    want = R.distill(z[1:], ids[1:, :1], t[1:, :1])
    R.close(loss[1:], want[0], 1e-5, "loss")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("K", CLASSES)
def test_policy_sizes(pkg, K, dtype):
    rng = np.random.default_rng(K + 1)
    n = 7 if K > 300 else int(rng.integers(1, 400))
    z, zd = logits(rng, n, K, DTYPES[dtype])
    check_policy(pkg, rng, z, zd, tau=1.0, beta=0.1, hess=K % 2 == 1)
    check_policy(pkg, rng, z, zd, tau=2.0, beta=0.0, hess=K % 2 == 0, ref=False)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("K", WIDE)
def test_wide_rows(pkg, K, dtype):
    rng = np.random.default_rng(K + 3)
    z, zd = logits(rng, 3, K, DTYPES[dtype], pad=K % 5)
    ids, t = slots(rng, 3, K, 40)
    check_distill(pkg.distill_grads(zd, ids.cuda(), t.cuda(), tau=1.5, hess=True), z, ids, t, None, 1.5, False, True)
    lt = log_probs(t, 0.9)
    check_distill(pkg.distill_grads(zd, ids.cuda(), lt.cuda(), tail=True), z, ids, lt, None, 1.0, True, False)
    check_policy(pkg, rng, z, zd, 1.0, 0.1, True)
    check_preference(pkg, z, zd, torch.tensor([5, 0, K], dtype=torch.int32), torch.tensor([0, 1, 3], dtype=torch.int32))


def check_policy(pkg, rng, z, zd, tau, beta, hess, ref=True, w=None):
    n, K = z.shape
    a = torch.from_numpy(rng.integers(0 if n > 2 else 1, K + 1, size=n).astype(np.int32))
    lp = torch.log_softmax(z.to(F8) / tau, 1).gather(1, (a.long() - 1).clamp(min=0)[:, None])[:, 0]
    ratio = rng.normal(size=n) * 0.3
    for edge in (np.log(0.8), np.log(1.3)):                        # away from where the gradient jumps
        ratio = np.where(abs(ratio - edge) < 0.01, edge + 0.02, ratio)
    old, adv = (lp - torch.from_numpy(ratio)).float(), torch.from_numpy(rng.normal(size=n).astype(np.float32))
    rf = (lp + torch.from_numpy(rng.normal(size=n) * 0.3)).float() if ref else None
    out = pkg.policy_grads(zd, a.cuda(), old.cuda(), adv.cuda(), ref_logp=None if rf is None else rf.cuda(), w=None if w is None else w.cuda(), tau=tau,
                           clip=(0.2, 0.3), beta=beta, hess=hess)
    loss, logp, grad, h, scale = R.policy(z, a, old, adv, rf, w, tau, (0.2, 0.3), beta)
    rel = R.part(z, tau) + R.U * 4 * logp.abs().nan_to_num()
    R.close(out[1], logp, rel + R.U * logp.abs(), "logp")
    R.close(out[0], loss, 4 * rel * scale + R.U * loss.abs(), "loss")
    p = torch.softmax(z.to(F8) / tau, 1).nan_to_num()
    d = scale / tau
    onehot = torch.zeros_like(p).scatter_(1, (a.long() - 1).clamp(min=0)[:, None], 1.0)
    R.close(out[2], grad, R.rounded(grad, z.dtype, 4 * rel[:, None], d[:, None] * (p + onehot)), "grad")
    if hess:
        wt = torch.ones(n, dtype=F8) if w is None else w.to(F8)
        R.close(out[3], h, R.rounded(h, z.dtype, 2 * rel[:, None], wt[:, None] / tau ** 2 * (p + p * p)), "hess")


@pytest.mark.parametrize("K", [6, 90, 1200, 9001, 66000])
def test_policy_masks_and_extremes(pkg, K):
    rng = np.random.default_rng(K)
    n = 8
    z, _ = logits(rng, n, K, torch.float32)
    a = torch.from_numpy(rng.integers(2, K + 1, size=n).astype(np.int32))
    w = torch.ones(n)
    a[0] = 0; z[0] = float("nan")                                  # not counted
    w[1], z[1] = 0.0, float("inf")
    z[2, : K // 2] = NINF; z[2, a[2].long() - 1] = 0.0
    z[3] = torch.finfo(torch.float32).min; z[3, a[3].long() - 1] = 0.0  # certain: log p = 0
    a[4] = K + 1
    lp = torch.log_softmax(z.to(F8), 1).gather(1, (a.long() - 1).clamp(0, K - 1)[:, None])[:, 0].nan_to_num()
    old, adv, ref = (lp - 0.1).float(), torch.ones(n), (lp + 0.2).float()
    old[0] = adv[0] = ref[0] = float("nan")
    adv[5], adv[6] = -1.0, 0.0
    old[7] = (lp[7] - 1.0).float()                                 # clipped: no gradient from the advantage
    out = pkg.policy_grads(z.cuda(), a.cuda(), old.cuda(), adv.cuda(), ref_logp=ref.cuda(), w=w.cuda(), beta=0.5, hess=True)
    assert all((o[:2] == 0).all() for o in out) and all(torch.isnan(o[4]).all() for o in out)
    keep = [2, 3, 5, 6, 7]
    want = R.policy(z[keep], a[keep], old[keep], adv[keep], ref[keep], w[keep], 1.0, (0.2, 0.2), 0.5)
    rel = R.part(z[keep])
    R.close(out[0][keep], want[0], 4 * rel * want[4] + R.U * want[0].abs(), "loss")
    R.close(out[2][keep], want[2], R.rounded(want[2], torch.float32, 4 * rel[:, None], (want[4] + 1)[:, None]), "grad")
    R.close(out[3][keep], want[3], R.rounded(want[3], torch.float32, 2 * rel[:, None], 1.0), "hess")
    loss, logp, g = pkg.policy_grads(z[keep].cuda(), a[keep].cuda(), old[keep].cuda(), adv[keep].cuda())   # without the KL term
    assert (g[4] == 0).all() and abs(loss[4].item() + 1.2) < 1e-6


def lengths(rng, P, longest):
    lens = rng.integers(0, longest + 1, size=2 * P)
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def check_preference(pkg, z, zd, label, seq, ref=None, w=None, beta=0.3, smooth=0.0, mean=False):
    out = pkg.preference_grads(zd, label.cuda(), seq.cuda(), ref_logp=None if ref is None else ref.cuda(), w=None if w is None else w.cuda(), beta=beta,
                               smooth=smooth, mean=mean)
    loss, margin, logp, grad = R.preference(z, label, seq, ref, w, beta, smooth, mean)
    live = label > 0
    rel = torch.where(live, R.part(torch.where(live[:, None], z.float(), torch.zeros(()))) , torch.zeros((), dtype=F8))
    R.close(out[2], logp, rel + R.U * logp.abs(), "logp")
    P = loss.numel()
    n = z.shape[0]
    each = rel + R.U * (logp.abs() + (0 if ref is None else ref.to(F8).nan_to_num().abs()))
    dm = torch.tensor([float(each[int(seq[2 * p]):int(seq[2 * p + 2])].sum()) * beta for p in range(P)], dtype=F8)
    if mean:      # what a mean is off by is at most what its worst row is
        dm = torch.tensor([2 * beta * float(each[int(seq[2 * p]):int(seq[2 * p + 2])].max()) if seq[2 * p + 2] > seq[2 * p] else 0.0 for p in range(P)], dtype=F8)
    R.close(out[1], margin, dm + R.U * margin.abs(), "margin")
    wt = torch.ones(P, dtype=F8) if w is None else w.to(F8).nan_to_num()
    R.close(out[0], loss, wt * (dm + 8 * R.U * (1 + margin.abs())), "loss")
    size = torch.zeros(n, dtype=F8)
    off = torch.zeros(n, dtype=F8)
    for p in range(P):
        a, b = int(seq[2 * p]), int(seq[2 * p + 2])
        size[a:b], off[a:b] = wt[p] * beta, dm[p] + 16 * R.U
    p = torch.where(live[:, None], torch.softmax(torch.where(live[:, None], z.to(F8), torch.zeros((), dtype=F8)), 1), torch.zeros((), dtype=F8))
    onehot = torch.zeros_like(p).scatter_(1, (label.long() - 1).clamp(min=0)[:, None], 1.0) * live[:, None]
    R.close(out[3], grad, R.rounded(grad, z.dtype, (2 * rel + off)[:, None], size[:, None] * (p + onehot)), "grad")
    return out


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("K", [3, 30, 257, 2500, 20011, 70000, 300001])
def test_rows_far_away(pkg, K, dtype):
    """Rows whose largest prediction is the type's lowest value, or far from zero: what counts is the distance to it."""
    rng = np.random.default_rng(K)
    dt = DTYPES[dtype]
    low = torch.finfo(dt).min
    z = torch.full((5, K), low, dtype=dt)                       # row 0: nothing but masks
    z[1, : K // 2 + 1] = NINF
    z[2] = low / 2
    z[2, 0] = z[2, K - 1] = low / 4                             # two classes are far above the others
    z[3] = torch.from_numpy(rng.normal(size=K).astype(np.float32)).to(dt) + (1000.0 if dtype == "f16" else 3.0e4)
    z[4, K - 1] = -low                                          # and one is far above zero
    a = torch.tensor([1, K, K, 2, K], dtype=torch.int32)
    old, adv = torch.tensor([-np.log(K), -1.0, -0.5, -8.0, -0.1], dtype=torch.float32), torch.ones(5)
    for tau in (1.0, 1e-3):
        out = pkg.policy_grads(z.cuda(), a.cuda(), old.cuda(), adv.cuda(), tau=tau, clip=(1.0, 3.0e38), hess=True)
        loss, logp, grad, h, scale = R.policy(z, a, old, adv, None, None, tau, (1.0, 3.0e38))
        rel = R.part(z, tau) + 4 * R.U * logp.abs().nan_to_num()
        R.close(out[1], logp, rel + R.U * logp.abs(), "logp")
        R.close(out[2], grad, R.rounded(grad, dt, 4 * rel[:, None], 2 * (scale / tau)[:, None]), "grad")
        h = torch.where(h > torch.finfo(dt).max * (1 + torch.finfo(dt).eps / 4), torch.full_like(h, float("inf")), h)      # more than half a step beyond the type's largest number
        R.close(out[3], h, R.rounded(h, dt, 4 * rel[:, None], 2 / tau ** 2), "hess")
    ids = torch.tensor([[1, 2], [K, K - 1], [1, K], [3, 1], [K, 0]], dtype=torch.int32)
    t = torch.zeros((5, 2))
    check_distill(pkg.distill_grads(z[[0, 2, 3]].cuda(), ids[[0, 2, 3]].cuda(), t[[0, 2, 3]].cuda(), hess=True), z[[0, 2, 3]], ids[[0, 2, 3]], t[[0, 2, 3]], None,
                  1.0, False, True)
    one = pkg.preference_grads(z.cuda(), a.cuda(), torch.tensor([0, 1, 3], dtype=torch.int32).cuda())
    want = R.preference(z[:3], a[:3], torch.tensor([0, 1, 3]))
    R.close(one[2][:3], want[2], R.part(z[:3]) + R.U * want[2].abs(), "logp")
    R.close(one[3][:3], want[3], R.rounded(want[3], dt, 4 * R.part(z[:3])[:, None], 0.2), "grad")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("K", [k for k in CLASSES if k > 1])
def test_preference_sizes(pkg, K, dtype):
    rng = np.random.default_rng(K + 2)
    P, longest = (2, 3) if K > 300 else (9, 40)
    seq = lengths(rng, P, longest)
    n = max(1, int(seq[-1]))
    z, zd = logits(rng, n, K, DTYPES[dtype])
    label = torch.from_numpy(rng.integers(0, K + 1, size=n).astype(np.int32))
    ref = torch.from_numpy(-rng.random(n).astype(np.float32) * 8)
    check_preference(pkg, z, zd, label, torch.from_numpy(seq), ref, torch.from_numpy(rng.random(P).astype(np.float32)), smooth=0.1, mean=K % 2 == 0)


@pytest.mark.parametrize("K", [5, 300, 33000])
def test_preference_masks(pkg, K):
    """Empty sequences, sequences without a counted row, rows before, behind and between that do not count and hold NaN, a pair of weight 0."""
    rng = np.random.default_rng(K)
    seq = torch.tensor([2, 5, 5, 9, 9, 12, 13, 16, 18], dtype=torch.int32)      # pairs: (3, 0), (4, 0), (3, 1), (3, 2)
    n = 21
    z, _ = logits(rng, n, K, torch.float32)
    label = torch.from_numpy(rng.integers(1, K + 1, size=n).astype(np.int32))
    ref = torch.from_numpy(-rng.random(n).astype(np.float32))
    for i in (0, 1, 3, 9, 10, 11, 18, 19, 20):
        label[i], z[i], ref[i] = 0, float("nan"), float("nan")
    w = torch.tensor([1.0, 2.0, 0.5, 0.0])
    out = check_preference(pkg, z, z.cuda(), label, seq, ref, w)
    assert (out[3][[0, 1, 3, 9, 10, 11, 16, 17, 18, 19, 20]] == 0).all() and out[0][3] == 0
    # rows that count but lie outside of all sequences
    label[19] = 1; z[19] = 0.0; ref[19] = 0.0
    out2 = pkg.preference_grads(z.cuda(), label.cuda(), seq.cuda(), ref_logp=ref.cuda(), w=w.cuda(), beta=0.3)
    assert (out2[3][19] == 0).all() and torch.equal(out2[3][:18], out[3][:18])
    # a label that there is not: NaN for its pair, not for the others
    label[6] = K + 5
    out3 = pkg.preference_grads(z.cuda(), label.cuda(), seq.cuda(), ref_logp=ref.cuda(), w=w.cuda(), beta=0.3)
    assert torch.isnan(out3[0][1]) and torch.isnan(out3[3][6]).all() and torch.equal(out3[0][[0, 2, 3]], out[0][[0, 2, 3]])
    assert torch.equal(out3[3][9:18], out[3][9:18]) and torch.equal(out3[3][:5], out[3][:5])


def test_preference_long_sequences(pkg):
    rng = np.random.default_rng(5)
    for P, longest, mean in ((1, 3000, False), (300, 9, True), (3, 1, False)):
        seq = lengths(rng, P, longest)
        n, K = max(1, int(seq[-1])), 11
        z, zd = logits(rng, n, K, torch.float32)
        label = torch.from_numpy(rng.integers(0, K + 1, size=n).astype(np.int32))
        check_preference(pkg, z, zd, label, torch.from_numpy(seq), None, None, beta=0.02, mean=mean)


@pytest.mark.parametrize("K", [5, 18, 37, 64, 200, 1000, 1003, 4099, 20001, 131072])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("pad,shift", [(3, 0), (8, 8), (1, 3), (5, 1)])
def test_strides_and_alignment(pkg, K, dtype, pad, shift):
    """Rows apart by more than their classes, that begin anywhere: the same bits as rows that are packed, or as good."""
    rng = np.random.default_rng(K)
    n = 5
    z, zd = logits(rng, n, K, DTYPES[dtype], pad, shift)
    ids, t = slots(rng, n, K, min(K, 4))
    out = pkg.distill_grads(zd, ids.cuda(), t.cuda(), hess=True)
    check_distill(out, z, ids, t, None, 1.0, False, True)
    lt = log_probs(t, 0.9)
    check_distill(pkg.distill_grads(zd, ids.cuda(), lt.cuda(), tail=True), z, ids, lt, None, 1.0, True, False)
    check_policy(pkg, rng, z, zd, 1.0, 0.1, True)
    label = torch.from_numpy(rng.integers(0, K + 1, size=n).astype(np.int32))
    check_preference(pkg, z, zd, label, torch.tensor([0, 1, 3, 4, 5], dtype=torch.int32))


@pytest.mark.parametrize("K", [5, 40, 700, 5003, 40000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_output_strides_write_nothing_else(pkg, K, dtype):
    """Gradient and hessian with their own strides, through the C entry: the gaps stay as they were."""
    from evotrees_b200 import _lib
    rng = np.random.default_rng(K)
    n, dt = 6, DTYPES[dtype]
    z, zd = logits(rng, n, K, dt)
    ids, t = slots(rng, n, K, min(K, 3))
    want = pkg.distill_grads(zd, ids.cuda(), t.cuda(), hess=True)
    for ld, off in ((2 * K + 1, 0), (K + 8, 8), (K + 3, 1)):
        g = torch.full((n * ld + off + 1,), 77.0, dtype=dt, device="cuda")
        h = torch.full((n * ld + off + 1,), 78.0, dtype=dt, device="cuda")
        loss = torch.empty(n, device="cuda")
        idd, td = ids.cuda(), t.cuda()
        _lib.check(_lib.lib().evb_distill_grads(0, 0, zd.data_ptr(), _lib.EVB_F32 if dtype == "f32" else _lib.EVB_BF16, n, K, K, idd.data_ptr(), td.data_ptr(),
                                                _lib.EVB_F32, t.shape[1], 0, None, 1.0, loss.data_ptr(), g[off:].data_ptr(), ld, h[off:].data_ptr(), ld, None))
        torch.cuda.synchronize()
        for buf, w, mark in ((g, want[1], 77.0), (h, want[2], 78.0)):
            body = buf[off:off + n * ld].view(n, ld)
            assert torch.allclose(body[:, :K].float(), w.float(), rtol=2 * R.half_step(dt) + 1e-5, atol=1e-7)
            assert (body[:, K:] == mark).all() and (buf[:off] == mark).all() and (buf[off + n * ld:] == mark).all()
        assert torch.allclose(loss, want[0], rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("K", [4, 60, 600, 6000])
def test_gradients_against_differences(pkg, K):
    """Central differences of the calls' own losses: off by delta^2 / 6 of a third derivative (below 1 for these) and by what the losses' errors
    make of a division by 2 delta."""
    rng = np.random.default_rng(K)
    delta, n = 2.0 ** -5, 1
    z, _ = logits(rng, n, K, torch.float32)
    ids, t = slots(rng, n, K, 3, empty=0.0)
    a = torch.tensor([2], dtype=torch.int32)
    lp = torch.log_softmax(z, 1)[:, 1]
    label, seq = torch.tensor([1, 2, 3, 0, 1], dtype=torch.int32), torch.tensor([0, 2, 5], dtype=torch.int32)
    at = [int(ids[0, 0]) - 1, int(ids[0, 1]) - 1, 1, K - 1, int(z[0].argmax())]
    many = z.repeat(2 * len(at), 1)
    for j, k in enumerate(at):
        many[2 * j, k] += delta
        many[2 * j + 1, k] -= delta
    N = many.shape[0]
    step = lambda v, j: float((v[2 * j].double() - v[2 * j + 1].double())) / (2 * delta)     # noqa: E731
    rep = lambda v: v.repeat(*([N] + [1] * (v.dim() - 1))).cuda()                            # noqa: E731
    tol = delta ** 2 / 6 * 4 + 1e-5 / (2 * delta)
    for tail in (False, True):
        tt = log_probs(t, 0.9) if tail else t
        g = pkg.distill_grads(z.cuda(), ids.cuda(), tt.cuda(), tail=tail)[1]
        v = pkg.distill_grads(many.cuda(), rep(ids), rep(tt), tail=tail, grads=False)[0]
        for j, k in enumerate(at):
            assert abs(step(v, j) - g[0, k].item()) < tol
    for adv, shift in ((1.0, 0.02), (-1.0, 0.02), (1.0, 0.5)):       # the last: clipped
        old = lp - shift
        args = dict(beta=0.3, clip=(0.3, 0.3))
        g = pkg.policy_grads(z.cuda(), a.cuda(), old.cuda(), torch.tensor([adv]).cuda(), ref_logp=(lp + 0.4).cuda(), **args)[2]
        v = pkg.policy_grads(many.cuda(), rep(a), rep(old), torch.full((N,), adv).cuda(), ref_logp=rep(lp + 0.4), grads=False, **args)[0]
        for j, k in enumerate(at):
            assert abs(step(v, j) - g[0, k].item()) < tol
    rows = torch.from_numpy(rng.normal(size=(5, K)).astype(np.float32))
    g = pkg.preference_grads(rows.cuda(), label.cuda(), seq.cuda(), beta=0.7)[3]
    for i, k in ((0, 0), (0, 1), (1, K - 1), (2, 2), (4, 0), (3, 1)):
        v = []
        for d in (delta, -delta):
            r2 = rows.clone(); r2[i, k] += d
            v.append(pkg.preference_grads(r2.cuda(), label.cuda(), seq.cuda(), beta=0.7, grads=False)[0])
        assert abs(float(v[0].double() - v[1].double()) / (2 * delta) - g[i, k].item()) < tol


@pytest.mark.parametrize("K", [5, 100, 3000, 100000])
def test_losses_without_gradients_are_the_same(pkg, K):
    rng = np.random.default_rng(K)
    z, zd = logits(rng, 5, K, torch.bfloat16)
    ids, t = slots(rng, 5, K, 3)
    assert torch.equal(pkg.distill_grads(zd, ids.cuda(), t.cuda(), grads=False)[0], pkg.distill_grads(zd, ids.cuda(), t.cuda())[0])
    a, v = torch.ones(5, dtype=torch.int32).cuda(), torch.ones(5).cuda()
    one, two = pkg.policy_grads(zd, a, -v, v, grads=False), pkg.policy_grads(zd, a, -v, v)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    seq = torch.tensor([0, 2, 5], dtype=torch.int32).cuda()
    one, two = pkg.preference_grads(zd, a, seq, grads=False), pkg.preference_grads(zd, a, seq)
    assert all(torch.equal(x, y) for x, y in zip(one, two))


def test_no_rows_and_no_pairs(pkg):
    z = torch.empty((0, 7), device="cuda")
    i, f = torch.empty(0, dtype=torch.int32, device="cuda"), torch.empty(0, device="cuda")
    assert [tuple(o.shape) for o in pkg.distill_grads(z, i.view(0, 1).expand(0, 2).contiguous(), f.view(0, 1).expand(0, 2).contiguous())] == [(0,), (0, 7)]
    assert [tuple(o.shape) for o in pkg.policy_grads(z, i, f, f, hess=True)] == [(0,), (0,), (0, 7), (0, 7)]
    seq = torch.zeros(3, dtype=torch.int32, device="cuda")
    loss, margin, logp, g = pkg.preference_grads(z, i, seq)
    assert margin.tolist() == [0.0] and abs(loss[0].item() - np.log(2.0)) < 1e-6 and g.shape == (0, 7)
    z = torch.randn((4, 7), device="cuda")
    loss, margin, logp, g = pkg.preference_grads(z, torch.ones(4, dtype=torch.int32, device="cuda"), seq[:1])
    assert loss.shape == (0,) and (g == 0).all()
    torch.cuda.synchronize()


def test_equal_calls_give_equal_bits_in_graphs_and_on_streams(pkg):
    """Captured and replayed with other inputs, two graphs and two streams at the same time."""
    rng = np.random.default_rng(3)
    jobs = []
    for K, dt in ((5, torch.float32), (700, torch.bfloat16), (33000, torch.bfloat16)):
        n = 40
        zs = [logits(rng, n, K, dt)[1] for _ in range(2)]
        ids, t = slots(rng, n, K, 3)
        ids, t = ids.cuda(), t.cuda()
        a = torch.from_numpy(rng.integers(0, K + 1, size=n).astype(np.int32)).cuda()
        v = torch.from_numpy(rng.normal(size=n).astype(np.float32)).cuda()
        seq = torch.tensor([0, 11, 20, 32, 38], dtype=torch.int32).cuda()
        jobs.append((zs, lambda z, ids=ids, t=t, a=a, v=v, seq=seq: [*pkg.distill_grads(z, ids, t), *pkg.policy_grads(z, a, v - 3, v, ref_logp=v - 2, beta=0.1),
                                                                    *pkg.preference_grads(z, a, seq, ref_logp=v)]))
    torch.cuda.synchronize()
    plain = [[job(z) for z in zs] for zs, job in jobs]
    graphs = []
    for zs, job in jobs:
        z = zs[0].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = job(z)
        graphs.append((g, z, out))
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(3):
        for which in (1, 0):
            torch.cuda.synchronize()
            for (g, z, out), (zs, _), s in zip(graphs, jobs, streams):
                with torch.cuda.stream(s):
                    z.copy_(zs[which])
                    g.replay()
            torch.cuda.synchronize()
            for (g, z, out), want in zip(graphs, plain):
                for o, e in zip(out, want[which]):
                    assert torch.equal(torch.nan_to_num(o, nan=-7.0), torch.nan_to_num(e, nan=-7.0))
    with torch.cuda.stream(streams[0]):
        again = jobs[1][1](jobs[1][0][0])
    torch.cuda.synchronize()
    assert all(torch.equal(torch.nan_to_num(x, nan=-7.0), torch.nan_to_num(y, nan=-7.0)) for x, y in zip(again, plain[1][0]))


def test_offsets_beyond_32_bits(pkg):
    """More than 2^31 elements: the last rows are as good as the first."""
    K, n = 65600, 33000                                            # 2.16e9 elements of 2 bytes
    z = torch.empty((n, K), dtype=torch.bfloat16, device="cuda")
    for i in range(0, n, 3300):
        z[i:i + 3300].normal_()
    z[-1] = z[0]
    a = torch.full((n,), 17, dtype=torch.int32, device="cuda")
    v = torch.ones(n, device="cuda")
    loss, logp, g = pkg.policy_grads(z, a, -10 * v, v)
    assert torch.equal(g[-1], g[0]) and loss[-1] == loss[0]
    want = R.policy(z[-1:].cpu(), a[-1:].cpu(), -10 * v[-1:].cpu(), v[-1:].cpu())
    R.close(logp[-1:], want[1], R.part(z[-1:].cpu()) + 16 * R.U, "logp")
    ids = torch.full((n, 1), 17, dtype=torch.int32, device="cuda")
    l2, g2 = pkg.distill_grads(z, ids, v[:, None].contiguous())
    assert torch.equal(g2[-1], g2[0]) and l2[-1] == l2[0] and abs(l2[0].item() + logp[0].item()) < 1e-4

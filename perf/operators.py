"""The losses on rows of raw predictions -- distillation from a teacher's top logits, the clipped policy loss with a KL term, the
preference loss of paired log ratios -- as cases that can be timed and compared.

A case is one call of one of them: the loss and its gradient (for boosting also its hessian) on [rows, classes] raw predictions that
live on the GPU.  Two kinds of sizes: rows of a table with a few classes, as boosting rounds have them (float32, with hessians), and
rows of tokens over a vocabulary, as fine-tuning has them (16 bits mostly).  Class codes are 1..classes, 0 names none.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
NINF = float("-inf")


def _distill(**kw):
    return {"op": "distill", "dtype": "f32", "hess": False, "tail": False, "tau": 1.0, "masked": 0, "weights": False, **kw}


def _policy(**kw):
    return {"op": "policy", "dtype": "f32", "hess": False, "tau": 1.0, "low": 0.2, "high": 0.2, "beta": 0.05, "masked": 0, "ref": True, **kw}


def _preference(**kw):
    return {"op": "preference", "dtype": "f32", "beta": 0.1, "smooth": 0.0, "mean": False, "ref": True, "weights": False, "lens": 1, **kw}


def listed():
    return [
        # one boosting round's gradients on the package's smallest table: latency
        {"name": "distill_1503_x5", **_distill(rows=1503, classes=5, top=3, hess=True, weights=True, tau=2.0)},
        # the same at the size of the package's softmax benchmark (2M rows, five classes)
        {"name": "distill_2M_x5", **_distill(rows=2_000_000, classes=5, top=3, hess=True)},
        # a few hundred labels (tags, intents): rows that a warp can hold
        {"name": "distill_100k_x200", **_distill(rows=100_003, classes=200, top=10, tau=2.0)},
        # a batch of tokens, odd vocabulary, half precision, softened teacher
        {"name": "distill_777_x50021_f16", **_distill(rows=777, classes=50_021, top=20, dtype="f16", tau=2.0, masked=48)},
        # a batch of tokens against stored log-probabilities of the teacher's best 64, the rest as one class: the largest
        {"name": "distill_4096_x131072_tail", **_distill(rows=4096, classes=131_072, top=64, dtype="bf16", tail=True, masked=256)},
        # the last few tokens of an episode: latency
        {"name": "policy_16_x32768", **_policy(rows=16, classes=32_768, dtype="bf16")},
        # a tabular policy with 18 actions, one boosting round
        {"name": "policy_1M_x18", **_policy(rows=1_000_000, classes=18, hess=True, beta=0.0, ref=False)},
        # a middle-sized action space, float32
        {"name": "policy_20k_x1000", **_policy(rows=20_011, classes=1000, high=0.28, masked=2000)},
        # a rollout batch over an odd vocabulary, a tenth of it padding
        {"name": "policy_8192_x65537", **_policy(rows=8192, classes=65_537, dtype="bf16", masked=819)},
        # two short pairs: latency
        {"name": "preference_2_x1021", **_preference(pairs=2, longest=32, classes=1021, weights=True)},
        # an ordinary micro-batch
        {"name": "preference_16_x32768", **_preference(pairs=16, longest=256, classes=32_768, dtype="bf16")},
        # a long batch over a large vocabulary
        {"name": "preference_8_x131072", **_preference(pairs=8, longest=512, classes=131_072, dtype="bf16", smooth=0.1)},
    ]


LARGEST = 4096 * 131_072      # elements of the largest case


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["distill", "policy", "preference"])
    boost = op != "preference" and rng.random() < 0.4
    if boost:
        classes, rows, dtype = _log_uniform(rng, 2, 32), _log_uniform(rng, 100, 2_000_000), "f32"
    else:
        classes, dtype = _log_uniform(rng, 33, 131_072), rng.choice(["f32", "bf16", "bf16", "f16"])
        rows = _log_uniform(rng, 1, min(200_000, LARGEST * 2 // (classes * SIZES[dtype])))
    if op == "distill":
        tail = rng.random() < 0.4
        return _distill(rows=rows, classes=classes, dtype=dtype, hess=boost, top=_log_uniform(rng, 1, min(classes, 128)), tail=tail,
                        tau=1.0 if tail else rng.choice([1.0, 2.0, 1.5]), masked=0 if boost else rows // rng.choice([7, 16]), weights=boost)
    if op == "policy":
        return _policy(rows=rows, classes=classes, dtype=dtype, hess=boost, high=rng.choice([0.2, 0.28]), beta=rng.choice([0.0, 0.01, 0.1]),
                       masked=0 if boost else rows // rng.choice([5, 10]), ref=True)
    longest = _log_uniform(rng, 1, 512)
    pairs = _log_uniform(rng, 1, max(1, min(2000, rows // (2 * longest))))
    if 2 * pairs * longest * classes * SIZES[dtype] > 2 * LARGEST:
        longest = max(1, 2 * LARGEST // (2 * pairs * classes * SIZES[dtype]))
    return _preference(pairs=pairs, longest=longest, classes=classes, dtype=dtype, smooth=rng.choice([0.0, 0.1]), mean=rng.random() < 0.3,
                       weights=rng.random() < 0.5, lens=rng.randrange(1 << 20))


def _lengths(case):
    """Rows of every sequence and how many of them, its first ones, are prompt (not counted)."""
    r, top = random.Random(case["lens"]), case["longest"]
    lens = [r.randint((top + 1) // 2, top) for _ in range(2 * case["pairs"])]
    return lens, [n // 4 for n in lens]


def _rows(case):
    return sum(_lengths(case)[0]) if case["op"] == "preference" else case["rows"]


def _counted(case):
    if case["op"] == "preference":
        lens, prompt = _lengths(case)
        return sum(lens) - sum(prompt)
    return case["rows"] - case["masked"]


def work(case):
    """Rows that count are read once, every row of the gradient (and hessian) is written once; four operations an element: the
    difference, the exponential, the sum and the product."""
    n, counted, K, e = _rows(case), _counted(case), case["classes"], SIZES[case["dtype"]]
    nbytes = counted * K * e + n * K * e * (2 if case["hess"] else 1) if case["op"] != "preference" else counted * K * e + n * K * e
    if case["op"] == "distill":
        nbytes += n * case["top"] * (4 + e) + 8 * n
    elif case["op"] == "policy":
        nbytes += n * (4 * (5 if case["ref"] else 4) + 8)
    else:
        nbytes += n * 12 + 4 * (4 * case["pairs"] + 1) + 8 * case["pairs"]
    return {"bytes": nbytes, "flops": 4 * counted * K}


# ---------------------------------------------------------------------------------------------------------------- inputs
def _logits(n, K, dtype, gen, scale=2.0):
    """Raw predictions: a bell with a few classes standing out in every row, as trained models give them."""
    out = torch.empty((n, K), dtype=dtype, device="cuda")
    step = max(1, (1 << 28) // K)
    for i in range(0, n, step):
        rows = out[i:i + step]
        v = torch.randn(rows.shape, generator=gen, device="cuda") * scale
        peaks = torch.randint(0, K, (rows.shape[0], 4), generator=gen, device="cuda")
        v.scatter_add_(1, peaks, 4.0 + 3.0 * torch.rand(peaks.shape, generator=gen, device="cuda"))
        rows.copy_(v)
    return out


def _logp_of(z, code):
    """log p of the class `code` (1..K) of every row, in 32 bits, block by block."""
    out = torch.empty(z.shape[0], device="cuda")
    step = max(1, (1 << 28) // z.shape[1])
    for i in range(0, z.shape[0], step):
        x = z[i:i + step].float()
        out[i:i + step] = x.gather(1, (code[i:i + step].long() - 1)[:, None])[:, 0] - torch.logsumexp(x, 1)
    return out


def _some_code(z, gen):
    """The likeliest of 64 random classes of every row: what a sampler would have taken."""
    n, K = z.shape
    cand = torch.randint(0, K, (n, min(64, K)), generator=gen, device="cuda")
    return (cand.gather(1, z.gather(1, cand).float().argmax(1, keepdim=True))[:, 0] + 1).int()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    n, K, dtype = _rows(case), case["classes"], DTYPES[case["dtype"]]
    z = _logits(n, K, dtype, gen)
    st = {"case": case, "z": z}
    if own:
        import __graft_entry__
        st["evo"] = __graft_entry__.load_package()

    def masked_weights():
        w = None
        if case.get("masked"):
            w = torch.ones(n, device="cuda")
            w[torch.randperm(n, generator=gen, device="cuda")[:case["masked"]]] = 0.0
        elif case.get("weights"):
            w = 0.5 + torch.rand(n, generator=gen, device="cuda")
        return w

    if case["op"] == "distill":
        T = case["top"]
        ids = torch.empty((n, T), dtype=torch.int32, device="cuda")
        teacher = torch.empty((n, T), dtype=dtype, device="cuda")
        step = max(1, (1 << 27) // K)
        for i in range(0, n, step):     # the teacher agrees with the student more or less
            x = z[i:i + step].float() * 0.8 + torch.randn((min(step, n - i), K), generator=gen, device="cuda")
            if case["tail"]:
                x = torch.log_softmax(x, 1)
            v, k = x.topk(T, 1)
            ids[i:i + step], teacher[i:i + step] = (k + 1).int(), v.to(dtype)
        # a tenth of the rows were stored with fewer entries
        short = torch.rand(n, generator=gen, device="cuda") < 0.1
        keep = torch.randint(1, T + 1, (n, 1), generator=gen, device="cuda")
        ids[short[:, None] & (torch.arange(T, device="cuda")[None, :] >= keep)] = 0
        st.update(ids=ids, teacher=teacher, w=masked_weights())
    elif case["op"] == "policy":
        action = _some_code(z, gen)
        lp = _logp_of(z, action)
        ratio = 0.25 * torch.randn(n, generator=gen, device="cuda")     # of the present policy to the one that acted, its logarithm
        # the gradient jumps where the clip begins: a ratio that sits on the border to seven digits is a coin toss for any arithmetic
        for edge in (math.log1p(case["high"]), math.log1p(-case["low"])):
            ratio = torch.where((ratio - edge).abs() < 2e-3, torch.full_like(ratio, edge + 4e-3), ratio)
        w = masked_weights()
        if w is not None:
            action = torch.where(w > 0, action, torch.zeros_like(action))
        st.update(action=action, old=lp - ratio, adv=torch.randn(n, generator=gen, device="cuda"), w=w,
                  ref=lp + 0.3 * torch.randn(n, generator=gen, device="cuda") if case["ref"] else None)
    else:
        lens, prompt = _lengths(case)
        label = _some_code(z, gen)
        ref = _logp_of(z, label) + 0.2 * torch.randn(n, generator=gen, device="cuda")
        seq = np.concatenate([[0], np.cumsum(lens)])
        drop = np.concatenate([np.arange(a, a + p) for a, p in zip(seq[:-1], prompt)]).astype(np.int64)
        label[torch.from_numpy(drop).cuda()] = 0
        st.update(label=label, seq=torch.from_numpy(seq.astype(np.int32)).cuda(), ref=ref if case["ref"] else None,
                  w=0.5 + torch.rand(case["pairs"], generator=gen, device="cuda") if case["weights"] else None)
    torch.cuda.synchronize()
    return st


# ---------------------------------------------------------------------------------------------------------------- the plain forms
def _softmax_parts(x):
    m = x.max(1, keepdim=True).values
    e = torch.exp(x - m)
    s = e.sum(1, keepdim=True)
    return e / s, m + torch.log(s)


def _plain_distill(c, z, ids, teacher, w):
    n, K = z.shape
    x = z.float() / c["tau"]
    p, lse = _softmax_parts(x)
    t = teacher.float() / c["tau"]
    named = (ids > 0) & (t > NINF)
    k = (ids.long() - 1).clamp(min=0)
    t = torch.where(named, t, torch.full_like(t, NINF))
    if c["tail"]:
        q = torch.exp(t)
        qt = (1.0 - q.sum(1, keepdim=True)).clamp(min=0.0)
    else:
        tm = t.max(1, keepdim=True).values
        q = torch.exp(t - torch.where(tm > NINF, tm, torch.zeros_like(tm)))
        q = torch.where(named, q / q.sum(1, keepdim=True), torch.zeros_like(q))
        qt = torch.zeros_like(lse)
    xlogx = lambda v: torch.where(v > 0, v * torch.log(torch.where(v > 0, v, torch.ones_like(v))), torch.zeros_like(v))   # noqa: E731
    logp = x.gather(1, k) - lse
    loss = (xlogx(q) - torch.where(q > 0, q * logp, torch.zeros_like(q))).sum(1, keepdim=True)
    # the named classes' probabilities; slots that name none add to a spare column
    spare = torch.zeros((n, K + 1), device=z.device)
    named_q = spare.scatter_add(1, torch.where(named, k, torch.full_like(k, K)), torch.where(named, q, torch.zeros_like(q)))[:, :K]
    factor = q.sum(1, keepdim=True) + qt
    grad = factor * p - named_q
    if c["tail"]:
        is_named = spare.scatter(1, torch.where(named, k, torch.full_like(k, K)), 1.0)[:, :K] > 0
        rest = torch.where(is_named, torch.full_like(x, NINF), x)
        rp, rlse = _softmax_parts(torch.where(torch.isinf(rest).all(1, keepdim=True), torch.zeros_like(rest), rest))
        some = (~is_named).any(1, keepdim=True)
        qt = torch.where(some, qt, torch.zeros_like(qt))
        factor = q.sum(1, keepdim=True) + qt
        loss = loss + torch.where(qt > 0, xlogx(qt) - qt * (rlse - lse), torch.zeros_like(qt))
        grad = factor * p - named_q - torch.where(is_named, torch.zeros_like(rp), qt * rp)
    wt = torch.ones((n, 1), device=z.device) if w is None else w[:, None]
    live = (wt != 0) & named.any(1, keepdim=True)
    zero = torch.zeros((), device=z.device)
    out = [torch.where(live, wt * c["tau"] ** 2 * loss, zero)[:, 0], torch.where(live, wt * c["tau"] * grad, zero).to(z.dtype)]
    if c["hess"]:
        out.append(torch.where(live, wt * p * (1.0 - p), zero).to(z.dtype))
    return out


def _plain_policy(c, z, action, old, adv, ref, w):
    x = z.float() / c["tau"]
    p, lse = _softmax_parts(x)
    k = (action.long() - 1).clamp(min=0)[:, None]
    lp = (x.gather(1, k) - lse)[:, 0]
    r = torch.exp(lp - old)
    u, cl = r * adv, r.clamp(1.0 - c["low"], 1.0 + c["high"]) * adv
    loss, d = -torch.minimum(u, cl), torch.where(u <= cl, -u, torch.zeros_like(u))
    if ref is not None:
        kl = ref - lp
        loss, d = loss + c["beta"] * (torch.exp(kl) - kl - 1.0), d + c["beta"] * (1.0 - torch.exp(kl))
    wt = torch.ones_like(lp) if w is None else w
    live, zero = (action > 0) & (wt != 0), torch.zeros((), device=z.device)
    onehot = torch.zeros_like(x).scatter_(1, k, 1.0)
    out = [torch.where(live, wt * loss, zero), torch.where(live, lp, zero),
           torch.where(live[:, None], (wt * d / c["tau"])[:, None] * (onehot - p), zero).to(z.dtype)]
    if c["hess"]:
        out.append(torch.where(live[:, None], wt[:, None] * p * (1.0 - p) / c["tau"] ** 2, zero).to(z.dtype))
    return out


def _plain_preference(c, z, label, seq, ref, w):
    x = z.float()
    p, lse = _softmax_parts(x)
    k = (label.long() - 1).clamp(min=0)[:, None]
    counted = label > 0
    lp = torch.where(counted, (x.gather(1, k) - lse)[:, 0], torch.zeros((), device=z.device))
    ratio = torch.where(counted, lp.double() - (0.0 if ref is None else ref.double()), torch.zeros((), dtype=torch.float64, device=z.device))
    S, n = seq.numel() - 1, z.shape[0]
    of = torch.searchsorted(seq[1:].contiguous(), torch.arange(n, dtype=torch.int32, device=z.device), right=True)
    inside = of < S
    of = of.clamp(max=S - 1)
    live = counted & inside
    D = torch.zeros(S, dtype=torch.float64, device=z.device).index_add_(0, of, torch.where(live, ratio, torch.zeros_like(ratio)))
    share = torch.ones(S, device=z.device)
    if c["mean"]:
        share = 1.0 / torch.zeros(S, device=z.device).index_add_(0, of, live.float()).clamp(min=1.0)
        D = D * share.double()
    m = (c["beta"] * (D[0::2] - D[1::2])).float()
    wt = torch.ones_like(m) if w is None else w
    softplus = lambda v: v.clamp(min=0.0) + torch.log1p(torch.exp(-v.abs()))    # noqa: E731
    sigma = lambda v: 1.0 / (1.0 + torch.exp(-v))                               # noqa: E731
    e = c["smooth"]
    loss = wt * ((1.0 - e) * softplus(-m) + e * softplus(m))
    dm = wt * (e * sigma(m) - (1.0 - e) * sigma(-m))
    coef = torch.stack([dm, -dm], 1).reshape(-1) * c["beta"] * share
    onehot = torch.zeros_like(x).scatter_(1, k, 1.0)
    grad = torch.where(live[:, None], coef[of][:, None] * (onehot - p), torch.zeros((), device=z.device)).to(z.dtype)
    return [loss, m, lp, grad]


def run(st):
    c, z = st["case"], st["z"]
    if c["op"] == "distill":
        if own:
            return st["evo"].distill_grads(z, st["ids"], st["teacher"], w=st["w"], tau=c["tau"], tail=c["tail"], hess=c["hess"])
        return _plain_distill(c, z, st["ids"], st["teacher"], st["w"])
    if c["op"] == "policy":
        if own:
            return st["evo"].policy_grads(z, st["action"], st["old"], st["adv"], ref_logp=st["ref"], w=st["w"], tau=c["tau"],
                                          clip=(c["low"], c["high"]), beta=c["beta"], hess=c["hess"])
        return _plain_policy(c, z, st["action"], st["old"], st["adv"], st["ref"], st["w"])
    if own:
        return st["evo"].preference_grads(z, st["label"], st["seq"], ref_logp=st["ref"], w=st["w"], beta=c["beta"], smooth=c["smooth"], mean=c["mean"])
    return _plain_preference(c, z, st["label"], st["seq"], st["ref"], st["w"])


# ---------------------------------------------------------------------------------------------------------------- in 64 bits
def _blocks(n, K):
    step = max(1, (1 << 27) // K)
    return [(i, min(n, i + step)) for i in range(0, n, step)]


def exact(case, seed):
    """The definitions in 64 bits, block of rows by block of rows."""
    st = prepare(case, seed)
    z, n, K = st["z"], st["z"].shape[0], case["classes"]
    f8 = dict(dtype=torch.float64, device="cuda")
    grad = torch.zeros((n, K), **f8)
    if case["op"] == "preference":
        label = st["label"].long()
        lp = torch.zeros(n, **f8)
        for a, b in _blocks(n, K):
            logp = torch.log_softmax(z[a:b].double(), 1)
            lp[a:b] = torch.where(label[a:b] > 0, logp.gather(1, (label[a:b] - 1).clamp(min=0)[:, None])[:, 0], torch.zeros((), **f8))
        seq, mean = st["seq"].tolist(), case["mean"]
        diff = lp if st["ref"] is None else torch.where(label > 0, lp - st["ref"].double(), torch.zeros((), **f8))
        total, share = [], []
        for s in range(2 * case["pairs"]):
            part = slice(seq[s], seq[s + 1])
            share.append(1.0 / max(1, int((label[part] > 0).sum())) if mean else 1.0)
            total.append(float(diff[part].sum()) * share[-1])
        loss, margin = [], []
        for p in range(case["pairs"]):
            m, w, e = case["beta"] * (total[2 * p] - total[2 * p + 1]), 1.0 if st["w"] is None else float(st["w"][p]), case["smooth"]
            up, down = 1.0 / (1.0 + math.exp(-m)), 1.0 / (1.0 + math.exp(m))
            loss.append(-w * ((1.0 - e) * math.log(up) + e * math.log(down)))
            margin.append(m)
            slope = case["beta"] * w * (e * up - (1.0 - e) * down)
            for s, sign in ((2 * p, 1.0), (2 * p + 1, -1.0)):
                for a, b in _blocks(seq[s + 1] - seq[s], K):
                    a, b = a + seq[s], b + seq[s]
                    rows = (label[a:b] > 0).nonzero()[:, 0]
                    if rows.numel():
                        g = -torch.softmax(z[a:b][rows].double(), 1)
                        g[torch.arange(rows.numel(), device="cuda"), label[a:b][rows] - 1] += 1.0
                        grad[a + rows] = g * (sign * slope * share[s])
        return [torch.tensor(loss, **f8), torch.tensor(margin, **f8), lp, grad]
    w = torch.ones(n, **f8) if st["w"] is None else st["w"].double()
    loss, tau = torch.zeros(n, **f8), case["tau"]
    hess = torch.zeros((n, K), **f8) if case["hess"] else None
    if case["op"] == "policy":
        out_lp = torch.zeros(n, **f8)
        for a, b in _blocks(n, K):
            act = st["action"][a:b].long()
            use = (act > 0) & (w[a:b] != 0)
            act = (act - 1).clamp(min=0)[:, None]
            logp = torch.log_softmax(z[a:b].double() / tau, 1)
            lp = logp.gather(1, act)[:, 0]
            ratio, A = (lp - st["old"][a:b].double()).exp(), st["adv"][a:b].double()
            inner = torch.where(A >= 0, ratio < 1.0 + case["high"], ratio > 1.0 - case["low"])      # where the unclipped side counts
            side = torch.where(A >= 0, torch.full_like(A, 1.0 + case["high"]), torch.full_like(A, 1.0 - case["low"]))
            value, slope = torch.where(inner, -ratio * A, -side * A), torch.where(inner, -ratio * A, torch.zeros((), **f8))
            if st["ref"] is not None:
                gap = st["ref"][a:b].double() - lp
                value, slope = value + case["beta"] * (gap.expm1() - gap), slope - case["beta"] * gap.expm1()
            wu = torch.where(use, w[a:b], torch.zeros((), **f8))
            loss[a:b], out_lp[a:b] = wu * value, torch.where(use, lp, torch.zeros((), **f8))
            prob = logp.exp()
            grad[a:b] = -prob * (wu * slope / tau)[:, None]
            grad[a:b].scatter_add_(1, act, (wu * slope / tau)[:, None])
            if hess is not None:
                hess[a:b] = prob * (1.0 - prob) * (wu / tau ** 2)[:, None]
        return [loss, out_lp, grad] + ([hess] if hess is not None else [])
    for a, b in _blocks(n, K):
        code, t = st["ids"][a:b].long(), st["teacher"][a:b].double() / tau
        use = (code > 0) & (t > NINF)
        target = torch.zeros((b - a, K + 1), **f8)      # the teacher's probability of every class; column 0: none
        code = torch.where(use, code, torch.zeros_like(code))
        q = t.masked_fill(~use, NINF)
        q = q.exp() if case["tail"] else torch.nan_to_num(torch.softmax(q, 1), nan=0.0)
        target.scatter_add_(1, code, torch.where(use, q, torch.zeros((), **f8)))
        target = target[:, 1:]
        named = torch.zeros((b - a, K + 1), dtype=torch.bool, device="cuda").scatter_(1, code, True)[:, 1:]
        logp = torch.log_softmax(z[a:b].double() / tau, 1)
        prob = logp.exp()
        value = (torch.special.xlogy(target, target) - torch.where(target > 0, target * logp, torch.zeros((), **f8))).sum(1)
        mass = target.sum(1)
        g = prob * mass[:, None] - target
        if case["tail"]:
            other = (1.0 - mass).clamp(min=0.0) * (~named).any(1)
            rest = logp.masked_fill(named, NINF).logsumexp(1)
            value = value + torch.where(other > 0, torch.special.xlogy(other, other) - other * rest, torch.zeros((), **f8))
            g = g + prob * other[:, None] - torch.where(named, torch.zeros((), **f8), (logp - rest[:, None]).exp() * other[:, None])
        wu = torch.where(use.any(1), w[a:b], torch.zeros((), **f8))
        loss[a:b] = torch.where(wu != 0, wu * tau ** 2 * value, torch.zeros((), **f8))
        grad[a:b] = torch.where(wu[:, None] != 0, g * (wu * tau)[:, None], torch.zeros((), **f8))
        if hess is not None:
            hess[a:b] = prob * (1.0 - prob) * wu[:, None]
    return [loss, grad] + ([hess] if hess is not None else [])

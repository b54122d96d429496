"""The losses of `evotrees_b200.losses` in 64 bits, their gradients by differentiation, and how far 32-bit arithmetic may be off."""
import torch

F8 = torch.float64
U = 2.0 ** -24            # half a step of a 32-bit float, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _grad(loss_rows, z):
    return torch.autograd.grad(loss_rows.sum(), z)[0]


def distill(z, ids, teacher, w=None, tau=1.0, tail=False):
    """loss [n], grad, hess [n, K], and `scale`: what an error of one part in the probabilities costs the loss of a row."""
    n, K = z.shape
    w = torch.ones(n, dtype=F8) if w is None else w.to(F8)
    loss, grad, hess, scale = torch.zeros(n, dtype=F8), torch.zeros((n, K), dtype=F8), torch.zeros((n, K), dtype=F8), torch.zeros(n, dtype=F8)
    for i in range(n):
        use = (ids[i] != 0) & (teacher[i] != float("-inf"))
        if w[i] == 0 or not use.any():
            continue
        k, t = ids[i][use].long() - 1, teacher[i][use].to(F8)
        if (k < 0).any() or (k >= K).any():
            loss[i] = grad[i] = hess[i] = float("nan")
            continue
        x = z[i].to(F8).clone().requires_grad_(True)
        logp = torch.log_softmax(x / tau, 0)
        logq = t if tail else torch.log_softmax(t / tau, 0)
        q = logq.exp()
        lp = logp[k]
        value = (q * (logq - torch.where(q > 0, lp, torch.zeros_like(lp))))[q > 0].sum()
        cost = (q * (1 + (logq - lp.detach()).abs()))[q > 0].sum()
        if tail:
            named = torch.zeros(K, dtype=torch.bool)
            named[k] = True
            rest = logp[~named]
            qt = max(0.0, 1.0 - float(q.sum()))
            if rest.numel() and (rest > float("-inf")).any() and qt > 0:
                lt = torch.logsumexp(rest, 0)
                value = value + qt * (torch.log(torch.tensor(qt, dtype=F8)) - lt)
                # 1 - sum q is off by a few steps of 1, which counts with the logarithms it multiplies
                cost = cost + qt + 1 + abs(float(torch.log(torch.tensor(qt, dtype=F8)))) + abs(float(lt.detach()))
        r = w[i] * tau ** 2 * value
        loss[i], grad[i] = r.detach(), _grad(r, x)
        p = logp.detach().exp()
        hess[i] = w[i] * p * (1 - p)
        scale[i] = (w[i] * tau ** 2).abs() * cost
    return loss, grad, hess, scale


def policy(z, action, old, adv, ref=None, w=None, tau=1.0, clip=(0.2, 0.2), beta=0.0):
    n, K = z.shape
    w = torch.ones(n, dtype=F8) if w is None else w.to(F8)
    loss, logp_out, grad, hess, scale = (torch.zeros(n, dtype=F8), torch.zeros(n, dtype=F8), torch.zeros((n, K), dtype=F8),
                                         torch.zeros((n, K), dtype=F8), torch.zeros(n, dtype=F8))
    for i in range(n):
        a = int(action[i])
        if a == 0 or w[i] == 0:
            continue
        if a < 0 or a > K:
            loss[i] = logp_out[i] = grad[i] = hess[i] = float("nan")
            continue
        x = z[i].to(F8).clone().requires_grad_(True)
        logp = torch.log_softmax(x / tau, 0)
        lp = logp[a - 1]
        r, A = torch.exp(lp - old[i].to(F8)), adv[i].to(F8)
        u, c = r * A, r.clamp(1 - clip[0], 1 + clip[1]) * A
        value = -(u if float(u.detach()) <= float(c.detach()) else c.detach())
        cost = (r * A).abs().detach()
        if ref is not None:
            d = ref[i].to(F8) - lp
            value = value + beta * (torch.exp(d) - d - 1)
            cost = cost + beta * (1 + torch.exp(d) + d.abs()).detach()
        rr = w[i] * value
        loss[i], logp_out[i] = rr.detach(), lp.detach()
        grad[i] = _grad(rr, x) if rr.requires_grad else 0
        p = logp.detach().exp()
        hess[i] = w[i] * p * (1 - p) / tau ** 2
        scale[i] = w[i].abs() * cost
    return loss, logp_out, grad, hess, scale


def preference(z, label, seq, ref=None, w=None, beta=0.1, smooth=0.0, mean=False):
    n, K = z.shape
    P = (seq.numel() - 1) // 2
    x = torch.where(torch.isnan(z.to(F8)) & (label == 0)[:, None], torch.zeros((), dtype=F8), z.to(F8)).clone().requires_grad_(True)
    logp = torch.log_softmax(x, 1)
    counted = label > 0
    lp = torch.where(counted, logp.gather(1, (label.long() - 1).clamp(min=0)[:, None])[:, 0], torch.zeros((), dtype=F8))
    diff = lp if ref is None else torch.where(counted, lp - torch.nan_to_num(ref.to(F8)), torch.zeros((), dtype=F8))
    loss, margin, total = [], [], 0.0
    for p in range(P):
        D = []
        for s in (2 * p, 2 * p + 1):
            a, b = int(seq[s]), int(seq[s + 1])
            cnt = max(1, int(counted[a:b].sum())) if mean else 1
            D.append(diff[a:b].sum() / cnt)
        m = beta * (D[0] - D[1])
        wp = 1.0 if w is None else float(w[p])
        sp = torch.nn.functional.softplus
        v = wp * ((1 - smooth) * sp(-m) + smooth * sp(m))
        if wp != 0.0:
            total = total + v
        loss.append(float(v.detach()) if wp != 0.0 else 0.0)
        margin.append(float(m.detach()))
    grad = _grad(total, x) if torch.is_tensor(total) and total.requires_grad else torch.zeros((n, K), dtype=F8)
    return torch.tensor(loss, dtype=F8), torch.tensor(margin, dtype=F8), lp.detach(), torch.where(counted[:, None], grad, torch.zeros((), dtype=F8))


def part(z, tau=1.0):
    """Relative error that a probability of a row may have in 32 bits (and, in absolute terms, its logarithm).

    The exponent's argument (z - max) / tau is off by the rounding of its factor and its own, each half a step of it: two steps of U with
    the range, in log p once more for the sum it is compared with; doubled for safety.  A sum of K positive terms that 32 threads or more
    share has at most K / 32 roundings in a row and the steps that join them, each with a factor whose exponential has an error of 2 U:
    four a step.  The remaining operations (exponential, reciprocal, products, logarithm of the sum) are within 64 U."""
    f = z.to(F8)
    f = torch.where(torch.isfinite(f), f, torch.zeros((), dtype=F8))
    f = torch.maximum(f, f.max(1, keepdim=True).values - 120.0 * tau)      # below that a probability is zero in 32 bits
    span = (f.max(1).values - f.min(1).values) / tau
    return U * (4 * span + 4 * (z.shape[1] / 32 + 32) + 64)


def slots_part(teacher, tau=1.0):
    f = teacher.to(F8)
    f = torch.where(torch.isfinite(f), f, torch.zeros((), dtype=F8))
    return U * (4 * (f.max(1).values - f.min(1).values + f.abs().max(1).values) / tau + 4 * teacher.shape[1] + 64)


def close(got, want, tol, what):
    """Equal where `want` is not finite, else within `tol` (a tensor that broadcasts)."""
    got, want = got.detach().cpu().to(F8), want
    tol = torch.as_tensor(tol, dtype=F8).expand(want.shape) if not torch.is_tensor(tol) else tol.to(F8).expand(want.shape)
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    assert torch.equal(torch.nan_to_num(got[odd], nan=7.0), torch.nan_to_num(want[odd], nan=7.0)), f"{what}: infinities"
    err = torch.where(odd, torch.zeros((), dtype=F8), (got - want).abs() - tol)
    bad = err > 0
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((got - want)[bad].abs().max()):.3e} beyond "
                           f"{float(tol[bad].max()):.3e} (value {float(want[bad].abs().max()):.3e})")


def rounded(want, dtype, rel, floor):
    """Tolerance of a result that is right to `rel` of its parts (`floor`: their size) and rounded to `dtype` at the end."""
    # Half of the smallest step around zero counts too.  And the exponential's results below 2^-126, the smallest normal number, are zeros
    # (the instruction flushes them): a probability is off by less than 2^-126 then, a gradient by that times its factor, at most 2^4 here.
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps + 2.0 ** -122
    return rel * floor + (half_step(dtype) * (1 + rel)) * want.abs() + tiny

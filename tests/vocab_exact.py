"""The losses on the scores of a vocabulary in 64 bits, from their definitions, with the size of what an fp32 evaluation may be off by.
Gradients are the direction in which the loss falls, as the library has them.

Error of an fp32 evaluation, in units u = 2^-24 (half a step). An exponential exp((x - M)/tau) is off by 3u*|x - M|/tau from its
argument (difference, 1/tau and product are rounded) and 4u from the function (2^-22 of its result): weighted with the probabilities,
whose mean of |x - M|/tau is below ln(vocabulary) < 13, less than 3*13 + 4 = 43u of the sum. The sum has at most 64 terms in a row and
then trees of 5 + 8 levels: 77u. So S is off by less than 120u of itself, ln S by 120u + the logarithm's own 2u*ln S, and
  logp: |error| < 120u + 26u + 3u*|x_token - M|/tau        -> LOGP_ABS + LOGP_REL*|x_token - M|/tau below (150u and 4u)
A gradient c*(p - target): p is off by 120u + (3|x - M|/tau + 5)u of itself; where p matters for the bound, |x - M|/tau < 40: 250u.
c carries exp(logp - old) and exp(ref - logp), each off by the error of logp: a further 150u + 4u*|x_token - M|/tau of themselves, and
a few roundings: 500u of the sum of the terms' magnitudes covers both for |x_token - M|/tau < 30.  -> GRAD
"""
import torch

U = 2.0 ** -24
LOGP_ABS, LOGP_REL = 150 * U, 4 * U
GRAD = 500 * U


def rows(logits, tau):
    """M, S, p and which rows have a distribution at all."""
    x = logits.double()
    m = x.amax(dim=1)
    base = torch.where(torch.isinf(m) & (m < 0), torch.zeros_like(m), m)
    e = torch.exp((x - base[:, None]) / tau)
    s = e.sum(dim=1)
    return m, s, e / s[:, None], ~((s == 0) & ~torch.isnan(s))


def token_logp(logits, tokens, tau):
    """logp, saved, which rows count, the tolerance of logp, p."""
    m, s, p, any_ = rows(logits, tau)
    t = tokens.long()
    on = (t >= 0) & (t < logits.shape[1]) & any_
    xa = logits.double().gather(1, torch.where(on, t, torch.zeros_like(t))[:, None])[:, 0]
    logp = torch.where(on, (xa - m) / tau - torch.log(s), torch.zeros_like(xa))
    saved = torch.stack([torch.where(on, m, torch.zeros_like(m)), torch.where(on, s, torch.zeros_like(s))])
    gap = torch.where(on, (xa - m).abs() / tau, torch.zeros_like(xa))
    return logp, saved, on, LOGP_ABS + LOGP_REL * torch.where(torch.isfinite(gap), gap, torch.zeros_like(gap)), p


def gradient(p, tokens, on, g, size, tau):
    """g/tau*(target - p) and the magnitude that its error is a share of (size: that of the terms of g)."""
    target = torch.zeros_like(p)
    idx = torch.nonzero(on)[:, 0]
    target[idx, tokens.long()[idx]] = 1.0
    live = (on & (g != 0))[:, None]
    zero = torch.zeros_like(p)
    return torch.where(live, (target - p) * (g / tau)[:, None], zero), torch.where(live, (target + p) * (size / tau)[:, None], zero)


def policy(logits, tokens, old_logp, advantages, ref_logp, mask, low, high, kl_coef, tau, scale):
    logp, _, on, tol, p = token_logp(logits, tokens, tau)
    w = torch.full_like(logp, scale) if mask is None else mask.double() * scale
    on = on & (True if mask is None else mask != 0)
    zero = torch.zeros_like(logp)
    logp = torch.where(on, logp, zero)
    ratio, a = torch.exp(logp - old_logp.double()), advantages.double()
    free, held = ratio * a, ratio.clamp(1 - low, 1 + high) * a
    loss, g, size = -torch.minimum(free, held), torch.where(held < free, zero, free), torch.where(held < free, zero, free.abs())
    err = free.abs()
    kl, kl_err = zero, zero
    if ref_logp is not None:
        d = ref_logp.double() - logp
        kl = torch.where(on, torch.expm1(d) - d, zero)
        kl_err = torch.exp(d) + 1 + d.abs()
        loss, g, size = loss + kl_coef * kl, g + kl_coef * torch.expm1(d), size + abs(kl_coef) * (torch.exp(d) + 1)
        err = err + abs(kl_coef) * kl_err
    on = on & (w != 0)
    loss, g, size = (torch.where(on, w * v, zero) for v in (loss, g, size))
    d_logits, d_size = gradient(p, tokens, on, g, size.abs(), tau)
    return {"loss": (loss, GRAD * w.abs() * err), "logp": (logp, tol), "kl": (kl, GRAD * kl_err), "dlogits": (d_logits, GRAD * d_size)}


def preference(logits, tokens, offsets, ref_logp, squared, beta, smoothing, average, tau, scale):
    """Also which rows lie in a sequence. Sums are in double on the kernel's side too: what is off is the sum of the terms' errors."""
    logp, saved, on, tol, p = token_logp(logits, tokens, tau)
    ends = offsets.tolist()
    t = len(tokens)
    pairs = len(ends) // 2
    inside = torch.zeros(t, dtype=torch.bool, device=logits.device)
    inside[ends[0]:ends[-1]] = True
    q, q_tol, share = [], [], []
    for i in range(2 * pairs):
        part = slice(ends[i], ends[i + 1])
        n = int(on[part].sum())
        by = 1.0 / n if average and n else 1.0
        q.append(logp[part][on[part]].sum() * by - ref_logp[i].double())
        q_tol.append(tol[part][on[part]].sum() * by + U * q[-1].abs())
        share.append(by)
    loss, loss_tol, g, size = [], [], torch.zeros_like(logp), torch.zeros_like(logp)
    for i in range(pairs):
        h, h_tol = q[2 * i] - q[2 * i + 1], q_tol[2 * i] + q_tol[2 * i + 1]
        if squared:
            off = h - 0.5 / beta
            value, dh, bend = off * off, 2 * off, 2.0 + 0 * h
        else:
            m = beta * h
            value = (1 - smoothing) * torch.nn.functional.softplus(-m) + smoothing * torch.nn.functional.softplus(m)
            dh, bend = beta * (smoothing * torch.sigmoid(m) - (1 - smoothing) * torch.sigmoid(-m)), beta * beta / 4 + 0 * h
        loss.append(value * scale)
        loss_tol.append(scale * (dh.abs() * h_tol + bend * h_tol ** 2 + 16 * U * (value + (1 if not squared else 0))))
        for side, sign in ((0, -1.0), (1, 1.0)):
            part = slice(ends[2 * i + side], ends[2 * i + side + 1])
            by = share[2 * i + side] * scale
            g[part] = torch.where(on[part], sign * dh * by, torch.zeros_like(g[part]))
            size[part] = (dh.abs() + (bend * h_tol + beta * 16 * U) / GRAD) * by
    d_logits, d_size = gradient(p, tokens, on & inside, g, size, tau)
    keep = inside.double()
    return {"loss": (torch.stack(loss), torch.stack(loss_tol)), "rewards": (beta * torch.stack(q), beta * torch.stack(q_tol) + 4 * U * (beta * torch.stack(q)).abs()),
            "logp": (logp * keep, tol), "dlogp": (g, size * GRAD), "dlogits": (d_logits, GRAD * d_size), "inside": inside}


def distill(logits, ids, teacher, mask, tau, scale):
    m, s, p, any_ = rows(logits, tau)
    t, v = logits.shape
    ids = ids.long()
    kept = (ids >= 0) & (ids < v)
    at = torch.where(kept, ids, torch.zeros_like(ids))
    top = torch.where(kept, teacher.double(), torch.full_like(teacher.double(), -float("inf")))
    peak = top.amax(dim=1)
    any_ = any_ & ~(torch.isinf(peak) & (peak < 0))
    peak = torch.where(torch.isinf(peak), torch.zeros_like(peak), peak)
    e = torch.exp((top - peak[:, None]) / tau)
    q = e / e.sum(dim=1, keepdim=True).clamp(min=1e-300)
    lnq = (top - peak[:, None]) / tau - torch.log(e.sum(dim=1, keepdim=True))
    lnp = (logits.double().gather(1, at) - m[:, None]) / tau - torch.log(s)[:, None]
    w = torch.full_like(m, scale) if mask is None else mask.double() * scale
    on = any_ & (w != 0)
    zero = torch.zeros_like(q)
    live = q > 0
    terms = torch.where(live, q * (lnq - lnp), zero)
    mass = torch.where(live, q * (lnq.abs() + lnp.abs() + 1), zero)
    target = torch.zeros(t, v, dtype=torch.float64, device=logits.device)
    target.scatter_add_(1, at, torch.where(kept & live, q, zero))
    row = on[:, None]
    none = torch.zeros(t, v, dtype=torch.float64, device=logits.device)
    return {"loss": (torch.where(on, w * tau * tau * terms.sum(dim=1), 0 * w), GRAD * torch.where(on, w.abs() * tau * tau * mass.sum(dim=1), 0 * w)),
            "dlogits": (torch.where(row, (w * tau)[:, None] * (target - p), none), GRAD * torch.where(row, (w.abs() * tau)[:, None] * (p + target), none))}


def check(got, want, tolerance, what):
    """fp32 results against (value, tolerance); a 16-bit one may be half a step further (an fp16 one half its smallest step at least)."""
    want, tolerance = want.to(got.device), tolerance.to(got.device)
    half = torch.finfo(got.dtype).eps / 2
    least = 2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -126
    g = got.double()
    special = ~torch.isfinite(want)
    same = (torch.isnan(g) & torch.isnan(want)) | (g == want)
    bound = tolerance + (half * (want.abs() + tolerance) if got.dtype != torch.float32 else 2 * U * want.abs()) + least
    bad = torch.where(special, ~same, ~((g - want).abs() <= bound))
    if bool(bad.any()):
        at = tuple(int(i) for i in torch.nonzero(bad)[0])
        raise AssertionError("%s: %d of %d outside tolerance; first at %s: got %r want %r bound %r" % (
            what, int(bad.sum()), bad.numel(), at, float(g[at]), float(want[at]), float(bound[at])))

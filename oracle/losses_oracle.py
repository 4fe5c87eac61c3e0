"""The losses over many classes in 64 bits, with the logits in memory, by their formulas; and how far results in the kernels'
number formats may be off.  Test infrastructure only."""
import math

import torch


def softmax_targets(x, w, target, scale=1.0, ignore_index=-100):
    """Losses of rows, which rows count, and the gradients of the raw products x . w for an upstream gradient of one to a row."""
    z = scale * (x.double() @ w.double().t())
    ok = target != ignore_index
    n, t = torch.arange(len(x), device=x.device), torch.where(ok, target, 0).long()
    lse = torch.logsumexp(z, 1)
    e = torch.exp(z - lse.unsqueeze(1))
    others = z.clone()
    others[n, t] = -math.inf
    apart = torch.logsumexp(others, 1) - z[n, t]
    rows = torch.where(ok, torch.logaddexp(apart, torch.zeros_like(apart)), 0.0)      # lse - z[t] and P - 1 without the differences
    e[n, t] = -torch.sigmoid(apart)
    return rows, ok, torch.where(ok.unsqueeze(1), scale * e, 0.0)


def teacher(x, w, logits, ids, temperature=1.0):
    z = x.double() @ w.double().t() / temperature
    logp = z - torch.logsumexp(z, 1, keepdim=True)
    there = (ids >= 0) & (logits.double() > -math.inf)
    ok = there.any(1)
    t = torch.where(there, logits.double() / temperature, -1e300)
    q = torch.where(there & ok.unsqueeze(1), torch.softmax(t, 1), 0.0)
    at = torch.where(there, ids, 0).long()
    rows = temperature ** 2 * (torch.xlogy(q, q) - torch.where(q > 0, q * logp.gather(1, at), 0.0)).sum(1)
    e = torch.exp(logp)
    e.scatter_add_(1, at, -q)
    return torch.where(ok, rows, 0.0), ok, torch.where(ok.unsqueeze(1), temperature * e, 0.0)


def margin(x, w, target, m=0.2, scale=32.0, ignore_index=-100):
    """w [V, K, D].  The third result is by the cosines, [N, V * K]: zero but at a class's nearest row; the fourth the cosines."""
    V, K, D = w.shape
    ux, uw = unit(x.double()), unit(w.double().view(V * K, D))
    every = ux @ uw.t()
    cosine, which = every.view(-1, V, K).max(2)
    ok = target != ignore_index
    n, t = torch.arange(len(x), device=x.device), torch.where(ok, target, 0).long()
    c = cosine[n, t]
    near = c > math.cos(math.pi - m)
    moved = torch.where(near, c * math.cos(m) - torch.sqrt((1 - c * c).clamp(min=0)) * math.sin(m), c - m * math.sin(math.pi - m))
    slope = torch.where(near, math.cos(m) + math.sin(m) * c / torch.sqrt((1 - c * c).clamp(min=1e-6)), 1.0)
    z = scale * cosine
    z[n, t] = scale * moved
    lse = torch.logsumexp(z, 1)
    e = torch.exp(z - lse.unsqueeze(1))
    others = z.clone()
    others[n, t] = -math.inf
    apart = torch.logsumexp(others, 1) - z[n, t]
    rows = torch.where(ok, torch.logaddexp(apart, torch.zeros_like(apart)), 0.0)
    e[n, t] = -torch.sigmoid(apart) * slope
    e = torch.where(ok.unsqueeze(1), scale * e, 0.0)
    full = torch.zeros(len(x), V, K, dtype=torch.float64, device=x.device).scatter_(2, which.unsqueeze(2), e.unsqueeze(2))
    return rows, ok, full.view(-1, V * K), every


def unit(v):
    length = v.norm(dim=1, keepdim=True)
    return torch.where(length > 1e-12, v / length.clamp(min=1e-12), 0.0)


def shares(ok, reduction, up):
    """Upstream gradient of every row: `up` is a number, or one to a row for "none"."""
    if reduction == "none":
        return up.double()
    return ok.double() * float(up) / (max(1, int(ok.sum())) if reduction == "mean" else 1)


def reduced(rows, ok, reduction):
    return rows if reduction == "none" else rows.sum() / (max(1, int(ok.sum())) if reduction == "mean" else 1)


def linear_gradients(x, w, e, g):
    """dx, dw, and (for a row's factor f) the sums of f times the magnitudes of what each is made of."""
    x, w, e = x.double(), w.double(), e * g.unsqueeze(1)
    return e @ w, e.t() @ x, lambda f: (e.abs() * f.unsqueeze(1) @ w.abs(), (e.abs() * f.unsqueeze(1)).t() @ x.abs())


def margin_gradients(x, w, e, g):
    """The same by x and w [V * K, D] (in the magnitudes, with the part along the row that goes)."""
    x, w = x.double(), w.double().reshape(-1, w.shape[-1])
    ux, uw, lx, lw = unit(x), unit(w), x.norm(dim=1, keepdim=True), w.norm(dim=1, keepdim=True)
    ix, iw = torch.where(lx > 1e-12, 1 / lx, 0.0), torch.where(lw > 1e-12, 1 / lw, 0.0)
    e = e * g.unsqueeze(1)
    away = lambda a, u: a - u * (a * u).sum(1, keepdim=True)
    more = lambda a, u: a + u.abs() * (a * u.abs()).sum(1, keepdim=True)
    return ix * away(e @ uw, ux), iw * away(e.t() @ ux, uw), lambda f: (
        ix * more(e.abs() * f.unsqueeze(1) @ uw.abs(), ux), iw * more((e.abs() * f.unsqueeze(1)).t() @ ux.abs(), uw))


def undecided(x, w, e, cosines, g):
    """What margin_gradients' two results may be off by where a class's two nearest rows are no further apart than their cosines'
    errors in fp32 (D roundings of the sum's magnitudes and the last ones, for either): the class's share goes to either of the
    two.  That is at most all of it, counted at both."""
    V, K, D = w.shape
    if K == 1:
        return 0.0, 0.0
    most = (unit(x.double()).abs() @ unit(w.double().view(V * K, D)).abs().t()).view(-1, V, K).amax(2)
    two, at = cosines.view(-1, V, K).topk(2, 2)
    close = two[..., 0] - two[..., 1] <= 2 * 2.0 ** -24 * (D * most + 4)
    share = (e.view(-1, V, K).abs().sum(2) * close).unsqueeze(2).expand(-1, -1, 2)
    both = torch.zeros(len(x), V, K, dtype=torch.float64, device=x.device).scatter_(2, at, share).view(-1, V * K)
    return margin_gradients(x, w, both, g)[2](torch.ones(len(x), dtype=torch.float64, device=x.device))


def logit_bound(x, w, scale):
    """How far a row's logits and the logarithm of its sum may be off in fp32: D roundings of a product's sums, relative to its
    magnitudes, and a few of the logarithm's, relative to itself (base 2: at most 2^-20 of it)."""
    most = (x.double().abs() @ w.double().abs().t()).amax(1) * scale
    return 2 * x.shape[1] * 2.0 ** -24 * most + 2.0 ** -20 * (1 + most)


def gradient_bounds(dx, dw, magnitudes, delta, dtype, least=0.0):
    """An element of a gradient is a sum whose terms' factors dz are off by `delta` of their row (its logits; twice, for the
    logarithm's too) and half a step of `dtype`, the sum itself by as many roundings in fp32 (2^-13 stands for those), and it
    is rounded to `dtype` at the end.  fp16's smallest step is 2^-24."""
    u = torch.finfo(dtype).eps / 2
    small = (2.0 ** -25 if dtype == torch.float16 else 0.0) + least
    mx, mw = magnitudes(1.01 * u + 2 * delta + 2.0 ** -13)
    return mx + 1.01 * u * dx.abs() + small, mw + 1.01 * u * dw.abs() + small

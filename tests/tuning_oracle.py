"""Plain 64-bit restatements of the tuning operators' formulas, for the tests (CPU, torch.float64)."""
import math

import torch

IGNORE = -100


def row_logps(logits, targets, temperature=1.0):
    """(lp, softmax) per row; lp is 0 at ignored rows and NaN for a target outside the vocabulary."""
    x = logits.detach().double().cpu() / temperature
    t = targets.cpu().long()
    v = x.shape[-1]
    m = x.max(-1, keepdim=True).values
    e = torch.exp(torch.where(torch.isinf(m) & (m < 0), x, x - m))
    s = e.sum(-1, keepdim=True)
    lp = x.gather(-1, t.clamp(0, v - 1)[..., None])[..., 0] - m[..., 0] - torch.log(s[..., 0])
    lp = torch.where((t < 0) | (t >= v), math.nan, lp)
    return torch.where(t == IGNORE, 0.0, lp), e / s


def logit_grad(p, targets, slope, temperature=1.0):
    """c_r (1{j = t_r} - p[r, j]) with c = slope / T, and |c| per row; rows of slope 0 are zero whatever p holds."""
    t = targets.cpu().long().clamp(0, p.shape[-1] - 1)
    hot = torch.zeros_like(p).scatter_(-1, t[..., None], 1.0)
    g = (slope / temperature)[..., None] * (hot - p)
    return torch.where(slope[..., None] == 0, 0.0, g), (slope / temperature).abs()[..., None]


def spans(cu):
    return list(zip(cu[:-1], cu[1:]))


def policy(logits, targets, old, adv, ref, *, clip_low=0.2, clip_high=0.2, kl_coef=0.0, cu=None, reduction="token",
           temperature=1.0):
    """loss, logps, kl, clip_fraction, (grad, |c|); rows are 1-D, `adv` one per row or per sequence of `cu`."""
    lp, p = row_logps(logits, targets, temperature)
    n = lp.numel()
    keep = targets.cpu() != IGNORE
    seq = torch.full((n,), -1, dtype=torch.long)
    if cu is not None:
        for i, (a, b) in enumerate(spans(cu)):
            seq[a:b] = i
        keep = keep & (seq >= 0)
    w = torch.zeros(n, dtype=torch.float64)
    if reduction == "token":
        w[keep] = 1.0 / max(1, int(keep.sum()))
    elif reduction == "sum":
        w[keep] = 1.0
    else:
        counts = [int(keep[a:b].sum()) for a, b in spans(cu)]
        live = sum(c > 0 for c in counts)
        for (a, b), c in zip(spans(cu), counts):
            if c:
                w[a:b] = keep[a:b].double() / c / live
    adv = adv.double().cpu()
    a = adv if adv.numel() == n and (cu is None or adv.shape == targets.shape) else adv[seq.clamp_min(0)]
    ratio = torch.exp(lp - old.double().cpu())
    free, held = ratio * a, ratio.clamp(1 - clip_low, 1 + clip_high) * a
    clipped = held < free
    term = -torch.where(clipped, held, free)
    slope = torch.where(clipped, 0.0, -free)
    kl = torch.zeros(n, dtype=torch.float64)
    if ref is not None:
        d = ref.double().cpu() - lp
        kl = torch.exp(d) - d - 1
        term = term + kl_coef * kl
        slope = slope + kl_coef * (1 - torch.exp(d))
    zero = torch.zeros((), dtype=torch.float64)
    pick = lambda v: torch.where(w > 0, v, zero)  # noqa: E731
    slope = pick(slope) * w
    lp = torch.where(keep, lp, 0.0)
    return (pick(term) * w).sum(), lp, (pick(kl) * w).sum(), (clipped * w).sum(), logit_grad(p, targets, slope, temperature)


def preference(logits, targets, ref, cu, *, beta=0.1, label_smoothing=0.0, margin=0.0, kind="sigmoid", average=False,
               temperature=1.0):
    """loss, chosen rewards, rejected rewards, logps, (grad, |c|)."""
    lp, p = row_logps(logits, targets, temperature)
    keep = targets.cpu() != IGNORE
    inside = torch.zeros_like(keep)
    d, norm = [], []
    for a, b in spans(cu):
        inside[a:b] = True
        k = keep[a:b]
        x = (lp[a:b] - (0.0 if ref is None else ref.double().cpu()[a:b]))[k].sum()
        c = max(1, int(k.sum())) if average else 1
        d.append(x / c)
        norm.append(c)
    d = torch.stack(d)
    pairs = len(d) // 2
    h = (beta * (d[:pairs] - d[pairs:]) - margin).requires_grad_(True)
    e = label_smoothing
    ls = torch.nn.functional.logsigmoid
    each = {"sigmoid": lambda: -(1 - e) * ls(h) - e * ls(-h), "hinge": lambda: (1 - h).clamp_min(0),
            "squared": lambda: (h - 0.5) ** 2}[kind]()
    loss = each.mean()
    loss.backward()
    slope = torch.zeros(lp.numel(), dtype=torch.float64)
    for i in range(pairs):
        for s, sign in ((i, 1.0), (pairs + i, -1.0)):
            a, b = spans(cu)[s]
            slope[a:b] = sign * beta * h.grad[i] / norm[s] * keep[a:b]
    lp = torch.where(inside & keep, lp, 0.0)
    return loss.detach(), beta * d[:pairs], beta * d[pairs:], lp, logit_grad(p, targets, slope, temperature)

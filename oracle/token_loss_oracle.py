"""TEST INFRASTRUCTURE ONLY.  float64 numpy forms of the log-probabilities of given tokens and of the two losses on them (clipped policy
loss with a KL term, paired log ratios), with their gradients with respect to the logits, written from the formulas.  The reference has
no trainer, so there is nothing of its own to pin them against.  Only tests may import this module."""
import numpy as np


def live_tokens(z, targets, mask):
    live = (targets >= 0) & (targets < z.shape[-1])
    return live if mask is None else live & mask


def log_probs(z, targets, mask=None, tau=1.0):
    """(lp [...], softmax [..., V], live [...]) of logits [..., V]; rows that do not count give 0."""
    live = live_tokens(z, targets, mask)
    x = np.where(live[..., None], np.asarray(z, np.float64), 0.0) / tau
    top = x.max(-1, keepdims=True)
    e = np.exp(x - top)
    total = e.sum(-1, keepdims=True)
    at = np.where(live, targets, 0)[..., None]
    lp = np.take_along_axis(x - top, at, -1)[..., 0] - np.log(total[..., 0])
    return np.where(live, lp, 0.0), e / total, live


def logit_gradient(p, targets, live, coefficient, tau=1.0):
    """coefficient (1[j = target] - p_j) / tau, zeros in rows that do not count."""
    c = np.where(live, coefficient, 0.0) / tau
    g = -c[..., None] * p
    at = np.where(live, targets, 0)[..., None]
    np.put_along_axis(g, at, np.take_along_axis(g, at, -1) + c[..., None], -1)
    return np.where(live[..., None], g, 0.0)


def policy(z, targets, adv, old, ref=None, mask=None, low=0.2, high=0.2, kl=0.0, tau=1.0, reduction="mean", scale=1.0):
    """(loss, lp, gradient, d loss / d lp) for [S, T, V] logits."""
    lp, p, live = log_probs(z, targets, mask, tau)
    rho = np.exp(lp - old)
    free, clipped = rho * adv, np.clip(rho, 1 - low, 1 + high) * adv
    each, slope = -np.minimum(free, clipped), np.where(free <= clipped, -free, 0.0)
    if kl:
        d = ref - lp
        each, slope = each + kl * (np.expm1(d) - d), slope - kl * np.expm1(d)
    n = live.sum(-1, keepdims=True)
    w = {"mean": 1.0 / max(1, n.sum()), "sequence_mean": 1.0 / (np.maximum(n, 1) * len(n)), "sum": 1.0}[reduction] * scale
    c = np.where(live, slope * w, 0.0)
    return np.where(live, each * w, 0.0).sum(), lp, logit_gradient(p, targets, live, c, tau), c


def preference(z, targets, ref=None, mask=None, beta=0.1, smoothing=0.0, margin=0.0, average=False, scale=1.0):
    """(loss, sequences' lp, gradient, d loss / d lp of each sequence) for [2P, T, V] logits."""
    lp, p, live = log_probs(z, targets, mask)
    n = np.maximum(live.sum(-1), 1) if average else np.ones(len(lp))
    seq = lp.sum(-1) / n
    over = seq - (0.0 if ref is None else ref)
    pairs = len(lp) // 2
    d = beta * (over[:pairs] - over[pairs:]) - margin
    loss = scale * np.mean((1 - smoothing) * np.logaddexp(0.0, -d) + smoothing * np.logaddexp(0.0, d))
    slope = -beta * scale / pairs * (1 - smoothing - 1 / (1 + np.exp(-d)))
    c = np.concatenate((slope, -slope)) / n
    return loss, seq, logit_gradient(p, targets, live, c[:, None]), c

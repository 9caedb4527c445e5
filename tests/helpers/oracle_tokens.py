"""Definitions in 64 bits of the per-token vocabulary ops and the error that fp32 kernels may have."""
import math

import torch


def scores(logits, tokens, top_k, temperature):
    """(logprob, entropy, top_logprob, top_index, log-probabilities) of whole-vocabulary logits."""
    z = logits.detach().double()
    logp = torch.log_softmax(z / temperature, 1)
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, p).sum(1)
    known = tokens < z.shape[1]
    lp = logp.gather(1, tokens.clamp(0, z.shape[1] - 1)[:, None])[:, 0]
    lp = torch.where(tokens < 0, 0.0, torch.where(known, lp, math.nan))
    order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top_k]
    return lp, entropy, logp.gather(1, order), order, logp


def scores_grad(logits, tokens, top_index, g, h, u, temperature):
    _, entropy, _, _, logp = scores(logits, tokens, 0, temperature)
    p = logp.exp()
    rows = len(tokens)
    g = torch.zeros(rows, dtype=torch.float64, device=p.device) if g is None else torch.where(tokens >= 0, g.double(), 0.0)
    dx = -p * g[:, None]
    dx.scatter_add_(1, tokens.clamp_min(0)[:, None], g[:, None])
    if h is not None:
        dx -= torch.where(p > 0, p * (logp + entropy[:, None]), 0.0) * h.double()[:, None]
    if u is not None:
        dx -= p * u.double().sum(1, keepdim=True)
        dx.scatter_add_(1, top_index, u.double())
    return dx / temperature


def distill(logits, index, logit, dloss, temperature):
    """(loss, d logits)."""
    logp = torch.log_softmax(logits.detach().double() / temperature, 1)
    t = logit.double() / temperature
    some = ~(t == -math.inf).all(1, keepdim=True)
    log_q = torch.log_softmax(torch.where(some, t, 0.0), 1)
    q = torch.where(some, log_q.exp(), 0.0)
    used = q > 0
    loss = torch.where(used, q * (log_q - logp.gather(1, index.clamp(0, logp.shape[1] - 1))), 0.0).sum(1)
    dx = torch.where(some, logp.exp(), 0.0)
    dx = dx.scatter_add(1, torch.where(used, index, 0), torch.where(used, -q, 0.0))
    return loss, dx * (dloss.double()[:, None] / temperature)


def statistic_tolerance(logits, temperature):
    """Absolute error allowed to an fp32 log-probability, entropy or loss. A difference z - m is exact to
    2^-24 of itself, its product with log2(e) / T to 2^-23: an exponent of magnitude t is off by
    t 2^-23, the approximate exponential by 2^-22 of its value, the logarithm by 2^-22 (2^-22 of the
    result beyond 2); the fp32 sums of up to 1000 terms per thread add at most 1000 2^-24 / 2 relative
    and in practice far less. Exponents that matter are bounded by the range of the finite logits."""
    z = logits.detach().double()
    z = torch.where(z.isfinite(), z, 0.0)
    span = (z.amax(1) - z.amin(1)).clamp_max(100.0) / temperature
    return 2.0 ** -18 + 2.0 ** -21 * span


def grad_error(got, want, noise):
    """Largest excess of |got - want| over half a unit of the type plus `noise` (absolute, per row), as a
    multiple of it: <= 1 passes. fp16 gradients below its smallest normal number are off by up to 2^-25."""
    half = torch.finfo(got.dtype).eps / 2 * 1.001
    floor = 2.0 ** -25 if got.dtype == torch.float16 else 1e-37
    err = (got.double() - want).abs()
    bound = half * want.abs() + noise[:, None] + floor
    worst = (err / bound).max().item() if err.numel() else 0.0
    return worst if worst == worst else math.inf

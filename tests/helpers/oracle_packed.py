"""Packed-document attention in 64 bits, with a bound on the error of a kernel that rounds the
probabilities, their gradients and its results to the input type.

With u = half a unit of the type and eta = 2^-15 for all fp32 steps (sums of up to 2^9 products per
tensor-core pass, exponentials, the log-sum-exp), per element:
  out   u |O| + (u + eta) P|V| + 2^-25 sum|V| (fp16 probabilities below the smallest normal number)
  D     E = |dO| . (bound of out) + eta |dO| . P|V|      (D = dO . O takes the rounded O)
  dS    (u + eta) |dS| + P (E + eta |dO||V|)
  dV    u |dV| + (u + eta) P^T|dO|
  dQ    u |dQ| + scale (bound of dS) |K|,   dK likewise with its transpose and |Q|
"""
import torch


def documents(lengths):
    at = 0
    for n in lengths:
        if n:
            yield slice(at, at + n)
        at += n


def attention(q, k, v, lengths, causal, scale=None, d_out=None):
    """{name: (value, bound)} of out and, with d_out, dq, dk, dv, all double; rows of no document are 0."""
    u, eta, floor = torch.finfo(q.dtype).eps / 2, 2.0 ** -15, 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    scale = q.shape[2] ** -0.5 if scale is None else scale
    group = q.shape[1] // k.shape[1]
    res = {name: tuple(torch.zeros(t.shape, dtype=torch.float64, device=q.device) for _ in range(2))
           for name, t in (("out", q), ("dq", q), ("dk", k), ("dv", k))}
    for rows in documents(lengths):
        qd, kd, vd = (t[rows].detach().double().transpose(0, 1) for t in (q, k, v))
        kd, vd = kd.repeat_interleave(group, 0), vd.repeat_interleave(group, 0)
        x = qd @ kd.transpose(1, 2) * scale
        if causal:
            n = x.shape[-1]
            x.masked_fill_(torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1), float("-inf"))
        p = torch.softmax(x, -1)
        o = p @ vd
        spread = p @ vd.abs()
        o_bound = u * o.abs() + (u + eta) * spread + floor * vd.abs().sum(1, keepdim=True)

        def put(name, value, bound, shared):
            for dst, t in zip(res[name], (value, bound)):
                t = t.unflatten(0, (-1, group)).sum(1) if shared else t
                dst[rows] = t.transpose(0, 1)
        put("out", o, o_bound, False)
        if d_out is None:
            continue
        do = d_out[rows].double().transpose(0, 1)
        dp = do @ vd.transpose(1, 2)
        ds = p * (dp - (do * o).sum(-1, keepdim=True))
        e = (do.abs() * (o_bound + eta * spread)).sum(-1, keepdim=True)
        ds_bound = (u + eta) * ds.abs() + p * (e + eta * (do.abs() @ vd.abs().transpose(1, 2))) + floor
        put("dv", p.transpose(1, 2) @ do, ((u + eta) * p + floor).transpose(1, 2) @ do.abs(), True)
        put("dq", scale * ds @ kd, scale * ds_bound @ kd.abs(), False)
        put("dk", scale * ds.transpose(1, 2) @ qd, scale * ds_bound.transpose(1, 2) @ qd.abs(), True)
    if d_out is not None:
        for name in ("dq", "dk", "dv"):
            value, bound = res[name]
            res[name] = (value, bound + u * value.abs())
    return res


def excess(got, value_and_bound):
    """Largest |got - value| as a multiple of its bound: <= 1 passes, NaN does not."""
    value, bound = value_and_bound
    if got.numel() == 0:
        return 0.0
    small = 2.0 ** -25 if got.dtype == torch.float16 else 1e-37      # the type's own subnormal step
    worst = ((got.double() - value).abs() / (1.02 * bound + small)).max().item()
    return worst if worst == worst else float("inf")

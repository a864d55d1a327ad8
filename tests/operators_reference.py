"""64-bit restatements of the embedding and windowed-attention products, with the error each result may carry.

``u`` is half a step of a type relative to the value. The bounds count every rounding of the method: products and sums in
fp32 (n terms: n * u32), one rounding of the softmax weights (and of their gradients) to the inputs' type, one of the
result, and for fp16 the absolute step of its subnormal numbers (2^-25).
"""

import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# The absolute part of a rounding. fp32 (and bf16, which has its exponents) holds no number between 0 and 2^-149, and an
# exponential below 2^-126 may be taken as 0: exp(-135) = 2.3e-59 is 0 in fp32, with an error of 100 % that no relative bound
# covers and 2^-126 does.
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}
U32 = U[torch.float32]


def positions(lq, lk, window, sinks, device):
    """[lq, lk] mask of the seen pairs."""
    p = torch.arange(lk - lq, lk, device=device)[:, None]
    j = torch.arange(lk, device=device)[None, :]
    return (j <= p) & ((j > p - window) | (j < sinks))


def clean(x, seen):
    """Rows nobody sees as zeros, so that nothing in them enters the reference."""
    return torch.where(seen.reshape(-1, *[1] * (x.dim() - 1)), x.double(), torch.zeros((), dtype=torch.float64, device=x.device))


def attention(q, k, v, window, sinks, scale, dout=None):
    """One sequence: q [lq, hq, d], k, v [lk, hk, d]. Returns {name: (value, allowed error)}; with dout the gradients too."""
    t = q.dtype
    u, tiny = U[t], TINY[t]
    mask = positions(q.shape[0], k.shape[0], window, sinks, q.device)
    group = q.shape[1] // k.shape[1]
    q, k, v = q.double(), clean(k, mask.any(0)), clean(v, mask.any(0))
    kx, vx = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    d, n = q.shape[2], max(1, k.shape[0])
    s = torch.einsum("ihd,jhd->hij", q, kx) * scale
    # a score's error: d products and sums, the scale, and the exponential's argument in base 2
    ds = (d + 8) * U32 * torch.einsum("ihd,jhd->hij", q.abs(), kx.abs()) * abs(scale)
    s = s.masked_fill(~mask, -torch.inf)
    ds = ds.masked_fill(~mask, 0.0)
    lse = torch.logsumexp(s, -1)
    p = torch.where(mask, torch.exp(s - torch.where(lse.isinf(), 0.0, lse)[..., None]), 0.0)
    worst = ds.amax(-1) if k.shape[0] else torch.zeros_like(lse)
    rel = 2 * worst + (n + 24) * U32 + 4 * U32 * s.masked_fill(~mask, 0).abs().amax(-1) if k.shape[0] else worst  # of a weight
    o = torch.einsum("hij,jhd->ihd", p, vx)
    oa = torch.einsum("hij,jhd->ihd", p, vx.abs())
    seen_v = torch.einsum("hij,jhd->ihd", mask.double().expand_as(p), vx.abs())
    weight = u if t != torch.float32 else 0.0
    r = rel.permute(1, 0)[..., None]
    o_err = (weight + r) * oa + u * o.abs() + tiny * (1 + seen_v)
    out = {"out": (o, o_err * 1.01), "lse": (lse, rel + 4 * U32 * (1 + lse.abs().nan_to_num(posinf=0.0)))}
    if dout is None:
        return out
    g = dout.double()
    dp = torch.einsum("ihd,jhd->hij", g, vx)
    dpa = torch.einsum("ihd,jhd->hij", g.abs(), vx.abs())
    delta = (g * o).sum(-1).permute(1, 0)[..., None]
    # delta comes from the rounded O; dP and delta are sums of d terms in fp32
    ddelta = (g.abs() * o_err).sum(-1).permute(1, 0)[..., None] + (d + 4) * U32 * (g * o).abs().sum(-1).permute(1, 0)[..., None]
    grad = p * (dp - delta)
    # (a weight that is flushed to 0 takes its gradient along: 2^-126 of |dP| + |delta|)
    grad_err = (p * ((d + 4) * U32 * dpa + ddelta) + (weight + rel[..., None] + 4 * U32) * grad.abs()
                + mask * (tiny + TINY[torch.float32] * (dpa + delta.abs())))
    p_err = (weight + rel[..., None]) * p + tiny * mask

    def shared(x):  # sums over the query heads of a key head
        return x.unflatten(1, (-1, group)).sum(2)

    m = q.shape[0] * group + 4
    ga, qa, ka = g.abs(), q.abs(), kx.abs()
    dv = shared(torch.einsum("hij,ihd->jhd", p, g))
    dv_err = shared(torch.einsum("hij,ihd->jhd", p_err + m * U32 * p, ga)) + u * dv.abs() + tiny
    dk = shared(torch.einsum("hij,ihd->jhd", grad, q)) * scale
    dk_err = shared(torch.einsum("hij,ihd->jhd", grad_err + m * U32 * grad.abs(), qa)) * abs(scale) + u * dk.abs() + tiny
    dq = torch.einsum("hij,jhd->ihd", grad, kx) * scale
    dq_err = torch.einsum("hij,jhd->ihd", grad_err + (n + 4) * U32 * grad.abs(), ka) * abs(scale) + u * dq.abs() + tiny
    out.update(dq=(dq, 1.01 * dq_err), dk=(dk, 1.01 * dk_err), dv=(dv, 1.01 * dv_err))
    return out


def close(got, want, what):
    """Every element within its own bound; infinities (an empty row's lse) equal."""
    value, allowed = want
    got = got.double()
    same = (got == value) | ((got - value).abs() <= allowed)
    assert bool(same.all()), (
        f"{what}: {int((~same).sum())} of {same.numel()} outside; worst {float(((got - value).abs() / allowed.clamp_min(1e-300))[~same].nan_to_num(9e9).max()):.3g} "
        f"of the allowed error, first at {torch.nonzero(~same)[0].tolist()}")


def gradient(indices, dy, rows, alpha, beta, table, base=0):
    """dE = alpha * S^T dY + beta * dE and its allowed error."""
    t = table.dtype
    ids = indices.long() - base
    ok = (ids >= 0) & (ids < rows)
    ids, y = ids[ok], dy.double()[ok]
    total = torch.zeros(rows, dy.shape[1], dtype=torch.float64, device=dy.device).index_add_(0, ids, y)
    size = torch.zeros_like(total).index_add_(0, ids, y.abs())
    n = torch.bincount(ids, minlength=rows).double()[:, None]
    old = torch.zeros_like(total) if beta == 0 else table.double() * beta
    value = alpha * total + old
    err = (n + 3) * U32 * abs(alpha) * size + 2 * U32 * old.abs() + U[t] * value.abs() + TINY[t]
    return value, 1.01 * err

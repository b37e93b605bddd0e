"""Attention and its gradient in 64 bits, with bounds on what rounding may cost (test infrastructure).

Every tolerance is counted from the formulas.  u is half a step of the inputs' type (0 where weights are not rounded), e = 2^-23
the most one 32-bit addition of the tensor cores loses.  A score is off by E d with E = scale sum |q| |k| and
d = (D + 8) e (+ 2^-21 for the products of split float32 values), a weight so by the factor exp(2 E d) and the two 2^-22 of ex2
and of the sum.
"""
import math

import torch

STEP = 2.0 ** -23


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def visible(N, M, P, length, causal):
    """(N, P + M) truth values: which keys of [prefix, own] a query sees."""
    own = torch.arange(M)[None, :] < max(0, min(M, length))
    own = own.expand(N, M)
    if causal:
        own = own & (torch.arange(M)[None, :] <= max(0, min(M, length)) - N + torch.arange(N)[:, None])
    return torch.cat([torch.ones(N, P, dtype=torch.bool), own], dim=1)


def _one(q, k, v, seen, scale, dtype):
    """One head of one batch entry: weights, output, lse and the bound of the output."""
    D = q.shape[-1]
    k, v = k.clone(), v.clone()
    hidden = ~seen.any(dim=0)
    k[hidden], v[hidden] = 0.0, 0.0                  # never used, whatever they hold
    s = (q @ k.T) * scale
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(dim=1, keepdim=True) if s.shape[1] else torch.full((q.shape[0], 1), -math.inf, dtype=torch.float64)
    w = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
    total = w.sum(dim=1, keepdim=True)
    p = w / total.masked_fill(total == 0.0, 1.0)
    out = p @ v
    lse = (top + torch.log(total)).squeeze(1)
    u = _half_step(dtype)
    off = (D + 8) * STEP + (2.0 ** -21 if dtype == torch.float32 else 0.0)
    E = scale * (q.abs() @ k.abs().T)
    E = E.masked_fill(~seen, 0.0).amax(dim=1, keepdim=True) if E.shape[1] else torch.zeros_like(top)
    weight = torch.expm1(2.0 * E * off) + 2.0 ** -20 + s.shape[1] / 8 * STEP     # relative error of a normalised weight
    rounded = 0.0 if dtype == torch.float32 else u
    bound = u * out.abs() + (p @ v.abs()) * (weight + rounded)
    if dtype == torch.float32:
        bound = bound + (p @ v.abs()) * 2.0 ** -21
    if dtype == torch.float16:
        # half of the smallest step: of the result, and of a weight, which the kernels multiply by 2^8 before they round it
        bound = bound + 2.0 ** -25 + 2.0 ** -33 * v.abs().sum(dim=0)
    return p, out, lse, bound, weight, E * off


def attention(q, k, v, lengths=None, scale=None, prefix=None):
    """q (L, N, H, D), k, v (L or 1, M, Hk, D) of any type; prefix: (k, v) of (P, Hk, D).  Returns out, lse and their bounds."""
    dtype = q.dtype
    k, v = (t.expand(max(q.shape[0], k.shape[0]), *t.shape[1:]).cpu().double() for t in (k, v))
    q = q.expand(max(q.shape[0], k.shape[0]), *q.shape[1:]).cpu().double()
    L, N, H, D = q.shape
    M, Hk = k.shape[1:3]
    P = 0 if prefix is None else prefix[0].shape[0]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out, bound = torch.zeros(L, N, H, D, dtype=torch.float64), torch.zeros(L, N, H, D, dtype=torch.float64)
    lse, lse_bound = torch.zeros(L, H, N, dtype=torch.float64), torch.zeros(L, H, N, dtype=torch.float64)
    for l in range(L):
        seen = visible(N, M, P, M if lengths is None else int(lengths[l]), prefix is not None)
        for h in range(H):
            hk = h // (H // Hk)
            kk, vv = k[l, :, hk], v[l, :, hk]
            if prefix is not None:
                kk, vv = (torch.cat([a[:, hk].cpu().double(), b]) for a, b in zip(prefix, (kk, vv)))
            _, out[l, :, h], lse[l, h], bound[l, :, h], weight, score = _one(q[l, :, h], kk, vv, seen, scale, dtype)
            lse_bound[l, h] = (weight + score).squeeze(1) + 4 * STEP * (1.0 + lse[l, h].abs().nan_to_num(posinf=0.0, neginf=0.0))
    return out, lse, bound, lse_bound


def attention_grad(q, k, v, grad_out, lengths=None, scale=None):
    """{name: (gradient, bound)} for grad_q, grad_k, grad_v, each with its input's shape (sums over broadcast extents)."""
    dtype = q.dtype
    qb, kb = q.shape[0], k.shape[0]
    L = max(qb, kb, grad_out.shape[0])
    q, k, v, g = (t.expand(L, *t.shape[1:]).cpu().double() for t in (q, k, v, grad_out))
    _, N, H, D = q.shape
    M, Hk = k.shape[1:3]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    u = _half_step(dtype)
    rounded = 2.0 ** -21 if dtype == torch.float32 else u
    f16 = dtype == torch.float16
    sums = {n: [torch.zeros(s, dtype=torch.float64) for _ in range(2)]
            for n, s in (("grad_q", q.shape), ("grad_k", k.shape), ("grad_v", k.shape))}
    terms = max(M, N * L * H // Hk) / 8 * STEP
    # float16: ds is multiplied by at least 2^13 / x, x = D max|dout| max|v| of the keys that are seen, before it is rounded, and half of the
    # smallest step there is 2^-25
    there = torch.stack([torch.arange(M) < (M if lengths is None else int(lengths[l])) for l in range(L)])
    v_peak = v.abs().amax(dim=-1).masked_fill(~there[:, :, None], 0.0).amax(dim=(0, 1)) if M else torch.zeros(Hk)
    for l in range(L):
        seen = visible(N, M, 0, M if lengths is None else int(lengths[l]), False)
        for h in range(H):
            hk = h // (H // Hk)
            p, out, _, out_bound, weight, _ = _one(q[l, :, h], k[l, :, hk], v[l, :, hk], seen, scale, dtype)
            kk, vv = k[l, :, hk].clone(), v[l, :, hk].clone()
            kk[~seen.any(dim=0)], vv[~seen.any(dim=0)] = 0.0, 0.0
            qq, gg = q[l, :, h], g[l, :, h]
            # the gradient takes p from the rounded 32-bit lse: two more roundings of the score
            weight = weight + 2.0 ** -20 + 8 * STEP * (scale * (qq @ kk.T)).abs().masked_fill(~seen, 0.0).amax(dim=1, keepdim=True) if M else weight
            dp, delta = gg @ vv.T, (gg * out).sum(dim=1, keepdim=True)
            ds = p * (dp - delta)
            # dp is a sum of D products, delta takes the output as it was rounded
            dp_off = (gg.abs() @ vv.abs().T) * ((D + 8) * STEP + (2.0 ** -21 if dtype == torch.float32 else 0.0))
            delta_off = (gg.abs() * out_bound).sum(dim=1, keepdim=True) + (gg * out).abs().sum(dim=1, keepdim=True) * D * STEP
            ds_off = ds.abs() * (weight + rounded + terms) + p * (1.0 + weight) * (dp_off + delta_off)
            p_off = p * (weight + rounded + terms)
            if f16:
                ds_off = ds_off + 2.0 ** -38 * D * float(g[:, :, hk * (H // Hk):(hk + 1) * (H // Hk)].abs().max() * v_peak[hk])
                p_off = p_off + 2.0 ** -33
            for name, value, off in (("grad_q", scale * ds @ kk, scale * ds_off @ kk.abs()),
                                     ("grad_k", scale * ds.T @ qq, scale * ds_off.T @ qq.abs()),
                                     ("grad_v", p.T @ gg, p_off.T @ gg.abs())):
                at = h if name == "grad_q" else hk
                sums[name][0][l, :, at] += value
                sums[name][1][l, :, at] += off
    found = {}
    for name, (value, off) in sums.items():
        if (qb if name == "grad_q" else kb) == 1:
            value, off = value.sum(dim=0, keepdim=True), off.sum(dim=0, keepdim=True)
        found[name] = (value, off + u * value.abs() + (2.0 ** -25 if f16 else 0.0) + 2.0 ** -140)
    return found

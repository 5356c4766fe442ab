"""Plain 64-bit forms of causal attention over packed sequences, of its gradients
and of head norms, with the bounds that their roundings obey, for the tests."""
import math

import torch

BF16 = 2.0 ** -8   # half a step of bf16, relative
FP32 = 2.0 ** -24


def packed(q, k, v, lens, first=0, dO=None, o=None):
    """Per sequence and head, in float64: o and lse (dO None), or dq, dk, dv; each as
    (value, bound without the output's own rounding). `o` is what the kernel is given.

    The kernel's S has fp32 sums of D products (relative to the sum of magnitudes: D 2^-24);
    P = exp(S - lse) is off by that, by exp2's 2^-21 and by the 2^-23 of its argument, and is
    rounded to bf16 for P V and P^T dO, as dS is for the products with k and q. Delta = dO . o
    takes the rounded o."""
    H, Hk, D = q.shape[1], k.shape[1], q.shape[2]
    G, scale = H // Hk, D ** -0.5
    f64 = lambda x: None if x is None else x.double()  # noqa: E731
    q, k, v, dO, o = (f64(x) for x in (q, k, v, dO, o))
    zero = lambda x: (torch.zeros_like(x), torch.zeros_like(x))  # noqa: E731
    out, lse = zero(q), zero(q[..., 0].t().contiguous())
    dq, dk, dv = zero(q), zero(k), zero(v)
    a = first
    for n in lens:
        b = a + n
        if n == 0:
            continue
        future = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
        for h in range(H):
            x, y, z = q[a:b, h], k[a:b, h // G], v[a:b, h // G]
            s = (scale * x @ y.T).masked_fill(future, -math.inf)
            ls = torch.logsumexp(s, 1)
            p = torch.exp(s - ls[:, None])
            mag = scale * x.abs() @ y.abs().T
            top = mag.masked_fill(future, 0).amax(1, keepdim=True)
            ep = 2 * D * FP32 * top + 4 * FP32 * (s.masked_fill(future, 0).abs() + ls[:, None].abs()) + 2.0 ** -19
            if dO is None:
                out[0][a:b, h] = p @ z
                out[1][a:b, h] = (p * (BF16 + ep)) @ z.abs()
                lse[0][h, a:b] = ls
                lse[1][h, a:b] = ep.amax(1) + 2.0 ** -22 * ls.abs()
                continue
            g = dO[a:b, h]
            dp = g @ z.T
            delta = (p * dp).sum(1, keepdim=True)
            ds = p * (dp - delta)
            # Delta from the given o, and its own and dP's fp32 sums
            given = (g * o[a:b, h]).sum(1, keepdim=True)
            off = (given - delta).abs() + D * FP32 * ((g.abs() * o[a:b, h].abs()).sum(1, keepdim=True) + g.abs() @ z.abs().T)
            eds = ds.abs() * (BF16 + ep) + p * off * (1 + BF16)
            dv[0][a:b, h // G] += p.T @ g
            dv[1][a:b, h // G] += (p * (BF16 + ep)).T @ g.abs()
            dq[0][a:b, h] = scale * ds @ y
            dq[1][a:b, h] = scale * eds @ y.abs()
            dk[0][a:b, h // G] += scale * ds.T @ x
            dk[1][a:b, h // G] += scale * eds.T @ x.abs()
        a = b
    # fp32 sums of up to 1900 products: n 2^-24 of the magnitudes, 3% of 2^-8
    grow = lambda t: (t[0], t[1] * 1.03 + 1e-30)  # noqa: E731
    return (grow(out), lse) if dO is None else tuple(grow(t) for t in (dq, dk, dv))


def paged(q, k, v, on, step):
    """o, its bound and lse of one query [H, D] over keys k, v [n, Hk, D] where `on` [n]; `step`: the
    rounding of P (0: none)."""
    H, D = q.shape
    G = H // k.shape[1]
    q, k, v = q.double(), k.double()[on].repeat_interleave(G, 1), v.double()[on].repeat_interleave(G, 1)
    s = torch.einsum("hd,nhd->hn", q, k) * D ** -0.5
    mag = torch.einsum("hd,nhd->hn", q.abs(), k.abs()) * D ** -0.5
    if s.shape[1] == 0:
        return torch.zeros_like(q), torch.zeros_like(q), torch.full((H,), -math.inf, device=q.device)
    lse = torch.logsumexp(s, 1)
    p = torch.exp(s - lse[:, None])
    ep = 2 * D * FP32 * mag.amax(1, keepdim=True) + 4 * FP32 * (s.abs() + lse[:, None].abs()) + 2.0 ** -19
    # sums over the keys in fp32, in lanes and splits: chains of 2^10 terms at most
    o = torch.einsum("hn,nhd->hd", p, v)
    return o, torch.einsum("hn,nhd->hd", p * (step + ep + 2.0 ** -14 * (step > 0) + 2.0 ** -16), v.abs()), lse


def rms(x, gamma, eps):
    """x / sqrt(mean x^2 + eps) * gamma in float64 (gamma None: x)."""
    x = x.double()
    return x if gamma is None else x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * gamma.double()

"""Plain 64-bit forms of the rotary positions and of linear attention with a
decay per head, for the tests of both."""
import torch


def turn(x, positions, sections, base=10000.0, layout="halves", freqs="shared", inverse=False):
    """Rotary positions of x [B, L, H, D] in float64 (positions int [axes, B, L])."""
    x = x.double()
    P = sum(sections)
    ang, i = [], 0
    for a, n in enumerate(sections):
        for j in range(n):
            f = j / n if freqs == "per_axis" else i / P
            ang.append(positions[a].double() * base ** -f)
            i += 1
    ang = torch.stack(ang, -1)[:, :, None]
    c, s = ang.cos(), ang.sin() * (-1.0 if inverse else 1.0)
    y = x.clone()
    a, b = (slice(0, P), slice(P, 2 * P)) if layout == "halves" else (slice(0, 2 * P, 2), slice(1, 2 * P, 2))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def mix(q, k, v, log_decay, lens=None, state=None, scale=None, absolute=False):
    """(o, final state) of linear attention in float64 as the quadratic form, differentiable.
    absolute: every product taken of magnitudes (the sum that rounding errors scale with)."""
    B, L, H, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    lam = torch.exp(log_decay.double())
    q, k, v = q.double(), k.double(), v.double()
    if absolute:
        q, k, v = q.abs(), k.abs(), v.abs()
        state = None if state is None else state.abs()
    outs, states = [], []
    for b in range(B):
        n = L if lens is None else max(0, min(L, int(lens[b])))
        t = torch.arange(n, device=q.device)
        e = t[:, None] - t
        qb, kb, vb = (x[b, :n].transpose(0, 1) for x in (q, k, v))  # [H, n, D]
        M = torch.where(e >= 0, lam[:, None, None] ** e.clamp(min=0), 0.0)
        o = ((qb @ kb.transpose(1, 2)) * M) @ vb
        S = (kb * (lam[:, None] ** (n - 1 - t))[..., None]).transpose(1, 2) @ vb
        if state is not None:
            s0 = state[b].double()
            o = o + (lam[:, None] ** (t + 1))[..., None] * (qb @ s0)
            S = S + (lam ** n)[:, None, None] * s0
        pad = torch.zeros(L - n, H, D, dtype=torch.float64, device=q.device)
        outs.append(torch.cat([scale * o.transpose(0, 1), pad]))
        states.append(S)
    return torch.stack(outs), torch.stack(states)


def mix_grads(q, k, v, log_decay, dO, lens=None, state=None, d_state=None, scale=None):
    """Gradients (dq, dk, dv, d_state_in) of mix by autograd in float64; dO past the lengths is
    not used. state None: the last is the gradient with respect to a zero state."""
    B, L, H, D = q.shape
    if lens is not None:
        live = torch.arange(L, device=q.device) < lens.to(q.device)[:, None].clamp(0, L)
        q, k, v, dO = (torch.where(live[..., None, None], x.double(), 0.0) for x in (q, k, v, dO))
    x = [t.double().detach().requires_grad_() for t in (q, k, v)]
    s = (torch.zeros(B, H, D, D, dtype=torch.float64, device=q.device) if state is None
         else state.double()).detach().requires_grad_()
    o, S = mix(*x, log_decay, lens, s, scale)
    loss = (o * dO.double()).sum()
    if d_state is not None:
        loss = loss + (S * d_state.double()).sum()
    loss = loss + 0.0 * s.sum()
    return torch.autograd.grad(loss, x + [s])


def mix_grads_absolute(q, k, v, log_decay, dO, lens=None, state=None, d_state=None, scale=None):
    """The gradients' sums of magnitudes (mix_grads of magnitudes: every term is positive)."""
    m = [t if t is None else t.abs() for t in (q, k, v, dO, state, d_state)]
    return mix_grads(m[0], m[1], m[2], log_decay, m[3], lens, m[4], m[5], scale)

"""Sizes, plain forms and work of the positional and linear-attention operators.

Three operators that stand beside the softmax attention of this framework and
share its [B, L, H, D] tensors:

  rope    rotary positions of q and k with one to four position axes (a text
          index, or time / height / width of a video token), and its adjoint;
  mix     causal linear attention with a decay per head over a prompt or a
          training sequence, from an optional carried state, its backward;
  step    the same recurrence for one new token per sequence (serving).

`own` false computes each in elementary torch operations; true calls the
framework's kernels through pa_capi.
"""
import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pure-attention_b200")
_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _capi():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import pa_capi
    return pa_capi


# ---------------------------------------------------------------- cases
def _rope(name, direction, B, L, H, Hk, D, dtype, sections, layout, freqs, far):
    return {"name": name, "op": "rope", "dir": direction, "B": B, "L": L, "H": H, "Hk": Hk, "D": D,
            "dtype": dtype, "sections": sections, "layout": layout, "freqs": freqs, "far": far}


def _mix(name, direction, B, L, H, D, dtype, ragged, states):
    return {"name": name, "op": "mix", "dir": direction, "B": B, "L": L, "H": H, "D": D,
            "dtype": dtype, "ragged": ragged, "states": states}


def _step(name, B, H, D, dtype):
    return {"name": name, "op": "step", "B": B, "H": H, "D": D, "dtype": dtype}


def listed():
    return [
        # one new token of each of 16 sequences being generated, far into its context
        _rope("rope, new tokens", "fwd", 16, 1, 8, 8, 64, "bf16", "32", "halves", "shared", 200000),
        # q and k of the attention benchmark's batch, tokens of a video (time, height, width)
        _rope("rope, video batch", "fwd", 8, 4096, 16, 16, 64, "bf16", "8,12,12", "halves", "shared", 64),
        # gradients of the fp32 training path: images (height, width), shared k heads, odd length
        _rope("rope gradient, images", "bwd", 5, 1177, 8, 2, 64, "fp32", "16,16", "pairs", "per_axis", 64),
        # a short prompt: latency counts
        _mix("prompt, 100 tokens", "fwd", 1, 100, 8, 64, "bf16", False, True),
        # the pre-LN block of the fp32 layers (E = 512)
        _mix("block, fp32", "fwd", 8, 1024, 8, 64, "fp32", False, False),
        # the attention benchmark's batch
        _mix("batch, bf16", "fwd", 8, 4096, 16, 64, "bf16", False, False),
        # the attention benchmark's long sequences: few heads to share the GPU
        _mix("long, head dim 128", "fwd", 2, 16384, 16, 128, "bf16", False, True),
        _mix("batch gradient, bf16", "bwd", 8, 4096, 16, 64, "bf16", False, False),
        # a padded batch trained in pieces: lengths differ, states and their gradients carried
        _mix("ragged gradient, fp32", "bwd", 3, 1999, 8, 64, "fp32", True, True),
        _mix("long gradient, head dim 128", "bwd", 1, 8192, 16, 128, "bf16", False, False),
        # one user, and a serving batch
        _step("new token, one user", 1, 8, 64, "bf16"),
        _step("new tokens, 64 users", 64, 16, 128, "bf16"),
    ]


def _between(rng, lo, hi):
    """A whole number, spread over the logarithm of its range."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "mix", "mix", "step"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    D = rng.choice([64, 128]) if dtype == "bf16" else rng.choice([32, 64])
    H = rng.choice([1, 2, 4, 6, 8, 12, 16])
    if op == "step":
        c = _step("", _between(rng, 1, 64), H, D, dtype)
    elif op == "rope":
        pairs = D // 2 if rng.random() < 0.7 else D // 4
        axes = rng.choice([1, 2, 3])
        cuts = sorted(rng.sample(range(1, pairs), axes - 1))
        sections = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
        L = _between(rng, 1, 16384)
        B = _between(rng, 1, max(1, min(16, 32768 // L)))
        c = _rope("", rng.choice(["fwd", "bwd"]), B, L, H, rng.choice([h for h in (1, 2, 4, 6, 8, 12, 16) if H % h == 0]),
                  D, dtype, ",".join(map(str, sections)), rng.choice(["halves", "pairs"]),
                  rng.choice(["shared", "per_axis"]), rng.choice([64, 4096, 200000]))
    else:
        direction = rng.choice(["fwd", "bwd"])
        L = _between(rng, 1, 16384)
        most = (8 * 4096 * 16 * 64) // (L * H * D)
        if dtype == "fp32":
            most //= 2
        c = _mix("", direction, _between(rng, 1, max(1, min(16, most))), L, H, D, dtype,
                 rng.random() < 0.5, rng.random() < 0.5)
    del c["name"]
    return c


def _lengths(c):
    """Valid tokens of each sequence: all of them, or a padded batch whose sequences get shorter."""
    return [max(1, c["L"] * (c["B"] - b) // c["B"]) if c.get("ragged") else c["L"] for b in range(c["B"])]


def work(c):
    e = 2 if c["dtype"] == "bf16" else 4
    if c["op"] == "rope":
        values = c["B"] * c["L"] * (c["H"] + c["Hk"]) * c["D"]
        axes = len(c["sections"].split(","))
        return {"bytes": 2 * values * e + 4 * axes * c["B"] * c["L"], "flops": 3 * values}
    state = 4 * c["B"] * c["H"] * c["D"] * c["D"]
    if c["op"] == "step":
        token = c["B"] * c["H"] * c["D"] * e
        return {"bytes": 2 * state + 4 * token, "flops": 4 * c["B"] * c["H"] * c["D"] ** 2}
    tokens = sum(_lengths(c)) * c["H"]
    out = c["B"] * c["L"] * c["H"]
    if c["dir"] == "fwd":  # reads q, k, v; the recurrence updates the state and reads it
        return {"bytes": (3 * tokens + out) * c["D"] * e + (2 * state if c["states"] else state),
                "flops": 4 * tokens * c["D"] ** 2}
    # reads q, k, v, dO; two recurrences, and three reads of their states
    return {"bytes": (4 * tokens + 3 * out) * c["D"] * e + (3 * state if c["states"] else 0),
            "flops": 10 * tokens * c["D"] ** 2}


# ---------------------------------------------------------------- inputs
def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[c["dtype"]]

    def normal(*shape, std=1.0, dtype=t):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    B, H, D = c["B"], c["H"], c["D"]
    s = {"case": c}
    if c["op"] == "rope":
        L, sections = c["L"], [int(n) for n in c["sections"].split(",")]
        s["x"] = (normal(B, L, H, D), normal(B, L, c["Hk"], D))
        s["positions"] = torch.randint(0, c["far"], (len(sections), B, L), generator=g, device="cuda",
                                       dtype=torch.int32)
        s["sections"] = sections
        return s
    # heads that forget within a few tokens to heads that keep hundreds
    s["log_decay"] = -torch.exp2(-8.0 * torch.arange(1, H + 1, device="cuda", dtype=torch.float32) / H)
    if c["op"] == "step":
        s["q"], s["k"], s["v"] = (normal(B, 1, H, D, std=0.5) for _ in range(3))
        s["state"] = normal(B, H, D, D, dtype=torch.float32)
        s["next"] = torch.empty_like(s["state"])
        return s
    L = c["L"]
    s["q"], s["k"], s["v"] = (normal(B, L, H, D, std=0.5) for _ in range(3))
    s["lens"] = torch.tensor(_lengths(c), device="cuda", dtype=torch.int32) if c["ragged"] else None
    s["state"] = normal(B, H, D, D, dtype=torch.float32) if c["states"] else None
    if c["dir"] == "bwd":
        s["dO"] = normal(B, L, H, D, std=0.5)
        s["dstate"] = normal(B, H, D, D, dtype=torch.float32) if c["states"] else None
    return s


# ---------------------------------------------------------------- plain forms
def _angles(s):
    """cos and sin [B, L, 1, pairs]; far positions need 64 bits."""
    c, sections = s["case"], s["sections"]
    pairs = sum(sections)
    n = torch.tensor(sections, device="cuda")
    axis = torch.repeat_interleave(torch.arange(len(sections), device="cuda"), n, output_size=pairs)
    i = torch.arange(pairs, device="cuda", dtype=torch.float64)
    if c["freqs"] == "per_axis":
        first = torch.cumsum(n, 0) - n
        frac = (i - first[axis]) / n[axis]
    else:
        frac = i / pairs
    a = s["positions"].double()[axis].permute(1, 2, 0) * 10000.0 ** -frac
    return a.cos().float().unsqueeze(2), a.sin().float().unsqueeze(2)


def _plain_rope(s):
    c = s["case"]
    cos, sin = _angles(s)
    if c["dir"] == "bwd":
        sin = -sin
    P = cos.shape[-1]

    def turn(x):
        f = x.float()
        y = f.clone()
        a, b = (slice(0, P), slice(P, 2 * P)) if c["layout"] == "halves" else (slice(0, 2 * P, 2), slice(1, 2 * P, 2))
        y[..., a] = f[..., a] * cos - f[..., b] * sin
        y[..., b] = f[..., b] * cos + f[..., a] * sin
        return y.to(x.dtype)

    return turn(s["x"][0]), turn(s["x"][1])


def _chunks(q, k, v, n, ld, first, lead, C=128):
    """sum_{s <= t} decay^(t-s) (q_t . k_s) v_s + decay^(t+1-lead) q_t first, over [B, L, H, D] in
    chunks of C: within a chunk as a masked product, across chunks through the chunks' states."""
    B, L, H, D = q.shape
    nC = -(-L // C)
    valid = (torch.arange(L, device=q.device) < n[:, None])[:, :, None, None]
    k, v = torch.where(valid, k, 0), torch.where(valid, v, 0)

    def cut(x):
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, nC * C - L))
        return x.view(B, nC, C, H, -1).permute(0, 3, 1, 2, 4)

    qc, kc, vc = cut(q), cut(k), cut(v)
    r = torch.arange(C, device=q.device)
    d = (r[:, None] - r).float()
    inside = torch.where(d >= 0, torch.exp(d.clamp(min=0) * ld[:, None, None]), 0)
    o = ((qc @ kc.transpose(-1, -2)) * inside[:, None]) @ vc
    kv = (kc * torch.exp((C - 1 - r).float() * ld[:, None])[:, None, :, None]).transpose(-1, -2) @ vc
    e = torch.arange(nC, device=q.device)
    d = (e[:, None] - 1 - e).float()
    across = torch.where(d >= 0, torch.exp(d.clamp(min=0) * C * ld[:, None, None]), 0)
    before = (across @ kv.flatten(3)).view(B, H, nC, k.shape[-1], v.shape[-1])
    o = o + torch.exp((r + 1).float() * ld[:, None])[:, None, :, None] * (qc @ before)
    o = o.permute(0, 2, 3, 1, 4).reshape(B, nC * C, H, -1)[:, :L]
    if first is not None:
        t = torch.arange(L, device=q.device, dtype=torch.float32)
        o = o + torch.exp((t + 1 - lead)[:, None] * ld)[..., None] * torch.einsum("blhd,bhde->blhe", q, first)
    return torch.where(valid, o, 0)


def _sum_state(k, v, power, ld, n):
    """sum_s decay^power_s k_s v_s^T over the valid tokens, [B, H, D, D]; power [B, L]."""
    valid = torch.arange(k.shape[1], device=k.device) < n[:, None]
    w = torch.where(valid[..., None], torch.exp(power.float()[..., None] * ld), 0)
    return (torch.where(valid[..., None, None], k, 0) * w[..., None]).permute(0, 2, 3, 1) @ torch.where(
        valid[..., None, None], v, 0).permute(0, 2, 1, 3)


def _plain_mix(s):
    c, ld = s["case"], s["log_decay"]
    B, L, D = c["B"], c["L"], c["D"]
    scale = D ** -0.5
    q, k, v = (s[x].float() for x in "qkv")
    n = s["lens"] if s["lens"] is not None else torch.full((B,), L, device=q.device, dtype=torch.int32)
    t = torch.arange(L, device=q.device)
    kept = torch.exp(n.float()[:, None] * ld)[..., None, None]  # decay^n [B, H, 1, 1]
    typ = s["q"].dtype
    if c["dir"] == "fwd":
        o = scale * _chunks(q, k, v, n, ld, s["state"], 0)
        state = _sum_state(k, v, (n[:, None] - 1 - t).clamp(min=0), ld, n)
        if s["state"] is not None:
            state = state + kept * s["state"]
        return o.to(typ), state
    dO, ds = s["dO"].float(), s["dstate"]
    back = (n[:, None] - 1 - t)
    back = torch.where(back >= 0, back, t)[..., None, None].expand_as(q).long()  # each sequence's tokens reversed

    def rev(x):
        return torch.gather(x, 1, back)

    u = ds / scale if ds is not None else None
    dq = scale * _chunks(dO, v, k, n, ld, s["state"].transpose(-1, -2) if s["state"] is not None else None, 0)
    dv = scale * rev(_chunks(rev(k), rev(q), rev(dO), n, ld, u, 1))
    dk = scale * rev(_chunks(rev(v), rev(dO), rev(q), n, ld, u.transpose(-1, -2) if u is not None else None, 1))
    out = [dq.to(typ), dk.to(typ), dv.to(typ)]
    if ds is not None:
        out.append(scale * _sum_state(q, dO, (t + 1).expand(B, L), ld, n) + kept * ds)
    return out


def _plain_step(s):
    q, k, v = (s[x].float()[:, 0] for x in "qkv")
    state = torch.exp(s["log_decay"])[:, None, None] * s["state"] + k[..., :, None] * v[..., None, :]
    o = s["case"]["D"] ** -0.5 * (q[..., None, :] @ state)[..., 0, :]
    return o[:, None].to(s["q"].dtype), state


def run(s):
    c = s["case"]
    if not own:
        return {"rope": _plain_rope, "mix": _plain_mix, "step": _plain_step}[c["op"]](s)
    pa = _capi()
    if c["op"] == "rope":
        x, y = s["x"]
        desc = pa.rope_desc(x, y, s["sections"], layout=c["layout"], freqs=c["freqs"])
        xo, yo = torch.empty_like(x), torch.empty_like(y)
        (pa.rope_fwd if c["dir"] == "fwd" else pa.rope_bwd)(x, y, s["positions"], xo, yo, desc)
        return xo, yo
    if c["op"] == "step":
        o = torch.empty_like(s["q"])
        pa.linear_attn_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], o, s["next"])
        return o, s["next"]
    if c["dir"] == "fwd":
        o = torch.empty_like(s["q"])
        state = torch.empty(c["B"], c["H"], c["D"], c["D"], device="cuda")
        pa.linear_attn_fwd(s["q"], s["k"], s["v"], s["log_decay"], o, seq_lens=s["lens"],
                           state_in=s["state"], state_out=state)
        return o, state
    dq, dk, dv = (torch.empty_like(s["q"]) for _ in range(3))
    dstate = torch.empty_like(s["dstate"]) if s["dstate"] is not None else None
    pa.linear_attn_bwd(s["q"], s["k"], s["v"], s["dO"], s["log_decay"], dq, dk, dv, seq_lens=s["lens"],
                       state_in=s["state"], d_state_out=s["dstate"], d_state_in=dstate)
    return [dq, dk, dv] + ([dstate] if dstate is not None else [])


# ---------------------------------------------------------------- from the definitions, in 64 bits
def _exact_rope(s):
    c = s["case"]
    w = []
    for a, n in enumerate(s["sections"]):
        for i in range(n):
            f = i / n if c["freqs"] == "per_axis" else len(w) / sum(s["sections"])
            w.append(s["positions"][a].double() * math.pow(10000.0, -f))
    z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.stack(w, -1))[:, :, None]
    if c["dir"] == "bwd":
        z = z.conj()
    P = z.shape[-1]
    out = []
    for x in s["x"]:
        x = x.double()
        head, tail = x[..., :2 * P], x[..., 2 * P:]
        if c["layout"] == "halves":
            r = torch.complex(head[..., :P].contiguous(), head[..., P:].contiguous()) * z
            out.append(torch.cat([r.real, r.imag, tail], -1))
        else:
            r = torch.view_as_complex(head.reshape(*head.shape[:-1], P, 2).contiguous()) * z
            out.append(torch.cat([torch.view_as_real(r).flatten(-2), tail], -1))
    return tuple(out)


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "rope":
        return _exact_rope(s)
    q, k, v = (s[x].double() for x in "qkv")
    B, L, H, D = q.shape
    scale = D ** -0.5
    lam = torch.exp(s["log_decay"].double())[:, None, None]
    S = s["state"].double() if s["state"] is not None else torch.zeros(B, H, D, D, dtype=torch.float64, device="cuda")
    n = _lengths(c) if c["op"] == "mix" else [1] * B
    live = torch.tensor(n, device="cuda")[:, None] > torch.arange(L, device="cuda")  # [B, L]
    o, dq = torch.zeros_like(q), torch.zeros_like(q)
    bwd = c.get("dir") == "bwd"
    dO = s["dO"].double() if bwd else None
    ragged = bool(c.get("ragged"))
    for t in range(L):
        new = lam * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        S = torch.where(live[:, t, None, None, None], new, S) if ragged else new
        if bwd:
            dq[:, t] = scale * (S @ dO[:, t, :, :, None])[..., 0]
        else:
            o[:, t] = scale * (q[:, t, :, None, :] @ S)[..., 0, :]
    if not bwd:
        return o * live[..., None, None], S
    U = s["dstate"].double() if s["dstate"] is not None else torch.zeros_like(S)
    dk, dv = torch.zeros_like(q), torch.zeros_like(q)
    for t in reversed(range(L)):  # U: the gradient of the state after token t
        on = live[:, t, None, None, None]
        add = scale * q[:, t, :, :, None] * dO[:, t, :, None, :]
        new = U + add
        dk[:, t] = (new @ v[:, t, :, :, None])[..., 0]
        dv[:, t] = (k[:, t, :, None, :] @ new)[..., 0, :]
        new = lam * new
        U = torch.where(on, new, U) if ragged else new
    out = [x * live[..., None, None] for x in (dq, dk, dv)]
    return out + [U] if s["dstate"] is not None else out

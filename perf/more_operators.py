"""Sizes, plain forms and work of causal attention over packed prompts, of
attention over a paged cache, and of head norms with rotary positions.

Three operators of a causal model with shared key-value heads, beside the
bidirectional attention and the rotary positions that the framework has:

  packed  causal attention over sequences of different lengths laid end to end
          ([T, H, D] with cumulative lengths), heads of k and v shared by
          groups of q's heads: a batch of prompts, or a packed training batch
          with its gradients;
  paged   attention of one new token of each sequence over its cache, whose
          pages lie anywhere in a pool (serving);
  norm    the root-mean-square norm of each head of q and k, their rotary
          positions, and optionally k and v written into the cache's pages, in
          one pass; its backward.

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
_EPS = 1e-6


def _capi():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import pa_capi
    return pa_capi


# ---------------------------------------------------------------- cases
def _packed(name, direction, seqs, longest, ragged, H, Hk, D, fused):
    return {"name": name, "op": "packed", "dir": direction, "seqs": seqs, "longest": longest,
            "ragged": ragged, "H": H, "Hk": Hk, "D": D, "dtype": "bf16", "fused": fused}


def _paged(name, B, longest, ragged, H, Hk, D, dtype, page):
    return {"name": name, "op": "paged", "B": B, "longest": longest, "ragged": ragged, "H": H,
            "Hk": Hk, "D": D, "dtype": dtype, "page": page}


def _norm(name, kind, B, L, H, Hk, D, dtype, sections, layout, fused, page):
    return {"name": name, "op": "norm", "kind": kind, "B": B, "L": L, "H": H, "Hk": Hk, "D": D,
            "dtype": dtype, "sections": sections, "layout": layout, "fused": fused, "page": page}


def listed():
    return [
        # a short prompt of one user: latency counts
        _packed("prompt, 100 tokens", "fwd", 1, 100, False, 8, 2, 64, True),
        # prompts of 16 users in one call, from a few tokens to thousands, one of them empty
        _packed("prompts, ragged", "fwd", 16, 3907, True, 16, 2, 128, True),
        # the attention benchmark's long sequence, as a prompt
        _packed("long prompt", "fwd", 1, 16384, False, 16, 4, 128, False),
        # a packed training batch of the attention benchmark's heads
        _packed("packed gradient", "bwd", 8, 4096, True, 16, 16, 64, False),
        # a long document, shared heads
        _packed("long gradient, shared heads", "bwd", 1, 8192, False, 16, 4, 128, False),
        # one user's next token: latency counts
        _paged("new token, one user", 1, 1531, False, 8, 2, 64, "bf16", 16),
        # a serving batch, contexts of all lengths
        _paged("new tokens, 64 users", 64, 8192, True, 16, 4, 128, "bf16", 64),
        # few users far into long documents: the cache's length has to be shared out
        _paged("new tokens, long contexts", 2, 131072, False, 16, 2, 128, "bf16", 128),
        # the fp32 layers' heads, each with its own keys
        _paged("new tokens, fp32", 7, 3001, True, 8, 8, 64, "fp32", 32),
        # one new token of each of 16 sequences: normed, turned and into the cache
        _norm("norm to cache, new tokens", "cache", 16, 1, 8, 2, 64, "bf16", "32", "halves", True, 16),
        # q and k of a prompt batch, slices of one projection's output
        _norm("norm, batch", "fwd", 8, 4096, 16, 2, 128, "bf16", "64", "halves", True, 0),
        # gradients of the fp32 training path: images (height, width), odd length
        _norm("norm gradient, images", "bwd", 5, 1177, 8, 2, 64, "fp32", "16,16", "pairs", False, 0),
    ]


def _between(rng, lo, hi):
    """A whole number, spread over the logarithm of its range."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["packed", "packed", "paged", "norm"])
    Hk = rng.choice([1, 2, 3, 4, 8])
    H = Hk * rng.choice([1, 2, 3, 4, 8] if Hk <= 4 else [1, 2])
    if op == "packed":
        D, bwd = rng.choice([64, 128]), rng.random() < 0.5
        longest = _between(rng, 1, 8192 if bwd else 16384)
        scores = 8 * 16 * 4096 ** 2 * 64 // D if bwd else 16 * 16384 ** 2  # values of all heads' score matrices
        tokens = 65536 // max(1, H * D // 1024)
        seqs = _between(rng, 1, max(1, min(32, scores // (H * longest ** 2), tokens // longest)))
        while H * longest ** 2 * seqs > scores:
            longest = longest * 3 // 4
        c = _packed("", "bwd" if bwd else "fwd", seqs, longest, rng.random() < 0.7, H, Hk, D,
                    rng.random() < 0.5)
    elif op == "paged":
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        D = rng.choice([64, 128]) if dtype == "bf16" else rng.choice([32, 64])
        B = _between(rng, 1, 64)
        most = (64 * 8192 * 4 * 128) // (B * Hk * D * (1 if dtype == "bf16" else 2))
        c = _paged("", B, _between(rng, 1, min(131072, most)), rng.random() < 0.7, H, Hk, D, dtype,
                   rng.choice([16, 24, 32, 64, 128]))
    else:
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        D = rng.choice([64, 80, 128])
        kind = rng.choice(["fwd", "bwd", "cache"])
        pairs = D // 2 if rng.random() < 0.7 else D // 4
        cuts = sorted(rng.sample(range(1, pairs), rng.choice([0, 0, 1])))
        sections = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
        L = 1 if kind == "cache" and rng.random() < 0.5 else _between(rng, 1, 8192)
        most = (8 * 4096 * 18 * 128) // (L * (H + 2 * Hk) * D * (1 if dtype == "bf16" else 2))
        c = _norm("", kind, _between(rng, 1, max(1, min(64, most))), L, H, Hk, D, dtype,
                  ",".join(map(str, sections)), rng.choice(["halves", "pairs"]), rng.random() < 0.5,
                  rng.choice([16, 64]) if kind == "cache" else 0)
    del c["name"]
    return c


def _lengths(n, longest, ragged, empty):
    """Tokens of each sequence: all alike, or from few to `longest` in no order, some odd, one of
    them empty where that is asked for."""
    if not ragged:
        return [longest] * n
    lens = [max(1, longest * (i + 1) ** 2 // n ** 2) for i in range(n)]
    if empty and n > 3:
        lens[1] = 0
    return lens[1::2] + lens[0::2][::-1]


def _lens(c):
    n = c["seqs"] if c["op"] == "packed" else c["B"]
    return _lengths(n, c["longest"], c["ragged"], c["op"] == "packed")


def work(c):
    e = 2 if c["dtype"] == "bf16" else 4
    H, Hk, D = c["H"], c["Hk"], c["D"]
    if c["op"] == "packed":
        T, pairs = sum(_lens(c)), sum(n * (n + 1) // 2 for n in _lens(c))
        q, k = T * H * D * e, T * Hk * D * e
        if c["dir"] == "fwd":  # q, k, v in, o out; q.k and p.v
            return {"bytes": 2 * q + 2 * k + 4 * H * T, "flops": 4 * pairs * H * D}
        # q, k, v, o, dO in, dq, dk, dv out; five products
        return {"bytes": 4 * q + 4 * k + 4 * H * T, "flops": 10 * pairs * H * D}
    if c["op"] == "paged":
        keys = sum(_lens(c))
        return {"bytes": 2 * keys * Hk * D * e + 2 * c["B"] * H * D * e + 4 * sum(-(-n // c["page"]) for n in _lens(c)),
                "flops": 4 * keys * H * D}
    tokens = c["B"] * c["L"]
    x = tokens * (H + Hk) * D * e
    angles = 4 * tokens * len(c["sections"].split(","))
    if c["kind"] == "bwd":  # x and the gradient in, the gradient out
        return {"bytes": 3 * x + angles, "flops": 12 * tokens * (H + Hk) * D}
    v = 2 * tokens * Hk * D * e if c["kind"] == "cache" else 0
    return {"bytes": 2 * x + v + angles, "flops": 7 * tokens * (H + Hk) * D}


# ---------------------------------------------------------------- inputs
def _pages(c, g, lens):
    """Page numbers of each sequence's tokens [B, most pages], from a pool in random order, -1
    behind a sequence's last page; and the pool's size (a few pages belong to no one)."""
    per = [-(-n // c["page"]) for n in lens]
    width, used = max(1, max(per)), sum(per)
    pool = torch.randperm(used + 3, generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    n = torch.tensor(per, device="cuda")
    first = torch.cumsum(n, 0) - n
    at = torch.arange(width, device="cuda")
    table = torch.where(at < n[:, None], pool[(first[:, None] + at).clamp(max=used + 2)], -1)
    return table.to(torch.int32), used + 3


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[c["dtype"]]

    def normal(*shape, std=1.0, dtype=t):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    def qkv(*lead):
        """q, k, v [..., heads, D]: slices of one projection's output, or tensors of their own."""
        sizes = (H, Hk, Hk)
        if c["fused"]:
            parts = normal(*lead, (H + 2 * Hk) * D).split([n * D for n in sizes], -1)
            return [x.unflatten(-1, (n, D)) for x, n in zip(parts, sizes)]
        return [normal(*lead, n, D) for n in sizes]

    H, Hk, D = c["H"], c["Hk"], c["D"]
    s = {"case": c}
    if c["op"] == "packed":
        lens = _lens(c)
        T = sum(lens)
        s["q"], s["k"], s["v"] = qkv(T)
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        s["cu"] = torch.tensor(cu, device="cuda", dtype=torch.int32)
        if c["dir"] == "bwd":
            s["dO"] = normal(T, H, D)
            # a training step has o and lse from its forward
            with torch.no_grad():
                s["o"], s["lse"] = _plain_packed_fwd(s)
        return s
    if c["op"] == "paged":
        lens = _lens(c)
        s["table"], pages = _pages(c, g, lens)
        s["lens"] = torch.tensor(lens, device="cuda", dtype=torch.int32)
        s["q"] = normal(c["B"], H, D)
        s["k_cache"], s["v_cache"] = (normal(pages, c["page"], Hk, D) for _ in range(2))
        return s
    B, L, sections = c["B"], c["L"], [int(n) for n in c["sections"].split(",")]
    s["sections"] = sections
    s["q"], s["k"], s["v"] = qkv(B, L)
    s["positions"] = torch.randint(0, 100000, (len(sections), B, L), generator=g, device="cuda", dtype=torch.int32)
    s["gq"], s["gk"] = (1 + normal(D, std=0.1, dtype=torch.float32) for _ in range(2))
    if c["kind"] == "bwd":
        s["dq_out"], s["dk_out"] = normal(B, L, H, D), normal(B, L, Hk, D)
    if c["kind"] == "cache":
        # each sequence's tokens in pages of its own, the new ones behind `before` older ones
        before = 1000 if L == 1 else 0
        lens = [before + L] * B
        table, pages = _pages(c, g, lens)
        at = before + torch.arange(L, device="cuda")
        s["slots"] = (table[:, at // c["page"]] * c["page"] + at % c["page"]).to(torch.int32)
        s["k_cache"], s["v_cache"] = (normal(pages, c["page"], Hk, D) for _ in range(2))
    return s


# ---------------------------------------------------------------- plain forms
def _rows(s):
    """Token of each row of the padded batch [n, Lmax], whether there is one, and each token's
    sequence and place."""
    c, cu = s["case"], s["cu"].long()
    T, Lm = s["q"].shape[0], max(_lens(c))
    r = torch.arange(Lm, device="cuda")
    valid = r < (cu[1:] - cu[:-1])[:, None]
    rows = (cu[:-1, None] + r).clamp(max=T - 1)
    t = torch.arange(T, device="cuda")
    seq = torch.bucketize(t, cu[1:], right=True)
    return rows, valid, seq, t - cu[seq]


def _probabilities(s, rows, valid):
    """Causal softmax of the padded batch [n, H, Lmax, Lmax] and its row log-sums."""
    c = s["case"]
    G = c["H"] // c["Hk"]
    q = s["q"].float()[rows].transpose(1, 2) * c["D"] ** -0.5
    k = s["k"].float()[rows].transpose(1, 2).repeat_interleave(G, 1)
    x = q @ k.transpose(-1, -2)
    r = torch.arange(rows.shape[1], device="cuda")
    x.masked_fill_((r > r[:, None]) | ~valid[:, None, None, :], -torch.inf)
    m = x.amax(-1, keepdim=True).clamp(min=-1e30)
    x.sub_(m).exp_()
    total = x.sum(-1, keepdim=True).clamp(min=1e-30)
    return x.div_(total), (m + total.log())[..., 0]


def _plain_packed_fwd(s):
    c = s["case"]
    rows, valid, seq, at = _rows(s)
    p, lse = _probabilities(s, rows, valid)
    v = s["v"].float()[rows].transpose(1, 2).repeat_interleave(c["H"] // c["Hk"], 1)
    v = torch.where(valid[:, None, :, None], v, 0)
    o = (p @ v)[seq, :, at]  # [T, H, D]
    return o.to(s["q"].dtype), lse[seq, :, at].t().contiguous()


def _plain_packed_bwd(s):
    c = s["case"]
    G, n, scale = c["H"] // c["Hk"], c["seqs"], c["D"] ** -0.5
    rows, valid, seq, at = _rows(s)
    p, _ = _probabilities(s, rows, valid)
    on = valid[:, None, :, None]
    k, v = (torch.where(on, s[x].float()[rows].transpose(1, 2), 0).repeat_interleave(G, 1) for x in "kv")
    q, dO, o = (torch.where(on, s[x].float()[rows].transpose(1, 2), 0) for x in ("q", "dO", "o"))
    dv = p.transpose(-1, -2) @ dO
    ds = dO @ v.transpose(-1, -2)
    ds.sub_((dO * o).sum(-1, keepdim=True)).mul_(p)
    dq = scale * (ds @ k)
    dk = scale * (ds.transpose(-1, -2) @ q)
    dk, dv = (x.view(n, c["Hk"], G, *x.shape[2:]).sum(2) for x in (dk, dv))
    return [x[seq, :, at].to(s["q"].dtype) for x in (dq, dk, dv)]


def _plain_paged(s):
    c = s["case"]
    B, H, Hk, D = c["B"], c["H"], c["Hk"], c["D"]
    pages = s["table"].clamp(min=0).long()
    k, v = (s[x][pages].flatten(1, 2).float() for x in ("k_cache", "v_cache"))  # [B, S, Hk, D]
    on = torch.arange(k.shape[1], device="cuda") < s["lens"][:, None]
    q = s["q"].float().view(B, Hk, H // Hk, D) * D ** -0.5
    x = q @ k.permute(0, 2, 3, 1)
    x = x.masked_fill(~on[:, None, None], -torch.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    v = torch.where(on[..., None, None], v, 0)
    o = (x @ v.transpose(1, 2)) / x.sum(-1, keepdim=True)
    return o.view(B, H, D).to(s["q"].dtype)


def _turned(s, x, inverse):
    """x (fp32) turned by its tokens' positions; the angles of far positions need 64 bits."""
    c, sections = s["case"], s["sections"]
    P = sum(sections)
    n = torch.tensor(sections, device="cuda")
    axis = torch.repeat_interleave(torch.arange(len(sections), device="cuda"), n, output_size=P)
    i = torch.arange(P, device="cuda", dtype=torch.float64)
    a = s["positions"].double()[axis].permute(1, 2, 0) * 10000.0 ** -(i / P)
    cos, sin = a.cos().float().unsqueeze(2), a.sin().float().unsqueeze(2)
    if inverse:
        sin = -sin
    y = x.clone()
    a, b = (slice(0, P), slice(P, 2 * P)) if c["layout"] == "halves" else (slice(0, 2 * P, 2), slice(1, 2 * P, 2))
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    return y


def _inverse_rms(x):
    return torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)


def _plain_norm(s):
    c = s["case"]
    q, k = s["q"].float(), s["k"].float()
    if c["kind"] == "bwd":
        def back(x, gamma, dy):
            r, dn = _inverse_rms(x), _turned(s, dy.float(), True)
            xhat, u = x * r, dn * gamma
            dx = r * (u - xhat * (u * xhat).mean(-1, keepdim=True))
            # long sums of many tokens
            return dx.to(dy.dtype), (dn * xhat).sum((0, 1, 2), dtype=torch.float64).float()
        (dq, dgq), (dk, dgk) = back(q, s["gq"], s["dq_out"]), back(k, s["gk"], s["dk_out"])
        return dq, dk, dgq, dgk
    qo = _turned(s, q * _inverse_rms(q) * s["gq"], False).to(s["q"].dtype)
    ko = _turned(s, k * _inverse_rms(k) * s["gk"], False).to(s["k"].dtype)
    if c["kind"] == "fwd":
        return qo, ko
    slots = s["slots"].flatten().long()
    s["k_cache"].view(-1, c["Hk"], c["D"])[slots] = ko.flatten(0, 1)
    s["v_cache"].view(-1, c["Hk"], c["D"])[slots] = s["v"].flatten(0, 1)
    return qo, s["k_cache"], s["v_cache"]


def _own_packed(s):
    c, pa = s["case"], _capi()
    T, H = s["q"].shape[:2]
    if c["dir"] == "fwd":
        o = torch.empty(T, H, c["D"], dtype=s["q"].dtype, device="cuda")
        lse = torch.empty(H, T, device="cuda")
        pa.packed_attn_fwd(s["q"], s["k"], s["v"], s["cu"], o, lse)
        return o, lse
    dq, dk, dv = (torch.empty(x.shape, dtype=x.dtype, device="cuda") for x in (s["q"], s["k"], s["v"]))
    pa.packed_attn_bwd(s["q"], s["k"], s["v"], s["o"], s["dO"], s["lse"], s["cu"], dq, dk, dv)
    return [dq, dk, dv]


def _own_paged(s):
    o = torch.empty_like(s["q"])
    _capi().paged_attn_step(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], o)
    return o


def _own_norm(s):
    c, pa = s["case"], _capi()
    q, k = s["q"], s["k"]
    d = pa.rope_desc(q, k, s["sections"], layout=c["layout"])
    new = lambda x: torch.empty(x.shape, dtype=x.dtype, device="cuda")  # noqa: E731
    if c["kind"] == "bwd":
        dq, dk, dgq, dgk = new(q), new(k), new(s["gq"]), new(s["gk"])
        pa.qk_norm_rope_bwd(s["dq_out"], s["dk_out"], q, k, s["gq"], s["gk"], s["positions"], dq, dk, dgq, dgk, d,
                            eps=_EPS)
        return dq, dk, dgq, dgk
    qo = new(q)
    if c["kind"] == "cache":
        pa.qk_norm_rope_cache(q, k, s["v"], s["gq"], s["gk"], s["positions"], s["slots"], qo, s["k_cache"],
                              s["v_cache"], d, eps=_EPS)
        return qo, s["k_cache"], s["v_cache"]
    ko = new(k)
    pa.qk_norm_rope_fwd(q, k, s["gq"], s["gk"], s["positions"], qo, ko, d, eps=_EPS)
    return qo, ko


def run(s):
    c = s["case"]
    if own:
        return {"packed": _own_packed, "paged": _own_paged, "norm": _own_norm}[c["op"]](s)
    if c["op"] == "packed":
        return (_plain_packed_fwd if c["dir"] == "fwd" else _plain_packed_bwd)(s)
    return (_plain_paged if c["op"] == "paged" else _plain_norm)(s)


# ---------------------------------------------------------------- from the definitions, in 64 bits
def _exact_packed(s):
    """One sequence and head after the other."""
    c, cu = s["case"], s["cu"].tolist()
    G, bwd = c["H"] // c["Hk"], c["dir"] == "bwd"
    scale = 1.0 / math.sqrt(c["D"])
    names = ("q", "k", "v") + (("dO",) if bwd else ())
    x = {n: s[n].double() for n in names}
    out = {n: torch.zeros_like(x[n]) for n in "qkv"}  # gradients; "q" holds o of a forward
    lse = torch.zeros(c["H"], x["q"].shape[0], dtype=torch.float64, device="cuda")
    for a, b in zip(cu, cu[1:]):
        if a == b:
            continue
        future = torch.ones(b - a, b - a, dtype=torch.bool, device="cuda").triu(1)
        for h in range(c["H"]):
            q, k, v = x["q"][a:b, h], x["k"][a:b, h // G], x["v"][a:b, h // G]
            w = torch.where(future, -math.inf, scale * (q @ k.T))
            z = torch.logsumexp(w, 1)
            w = torch.exp(w - z[:, None])
            if not bwd:
                out["q"][a:b, h], lse[h, a:b] = w @ v, z
                continue
            dO = x["dO"][a:b, h]
            out["v"][a:b, h // G] += w.T @ dO
            dp = dO @ v.T
            dw = w * (dp - (w * dp).sum(1, keepdim=True))
            out["q"][a:b, h] = scale * (dw @ k)
            out["k"][a:b, h // G] += scale * (dw.T @ q)
    return [out["q"], out["k"], out["v"]] if bwd else (out["q"], lse)


def _exact_paged(s):
    c = s["case"]
    G, S = c["H"] // c["Hk"], c["page"]
    o = torch.zeros(c["B"], c["H"], c["D"], dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        t = torch.arange(n, device="cuda")
        at = s["table"][b, t // S].long(), t % S
        k, v = s["k_cache"][at].double(), s["v_cache"][at].double()
        for h in range(c["H"]):
            w = torch.softmax(k[:, h // G] @ s["q"][b, h].double() / math.sqrt(c["D"]), 0)
            o[b, h] = w @ v[:, h // G]
    return o


def _exact_norm(s):
    c = s["case"]
    w = [s["positions"][a].double() * 10000.0 ** (-i / sum(s["sections"])) for i, a in
         enumerate(a for a, n in enumerate(s["sections"]) for _ in range(n))]
    z = torch.stack(w, -1)[:, :, None]
    z = torch.polar(torch.ones_like(z), z)
    P = z.shape[-1]

    def turn(x, z):
        head, tail = x[..., :2 * P], x[..., 2 * P:]
        if c["layout"] == "halves":
            r = torch.complex(head[..., :P].contiguous(), head[..., P:].contiguous()) * z
            return torch.cat([r.real, r.imag, tail], -1)
        r = torch.view_as_complex(head.reshape(*head.shape[:-1], P, 2).contiguous()) * z
        return torch.cat([torch.view_as_real(r).flatten(-2), tail], -1)

    def normed(x, gamma):
        return turn(x / torch.sqrt(x.square().mean(-1, keepdim=True) + _EPS) * gamma, z)

    q, k, gq, gk = (s[n].double() for n in ("q", "k", "gq", "gk"))
    if c["kind"] == "bwd":
        with torch.enable_grad():
            leaves = [x.detach().clone().requires_grad_() for x in (q, k, gq, gk)]
            total = (normed(leaves[0], leaves[2]) * s["dq_out"].double()).sum()
            total = total + (normed(leaves[1], leaves[3]) * s["dk_out"].double()).sum()
            return tuple(torch.autograd.grad(total, leaves))
    if c["kind"] == "fwd":
        return normed(q, gq), normed(k, gk)
    caches = [s["k_cache"].double(), s["v_cache"].double()]
    slots = s["slots"].long()
    for cache, x in zip(caches, (normed(k, gk), s["v"].double())):
        cache[slots // c["page"], slots % c["page"]] = x
    return normed(q, gq), caches[0], caches[1]


def exact(c, seed):
    s = prepare(c, seed)
    return {"packed": _exact_packed, "paged": _exact_paged, "norm": _exact_norm}[c["op"]](s)

"""Head norms with rotary positions, through the C ABI against their 64-bit form.

Per value, with m = |n_a| + |n_b| of its pair of normed values: the output's rounding; the
rotation's 2^-21 m (as for the rotary positions alone); r = (mean x^2 + eps)^-1/2 from a sum of
positive terms in chains of at most 32 fp32 additions, 2^-20, rsqrt's 2^-22 and three
products: together 2^-19 m. Gradients: the same of every term of u - x r^2 mean(u x), 2^-18 of
their magnitudes; dgamma: fp32 sums in chains of at most 400 terms, 2^-15 of the magnitudes."""
import pytest

torch = pytest.importorskip("torch")
import causal_ref as ref  # noqa: E402
from seq_ref import turn  # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32
STEP = {BF16: 2.0 ** -8, F32: 2.0 ** -24}
EPS = 1e-6
pytestmark = pytest.mark.gpu

CASES = [  # B, L, H, Hk, D, sections, layout, freqs, slices
    (1, 1, 1, 1, 64, [32], "halves", "shared", False),
    (16, 1, 8, 2, 64, [32], "halves", "shared", True),
    (3, 37, 4, 2, 128, [64], "halves", "shared", True),
    (2, 129, 6, 1, 128, [20, 22, 22], "pairs", "per_axis", False),
    (2, 33, 3, 3, 64, [8, 8], "halves", "per_axis", True),     # half of each head turns
    (1, 50, 5, 1, 64, [3, 4, 1, 5], "pairs", "shared", False),  # runs that are no whole vectors
    (1, 61, 2, 2, 80, [22, 18], "halves", "shared", True),
    (2, 7, 3, 1, 8, [1, 2], "halves", "shared", False),
    (1, 900, 16, 4, 256, [128], "halves", "shared", True),
    (1, 70, 2, 1, 256, [1], "pairs", "shared", False),          # nearly all passes through
    (1, 70, 2, 1, 256, [3], "halves", "shared", False),
    (5, 1177, 8, 2, 64, [16, 16], "pairs", "per_axis", False),
    (1, 30, 5, 0, 128, [64], "halves", "shared", False),        # no k
]


def _data(case, dtype, seed=0):
    B, L, H, Hk, D, sections, layout, freqs, fused = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = (normal(B, L, (H + 2 * Hk) * D) * torch.exp(normal(B, L, 1))).to(dtype)
    parts = x.split([H * D, Hk * D, Hk * D], -1)
    q, k, v = (p.unflatten(-1, (n, D)) if fused else p.reshape(B, L, n, D) for p, n in zip(parts, (H, Hk, Hk)))
    pos = torch.randint(-70000, 70000, (len(sections), B, L), generator=g, device="cuda", dtype=torch.int32)
    gq, gk = (1 + 0.3 * normal(D) for _ in range(2))
    dq, dk = normal(B, L, H, D).to(dtype), normal(B, L, Hk, D).to(dtype)
    import pa_capi
    desc = pa_capi.rope_desc(q, k if Hk else None, sections, layout=layout, freqs=freqs)
    if not Hk:
        k = v = gk = dk = None
    return q, k, v, pos, gq, gk, dq, dk, desc


def _pair_sum(x, case):
    """|x_a| + |x_b| of each value's pair."""
    sections, layout = case[5], case[6]
    P, m = sum(sections), x.abs()
    y = m.clone()
    a, b = (slice(0, P), slice(P, 2 * P)) if layout == "halves" else (slice(0, 2 * P, 2), slice(1, 2 * P, 2))
    y[..., a] = y[..., b] = m[..., a] + m[..., b]
    return y


def _near(got, want, mag, rel, step):
    off = (got.double() - want).abs() - (step * want.abs() + rel * mag)
    assert torch.isfinite(got.double()).all() and off.max() <= 0, float(off.max())


def _forward_ok(y, x, gamma, pos, case, eps=EPS):
    n = ref.rms(x, gamma, eps)
    want = turn(n, pos, case[5], layout=case[6], freqs=case[7])
    _near(y, want, _pair_sum(n, case), 2.0 ** -19, STEP[x.dtype])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", CASES)
def test_forward_matches_formula(case, dtype):
    import pa_capi
    q, k, _, pos, gq, gk, _, _, desc = _data(case, dtype)
    new = lambda x: None if x is None else torch.full(x.shape, float("nan"), dtype=dtype, device="cuda")  # noqa: E731
    for a, b in ((gq, gk), (None, gk), (gq, None)):
        qo, ko = new(q), new(k)
        pa_capi.qk_norm_rope_fwd(q, k, a, b, pos, qo, ko, desc, EPS)
        for y, x, gamma in ((qo, q, a), (ko, k, b)):
            if x is not None:
                _forward_ok(y, x, gamma, pos, case)
    # in place
    q1, k1 = (None if x is None else x.contiguous().clone() for x in (q, k))
    pa_capi.qk_norm_rope_fwd(q1, k1, gq, None, pos, q1, k1, desc, EPS)
    _forward_ok(q1, q, gq, pos, case)
    assert k is None or torch.equal(k1, ko)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", CASES)
def test_gradients_match_formula(case, dtype):
    import pa_capi
    q, k, _, pos, gq, gk, dqo, dko, desc = _data(case, dtype, 1)

    def formula(x, gamma, dy):
        """dx, dgamma and the magnitudes of their terms."""
        x, dy = x.double(), dy.double()
        dn = turn(dy, pos, case[5], layout=case[6], freqs=case[7], inverse=True)
        mag = _pair_sum(dy, case)  # bounds |dn|
        if gamma is None:
            return dn, None, mag, None
        gamma = gamma.double()
        r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        u = dn * gamma
        dx = r * (u - x * r ** 2 * (u * x).mean(-1, keepdim=True))
        mu = mag * gamma.abs()
        return (dx, (dn * x * r).sum((0, 1, 2)), r * (mu + x.abs() * r ** 2 * (mu * x.abs()).mean(-1, keepdim=True)),
                (mag * x.abs() * r).sum((0, 1, 2)))

    for a, b, add in ((gq, gk, False), (gq, gk, True), (None, gk, False)):
        old = 0.5 if add else float("nan")
        dq, dk, dgq, dgk = (None if x is None else torch.full(x.shape, old, dtype=x.dtype, device="cuda")
                            for x in (q, k, a, b))
        pa_capi.qk_norm_rope_bwd(dqo, dko, q, k, a, b, pos, dq, dk, dgq, dgk, desc, EPS, accumulate=add)
        for x, gamma, dy, dx, dg in ((q, a, dqo, dq, dgq), (k, b, dko, dk, dgk)):
            if x is None:
                continue
            wx, wg, mx, mg = formula(x, gamma, dy)
            _near(dx, wx + 0.5 * add, mx, 2.0 ** -18, STEP[dtype])
            if gamma is not None:
                _near(dg, wg + 0.5 * add, mg, 2.0 ** -15, 2.0 ** -22)
    # in place, and with the weights' gradients not wanted
    g1, h1 = dqo.clone(), None if dko is None else dko.clone()
    pa_capi.qk_norm_rope_bwd(g1, h1, q, k, None, gk, pos, g1, h1, None, None, desc, EPS)
    assert torch.equal(g1, dq) and (dk is None or torch.equal(h1, dk))


def test_gradients_against_differences():
    """fp32: the loss moved along random directions of each input, in float64 from the kernel's outputs."""
    import pa_capi
    case = (2, 9, 3, 1, 64, [16, 16], "halves", "shared", False)
    q, k, _, pos, gq, gk, dqo, dko, desc = _data(case, F32, 3)
    q, k = (x / x.square().mean(-1, keepdim=True).sqrt() for x in (q, k))
    grads = [torch.empty_like(x) for x in (q, k, gq, gk)]
    pa_capi.qk_norm_rope_bwd(dqo, dko, q, k, gq, gk, pos, *grads, desc, EPS)

    def loss(q, k, gq, gk):
        qo, ko = torch.empty_like(q), torch.empty_like(k)
        pa_capi.qk_norm_rope_fwd(q, k, gq, gk, pos, qo, ko, desc, EPS)
        return (qo.double() * dqo.double()).sum() + (ko.double() * dko.double()).sum()

    for i, gr in enumerate(grads):
        x = [q, k, gq, gk]
        d = torch.randn(gr.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i))
        d = d + torch.sign(gr)
        h = 2.0 ** -7
        up, down = ([y + s * h * d if j == i else y for j, y in enumerate(x)] for s in (1, -1))
        along = (gr.double() * (up[i].double() - down[i].double())).sum()
        change = loss(*up) - loss(*down)
        # third derivatives times h^2, and fp32 roundings of the outputs over h
        assert abs(change - along) <= 0.01 * abs(along), (i, float(change), float(along))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", [c for c in CASES if c[3]])
def test_cache_holds_the_turned_keys_and_values(case, dtype):
    import pa_capi
    B, L, H, Hk, D = case[:5]
    q, k, v, pos, gq, gk, _, _, desc = _data(case, dtype, 4)
    page, T = 16, B * L
    pages = -(-T // page) + 2
    g = torch.Generator(device="cuda").manual_seed(5)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:T].to(torch.int32).view(B, L)
    if T > 4:  # tokens that are not stored
        flat = slots.view(-1)
        flat[1], flat[2], flat[-1] = -1, pages * page, 2 ** 31 - 1
    kc, vc = (torch.full((pages, page, Hk, D), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    qo, ko = torch.empty(q.shape, dtype=dtype, device="cuda"), torch.empty(k.shape, dtype=dtype, device="cuda")
    q1, k1 = torch.empty_like(qo), torch.empty_like(ko)
    pa_capi.qk_norm_rope_fwd(q, k, gq, gk, pos, q1, k1, desc, EPS)
    for out in (ko, None):
        kc.fill_(7.0), vc.fill_(7.0)
        pa_capi.qk_norm_rope_cache(q, k, v, gq, gk, pos, slots, qo, kc, vc, desc, EPS, k_out=out)
        assert torch.equal(qo, q1) and (out is None or torch.equal(out, k1))
        s = slots.flatten().long()
        on = (s >= 0) & (s < pages * page)
        wk, wv = torch.full_like(kc, 7.0), torch.full_like(vc, 7.0)
        wk.view(-1, Hk, D)[s[on]] = k1.view(T, Hk, D)[on]
        wv.view(-1, Hk, D)[s[on]] = v.reshape(T, Hk, D)[on]
        assert torch.equal(kc, wk) and torch.equal(vc, wv)


def test_zero_rows_and_rows_that_are_not_finite():
    """A head of zeros is normed to zeros; a NaN or infinity stays in its head."""
    import pa_capi
    case = (1, 40, 4, 2, 64, [32], "halves", "shared", False)
    q, k, _, pos, gq, gk, dqo, dko, desc = _data(case, BF16, 6)
    q[0, 3, 1] = 0
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    pa_capi.qk_norm_rope_fwd(q, k, gq, gk, pos, qo, ko, desc, EPS)
    assert (qo[0, 3, 1] == 0).all()
    _forward_ok(qo, q, gq, pos, case)
    q1 = q.clone()
    q1[0, 5, 2, 7], q1[0, 6, 0, 1] = float("nan"), float("inf")
    q2 = torch.empty_like(q)
    pa_capi.qk_norm_rope_fwd(q1, k, gq, gk, pos, q2, ko, desc, EPS)
    same = torch.ones(40, 4, dtype=torch.bool, device="cuda")
    same[5, 2] = same[6, 0] = False
    assert torch.equal(q2[0][same], qo[0][same])


def test_runs_repeat_and_workspaces_may_hold_anything():
    import pa_capi
    case = (3, 700, 4, 2, 128, [64], "halves", "shared", True)
    q, k, _, pos, gq, gk, dqo, dko, desc = _data(case, BF16, 7)
    outs = []
    for fill in (0, 255, 127):
        ws = torch.full((1 << 23,), fill, dtype=torch.uint8, device="cuda")
        out = [torch.empty(x.shape, dtype=x.dtype, device="cuda") for x in (q, k, gq, gk)]
        pa_capi.qk_norm_rope_bwd(dqo, dko, q, k, gq, gk, pos, *out, desc, EPS, workspace=ws)
        outs.append(out)
    for out in outs[1:]:
        for x, y in zip(out, outs[0]):
            assert torch.equal(x, y)


def test_captured_calls_follow_rewritten_inputs():
    import pa_capi
    case = (2, 65, 4, 2, 64, [32], "halves", "shared", False)
    q, k, v, pos, gq, gk, dqo, dko, desc = _data(case, BF16, 8)
    kc, vc = (torch.zeros(20, 16, 2, 64, dtype=BF16, device="cuda") for _ in range(2))
    slots = torch.arange(130, device="cuda", dtype=torch.int32).view(2, 65)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    grads = [torch.empty_like(x) for x in (q, k, gq, gk)]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        pa_capi.qk_norm_rope_cache(q, k, v, gq, gk, pos, slots, qo, kc, vc, desc, EPS, k_out=ko)
        pa_capi.qk_norm_rope_bwd(dqo, dko, q, k, gq, gk, pos, *grads, desc, EPS)
    for seed in (8, 9):
        new = _data(case, BF16, seed)
        for x, y in zip((q, k, v, pos, gq, gk, dqo, dko), new):
            x.copy_(y)
        slots.add_(7)
        graph.replay()
        q1, k1 = torch.empty_like(q), torch.empty_like(k)
        pa_capi.qk_norm_rope_fwd(q, k, gq, gk, pos, q1, k1, desc, EPS)
        assert torch.equal(qo, q1) and torch.equal(ko, k1)
        assert torch.equal(kc.view(-1, 2, 64)[slots.flatten().long()], k1.view(-1, 2, 64))
        want = [torch.empty_like(x) for x in (q, k, gq, gk)]
        pa_capi.qk_norm_rope_bwd(dqo, dko, q, k, gq, gk, pos, *want, desc, EPS)
        for x, y in zip(grads, want):
            assert torch.equal(x, y)


def test_offsets_past_32_bits():
    """Tokens whose offsets pass 2^31 values, and a cache row there."""
    import pa_capi
    L, H, D, wide = 34000, 2, 64, 65536
    big = torch.empty(1, L, wide, dtype=BF16, device="cuda")
    case = (1, L, H, 1, D, [32], "halves", "shared", False)
    q, k, v, pos, gq, gk, _, _, desc = _data(case, BF16, 10)
    views = [big[..., i * 256:i * 256 + n * D].unflatten(-1, (n, D)) for i, n in enumerate((H, 1, 1))]
    for x, y in zip(views, (q, k, v)):
        x.copy_(y)
    rows = 2 ** 31 // D + 40000
    kc, vc = (torch.empty(rows, 1, 1, D, dtype=BF16, device="cuda") for _ in range(2))
    slots = (rows - 1 - torch.arange(L, device="cuda", dtype=torch.int64)).to(torch.int32).view(1, L)
    qo, ko, q1, k1 = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q), torch.empty_like(k)
    pa_capi.qk_norm_rope_fwd(q, k, gq, gk, pos, q1, k1, desc, EPS)
    pa_capi.qk_norm_rope_cache(*views, gq, gk, pos, slots, qo, kc, vc, desc, EPS, k_out=ko)
    assert torch.equal(qo, q1) and torch.equal(ko, k1)
    assert torch.equal(kc[rows - L:].flip(0).view(L, D), k1.view(L, D))
    assert torch.equal(vc[rows - L:].flip(0).view(L, D), v.view(L, D))

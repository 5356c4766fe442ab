"""Rotary positions through the C ABI against their 64-bit form.

Tolerance per value, with m = |x_a| + |x_b| of its pair: the output's rounding
(bf16 2^-8, fp32 2^-24 of the value), and for cosine and sine an angle held as an
fp32 fraction of a turn (2^-25 of a turn at most half, i.e. 2 pi 2^-26 = 9.4e-8),
sincospi's 2 ulp (2^-22) and two fp32 products and a sum (3 x 2^-24): together
under 2^-21 m."""
import pytest

torch = pytest.importorskip("torch")
from seq_ref import turn  # noqa: E402

STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _data(B, L, H, D, dtype, axes, far, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, L, H, D, generator=g).to(dtype).cuda()
    pos = torch.randint(-far, far, (axes, B, L), generator=g, dtype=torch.int32).cuda()
    return x, pos


def _check(y, x, want, sections, layout):
    P = sum(sections)
    m = x.double().abs()
    pair = m.clone()
    a, b = (slice(0, P), slice(P, 2 * P)) if layout == "halves" else (slice(0, 2 * P, 2), slice(1, 2 * P, 2))
    pair[..., a] = pair[..., b] = m[..., a] + m[..., b]
    tol = STEP[y.dtype] * want.abs() + 2.0 ** -21 * pair
    tol[..., 2 * P:] = 0  # passed through as it is
    assert ((y.double() - want).abs() <= tol).all()


CASES = [  # B, L, Hq, Hk, D, sections, layout, freqs, far
    (2, 1, 8, 8, 64, [32], "halves", "shared", 1 << 18),
    (1, 1, 1, 1, 128, [64], "pairs", "shared", 2 ** 31 - 1),
    (3, 37, 4, 2, 64, [8, 12, 12], "halves", "shared", 64),
    (2, 129, 6, 1, 128, [20, 22, 22], "pairs", "per_axis", 4096),
    (2, 33, 3, 3, 64, [8, 8], "halves", "per_axis", 100),        # half of each head turns
    (1, 50, 5, 1, 64, [3, 4, 1, 5], "pairs", "shared", 1000),     # runs that are no whole vectors
    (1, 50, 2, 2, 48, [5, 6], "halves", "per_axis", 1000),
    (2, 7, 3, 1, 6, [1, 2], "pairs", "shared", 50),               # heads smaller than a vector
    (1, 5, 2, 1, 7, [3], "halves", "shared", 50),                 # odd head size
    (1, 3000, 16, 4, 256, [128], "halves", "shared", 200000),     # several tokens a block
    (5, 1777, 2, 1, 64, [16, 16], "pairs", "per_axis", 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", CASES)
def test_rope_matches_formula(case, dtype):
    import pa_capi
    B, L, Hq, Hk, D, sections, layout, freqs, far = case
    q, pos = _data(B, L, Hq, D, dtype, len(sections), far, 1)
    k, _ = _data(B, L, Hk, D, dtype, 1, 2, 2)
    desc = pa_capi.rope_desc(q, k, sections, layout=layout, freqs=freqs)
    qo, ko = torch.full_like(q, float("nan")), torch.full_like(k, float("nan"))
    pa_capi.rope_fwd(q, k, pos, qo, ko, desc)
    for x, y in ((q, qo), (k, ko)):
        _check(y, x, turn(x, pos, sections, layout=layout, freqs=freqs), sections, layout)
    # the gradient turns back, overwriting or adding
    pa_capi.rope_bwd(q, k, pos, qo, ko, desc)
    for x, y in ((q, qo), (k, ko)):
        _check(y, x, turn(x, pos, sections, layout=layout, freqs=freqs, inverse=True), sections, layout)
    q0, k0 = torch.randn_like(q), torch.randn_like(k)
    q1, k1 = q0.clone(), k0.clone()
    pa_capi.rope_bwd(q, k, pos, q1, k1, desc, accumulate=True)
    for y, y0, x in ((q1, q0, q), (k1, k0, k)):
        want = y0.double() + turn(x, pos, sections, layout=layout, freqs=freqs, inverse=True)
        tol = STEP[dtype] * want.abs() + 2.0 ** -20 * (y0.double().abs() + 2 * x.double().abs().amax())
        assert ((y.double() - want).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["halves", "pairs"])
def test_rope_in_place_and_q_alone(layout):
    import pa_capi
    q, pos = _data(2, 300, 4, 64, torch.float32, 2, 500, 3)
    k, _ = _data(2, 300, 2, 64, torch.float32, 1, 2, 4)
    sections = [10, 22]
    desc = pa_capi.rope_desc(q, k, sections, layout=layout)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    pa_capi.rope_fwd(q, k, pos, qo, ko, desc)
    a, b = q.clone(), k.clone()
    pa_capi.rope_fwd(a, b, pos, a, b, desc)
    assert torch.equal(a, qo) and torch.equal(b, ko)
    alone = torch.empty_like(q)
    pa_capi.rope_fwd(q, None, pos, alone, None, pa_capi.rope_desc(q, None, sections, layout=layout))
    assert torch.equal(alone, qo)


@pytest.mark.gpu
def test_rope_gradient_is_the_adjoint_and_products_depend_on_distance():
    """<turn(x), y> = <x, turn^-1(y)> (differences: the turn is linear), and with one axis
    q.k depends on the distance of the positions alone, far out as well."""
    import pa_capi
    x, pos = _data(2, 65, 4, 128, torch.float32, 3, 1 << 20, 5)
    y = torch.randn_like(x)
    sections = [16, 24, 24]
    desc = pa_capi.rope_desc(x, None, sections)
    tx, ty = torch.empty_like(x), torch.empty_like(x)
    pa_capi.rope_fwd(x, None, pos, tx, None, desc)
    pa_capi.rope_bwd(y, None, pos, ty, None, desc)
    a, b = (tx.double() * y.double()).sum(), (x.double() * ty.double()).sum()
    assert abs(a - b) <= 2.0 ** -20 * (x.double().abs() * y.double().abs()).sum()
    q, _ = _data(1, 1, 1, 64, torch.float32, 1, 2, 6)
    q = q.expand(1, 2, 1, 64).contiguous()
    dots = []
    for start in (0, 123456789):
        p = torch.tensor([[[start, start + 77]]], dtype=torch.int32, device="cuda")
        out = torch.empty_like(q)
        pa_capi.rope_fwd(q, None, p, out, None, pa_capi.rope_desc(q))
        dots.append((out[0, 0, 0].double() * out[0, 1, 0].double()).sum())
    assert abs(dots[0] - dots[1]) <= 2.0 ** -19 * (q[0, 0, 0].double() ** 2).sum()


@pytest.mark.gpu
def test_rope_on_a_stream_and_in_a_graph():
    import pa_capi
    q, pos = _data(2, 64, 4, 64, torch.bfloat16, 1, 1000, 7)
    desc = pa_capi.rope_desc(q)
    want, out = torch.empty_like(q), torch.empty_like(q)
    pa_capi.rope_fwd(q, None, pos, want, None, desc)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pa_capi.rope_fwd(q, None, pos, out, None, desc)
    out.fill_(0)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.gpu
def test_rope_past_2_31_values():
    import pa_capi
    B, L, H, D = 1, (1 << 19) + 77, 64, 64
    q = torch.zeros(B, L, H, D, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(9)
    tail = torch.randn(B, 90, H, D, generator=g).bfloat16().cuda()
    q[:, -90:] = tail
    pos = torch.arange(L, dtype=torch.int32, device="cuda").reshape(1, 1, L)
    pa_capi.rope_fwd(q, None, pos, q, None, pa_capi.rope_desc(q))
    want = turn(tail, pos[:, :, -90:], [32])
    _check(q[:, -90:], tail, want, [32], "halves")
    assert not q[:, :-90].any()


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,sections", [(64, [8, 16]), (128, [64]), (50, [3, 7]), (7, [2]), (130, [9])])
def test_rope_in_place_in_every_form(dtype, layout, D, sections):
    """Whole vectors and single values, forward and gradient: an output over its own input gives the bits
    of one beside it. With heads of 130 a thread takes several groups of four, one after another."""
    import pa_capi
    q, pos = _data(2, 290, 16, D, dtype, len(sections), 3000, 10)
    k, _ = _data(2, 290, 3, D, dtype, 1, 2, 11)
    desc = pa_capi.rope_desc(q, k, sections, layout=layout)
    for turn_by in (pa_capi.rope_fwd, pa_capi.rope_bwd):
        qo, ko = torch.empty_like(q), torch.empty_like(k)
        turn_by(q, k, pos, qo, ko, desc)
        a, b = q.clone(), k.clone()
        turn_by(a, b, pos, a, b, desc)
        assert torch.equal(a, qo) and torch.equal(b, ko)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Hq,Hk,D,sections", [(70, 9, 256, [60, 68]), (1, 11, 130, [9]), (40, 40, 90, [20, 25])])
def test_rope_more_heads_than_a_block_takes_at_once(dtype, layout, Hq, Hk, D, sections):
    """A thread then goes through several groups of four heads with the angles of the first, from q on into k."""
    import pa_capi
    q, pos = _data(2, 190, Hq, D, dtype, len(sections), 5000, 12)
    k, _ = _data(2, 190, Hk, D, dtype, 1, 2, 13)
    desc = pa_capi.rope_desc(q, k, sections, layout=layout)
    qo, ko = torch.full_like(q, float("nan")), torch.full_like(k, float("nan"))
    pa_capi.rope_fwd(q, k, pos, qo, ko, desc)
    for x, y in ((q, qo), (k, ko)):
        _check(y, x, turn(x, pos, sections, layout=layout), sections, layout)
    pa_capi.rope_bwd(q, k, pos, qo, ko, desc)
    for x, y in ((q, qo), (k, ko)):
        _check(y, x, turn(x, pos, sections, layout=layout, inverse=True), sections, layout)

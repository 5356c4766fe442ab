"""Causal attention over packed sequences with shared key-value heads, through the
C ABI against its 64-bit form (bounds in causal_ref.packed, plus the rounding of
each output)."""
import pytest

torch = pytest.importorskip("torch")
import causal_ref as ref  # noqa: E402

BF16 = torch.bfloat16
pytestmark = pytest.mark.gpu


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda").to(BF16)


def _inputs(lens, H, Hk, D, seed=0, before=0, behind=0, fused=False, fill=float("nan")):
    """q, k, v, cu of sequences behind `before` and in front of `behind` tokens of no sequence."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = before + sum(lens) + behind
    x = _normal(g, T, (H + 2 * Hk) * D)
    x[:before] = fill
    x[T - behind:] = fill
    parts = x.split([H * D, Hk * D, Hk * D], 1)
    qkv = [p.unflatten(1, (n, D)) if fused else p.reshape(T, n, D) for p, n in zip(parts, (H, Hk, Hk))]
    cu = torch.cumsum(torch.tensor([before] + lens), 0).to(torch.int32).cuda()
    return (*qkv, cu)


def _fwd(q, k, v, cu, **kw):
    import pa_capi
    o = torch.full(q.shape, 7.0, dtype=BF16, device="cuda")
    lse = torch.full((q.shape[1], q.shape[0]), 7.0, device="cuda")
    pa_capi.packed_attn_fwd(q, k, v, cu, o, lse, **kw)
    return o, lse


def _bwd(q, k, v, cu, dO, fill=7.0, o=None, lse=None, **kw):
    import pa_capi
    if o is None:
        o, lse = _fwd(q, k, v, cu)
    dq, dk, dv = (torch.full(x.shape, fill, dtype=BF16, device="cuda") for x in (q, k, v))
    pa_capi.packed_attn_bwd(q, k, v, o, dO, lse, cu, dq, dk, dv, **kw)
    return dq, dk, dv


def _near(got, want, bound, step=2.0 ** -8):
    off = (got.double() - want).abs() - (bound + step * want.abs())
    assert torch.isfinite(got.double()).all() and off.max() <= 0, float(off.max())


CASES = [  # lens, H, Hk, D, tokens before and behind, slices of one tensor
    ([1], 1, 1, 64, 0, 0, False),
    ([1, 0, 2, 1], 2, 1, 128, 0, 0, True),
    ([100], 8, 2, 64, 0, 0, True),
    ([127, 128, 129], 4, 2, 64, 3, 5, False),
    ([255, 0, 256, 257], 3, 1, 128, 0, 9, True),
    ([513, 64, 0, 300], 6, 3, 64, 1, 0, False),
    ([5, 700, 31], 8, 1, 128, 2, 130, True),
    ([1025], 5, 5, 64, 0, 0, True),
    ([640, 641], 4, 4, 128, 0, 1, False),
    ([0, 0, 17], 16, 2, 64, 0, 0, False),
    ([3] * 70 + [260], 2, 2, 64, 0, 0, True),
    ([1500], 12, 4, 128, 0, 0, False),
]


@pytest.mark.parametrize("case", CASES)
def test_forward_matches_formula(case):
    lens, H, Hk, D, before, behind, fused = case
    q, k, v, cu = _inputs(lens, H, Hk, D, 1, before, behind, fused)
    o, lse = _fwd(q, k, v, cu)
    (want, bound), (wl, bl) = ref.packed(q, k, v, lens, before)
    a, b = before, before + sum(lens)
    _near(o[a:b], want[a:b], bound[a:b])
    _near(lse[:, a:b], wl[:, a:b], bl[:, a:b], 2.0 ** -22)
    for x in (o[:a], o[b:], lse[:, :a], lse[:, b:]):  # tokens of no sequence stay as they were
        assert (x == 7).all()


@pytest.mark.parametrize("case", CASES)
def test_gradients_match_formula(case):
    lens, H, Hk, D, before, behind, fused = case
    q, k, v, cu = _inputs(lens, H, Hk, D, 2, before, behind, fused)
    a, b = before, before + sum(lens)
    dO = _normal(torch.Generator(device="cuda").manual_seed(3), *q.shape)
    dO[:a] = dO[b:] = float("nan")
    o, lse = _fwd(q, k, v, cu)
    want = ref.packed(q, k, v, lens, before, dO, o)
    got = _bwd(q, k, v, cu, dO, o=o, lse=lse)
    for x, (w, bound) in zip(got, want):
        _near(x[a:b], w[a:b], bound[a:b])
        assert (x[:a] == 7).all() and (x[b:] == 7).all()
    # added to what is there
    got = _bwd(q, k, v, cu, dO, 0.5, o, lse, accumulate=True)
    for x, (w, bound) in zip(got, want):
        _near(x[a:b], 0.5 + w[a:b], bound[a:b])
        assert (x[:a] == 0.5).all() and (x[b:] == 0.5).all()


def test_gradients_against_differences():
    """The loss sum(o * w), moved along a direction of each input. The difference of two outputs keeps
    their roundings: 2^-8 of the loss's terms each, over the step."""
    lens, H, Hk, D = [70, 131], 4, 2, 64
    q, k, v, cu = _inputs(lens, H, Hk, D, 5)
    w = _normal(torch.Generator(device="cuda").manual_seed(6), *q.shape)
    grads = _bwd(q, k, v, cu, w)
    step = 0.25
    for i, gr in enumerate(grads):
        d = torch.sign(gr.float())  # along the gradient: the change stands out of the roundings
        moved = []
        for s in (step, -step):
            x = [q, k, v]
            x[i] = (x[i].float() + s * d * 0.1).to(BF16)
            moved.append((_fwd(*x, cu)[0].double(), x[i].double()))
        change = ((moved[0][0] - moved[1][0]) * w.double()).sum()
        along = (gr.double() * (moved[0][1] - moved[1][1])).sum()
        # curvature and roundings: a tenth, which the sign or a factor of two would not pass
        assert abs(change - along) <= 0.1 * abs(along), (i, float(change), float(along))


def test_gradient_into_slices_of_one_tensor():
    lens, H, Hk, D = [130, 7], 4, 2, 64
    q, k, v, cu = _inputs(lens, H, Hk, D, 7, fused=True)
    dO = _normal(torch.Generator(device="cuda").manual_seed(8), *q.shape)
    want = _bwd(q, k, v, cu, dO)
    import pa_capi
    o, lse = _fwd(q, k, v, cu)
    one = torch.zeros(q.shape[0], (H + 2 * Hk) * D, dtype=BF16, device="cuda")
    parts = [p.unflatten(1, (n, D)) for p, n in zip(one.split([H * D, Hk * D, Hk * D], 1), (H, Hk, Hk))]
    pa_capi.packed_attn_bwd(q, k, v, o, dO, lse, cu, *parts)
    for x, w in zip(parts, want):
        assert torch.equal(x, w)


@pytest.mark.parametrize("D,H,Hk", [(64, 4, 2), (128, 3, 3)])
def test_other_sequences_keep_their_bits(D, H, Hk):
    """NaN and infinities in one sequence, and in tokens of none, reach no other sequence; within a
    sequence they reach no o and dq of a block of 128 tokens before theirs."""
    lens = [140, 300, 90]
    q, k, v, cu = _inputs(lens, H, Hk, D, 9, 1, 60, fill=0.0)
    dO = _normal(torch.Generator(device="cuda").manual_seed(10), *q.shape)
    o, lse = _fwd(q, k, v, cu)
    grads = _bwd(q, k, v, cu, dO, o=o, lse=lse)
    for bad in (float("nan"), float("inf")):
        x = [t.clone() for t in (q, k, v, dO)]
        for t in x:
            t[:1] = t[531:] = bad
            t[141 + 130:141 + 140] = bad  # in the second block of the second sequence
        o1, lse1 = _fwd(*x[:3], cu)
        for lo, hi in ((1, 141), (141, 141 + 128), (441, 531)):
            assert torch.equal(o1[lo:hi], o[lo:hi]) and torch.equal(lse1[:, lo:hi], lse[:, lo:hi])
        g1 = _bwd(*x[:3], cu, x[3], o=o1, lse=lse1)
        for y, w in zip(g1, grads):
            assert torch.equal(y[1:141], w[1:141]) and torch.equal(y[441:531], w[441:531])
        assert torch.equal(g1[0][141:269], grads[0][141:269])


def test_large_scores_and_scale():
    """Scores far apart: rows that keep one key, and scores whose exponentials would overflow."""
    lens, H, Hk, D = [260], 2, 1, 64
    q, k, v, cu = _inputs(lens, H, Hk, D, 11)
    q = (q.float() * 30).to(BF16)
    o, lse = _fwd(q, k, v, cu)
    (want, bound), (wl, bl) = ref.packed(q, k, v, lens)
    _near(o, want, bound)
    _near(lse, wl, bl, 2.0 ** -22)
    # the scale as an argument
    q1 = (q.float() * 0.25).to(BF16)
    o1, lse1 = _fwd(q1, k, v, cu, scale=4 * D ** -0.5)
    assert torch.equal(o1, o) and torch.allclose(lse1, lse, rtol=2.0 ** -20)


def test_runs_repeat_bit_for_bit_and_workspaces_may_hold_anything():
    import pa_capi
    lens, H, Hk, D = [900, 3, 411, 0, 200], 8, 2, 64
    q, k, v, cu = _inputs(lens, H, Hk, D, 12)
    dO = _normal(torch.Generator(device="cuda").manual_seed(13), *q.shape)
    d = pa_capi.packed_attn_desc(q, k, v, cu)
    o, lse = _fwd(q, k, v, cu)
    first = _bwd(q, k, v, cu, dO, o=o, lse=lse)
    for fill in (0, 255, 127):
        ws = torch.full((pa_capi.packed_attn_fwd_workspace_size(d),), fill, dtype=torch.uint8, device="cuda")
        o1, lse1 = _fwd(q, k, v, cu, workspace=ws)
        assert torch.equal(o1, o) and torch.equal(lse1, lse)
        ws = torch.full((pa_capi.packed_attn_bwd_workspace_size(d),), fill, dtype=torch.uint8, device="cuda")
        for x, w in zip(_bwd(q, k, v, cu, dO, o=o, lse=lse, workspace=ws), first):
            assert torch.equal(x, w)


def test_captured_calls_follow_rewritten_inputs_and_lengths():
    import pa_capi
    H, Hk, D = 4, 2, 64
    q, k, v, cu = _inputs([200, 56, 300], H, Hk, D, 14)
    dO = _normal(torch.Generator(device="cuda").manual_seed(15), *q.shape)
    o, lse = torch.empty_like(q), torch.empty(H, q.shape[0], device="cuda")
    grads = [torch.empty_like(x) for x in (q, k, v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        pa_capi.packed_attn_fwd(q, k, v, cu, o, lse)
        pa_capi.packed_attn_bwd(q, k, v, o, dO, lse, cu, *grads)
    for lens in ([200, 56, 300], [1, 554, 1], [0, 556, 0]):
        q2, k2, v2, cu2 = _inputs(lens, H, Hk, D, 16 + lens[0])
        for x, y in ((q, q2), (k, k2), (v, v2), (cu, cu2)):
            x.copy_(y)
        graph.replay()
        o2, lse2 = _fwd(q2, k2, v2, cu2)
        assert torch.equal(o, o2) and torch.equal(lse, lse2)
        for x, w in zip(grads, _bwd(q2, k2, v2, cu2, dO, o=o2, lse=lse2)):
            assert torch.equal(x, w)


def test_two_streams_at_once():
    q, k, v, cu = _inputs([800, 31], 8, 2, 128, 17)
    want = _fwd(q, k, v, cu)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(_fwd(q, k, v, cu))
    got.append(_fwd(q, k, v, cu, stream=streams[0].cuda_stream))
    torch.cuda.synchronize()
    for o, lse in got[:-1]:
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])


def test_offsets_past_32_bits():
    """Tokens so far apart that their offsets pass 2^31 values."""
    T, D, wide = 34000, 64, 65536
    big = torch.empty(T, wide, dtype=BF16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(18)
    small = [_normal(g, T, 1, D) for _ in range(3)]
    views = [big[:, i * D:(i + 1) * D].unflatten(1, (1, D)) for i in range(6)]
    for x, y in zip(views, small):
        x.copy_(y)
    cu = torch.tensor([*range(0, 33900, 300), 33900, T], dtype=torch.int32, device="cuda")
    dO = _normal(g, T, 1, D)
    want, got = _fwd(*small, cu), _fwd(*views[:3], cu)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    import pa_capi
    ws = _bwd(*small, cu, dO, o=want[0], lse=want[1])
    pa_capi.packed_attn_bwd(*views[:3], want[0], dO, want[1], cu, *views[3:])
    for x, w in zip(views[3:], ws):
        assert torch.equal(x, w)


def test_lengths_out_of_bounds_stay_in_bounds():
    """Entries past the tokens, below zero or descending are clamped; sequences apart from them hold."""
    q, k, v, _ = _inputs([400], 2, 1, 64, 19)
    for cu, lens, first in (([-5, 130, 9999], [130, 270], 0), ([100, 50, 300], [0, 200], 100), ([400, 400], [0], 400)):
        o, lse = _fwd(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"))
        (want, bound), _ = ref.packed(q, k, v, lens, first)
        a, b = first, first + sum(lens)
        assert (o[:a] == 7).all() and (o[b:] == 7).all()
        if b > a:
            _near(o[a:b], want[a:b], bound[a:b])


@pytest.mark.parametrize("H, Hk, D", [(16, 16, 64), (16, 16, 128), (24, 8, 64)])
def test_more_work_than_the_gpu_holds_at_once(H, Hk, D):
    """Several items for each CTA, of long and short sequences, full and ragged."""
    lens = [300, 0, 77, 640, 129, 512, 33, 255, 1, 128]
    q, k, v, cu = _inputs(lens, H, Hk, D, 20, fused=True)
    dO = _normal(torch.Generator(device="cuda").manual_seed(21), *q.shape)
    o, lse = _fwd(q, k, v, cu)
    (want, bound), (wl, bl) = ref.packed(q, k, v, lens, 0)
    _near(o, want, bound)
    _near(lse, wl, bl, 2.0 ** -22)
    for x, (w, b) in zip(_bwd(q, k, v, cu, dO, o=o, lse=lse), ref.packed(q, k, v, lens, 0, dO, o)):
        _near(x, w, b)


def test_calls_after_a_failed_wait_leave_their_outputs():
    """While the device's status word is set, the kernels skip their work; cleared, they run."""
    import pa_capi
    q, k, v, cu = _inputs([200, 77], 4, 2, 64, 22)
    dO = _normal(torch.Generator(device="cuda").manual_seed(23), *q.shape)
    want = _fwd(q, k, v, cu)
    grads = _bwd(q, k, v, cu, dO, o=want[0], lse=want[1])
    assert pa_capi.device_status() == 0
    pa_capi.wait_selftest(100_000_000, arrive=False)
    skipped = [*_fwd(q, k, v, cu), *_bwd(q, k, v, cu, dO, o=want[0], lse=want[1])]
    assert pa_capi.device_status(clear=True) == 6  # PA_ERR_TIMEOUT
    for x in skipped:
        assert (x == 7).all()
    again = [*_fwd(q, k, v, cu), *_bwd(q, k, v, cu, dO, o=want[0], lse=want[1])]
    assert pa_capi.device_status() == 0
    for x, y in zip(again, [*want, *grads]):
        assert torch.equal(x, y)


@pytest.mark.parametrize("lens, T, H, Hk, D", [
    ([5, 0, 130, 1], 140, 8, 2, 64),              # as many units as the GPU has SMs at most: no list
    ([0] * 15 + [200], 200, 4, 4, 128),
    ([0] * 16 + [200], 200, 4, 4, 128),           # one sequence more: a list
    ([16, 0, 3, 128, 129], 276, 16, 16, 64),      # (units and heads on both sides of 148)
    ([16, 0, 3, 128, 129], 276, 24, 8, 64),
    ([1] * 9, 9, 12, 3, 128),
])
def test_few_units_and_many_sequences(lens, T, H, Hk, D):
    """Small calls, which find their work without a list, and the same sizes with one."""
    q, k, v, cu = _inputs(lens, H, Hk, D, 24)
    assert q.shape[0] == sum(lens) <= T
    dO = _normal(torch.Generator(device="cuda").manual_seed(25), *q.shape)
    o, lse = _fwd(q, k, v, cu)
    (want, bound), (wl, bl) = ref.packed(q, k, v, lens, 0)
    _near(o, want, bound)
    _near(lse, wl, bl, 2.0 ** -22)
    for x, (w, b) in zip(_bwd(q, k, v, cu, dO, o=o, lse=lse), ref.packed(q, k, v, lens, 0, dO, o)):
        _near(x, w, b)


@pytest.mark.parametrize("D", [64, 128])
def test_many_sequences_of_one_tile(D):
    """Items of one tile, several to a CTA: an item's sums are read while the next one's are computed."""
    lens, H = [700] + [90, 128, 1, 33] * 25, 12
    q, k, v, cu = _inputs(lens, H, H, D, 26)
    dO = _normal(torch.Generator(device="cuda").manual_seed(27), *q.shape)
    o, lse = _fwd(q, k, v, cu)
    (want, bound), _ = ref.packed(q, k, v, lens, 0)
    _near(o, want, bound)
    want = ref.packed(q, k, v, lens, 0, dO, o)
    for _ in range(10):
        for x, (w, b) in zip(_bwd(q, k, v, cu, dO, o=o, lse=lse), want):
            _near(x, w, b)

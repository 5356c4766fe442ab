"""Attention of one new token of each sequence over its paged cache, through the C ABI
against its 64-bit form (bounds in causal_ref.paged)."""
import pytest

torch = pytest.importorskip("torch")
import causal_ref as ref  # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32
STEP = {BF16: 2.0 ** -8, F32: 2.0 ** -24}
pytestmark = pytest.mark.gpu


def _cache(lens, page, Hk, D, dtype, seed=0, spare=3, width=0, stale=float("nan")):
    """Pools in which each sequence's tokens lie in pages of random numbers; every other place of the
    pools is `stale`; table entries behind a sequence's pages name no page or a stale one."""
    g = torch.Generator().manual_seed(seed)
    per = [-(-n // page) for n in lens]
    pages = sum(per) + spare
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(1, width, *per)), -1, dtype=torch.int32)
    kc, vc = (torch.full((pages, page, Hk, D), stale, dtype=dtype) for _ in range(2))
    at = 0
    for b, n in enumerate(lens):
        mine = order[at:at + per[b]]
        at += per[b]
        table[b, :per[b]] = mine
        table[b, per[b]:] = int(order[-1]) if b % 2 else -1
        for i, p in enumerate(mine.tolist()):
            m = min(page, n - i * page)
            for c in (kc, vc):
                c[p, :m] = torch.randn(m, Hk, D, generator=g).to(dtype)
    return kc.cuda(), vc.cuda(), table.cuda()


def _query(B, H, D, dtype, seed, wide=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(B, (H + wide) * D, generator=g).to(dtype).cuda()
    return q[:, :H * D].unflatten(1, (H, D)) if wide else q.view(B, H, D)


def _step(q, kc, vc, table, lens, **kw):
    import pa_capi
    o, lse = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda"), torch.full(q.shape[:2], 7.0, device="cuda")
    pa_capi.paged_attn_step(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), o, lse, **kw)
    return o, lse


def _check(q, kc, vc, table, lens, o, lse, reads=None):
    page = kc.shape[1]
    for b, n in enumerate(lens):
        n = max(0, min(n, table.shape[1] * page))
        t = torch.arange(n, device="cuda")
        p = table[b, t // page].long()
        on = (p >= 0) & (p < kc.shape[0])
        k, v = (c[p.clamp(0, kc.shape[0] - 1), t % page] for c in (kc, vc))
        k, v = (torch.where(on[:, None, None], x, 0) for x in (k, v))
        want, bound, wl = ref.paged(q[b], k, v, on, STEP[BF16] if q.dtype is BF16 else 0.0)
        assert torch.isfinite(o[b].double()).all()
        off = (o[b].double() - want).abs() - (bound + STEP[q.dtype] * want.abs())
        assert off.max() <= 0, (b, n, float(off.max()))
        if on.any():
            assert ((lse[b].double() - wl).abs() <= 2.0 ** -16 * (1 + wl.abs())).all()
        else:
            assert (o[b] == 0).all() and (lse[b] == -torch.inf).all()


CASES = [  # lens, page, H, Hk, D of bf16 (fp32: half), slices
    ([1], 16, 1, 1, 64, 0),
    ([0, 1, 2, 15, 16, 17], 16, 8, 2, 64, 5),
    ([100, 0, 333], 24, 4, 4, 128, 0),
    ([63, 64, 65, 127, 128, 129], 64, 6, 2, 128, 1),
    ([1000, 7], 1, 3, 3, 64, 0),
    ([500, 499], 7, 16, 1, 128, 0),
    ([2047], 128, 24, 3, 64, 2),
    ([4000, 5], 96, 40, 2, 64, 0),     # 20 heads of q to one of k
    ([300], 300, 72, 1, 128, 0),       # 72
    ([9000], 64, 2, 1, 128, 0),
    ([30] * 300, 16, 4, 2, 64, 0),     # more sequences than blocks
    ([20000, 1, 0, 700, 3], 32, 8, 8, 64, 0),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", CASES)
def test_step_matches_formula(case, dtype):
    lens, page, H, Hk, D, wide = case
    D = D if dtype is BF16 else D // 2
    kc, vc, table = _cache(lens, page, Hk, D, dtype, 1)
    q = _query(len(lens), H, D, dtype, 2, wide)
    o, lse = _step(q, kc, vc, table, lens)
    _check(q, kc, vc, table, lens, o, lse)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_pages_that_are_none_are_left_out(dtype):
    """Numbers below zero and past the pool, at the beginning, inside and at the end; a sequence of
    none but such pages; and lengths past the table and below zero."""
    lens = [200, 200, 64, 40, 128]
    kc, vc, table = _cache(lens, 16, 2, 64, dtype, 3, width=13)
    table[0, 0] = -1
    table[0, 5] = kc.shape[0]
    table[0, 12] = 2 ** 31 - 1
    table[1, 1:12] = -2 ** 31
    table[2, :] = -1
    table[4, 2:6] = kc.shape[0] + 7
    q = _query(5, 4, 64, dtype, 4)
    o, lse = _step(q, kc, vc, table, lens)
    _check(q, kc, vc, table, lens, o, lse)
    lens = [2 ** 31 - 1, -5, -2 ** 31, 40, 500]
    table[0, 6:] = table[4, 8:] = -1
    last = torch.where((table[0] >= 0) & (table[0] < kc.shape[0]))[0][-1]
    kc[table[0, last]], vc[table[0, last]] = 1.0, 2.0
    o, lse = _step(q, kc, vc, table, lens)
    _check(q, kc, vc, table, lens, o, lse)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_large_scores_and_infinite_masks(dtype):
    """One key far above the others, wherever it lies; keys of -infinity scores are as if masked."""
    lens = [700, 700, 700]
    kc, vc, table = _cache(lens, 32, 1, 64, dtype, 5)
    q = _query(3, 2, 64, dtype, 6) * 20
    for b, t in ((0, 0), (1, 350), (2, 699)):
        kc[table[b, t // 32], t % 32] = (q[b, 0].float() * 0.5).to(dtype)
    o, lse = _step(q, kc, vc, table, lens)
    _check(q, kc, vc, table, lens, o, lse)


def test_runs_repeat_and_workspaces_may_hold_anything():
    import pa_capi
    lens = [5000, 3, 0, 900, 64, 2222]
    kc, vc, table = _cache(lens, 64, 2, 128, BF16, 7)
    q = _query(6, 8, 128, BF16, 8)
    o, lse = _step(q, kc, vc, table, lens)
    n = pa_capi.paged_attn_step_workspace_size(pa_capi.paged_attn_desc(q, kc, table))
    for fill in (0, 255, 127):
        ws = torch.full((n,), fill, dtype=torch.uint8, device="cuda")
        o1, lse1 = _step(q, kc, vc, table, lens, workspace=ws)
        assert torch.equal(o, o1) and torch.equal(lse, lse1)
    # without lse
    o1 = torch.empty_like(o)
    pa_capi.paged_attn_step(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), o1)
    assert torch.equal(o, o1)


def test_captured_step_follows_growing_lengths():
    import pa_capi
    lens = [70, 1, 500]
    kc, vc, table = _cache([900] * 3, 16, 2, 64, BF16, 9)
    q = _query(3, 8, 64, BF16, 10)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    o = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        pa_capi.paged_attn_step(q, kc, vc, table, n, o)
    for grow in (0, 1, 15, 399):
        now = [x + grow for x in lens]
        n.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        want, lse = _step(q, kc, vc, table, now)
        assert torch.equal(o, want)
        _check(q, kc, vc, table, now, want, lse)


def test_two_streams_at_once():
    lens = [3000, 1700]
    kc, vc, table = _cache(lens, 64, 2, 128, BF16, 11)
    q = _query(2, 8, 128, BF16, 12)
    want = _step(q, kc, vc, table, lens)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(_step(q, kc, vc, table, lens))
    torch.cuda.synchronize()
    for o, lse in got:
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])


def test_pages_past_32_bit_offsets():
    """The last pages of a pool of more than 2^31 values."""
    Hk, D, page = 16, 128, 128
    pages = 2 ** 31 // (Hk * D * page) + 5
    kc, vc = (torch.zeros(pages, page, Hk, D, dtype=BF16, device="cuda") for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(13)
    for c in (kc, vc):
        c[-3:] = torch.randn(3, page, Hk, D, generator=g, device="cuda").to(BF16)
    table = torch.tensor([[pages - 1, pages - 3, pages - 2]], dtype=torch.int32, device="cuda")
    q = _query(1, 32, D, BF16, 14)
    o, lse = _step(q, kc, vc, table, [300])
    _check(q, kc, vc, table, [300], o, lse)

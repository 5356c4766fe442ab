"""Causal attention and head norms where they can go wrong beyond their own files' cases: scores of
-infinity, more items than SMs in every form, thousands of sequences, workspaces that are used again at once,
streams given by handle, errors recorded while kernels run, gradients of a whole training batch."""
import math

import pytest

torch = pytest.importorskip("torch")
import causal_ref as ref  # noqa: E402
from seq_ref import turn  # noqa: E402
from test_packed_attention_gpu import _bwd, _fwd, _inputs, _near, _normal  # noqa: E402
from test_paged_attention_gpu import _cache, _query, _step  # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32


def _hidden_form(q, k, v, lens, hidden):
    """o and lse of causal_ref.packed (each with its bound) where the tokens `hidden` [T] have scores of -infinity with
    every query: their weight is 0, and a row that sees no other has o 0 and lse -infinity."""
    H, Hk, D = q.shape[1], k.shape[1], q.shape[2]
    G, scale = H // Hk, D ** -0.5
    q, k, v = q.double(), torch.where(hidden[:, None, None], 0, k.double()), v.double()
    o, eo = torch.zeros_like(q), torch.zeros_like(q)
    lse, el = (torch.zeros(H, q.shape[0], dtype=torch.float64, device=q.device) for _ in range(2))
    a = 0
    for n in lens:
        b = a + n
        out = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1) | hidden[a:b]
        none = out.all(1, keepdim=True)
        for h in range(H):
            x, y, z = q[a:b, h], k[a:b, h // G], v[a:b, h // G]
            s = (scale * x @ y.T).masked_fill(out, -math.inf)
            ls = torch.logsumexp(s, 1, keepdim=True)
            some = torch.where(none, 0, ls)
            p = torch.exp(s - some)
            top = (scale * x.abs() @ y.abs().T).masked_fill(out, 0).amax(1, keepdim=True)
            ep = 2 * D * 2.0 ** -24 * top + 2.0 ** -22 * (s.masked_fill(out, 0).abs() + some.abs()) + 2.0 ** -19
            o[a:b, h], eo[a:b, h] = p @ z, (p * (2.0 ** -8 + ep)) @ z.abs() * 1.03 + 1e-30
            lse[h, a:b], el[h, a:b] = ls[:, 0], ep.amax(1) + 2.0 ** -22 * some[:, 0].abs()
        a = b
    return (o, eo), (lse, el)


def test_hidden_form_is_the_causal_one():
    """(On the CPU.) Where nothing is hidden; and hidden first tokens are as if they were not there."""
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(37, n, 8, generator=g).to(BF16) for n in (4, 2, 2))
    lens, some = [20, 17], torch.zeros(37, dtype=torch.bool)
    for x, y in zip(ref.packed(q, k, v, lens), _hidden_form(q, k, v, lens, some)):
        assert torch.allclose(x[0], y[0], rtol=1e-12, atol=1e-15) and torch.allclose(x[1], y[1], rtol=1e-12, atol=1e-15)
    some[:5] = True
    (o1, _), (ls1, _) = _hidden_form(q, k, v, lens, some)
    (o2, _), (ls2, _) = ref.packed(q[5:], k[5:], v[5:], [15, 17])
    assert torch.allclose(o1[5:], o2) and torch.allclose(ls1[:, 5:], ls2)
    assert (o1[:5] == 0).all() and (ls1[:, :5] == -torch.inf).all()


HIDDEN = [  # lens, H, Hk, D, hidden tokens
    ([300, 40, 200], 4, 2, 64, [*range(130), 200, 259, *range(300, 340), 340, 490]),
    ([300, 40, 200], 4, 2, 128, [*range(130), 200, 259, *range(300, 340), 340, 490]),
    ([700], 3, 1, 128, [*range(256), 300, 301, 511, 512]),   # groups of one: two tiles of a head
    ([129, 1, 1, 640], 3, 1, 64, [*range(128), 129, *range(131, 131 + 400)]),
    ([150] * 60, 8, 4, 64, [*range(0, 9000, 3), *range(150, 300)]),
]


def _hide(q, k, hidden, col=3):
    """-infinity in one column of the hidden keys, which every query meets with a value above zero."""
    q, k = q.clone(), k.clone()
    q[..., col] = q[..., col].abs() + 0.5
    k[hidden, :, col] = -torch.inf
    return q, k


@pytest.mark.gpu
@pytest.mark.parametrize("lens, H, Hk, D, hide", HIDDEN)
def test_packed_scores_of_minus_infinity_are_as_if_masked(lens, H, Hk, D, hide):
    """Whole tiles of such keys before others, single ones, and rows that see no others."""
    q, k, v, cu = _inputs(lens, H, Hk, D, 30)
    hidden = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
    hidden[hide] = True
    q, k = _hide(q, k, hidden)
    o, lse = _fwd(q, k, v, cu)
    (want, bound), (wl, bl) = _hidden_form(q, k, v, lens, hidden)
    _near(o, want, bound)
    none = wl == -torch.inf
    assert none.any() and torch.equal(lse == -torch.inf, none)
    assert (o.transpose(0, 1)[none] == 0).all()
    _near(torch.where(none, 0, lse), torch.where(none, 0, wl), bl, 2.0 ** -22)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_paged_scores_of_minus_infinity_are_as_if_masked(dtype):
    """A leading block, whole pieces of a sequence that several blocks share, single keys, all keys of a sequence."""
    lens, page, H, Hk, D = [700, 9000, 300, 64], 32, 4, 2, 64
    kc, vc, table = _cache(lens, page, Hk, D, dtype, 32)
    q = _query(4, H, D, dtype, 33).clone()
    q[..., 3] = q[..., 3].abs() + 0.5
    hide = [[*range(64), 100, 699], [*range(1000, 6000), 8999], [*range(0, 300, 2)], [*range(64)]]
    for b, keys in enumerate(hide):
        t = torch.tensor(keys, device="cuda")
        kc[table[b, t // page].long(), t % page, :, 3] = -torch.inf
    o, lse = _step(q, kc, vc, table, lens)
    for b, n in enumerate(lens):
        t = torch.arange(n, device="cuda")
        on = torch.ones(n, dtype=torch.bool, device="cuda")
        on[hide[b]] = False
        p = table[b, t // page].long()
        want, bound, wl = ref.paged(q[b], kc[p, t % page], vc[p, t % page], on, 2.0 ** -8 if dtype is BF16 else 0.0)
        _near(o[b], want, bound, 2.0 ** -8 if dtype is BF16 else 2.0 ** -24)
        if on.any():
            assert ((lse[b].double() - wl).abs() <= 2.0 ** -16 * (1 + wl.abs())).all()
        else:
            assert (o[b] == 0).all() and (lse[b] == -torch.inf).all()


def _check_all(q, k, v, cu, lens, seed):
    dO = _normal(torch.Generator(device="cuda").manual_seed(seed), *q.shape)
    o, lse = _fwd(q, k, v, cu)
    (want, bound), (wl, bl) = ref.packed(q, k, v, lens, 0)
    _near(o, want, bound)
    _near(lse, wl, bl, 2.0 ** -22)
    for x, (w, b) in zip(_bwd(q, k, v, cu, dO, o=o, lse=lse), ref.packed(q, k, v, lens, 0, dO, o)):
        _near(x, w, b)


@pytest.mark.gpu
@pytest.mark.parametrize("H, Hk, D", [(32, 4, 64), (32, 4, 128), (64, 16, 64), (64, 16, 128), (48, 24, 128), (36, 12, 128)])
def test_several_items_a_block_in_groups(H, Hk, D):
    """Items of two heads of a group (even groups) and of one, forward and gradients, more than the SMs: at
    4 heads of k in forward and dq only, at 12 to 24 in dk and dv too."""
    lens = [300, 0, 77, 640, 129, 512, 33, 255, 1, 128]
    q, k, v, cu = _inputs(lens, H, Hk, D, 34, fused=True)
    _check_all(q, k, v, cu, lens, 35)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_thousands_of_sequences(D):
    """More than the threads that lay out the list of work: each takes a run of them, some empty."""
    lens = [3, 0, 1, 7, 2] * 250 + [300, 0, 130] + [0] * 900 + [5, 1] * 40
    assert len(lens) > 2048
    q, k, v, cu = _inputs(lens, 2, 1, D, 36)
    _check_all(q, k, v, cu, lens, 37)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_a_workspace_used_again_at_once(D):
    """Calls of other lengths follow each other on one stream with the same workspaces: each sees its own list of
    work and its own statistics."""
    import pa_capi
    T, H, Hk = 2400, 8, 4
    sets = []
    for i, lens in enumerate(([2400], [100] * 24, [1, 2399], [700, 0, 1000, 700], [5] * 480, [0] * 20 + [1200, 1200])):
        q, k, v, cu = _inputs(lens, H, Hk, D, 38 + i)
        dO = _normal(torch.Generator(device="cuda").manual_seed(50 + i), *q.shape)
        cu = torch.nn.functional.pad(cu, (0, 481 - cu.numel()), value=T)  # empty sequences behind: one size of workspace
        o, lse = _fwd(q, k, v, cu)
        sets.append((q, k, v, cu, dO, o, lse, _bwd(q, k, v, cu, dO, o=o, lse=lse)))
    d = pa_capi.packed_attn_desc(*sets[0][:4])
    wf, wb = (torch.empty(f(d), dtype=torch.uint8, device="cuda") for f in
              (pa_capi.packed_attn_fwd_workspace_size, pa_capi.packed_attn_bwd_workspace_size))
    got = [[torch.empty_like(x) for x in (s[5], s[6], *s[7])] for s in sets * 4]
    torch.cuda.synchronize()
    for (q, k, v, cu, dO, o, lse, _), out in zip(sets * 4, got):
        pa_capi.packed_attn_fwd(q, k, v, cu, out[0], out[1], workspace=wf)
        pa_capi.packed_attn_bwd(q, k, v, o, dO, lse, cu, *out[2:], workspace=wb)
    for s, out in zip(sets * 4, got):
        for x, w in zip(out, (s[5], s[6], *s[7])):
            assert torch.equal(x, w)


@pytest.mark.gpu
def test_calls_on_a_stream_given_by_its_handle():
    """Each operator with the handle of another stream than the current one, and with the default stream's: what it
    reads was written there, and its result is that of the current stream."""
    import pa_capi as pa
    q, k, v, cu = _inputs([500, 31], 8, 2, 64, 60)
    T, g = q.shape[0], torch.Generator(device="cuda").manual_seed(61)
    dO = _normal(g, *q.shape)
    kc, vc, table = _cache([300, 900], 16, 2, 64, BF16, 62)
    q1, lens = _query(2, 8, 64, BF16, 63), torch.tensor([300, 900], dtype=torch.int32, device="cuda")
    x, y, z = (t.view(1, T, -1, 64) for t in (q, k, v))
    pos, gamma = torch.arange(T, device="cuda", dtype=torch.int32).view(1, 1, T), torch.rand(64, generator=g, device="cuda")
    slots = torch.randperm(600, generator=g, device="cuda")[:T].to(torch.int32).view(1, T)
    desc = pa.rope_desc(x, y)
    ins = {n: t.contiguous() for n, t in dict(q=q, k=k, v=v, dO=dO, kc=kc, vc=vc, q1=q1).items()}
    o, lse = _fwd(q, k, v, cu)

    def calls(i, **kw):
        x, y, z = (i[n].view(1, T, -1, 64) for n in "qkv")
        return {
            "packed": ((o, lse), lambda a, b: pa.packed_attn_fwd(i["q"], i["k"], i["v"], cu, a, b, **kw)),
            "packed gradient": ((q, k, v), lambda *a: pa.packed_attn_bwd(i["q"], i["k"], i["v"], o, i["dO"], lse, cu, *a,
                                                                        **kw)),
            "paged": ((q1, lse[:, :2].t().contiguous()), lambda a, b: pa.paged_attn_step(
                i["q1"], i["kc"], i["vc"], table, lens, a, b, **kw)),
            "norm": ((x, y), lambda a, b: pa.qk_norm_rope_fwd(x, y, gamma, gamma, pos, a, b, desc, **kw)),
            "norm to cache": ((x, kc, vc), lambda a, b, c: pa.qk_norm_rope_cache(x, y, z, gamma, gamma, pos, slots, a, b, c,
                                                                                desc, **kw)),
            "norm gradient": ((x, y, gamma, gamma), lambda *a: pa.qk_norm_rope_bwd(
                i["dO"].view(1, T, -1, 64), y, x, y, gamma, gamma, pos, *a, desc, **kw)),
        }

    side = torch.cuda.Stream()
    for name, (like, call) in calls(ins).items():
        want = [torch.zeros_like(t) for t in like]
        call(*want)
        for handle in (side, torch.cuda.default_stream()):
            late = {n: torch.zeros_like(t) for n, t in ins.items()}
            got = [torch.zeros_like(t) for t in like]
            other = torch.cuda.Stream()  # the current stream of the call, on which nothing is waited for
            torch.cuda.synchronize()
            with torch.cuda.stream(handle):
                torch.cuda._sleep(2_000_000)  # about a millisecond
                for n, t in ins.items():
                    late[n].copy_(t)
            with torch.cuda.stream(other):
                calls(late, stream=handle.cuda_stream)[name][1](*got)
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b), (name, handle)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, B, L", [(BF16, 8, 4096), (F32, 4, 4096)])
def test_norm_gradients_of_a_training_batch(dtype, B, L):
    """32768 tokens of 16 + 2 heads of 128. dgamma: a thread adds at most 16 tiles x 8 heads, a block 32 threads, a sum
    10 blocks and 32 parts: chains of 202 terms, 202 2^-24 < 2^-16 of the magnitudes, with 2^-18 of each term
    as for dx; together below the 2^-15 of the smaller cases."""
    import pa_capi
    H, Hk, D, eps = 16, 2, 128, 1e-6
    g = torch.Generator(device="cuda").manual_seed(70)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    q, k, _ = (p.unflatten(-1, (n, D)) for p, n in zip(
        normal(B, L, (H + 2 * Hk) * D).to(dtype).split([H * D, Hk * D, Hk * D], -1), (H, Hk, Hk)))
    gq, gk = 1 + 0.3 * normal(D), 1 + 0.3 * normal(D)
    dqo, dko = normal(B, L, H, D).to(dtype), normal(B, L, Hk, D).to(dtype)
    pos = torch.randint(0, 100000, (1, B, L), generator=g, device="cuda", dtype=torch.int32)
    dq, dk, dgq, dgk = (torch.empty(x.shape, dtype=x.dtype, device="cuda") for x in (q, k, gq, gk))
    pa_capi.qk_norm_rope_bwd(dqo, dko, q, k, gq, gk, pos, dq, dk, dgq, dgk, pa_capi.rope_desc(q, k), eps)
    step = {BF16: 2.0 ** -8, F32: 2.0 ** -24}[dtype]
    for x, gamma, dy, dx, dg in ((q, gq, dqo, dq, dgq), (k, gk, dko, dk, dgk)):
        wg, mg = torch.zeros(D, dtype=torch.float64, device="cuda"), torch.zeros(D, dtype=torch.float64, device="cuda")
        for b in range(B):
            xb, db, gd = x[b:b + 1].double(), dy[b:b + 1].double(), gamma.double()
            dn = turn(db, pos[:, b:b + 1], [D // 2], inverse=True)
            m = db.abs()
            mag = (m[..., :D // 2] + m[..., D // 2:]).repeat(1, 1, 1, 2)
            r = (xb.square().mean(-1, keepdim=True) + eps).rsqrt()
            u, mu = dn * gd, mag * gd.abs()
            want = r * (u - xb * r ** 2 * (u * xb).mean(-1, keepdim=True))
            bound = r * (mu + xb.abs() * r ** 2 * (mu * xb.abs()).mean(-1, keepdim=True))
            _near(dx[b:b + 1], want, 2.0 ** -18 * bound, step)
            wg += (dn * xb * r).sum((0, 1, 2))
            mg += (mag * xb.abs() * r).sum((0, 1, 2))
        _near(dg, wg, 2.0 ** -15 * mg, 2.0 ** -22)


@pytest.mark.gpu
@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("lens, H, Hk, D", [([12000, 1, 4000], 16, 4, 64), ([12000, 1, 4000], 16, 16, 64),
                                            ([9000, 77, 300], 16, 4, 128), ([9000, 77, 300], 9, 9, 128)])
def test_calls_that_a_recorded_error_interrupts(lens, H, Hk, D, backward):
    """An error that another kernel records in the middle of a row of calls: the one that runs then ends within a
    few milliseconds (a wait for a copy that was never sent takes 20), those behind it leave their outputs, and once
    the error is cleared the same calls give the same bits: no copy or product of an ended block is still on its way."""
    import pa_capi
    q, k, v, cu = _inputs(lens, H, Hk, D, 80)
    dO = _normal(torch.Generator(device="cuda").manual_seed(81), *q.shape)
    o, lse = _fwd(q, k, v, cu)
    want = _bwd(q, k, v, cu, dO, o=o, lse=lse) if backward else (o, lse)
    outs = [[torch.full_like(x, 7.0) for x in want] for _ in range(16)]
    assert pa_capi.device_status() == 0

    def call(out):
        if backward:
            pa_capi.packed_attn_bwd(q, k, v, o, dO, lse, cu, *out)
        else:
            pa_capi.packed_attn_fwd(q, k, v, cu, *out)

    call(outs[-1])  # (memory and launches are ready)
    outs[-1] = [torch.full_like(x, 7.0) for x in want]
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    side, limit = torch.cuda.Stream(), 2_000_000
    torch.cuda.synchronize()
    pa_capi.wait_selftest(limit, arrive=False, stream=side.cuda_stream)
    try:
        a.record()
        for out in outs:
            call(out)
        b.record()
        torch.cuda.synchronize()
        assert pa_capi.device_status(clear=False) == 6  # PA_ERR_TIMEOUT
        assert a.elapsed_time(b) < limit * 1e-6 + 12, a.elapsed_time(b)
        assert all(torch.equal(x, y) for x, y in zip(outs[0], want))  # before it
        assert all((x == 7).all() for x in outs[-1])                  # behind it
    finally:
        pa_capi.device_status(clear=True)
    for out in outs[:4]:
        call(out)
    for out in outs[:4]:
        assert all(torch.equal(x, y) for x, y in zip(out, want))
    assert pa_capi.device_status() == 0

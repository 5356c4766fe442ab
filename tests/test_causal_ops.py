"""Argument checks of packed causal attention, paged attention and head norms: the C ABI's
status codes before any device work, and the Python binding's refusals (no GPU)."""
import ctypes

import pytest

NULL, SHAPE, DTYPE, ALIGN, UNSUPPORTED, WORKSPACE = 8, 1, 2, 3, 4, 7
BIG = 1 << 44
# pointers far apart
P = [i << 45 for i in range(1, 16)]


def _packed(**kw):
    import pa_capi
    f = dict(tokens=100, num_seqs=3, num_heads=4, num_kv_heads=2, head_dim=64, dtype=pa_capi.PA_BF16)
    f.update(kw)
    return ctypes.byref(pa_capi.PackedAttnDesc(**f))


def _packed_calls(desc, a=P, ws=P[12], nb=BIG):
    import pa_capi
    lib = pa_capi.load()
    return (lib.pa_packed_attn_fwd(desc, *a[:6], ws, nb, None),
            lib.pa_packed_attn_bwd(desc, *a[:10], 0, ws, nb, None))


@pytest.mark.parametrize("kw,status", [
    (dict(tokens=0), SHAPE), (dict(num_seqs=0), SHAPE), (dict(num_heads=0), SHAPE), (dict(num_kv_heads=0), SHAPE),
    (dict(num_kv_heads=3), SHAPE), (dict(head_dim=0), SHAPE), (dict(head_dim=96), UNSUPPORTED),
    (dict(head_dim=32), UNSUPPORTED), (dict(dtype=0), DTYPE), (dict(dtype=7), DTYPE), (dict(tokens=2 ** 31 - 1), SHAPE),
    (dict(tokens=2 ** 31 - 1000, num_heads=1 << 10, num_kv_heads=1), SHAPE), (dict(num_seqs=2 ** 31 - 1), SHAPE),
    (dict(softmax_scale=float("nan")), SHAPE), (dict(softmax_scale=float("inf")), SHAPE),
    (dict(softmax_scale=1e-30), SHAPE), (dict(q_stride=255), SHAPE), (dict(q_stride=260), ALIGN),
    (dict(k_stride=-128), SHAPE), (dict(v_stride=64), SHAPE), (dict(v_stride=129), ALIGN),
    (dict(dq_stride=8), SHAPE), (dict(dk_stride=132), ALIGN), (dict(dv_stride=-8), SHAPE),
])
def test_packed_descriptor_refusals(kw, status):
    import pa_capi
    lib = pa_capi.load()
    assert _packed_calls(_packed(**kw)) == (status, status)
    assert lib.pa_packed_attn_fwd_workspace_size(_packed(**kw)) == 0
    assert lib.pa_packed_attn_bwd_workspace_size(_packed(**kw)) == 0


def test_packed_pointer_refusals():
    import pa_capi
    lib = pa_capi.load()
    assert _packed_calls(None) == (NULL, NULL)
    for i in range(10):
        a = list(P)
        a[i] = None
        assert _packed_calls(_packed(), a)[1] == NULL
        assert i >= 6 or _packed_calls(_packed(), a)[0] == NULL
        a[i] = P[i] + 2
        assert _packed_calls(_packed(), a)[1] == ALIGN
        assert i >= 6 or _packed_calls(_packed(), a)[0] == ALIGN
    for size, call in ((lib.pa_packed_attn_fwd_workspace_size, 0), (lib.pa_packed_attn_bwd_workspace_size, 1)):
        need = size(_packed())
        assert need > 0
        assert _packed_calls(_packed(), nb=need - 1)[call] == WORKSPACE
        assert _packed_calls(_packed(), ws=None)[call] == WORKSPACE
        assert _packed_calls(_packed(), ws=P[12] + 16)[call] == ALIGN


def test_packed_overlaps_are_refused():
    """fwd: q, k, v, cu, o, lse; bwd: q, k, v, o, dO, lse, cu, dq, dk, dv."""
    row = 4 * 64 * 2
    for out, others, call in ((4, (0, 1, 2, 3, 5), 0), (5, (0, 1, 2, 3), 0), (7, (0, 1, 2, 3, 4, 5, 6, 8, 9), 1),
                              (8, (0, 6, 9), 1), (9, (1, 3), 1)):
        for i in others:
            a = list(P)
            a[out] = a[i]
            assert _packed_calls(_packed(), a)[call] == SHAPE
            if call == 0 and out == 4 and i in (0, 1, 2):
                a[out] = a[i] + 99 * (row if i == 0 else row // 2)  # the last token's row
                assert _packed_calls(_packed(), a)[call] == SHAPE
    # the workspace over an input; gradients over slices of the same tensor as the inputs
    assert _packed_calls(_packed(), ws=P[0]) == (SHAPE, SHAPE)
    a = list(P)
    a[7] = a[0] + row // 2
    assert _packed_calls(_packed(q_stride=512, dq_stride=512), a)[1] == SHAPE


def _paged(**kw):
    import pa_capi
    f = dict(batch=3, num_heads=4, num_kv_heads=2, head_dim=64, dtype=pa_capi.PA_BF16, page_size=16, num_pages=9,
             max_pages=4)
    f.update(kw)
    return ctypes.byref(pa_capi.PagedAttnDesc(**f))


def _paged_call(desc, a=P, ws=P[12], nb=BIG):
    import pa_capi
    return pa_capi.load().pa_paged_attn_step(desc, *a[:7], ws, nb, None)


@pytest.mark.parametrize("kw,status", [
    (dict(batch=0), SHAPE), (dict(num_heads=0), SHAPE), (dict(num_kv_heads=0), SHAPE), (dict(num_kv_heads=3), SHAPE),
    (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=32), UNSUPPORTED), (dict(dtype=0, head_dim=128), UNSUPPORTED),
    (dict(dtype=3), DTYPE), (dict(page_size=0), SHAPE), (dict(num_pages=0), SHAPE), (dict(max_pages=-1), SHAPE),
    (dict(page_size=1 << 16, max_pages=1 << 16), SHAPE), (dict(page_size=1 << 16, num_pages=1 << 16), SHAPE),
    (dict(batch=1 << 28, num_heads=1, num_kv_heads=1), SHAPE), (dict(q_stride=128), SHAPE), (dict(q_stride=260), ALIGN),
    (dict(softmax_scale=float("nan")), SHAPE),
])
def test_paged_descriptor_refusals(kw, status):
    import pa_capi
    assert _paged_call(_paged(**kw)) == status
    assert pa_capi.load().pa_paged_attn_step_workspace_size(_paged(**kw)) == 0


def test_paged_pointer_refusals():
    """q, k_cache, v_cache, page_table, seq_lens, o, lse."""
    import pa_capi
    assert _paged_call(None) == NULL
    for i in range(7):
        a = list(P)
        if i < 6:  # lse may be NULL
            a[i] = None
            assert _paged_call(_paged(), a) == NULL
        a[i] = P[i] + 2
        assert _paged_call(_paged(), a) == ALIGN
        if i < 5:
            a[i] = P[i]
            for out in (5, 6):
                a[out] = P[i]
                assert _paged_call(_paged(), a) == SHAPE
                a[out] = P[out]
    need = pa_capi.load().pa_paged_attn_step_workspace_size(_paged())
    assert need > 0
    assert _paged_call(_paged(), nb=need - 1) == WORKSPACE
    assert _paged_call(_paged(), ws=None) == WORKSPACE
    assert _paged_call(_paged(), ws=P[12] + 128) == ALIGN
    assert _paged_call(_paged(), ws=P[1]) == SHAPE


def _norm(eps=1e-6, q_stride=0, k_stride=0, v_stride=0, dq_stride=0, dk_stride=0, **kw):
    import pa_capi
    f = dict(batch=1, seq_len=8, num_heads=2, num_kv_heads=1, head_dim=64, dtype=pa_capi.PA_BF16, layout=0,
             freqs=0, axes=2, sections=(ctypes.c_int32 * 4)(8, 8, 0, 0), base=10000.0)
    f.update(kw)
    if isinstance(f["sections"], tuple):
        f["sections"] = (ctypes.c_int32 * 4)(*f["sections"])
    return ctypes.byref(pa_capi.QkNormDesc(pa_capi.RopeDesc(**f), eps, q_stride, k_stride, v_stride, dq_stride,
                                           dk_stride))


def _norm_calls(desc, fwd=P, cache=P, bwd=P, slots=100, ws=P[12], nb=BIG):
    """fwd: q, k, gq, gk, positions, q_out, k_out; cache: q, k, v, gq, gk, positions, slots, q_out, k_out,
    k_cache, v_cache; bwd: dq_out, dk_out, q, k, gq, gk, positions, dq, dk, dgq, dgk."""
    import pa_capi
    lib = pa_capi.load()
    return (lib.pa_qk_norm_rope_fwd(desc, *fwd[:7], None),
            lib.pa_qk_norm_rope_cache(desc, *cache[:11], slots, None),
            lib.pa_qk_norm_rope_bwd(desc, *bwd[:11], 0, ws, nb, None))


@pytest.mark.parametrize("kw,status", [
    (dict(batch=0), SHAPE), (dict(num_heads=0), SHAPE), (dict(num_kv_heads=-1), SHAPE), (dict(head_dim=264), UNSUPPORTED),
    (dict(head_dim=44), UNSUPPORTED), (dict(head_dim=50, dtype=0), UNSUPPORTED), (dict(dtype=5), DTYPE),
    (dict(axes=0), SHAPE), (dict(sections=(30, 3, 0, 0)), SHAPE), (dict(base=1.0), SHAPE), (dict(eps=-1.0), SHAPE),
    (dict(eps=float("nan")), SHAPE), (dict(eps=float("inf")), SHAPE), (dict(q_stride=64), SHAPE),
    (dict(q_stride=132), ALIGN), (dict(k_stride=-64), SHAPE), (dict(v_stride=68), ALIGN), (dict(dq_stride=32), SHAPE),
    (dict(dk_stride=66), ALIGN), (dict(dtype=0, k_stride=66), ALIGN),
])
def test_norm_descriptor_refusals(kw, status):
    import pa_capi
    assert _norm_calls(_norm(**kw)) == (status,) * 3
    assert pa_capi.load().pa_qk_norm_rope_bwd_workspace_size(_norm(**kw)) == 0


def test_norm_pointer_refusals():
    import pa_capi
    assert _norm_calls(None) == (NULL,) * 3
    optional = ((2, 3), (3, 4, 8), (4, 5, 9, 10))
    for call, n in enumerate((7, 11, 11)):
        for i in range(n):
            a = [list(P) for _ in range(3)]
            if i not in optional[call]:
                a[call][i] = None
                assert _norm_calls(_norm(), *a)[call] == NULL, (call, i)
            a[call][i] = P[i] + 2
            assert _norm_calls(_norm(), *a)[call] == ALIGN, (call, i)
    # the gradient of a weight that is not there
    for g, dg in ((4, 9), (5, 10)):
        a = list(P)
        a[g] = None
        assert _norm_calls(_norm(), bwd=a)[2] == NULL
    # a cache without keys, or without places
    assert _norm_calls(_norm(num_kv_heads=0))[1] == SHAPE
    assert _norm_calls(_norm(), slots=0)[1] == SHAPE
    assert _norm_calls(_norm(), slots=2 ** 31)[1] == SHAPE
    need = pa_capi.load().pa_qk_norm_rope_bwd_workspace_size(_norm())
    assert need > 0
    assert _norm_calls(_norm(), nb=need - 1)[2] == WORKSPACE
    assert _norm_calls(_norm(), ws=None)[2] == WORKSPACE
    assert _norm_calls(_norm(), ws=P[12] + 64)[2] == ALIGN


def test_norm_overlaps_are_refused():
    def one(call, out, i, shift=0, **kw):
        a = [list(P) for _ in range(3)]
        a[call][out] = a[call][i] + shift
        return _norm_calls(_norm(**kw), *a)[call]
    for call, outs, ins in ((0, (5, 6), range(5)), (1, (7, 8, 9, 10), range(7)), (2, (7, 8, 9, 10), range(7))):
        for o in outs:
            for i in ins:
                # in place: q_out over q, k_out over k, dq over dq_out, dk over dk_out
                if (call, o, i) in ((0, 5, 0), (0, 6, 1), (1, 7, 0), (1, 8, 1), (2, 7, 0), (2, 8, 1)):
                    continue
                assert one(call, o, i) == SHAPE, (call, o, i)
    # in place, but not over the whole of itself, or over tokens that lie apart
    assert one(0, 5, 0, 16) == SHAPE and one(0, 6, 1, 16) == SHAPE
    assert one(0, 5, 0, q_stride=256) == SHAPE and one(0, 6, 1, k_stride=128) == SHAPE
    assert one(2, 7, 0, dq_stride=256) == SHAPE
    import pa_capi
    a = list(P)
    a[7] = a[0]  # adding in place would read what it has written
    assert pa_capi.load().pa_qk_norm_rope_bwd(_norm(), *a[:11], 1, P[12], BIG, None) == SHAPE


def test_binding_refuses_tensors_that_do_not_fit():
    torch = pytest.importorskip("torch")
    import pa_capi
    b = torch.bfloat16
    q, k, v = torch.zeros(10, 4, 64, dtype=b), torch.zeros(10, 2, 64, dtype=b), torch.zeros(10, 2, 64, dtype=b)
    cu, o, lse = torch.zeros(3, dtype=torch.int32), torch.zeros(10, 4, 64, dtype=b), torch.zeros(4, 10)

    def fwd(**kw):
        a = dict(q=q, k=k, v=v, cu_seqlens=cu, o=o, lse=lse)
        a.update(kw)
        pa_capi.packed_attn_fwd(**a)

    bad = [dict(k=k[:9]), dict(v=torch.zeros(10, 3, 64, dtype=b)), dict(k=k.float()), dict(o=o[:, :2]),
           dict(lse=lse.t().contiguous()), dict(cu_seqlens=cu.long()), dict(cu_seqlens=cu[None]),
           dict(q=torch.zeros(10, 64, 4, dtype=b).transpose(1, 2)), dict(k=torch.zeros(1, 2, 64, dtype=b).expand(10, 2, 64)),
           dict(q=torch.zeros(20, 8, 64, dtype=b)[:10, ::2]), {}]  # the last: not on a CUDA device
    for kw in bad:
        with pytest.raises(ValueError):
            fwd(**kw)
    kc, table, lens = torch.zeros(5, 16, 2, 64, dtype=b), torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    q3 = q[:3]

    def step(**kw):
        a = dict(q=q3, k_cache=kc, v_cache=kc.clone(), page_table=table, seq_lens=lens, o=torch.zeros_like(q3))
        a.update(kw)
        pa_capi.paged_attn_step(**a)

    for kw in (dict(v_cache=kc[:4]), dict(k_cache=kc.float()), dict(page_table=table[:2]), dict(page_table=table.long()),
               dict(seq_lens=lens[:2]), dict(o=q), dict(lse=torch.zeros(3, 3)), dict(q=q3.float()),
               dict(page_table=table.t()), dict(k_cache=torch.zeros(5, 16, 2, 32, dtype=b),
                                                v_cache=torch.zeros(5, 16, 2, 32, dtype=b)), {}):
        with pytest.raises(ValueError):
            step(**kw)
    x, y = torch.zeros(2, 5, 4, 64, dtype=b), torch.zeros(2, 5, 2, 64, dtype=b)
    d, g, pos = pa_capi.rope_desc(x, y), torch.zeros(64), torch.zeros(1, 2, 5, dtype=torch.int32)

    def norm(**kw):
        a = dict(q=x, k=y, gamma_q=g, gamma_k=g, positions=pos, q_out=x.clone(), k_out=y.clone(), desc=d)
        a.update(kw)
        pa_capi.qk_norm_rope_fwd(**a)

    for kw in (dict(k=None), dict(gamma_q=g.to(b)), dict(gamma_k=g[:32]), dict(positions=pos[0]), dict(q_out=x[:, :4]),
               dict(q=x.transpose(1, 2)), dict(k_out=y.float()),
               dict(q=torch.zeros(2, 6, 4, 64, dtype=b)[:, :5]), {}):
        with pytest.raises(ValueError):
            norm(**kw)


def test_binding_takes_slices_as_strides():
    torch = pytest.importorskip("torch")
    import pa_capi
    x = torch.zeros(10, 512, dtype=torch.bfloat16)
    q, k, v = (p.unflatten(1, (-1, 64)) for p in x.split([256, 128, 128], 1))
    d = pa_capi.packed_attn_desc(q, k, v, torch.zeros(3, dtype=torch.int32))
    assert (d.tokens, d.num_seqs, d.num_heads, d.num_kv_heads, d.head_dim) == (10, 2, 4, 2, 64)
    assert (d.q_stride, d.k_stride, d.v_stride, d.dq_stride) == (512, 512, 512, 0)
    y = torch.zeros(2, 5, 512, dtype=torch.bfloat16)[..., :256].unflatten(-1, (4, 64))
    assert pa_capi._token_stride("f", "q", y, 4, 64, -1, torch.bfloat16, 10) == 512
    assert pa_capi._token_stride("f", "q", y[:, :1], 4, 64, -1, torch.bfloat16, 2) == 512 * 5
    assert pa_capi._token_stride("f", "q", y[:1, :1], 4, 64, -1, torch.bfloat16, 1) == 256

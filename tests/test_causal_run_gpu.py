"""The operators of a causal model together: prompts are normed, turned and written into a paged
cache, attend within themselves, and then go on token by token from the cache."""
import pytest

torch = pytest.importorskip("torch")
import causal_ref as ref  # noqa: E402
from seq_ref import turn  # noqa: E402

BF16 = torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,D,page", [(4, 2, 64, 16), (6, 2, 128, 24), (8, 8, 64, 64)])
def test_prompts_and_generation(H, Hk, D, page):
    """Each token of each step, prompt or generated, against the 64-bit attention of the keys and values
    that the model made so far; a generated token sees what it would as the last of a longer prompt."""
    import pa_capi as pa
    lens, steps, eps = [130, 1, 0, 77], 20, 1e-6
    n, T = len(lens), sum(lens)
    g = torch.Generator(device="cuda").manual_seed(0)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    gq, gk = 1 + 0.2 * normal(D), 1 + 0.2 * normal(D)
    per = -(-(max(lens) + steps) // page)
    table = torch.randperm(n * per, generator=g, device="cuda").to(torch.int32).view(n, per)
    kc, vc = (torch.full((n * per, page, Hk, D), float("nan"), dtype=BF16, device="cuda") for _ in range(2))

    def qkv(B, L):
        parts = normal(B, L, (H + 2 * Hk) * D).to(BF16).split([H * D, Hk * D, Hk * D], -1)
        return [p.unflatten(-1, (m, D)) for p, m in zip(parts, (H, Hk, Hk))]

    def slots_of(seq, at):
        return (table[seq, at // page] * page + at % page).to(torch.int32)

    # the prompts, packed
    cu = torch.cumsum(torch.tensor([0] + lens), 0).to(torch.int32).cuda()
    seq = torch.repeat_interleave(torch.arange(n), torch.tensor(lens)).cuda()
    at = torch.cat([torch.arange(m) for m in lens]).cuda()
    q, k, v = qkv(1, T)
    pos = at.to(torch.int32).view(1, 1, T)
    qo, ko = torch.empty(1, T, H, D, dtype=BF16, device="cuda"), torch.empty(1, T, Hk, D, dtype=BF16, device="cuda")
    pa.qk_norm_rope_cache(q, k, v, gq, gk, pos, slots_of(seq, at).view(1, T), qo, kc, vc, pa.rope_desc(qo, ko), eps,
                          k_out=ko)
    o, lse = torch.empty(T, H, D, dtype=BF16, device="cuda"), torch.empty(H, T, device="cuda")
    pa.packed_attn_fwd(qo[0], ko[0], v[0], cu, o, lse)
    (want, bound), _ = ref.packed(qo[0], ko[0], v[0], lens)
    assert ((o.double() - want).abs() <= bound + 2.0 ** -8 * want.abs()).all()
    n64 = turn(ref.rms(q, gq, eps), pos, [D // 2])
    assert torch.allclose(qo.double(), n64, rtol=2.0 ** -7, atol=1e-4)

    # token by token
    keys = [[ko[0, cu[b]:cu[b + 1]], v[0, cu[b]:cu[b + 1]]] for b in range(n)]
    now = torch.tensor(lens, device="cuda")
    every = torch.arange(n, device="cuda")
    for _ in range(steps):
        q, k, v = qkv(n, 1)
        pos = now.to(torch.int32).view(1, n, 1)
        qo, ko = torch.empty(n, 1, H, D, dtype=BF16, device="cuda"), torch.empty(n, 1, Hk, D, dtype=BF16, device="cuda")
        pa.qk_norm_rope_cache(q, k, v, gq, gk, pos, slots_of(every, now).view(n, 1), qo, kc, vc, pa.rope_desc(qo, ko),
                              eps, k_out=ko)
        now = now + 1
        o = torch.empty(n, H, D, dtype=BF16, device="cuda")
        pa.paged_attn_step(qo[:, 0], kc, vc, table, now.to(torch.int32), o)
        for b in range(n):
            keys[b] = [torch.cat(p) for p in zip(keys[b], (ko[b], v[b]))]
            on = torch.ones(keys[b][0].shape[0], dtype=torch.bool, device="cuda")
            want, bound, _ = ref.paged(qo[b, 0], *keys[b], on, 2.0 ** -8)
            assert ((o[b].double() - want).abs() <= bound + 2.0 ** -8 * want.abs()).all()
    # the last token of a longer prompt
    lens = [m + steps for m in lens]
    last = torch.cumsum(torch.tensor(lens), 0).cuda() - 1
    cu = torch.cumsum(torch.tensor([0] + lens), 0).to(torch.int32).cuda()
    ks, vs = (torch.cat([kv[i] for kv in keys]) for i in range(2))
    qs = torch.zeros(sum(lens), H, D, dtype=BF16, device="cuda")
    qs[last] = qo[:, 0]
    whole, lse = torch.empty_like(qs), torch.empty(H, qs.shape[0], device="cuda")
    pa.packed_attn_fwd(qs, ks, vs, cu, whole, lse)
    (want, bound), _ = ref.packed(qs, ks, vs, lens)
    for x in (whole[last], o):
        assert ((x.double() - want[last]).abs() <= 2 * bound[last] + 2.0 ** -8 * want[last].abs()).all()

"""Causal attention and head norms where they can go wrong beyond their own files' cases: scores of
-infinity."""
import math

import pytest

torch = pytest.importorskip("torch")
import causal_ref as ref  # noqa: E402
from test_packed_attention_gpu import _fwd, _inputs, _near  # noqa: E402
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

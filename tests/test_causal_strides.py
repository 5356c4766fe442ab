"""Layouts that a 32-bit descriptor cannot hold are refused by the Python binding (no GPU, no memory:
the tensors are on the meta device)."""
import pytest

torch = pytest.importorskip("torch")

FAR = (2 ** 31, 2 ** 32, 2 ** 32 + 256, 2 ** 33 + 512, 2 ** 40)


def _apart(step, *shape):
    """bf16 [tokens, heads, D] with `step` values from token to token."""
    return torch.empty_strided(shape, (step, shape[2], 1), dtype=torch.bfloat16, device="meta")


@pytest.mark.parametrize("step", FAR)
def test_tokens_too_far_apart_are_refused(step):
    import pa_capi
    cu = torch.zeros(3, dtype=torch.int32)
    near = {"q": _apart(256, 2, 4, 64), "k": _apart(128, 2, 2, 64), "v": _apart(128, 2, 2, 64)}
    for name, x in near.items():
        far = dict(near, **{name: _apart(step, *x.shape)})
        with pytest.raises(ValueError, match=name):
            pa_capi.packed_attn_desc(**far, cu_seqlens=cu)
        with pytest.raises(ValueError, match="d" + name):
            pa_capi.packed_attn_desc(**near, cu_seqlens=cu, **{"d" + name: _apart(step, *x.shape)})
    cache, table = torch.empty(5, 16, 2, 64, dtype=torch.bfloat16, device="meta"), torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="q"):
        pa_capi.paged_attn_desc(_apart(step, 2, 4, 64), cache, table)
    x = torch.empty_strided((1, 2, 4, 64), (2 * step, step, 64, 1), dtype=torch.bfloat16, device="meta")
    with pytest.raises(ValueError, match="q"):
        pa_capi._token_stride("qk_norm_rope_fwd", "q", x, 4, 64, -1, torch.bfloat16, 2)


def test_the_widest_tokens_are_taken():
    import pa_capi
    step = 2 ** 31 - 8
    d = pa_capi.packed_attn_desc(_apart(step, 2, 4, 64), _apart(128, 2, 2, 64), _apart(128, 2, 2, 64),
                                 torch.zeros(3, dtype=torch.int32))
    assert (d.q_stride, d.k_stride) == (step, 128)


def test_counts_past_32_bits_are_refused():
    """More sequences, or pages of a sequence, than an int32 counts."""
    import pa_capi
    q, k = _apart(256, 2, 4, 64), _apart(128, 2, 2, 64)
    many = torch.empty(2 ** 32 + 3, dtype=torch.int32, device="meta")
    with pytest.raises(ValueError, match="cu_seqlens"):
        pa_capi.packed_attn_desc(q, k, k, many)
    cache = torch.empty(5, 16, 2, 64, dtype=torch.bfloat16, device="meta")
    with pytest.raises(ValueError, match="page_table"):
        pa_capi.paged_attn_desc(q, cache, torch.empty(2, 2 ** 32 + 4, dtype=torch.int32, device="meta"))

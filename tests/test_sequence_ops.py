"""Argument checks of the rotary positions and of linear attention: the C ABI's
status codes before any device work, and the Python binding's refusals (no GPU)."""
import ctypes

import pytest

NULL, SHAPE, DTYPE, ALIGN, UNSUPPORTED, WORKSPACE = 8, 1, 2, 3, 4, 7


def _rope(**kw):
    import pa_capi
    f = dict(batch=1, seq_len=8, num_heads=2, num_kv_heads=1, head_dim=64, dtype=pa_capi.PA_BF16, layout=0,
             freqs=0, axes=2, sections=(ctypes.c_int32 * 4)(8, 8, 0, 0), base=10000.0)
    f.update(kw)
    if isinstance(f["sections"], tuple):
        f["sections"] = (ctypes.c_int32 * 4)(*f["sections"])
    return ctypes.byref(pa_capi.RopeDesc(**f))


@pytest.mark.parametrize("kw,status", [
    (dict(batch=0), SHAPE), (dict(seq_len=0), SHAPE), (dict(num_heads=0), SHAPE), (dict(num_kv_heads=-1), SHAPE),
    (dict(head_dim=0), SHAPE), (dict(head_dim=258), UNSUPPORTED), (dict(dtype=5), DTYPE), (dict(layout=2), UNSUPPORTED),
    (dict(freqs=-1), UNSUPPORTED), (dict(axes=0), SHAPE), (dict(axes=5), SHAPE), (dict(sections=(8, 0, 0, 0)), SHAPE),
    (dict(sections=(30, 3, 0, 0)), SHAPE), (dict(sections=(2 ** 31 - 1, 2 ** 31 - 1, 0, 0)), SHAPE),
    (dict(base=1.0), SHAPE), (dict(base=float("nan")), SHAPE), (dict(base=float("inf")), SHAPE),
    (dict(batch=1 << 16, seq_len=1 << 16), SHAPE), (dict(num_heads=1 << 25), SHAPE),
])
def test_rope_descriptor_refusals(kw, status):
    import pa_capi
    lib = pa_capi.load()
    assert lib.pa_rope_fwd(_rope(**kw), 16, 32, 64, 128, 256, None) == status
    assert lib.pa_rope_bwd(_rope(**kw), 16, 32, 64, 128, 256, 0, None) == status


def test_rope_pointer_refusals():
    import pa_capi
    lib = pa_capi.load()
    assert lib.pa_rope_fwd(None, 16, 32, 64, 128, 256, None) == NULL
    for i in range(5):
        a = [16, 32, 64, 128, 256]
        a[i] = None
        assert lib.pa_rope_fwd(_rope(), *a, None) == NULL
        a[i] = 18  # misaligned for values, and for positions
        assert lib.pa_rope_fwd(_rope(), *a, None) == ALIGN
    # adding in place would read what it has written
    assert lib.pa_rope_bwd(_rope(), 16, 32, 64, 16, 256, 1, None) == SHAPE
    assert lib.pa_rope_bwd(_rope(), 16, 32, 64, 128, 32, 1, None) == SHAPE


def _desc(B=2, L=128, H=2, D=64, dtype=1, scale=0.0):
    import pa_capi
    return ctypes.byref(pa_capi.AttnDesc(B, L, H, D, dtype, scale))


@pytest.mark.parametrize("kw,status", [
    (dict(B=0), SHAPE), (dict(L=0), SHAPE), (dict(L=-3), SHAPE), (dict(H=0), SHAPE), (dict(D=96), UNSUPPORTED),
    (dict(D=32), UNSUPPORTED), (dict(dtype=0, D=128), UNSUPPORTED), (dict(dtype=9), DTYPE),
    (dict(B=1 << 16, H=1 << 10), SHAPE),
])
def test_linear_attention_descriptor_refusals(kw, status):
    import pa_capi
    lib = pa_capi.load()
    big = 1 << 40
    assert lib.pa_linear_attn_fwd(_desc(**kw), 16, 32, 48, 64, None, None, 80, None, 256, big, None) == status
    assert lib.pa_linear_attn_bwd(_desc(**kw), 16, 32, 48, 64, 80, None, None, None, 96, 112, 128, None, 0, 256,
                                  big, None) == status
    assert lib.pa_linear_attn_step(_desc(**dict(kw, L=kw.get("L", 1))), 16, 32, 48, 64, 80, 96, 112, None) == status
    assert lib.pa_linear_attn_fwd_workspace_size(_desc(**kw)) == 0
    assert lib.pa_linear_attn_bwd_workspace_size(_desc(**kw)) == 0


def test_linear_attention_pointer_refusals():
    import pa_capi
    lib = pa_capi.load()
    big = 1 << 40
    fwd = lambda q=16, k=32, v=48, ld=64, n=None, s=None, o=80, so=None, ws=256, nb=big: lib.pa_linear_attn_fwd(
        _desc(), q, k, v, ld, n, s, o, so, ws, nb, None)
    assert lib.pa_linear_attn_fwd(None, 16, 32, 48, 64, None, None, 80, None, 256, big, None) == NULL
    for name in ("q", "k", "v", "ld", "o"):
        assert fwd(**{name: None}) == NULL
    for name in ("q", "k", "v", "o", "s", "so"):
        assert fwd(**{name: 8}) == ALIGN
    assert fwd(ld=66) == ALIGN and fwd(n=66) == ALIGN
    for name in ("q", "k", "v"):
        assert fwd(**{name: 80}) == SHAPE  # an input as the output
    bwd = lambda q=16, k=32, v=48, dO=64, ld=80, n=None, s=None, ds=None, dq=96, dk=112, dv=128, dsi=None, ws=256, \
        nb=big: lib.pa_linear_attn_bwd(_desc(), q, k, v, dO, ld, n, s, ds, dq, dk, dv, dsi, 0, ws, nb, None)
    for name in ("q", "k", "v", "dO", "ld", "dq", "dk", "dv"):
        assert bwd(**{name: None}) == NULL
    for name in ("q", "k", "v", "dO", "dq", "dk", "dv", "s", "ds", "dsi"):
        assert bwd(**{name: 8}) == ALIGN
    assert bwd(dq=16) == SHAPE and bwd(dk=64) == SHAPE and bwd(dv=96) == SHAPE
    assert bwd(s=160, dsi=160) == SHAPE and bwd(ds=160, dsi=160) == SHAPE
    step = lambda L=1, q=16, k=32, v=48, ld=64, s=80, o=96, so=112: lib.pa_linear_attn_step(
        _desc(L=L), q, k, v, ld, s, o, so, None)
    assert step(L=2) == SHAPE and step(o=16) == SHAPE
    for name in ("q", "k", "v", "ld", "s", "o", "so"):
        assert step(**{name: None}) == NULL
        if name != "ld":
            assert step(**{name: 8}) == ALIGN


def test_binding_refusals():
    """Types, shapes, layouts and devices that the kernels would misread are refused by name."""
    torch = pytest.importorskip("torch")
    import pa_capi
    q = torch.zeros(2, 8, 4, 64)
    ld = torch.zeros(4)
    with pytest.raises(ValueError, match="current CUDA device"):
        pa_capi.linear_attn_fwd(q, q, q, ld, q)
    with pytest.raises(ValueError, match="k must be"):
        pa_capi.linear_attn_fwd(q, q[:, :4], q, ld, q, workspace=q)
    with pytest.raises(TypeError):
        pa_capi.linear_attn_fwd(q.double(), q, q, ld, q)
    with pytest.raises(ValueError, match="sections|axes"):
        pa_capi.rope_desc(q, q, [1] * 5)
    with pytest.raises(KeyError):
        pa_capi.rope_desc(q, q, layout="both")
    d = pa_capi.rope_desc(q, q)
    with pytest.raises(ValueError, match="kv heads"):
        pa_capi.rope_fwd(q, None, torch.zeros(1, 2, 8, dtype=torch.int32), q, None, d)
    with pytest.raises(ValueError):
        pa_capi.rope_fwd(q, q, torch.zeros(1, 2, 8, dtype=torch.int64), q, q, d)
    with pytest.raises(ValueError, match="v must be contiguous"):
        pa_capi.linear_attn_fwd(q, q, q.transpose(1, 2).contiguous().transpose(1, 2), ld, q)
    with pytest.raises(ValueError, match="state_in must be"):
        pa_capi.linear_attn_step(q, q, q, ld, torch.zeros(2, 4, 64, 32), q, q)


def test_rope_refuses_outputs_over_the_other_tensor():
    import pa_capi
    lib = pa_capi.load()
    for a in ((16, 32, 64, 128, 128), (16, 32, 64, 32, 256), (16, 32, 64, 128, 16)):
        assert lib.pa_rope_fwd(_rope(), *a, None) == SHAPE
        assert lib.pa_rope_bwd(_rope(), *a, 0, None) == SHAPE


@pytest.mark.parametrize("scale", [1e-30, 1e-44, 1e30, float("inf")])
def test_linear_attention_scale_refusals(scale):
    import pa_capi
    lib = pa_capi.load()
    big = 1 << 40
    assert lib.pa_linear_attn_fwd(_desc(scale=scale), 16, 32, 48, 64, None, None, 80, None, 256, big, None) == SHAPE
    assert lib.pa_linear_attn_bwd(_desc(scale=scale), 16, 32, 48, 64, 80, None, None, None, 96, 112, 128, None, 0,
                                  256, big, None) == SHAPE
    assert lib.pa_linear_attn_step(_desc(L=1, scale=scale), 16, 32, 48, 64, 80, 96, 112, None) == SHAPE
    assert lib.pa_linear_attn_fwd_workspace_size(_desc(L=9000, scale=scale)) == 0


@pytest.mark.parametrize("e,h", [(64, 0), (0, 1), (64, 3)])
def test_layer_refuses_heads_that_do_not_divide(e, h):
    import PureAttention
    with pytest.raises(RuntimeError, match="not divisible"):
        PureAttention.LinearAttention(e, h, sections=[4])


def test_binding_refuses_workspaces_that_the_kernel_must_not_write():
    """A workspace of another device, or a view that counts more bytes than its memory holds, is
    refused like any other tensor of the call, before the library sees it."""
    torch = pytest.importorskip("torch")
    import pa_capi

    class OnGpu:  # what the helper asks of q
        shape, dtype, device = (1, 4100, 2, 64), torch.bfloat16, "cuda:0"

        def __init__(self, index):
            self.index = index

        def get_device(self):
            return self.index

    d = pa_capi.AttnDesc(1, 4100, 2, 64, pa_capi.PA_BF16, 0.0)
    plain = torch.empty(1 << 22, dtype=torch.uint8)
    view = torch.empty(1, dtype=torch.uint8).expand(1 << 22)
    strided = torch.empty(1 << 12, dtype=torch.uint8)[::2]
    for size_of in (pa_capi.linear_attn_fwd_workspace_size, pa_capi.linear_attn_bwd_workspace_size):
        for ws in (plain, torch.empty(1 << 22, dtype=torch.uint8, device="meta")):
            with pytest.raises(ValueError, match="workspace must be on"):
                pa_capi._linear_attn_ws(size_of, d, ws, OnGpu(0), None)
        for ws in (view, strided):
            with pytest.raises(ValueError, match="workspace must be contiguous"):
                pa_capi._linear_attn_ws(size_of, d, ws, OnGpu(-1), None)
        assert pa_capi._linear_attn_ws(size_of, d, plain, OnGpu(-1), None) == (plain, 1 << 22)


# 2 x 128 tokens of 2 heads of 64 in bf16 and 2 x 2 states of 64 x 64: 64 KB each, so addresses 64 KB apart
# are tensors side by side
K64 = 1 << 16


def _spans(n):
    return [(i + 1) * K64 for i in range(n)]


@pytest.mark.parametrize("shift", [16, K64 - 16, 16 - K64, -16, 0])
def test_linear_attention_refuses_tensors_that_share_bytes(shift):
    """Each output over each input, each other output and the workspace, by 16 bytes, by all but 16, and whole."""
    import pa_capi
    lib = pa_capi.load()

    def each(call, names, outputs, free=()):
        at = dict(zip(names, _spans(len(names))))
        for o in outputs:
            for other in names:
                if other != o and (o, other, shift) not in free:
                    assert call(dict(at, **{o: at[other] + shift})) == SHAPE, (o, other)

    names = ["q", "k", "v", "s", "o", "so", "ld", "n"]
    small = ("ld", "n")  # shorter than the shift: only what lies over them meets them
    skip = [(o, x, d) for o in ("o", "so", "dq", "dk", "dv", "dsi") for x in small for d in (16, K64 - 16)]
    each(lambda a: lib.pa_linear_attn_fwd(_desc(), a["q"], a["k"], a["v"], a["ld"], a["n"], a["s"], a["o"], a["so"],
                                          None, 0, None), names, ("o", "so"), [*skip, ("so", "s", 0)])
    names = ["q", "k", "v", "dO", "s", "ds", "dq", "dk", "dv", "dsi", "ld", "n"]
    each(lambda a: lib.pa_linear_attn_bwd(_desc(), a["q"], a["k"], a["v"], a["dO"], a["ld"], a["n"], a["s"], a["ds"],
                                          a["dq"], a["dk"], a["dv"], a["dsi"], 0, None, 0, None),
         names, ("dq", "dk", "dv", "dsi"), skip)
    # one token: 256 sequences of 2 heads for tensors of 64 KB, 8 MB of states
    names = ["q", "k", "v", "o", "ld"]
    base = dict(zip(names, _spans(5)), s=1 << 24, so=1 << 25)
    step = lambda a: lib.pa_linear_attn_step(_desc(B=256, L=1), a["q"], a["k"], a["v"], a["ld"], a["s"], a["o"],
                                             a["so"], None)
    for x in ("q", "k", "v"):
        assert step(dict(base, o=base[x] + shift)) == SHAPE
    assert step(dict(base, o=base["s"] + shift)) == SHAPE
    if shift:
        assert step(dict(base, so=base["s"] + shift)) == SHAPE
    assert step(dict(base, so=base["o"] + shift)) == SHAPE


def test_linear_attention_refuses_a_workspace_over_a_tensor():
    """And takes one beside it: then a workspace that is too small is what is wrong."""
    import pa_capi
    lib = pa_capi.load()
    desc = ctypes.byref(pa_capi.AttnDesc(1, 8192, 2, 64, pa_capi.PA_BF16, 0.0))  # tensors of 2 MB
    need = lib.pa_linear_attn_fwd_workspace_size(desc)
    assert need > 0
    M2 = 2 << 20
    fwd = lambda ws, nb: lib.pa_linear_attn_fwd(desc, M2, 2 * M2, 3 * M2, 64, None, None, 4 * M2, None, ws, nb, None)
    for ws in (M2, 2 * M2 + 256, 4 * M2 - 256, 5 * M2 - 256):
        assert fwd(ws, need) == SHAPE
    assert fwd(5 * M2, need - 1) == WORKSPACE
    assert fwd(None, 0) == WORKSPACE


@pytest.mark.parametrize("shift", [16, 1024, -16])
def test_rope_refuses_tensors_that_share_bytes(shift):
    """8 tokens of 2 heads of 64 in bf16 (2 KB) and of 1 (1 KB); positions 64 bytes."""
    import pa_capi
    lib = pa_capi.load()
    q, k, pos, qo, ko = 1 << 16, 2 << 16, 3 << 16, 4 << 16, 5 << 16
    in_k = shift if abs(shift) < 1024 else 512
    for a in ((q, k, pos, q + shift, ko), (q, k, pos, k + in_k, ko), (q, k, pos, k, ko), (q, k, pos, qo, q + shift),
              (q, k, pos, qo, k + in_k), (q, k, pos, qo, qo + shift), (q, k, pos, pos - 16, ko),
              (q, k, pos, q, q + shift), (q, k, pos, qo, pos - 1008)):
        assert lib.pa_rope_fwd(_rope(), *a, None) == SHAPE, a
        assert lib.pa_rope_bwd(_rope(), *a, 0, None) == SHAPE, a
        assert lib.pa_rope_bwd(_rope(), *a, 1, None) == SHAPE, a

"""Linear attention with a decay per head through the C ABI against its 64-bit
quadratic form: forward, backward, carried states and the single-token step.

Tolerances, per value, from the roundings of the kernels. `mag` is the same sum
with every factor's magnitude, so an error of r in every factor moves a value by
at most r * mag.
  bf16 operands: each term of an output has one factor rounded to bf16 on the way, a score or
      the state entering its chunk (2^-8 of `mag`), and the output's rounding (2^-8 of the
      value); the states' own errors (next but one) are inside 2^-8 x 0.02: 2^-8 (|value| + 1.02 mag).
  fp32 operands (split products): an operand in two bf16 parts is off by 2^-16,
      the product drops the low parts' product, 2^-16: 3 x 2^-16 a product, two
      products in a row and two splits of the state: 12 x 2^-16 < 2^-12 of mag.
  states from bf16 operands: values times decay in two parts 2^-16 and fp32 sums:
      2^-15 of mag; from fp32 operands 2^-12.
Norm-wise, roundings of random sign: bf16 2^-8 x 2 (the output's own rounding and one more), fp32 2^-15."""
import pytest

torch = pytest.importorskip("torch")
from conftest import rel_err  # noqa: E402
from seq_ref import mix, mix_grads, mix_grads_absolute  # noqa: E402

REL = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -12}
NORM = {torch.bfloat16: 2.0 ** -7, torch.float32: 2.0 ** -15}
STATE = {torch.bfloat16: 2.0 ** -15, torch.float32: 2.0 ** -12}


def _close(got, want, mag, r, step):
    err = (got.double() - want).abs()
    tol = step * want.abs() + 1.02 * r * mag + 1e-30
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{worst} of the tolerance"


def _inputs(B, L, H, D, dtype, seed, decays=None, states=False):
    g = torch.Generator().manual_seed(seed)
    q, k, v, dO = ((0.5 * torch.randn(B, L, H, D, generator=g)).to(dtype).cuda() for _ in range(4))
    if decays is None:
        decays = [-(2.0 ** -(8.0 * (h + 1) / H)) for h in range(H)]
    ld = torch.tensor(decays, dtype=torch.float32).cuda()
    s, ds = ((torch.randn(B, H, D, D, generator=g).cuda() if states else None) for _ in range(2))
    return q, k, v, dO, ld, s, ds


def _forward(q, k, v, ld, **kw):
    import pa_capi
    B, L, H, D = q.shape
    o = torch.full_like(q, float("nan"))
    so = torch.full((B, H, D, D), float("nan"), device="cuda")
    pa_capi.linear_attn_fwd(q, k, v, ld, o, state_out=so, **kw)
    assert pa_capi.device_status() == 0
    return o, so


def _check_forward(q, k, v, ld, lens=None, s=None, scale=None):
    import pa_capi
    desc = pa_capi.attn_desc(q, scale=scale or 0.0)
    o, so = _forward(q, k, v, ld, seq_lens=lens, state_in=s, desc=desc)
    want, ws = mix(q, k, v, ld, lens, s, scale)
    mag, ms = mix(q, k, v, ld, lens, s, scale, absolute=True)
    t = q.dtype
    _close(o, want, mag, REL[t], 2.0 ** -8 if t == torch.bfloat16 else 2.0 ** -24)
    _close(so, ws, ms, STATE[t], 2.0 ** -24)
    if want.norm() > 0:
        assert rel_err(o.double().cpu(), want.cpu()) < NORM[t]
    return o, so


TYPES = [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 32), (torch.float32, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", TYPES)
@pytest.mark.parametrize("L", [1, 2, 63, 64, 65, 127, 128, 129, 257, 500])
def test_forward_lengths(dtype, D, L):
    q, k, v, _, ld, _, _ = _inputs(2, L, 3, D, dtype, L)
    _check_forward(q, k, v, ld)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", TYPES)
def test_forward_state_and_ragged(dtype, D):
    """Padded batch: lengths of zero, one, a tile's border, full, and beyond the range; the padding
    holds NaN and infinities, which must reach neither outputs nor states."""
    q, k, v, _, ld, s, _ = _inputs(7, 300, 2, D, dtype, 5, states=True)
    lens = torch.tensor([0, 1, 128, 129, 300, 999, -4], dtype=torch.int32)
    for b in range(7):
        n = max(0, min(300, int(lens[b])))
        for x in (q, k, v):
            x[b, n:] = float("nan")
            x[b, n::2] = float("inf")
    o, so = _check_forward(q, k, v, ld, lens.cuda(), s)
    for b in range(7):
        assert (o[b, max(0, min(300, int(lens[b]))):] == 0).all()
    assert torch.equal(so[0], s[0]) and torch.equal(so[6], s[6])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", TYPES)
def test_forward_decays(dtype, D):
    """No decay, a fast one, one that underflows within a tile, zero (each token alone), a growing one."""
    decays = [0.0, -0.7, -9.0, -1e3, float("-inf"), 0.01]
    q, k, v, _, ld, s, _ = _inputs(1, 280, 6, D, dtype, 6, decays, states=True)
    _check_forward(q, k, v, ld, None, s)


@pytest.mark.gpu
def test_forward_scale_and_values_of_all_sizes():
    q, k, v, _, ld, s, _ = _inputs(2, 200, 2, 64, torch.bfloat16, 7, states=True)
    _check_forward(q, k, v, ld, None, s, scale=1.0)
    _check_forward(q * 2.0 ** 40, k * 2.0 ** -30, v * 2.0 ** 20, ld, None, s * 2.0 ** -10)
    z = torch.zeros_like(q)
    o, so = _forward(z, z, z, ld)
    assert (o == 0).all() and (so == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", TYPES)
@pytest.mark.parametrize("B,H,L", [(1, 1, 4100), (2, 8, 1500), (1, 3, 9000)])
def test_long_sequences_of_few_heads(dtype, D, B, H, L):
    """Few (sequence, head) pairs: the work of one is split over the GPU and joined."""
    q, k, v, dO, ld, s, ds = _inputs(B, L, H, D, dtype, 8, states=True)
    lens = torch.tensor([L - 77 * b for b in range(B)], dtype=torch.int32).cuda()
    _check_forward(q, k, v, ld, lens, s)
    _check_backward(q, k, v, dO, ld, lens, s, ds)


def _check_backward(q, k, v, dO, ld, lens=None, s=None, ds=None, accumulate=False):
    import pa_capi
    t = q.dtype
    base = [torch.randn_like(q) if accumulate else torch.full_like(q, float("nan")) for _ in range(3)]
    g = [x.clone() for x in base]
    dsi = torch.full((*q.shape[:1], q.shape[2], q.shape[3], q.shape[3]), float("nan"), device="cuda")
    pa_capi.linear_attn_bwd(q, k, v, dO, ld, *g, seq_lens=lens, state_in=s, d_state_out=ds,
                            d_state_in=dsi, accumulate=accumulate)
    assert pa_capi.device_status() == 0
    want = mix_grads(q, k, v, ld, dO, lens, s, ds)
    mag = mix_grads_absolute(q, k, v, ld, dO, lens, s, ds)
    step = 2.0 ** -8 if t == torch.bfloat16 else 2.0 ** -24
    for got, w, m, b0 in zip(g, want, mag, base):
        w = w + b0.double() if accumulate else w
        _close(got, w, m, REL[t], step * 1.01)
        if w.norm() > 0:
            assert rel_err(got.double().cpu(), w.cpu()) < NORM[t]
    _close(dsi, want[3], mag[3], STATE[t], 2.0 ** -24)
    return g, dsi


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", TYPES)
@pytest.mark.parametrize("L", [1, 2, 64, 127, 129, 300])
def test_backward_lengths(dtype, D, L):
    q, k, v, dO, ld, s, ds = _inputs(2, L, 3, D, dtype, 20 + L, states=True)
    _check_backward(q, k, v, dO, ld)
    _check_backward(q, k, v, dO, ld, None, s, ds)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", TYPES)
def test_backward_ragged_and_accumulating(dtype, D):
    q, k, v, dO, ld, s, ds = _inputs(5, 260, 2, D, dtype, 30, [-0.3, float("-inf")], states=True)
    lens = torch.tensor([0, 1, 128, 131, 260], dtype=torch.int32)
    for b in range(5):
        for x in (q, k, v, dO):
            x[b, int(lens[b]):] = float("nan")
    lens = lens.cuda()
    g, dsi = _check_backward(q, k, v, dO, ld, lens, s, ds)
    for b in range(5):
        for x in g:
            assert (x[b, int(lens[b]):] == 0).all()
    assert rel_err(dsi[0].cpu(), ds[0].cpu()) < 2.0 ** -22  # no token: the gradient passes through
    q, k, v, dO, ld, s, ds = _inputs(3, 150, 2, D, dtype, 31, states=True)
    _check_backward(q, k, v, dO, ld, torch.tensor([150, 0, 9], dtype=torch.int32).cuda(), s, ds, accumulate=True)


@pytest.mark.gpu
def test_gradients_against_differences():
    """o is linear in each of q, k, v and the state, so a difference of the forward over any step is
    the gradient along it: <dO, o(q + d) - o(q)> = <dq, d>, with the state's part for k, v, S_0."""
    import pa_capi
    q, k, v, dO, ld, s, ds = _inputs(2, 190, 3, 64, torch.float32, 40, states=True)
    g = [torch.empty_like(q) for _ in range(3)]
    dsi = torch.empty_like(s)
    pa_capi.linear_attn_bwd(q, k, v, dO, ld, *g, state_in=s, d_state_out=ds, d_state_in=dsi)

    def value(q, k, v, s):
        o, so = _forward(q, k, v, ld, state_in=s)
        return (o.double() * dO).sum() + (so.double() * ds).sum()

    x = [q, k, v, s]
    for i, grad in enumerate([*g, dsi]):
        d = torch.randn_like(x[i])
        hi, lo = list(x), list(x)
        hi[i], lo[i] = x[i] + d, x[i] - d
        diff = (value(*hi) - value(*lo)) / 2
        want = (grad.double() * d).sum()
        scale = grad.double().norm() * d.double().norm()
        assert abs(diff - want) <= 2.0 ** -12 * scale


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64])
def test_bf16_math_of_fp32_tensors(D):
    """set_f32_math("bf16"): as bf16 operands (v times its decay and the states excepted, which keep
    two parts), so against inputs rounded to bf16 the bf16 tolerance holds with an fp32 output."""
    import pa_capi
    q, k, v, dO, ld, s, ds = _inputs(3, 290, 2, D, torch.float32, 90, states=True)
    q, k, v, dO = (x.bfloat16().float() for x in (q, k, v, dO))
    lens = torch.tensor([290, 130, 7], dtype=torch.int32).cuda()
    pa_capi.set_f32_math("bf16")
    try:
        o, so = _forward(q, k, v, ld, seq_lens=lens, state_in=s)
        g = [torch.empty_like(q) for _ in range(3)]
        dsi = torch.empty_like(s)
        pa_capi.linear_attn_bwd(q, k, v, dO, ld, *g, seq_lens=lens, state_in=s, d_state_out=ds, d_state_in=dsi)
    finally:
        pa_capi.set_f32_math("split3")
    want, ws = mix(q, k, v, ld, lens, s)
    mag, ms = mix(q, k, v, ld, lens, s, absolute=True)
    _close(o, want, mag, 2.0 ** -8, 2.0 ** -24)
    _close(so, ws, ms, 2.0 ** -15, 2.0 ** -24)
    wg, mg = mix_grads(q, k, v, ld, dO, lens, s, ds), mix_grads_absolute(q, k, v, ld, dO, lens, s, ds)
    for got, w, m in zip(g, wg, mg):
        _close(got, w, m, 2.0 ** -8, 2.0 ** -24)
    _close(dsi, wg[3], mg[3], 2.0 ** -15, 2.0 ** -24)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", TYPES)
@pytest.mark.parametrize("B,H", [(1, 1), (5, 3), (64, 4)])
def test_step_matches_formula(dtype, D, B, H):
    import pa_capi
    q, k, v, _, ld, s, _ = _inputs(B, 1, H, D, dtype, 50 + B, states=True)
    o, so = torch.empty_like(q), torch.empty_like(s)
    pa_capi.linear_attn_step(q, k, v, ld, s, o, so)
    want, ws = mix(q, k, v, ld, None, s)
    mag, ms = mix(q, k, v, ld, None, s, absolute=True)
    step = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    _close(o, want, mag, 2.0 ** -20, step)
    _close(so, ws, ms, 2.0 ** -22, 2.0 ** -24)
    inplace = s.clone()
    pa_capi.linear_attn_step(q, k, v, ld, inplace, o, inplace)
    assert torch.equal(inplace, so)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", TYPES)
def test_prompt_in_pieces_then_tokens_equals_one_pass(dtype, D):
    """A prompt in two pieces with the state carried (in place), then single tokens: the same outputs
    as one pass over all of it."""
    import pa_capi
    B, L, H = 2, 220, 3
    q, k, v, _, ld, s, _ = _inputs(B, L, H, D, dtype, 60, states=True)
    want, ws = mix(q, k, v, ld, None, s)
    mag, ms = mix(q, k, v, ld, None, s, absolute=True)
    state, outs = s.clone(), []
    for a, b in ((0, 130), (130, 213)):
        part = [x[:, a:b].contiguous() for x in (q, k, v)]
        o = torch.empty_like(part[0])
        pa_capi.linear_attn_fwd(*part, ld, o, state_in=state, state_out=state)
        outs.append(o)
    for t in range(213, L):
        part = [x[:, t:t + 1].contiguous() for x in (q, k, v)]
        o = torch.empty_like(part[0])
        pa_capi.linear_attn_step(*part, ld, state, o, state)
        outs.append(o)
    _close(torch.cat(outs, 1), want, mag, REL[dtype], 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24)
    _close(state, ws, ms, STATE[dtype], 2.0 ** -22)


@pytest.mark.gpu
def test_same_bits_every_time_on_streams_and_in_graphs():
    """Two calls at once on two streams with a workspace each, and a captured call replayed with new
    inputs, give the bits of a call alone."""
    import pa_capi
    a = _inputs(1, 2100, 4, 64, torch.bfloat16, 70, states=True)
    b = _inputs(1, 2100, 4, 64, torch.bfloat16, 71, states=True)

    def call(x, out, ws):
        q, k, v, dO, ld, s, ds = x
        pa_capi.linear_attn_fwd(q, k, v, ld, out[0], state_in=s, state_out=out[1], workspace=ws[0])
        pa_capi.linear_attn_bwd(q, k, v, dO, ld, *out[2:5], state_in=s, d_state_out=ds, d_state_in=out[5],
                                workspace=ws[1])

    def buffers(x):
        d = pa_capi.attn_desc(x[0])
        n = (pa_capi.linear_attn_fwd_workspace_size(d), pa_capi.linear_attn_bwd_workspace_size(d))
        q, s = x[0], x[5]
        return ([torch.zeros_like(q), torch.zeros_like(s), *(torch.zeros_like(q) for _ in range(3)), torch.zeros_like(s)],
                [torch.empty(max(m, 256), dtype=torch.uint8, device="cuda") for m in n])

    alone = []
    for x in (a, b):
        out, ws = buffers(x)
        call(x, out, ws)
        alone.append(out)
    torch.cuda.synchronize()
    both = [buffers(x) for x in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for x, (out, ws), st in zip((a, b), both, streams):
            with torch.cuda.stream(st):
                call(x, out, ws)
    torch.cuda.synchronize()
    for (out, _), want in zip(both, alone):
        assert all(torch.equal(m, n) for m, n in zip(out, want))
    out, ws = buffers(a)
    x = [t.clone() for t in a]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(x, out, ws)
    for src, want in ((a, alone[0]), (b, alone[1])):
        for t, n in zip(x, src):
            t.copy_(n)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(m, n) for m, n in zip(out, want))
    assert pa_capi.device_status() == 0


@pytest.mark.gpu
def test_rotary_then_linear_attention_trains_as_in_64_bits():
    """The two together as a layer uses them: turn q and k, mix, and the gradients back through both."""
    import pa_capi
    from seq_ref import turn
    B, L, H, D = 2, 333, 4, 64
    q, k, v, dO, ld, _, _ = _inputs(B, L, H, D, torch.float32, 80)
    pos = torch.stack([torch.arange(L) // 49, torch.arange(L) // 7 % 7, torch.arange(L) % 7]).int()
    pos = pos[:, None].expand(3, B, L).contiguous().cuda()
    sections = [8, 12, 12]
    desc = pa_capi.rope_desc(q, k, sections)
    qr, kr, o = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q)
    pa_capi.rope_fwd(q, k, pos, qr, kr, desc)
    pa_capi.linear_attn_fwd(qr, kr, v, ld, o)
    g = [torch.empty_like(q) for _ in range(3)]
    pa_capi.linear_attn_bwd(qr, kr, v, dO, ld, *g)
    pa_capi.rope_bwd(g[0], g[1], pos, g[0], g[1], desc)
    x = [t.double().requires_grad_() for t in (q, k, v)]
    want, _ = mix(turn(x[0], pos, sections), turn(x[1], pos, sections), x[2], ld)
    assert rel_err(o.double().cpu(), want.detach().cpu()) < NORM[torch.float32]
    for got, w in zip(g, torch.autograd.grad((want * dO.double()).sum(), x)):
        assert rel_err(got.double().cpu(), w.cpu()) < NORM[torch.float32]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", TYPES)
def test_more_heads_than_sms_with_lengths_of_all_kinds(dtype, D):
    """Each block takes several (sequence, head) pairs one after another, some of them empty."""
    B, L, H = 61, 270, 5
    q, k, v, dO, ld, s, ds = _inputs(B, L, H, D, dtype, 90, states=True)
    g = torch.Generator().manual_seed(91)
    lens = torch.randint(-3, L + 9, (B,), generator=g, dtype=torch.int32)
    lens[::7] = 0
    lens[1::9] = 1
    lens[2::11] = 128
    for b in range(B):
        for x in (q, k, v, dO):
            x[b, max(0, int(lens[b])):] = float("nan")
    lens = lens.cuda()
    _check_forward(*(torch.nan_to_num(x) for x in (q, k, v)), ld, lens, s)
    o, _ = _forward(q, k, v, ld, seq_lens=lens, state_in=s)
    assert torch.isfinite(o).all()
    _check_backward(q, k, v, dO, ld, lens, s, ds)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", TYPES)
def test_segments_with_short_and_empty_sequences(dtype, D):
    """Long enough to be cut into segments, most of which the shorter sequences do not reach."""
    q, k, v, dO, ld, s, ds = _inputs(4, 4500, 2, D, dtype, 92, states=True)
    lens = torch.tensor([4500, 130, 0, 2049], dtype=torch.int32).cuda()
    _check_forward(q, k, v, ld, lens, s)
    _check_backward(q, k, v, dO, ld, lens, s, ds)
    _check_backward(q, k, v, dO, ld, lens, None, None, accumulate=True)


@pytest.mark.gpu
def test_past_2_31_values():
    """The last tokens of tensors of more than 2^31 values. With a decay of e^-0.7 what lies 400
    tokens back counts e^-280: the last 600 tokens alone give them."""
    import pa_capi
    B, L, H, D, W, C = 1, (1 << 19) + 77, 64, 64, 600, 200
    t, heads = torch.bfloat16, [0, 63]
    q, k, v, dO = (torch.empty(B, L, H, D, dtype=t, device="cuda").normal_(std=0.5) for _ in range(4))
    ld = torch.full((H,), -0.7, device="cuda")
    o = torch.full_like(q, float("nan"))
    so = torch.empty(B, H, D, D, device="cuda")
    pa_capi.linear_attn_fwd(q, k, v, ld, o, state_out=so)
    x = [y[:, -W:, heads].contiguous() for y in (q, k, v, dO)]
    want, ws = mix(*x[:3], ld[heads])
    mag, ms = mix(*x[:3], ld[heads], absolute=True)
    _close(o[:, -C:, heads], want[:, -C:], mag[:, -C:], REL[t], 2.0 ** -8)
    _close(so[:, heads], ws, ms, STATE[t], 2.0 ** -24)
    g = [o] + [torch.empty_like(q) for _ in range(2)]
    for y in g:
        y.fill_(1.0)
    pa_capi.linear_attn_bwd(q, k, v, dO, ld, *g, accumulate=True)
    assert pa_capi.device_status() == 0
    want = mix_grads(*x[:3], ld[heads], x[3])
    mag = mix_grads_absolute(*x[:3], ld[heads], x[3])
    for got, w, m in zip(g, want, mag):
        _close(got[:, -C:, heads], w[:, -C:] + 1.0, m[:, -C:], REL[t], 2.0 ** -8 * 1.01)


@pytest.mark.gpu
def test_workspace_of_a_call_on_a_stream_given_by_its_handle():
    """The workspace that the binding allocates belongs to the stream that the kernels run on."""
    import pa_capi
    q, k, v, dO, ld, _, _ = _inputs(1, 4100, 2, 64, torch.bfloat16, 93)
    want, _ = _forward(q, k, v, ld)
    side = torch.cuda.Stream()
    for handle, st in ((side.cuda_stream, side), (0, torch.cuda.default_stream())):
        outs = [torch.zeros_like(q) for _ in range(4)]
        torch.cuda.synchronize()
        for o in outs:
            pa_capi.linear_attn_fwd(q, k, v, ld, o, stream=handle)
            torch.full((1 << 22,), float("nan"), device="cuda")  # would take a freed workspace of its own stream
        st.synchronize()
        assert all(torch.equal(o, want) for o in outs)


@pytest.mark.gpu
def test_a_refused_scale_does_not_change_the_workspace_of_later_calls():
    import pa_capi
    q, k, v, _, ld, _, _ = _inputs(1, 4100, 2, 64, torch.bfloat16, 94)
    with pytest.raises(pa_capi.PaError):
        _forward(q, k, v, ld, desc=pa_capi.attn_desc(q, scale=1e-30))
    _check_forward(q, k, v, ld)
    assert pa_capi.linear_attn_fwd_workspace_size(pa_capi.attn_desc(q)) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", TYPES)
@pytest.mark.parametrize("B,L,H", [(1, 100, 2), (2, 900, 3), (1, 4100, 2), (61, 270, 5)])
def test_calls_after_a_recorded_error_end_at_once(dtype, D, B, L, H):
    """While an error of an earlier wait is recorded, a call waits for the copies that its blocks have already sent
    for and for nothing else: it ends within a few milliseconds (a wait for a copy that was never sent takes
    20), leaves its outputs as they were, and the same call is right once the error is cleared."""
    import pa_capi
    q, k, v, dO, ld, s, ds = _inputs(B, L, H, D, dtype, 95, states=True)
    want = (*_forward(q, k, v, ld, state_in=s), *(torch.empty_like(q) for _ in range(3)), torch.empty_like(s))

    def call(o, so, dq, dk, dv, dsi):
        pa_capi.linear_attn_fwd(q, k, v, ld, o, state_in=s, state_out=so)
        pa_capi.linear_attn_bwd(q, k, v, dO, ld, dq, dk, dv, state_in=s, d_state_out=ds, d_state_in=dsi)

    call(*want)
    out = [torch.full_like(x, float("nan")) for x in want]
    torch.cuda.synchronize()
    pa_capi.wait_selftest(1_000_000, arrive=False)
    try:
        assert pa_capi.device_status(clear=False) == 6
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        call(*out)
        b.record()
        torch.cuda.synchronize()
        assert a.elapsed_time(b) < 10
        assert all(torch.isnan(x).all() for x in out)
    finally:
        assert pa_capi.device_status(clear=True) == 6
    call(*out)
    assert pa_capi.device_status() == 0
    assert all(torch.equal(x, w) for x, w in zip(out, want))


@pytest.mark.gpu
def test_tensors_side_by_side_in_one_buffer():
    """Slices of one allocation that touch and do not overlap are separate tensors, the same tensor may be
    several inputs, and a slice that overlaps another by one vector is refused."""
    import pa_capi
    B, L, H, D = 1, 4100, 2, 64
    q, k, v, dO, ld, s, ds = _inputs(B, L, H, D, torch.bfloat16, 96, states=True)
    n = q.numel()
    buf = torch.empty(8 * n, dtype=q.dtype, device="cuda")
    a = [buf[i * n:(i + 1) * n].view(q.shape) for i in range(8)]
    for x, y in zip(a, (q, k, v, dO)):
        x.copy_(y)
    o, _ = _forward(q, k, v, ld)
    pa_capi.linear_attn_fwd(*a[:3], ld, a[4])
    assert torch.equal(a[4], o)
    want = [torch.empty_like(q) for _ in range(3)]
    pa_capi.linear_attn_bwd(q, k, v, dO, ld, *want)
    pa_capi.linear_attn_bwd(*a[:4], ld, *a[4:7])
    assert all(torch.equal(x, w) for x, w in zip(a[4:7], want))
    pa_capi.linear_attn_fwd(q, q, q, ld, o)
    _close(o, *(mix(q, q, q, ld, absolute=m)[0] for m in (False, True)), REL[q.dtype], 2.0 ** -8)
    off = buf[n * 3 - 8:n * 4 - 8].view(q.shape)
    with pytest.raises(pa_capi.PaError):
        pa_capi.linear_attn_fwd(*a[:3], ld, off)
    with pytest.raises(pa_capi.PaError):
        pa_capi.linear_attn_bwd(*a[:4], ld, a[4], a[5], buf[n * 6 - 8:n * 7 - 8].view(q.shape))
    pos = torch.arange(L, dtype=torch.int32, device="cuda").view(1, 1, L)
    desc = pa_capi.rope_desc(q, k)
    turned = [torch.empty_like(q) for _ in range(2)]
    pa_capi.rope_fwd(q, k, pos, *turned, desc)
    a[0].copy_(q)
    a[1].copy_(k)
    pa_capi.rope_fwd(a[0], a[1], pos, a[0], a[2], desc)  # q in place, k beside itself
    assert torch.equal(a[0], turned[0]) and torch.equal(a[2], turned[1])
    with pytest.raises(pa_capi.PaError):
        pa_capi.rope_fwd(a[0], a[1], pos, a[3], buf[n * 2 - 8:n * 3 - 8].view(q.shape), desc)


@pytest.mark.gpu
def test_the_bindings_workspace_is_allocated_on_the_stream_of_the_call(monkeypatch):
    """Whatever stream is current: memory that the allocator may hand out again on another one while the
    kernels still write it would change results now and then only, so the allocation itself is looked at; and
    the same memory is then asked for and overwritten on the current stream."""
    import pa_capi
    q, k, v, dO, ld, _, _ = _inputs(1, 4100, 2, 64, torch.bfloat16, 97)
    want = _forward(q, k, v, ld)[0], *(torch.empty_like(q) for _ in range(3))
    pa_capi.linear_attn_bwd(q, k, v, dO, ld, *want[1:])
    d = pa_capi.attn_desc(q)
    sizes = [pa_capi.linear_attn_fwd_workspace_size(d), pa_capi.linear_attn_bwd_workspace_size(d)]
    assert min(sizes) > 0
    empty, made = torch.empty, []

    def watched(*a, **kw):
        made.append((a[0], torch.cuda.current_stream().cuda_stream))
        return empty(*a, **kw)

    side = torch.cuda.Stream()
    default = torch.cuda.default_stream()
    for handle, expect, current in ((side.cuda_stream, side, default), (None, default, default), (None, side, side),
                                    (0, default, side)):
        outs = [[torch.zeros_like(q) for _ in range(4)] for _ in range(3)]
        torch.cuda.synchronize()
        with torch.cuda.stream(current):
            for o in outs:
                made.clear()
                with monkeypatch.context() as m:
                    m.setattr(torch, "empty", watched)
                    pa_capi.linear_attn_fwd(q, k, v, ld, o[0], stream=handle)
                    pa_capi.linear_attn_bwd(q, k, v, dO, ld, *o[1:], stream=handle)
                assert made == [(n, expect.cuda_stream) for n in sizes]
                if current is not expect:
                    for n in sizes * 2:
                        torch.full((n,), 255, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(x, w) for x, w in zip(o, want))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64])
def test_bf16_math_of_fp32_tensors_cut_into_segments(D):
    """As test_bf16_math_of_fp32_tensors, with sequences long enough for segment states, and lengths that end
    inside and between segments."""
    import pa_capi
    B, L, H = 2, 4100, 2
    q, k, v, dO, ld, s, ds = _inputs(B, L, H, D, torch.float32, 98, states=True)
    q, k, v, dO = (x.bfloat16().float() for x in (q, k, v, dO))
    assert pa_capi.linear_attn_fwd_workspace_size(pa_capi.attn_desc(q)) > 0
    for lens in (None, torch.tensor([4001, 1290], dtype=torch.int32).cuda()):
        pa_capi.set_f32_math("bf16")
        try:
            o, so = _forward(q, k, v, ld, seq_lens=lens, state_in=s)
            g = [torch.empty_like(q) for _ in range(3)]
            dsi = torch.empty_like(s)
            pa_capi.linear_attn_bwd(q, k, v, dO, ld, *g, seq_lens=lens, state_in=s, d_state_out=ds, d_state_in=dsi)
        finally:
            pa_capi.set_f32_math("split3")
        want, ws = mix(q, k, v, ld, lens, s)
        mag, ms = mix(q, k, v, ld, lens, s, absolute=True)
        _close(o, want, mag, 2.0 ** -8, 2.0 ** -24)
        _close(so, ws, ms, 2.0 ** -15, 2.0 ** -24)
        wg, mg = mix_grads(q, k, v, ld, dO, lens, s, ds), mix_grads_absolute(q, k, v, ld, dO, lens, s, ds)
        for got, w, m in zip(g, wg, mg):
            _close(got, w, m, 2.0 ** -8, 2.0 ** -24)
        _close(dsi, wg[3], mg[3], 2.0 ** -15, 2.0 ** -24)
        # one bf16 per operand, or these would not be the kernels of that mode: more than split products allow
        assert rel_err(o.double().cpu(), want.cpu()) > NORM[torch.float32]


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype,D", TYPES)
def test_how_far_a_value_that_is_not_finite_reaches(dtype, D, bad):
    """One such value in one valid token: outputs and dq of the chunks of 128 tokens before its own, and dk and dv of
    those after it, keep their bits, as do all other heads and sequences. Cut and uncut sequences."""
    import pa_capi
    for L, t in ((700, 300), (4100, 2050)):
        x = list(_inputs(2, L, 2, D, dtype, 99, states=True))
        ld, s, ds = x[4:]
        for i in range(4):  # q, k, v, dO in turn
            y = [z.clone() for z in x[:4]]
            y[i][1, t, 1, D // 2] = bad
            got = []
            for q, k, v, dO in (x[:4], y):
                o, so = _forward(q, k, v, ld, state_in=s)
                g = [torch.empty_like(q) for _ in range(3)]
                dsi = torch.empty_like(s)
                pa_capi.linear_attn_bwd(q, k, v, dO, ld, *g, state_in=s, d_state_out=ds, d_state_in=dsi)
                got.append((o, g[0], g[1], g[2], so, dsi))
            first, after = t // 128 * 128, (t // 128 + 1) * 128
            for n, (a, b) in enumerate(zip(*got)):
                assert torch.equal(a[0], b[0])
                if n >= 4:
                    assert torch.equal(a[1, 0], b[1, 0])
                    continue
                assert torch.equal(a[1, :, 0], b[1, :, 0])
                keep = slice(0, first) if n < 2 else slice(after, L)
                assert torch.equal(a[1, keep, 1], b[1, keep, 1])
            if i == 0:  # q alone: its own output, and no state
                assert torch.equal(got[0][4], got[1][4])
                clean = torch.ones(L, dtype=torch.bool)
                clean[t] = False
                assert torch.equal(got[0][0][1, clean], got[1][0][1, clean])
                assert not torch.isfinite(got[1][0][1, t, 1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", TYPES)
def test_replayed_steps_in_place_equal_a_loop(dtype, D):
    """A captured single-token step that updates its state in place, its token's buffers refilled before each
    replay, for more blocks than a wave holds."""
    import pa_capi
    B, H, n = 90, 16, 12
    q, k, v, _, ld, s, _ = _inputs(B, n, H, D, dtype, 100, states=True)
    token = [torch.empty_like(q[:, :1]).contiguous() for _ in range(4)]
    want, state = [], s.clone()
    for t in range(n):
        o = torch.empty_like(token[3])
        pa_capi.linear_attn_step(*(x[:, t:t + 1].contiguous() for x in (q, k, v)), ld, state, o, state)
        want.append(o)
    held = s.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pa_capi.linear_attn_step(*token[:3], ld, held, token[3], held)
    for t in range(n):
        for x, y in zip(token, (q, k, v)):
            x.copy_(y[:, t:t + 1])
        g.replay()
        assert torch.equal(token[3], want[t])
    assert torch.equal(held, state)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", TYPES)
def test_many_sequences_of_one_token(dtype, D):
    """Thousands of units of one token each through the chunks, and the gradients of both states."""
    B, H = 1300, 3
    q, k, v, dO, ld, s, ds = _inputs(B, 1, H, D, dtype, 101, states=True)
    lens = torch.ones(B, dtype=torch.int32)
    lens[::5] = 0
    _check_forward(q, k, v, ld, lens.cuda(), s)
    _check_backward(q, k, v, dO, ld, lens.cuda(), s, ds)

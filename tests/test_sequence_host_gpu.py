"""Rotary positions and linear attention through the PureAttention host layer: their graph nodes
against float64 autograd (fan-out, shared tensors, states, lengths), the LinearAttention layer's
training gradients, a prompt and single tokens against one pass, and a captured training step.

Tolerance: everything is fp32 with split products; a projection, the turn, the mix and a projection
in a row are each off by at most 2^-15 norm-wise (three products of hi and lo parts), their gradients by
a like number of stages: 8 x 2^-15 < 3e-4."""
import numpy as np
import pytest

from conftest import rel_err, seeded_normal

torch = pytest.importorskip("torch")
from seq_ref import mix, turn  # noqa: E402

TOL = 3e-4


@pytest.fixture(scope="module")
def pa():
    import PureAttention
    PureAttention.set_seed(4321)
    return PureAttention


def _t(pa, x, requires_grad=False):
    x = np.ascontiguousarray(x, dtype=np.float32)
    t = pa.Tensor(list(x.shape), requires_grad)
    t.to_device(x.ravel().tolist())
    return t


def _h(t):
    return np.asarray(t.to_host(), dtype=np.float64).reshape(t.shape())


def _g(t):
    return np.asarray(t.grad_to_host(), dtype=np.float64).reshape(t.shape())


def _ints(pa, x):
    return pa.IntTensor(list(x.shape), [int(v) for v in x.ravel()])


def _loss(pa, y, target):
    return pa.MSE()(y, _t(pa, target))


def _mse(y, target):
    return ((y - torch.from_numpy(target).double()) ** 2).mean()


@pytest.mark.gpu
@pytest.mark.parametrize("same", [False, True])
def test_rope_node(pa, same):
    """Gradients through the turn, added to what another consumer of the inputs contributes; with
    one tensor as q and k both contributions."""
    N, L, H, D = 2, 19, 3, 32
    q, k = seeded_normal(1, (N, L, H * D)), seeded_normal(2, (N, L, H * D))
    pos = np.random.default_rng(3).integers(0, 40, (2, N, L)).astype(np.int32)
    tq, tk = seeded_normal(4, (N, L, H * D)), seeded_normal(5, (N, L, H * D))
    Q = _t(pa, q, True)
    K = Q if same else _t(pa, k, True)
    qo, ko = pa.rope(Q, K, D, _ints(pa, pos), [6, 10])
    s = pa.add(pa.add(qo, ko), Q)  # Q feeds another consumer too
    loss = _loss(pa, s, tq)
    loss.backward()
    x = [torch.from_numpy(v).double().requires_grad_() for v in (q, k)]
    if same:
        x[1] = x[0]
    p = torch.from_numpy(pos)
    a, b = (turn(v.view(N, L, H, D), p, [6, 10]).view(N, L, -1) for v in x)
    _mse(a + b + x[0], tq).backward()
    assert rel_err(_h(qo), a.detach()) < 1e-6
    assert rel_err(_g(Q), x[0].grad) < TOL
    if not same:
        assert rel_err(_g(K), x[1].grad) < TOL
    # only k's output is used: q receives nothing
    Q2, K2 = _t(pa, q, True), _t(pa, k, True)
    _, ko = pa.rope(Q2, K2, D, _ints(pa, pos), [6, 10])
    _loss(pa, ko, tk).backward()
    assert not _g(Q2).any() and _g(K2).any()


@pytest.mark.gpu
@pytest.mark.parametrize("same", [False, True])
def test_linear_attention_node(pa, same):
    """Gradients of q, k, v and of the carried state, from those of the output and of the state after,
    over a padded batch."""
    N, L, H, D = 3, 140, 2, 64
    q, k, v = (seeded_normal(10 + i, (N, L, H * D), 0.5) for i in range(3))
    s = seeded_normal(14, (N, H, D, D))
    to, ts = seeded_normal(15, (N, L, H * D)), seeded_normal(16, (N, H, D, D))
    ld = np.array([-0.02, -0.6], np.float32)
    lens = np.array([140, 1, 77], np.int32)
    Q = _t(pa, q, True)
    K, V = (Q, Q) if same else (_t(pa, k, True), _t(pa, v, True))
    S = _t(pa, s, True)
    o, after = pa.linear_attention(Q, K, V, H, _t(pa, ld), _ints(pa, lens), S, True)
    # one scalar of both outputs: mse of the output, then a step through the state
    o2, _ = pa.linear_attention(_t(pa, q), _t(pa, k), _t(pa, v), H, _t(pa, ld), None, after)
    loss = _loss(pa, pa.add(o, o2), to)
    loss.backward()
    x = [torch.from_numpy(t).double().requires_grad_() for t in (q, k, v, s)]
    if same:
        x[1] = x[2] = x[0]
    heads = [t.view(N, L, H, D) for t in x[:3]]
    l = torch.from_numpy(ld)
    ro, rs = mix(*heads, l, torch.from_numpy(lens), x[3])
    c = [torch.from_numpy(t).double().view(N, L, H, D) for t in (q, k, v)]
    ro2, _ = mix(*c, l, None, rs)
    _mse((ro + ro2).reshape(N, L, -1), to).backward()
    assert rel_err(_h(o), ro.detach().reshape(N, L, -1)) < TOL
    assert rel_err(_h(after), rs.detach()) < TOL
    assert rel_err(_g(Q), x[0].grad) < TOL
    if not same:
        assert rel_err(_g(K), x[1].grad) < TOL and rel_err(_g(V), x[2].grad) < TOL
    assert rel_err(_g(S), x[3].grad) < TOL
    # only the state has a gradient: q contributes nothing to it
    Q3, K3, V3 = (_t(pa, t, True) for t in (q, k, v))
    _, after = pa.linear_attention(Q3, K3, V3, H, _t(pa, ld), None, None, True)
    _loss(pa, after, ts).backward()
    y = [torch.from_numpy(t).double().requires_grad_() for t in (q, k, v)]
    _, rs = mix(*[t.view(N, L, H, D) for t in y], l)
    _mse(rs, ts).backward()
    assert not _g(Q3).any()
    assert rel_err(_g(K3), y[1].grad) < TOL and rel_err(_g(V3), y[2].grad) < TOL


def _layer_ref(x, w, H, ld, pos, sections, state=None):
    """(y, state after) of the layer in float64; w: the four parameters."""
    N, L, E = x.shape
    q, k, v = (x @ w[0] + w[1]).split(E, -1)
    q, k, v = (t.reshape(N, L, H, E // H) for t in (q, k, v))
    q, k = turn(q, pos, sections), turn(k, pos, sections)
    o, after = mix(q, k, v, ld, None, state)
    return o.reshape(N, L, E) @ w[2] + w[3], after


@pytest.mark.gpu
def test_layer_trains_and_generates(pa):
    """LinearAttention with positions of an image grid: output and every parameter's gradient; then the
    same tokens as a prompt in two pieces and single tokens, the state carried."""
    N, L, E, H = 2, 150, 128, 2
    sections, ld = [12, 20], [-0.01, -0.3]
    layer = pa.LinearAttention(E, H, ld, sections)
    x, target = seeded_normal(20, (N, L, E)), seeded_normal(21, (N, L, E))
    pos = np.stack([np.arange(L) // 12, np.arange(L) % 12])[:, None].repeat(N, 1).astype(np.int32)
    X = _t(pa, x, True)
    y = layer.forward(X, _ints(pa, pos))
    _loss(pa, y, target).backward()
    w = [torch.from_numpy(_h(p)).requires_grad_() for p in layer.parameters()]
    rx = torch.from_numpy(x).double().requires_grad_()
    ry, rs = _layer_ref(rx, w, H, torch.tensor(ld), torch.from_numpy(pos), sections)
    _mse(ry, target).backward()
    assert rel_err(_h(y), ry.detach()) < TOL
    assert rel_err(_g(X), rx.grad) < TOL
    for p, r in zip(layer.parameters(), w):
        assert rel_err(_g(p), r.grad) < TOL
    out, state = [], None
    for a, b in ((0, 100), (100, 146), *((i, i + 1) for i in range(146, L))):
        y, state = layer.forward_state(_t(pa, x[:, a:b]), _ints(pa, pos[:, :, a:b]), None, state)
        out.append(_h(y))
    assert rel_err(np.concatenate(out, 1), ry.detach()) < TOL
    assert rel_err(_h(state), rs.detach()) < TOL
    assert pa.device_status() == 0


@pytest.mark.gpu
def test_captured_training_step_beside_an_eager_graph(pa):
    """Forward and backward captured into a CUDA graph while an eager graph of the same parameters is
    alive; replays give the eager gradients."""
    N, L, E, H = 1, 260, 128, 4
    x, target = seeded_normal(30, (N, L, E)), seeded_normal(31, (N, L, E))
    pos = np.arange(L)[None, None].astype(np.int32)
    prev, s = pa.get_stream(), torch.cuda.Stream()
    pa.set_stream(s.cuda_stream)
    try:
        with torch.cuda.stream(s):
            layer = pa.LinearAttention(E, H, sections=[16])
            X, T, P = _t(pa, x), _t(pa, target), _ints(pa, pos)
            mse = pa.MSE()

            def step():
                for p in layer.parameters():
                    p.zero_grad()
                loss = mse(layer.forward(X, P), T)
                loss.backward()
                return loss

            eager = step()  # stays alive
            want = [_g(p) for p in layer.parameters()]
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                step()
            for _ in range(2):
                g.replay()
            torch.cuda.synchronize()
            for p, w in zip(layer.parameters(), want):
                assert np.array_equal(_g(p), w)
            del eager, g
    finally:
        torch.cuda.synchronize()
        pa.set_stream(prev)


@pytest.mark.gpu
def test_host_refusals(pa):
    x = _t(pa, seeded_normal(40, (1, 4, 64)))
    ld = _t(pa, np.zeros(1, np.float32))
    two = pa.IntTensor([2, 1, 4], [0] * 8)
    with pytest.raises(RuntimeError, match="head dim"):
        pa.rope(x, x, 48, two, [8, 8])
    with pytest.raises(RuntimeError, match="positions"):
        pa.rope(x, x, 64, two, [8])
    with pytest.raises(RuntimeError, match="invalid shape"):
        pa.rope(x, x, 64, two, [30, 8])
    with pytest.raises(RuntimeError, match="axes"):
        pa.rope(x, x, 64, two, [])
    with pytest.raises(ValueError, match="layout"):
        pa.rope(x, x, 64, two, [8, 8], layout="other")
    with pytest.raises(RuntimeError, match="log decay"):
        pa.linear_attention(x, x, x, 2, ld)
    with pytest.raises(RuntimeError, match="Unsupported Head Dimension"):
        pa.linear_attention(x, x, x, 4, _t(pa, np.zeros(4, np.float32)))
    with pytest.raises(RuntimeError, match="constant"):
        pa.linear_attention(x, x, x, 1, _t(pa, np.zeros(1, np.float32), True))
    with pytest.raises(RuntimeError, match="lengths"):
        pa.linear_attention(x, x, x, 1, ld, two)
    with pytest.raises(RuntimeError, match="state"):
        pa.linear_attention(x, x, x, 1, ld, None, x)
    with pytest.raises(RuntimeError, match="positions go with"):
        pa.LinearAttention(64, 1, sections=[8]).forward(x)
    with pytest.raises(RuntimeError, match="fill the shape"):
        pa.IntTensor([2, 2], [1, 2, 3])


@pytest.fixture
def no_graph(pa):
    pa.set_grad_enabled(False)
    yield
    pa.set_grad_enabled(True)


@pytest.mark.gpu
def test_generation_without_a_graph(pa, no_graph):
    """With the graph off a layer whose parameters have gradients generates token by token: the same values,
    and neither the output nor the state has a graph behind it."""
    N, E, H, sections = 1, 128, 2, [32]
    layer = pa.LinearAttention(E, H, [-0.01, -0.3], sections)
    x = seeded_normal(50, (N, 300, E))
    pos = np.arange(300, dtype=np.int32).reshape(1, 1, 300)
    w = [torch.from_numpy(_h(p)) for p in layer.parameters()]
    want, ws = _layer_ref(torch.from_numpy(x).double(), w, H, torch.tensor([-0.01, -0.3]), torch.from_numpy(pos),
                          sections)
    out, state = [], None
    for a, b in ((0, 200), *((i, i + 1) for i in range(200, 300))):
        y, state = layer.forward_state(_t(pa, x[:, a:b]), _ints(pa, pos[:, :, a:b]), None, state)
        out.append(_h(y))
    assert rel_err(np.concatenate(out, 1), want) < TOL
    assert rel_err(_h(state), ws) < TOL
    for t in (y, state):
        with pytest.raises(RuntimeError, match="does not require"):
            t.backward()


@pytest.mark.gpu
def test_one_token_takes_the_single_token_kernel_without_a_graph(pa):
    """Tensors that need gradients give the bits of tensors that need none once the graph is off."""
    ld, s = _t(pa, np.array([-0.1, -0.4], np.float32)), seeded_normal(60, (2, 2, 64, 64))
    qkv = [seeded_normal(61 + i, (2, 1, 128)) for i in range(3)]
    plain = pa.linear_attention(*(_t(pa, x) for x in qkv), 2, ld, None, _t(pa, s), True)
    assert pa.grad_enabled()
    pa.set_grad_enabled(False)
    try:
        off = pa.linear_attention(*(_t(pa, x, True) for x in qkv), 2, ld, None, _t(pa, s, True), True)
    finally:
        pa.set_grad_enabled(True)
    on = pa.linear_attention(*(_t(pa, x, True) for x in qkv), 2, ld, None, _t(pa, s, True), True)
    for a, b, c in zip(plain, off, on):
        assert np.array_equal(_h(a), _h(b))
        assert rel_err(_h(c), _h(a)) < TOL


@pytest.mark.gpu
def test_replays_of_a_captured_step_follow_their_inputs(pa):
    """Inputs and targets are rewritten between replays, and the gradients overwritten with the rewritten
    step's: what a replay leaves is its own work. Each is then compared with an eager step on the same values."""
    N, L, E, H = 2, 390, 128, 2
    pos = np.broadcast_to(np.arange(L), (1, N, L)).astype(np.int32)
    prev, s = pa.get_stream(), torch.cuda.Stream()
    pa.set_stream(s.cuda_stream)
    try:
        with torch.cuda.stream(s):
            layer = pa.LinearAttention(E, H, sections=[32])
            X, T, P = _t(pa, seeded_normal(70, (N, L, E))), _t(pa, seeded_normal(71, (N, L, E))), _ints(pa, pos)
            mse = pa.MSE()

            def step():
                for p in layer.parameters():
                    p.zero_grad()
                loss = mse(layer.forward(X, P), T)
                loss.backward()
                return loss

            def put(seed):
                X.to_device(seeded_normal(seed, (N, L, E)).ravel().tolist())
                T.to_device(seeded_normal(seed + 1, (N, L, E)).ravel().tolist())

            eager = step()  # stays alive
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                step()
            grads = []
            for seed in (72, 74):
                put(seed)
                g.replay()
                torch.cuda.synchronize()
                grads.append([_g(p) for p in layer.parameters()])
            for seed, got in zip((72, 74), grads):
                put(seed)
                loss = step()
                for p, w in zip(layer.parameters(), got):
                    assert np.array_equal(_g(p), w)
            assert not any(np.array_equal(a, b) for a, b in zip(*grads))
            del eager, loss, g
    finally:
        torch.cuda.synchronize()
        pa.set_stream(prev)


@pytest.mark.gpu
def test_the_graph_switched_off_changes_no_value_of_any_layer(pa):
    """The other layers with the graph off give the bits that they give with it on; a graph recorded before
    runs its backward while it is off, and recording goes on afterwards."""
    N, L, E = 2, 70, 128
    x, target = seeded_normal(80, (N, L, E)), _t(pa, seeded_normal(81, (N, L, E)))
    ln, mha, lin, act, mix_layer, mse = (pa.LayerNorm(E), pa.MultiheadAttention(E, 2), pa.Linear(E, E), pa.ReLU(),
                                         pa.LinearAttention(E, 2), pa.MSE())
    layers = (ln, mha, lin, mix_layer)

    def run():
        X = _t(pa, x, True)
        h = pa.add(X, mha.forward(ln.forward(X)))
        h = pa.add(h, mix_layer.forward(ln.forward(h)))
        y = act.forward(lin.forward(h))
        return X, y, mse(y, target)

    X0, y0, loss0 = run()
    loss0.backward()
    want = [_g(X0), *(_g(p) for m in layers for p in m.parameters())]
    X1, y1, loss1 = run()
    for m in layers:
        for p in m.parameters():
            p.zero_grad()
    pa.set_grad_enabled(False)
    try:
        X2, y2, loss2 = run()
        for t in (y2, loss2):
            with pytest.raises(RuntimeError, match="does not require"):
                t.backward()
        loss1.backward()
        got = [_g(X1), *(_g(p) for m in layers for p in m.parameters())]
    finally:
        pa.set_grad_enabled(True)
    assert np.array_equal(_h(y2), _h(y0)) and np.array_equal(_h(loss2), _h(loss0))
    assert all(np.array_equal(a, b) for a, b in zip(got, want))
    assert not _g(X2).any()

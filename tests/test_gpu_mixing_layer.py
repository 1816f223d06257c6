"""The operators of a layer with a matrix state as a program uses them together: normalisation in 8 bits, products of 8-bit rows, rotary positions,
linear attention, normalisation of its heads; a prompt and then tokens one at a time, a training step, a generation step in a graph. Compared with the
same program in 64-bit numpy; what it checks is results and gradients, not how well a model learns."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

B, T, H, S, DIM, WIDE = 2, 37, 4, 2, 16, 24
WIDTH = 40
EPS = 1e-5
DECAY = 1 - 2.0 ** (-2.0 - np.arange(H))


def cls_of(m, dt):
    return m.SFloat if dt == np.float32 else m.DFloat


def weights(rng):
    return {"norm": 1 + 0.1 * rng.standard_normal(WIDTH), "head": 1 + 0.1 * rng.standard_normal(WIDE), "q": rng.standard_normal((H * DIM, WIDTH)) / 6,
            "k": rng.standard_normal((S * DIM, WIDTH)) / 6, "v": rng.standard_normal((S * WIDE, WIDTH)) / 6}


def norm(v, w):
    return v / np.sqrt((v * v).mean(-1, keepdims=True) + EPS) * w


def turned(x, positions, f):
    n = len(f)
    angle = (positions[..., None] * f)[..., None, :]
    c, s = np.cos(angle), np.sin(angle)
    y = x.copy()
    y[..., :n], y[..., n:2 * n] = x[..., :n] * c - x[..., n:2 * n] * s, x[..., n:2 * n] * c + x[..., :n] * s
    return y


def attention(q, k, v, state, decay):
    o = np.zeros(q.shape[:3] + (v.shape[-1],))
    k, v = (np.repeat(x, q.shape[2] // x.shape[2], axis=2) for x in (k, v))
    for t in range(q.shape[1]):
        state = decay[:, None, None] * state + k[:, t, :, :, None] * v[:, t, :, None, :]
        o[:, t] = q.shape[-1] ** -0.5 * (q[:, t, :, :, None] * state).sum(-2)
    return o, state


def host(y, w, positions, f, state, decay):
    """From rows y and the weights as they stand for: the heads' normalised output, and the state."""
    b, t = y.shape[:2]
    q, k, v = ((y @ w[n].T).reshape(b, t, -1, d) for n, d in (("q", DIM), ("k", DIM), ("v", WIDE)))
    o, state = attention(turned(q, positions, f), turned(k, positions, f), v, state, decay)
    return norm(o, w["head"]), state


def layer(m, x, w, held, positions, f, state):
    """The same with the library: 8-bit rows and weights."""
    b, t = x.shape[:2]
    rows = m.Fused.rmsnorm_q8(x, w["norm"], eps=EPS)
    q, k, v = (m.Fused.matmul_q8(*rows, *held[n]).reshape(b, t, -1, d) for n, d in (("q", DIM), ("k", DIM), ("v", WIDE)))
    q, k = (m.Fused.rotary(z, positions, f) for z in (q, k))
    o, state = m.Fused.linear_attention(q, k, v, w["decay"], state)
    return m.Fused.rmsnorm(o, w["head"], eps=EPS), state, rows


def stands_for(m, pair):
    q, scale = (z.to_numpy().astype(np.float64) for z in pair)
    return q * scale


@pytest.mark.parametrize("dt", [np.float32, np.float64])
def test_a_prompt_and_then_tokens(dt):
    """The prompt at once, the rest one by one with the state and the positions carried along: what the host's program gives for the same 8-bit
    rows at once, within 256 roundings of its size (sums of 40 and 16 terms, 40 steps, two norms)."""
    import cumo_amd as m
    cls = cls_of(m, dt)
    rng = np.random.default_rng(1)
    w = weights(rng)
    dw = {n: cls.cast(w[n].astype(dt)) for n in ("norm", "head")}
    dw["decay"] = cls.cast(DECAY.astype(dt))
    held = {n: m.Fused.quantize(cls.cast(w[n].astype(dt))) for n in ("q", "k", "v")}
    meant = {"head": w["head"].astype(dt).astype(np.float64), **{n: stands_for(m, held[n]) for n in held}}
    f, _ = m.Fused.rotary_frequencies(DIM, 100.0)
    x = rng.standard_normal((B, T + 5, WIDTH)).astype(dt)
    start = rng.integers(0, 5000, (B, 1))
    positions = start + np.arange(T + 5)
    got, rows, state = [], [], cls.cast(np.zeros((B, H, DIM, WIDE), dt))
    for part in [slice(0, T)] + [slice(n, n + 1) for n in range(T, T + 5)]:
        y, state, r = layer(m, cls.cast(np.ascontiguousarray(x[:, part])), dw, held, m.Int32.cast(np.ascontiguousarray(positions[:, part]).astype(np.int32)), f, state)
        got.append(y.to_numpy())
        rows.append(stands_for(m, r))
    want, last = host(np.concatenate(rows, axis=1), meant, positions, f.to_numpy(), np.zeros((B, H, DIM, WIDE)), DECAY.astype(dt).astype(np.float64))
    for z, s in ((np.concatenate(got, axis=1), want), (state.to_numpy(), last)):
        assert np.abs(z - s).max() <= 256 * np.finfo(dt).eps * np.abs(s).max()


def test_a_training_step():
    """Gradients of the projected rows and of the heads' weight through norm, attention and positions, against differences in 64 bits (h^2 times a
    third derivative, 1e-10, and the loss's rounding over h)."""
    import cumo_amd as m
    D = m.DFloat
    rng = np.random.default_rng(2)
    q, k, v = (rng.standard_normal((B, T, h, d)) for h, d in ((H, DIM), (S, DIM), (S, WIDE)))
    head, g = 1 + 0.1 * rng.standard_normal(WIDE), rng.standard_normal((B, T, H, WIDE))
    f, amplitude = m.Fused.rotary_frequencies(DIM - 4, 100.0, "yarn", 4.0, trained=30)
    positions = rng.integers(0, 50, (B, 1)) + np.arange(T)
    p = m.Int32.cast(positions.astype(np.int32))
    decay = D.cast(DECAY)

    def forward(q, k, v, head):
        q, k = (m.Fused.rotary(D.cast(z), p, f, interleaved=True, amplitude=amplitude) for z in (q, k))
        v = D.cast(v)
        o, last = m.Fused.linear_attention(q, k, v, decay)
        return m.Fused.rmsnorm(o, D.cast(head), eps=EPS), (q, k, v, o, last)

    y, (rq, rk, rv, o, last) = forward(q, k, v, head)
    gl = rng.standard_normal(last.shape)
    go, ghead = m.Fused.rmsnorm_grad(D.cast(g), o, D.cast(head), eps=EPS)
    gq, gk, gv = m.Fused.linear_attention_grad(go, rq, rk, rv, decay, None, D.cast(gl))
    gq, gk = (m.Fused.rotary(z, p, f, interleaved=True, inverse=True, amplitude=amplitude) for z in (gq, gk))

    def loss(**moved):
        y, kept = forward(**{**dict(q=q, k=k, v=v, head=head), **moved})
        return float((y.to_numpy() * g).sum() + (kept[-1].to_numpy() * gl).sum())

    for name, z, places in (("q", gq, [(0, 0, 0, 0), (1, 36, 3, 15), (0, 20, 2, 5)]), ("k", gk, [(0, 0, 1, 3), (1, 18, 0, 11), (0, 36, 1, 14)]),
                            ("v", gv, [(0, 0, 0, 23), (1, 17, 1, 2)]), ("head", ghead, [(0,), (23,)])):
        size = np.abs(z.to_numpy()).max()
        for at in places:
            both = []
            for sign in (1, -1):
                moved = {"q": q, "k": k, "v": v, "head": head}[name].copy()
                moved[at] += sign * 1e-5
                both.append(loss(**{name: moved}))
            assert abs((both[0] - both[1]) / 2e-5 - z.to_numpy()[at]) <= 1e-6 * max(1.0, size), (name, at)


def test_a_generation_step_captured_and_replayed():
    """One token through the layer in a graph, the state updated in place from replay to replay."""
    import cumo_amd as m
    from cumo_amd import _lib
    from test_gpu_index import hip_runtime
    hip, L = hip_runtime(), _lib.lib
    rng = np.random.default_rng(3)
    w = weights(rng)
    dw = {n: m.SFloat.cast(w[n].astype(np.float32)) for n in ("norm", "head")}
    held = {n: m.Fused.quantize(m.SFloat.cast(w[n].astype(np.float32))) for n in ("q", "k", "v")}
    f, _ = m.Fused.rotary_frequencies(DIM, 100.0)
    x = m.SFloat.cast(rng.standard_normal((B, 1, WIDTH)).astype(np.float32))
    p = m.Int32.cast(np.array([[17], [400]], np.int32))
    decay = m.SFloat.cast(DECAY.astype(np.float32))
    state = m.SFloat.cast(np.zeros((B, H, DIM, WIDE), np.float32))
    dw["decay"] = decay
    r8, rs = m.Int8(B, 1, WIDTH), m.SFloat(B, 1, 1)
    out = {n: m.SFloat(B, 1, h * d) for n, h, d in (("q", H, DIM), ("k", S, DIM), ("v", S, WIDE))}
    heads = {n: out[n].reshape(B, 1, h, d) for n, h, d in (("q", H, DIM), ("k", S, DIM), ("v", S, WIDE))}
    o, y = m.SFloat(B, 1, H, WIDE), m.SFloat(B, 1, H, WIDE)
    ref = lambda z: C.byref(z._desc())  # noqa: E731
    keep = {n: ref(z) for n, z in dict(x=x, p=p, f=f, decay=decay, state=state, r8=r8, rs=rs, o=o, y=y, norm=dw["norm"], head=dw["head"]).items()}
    flat, by_head = ({n: ref(z) for n, z in d.items()} for d in (out, heads))
    weight = {n: [ref(z) for z in pair] for n, pair in held.items()}

    def call():
        _lib.call(L.cumo_hip_na_rmsnorm_q8, keep["x"], keep["norm"], None, EPS, keep["r8"], keep["rs"], None)
        for n in ("q", "k", "v"):
            _lib.call(L.cumo_hip_na_matmul_q8, keep["r8"], keep["rs"], *weight[n], None, flat[n])
        for n in ("q", "k"):   # (in place)
            _lib.call(L.cumo_hip_na_rotary, by_head[n], keep["p"], keep["f"], 0, 0, 1.0, by_head[n])
        _lib.call(L.cumo_hip_na_linear_attention, by_head["q"], by_head["k"], by_head["v"], keep["decay"], keep["state"], None, DIM ** -0.5, keep["o"], keep["state"])
        _lib.call(L.cumo_hip_na_rmsnorm, keep["o"], keep["head"], None, EPS, keep["y"], None)

    stream = C.c_void_p(L.cumo_hip_stream_create())
    graph, ready = C.c_void_p(), C.c_void_p()
    m.synchronize()
    L.cumo_hip_set_stream(stream)
    try:
        assert hip.hipStreamBeginCapture(stream, 2) == 0
        capture = m.MemoryPool.capture_id()
        call()
        assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert hip.hipGraphInstantiate(C.byref(ready), graph, None, None, C.c_size_t(0)) == 0
        assert m.MemoryPool.captured_blocks(capture) == 2   # (the turned q and k; the state is written where it is)
        before = m.SFloat.cast(np.zeros((B, H, DIM, WIDE), np.float32))
        for _ in range(4):
            dirt = [m.SFloat(n).fill(float("nan")) for n in (64, 3000, 100000)]
            y.fill(9)
            assert hip.hipGraphLaunch(ready, stream) == 0
            m.synchronize()
            want, before, _ = layer(m, x, dw, held, p, f, before)
            assert (y.to_numpy() == want.to_numpy()).all() and (state.to_numpy() == before.to_numpy()).all()
            del dirt
    finally:
        L.cumo_hip_set_stream(None)
        if ready:
            hip.hipGraphExecDestroy(ready)
        if graph:
            hip.hipGraphDestroy(graph)
        L.cumo_hip_stream_destroy(stream)


def test_two_streams_at_once():
    """Calls with scratch (segments of a long sequence, parts of inner) on two streams beside each other: each answers what it does alone."""
    import cumo_amd as m
    from cumo_amd import _lib
    L = _lib.lib
    rng = np.random.default_rng(4)
    sets = []
    for _ in range(2):
        q, k, v = (m.SFloat.cast(rng.standard_normal((1, 3000, 2, d)).astype(np.float32)) for d in (40, 40, 24))
        a = m.SFloat.cast(np.array([0.9, 0.999], np.float32))
        x, w = (m.Fused.quantize(m.SFloat.cast(rng.standard_normal((n, 4000)).astype(np.float32))) for n in (100, 130))
        sets.append((q, k, v, a, x, w))
    run = lambda q, k, v, a, x, w: m.Fused.linear_attention(q, k, v, a) + m.Fused.linear_attention_grad(v, q, k, v, a) + [m.Fused.matmul_q8(*x, *w)]  # noqa: E731
    wants = [[z.to_numpy() for z in run(*s)] for s in sets]
    m.synchronize()
    streams = [C.c_void_p(L.cumo_hip_stream_create()) for _ in range(2)]
    try:
        for _ in range(5):
            got = []
            for s, given in zip(streams, sets):
                L.cumo_hip_set_stream(s)
                got.append([run(*given) for _ in range(3)][-1])
            for s, zs, want in zip(streams, got, wants):
                L.cumo_hip_set_stream(s)
                assert all((z.to_numpy() == w).all() for z, w in zip(zs, want))
            del got
    finally:
        L.cumo_hip_set_stream(None)
        for s in streams:
            L.cumo_hip_stream_destroy(s)


# (under a name of its own: the next test takes this one)
test_two_streams_with_results_from_the_pool = test_two_streams_at_once


def test_two_streams_at_once():
    """Calls with scratch (inner cut into parts, a sequence into segments, gradients of shared heads) on two streams in turn, with no wait between
    them: each answers what it does by itself."""
    import cumo_amd as m
    from cumo_amd import _lib
    L = _lib.lib
    ref = lambda z: C.byref(z._desc())  # noqa: E731
    sides = []
    for seed in (1, 2):
        rng = np.random.default_rng(seed)
        draw = lambda *n: m.SFloat.cast(rng.standard_normal(n).astype(np.float32))  # noqa: E731
        x, xs = m.Fused.quantize(draw(100, 4096))
        w, ws = m.Fused.quantize(draw(300, 4096))
        q, k, v, g = draw(1, 3000, 4, 24), draw(1, 3000, 2, 24), draw(1, 3000, 2, 20), draw(1, 3000, 4, 20)
        a = m.SFloat.cast(np.linspace(0.8, 0.999, 4).astype(np.float32))
        want = [m.Fused.matmul_q8(x, xs, w, ws)] + m.Fused.linear_attention(q, k, v, a) + m.Fused.linear_attention_grad(g, q, k, v, a)
        sides.append(([ref(z) for z in (x, xs, w, ws)], [ref(z) for z in (q, k, v, a)], ref(g), [z.to_numpy() for z in want], [m.SFloat(*z.shape) for z in want],
                      (x, xs, w, ws, q, k, v, a, g)))
    streams = [C.c_void_p(L.cumo_hip_stream_create()) for _ in range(2)]
    m.synchronize()
    try:
        for _ in range(5):
            for stream, (rows, heads, g, _, results, _) in zip(streams, sides):
                L.cumo_hip_set_stream(stream)
                z = [ref(y) for y in results]
                _lib.call(L.cumo_hip_na_matmul_q8, *rows, None, z[0])
                _lib.call(L.cumo_hip_na_linear_attention, *heads, None, None, 24 ** -0.5, z[1], z[2])
                _lib.call(L.cumo_hip_na_linear_attention_grad, g, *heads, None, None, None, 24 ** -0.5, z[3], z[4], z[5], None)
        L.cumo_hip_set_stream(None)
        m.synchronize()
        for _, _, _, want, results, _ in sides:
            assert all((z.to_numpy() == y).all() for z, y in zip(results, want))
    finally:
        L.cumo_hip_set_stream(None)
        for stream in streams:
            L.cumo_hip_stream_destroy(stream)

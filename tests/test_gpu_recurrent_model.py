"""The row operators and the recurrence as a program uses them together: a small language model whose layers are
normalisation, gates, recurrence and a product, trained and then sampled. Matrix products are mulsum over broadcast views, as
this library has them. Compared with the same program in 64-bit numpy; what it checks is results and gradients, not how
well the model learns."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

B, T, D, V = 3, 17, 12, 40
EPS = 1e-5


def weights(rng):
    w = {"embed": rng.standard_normal((V, D)), "norm": 1 + 0.1 * rng.standard_normal(D), "gate": 0.5 * rng.standard_normal((D, D)),
         "into": rng.standard_normal((D, D)) / 3, "last": 1 + 0.1 * rng.standard_normal(D), "out": rng.standard_normal((V, D)) / 3}
    return {k: v.astype(np.float64) for k, v in w.items()}


class Host:
    """The program in numpy, one step after the other; gradients by differences."""

    def logits(self, w, tokens, state=None):
        x = w["embed"][tokens]
        norm = lambda v, g: v / np.sqrt((v * v).mean(-1, keepdims=True) + EPS) * g  # noqa: E731
        y = norm(x, w["norm"])
        a = 1 / (1 + np.exp(-(y @ w["gate"].T) - 1))
        b = (1 - a) * (y @ w["into"].T)
        h = np.empty_like(a)
        state = np.zeros((x.shape[0], D)) if state is None else state
        for t in range(x.shape[1]):
            state = a[:, t] * state + b[:, t]
            h[:, t] = state
        return norm(h + x, w["last"]) @ w["out"].T, state


def product(m, x, w):
    """x [..., D] by the rows of w [N, D]."""
    rows = int(np.prod(x.shape[:-1]))
    flat = x.reshape(rows, 1, x.shape[-1])
    return flat.mulsum(w.reshape(1, *w.shape), axis=-1).reshape(*x.shape[:-1], w.shape[0])


def forward(m, w, x, state=None):
    """Embedded tokens to logits; what the backward pass needs beside them."""
    y = m.Fused.rmsnorm(x, w["norm"], eps=EPS)
    a = 1 / (m.NMath.exp(-(product(m, y, w["gate"]) + 1)) + 1)
    p = product(m, y, w["into"])
    b = (1 - a) * p
    h = m.Fused.recurrence(a, b, state, axis=1)
    z, s = m.Fused.rmsnorm(h, w["last"], x, EPS)
    return product(m, z, w["out"]), dict(x=x, y=y, a=a, p=p, h=h, z=z, s=s)


def backward(m, w, k, g):
    """Gradients of sum(g * logits) for the two norms' weights and the embedded tokens."""
    gz = product(m, g, w["out"].transpose())
    gh, g_last = m.Fused.rmsnorm_grad(gz, k["s"], w["last"], eps=EPS)   # of h, and of x by the residual
    ga, gb = m.Fused.recurrence_grad(gh, k["a"], k["h"], axis=1)
    gp = gb * (1 - k["a"])
    gate = (ga - gb * k["p"]) * k["a"] * (1 - k["a"])
    gy = product(m, gate, w["gate"].transpose()) + product(m, gp, w["into"].transpose())
    gx, g_norm = m.Fused.rmsnorm_grad(gy, k["x"], w["norm"], gh, EPS)   # what comes by the residual rides along
    return {"last": g_last, "norm": g_norm, "x": gx}


@pytest.mark.parametrize("dt", [np.float32, np.float64])
def test_a_training_step(dt):
    """Logits within 64 roundings of their size (a few dozen operations deep), gradients against differences in 64 bits."""
    import cumo_amd as m
    cls = m.SFloat if dt == np.float32 else m.DFloat
    rng = np.random.default_rng(1)
    w = weights(rng)
    tokens = rng.integers(0, V, (B, T))
    dw = {k: cls.cast(v.astype(dt)) for k, v in w.items()}
    x = cls.cast(w["embed"][tokens].astype(dt))
    logits, kept = forward(m, dw, x)
    want, _ = Host().logits(w, tokens)
    assert np.abs(logits.to_numpy() - want).max() <= 64 * np.finfo(dt).eps * np.abs(want).max()
    g = rng.standard_normal(want.shape)
    grads = backward(m, dw, kept, cls.cast(g.astype(dt)))
    # differences: h^2 / 6 times a third derivative (1e-10 here) and the loss's rounding (1e-13) over h
    for name in ("last", "norm"):
        for i in (0, 5, D - 1):
            both = []
            for sign in (1, -1):
                moved = {k: v.copy() for k, v in w.items()}
                moved[name][i] += sign * 1e-5
                both.append((Host().logits(moved, tokens)[0] * g).sum())
            size = np.abs(grads[name].to_numpy()).max()
            assert abs(grads[name].to_numpy()[i] - (both[0] - both[1]) / 2e-5) <= (1e-6 + 256 * np.finfo(dt).eps) * max(1.0, size), (name, i)
    # embedded tokens: a token's row gathers the gradients of every place that it stands at
    row = np.zeros((V, D))
    np.add.at(row, tokens, grads["x"].to_numpy().astype(np.float64))
    for token in tokens[0, :3]:
        both = []
        for sign in (1, -1):
            moved = {k: v.copy() for k, v in w.items()}
            moved["embed"][token, 4] += sign * 1e-5
            both.append((Host().logits(moved, tokens)[0] * g).sum())
        assert abs(row[token, 4] - (both[0] - both[1]) / 2e-5) <= (1e-6 + 256 * np.finfo(dt).eps) * np.abs(row).max()


@pytest.mark.parametrize("dt", [np.float32, np.float64])
def test_generation_carries_the_state(dt):
    """A prompt, then tokens one at a time with the state carried along: the logits of the whole sequence at once, and the
    tokens that the definition of sampling gives for them. In 8 bits the last norm is within a step of its scale."""
    import cumo_amd as m
    from test_gpu_sample import chosen
    cls = m.SFloat if dt == np.float32 else m.DFloat
    rng = np.random.default_rng(2)
    w = weights(rng)
    dw = {k: cls.cast(v.astype(dt)) for k, v in w.items()}
    tokens = rng.integers(0, V, (B, 5))
    logits, kept = forward(m, dw, cls.cast(w["embed"][tokens].astype(dt)))
    settings = dict(temperature=0.9, top_k=20, top_p=0.9, min_p=0.01)
    for step in range(6):
        u = rng.random(B).astype(dt)
        last = logits[:, logits.shape[1] - 1]
        token = m.Fused.sample(last, cls.cast(u), **settings).to_numpy()
        assert (token == chosen(last.to_numpy(), u, **settings)).all()
        tokens = np.concatenate([tokens, token[:, None]], axis=1)
        state = kept["h"][:, kept["h"].shape[1] - 1]
        logits, kept = forward(m, dw, cls.cast(w["embed"][token][:, None].astype(dt)), state)
        want, _ = Host().logits(w, tokens)
        assert np.abs(logits.to_numpy()[:, 0] - want[:, -1]).max() <= 64 * np.finfo(dt).eps * np.abs(want).max()
        q, scale, s = m.Fused.rmsnorm_q8(kept["h"], dw["last"], kept["x"], EPS)
        assert (s.to_numpy() == kept["s"].to_numpy()).all()
        z = kept["z"].to_numpy()
        assert (np.abs(m.Fused.dequantize(q, scale).to_numpy() - z) <= (0.5 + 1e-4) * scale.to_numpy()).all()


def test_a_generation_step_captured_and_replayed():
    """Norm, recurrence, norm and sample of one token in a graph: the state is updated in place from replay to replay."""
    import cumo_amd as m
    from cumo_amd import _lib
    from test_gpu_index import hip_runtime
    hip, L = hip_runtime(), _lib.lib
    rng = np.random.default_rng(3)
    rows, d, v = 4, 64, 640
    x, a, b = (m.SFloat.cast(rng.uniform(0.1, 0.9, (rows, 1, d)).astype(np.float32)) for _ in range(3))
    w, u, logits = m.SFloat.cast(rng.standard_normal(d).astype(np.float32)), m.SFloat.cast(rng.random(rows).astype(np.float32)), m.SFloat.cast(rng.standard_normal((rows, v)).astype(np.float32))
    state = m.SFloat.cast(np.zeros((rows, d), np.float32))
    h, y, s, token = m.SFloat(rows, 1, d), m.SFloat(rows, 1, d), m.SFloat(rows, 1, d), m.Int32(rows)
    ref = lambda z: C.byref(z._desc())  # noqa: E731
    view = state.reshape(rows, 1, d)
    args = [ref(z) for z in (a, b, state, h, view, w, x, y, s, logits, u, token)]
    ra, rb, rstate, rh, rview, rw, rx, ry, rs, rl, ru, rt = args

    def call():
        _lib.call(L.cumo_hip_na_recurrence, ra, rb, rstate, 1, rh)
        _lib.call(L.cumo_hip_na_store, rview, rh)
        _lib.call(L.cumo_hip_na_rmsnorm, rh, rw, rx, 1e-6, ry, rs)
        _lib.call(L.cumo_hip_na_sample, rl, ru, 0.7, None, 30, None, 0.9, None, 0.0, None, rt)

    ha, hb = a.to_numpy()[:, 0].astype(np.float64), b.to_numpy()[:, 0].astype(np.float64)
    want_token = m.Fused.sample(logits, u, 0.7, 30, 0.9).to_numpy()
    stream = C.c_void_p(L.cumo_hip_stream_create())
    graph, ready = C.c_void_p(), C.c_void_p()
    m.synchronize()
    L.cumo_hip_set_stream(stream)
    try:
        assert hip.hipStreamBeginCapture(stream, 2) == 0
        call()
        assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert hip.hipGraphInstantiate(C.byref(ready), graph, None, None, C.c_size_t(0)) == 0
        want = np.zeros((rows, d))
        for _ in range(4):
            dirt = [m.SFloat(k).fill(float("nan")) for k in (64, 3000, 100000)]
            token.fill(-7)
            assert hip.hipGraphLaunch(ready, stream) == 0
            m.synchronize()
            want = ha * want + hb
            assert np.abs(state.to_numpy() - want).max() <= 1e-6 and (token.to_numpy() == want_token).all()
            both = m.Fused.rmsnorm(h, w, x, 1e-6)
            assert (both[0].to_numpy() == y.to_numpy()).all() and (both[1].to_numpy() == s.to_numpy()).all()
            del dirt
    finally:
        L.cumo_hip_set_stream(None)
        if ready:
            hip.hipGraphExecDestroy(ready)
        if graph:
            hip.hipGraphDestroy(graph)
        L.cumo_hip_stream_destroy(stream)


@pytest.mark.parametrize("dt", [np.float32, np.float64])
def test_results_side_by_side_in_one_array(dt):
    """Two results as the left and the right half of rows, as their even and odd elements, as every other row, row by row in
    turn backwards: what calls answer by themselves, and nothing beside them changes."""
    import cumo_amd as m
    from cumo_amd import _lib
    L = _lib.lib
    cls = m.SFloat if dt == np.float32 else m.DFloat
    rng = np.random.default_rng(5)
    rows, d = 37, 21
    x, r, g, a = (cls.cast(rng.uniform(0.1, 0.9, (rows, d)).astype(dt)) for _ in range(4))
    y, s = m.Fused.rmsnorm(x, None, r)
    ga, gb = m.Fused.recurrence_grad(g, a, x, axis=0)
    ref = lambda z: C.byref(z._desc())  # noqa: E731
    every = slice(None)
    for wide, one, two in (((rows, 2 * d), (every, slice(0, d)), (every, slice(d, 2 * d))), ((rows, 2 * d + 1), (every, slice(0, 2 * d, 2)), (every, slice(1, 2 * d + 1, 2))),
                           ((rows, 2 * d + 6), (every, slice(d + 5, 5, -1)), (every, slice(d + 6, 2 * d + 6))), ((2 * rows, d), (slice(0, None, 2), every), (slice(1, None, 2), every)),
                           ((2 * rows, d + 3), (slice(None, None, -2), slice(0, d)), (slice(0, None, 2), slice(2, d + 2)))):
        for call, want in ((lambda p, q: (L.cumo_hip_na_rmsnorm, ref(x), None, ref(r), 1e-6, ref(p), ref(q)), (y, s)),
                           (lambda p, q: (L.cumo_hip_na_recurrence_grad, ref(g), ref(a), ref(x), None, 0, ref(p), ref(q), None), (ga, gb))):
            for order in (1, -1):
                buf = cls(*wide).fill(7)
                both = (buf[one], buf[two])[::order]
                _lib.call(*call(*both))
                got = buf.to_numpy()
                for at, w in zip((one, two)[::order], want):
                    assert (got[at] == w.to_numpy()).all(), (wide, one, two)
                    got[at] = 7
                assert (got == 7).all()


def test_what_captures_leave_to_their_graphs_can_be_given_back():
    """Captured calls with scratch and with copies of operands: in use until it is given back, a capture's at a time, and the pool
    is then as it was; the other capture's graph still runs."""
    import cumo_amd as m
    from cumo_amd import _lib
    from test_gpu_index import hip_runtime
    hip, L = hip_runtime(), _lib.lib
    rng = np.random.default_rng(6)
    draw = lambda *shape: m.SFloat.cast(rng.uniform(0.1, 0.9, shape).astype(np.float32))  # noqa: E731
    a, b, wide, w, u = draw(1, 3000, 8), draw(1, 3000, 8), draw(700, 520), draw(260), draw(700)
    x = wide[:, ::2]   # (rows whose elements are not neighbours are copied)
    h, gx, gw, token = m.SFloat(1, 3000, 8), m.SFloat(700, 260), m.SFloat(260), m.Int32(700)
    ref = lambda z: C.byref(z._desc())  # noqa: E731
    args = [ref(z) for z in (a, b, h, x, w, gx, gw, u, token)]

    def call():
        ra, rb, rh, rx, rw, rgx, rgw, ru, rt = args
        _lib.call(L.cumo_hip_na_recurrence, ra, rb, None, 1, rh)
        _lib.call(L.cumo_hip_na_rmsnorm_grad, rx, rx, rw, None, 1e-6, rgx, rgw)
        _lib.call(L.cumo_hip_na_sample, rx, ru, 1.0, None, 30, None, 0.9, None, 0.0, None, rt)

    results = (h, gx, gw, token)
    call()
    wants = [z.to_numpy() for z in results]
    assert m.MemoryPool.capture_id() == 0
    start, used = m.MemoryPool.captured_blocks(), m.MemoryPool.used_bytes()
    stream = C.c_void_p(L.cumo_hip_stream_create())
    m.synchronize()
    L.cumo_hip_set_stream(stream)
    made = []
    try:
        for _ in range(2):
            graph, ready = C.c_void_p(), C.c_void_p()
            assert hip.hipStreamBeginCapture(stream, 2) == 0
            capture = m.MemoryPool.capture_id()
            call()
            assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
            assert hip.hipGraphInstantiate(C.byref(ready), graph, None, None, C.c_size_t(0)) == 0
            made.append((capture, graph, ready))
            # recurrence's words, two copies and the parts of the gradient, a copy and the bins
            assert m.MemoryPool.captured_blocks(capture) == 6
        assert made[0][0] and made[1][0] and made[0][0] != made[1][0] and m.MemoryPool.captured_blocks() == start + 12
        for k in range(2):
            for _, _, ready in made[k:]:
                for z in results:
                    z.fill(0)
                held = [m.Int32((512 << s) // 4).fill(77) for s in range(15) for _ in range(2)]
                assert hip.hipGraphLaunch(ready, stream) == 0
                m.synchronize()
                assert all((z.to_numpy() == want).all() for z, want in zip(results, wants))
                assert all(int(v.ne(77).count_true()) == 0 for v in held)
                del held
            capture, graph, ready = made[k]
            assert hip.hipGraphExecDestroy(ready) == 0 and hip.hipGraphDestroy(graph) == 0
            assert m.MemoryPool.free_captured(capture) == 6 and m.MemoryPool.captured_blocks(capture) == 0
        assert m.MemoryPool.captured_blocks() == start and m.MemoryPool.used_bytes() == used
    finally:
        L.cumo_hip_set_stream(None)
        L.cumo_hip_stream_destroy(stream)

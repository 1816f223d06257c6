"""Linear attention with a decay for each head and its gradients, against the definition step by step in more bits.

Tolerances: an output is a sum of products. Whatever the order, each term passes at most 2 roundings a step (a decay and an addition
to the state), dim additions of the dot product and a few dozen products (powers of the decay, scales), so it is off by at most
(2 time + dim + wide + 64) half steps of the type (eps / 2), of the sum of the terms' magnitudes, which the reference works out beside the
values. The heads that share k and v add up in their order: a few roundings more."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = [np.float32, np.float64]
# batch, time, heads, shared heads, dim, wide: one step, a few, stretches of 16 and their ends, odd heads, the widest ones, long sequences
SHAPES = [(1, 1, 1, 1, 1, 1), (2, 1, 3, 3, 16, 16), (3, 1, 4, 2, 128, 128), (2, 1, 2, 1, 100, 72), (1, 1, 1, 1, 256, 250), (3, 2, 2, 1, 5, 7), (2, 3, 2, 2, 64, 36), (2, 15, 2, 2, 16, 16),
          (1, 16, 4, 2, 32, 64), (2, 17, 2, 2, 33, 20), (1, 31, 2, 2, 48, 17), (1, 33, 2, 2, 64, 128), (2, 100, 3, 1, 72, 100), (1, 257, 2, 2, 128, 128), (1, 130, 2, 1, 256, 256),
          (2, 64, 1, 1, 16, 256), (1, 300, 1, 1, 256, 16), (1, 47, 1, 1, 255, 1), (1, 47, 1, 1, 1, 255), (1, 2000, 1, 1, 8, 8), (1, 3001, 2, 2, 24, 40), (40, 70, 8, 8, 20, 30),
          (70, 40, 4, 4, 256, 16), (70, 40, 4, 2, 150, 20), (70, 40, 4, 4, 128, 20), (1, 1500, 2, 1, 128, 80), (1, 700, 1, 1, 256, 40), (1, 1111, 2, 2, 80, 12)]


def cls_of(m, dt):
    return m.SFloat if dt == np.float32 else m.DFloat


def made(rng, shape, dt, decay=None):
    b, t, h, s, d, e = shape
    draw = lambda *n: rng.standard_normal(n).astype(dt)  # noqa: E731
    x = {"q": draw(b, t, h, d), "k": draw(b, t, s, d), "v": draw(b, t, s, e), "state": 2 * draw(b, h, d, e), "g": draw(b, t, h, e), "glast": draw(b, h, d, e)}
    x["decay"] = (1 - 2.0 ** (-1 - 8 * rng.random(h))).astype(dt) if decay is None else np.resize(np.array(decay, dt), h)
    return x


def more(dt):
    return np.float64 if dt == np.float32 else np.longdouble


def reference(x, lengths=None, scale=None, state=True):
    """o, last and what their terms' magnitudes add up to."""
    wide = more(x["q"].dtype)
    b, t, h, d = x["q"].shape
    group = h // x["k"].shape[2]
    q = x["q"].astype(wide)
    k, v = (np.repeat(x[n].astype(wide), group, axis=2) for n in ("k", "v"))
    a = x["decay"].astype(wide)[:, None, None]
    scale = wide(d) ** wide(-0.5) if scale is None else wide(scale)
    lengths = np.full(b, t) if lengths is None else np.clip(lengths, 0, t)
    s = x["state"].astype(wide) if state else np.zeros((b, h, d, v.shape[-1]), wide)
    m = np.abs(s)
    o, om = np.zeros((b, t, h, v.shape[-1]), wide), np.zeros((b, t, h, v.shape[-1]), wide)
    for n in range(t):
        on = np.flatnonzero(n < lengths)
        s[on] = a * s[on] + k[on, n, :, :, None] * v[on, n, :, None, :]
        m[on] = np.abs(a) * m[on] + np.abs(k[on, n, :, :, None] * v[on, n, :, None, :])
        o[on, n] = scale * (q[on, n, :, :, None] * s[on]).sum(-2)
        om[on, n] = np.abs(scale) * (np.abs(q[on, n, :, :, None]) * m[on]).sum(-2)
    return (o, s), (om, m)


def reference_grad(x, lengths=None, scale=None, state=True, glast=True):
    """gq, gk, gv, gstate by the definition, and the magnitudes."""
    wide = more(x["q"].dtype)
    b, t, h, d = x["q"].shape
    shared = x["k"].shape[2]
    group = h // shared
    q, g = x["q"].astype(wide), x["g"].astype(wide)
    k, v = (np.repeat(x[n].astype(wide), group, axis=2) for n in ("k", "v"))
    e = v.shape[-1]
    a = x["decay"].astype(wide)[:, None, None]
    scale = wide(d) ** wide(-0.5) if scale is None else wide(scale)
    lengths = np.full(b, t) if lengths is None else np.clip(lengths, 0, t)
    out, size = [], []
    for f in (lambda z: z, np.abs):
        aa, sc = f(a), f(scale)
        s = f(x["state"].astype(wide)) if state else np.zeros((b, h, d, e), wide)
        gq, gk, gv = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
        for n in range(t):
            on = np.flatnonzero(n < lengths)
            s[on] = aa * s[on] + f(k[on, n, :, :, None] * v[on, n, :, None, :])
            gq[on, n] = sc * (s[on] * f(g[on, n, :, None, :])).sum(-1)
        behind = f(x["glast"].astype(wide)) if glast else np.zeros((b, h, d, e), wide)
        for n in range(t - 1, -1, -1):
            on = np.flatnonzero(n < lengths)
            here = behind[on] + sc * f(q[on, n, :, :, None] * g[on, n, :, None, :])
            gk[on, n] = (here * f(v[on, n, :, None, :])).sum(-1)
            gv[on, n] = (here * f(k[on, n, :, :, None])).sum(-2)
            behind[on] = aa * here
        each = lambda z: z.reshape(b, t, shared, group, -1).sum(3)  # noqa: E731
        (size if out else out).extend([gq, each(gk), each(gv), behind])
    return out, size


def close(got, want, size, shape, what=""):
    dt = got.dtype
    tol = (2 * shape[1] + shape[4] + shape[5] + shape[2] // shape[3] + 64) * np.finfo(dt).eps / 2
    assert got.shape == want.shape
    bad = ~(np.abs(got - want) <= tol * size + np.finfo(dt).tiny)
    assert not bad.any(), "%s: %r of %d, first at %r: got %r want %r" % (what, bad.sum(), bad.size, np.argwhere(bad)[0], got[bad][0], want[bad][0])


def on_device(m, x, names):
    cls = cls_of(m, x["q"].dtype)
    return [cls.cast(x[n]) for n in names]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_the_definition(dt, shape):
    import cumo_amd as m
    x = made(np.random.default_rng(sum(shape)), shape, dt)
    q, k, v, a, s = on_device(m, x, ("q", "k", "v", "decay", "state"))
    for state, scale in ((s, None), (None, 0.7)):
        (o, last), (om, lm) = reference(x, scale=scale, state=state is not None)
        got = m.Fused.linear_attention(q, k, v, a, state, scale=scale)
        assert [type(z) for z in got] == [type(q)] * 2
        close(got[0].to_numpy(), o, om, shape, "o")
        close(got[1].to_numpy(), last, lm, shape, "last")


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_gradients_match_the_definition(dt, shape):
    import cumo_amd as m
    x = made(np.random.default_rng(sum(shape) + 1), shape, dt)
    g, q, k, v, a, s, gl = on_device(m, x, ("g", "q", "k", "v", "decay", "state", "glast"))
    for state, glast, scale in ((s, gl, None), (None, None, 1.3)):
        want, size = reference_grad(x, scale=scale, state=state is not None, glast=glast is not None)
        got = m.Fused.linear_attention_grad(g, q, k, v, a, state, glast, scale=scale)
        assert len(got) == (4 if state is not None else 3)
        for n, z in enumerate(got):
            close(z.to_numpy(), want[n], size[n], shape, ("gq", "gk", "gv", "gstate")[n])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", [(5, 1, 2, 1, 20, 30), (6, 40, 4, 2, 33, 48), (5, 150, 2, 2, 64, 64), (4, 4000, 2, 1, 20, 24)])
def test_lengths(dt, shape):
    """Sequences of different lengths, none and more than there are steps among them. What stands behind them may be anything."""
    import cumo_amd as m
    b, t = shape[:2]
    x = made(np.random.default_rng(t), shape, dt)
    lengths = np.resize(np.array([t, 0, t // 2, t + 9, -3, max(t - 1, 1)], np.int32), b)
    held = np.clip(lengths, 0, t)
    dirty = {n: z.copy() for n, z in x.items()}
    for n, bad in (("q", np.nan), ("k", np.inf), ("v", np.nan), ("g", -np.inf)):
        for row in range(b):
            dirty[n][row, held[row]:] = bad
    dl = m.Int32.cast(lengths)
    g, q, k, v, a, s, gl = on_device(m, dirty, ("g", "q", "k", "v", "decay", "state", "glast"))
    (o, last), (om, lm) = reference(x, lengths)
    got = m.Fused.linear_attention(q, k, v, a, s, dl)
    close(got[0].to_numpy(), o, om, shape, "o")
    close(got[1].to_numpy(), last, lm, shape, "last")
    want, size = reference_grad(x, lengths)
    got = [z.to_numpy() for z in m.Fused.linear_attention_grad(g, q, k, v, a, s, gl, dl)]
    for n, z in enumerate(got):
        close(z, want[n], size[n], shape, ("gq", "gk", "gv", "gstate")[n])
    for row in range(b):
        assert all((z[row, held[row]:] == 0).all() for z in got[:3])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", [(1, 50, 5, 5, 20, 36), (1, 1500, 5, 5, 16, 16), (2, 1, 5, 5, 16, 16)])
def test_decays_of_every_kind(dt, shape):
    """None, all, a change of sign, a growing state: the powers are products, not exponentials of logarithms."""
    import cumo_amd as m
    x = made(np.random.default_rng(3), shape, dt, decay=[0.0, 1.0, -0.75, 1.002, 0.5])
    g, q, k, v, a, s, gl = on_device(m, x, ("g", "q", "k", "v", "decay", "state", "glast"))
    (o, last), (om, lm) = reference(x)
    got = m.Fused.linear_attention(q, k, v, a, s)
    close(got[0].to_numpy(), o, om, shape, "o")
    close(got[1].to_numpy(), last, lm, shape, "last")
    want, size = reference_grad(x)
    for n, z in enumerate(m.Fused.linear_attention_grad(g, q, k, v, a, s, gl)):
        close(z.to_numpy(), want[n], size[n], shape, ("gq", "gk", "gv", "gstate")[n])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("at", [0, 5, 15, 16, 37, 700])
def test_a_step_reaches_no_step_before_it(dt, where, bad, at):
    import cumo_amd as m
    shape = (2, 720, 2, 1, 20, 36)
    x = made(np.random.default_rng(at), shape, dt)
    (o, _), (om, _) = reference(x)
    x[where][1, at, 0, 3] = bad
    q, k, v, a, s = on_device(m, x, ("q", "k", "v", "decay", "state"))
    got, last = (z.to_numpy() for z in m.Fused.linear_attention(q, k, v, a, s))
    part = (2, at, 2, 1, 20, 36)
    close(got[1, :at], o[1, :at], om[1, :at], part)
    close(got[0], o[0], om[0], shape)
    reached = got[1, at:] if where == "k" else got[1, at:, :, 3]
    assert not np.isfinite(reached).any() and not np.isfinite(last[1] if where == "v" else last[1, :, 3]).all()
    if where == "v":
        keep = [n for n in range(36) if n != 3]
        close(got[1][:, :, keep], o[1][:, :, keep], om[1][:, :, keep], shape)


@pytest.mark.parametrize("dt", TYPES)
def test_gradients_reach_no_step_behind(dt):
    """A g that is no number: gq of other steps, gk and gv of later ones are as they were."""
    import cumo_amd as m
    shape, at = (1, 70, 2, 1, 20, 36), 37
    x = made(np.random.default_rng(9), shape, dt)
    want, size = reference_grad(x)
    x["g"][0, at, 1, 3] = np.nan
    got = [z.to_numpy() for z in m.Fused.linear_attention_grad(*on_device(m, x, ("g", "q", "k", "v", "decay", "state", "glast")))]
    others = [n for n in range(shape[1]) if n != at]
    close(got[0][:, others], want[0][:, others], size[0][:, others], shape, "gq")
    assert np.isnan(got[0][0, at, 1]).all()
    for n in (1, 2):
        close(got[n][:, at + 1:], want[n][:, at + 1:], size[n][:, at + 1:], shape, "gk gv")
        assert np.isnan(got[n][0, :at + 1]).any()


@pytest.mark.parametrize("dt", TYPES)
def test_a_prompt_in_pieces(dt):
    """The state handed on: pieces of every length, single tokens among them, answer what the whole does."""
    import cumo_amd as m
    shape = (2, 130, 4, 2, 40, 24)
    x = made(np.random.default_rng(4), shape, dt)
    (o, last), (om, lm) = reference(x)
    q, k, v, a, s = on_device(m, x, ("q", "k", "v", "decay", "state"))
    out, at = [], 0
    for n in (1, 1, 2, 16, 17, 3, 64, 1, 25):
        part = slice(at, at + n)
        y, s = m.Fused.linear_attention(q[:, part], k[:, part], v[:, part], a, s)
        out.append(y.to_numpy())
        at += n
    assert at == shape[1]
    close(np.concatenate(out, axis=1), o, om, shape, "o")
    close(s.to_numpy(), last, lm, shape, "last")


def layouts(m, cls, x):
    """The same numbers as they may lie: heads in front, side by side in one array, backwards, every other element."""
    b, t, h, d = x.shape
    yield cls.cast(np.ascontiguousarray(x.transpose(0, 2, 1, 3))).transpose(0, 2, 1, 3)
    wide = np.zeros((b, t, h, d + 7), x.dtype)
    wide[..., 3:3 + d] = x
    yield cls.cast(wide)[:, :, :, 3:3 + d]
    yield cls.cast(np.ascontiguousarray(x[::-1, ::-1, ::-1]))[::-1, ::-1, ::-1]
    every = np.zeros((b, t, h, 2 * d), x.dtype)
    every[..., ::2] = x
    yield cls.cast(every)[:, :, :, ::2]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", [(3, 1, 4, 2, 24, 20), (3, 37, 4, 2, 24, 20)])
def test_layouts(dt, shape):
    import cumo_amd as m
    cls = cls_of(m, dt)
    x = made(np.random.default_rng(5), shape, dt)
    plain = on_device(m, x, ("q", "k", "v", "decay", "state"))
    want = [z.to_numpy() for z in m.Fused.linear_attention(*plain)]
    g, gl = on_device(m, x, ("g", "glast"))
    want_grad = [z.to_numpy() for z in m.Fused.linear_attention_grad(g, *plain, gl)]
    for q, k, v, gg in zip(*(layouts(m, cls, x[n]) for n in ("q", "k", "v", "g"))):
        for w, z in zip(want, m.Fused.linear_attention(q, k, v, *plain[3:])):
            assert (z.to_numpy() == w).all()
        for w, z in zip(want_grad, m.Fused.linear_attention_grad(gg, q, k, v, *plain[3:], gl)):
            assert (z.to_numpy() == w).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("time", [1, 37])
def test_results_in_given_arrays(dt, time):
    """Results as windows, on top of operands, heads in front; nothing beside them changes."""
    import cumo_amd as m
    from cumo_amd import _lib
    L, cls = _lib.lib, cls_of(m, dt)
    ref = lambda z: C.byref(z._desc())  # noqa: E731
    shape = (2, time, 4, 4, 24, 24)
    x = made(np.random.default_rng(6), shape, dt)
    arrays = on_device(m, x, ("q", "k", "v", "decay", "state"))
    q, k, v, a, s = arrays
    want, last = (z.to_numpy() for z in m.Fused.linear_attention(*arrays))
    buf = cls(2, 4, time, 30).fill(7)
    o = buf[:, :, :, 4:28].transpose(0, 2, 1, 3)
    _lib.call(L.cumo_hip_na_linear_attention, ref(q), ref(k), ref(v), ref(a), ref(s), None, 24 ** -0.5, ref(o), None)
    assert (o.to_numpy() == want).all()
    got = buf.to_numpy()
    got[:, :, :, 4:28] = 7
    assert (got == 7).all()
    # o over q, the state over itself (a single step's where it is: nothing is held for it)
    _lib.call(L.cumo_hip_na_linear_attention, ref(q), ref(k), ref(v), ref(a), ref(s), None, 24 ** -0.5, ref(q), ref(s))
    assert (q.to_numpy() == want).all() and (s.to_numpy() == last).all()
    # the state of two of its sequences in the middle of a wider array, in place
    x = made(np.random.default_rng(7), shape, dt)
    wide = np.concatenate([x["state"], 5 * np.ones_like(x["state"])], axis=0)
    q, k, v, a = on_device(m, x, ("q", "k", "v", "decay"))
    held = cls.cast(wide)
    want, last = (z.to_numpy() for z in m.Fused.linear_attention(q, k, v, a, cls.cast(x["state"])))
    o = cls(2, time, 4, 24)
    _lib.call(L.cumo_hip_na_linear_attention, ref(q), ref(k), ref(v), ref(a), ref(held[0:2]), None, 24 ** -0.5, ref(o), ref(held[0:2]))
    assert (o.to_numpy() == want).all() and (held.to_numpy()[:2] == last).all() and (held.to_numpy()[2:] == 5).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("apart", [(1 << 26) - 256, 1 << 26, (1 << 26) + 256])
def test_steps_far_apart(dt, apart):
    """Rows in one array, as far apart as a stretch's offsets reach and further; the last is more than 2^32 bytes from the first."""
    import cumo_amd as m
    cls, shape = cls_of(m, dt), (1, 70, 2, 1, 16, 16)
    x = made(np.random.default_rng(apart), shape, dt)
    q, k, v, a, s = on_device(m, x, ("q", "k", "v", "decay", "state"))
    g, gl = on_device(m, x, ("g", "glast"))
    want = [z.to_numpy() for z in m.Fused.linear_attention(q, k, v, a, s) + m.Fused.linear_attention_grad(g, q, k, v, a, s, gl)]
    buf = cls(1, 70, apart // (16 * np.dtype(dt).itemsize), 16)
    parts = [buf[:, :, 0:2], buf[:, :, 2:3], buf[:, :, 3:4], buf[:, :, 4:6]]
    for part, z in zip(parts, (q, k, v, g)):
        part.store(z)
    q, k, v, g = parts
    got = [z.to_numpy() for z in m.Fused.linear_attention(q, k, v, a, s) + m.Fused.linear_attention_grad(g, q, k, v, a, s, gl)]
    (o, last), (om, lm) = reference(x)
    close(got[0], o, om, shape, "o")
    close(got[1], last, lm, shape, "last")
    grads, size = reference_grad(x)
    for n in range(4):
        close(got[2 + n], grads[n], size[n], shape, ("gq", "gk", "gv", "gstate")[n])
    # (the same way of working, or one step at a time)
    if apart <= 1 << 26:
        assert all((z == w).all() for z, w in zip(got, want))


@pytest.mark.parametrize("dt", TYPES)
def test_nothing_to_do(dt):
    import cumo_amd as m
    cls = cls_of(m, dt)
    make = lambda *n: cls(*n)  # noqa: E731
    s = cls.cast(np.arange(24, dtype=dt).reshape(1, 2, 3, 4))
    o, last = m.Fused.linear_attention(make(1, 0, 2, 3), make(1, 0, 2, 3), make(1, 0, 2, 4), cls.cast(np.ones(2, dt)), s)
    assert o.shape == (1, 0, 2, 4) and (last.to_numpy() == s.to_numpy()).all()
    o, last = m.Fused.linear_attention(make(1, 0, 2, 3), make(1, 0, 2, 3), make(1, 0, 2, 4), cls.cast(np.ones(2, dt)))
    assert (last.to_numpy() == 0).all()
    gq, gk, gv, gs = m.Fused.linear_attention_grad(make(1, 0, 2, 4), make(1, 0, 2, 3), make(1, 0, 2, 3), make(1, 0, 2, 4), cls.cast(np.ones(2, dt)), s, s)
    assert gq.shape == (1, 0, 2, 3) and (gs.to_numpy() == s.to_numpy()).all()
    # the same with heads that share k and v
    s4 = cls.cast(np.arange(48, dtype=dt).reshape(1, 4, 3, 4))
    gq, gk, gv, gs = m.Fused.linear_attention_grad(make(1, 0, 4, 4), make(1, 0, 4, 3), make(1, 0, 2, 3), make(1, 0, 2, 4), cls.cast(np.ones(4, dt)), s4, s4)
    assert gk.shape == (1, 0, 2, 3) and (gs.to_numpy() == s4.to_numpy()).all()
    gq, gk, gv = m.Fused.linear_attention_grad(make(1, 3, 4, 0), make(1, 3, 4, 0), make(1, 3, 2, 0), make(1, 3, 2, 0), cls.cast(np.ones(4, dt)))
    assert gq.shape == (1, 3, 4, 0) and gk.shape == gv.shape == (1, 3, 2, 0)
    for shape in ((0, 5, 2, 3), (2, 5, 0, 3)):
        q, a = make(*shape), make(shape[2])
        o, last = m.Fused.linear_attention(q, q, q, a)
        assert o.shape == shape and last.shape == (shape[0], shape[2], 3, 3)
    # no elements of k: nothing is seen; none of v: nothing is written
    ones = lambda *n: cls(*n).fill(1)  # noqa: E731
    for time in (1, 40):
        o, last = m.Fused.linear_attention(make(1, time, 2, 0), make(1, time, 2, 0), ones(1, time, 2, 4), ones(2))
        assert (o.to_numpy() == 0).all() and last.shape == (1, 2, 0, 4)
        gq, gk, gv = m.Fused.linear_attention_grad(ones(1, time, 2, 4), make(1, time, 2, 0), make(1, time, 2, 0), ones(1, time, 2, 4), ones(2))
        assert (gv.to_numpy() == 0).all() and gq.shape == (1, time, 2, 0)
        o, last = m.Fused.linear_attention(ones(1, time, 2, 4), ones(1, time, 2, 4), make(1, time, 2, 0), ones(2))
        assert o.shape == (1, time, 2, 0)
        gq, gk, gv = m.Fused.linear_attention_grad(make(1, time, 2, 0), ones(1, time, 2, 4), ones(1, time, 2, 4), make(1, time, 2, 0), ones(2))
        assert (gq.to_numpy() == 0).all() and (gk.to_numpy() == 0).all()


def test_gradients_match_differences():
    """d of sum(g o) + sum(glast last) by central differences in double, off by h^2 times a third derivative (the loss is of the third degree in
    all of them together, in one number at a time of the first: none) and by the loss's rounding over h."""
    import cumo_amd as m
    shape = (2, 21, 4, 2, 6, 5)
    x = made(np.random.default_rng(8), shape, np.float64)
    lengths = m.Int32.cast(np.array([21, 13], np.int32))

    def loss(x):
        o, last = m.Fused.linear_attention(*on_device(m, x, ("q", "k", "v", "decay", "state")), lengths)
        return float((o.to_numpy() * x["g"]).sum() + (last.to_numpy() * x["glast"]).sum())

    got = m.Fused.linear_attention_grad(*on_device(m, x, ("g", "q", "k", "v", "decay", "state", "glast")), lengths)
    size = sum(np.abs(z.to_numpy()).max() for z in got)
    for name, z, places in zip(("q", "k", "v", "state"), got, ([(0, 0, 0, 0), (0, 20, 3, 5), (1, 12, 2, 1), (1, 13, 0, 0)], [(0, 0, 1, 3), (0, 17, 0, 0), (1, 5, 1, 2)],
                                                              [(0, 20, 1, 4), (1, 0, 0, 0), (1, 20, 0, 1)], [(0, 0, 0, 0), (1, 3, 5, 4)])):
        for at in places:
            both = []
            for sign in (1, -1):
                moved = {**x, name: x[name].copy()}
                moved[name][at] += sign * 1e-4
                both.append(loss(moved))
            assert abs((both[0] - both[1]) / 2e-4 - z.to_numpy()[at]) <= 1e-8 * size, (name, at)


@pytest.mark.parametrize("time", [1, 50, 3000])
def test_captured_on_another_stream(time):
    """A step, a prompt and a long one, with their gradients, in a graph: every replay answers what the calls by themselves do."""
    import cumo_amd as m
    from cumo_amd import _lib
    from test_gpu_index import hip_runtime
    hip, L = hip_runtime(), _lib.lib
    shape = (2, time, 4, 2, 24, 20)
    x = made(np.random.default_rng(time), shape, np.float32)
    lengths = m.Int32.cast(np.array([time, max(time - 5, 1)], np.int32))
    g, q, k, v, a, s, gl = on_device(m, x, ("g", "q", "k", "v", "decay", "state", "glast"))
    wants = [z.to_numpy() for z in m.Fused.linear_attention(q, k, v, a, s, lengths) + m.Fused.linear_attention_grad(g, q, k, v, a, s, gl, lengths)]
    results = [m.SFloat(*w.shape) for w in wants]
    ref = lambda z: C.byref(z._desc())  # noqa: E731
    rg, rq, rk, rv, ra, rs, rgl, rl = (ref(z) for z in (g, q, k, v, a, s, gl, lengths))
    rr = [ref(z) for z in results]
    stream = C.c_void_p(L.cumo_hip_stream_create())
    graph, ready = C.c_void_p(), C.c_void_p()
    m.synchronize()
    L.cumo_hip_set_stream(stream)
    try:
        assert hip.hipStreamBeginCapture(stream, 2) == 0
        _lib.call(L.cumo_hip_na_linear_attention, rq, rk, rv, ra, rs, rl, 24 ** -0.5, rr[0], rr[1])
        _lib.call(L.cumo_hip_na_linear_attention_grad, rg, rq, rk, rv, ra, rs, rgl, rl, 24 ** -0.5, *rr[2:])
        assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert hip.hipGraphInstantiate(C.byref(ready), graph, None, None, C.c_size_t(0)) == 0
        for _ in range(3):
            dirt = [m.SFloat(n).fill(float("nan")) for n in (64, 3000, 100000)]
            for z in results:
                z.fill(5)
            assert hip.hipGraphLaunch(ready, stream) == 0
            m.synchronize()
            assert all((z.to_numpy() == w).all() for z, w in zip(results, wants))
            again = m.Fused.linear_attention(q, k, v, a, s, lengths)
            assert all((z.to_numpy() == w).all() for z, w in zip(again, wants))
            del dirt
    finally:
        L.cumo_hip_set_stream(None)
        if ready:
            hip.hipGraphExecDestroy(ready)
        if graph:
            hip.hipGraphDestroy(graph)
        L.cumo_hip_stream_destroy(stream)


@pytest.mark.parametrize("time", [3000, 40000])
def test_slow_decays_stay_powers(time):
    """States that forget over hundreds to thousands of steps pass a multiplication and five roundings or so a stretch of sixteen. Those fall on either
    side: a window of 4000 steps, 250 stretches, 1250 roundings, is off by sqrt(1250) half steps in norm, 2.1e-6; three times that is
    allowed. A decay that is off on one side would add up to 250 of its own roundings over the window, and more over longer ones."""
    import cumo_amd as m
    rng = np.random.default_rng(time)
    a = (1 - 10.0 ** -np.linspace(2.0, 3.6, 12)).astype(np.float32)
    shape = (1, time, 12, 12, 16, 16)
    x = made(rng, shape, np.float32)
    x["decay"] = a
    _, last = m.Fused.linear_attention(*on_device(m, x, ("q", "k", "v", "decay", "state")))
    steps = np.arange(time - 1, -1, -1)
    for h in range(12):
        by = a[h].astype(np.float64) ** steps
        want = a[h].astype(np.float64) ** time * x["state"][0, h] + (x["k"][0, :, h].astype(np.float64) * by[:, None]).T @ x["v"][0, :, h].astype(np.float64)
        got = last.to_numpy()[0, h]
        assert np.linalg.norm(got - want) <= 3 * 35 * 2.0 ** -24 * np.linalg.norm(want), (h, np.linalg.norm(got - want) / np.linalg.norm(want))


def test_slow_decays_stay_powers_in_double():
    """The same in double: 188 stretches, 940 roundings, three times sqrt(940) half steps in norm; powers by squares in double alone would be off by seven
    half steps a stretch on one side, over those that a decay of 1 - 10^-3.6 remembers."""
    import cumo_amd as m
    time = 3000
    a = 1 - 10.0 ** -np.linspace(2.0, 3.6, 4)
    x = made(np.random.default_rng(time), (1, time, 4, 4, 16, 16), np.float64)
    x["decay"] = a
    _, last = m.Fused.linear_attention(*on_device(m, x, ("q", "k", "v", "decay", "state")))
    (_, want), _ = reference(x)
    for h in range(4):
        off = np.linalg.norm((last.to_numpy()[0, h] - want[0, h]).astype(float)) / np.linalg.norm(want[0, h].astype(float))
        assert off <= 3 * 31 * 2.0 ** -53, (h, off)

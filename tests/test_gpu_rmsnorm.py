"""Root-mean-square normalisation, its 8-bit form and its gradients, against the formulas in 64 bits and more.

Tolerances: sums are in double and a result is rounded to its type once, so it is within half a step of its type
(eps / 2, relative) and what the double sums lose: at most (n + 16) 2^-53 of the sum of the terms' magnitudes for n
terms."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = [np.float32, np.float64]
U64 = 2.0 ** -53
# rows that are part of a vector, one vector, an odd length; lengths at which the lanes of a row change, more than a block's registers hold
SHAPES = [(1, 1), (3, 2), (5, 3), (2, 4), (7, 7), (33, 8), (70, 31), (9, 64), (64, 65), (4, 128), (1000, 129), (3, 5, 256), (40, 257), (5, 511),
          (6, 1023), (4, 1024), (1, 4096), (3, 4095), (5, 8190), (4, 8192), (2, 8193), (3, 16385), (2, 33001), (1, 70001), (300, 2050)]


def cls_of(m, dt):
    return m.SFloat if dt == np.float32 else m.DFloat


def half_step(dt):
    return np.finfo(dt).eps / 2


def reference(s, w, eps):
    v = s.astype(np.longdouble)
    r = 1 / np.sqrt((v * v).mean(axis=-1, keepdims=True) + np.longdouble(eps))
    return v * r * (1 if w is None else w.astype(np.longdouble)), r


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_rmsnorm_matches_the_formula(dt, shape):
    import cumo_amd as m
    cls = cls_of(m, dt)
    rng = np.random.default_rng(shape[-1])
    n = shape[-1]
    x = (rng.standard_normal(shape) * 2 + 0.3).astype(dt)
    res = (rng.standard_normal(shape) * 5).astype(dt)
    w = rng.standard_normal(n).astype(dt)
    tol = half_step(dt) + (n + 16) * U64
    for weight in (None, w):
        dw = None if weight is None else cls.cast(weight)
        want, _ = reference(x, weight, 1e-6)
        got = m.Fused.rmsnorm(cls.cast(x), dw)
        assert type(got) is cls and got.shape == shape
        assert (np.abs(got.to_numpy() - want) <= tol * np.abs(want)).all()
        s = x + res
        want, _ = reference(s, weight, 1e-3)
        y, total = m.Fused.rmsnorm(cls.cast(x), dw, cls.cast(res), 1e-3)
        assert (total.to_numpy() == s).all()
        assert (np.abs(y.to_numpy() - want) <= tol * np.abs(want)).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_rmsnorm_q8_matches_the_formula(dt, shape):
    import cumo_amd as m
    cls = cls_of(m, dt)
    rng = np.random.default_rng(shape[-1] + 1)
    n = shape[-1]
    x = (rng.standard_normal(shape) * 2).astype(dt)
    res = (rng.standard_normal(shape) * 5).astype(dt)
    w = rng.standard_normal(n).astype(dt)
    for weight, residual in ((None, None), (w, res)):
        s = x if residual is None else x + residual
        want, _ = reference(s, weight, 1e-6)
        args = [None if a is None else cls.cast(a) for a in (weight, residual)]
        out = m.Fused.rmsnorm_q8(cls.cast(x), *args)
        q, scale = out[0], out[1]
        assert type(q) is m.Int8 and q.shape == shape and type(scale) is cls and scale.shape == shape[:-1] + (1,)
        if residual is not None:
            assert (out[2].to_numpy() == s).all()
        hq, hs = q.to_numpy().astype(np.longdouble), scale.to_numpy().astype(np.longdouble)
        most = np.abs(want).max(axis=-1, keepdims=True)
        assert (np.abs(hs - most / 127) <= (half_step(dt) + (n + 16) * U64) * most / 127).all()
        # half a step of the integers, and what y and the quotient lost (relative to quotients of up to 127)
        assert (np.abs(hq - want / hs) <= 0.5 + 127 * 4 * (n + 16) * U64).all()
        assert (np.abs(hq).max(axis=-1) == 127).all()
        back = m.Fused.dequantize(q, scale)
        assert type(back) is cls and (back.to_numpy() == q.to_numpy().astype(dt) * scale.to_numpy()).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", SHAPES + [(5000, 3), (2000, 70)])
def test_rmsnorm_grad_matches_the_formula(dt, shape):
    import cumo_amd as m
    cls = cls_of(m, dt)
    rng = np.random.default_rng(shape[-1] + 2)
    n = shape[-1]
    rows = int(np.prod(shape[:-1]))
    s, g, gs = ((rng.standard_normal(shape) * k).astype(dt) for k in (3, 1, 2))
    w = rng.standard_normal(n).astype(dt)
    for weight, gsum in ((None, None), (w, None), (None, gs), (w, gs)):
        ls, lg = s.astype(np.longdouble), g.astype(np.longdouble)
        _, r = reference(s, None, 1e-6)
        gw = lg * (1 if weight is None else weight.astype(np.longdouble))
        c = r * r * (gw * ls).mean(axis=-1, keepdims=True)
        want = r * (gw - ls * c) + (0 if gsum is None else gsum.astype(np.longdouble))
        size = r * (np.abs(gw) + np.abs(ls) * r * r * np.abs(gw * ls).mean(axis=-1, keepdims=True)) + (0 if gsum is None else np.abs(gsum))
        args = [None if a is None else cls.cast(a) for a in (weight, gsum)]
        out = m.Fused.rmsnorm_grad(cls.cast(g), cls.cast(s), *args)
        gx = (out if weight is None else out[0]).to_numpy()
        assert (np.abs(gx - want) <= half_step(dt) * np.abs(want) + 2 * (n + 16) * U64 * size).all()
        if weight is not None:
            terms = lg * ls * r
            want = terms.reshape(rows, n).sum(axis=0)
            size = np.abs(terms).reshape(rows, n).sum(axis=0)
            assert out[1].shape == (n,)
            assert (np.abs(out[1].to_numpy() - want) <= half_step(dt) * np.abs(want) + (rows + n + 16) * U64 * size).all()


def test_rmsnorm_grad_matches_differences():
    """d/dx of sum(g y) + sum(gs s) by central differences in double: off by h^2 times a third derivative (about 1) and
    by the loss's rounding over h."""
    import cumo_amd as m
    rng = np.random.default_rng(5)
    x, res, g, gs = (rng.standard_normal((3, 17)) for _ in range(4))
    w = rng.standard_normal(17)

    def loss(x, w):
        y, s = m.Fused.rmsnorm(m.DFloat.cast(x), m.DFloat.cast(w), m.DFloat.cast(res), 1e-2)
        return float((y.to_numpy() * g).sum() + (s.to_numpy() * gs).sum())

    gx, gw = m.Fused.rmsnorm_grad(*(m.DFloat.cast(a) for a in (g, x + res, w, gs)), 1e-2)
    h = 1e-5
    for k in [(0, 0), (1, 16), (2, 5)]:
        d = np.zeros_like(x)
        d[k] = h
        assert abs((loss(x + d, w) - loss(x - d, w)) / (2 * h) - gx.to_numpy()[k]) < 1e-8
    for k in (0, 16):
        d = np.zeros_like(w)
        d[k] = h
        assert abs((loss(x, w + d) - loss(x, w - d)) / (2 * h) - gw.to_numpy()[k]) < 1e-8


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n", [5, 64, 1500, 9000])
def test_rmsnorm_of_views(dt, n):
    """Windows, every other row, rows backwards, transposed and stepped columns, weights that are views."""
    import cumo_amd as m
    cls = cls_of(m, dt)
    rng = np.random.default_rng(n)
    h, r, g = (rng.standard_normal((6, 2 * n + 3)).astype(dt) for _ in range(3))
    w = rng.standard_normal(3 * n).astype(dt)
    x, res, dg, dw = cls.cast(h), cls.cast(r), cls.cast(g), cls.cast(w)
    keys = [(slice(None), slice(1, n + 1)), (slice(None, None, 2), slice(0, n)), (slice(None, None, -1), slice(2, n + 2)), (slice(None), slice(0, 2 * n, 2)),
            (slice(None), slice(n - 1, None, -1)), (slice(2, 3), slice(3, n + 3)), (slice(0, 0), slice(0, n))]
    for key in keys:
        plain = [a[key].copy() for a in (h, r, g)]
        want = [a.to_numpy() for a in m.Fused.rmsnorm(cls.cast(plain[0]), cls.cast(w[::3].copy()), cls.cast(plain[1]))]
        got = m.Fused.rmsnorm(x[key], dw[::3], res[key])
        assert all((a.to_numpy() == b).all() for a, b in zip(got, want)), key
        want = [a.to_numpy() for a in m.Fused.rmsnorm_q8(cls.cast(plain[0]), cls.cast(w[::3].copy()), cls.cast(plain[1]))]
        got = m.Fused.rmsnorm_q8(x[key], dw[::3], res[key])
        assert all((a.to_numpy() == b).all() for a, b in zip(got, want)), key
        want = [a.to_numpy() for a in m.Fused.rmsnorm_grad(cls.cast(plain[2]), cls.cast(plain[0]), cls.cast(w[::3].copy()), cls.cast(plain[1]))]
        got = m.Fused.rmsnorm_grad(dg[key], x[key], dw[::3], res[key])
        assert all((a.to_numpy() == b).all() for a, b in zip(got, want)), key
    t = np.ascontiguousarray(h[:, :4].T)   # [4, 6] transposed
    got = m.Fused.rmsnorm(cls.cast(t).transpose())
    assert (got.to_numpy() == m.Fused.rmsnorm(cls.cast(t.T.copy())).to_numpy()).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n", [6, 300, 5000, 40000])
def test_rmsnorm_special_rows(dt, n):
    """A row of zeros, a NaN, an infinity, the largest numbers, subnormal ones; the rows beside them stay as they are."""
    import cumo_amd as m
    cls = cls_of(m, dt)
    big, tiny = np.finfo(dt).max, np.finfo(dt).smallest_subnormal
    h = np.random.default_rng(n).standard_normal((7, n)).astype(dt)
    h[1] = 0
    h[2, n // 2] = np.nan
    h[3, n - 1] = np.inf
    h[4] = tiny
    if dt == np.float32:   # (squares of DFloat's largest are beyond double: r is 0 there)
        h[5] = big
    y = m.Fused.rmsnorm(cls.cast(h)).to_numpy()
    assert (y[1] == 0).all() and np.isnan(y[2]).all() and np.isnan(y[3, n - 1]) and (np.delete(y[3], n - 1) == 0).all()
    assert (y[4] >= 0).all() and np.isfinite(y[4]).all()
    if dt == np.float32:
        assert np.abs(y[5] - 1).max() <= 2.0 ** -24
    for k in (0, 6):
        assert (y[k] == m.Fused.rmsnorm(cls.cast(h[k])).to_numpy()).all()
    q, scale = m.Fused.rmsnorm_q8(cls.cast(h))
    q, scale = q.to_numpy(), scale.to_numpy()
    assert scale[1] == 0 and (q[1] == 0).all()
    assert np.isnan(scale[2]) and (q[2] == 0).all()
    assert np.isnan(scale[3]) and (q[3] == 0).all()
    for k in (0, 6):
        one = m.Fused.rmsnorm_q8(cls.cast(h[k]))
        assert (q[k] == one[0].to_numpy()).all() and (scale[k] == one[1].to_numpy()).all()
    g = np.ones_like(h)
    gx, gw = m.Fused.rmsnorm_grad(cls.cast(g[:2]), cls.cast(h[:2]), cls.cast(np.ones(n, dt)), eps=1e-2)
    assert np.abs(gx.to_numpy()[1] - 10).max() <= 10 * (half_step(dt) + 8 * U64)   # r = 1 / sqrt(eps) where s is 0
    # eps 0 and a row of zeros: r is infinite, as the formula says
    assert np.isnan(m.Fused.rmsnorm(cls.cast(h[1:2]), eps=0.0).to_numpy()).all()


@pytest.mark.parametrize("dt", TYPES)
def test_rmsnorm_of_nothing(dt):
    import cumo_amd as m
    cls = cls_of(m, dt)
    for shape in [(0,), (0, 5), (3, 0), (2, 0, 4)]:
        x = cls.cast(np.zeros(shape, dt))
        w = cls.cast(np.ones(shape[-1], dt))
        y, s = m.Fused.rmsnorm(x, w, x)
        assert y.shape == s.shape == shape
        q, scale = m.Fused.rmsnorm_q8(x, w)
        assert q.shape == shape and scale.shape == shape[:-1] + (1,) and (scale.to_numpy() == 0).all()
        assert m.Fused.dequantize(q, scale).shape == shape
        gx, gw = m.Fused.rmsnorm_grad(x, x, w, x)
        assert gx.shape == shape and gw.shape == shape[-1:] and (gw.to_numpy() == 0).all()


def replayed(m, call, results, wants, times=3):
    """Captures `call` and replays it with the program's own work and the pool's memory in use in between."""
    from cumo_amd import _lib
    from test_gpu_index import hip_runtime
    hip = hip_runtime()
    stream = C.c_void_p(_lib.lib.cumo_hip_stream_create())
    graph, ready = C.c_void_p(), C.c_void_p()
    m.synchronize()
    _lib.lib.cumo_hip_set_stream(stream)
    try:
        call()
        assert hip.hipStreamBeginCapture(stream, 2) == 0
        call()
        assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert hip.hipGraphInstantiate(C.byref(ready), graph, None, None, C.c_size_t(0)) == 0
        # (every size of block that the pool could have kept from the capture, a few of each)
        held = [m.Int32((512 << k) // 4).fill(77) for k in range(0, 15) for _ in range(3)]
        for _ in range(times):
            for z in results:
                if type(z) is not m.Int8:
                    z.fill(0)
            assert hip.hipGraphLaunch(ready, stream) == 0
            m.synchronize()
            for z, want in zip(results, wants):
                assert (z.to_numpy() == want).all()
            assert all(int(a.ne(77).count_true()) == 0 for a in held)
        del held
    finally:
        _lib.lib.cumo_hip_set_stream(None)
        if ready:
            hip.hipGraphExecDestroy(ready)
        if graph:
            hip.hipGraphDestroy(graph)
        _lib.lib.cumo_hip_stream_destroy(stream)


@pytest.mark.parametrize("shape", [(1, 4096), (3000, 257), (40, 9000)])
def test_rmsnorm_captured_and_replayed(shape):
    import cumo_amd as m
    from cumo_amd import _lib
    rng = np.random.default_rng(3)
    x, r, g = (m.SFloat.cast(rng.standard_normal(shape).astype(np.float32)) for _ in range(3))
    w = m.SFloat.cast(rng.standard_normal(shape[1]).astype(np.float32))
    y, s = m.Fused.rmsnorm(x, w, r)
    q, scale, s2 = m.Fused.rmsnorm_q8(x, w, r)
    gx, gw = m.Fused.rmsnorm_grad(g, s, w, r)
    results = [y, q, scale, s2, gx, gw]
    wants = [a.to_numpy() for a in results]
    inputs = [a._desc() for a in (x, w, r, g, s)]
    outs = [a._desc() for a in results + [s]]
    dx, dw, dr, dg, ds = (C.byref(d) for d in inputs)
    oy, oq, oscale, os2, ogx, ogw, os = (C.byref(d) for d in outs)

    def call():
        _lib.call(_lib.lib.cumo_hip_na_rmsnorm, dx, dw, dr, 1e-6, oy, os)
        _lib.call(_lib.lib.cumo_hip_na_rmsnorm_q8, dx, dw, dr, 1e-6, oq, oscale, os2)
        _lib.call(_lib.lib.cumo_hip_na_rmsnorm_grad, dg, ds, dw, dr, 1e-6, ogx, ogw)

    replayed(m, call, results, wants)


@pytest.mark.parametrize("dt", TYPES)
def test_rmsnorm_into_given_arrays(dt):
    """Results written over their operands, into windows of larger arrays and across operands; nothing beside them changes."""
    import cumo_amd as m
    from cumo_amd import _lib
    cls = cls_of(m, dt)
    rng = np.random.default_rng(8)
    h, r = (rng.standard_normal((9, 101)).astype(dt) for _ in range(2))
    want, s = (a.to_numpy() for a in m.Fused.rmsnorm(cls.cast(h), None, cls.cast(r)))

    def call(x, res, y, total):
        d = [a._desc() for a in (x, res, y, total)]
        _lib.call(_lib.lib.cumo_hip_na_rmsnorm, C.byref(d[0]), None, C.byref(d[1]), 1e-6, C.byref(d[2]), C.byref(d[3]))

    x, res = cls.cast(h), cls.cast(r)
    call(x, res, x, res)   # element on element
    assert (x.to_numpy() == want).all() and (res.to_numpy() == s).all()
    wide, total = cls(12, 110).fill(5), cls(101, 9).fill(6)
    call(cls.cast(h), cls.cast(r), wide[1:10, 3:104], total.transpose())
    assert (wide[1:10, 3:104].to_numpy() == want).all() and (total.to_numpy() == s.T).all()
    rest = wide.to_numpy()
    rest[1:10, 3:104] = 5
    assert (rest == 5).all()
    # one row further down in the same memory
    buf = cls(10, 101)
    buf[:9].store(cls.cast(h))
    total = cls(9, 101)
    call(buf[:9], cls.cast(r), buf[1:], total)
    assert (buf[1:].to_numpy() == want).all() and (total.to_numpy() == s).all()
    # Int8 rows into a window with steps
    q, scale, _ = (a.to_numpy() for a in m.Fused.rmsnorm_q8(cls.cast(h), None, cls.cast(r)))
    z, zs = m.Int8.cast(np.full((9, 210), 3, np.int8)), cls(9, 1)
    d = [a._desc() for a in (cls.cast(h), cls.cast(r))]
    keep = (cls.cast(h), cls.cast(r))
    d = [a._desc() for a in keep + (z[:, 2:204:2], zs, total)]
    _lib.call(_lib.lib.cumo_hip_na_rmsnorm_q8, C.byref(d[0]), None, C.byref(d[1]), 1e-6, C.byref(d[2]), C.byref(d[3]), C.byref(d[4]))
    got = z.to_numpy()
    assert (got[:, 2:204:2] == q).all() and (zs.to_numpy() == scale).all()
    got[:, 2:204:2] = 3
    assert (got == 3).all()


def test_rmsnorm_on_another_stream_and_recorded():
    import cumo_amd as m
    from cumo_amd import _lib
    rng = np.random.default_rng(9)
    h = rng.standard_normal((200, 1000)).astype(np.float32)
    x, w = m.SFloat.cast(h), m.SFloat.cast(h[0])
    want = m.Fused.rmsnorm(x, w).to_numpy()
    stream = C.c_void_p(_lib.lib.cumo_hip_stream_create())
    m.synchronize()
    _lib.lib.cumo_hip_set_stream(stream)
    try:
        assert (m.Fused.rmsnorm(x, w).to_numpy() == want).all()
    finally:
        _lib.lib.cumo_hip_set_stream(None)
        _lib.lib.cumo_hip_stream_destroy(stream)
    with _lib.record() as calls:
        y, s = m.Fused.rmsnorm(x, w, x)
        g, gw = m.Fused.rmsnorm_grad(y, s, w)
    want = [a.to_numpy() for a in (y, s, g, gw)]
    for a in (y, s, g, gw):
        a.fill(0)
    _lib.replay(calls, 2)
    assert all((a.to_numpy() == b).all() for a, b in zip((y, s, g, gw), want))


def test_int8_arrays_are_copied_viewed_and_read_back():
    import cumo_amd as m
    h = np.random.default_rng(4).integers(-128, 128, (7, 13)).astype(np.int8)
    a = m.Int8.cast(h)
    assert (a.to_numpy() == h).all() and (a[::2, 1::3].copy().to_numpy() == h[::2, 1::3]).all() and (a.transpose().copy().to_numpy() == h.T).all()
    assert (a[[3, 0, 3]].to_numpy() == h[[3, 0, 3]]).all() and a[2, 5].extract_cpu() == h[2, 5]
    assert (a[np.array([3, 0, -1])].to_numpy() == h[[3, 0, -1]]).all()
    assert (a.reshape(91)[4:60].to_numpy() == h.reshape(91)[4:60]).all()
    with pytest.raises(TypeError):
        (m.SFloat.cast(h.astype(np.float32)) > 0).mask(a)


@pytest.mark.parametrize("dt,size", [(np.float32, 1e-43), (np.float32, 1e-39), (np.float32, 1e38), (np.float64, 1e-321), (np.float64, 1e-310), (np.float64, 1e307)])
@pytest.mark.parametrize("n", [5, 700, 4099, 33001])
def test_rmsnorm_q8_of_weights_at_the_ends_of_their_type(dt, size, n):
    """A scale is off by half a step of its type, near 0 of the smallest number's (and a little: largest / 127 is rounded twice
    there); what is above 127 of them is 127."""
    import cumo_amd as m
    cls = cls_of(m, dt)
    rng = np.random.default_rng(n)
    s = (rng.standard_normal((3, n)) * 7).astype(dt)
    w = (np.sign(rng.standard_normal(n)) * rng.uniform(0.3, 1.7, n) * size).astype(dt)
    want, _ = reference(s, w, 1e-6)
    q, scale = (a.to_numpy() for a in m.Fused.rmsnorm_q8(cls.cast(s), cls.cast(w)))
    hs = scale.astype(np.longdouble)
    least = np.longdouble(np.finfo(dt).smallest_subnormal)
    most = np.abs(want).max(axis=-1, keepdims=True)
    assert (np.abs(hs - most / 127) <= 0.51 * least + (half_step(dt) + (n + 16) * U64) * most / 127).all()
    quotient = np.where(hs > 0, want / np.where(hs > 0, hs, 1), 0)
    assert (np.abs(q - np.clip(quotient, -127, 127)) <= 0.5 + 127 * 4 * (n + 16) * U64).all()


def test_gradient_of_a_weight_longer_than_one_launch_of_its_parts():
    import cumo_amd as m
    n = (1 << 26) + 37
    s, g, w = m.SFloat(2, n).fill(1), m.SFloat(2, n).fill(0.5), m.SFloat(n).fill(2)
    gx, gw = m.Fused.rmsnorm_grad(g, s, w, eps=0.0)
    for k in (slice(0, 50), slice((1 << 24) - 50, (1 << 24) + 50), slice(n - 50, n)):
        assert (gw[k].to_numpy() == 1.0).all()                   # r = 1: 2 rows of 0.5
        assert (gx[:, k].to_numpy() == 0.0).all()                # along s nothing is left

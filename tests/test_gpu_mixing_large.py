"""The forms that rotary, single steps of linear attention, quantize and the product of 8-bit rows take past the caches, which arrays from 48 MiB on
choose by themselves; with vectors of 16 bytes on boundaries of one element alone (heads of odd length, a state in a window, rows of odd length).

Tolerances are those of the small tests; a form past the caches does the same operations in the same order as the others, so that the two agree bit by bit."""
import ctypes as C

import numpy as np
import pytest

from test_gpu_matmul_q8 import check, product
from test_gpu_rotary import close as close_rotary, reference as rotary_reference

pytestmark = pytest.mark.gpu

TYPES = [np.float32, np.float64]


def cls_of(m, dt):
    return m.SFloat if dt == np.float32 else m.DFloat


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,pairs", [(33, 16), (41, 16), (40, 16)])
def test_rotary(dt, interleaved, dim, pairs):
    """All at once, and in parts so small that they go through the caches; a window of longer heads, backwards in time."""
    import cumo_amd as m
    cls, shape = cls_of(m, dt), (3, 10010, 7, dim)
    rng = np.random.default_rng(dim)
    x = rng.standard_normal(shape, dtype=dt)
    p = rng.integers(0, 200000, shape[:2]).astype(np.int32)
    f = 10000.0 ** (-np.arange(pairs) / pairs)
    df, dp, dx = m.DFloat.cast(f), m.Int32.cast(p), cls.cast(x)
    y = m.Fused.rotary(dx, dp, df, interleaved, False, 1.25).to_numpy()
    for n in range(0, shape[1], 1001):
        part = m.Fused.rotary(cls.cast(np.ascontiguousarray(x[:, n:n + 1001])), m.Int32.cast(np.ascontiguousarray(p[:, n:n + 1001])), df, interleaved, False, 1.25)
        assert (part.to_numpy() == y[:, n:n + 1001]).all()
    some = slice(0, None, 997)
    close_rotary(y[:, some], *rotary_reference(x[:, some], p[:, some], f, interleaved, False, 1.25))
    buf = cls(shape[0], shape[1], shape[2], dim + 2).fill(7)
    window = buf[:, ::-1, :, 1:dim + 1]
    window.store(dx)
    out = cls(shape[0], shape[1], shape[2], dim + 2).fill(7)
    ref = lambda z: C.byref(z._desc())  # noqa: E731
    from cumo_amd import _lib
    _lib.call(_lib.lib.cumo_hip_na_rotary, ref(window), ref(dp), ref(df), int(interleaved), 0, 1.25, ref(out[:, :, :, 1:dim + 1]))
    got = out.to_numpy()
    assert (got[..., 1:dim + 1] == y).all() and (got[..., 0] == 7).all() and (got[..., dim + 1] == 7).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("wide", [64, 68])
def test_single_steps(dt, wide):
    """Every state on a boundary of one element, new and where it was; without one; quarters by themselves go through the caches."""
    import cumo_amd as m
    from cumo_amd import _lib
    cls, (b, h, d) = cls_of(m, dt), (96, 16, 66)
    rng = np.random.default_rng(wide)
    draw = lambda *n: rng.standard_normal(n, dtype=dt)  # noqa: E731
    q, k, v, s = draw(b, 1, h, d), draw(b, 1, h // 2, d), draw(b, 1, h // 2, wide), draw(b, h, d, wide)
    a = (1 - 2.0 ** (-1 - 8 * rng.random(h))).astype(dt)
    dq, dk, dv, da, ds = (cls.cast(z) for z in (q, k, v, a, s))
    o, last = (z.to_numpy() for z in m.Fused.linear_attention(dq, dk, dv, da, ds))
    for part in [slice(n, n + 24) for n in range(0, b, 24)]:   # (384 heads: a block to each, as for all of them)
        few = m.Fused.linear_attention(*(cls.cast(np.ascontiguousarray(z[part])) for z in (q, k, v)), da, cls.cast(np.ascontiguousarray(s[part])))
        assert (few[0].to_numpy() == o[part]).all() and (few[1].to_numpy() == last[part]).all()
    # by the definition: two roundings a number of the state (three more in numpy), and 66 + 64 a sum
    kk, vv = (np.repeat(z[:, 0].astype(np.float64), 2, axis=1) for z in (k, v))
    aa = a.astype(np.float64)[:, None, None]
    want = aa * s + kk[..., None] * vv[..., None, :]
    size = np.abs(aa * s) + np.abs(kk[..., None] * vv[..., None, :])
    half = np.finfo(dt).eps / 2
    assert (np.abs(last - want) <= 5 * half * size).all()
    qq = q[:, 0].astype(np.float64)[..., None]
    assert (np.abs(o[:, 0] - d ** -0.5 * (qq * want).sum(-2)) <= (d + 64) * half * d ** -0.5 * (np.abs(qq) * size).sum(-2)).all()
    # the state in a window that starts behind one element, read there, and then written there
    flat = cls(1 + s.size).fill(7)
    flat[1:1 + s.size].store(ds.reshape(s.size))
    at = ds._desc()
    at.ptr, at.offset = flat._desc().ptr, flat._desc().offset + np.dtype(dt).itemsize
    out, new = cls(b, 1, h, wide), cls(b, h, d, wide)
    ref = lambda z: C.byref(z._desc())  # noqa: E731
    for z in (ref(new), C.byref(at)):
        _lib.call(_lib.lib.cumo_hip_na_linear_attention, ref(dq), ref(dk), ref(dv), ref(da), C.byref(at), None, d ** -0.5, ref(out), z)
        assert (out.to_numpy() == o).all()
    assert (new.to_numpy() == last).all()
    held = flat.to_numpy()
    assert held[0] == 7 and (held[1:].reshape(s.shape) == last).all()
    empty = m.Fused.linear_attention(dq, dk, dv, da)[1].to_numpy()
    assert (empty == (kk.astype(dt)[..., None] * vv.astype(dt)[..., None, :])).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,cols", [(2600, 4095), (2600, 4096), (90000, 123)])
def test_quantize(dt, rows, cols):
    import cumo_amd as m
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((rows, cols), dtype=dt) * np.exp(rng.standard_normal((rows, 1))).astype(dt)
    q, scale = (z.to_numpy() for z in m.Fused.quantize(cls_of(m, dt).cast(x)))
    most = np.abs(x).max(axis=-1, keepdims=True).astype(np.longdouble)
    assert (np.abs(scale - most / 127) <= (np.finfo(dt).eps / 2 + 2.0 ** -53) * most / 127).all()
    wide = np.float64 if dt == np.float32 else np.longdouble   # (a quotient of two floats is no nearer than 2^-48 to a half that it is not)
    assert all((q[n:n + 1000] == np.rint(x[n:n + 1000].astype(wide) / scale[n:n + 1000].astype(wide))).all() for n in range(0, rows, 1000))


@pytest.mark.parametrize("dt,rows,inner,cols", [(np.float32, 4103, 70, 3301), (np.float64, 4103, 70, 3301), (np.float64, 2503, 130, 2603), (np.float64, 2503, 130, 2604)])
def test_product(dt, rows, inner, cols):
    """Tiles of 256 and of 128 (of 64 there are too few for results so large)."""
    import cumo_amd as m
    cls = cls_of(m, dt)
    rng = np.random.default_rng(cols)
    x, w = (rng.integers(-127, 128, s).astype(np.int8) for s in ((rows, inner), (cols, inner)))
    xs, ws = (np.exp(rng.standard_normal((n, 1))).astype(dt) for n in (rows, cols))
    bias = (100 * rng.standard_normal(cols)).astype(dt)
    for b in (None, bias):
        y = m.Fused.matmul_q8(m.Int8.cast(x), cls.cast(xs), m.Int8.cast(w), cls.cast(ws), None if b is None else cls.cast(b))
        check(y.to_numpy(), *product(x, xs, w, ws, b, dt))

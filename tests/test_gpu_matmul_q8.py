"""Rows in 8 bits and the product of such rows, against whole numbers and 64 bits.

Tolerances: quantize is exact but for the scale's one rounding (half a step). The product's sum is a whole number and exact; three roundings in
double and the one of the result follow."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = [np.float32, np.float64]
ROWS = [(1, 1), (3, 2), (5, 3), (2, 4), (7, 7), (33, 8), (70, 31), (9, 64), (64, 65), (4, 128), (1000, 129), (3, 5, 256), (40, 257), (5, 511), (6, 1023), (4, 1024), (1, 4096), (3, 4095),
        (5, 8190), (4, 8192), (2, 8193), (3, 16385), (2, 33001), (1, 70001), (300, 2050)]


def cls_of(m, dt):
    return m.SFloat if dt == np.float32 else m.DFloat


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", ROWS)
def test_quantize_matches_the_definition(dt, shape):
    import cumo_amd as m
    rng = np.random.default_rng(sum(shape))
    x = (rng.standard_normal(shape) * np.exp(rng.standard_normal(shape[:-1] + (1,)))).astype(dt)
    q, scale = m.Fused.quantize(cls_of(m, dt).cast(x))
    assert type(q) is m.Int8 and q.shape == shape and scale.shape == shape[:-1] + (1,)
    most, hs = np.abs(x).max(axis=-1, keepdims=True).astype(np.longdouble), scale.to_numpy().astype(np.longdouble)
    # (the quotient is a double before it is rounded to the type)
    assert (np.abs(hs - most / 127) <= (np.finfo(dt).eps / 2 + 2.0 ** -53) * most / 127).all()
    assert (q.to_numpy() == np.rint(x.astype(np.longdouble) / hs)).all()


@pytest.mark.parametrize("dt", TYPES)
def test_quantize_halves_go_to_even_numbers(dt):
    """Scales that are no powers of two, elements exactly between two steps."""
    import cumo_amd as m
    x = np.zeros((40, 300), dt)
    for r, scale in enumerate(np.arange(1, 41) * 3):
        x[r, :253] = (np.arange(253) - 126.5) * scale
        x[r, 254] = -127 * scale
    q, scale = m.Fused.quantize(cls_of(m, dt).cast(x))
    assert (scale.to_numpy()[:, 0] == np.arange(1, 41) * 3).all()
    want = np.rint(np.concatenate([np.arange(253) - 126.5, [0, -127], np.zeros(45)]))
    assert (q.to_numpy() == want).all()


@pytest.mark.parametrize("dt", TYPES)
def test_quantize_of_unusual_rows(dt):
    """Zeros; a NaN; an infinity; the least and the largest numbers."""
    import cumo_amd as m
    info = np.finfo(dt)
    least = info.smallest_subnormal
    x = np.zeros((9, 20), dt)
    x[1, 3], x[1, 4] = np.nan, 5
    x[2, 3], x[2, 4] = -np.inf, 5
    x[3, :3] = info.max, -info.max, info.max / 3
    x[4, :3] = info.tiny, -info.tiny / 2, info.tiny / 4
    x[5, :3] = 127 * least, -63 * least, 2 * least
    x[6, :2] = least, -least
    x[7, :3] = 254 * least, -127 * least, 3 * least
    x[8] = -1
    q, scale = (z.to_numpy() for z in m.Fused.quantize(cls_of(m, dt).cast(x)))
    assert (q[:3] == 0).all() and scale[0, 0] == 0 and np.isnan(scale[1, 0]) and scale[2, 0] == np.inf
    wide = x.astype(np.longdouble)
    for r in range(3, 9):
        s = scale[r, 0].astype(np.longdouble)
        want = np.clip(np.rint(wide[r] / s), -127, 127) if s > 0 else np.zeros(20)
        assert (q[r] == want).all(), r
    assert scale[6, 0] == 0 and scale[5, 0] == least


@pytest.mark.parametrize("dt", TYPES)
def test_quantize_layouts(dt):
    import cumo_amd as m
    cls = cls_of(m, dt)
    x = np.random.default_rng(5).standard_normal((6, 10, 33)).astype(dt)
    want = [z.to_numpy() for z in m.Fused.quantize(cls.cast(x))]
    for view in (cls.cast(np.ascontiguousarray(x.transpose())).transpose(), cls.cast(np.ascontiguousarray(x[::-1, ::-1, ::-1]))[::-1, ::-1, ::-1]):
        assert all((z.to_numpy() == w).all() for z, w in zip(m.Fused.quantize(view), want))
    assert m.Fused.quantize(cls(4, 0))[1].to_numpy().tolist() == [[0]] * 4
    assert m.Fused.quantize(cls(0, 4))[0].shape == (0, 4)


def product(x, xs, w, ws, bias, dt):
    """In 64 bits (SFloat) and more, with the sums as whole numbers."""
    wide = np.float64 if dt == np.float32 else np.longdouble
    total = x.astype(np.int64) @ w.astype(np.int64).T if x.size * w.shape[0] < 4e7 else (x.astype(np.float64) @ w.astype(np.float64).T)
    y = total.astype(wide) * xs.astype(wide) * ws.astype(wide).reshape(-1)
    size = np.abs(y) + (0 if bias is None else np.abs(bias))
    return y if bias is None else y + bias.astype(wide), size


def check(got, want, size):
    dt = got.dtype
    assert got.shape == want.shape
    bad = ~(np.abs(got - want) <= np.finfo(dt).eps / 2 * np.abs(want) + 4 * 2.0 ** -53 * size)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[0], got[bad][0], want[bad][0])


# rows, inner, cols: one row, a few, tiles and their ends, inner lengths that end inside every kind of piece
SIZES = [(1, 1, 1), (1, 16, 3), (1, 64, 64), (1, 4096, 512), (1, 4097, 130), (2, 63, 17), (3, 128, 100), (7, 65, 33), (16, 256, 256), (16, 1000, 300), (17, 129, 64), (33, 320, 70),
         (48, 513, 257), (64, 64, 64), (65, 127, 129), (100, 2048, 200), (128, 128, 128), (130, 192, 250), (255, 1030, 511), (256, 256, 256), (257, 64, 1025), (300, 4100, 520),
         (513, 384, 513), (1000, 70, 1000), (1030, 1024, 1540), (2050, 200, 2100), (5, 20000, 40), (200, 131071, 3), (1, 131071, 300)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,inner,cols", SIZES)
def test_matmul_matches_whole_numbers(dt, rows, inner, cols):
    import cumo_amd as m
    cls = cls_of(m, dt)
    rng = np.random.default_rng(rows + inner + cols)
    x, w = (rng.integers(-127, 128, s).astype(np.int8) for s in ((rows, inner), (cols, inner)))
    xs, ws = (np.exp(rng.standard_normal((n, 1))).astype(dt) for n in (rows, cols))
    bias = (100 * rng.standard_normal(cols)).astype(dt)
    dx, dw = m.Int8.cast(x), m.Int8.cast(w)
    for b in (None, bias):
        y = m.Fused.matmul_q8(dx, cls.cast(xs), dw, cls.cast(ws), None if b is None else cls.cast(b))
        assert type(y) is cls
        check(y.to_numpy(), *product(x, xs, w, ws, b, dt))


@pytest.mark.parametrize("rows", [70, 300, 3000])
@pytest.mark.parametrize("inner", [1, 2, 5, 15, 16, 17, 31, 33, 47, 112, 113, 127, 143, 255, 257, 271])
def test_matmul_of_tiles_whose_rows_end_anywhere(rows, inner):
    """Whole arrays and windows of rows that stand among others' bytes."""
    import cumo_amd as m
    rng = np.random.default_rng(rows + inner)
    x, w = (rng.integers(-127, 128, (n, inner + 20)).astype(np.int8) for n in (rows, 3100))
    xs, ws = (rng.random((n, 1)).astype(np.float32) for n in (rows, 3100))
    for part in (slice(0, inner), slice(9, 9 + inner)):
        for forms in (lambda z: m.Int8.cast(np.ascontiguousarray(z[:, part])), lambda z: m.Int8.cast(z)[:, part]):
            y = m.Fused.matmul_q8(forms(x), m.SFloat.cast(xs), forms(w), m.SFloat.cast(ws))
            check(y.to_numpy(), *product(x[:, part], xs, w[:, part], ws, None, np.float32))


@pytest.mark.parametrize("rows", [1, 20, 300])
def test_matmul_sums_reach_the_ends_of_32_bits(rows):
    """131071 products of -128 by -128, of 127 by -128."""
    import cumo_amd as m
    n = 131071
    x, w = np.full((rows, n), -128, np.int8), np.full((4, n), -128, np.int8)
    w[1] = 127
    w[2, ::2] = 127
    one = m.DFloat.cast(np.ones((rows, 1))), m.DFloat.cast(np.ones((4, 1)))
    y = m.Fused.matmul_q8(m.Int8.cast(x), one[0], m.Int8.cast(w), one[1]).to_numpy()
    assert (y == (w.astype(np.int64).sum(axis=1) * -128)).all() and y[0, 0] == 16384 * n


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows", [3, 70, 600])
def test_matmul_layouts(dt, rows):
    """Batches, windows of rows on any boundary, rows far apart, repeated and backwards, transposed and every other element; results in windows."""
    import cumo_amd as m
    from cumo_amd import _lib
    cls = cls_of(m, dt)
    rng = np.random.default_rng(rows)
    x, w = rng.integers(-127, 128, (rows, 131)).astype(np.int8), rng.integers(-127, 128, (90, 131)).astype(np.int8)
    xs, ws = rng.random((rows, 1)).astype(dt), rng.random((90, 1)).astype(dt)
    dxs, dws = cls.cast(xs), cls.cast(ws)
    want = m.Fused.matmul_q8(m.Int8.cast(x), dxs, m.Int8.cast(w), dws).to_numpy()

    def forms(a):
        wide = np.full((a.shape[0], 200), 99, np.int8)
        wide[:, 7:138] = a
        yield m.Int8.cast(wide)[:, 7:138]
        yield m.Int8.cast(np.ascontiguousarray(a[::-1]))[::-1]
        yield m.Int8.cast(np.ascontiguousarray(a.T)).transpose()
        every = np.zeros((a.shape[0], 262), np.int8)
        every[:, ::2] = a
        yield m.Int8.cast(every)[:, ::2]

    for fx, fw in zip(forms(x), forms(w)):
        assert (m.Fused.matmul_q8(fx, dxs, fw, dws).to_numpy() == want).all()
    batch = m.Fused.matmul_q8(m.Int8.cast(x).reshape(rows, 1, 131), dxs.reshape(rows, 1, 1), m.Int8.cast(w), dws)
    assert batch.shape == (rows, 1, 90) and (batch.to_numpy()[:, 0] == want).all()
    one = m.Fused.matmul_q8(m.Int8.cast(x[0]), cls.cast(xs[0]), m.Int8.cast(w), dws)
    assert one.shape == (90,) and (one.to_numpy() == want[0]).all()
    ref = lambda z: C.byref(z._desc())  # noqa: E731
    dx, dw = m.Int8.cast(x), m.Int8.cast(w)
    for shape, part in (((rows, 97), (slice(None), slice(3, 93))), ((rows, 180), (slice(None), slice(0, 180, 2))), ((2 * rows, 90), (slice(None, None, -2), slice(None)))):
        buf = cls(*shape).fill(7)
        y = buf[part]
        _lib.call(_lib.lib.cumo_hip_na_matmul_q8, ref(dx), ref(dxs), ref(dw), ref(dws), None, ref(y))
        got = buf.to_numpy()
        assert (got[part] == want).all()
        got[part] = 7
        assert (got == 7).all()


@pytest.mark.parametrize("dt", TYPES)
def test_matmul_of_nothing_and_of_no_numbers(dt):
    """No rows, no columns, rows of no elements (the bias, or 0); scales of 0, infinity and NaN stay in their rows and columns."""
    import cumo_amd as m
    cls = cls_of(m, dt)
    one = lambda *n: cls(*n).fill(1)  # noqa: E731
    assert m.Fused.matmul_q8(m.Int8(0, 5), one(0, 1), m.Int8(3, 5), one(3, 1)).shape == (0, 3)
    assert m.Fused.matmul_q8(m.Int8(4, 5), one(4, 1), m.Int8(0, 5), one(0, 1)).shape == (4, 0)
    y = m.Fused.matmul_q8(m.Int8(4, 0), one(4, 1), m.Int8(3, 0), one(3, 1), cls.cast(np.array([1, 2, 3], dt)))
    assert (y.to_numpy() == [[1, 2, 3]] * 4).all()
    x = np.ones((20, 40), np.int8)
    xs, ws = np.ones((20, 1), dt), np.ones((30, 1), dt)
    xs[3], xs[4], ws[5], ws[6] = np.nan, 0, np.inf, np.nan
    y = m.Fused.matmul_q8(m.Int8.cast(x), cls.cast(xs), m.Int8.cast(np.ones((30, 40), np.int8)), cls.cast(ws)).to_numpy()
    want = 40.0 * xs.astype(np.float64) * ws.astype(np.float64).T
    assert ((y == want) | (np.isnan(y) & np.isnan(want))).all()


def test_matmul_of_more_columns_than_blocks_of_sixteen_reach():
    """2^27 columns and some, two rows: more than 2^32 lanes if every sixteen columns were a block's."""
    import cumo_amd as m
    cols = (1 << 27) + 37
    w = (np.arange(cols, dtype=np.uint32) * np.uint32(2654435761) >> np.uint32(24)).astype(np.uint8).view(np.int8).reshape(cols, 1)
    y = m.Fused.matmul_q8(m.Int8.cast(np.array([[3], [-5]], np.int8)), m.SFloat.cast(np.ones((2, 1), np.float32)), m.Int8.cast(w), m.SFloat(cols, 1).fill(1)).to_numpy()
    for r, x in enumerate((3, -5)):
        assert (y[r] == np.int16(x) * w[:, 0].astype(np.int16)).all()


@pytest.mark.parametrize("rows", [4, 200])
def test_captured_on_another_stream(rows):
    import cumo_amd as m
    from cumo_amd import _lib
    from test_gpu_index import hip_runtime
    hip, L = hip_runtime(), _lib.lib
    rng = np.random.default_rng(rows)
    x, w = (m.SFloat.cast(rng.standard_normal(s).astype(np.float32)) for s in ((rows, 1100), (700, 1100)))
    qw, ws = m.Fused.quantize(w)
    q, xs = m.Fused.quantize(x)
    want = m.Fused.matmul_q8(q, xs, qw, ws).to_numpy()
    y = m.SFloat(rows, 700)
    q.store_binary(bytes(rows * 1100))
    ref = lambda z: C.byref(z._desc())  # noqa: E731
    args = [ref(z) for z in (x, q, xs, qw, ws, y)]
    stream = C.c_void_p(L.cumo_hip_stream_create())
    graph, ready = C.c_void_p(), C.c_void_p()
    m.synchronize()
    L.cumo_hip_set_stream(stream)
    try:
        assert hip.hipStreamBeginCapture(stream, 2) == 0
        _lib.call(L.cumo_hip_na_quantize, args[0], args[1], args[2])
        _lib.call(L.cumo_hip_na_matmul_q8, args[1], args[2], args[3], args[4], None, args[5])
        assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert hip.hipGraphInstantiate(C.byref(ready), graph, None, None, C.c_size_t(0)) == 0
        for _ in range(3):
            dirt = [m.SFloat(n).fill(float("nan")) for n in (64, 3000, 100000)]
            y.fill(5)
            assert hip.hipGraphLaunch(ready, stream) == 0
            m.synchronize()
            assert (y.to_numpy() == want).all()
            assert (m.Fused.matmul_q8(q, xs, qw, ws).to_numpy() == want).all()
            del dirt
    finally:
        L.cumo_hip_set_stream(None)
        if ready:
            hip.hipGraphExecDestroy(ready)
        if graph:
            hip.hipGraphDestroy(graph)
        L.cumo_hip_stream_destroy(stream)

"""What the row operators and the recurrence refuse, without a GPU: the error's kind, nothing allocated, results left as
they came. Operands are made-up addresses; a refused call reads none of them."""
import ctypes as C

import pytest

from cumo_amd import _lib
from cumo_amd._lib import NArrayDesc

L = _lib.lib
SF, DF, I32, I64, U64, BIT, I8 = range(7)
ELMSZ = {SF: 4, DF: 8, I32: 4, I64: 8, U64: 8, BIT: 1, I8: 1}
ARGUMENT, SHAPE, TYPE, DIMENSION = 3, 4, 6, 8


@pytest.fixture(autouse=True)
def host_pool():
    L.cumo_hip_pool_free_all_blocks()
    assert L.cumo_hip_pool_use_host_backend(1) == 0
    yield
    L.cumo_hip_pool_free_all_blocks()
    assert L.cumo_hip_pool_total_bytes() == 0, "a refused call kept memory"
    assert L.cumo_hip_pool_use_host_backend(0) == 0
    L.cumo_hip_last_error(None)


_at = [0x10000000]


def view(type_, *shape, ptr=None):
    d = NArrayDesc()
    d.type, d.ndim, d.offset = type_, len(shape), 0
    _at[0] += 0x10000000
    d.ptr = _at[0] if ptr is None else ptr
    s = ELMSZ[type_]
    for k in range(len(shape) - 1, -1, -1):
        d.shape[k], d.stride[k] = shape[k], s
        s *= shape[k]
    return d


def refused(kind, f, *args):
    args = [C.byref(a) if isinstance(a, NArrayDesc) else a for a in args]
    mallocs = L.cumo_hip_pool_device_malloc_calls()
    assert f(*args) == kind
    msg = C.c_char_p()
    assert L.cumo_hip_last_error(C.byref(msg)) == kind and msg.value
    assert L.cumo_hip_pool_device_malloc_calls() == mallocs
    for a in args:
        if hasattr(a, "_obj") and isinstance(a._obj, NArrayDesc):
            assert a._obj.ndim == 0 or a._obj.ptr


def new():
    return NArrayDesc()


def test_rmsnorm():
    f = L.cumo_hip_na_rmsnorm
    x = view(SF, 4, 8)
    refused(TYPE, f, view(I32, 4, 8), None, None, 1e-6, new(), None)
    refused(TYPE, f, view(I8, 4, 8), None, None, 1e-6, new(), None)
    refused(TYPE, f, x, view(DF, 8), None, 1e-6, new(), None)
    refused(TYPE, f, x, None, view(DF, 4, 8), 1e-6, new(), new())
    refused(DIMENSION, f, view(SF), None, None, 1e-6, new(), None)
    refused(SHAPE, f, x, view(SF, 7), None, 1e-6, new(), None)
    refused(SHAPE, f, x, view(SF, 1, 8), None, 1e-6, new(), None)
    refused(SHAPE, f, x, None, view(SF, 1, 8), 1e-6, new(), new())
    for eps in (-1.0, float("nan"), float("inf")):
        refused(ARGUMENT, f, x, None, None, eps, new(), None)
    refused(ARGUMENT, f, x, None, None, 1e-6, new(), new())           # a sum without a residual
    refused(ARGUMENT, f, x, None, view(SF, 4, 8), 1e-6, new(), None)  # a residual without a sum
    refused(ARGUMENT, f, None, None, None, 1e-6, new(), None)
    refused(ARGUMENT, f, x, None, None, 1e-6, None, None)
    refused(TYPE, f, x, None, None, 1e-6, view(DF, 4, 8), None)
    refused(SHAPE, f, x, None, None, 1e-6, view(SF, 8, 4), None)
    y = view(SF, 4, 8)
    refused(ARGUMENT, f, x, None, view(SF, 4, 8), 1e-6, y, view(SF, 4, 8, ptr=y.ptr + 64))   # results in one another
    q = L.cumo_hip_na_rmsnorm_q8
    refused(ARGUMENT, q, x, None, None, 1e-6, new(), None, None)
    refused(TYPE, q, x, None, None, 1e-6, view(SF, 4, 8), new(), None)
    refused(SHAPE, q, x, None, None, 1e-6, view(I8, 4, 8), view(SF, 4), None)
    refused(TYPE, q, view(BIT, 4, 8), None, None, 1e-6, new(), new(), None)


def test_dequantize():
    f = L.cumo_hip_na_dequantize
    refused(TYPE, f, view(SF, 4, 8), view(SF, 4, 1), new())
    refused(TYPE, f, view(I8, 4, 8), view(I32, 4, 1), new())
    refused(SHAPE, f, view(I8, 4, 8), view(SF, 4), new())
    refused(SHAPE, f, view(I8, 4, 8), view(SF, 1, 1), new())
    refused(DIMENSION, f, view(I8), view(SF), new())
    refused(TYPE, f, view(I8, 4, 8), view(SF, 4, 1), view(DF, 4, 8))


def test_rmsnorm_grad():
    f = L.cumo_hip_na_rmsnorm_grad
    g, s, w = view(SF, 4, 8), view(SF, 4, 8), view(SF, 8)
    refused(SHAPE, f, g, view(SF, 4, 7), None, None, 1e-6, new(), None)
    refused(TYPE, f, g, view(DF, 4, 8), None, None, 1e-6, new(), None)
    refused(SHAPE, f, g, s, None, view(SF, 8), 1e-6, new(), None)
    refused(TYPE, f, g, s, None, view(DF, 4, 8), 1e-6, new(), None)
    refused(ARGUMENT, f, g, s, w, None, 1e-6, new(), None)
    refused(ARGUMENT, f, g, s, None, None, 1e-6, new(), new())
    refused(ARGUMENT, f, g, None, None, None, 1e-6, new(), None)
    refused(ARGUMENT, f, g, s, None, None, -1e-6, new(), None)
    refused(SHAPE, f, g, s, w, None, 1e-6, new(), view(SF, 4, 8))
    gx = view(SF, 4, 8)
    refused(ARGUMENT, f, g, s, w, None, 1e-6, gx, view(SF, 8, ptr=gx.ptr))


def test_recurrence():
    f = L.cumo_hip_na_recurrence
    a, b = view(SF, 2, 9, 5), view(SF, 2, 9, 5)
    for axis in (-1, 3):
        refused(DIMENSION, f, a, b, None, axis, new())
    refused(DIMENSION, f, view(SF), view(SF), None, 0, new())
    refused(SHAPE, f, a, view(SF, 2, 1, 5), None, 1, new())
    refused(SHAPE, f, a, view(SF, 9, 5), None, 1, new())
    refused(TYPE, f, a, view(DF, 2, 9, 5), None, 1, new())
    refused(TYPE, f, view(I32, 4), view(I32, 4), None, 0, new())
    refused(SHAPE, f, a, b, view(SF, 2, 9), 1, new())
    refused(SHAPE, f, a, b, view(SF, 2, 1, 5), 1, new())
    refused(TYPE, f, a, b, view(DF, 2, 5), 1, new())
    refused(ARGUMENT, f, a, None, None, 1, new())
    refused(SHAPE, f, a, b, None, 1, view(SF, 2, 9, 4))
    q = L.cumo_hip_na_recurrence_grad
    h, h0 = view(SF, 2, 9, 5), view(SF, 2, 5)
    refused(SHAPE, q, a, b, view(SF, 2, 9, 6), None, 1, new(), new(), None)
    refused(TYPE, q, a, b, view(DF, 2, 9, 5), None, 1, new(), new(), None)
    refused(ARGUMENT, q, a, b, h, h0, 1, new(), new(), None)
    refused(ARGUMENT, q, a, b, h, None, 1, new(), new(), new())
    ga = view(SF, 2, 9, 5)
    refused(ARGUMENT, q, a, b, h, None, 1, ga, view(SF, 2, 9, 5, ptr=ga.ptr + 4), None)


def test_sample():
    f = L.cumo_hip_na_sample
    x, u = view(SF, 4, 100), view(SF, 4)

    def call(x=x, u=u, t=1.0, ts=None, k=0, ks=None, p=1.0, ps=None, m=0.0, ms=None, z=None):
        return x, u, t, ts, k, ks, p, ps, m, ms, z or new()

    nan = float("nan")
    refused(TYPE, f, *call(x=view(I32, 4, 100)))
    refused(TYPE, f, *call(u=view(I32, 4)))
    refused(DIMENSION, f, *call(x=view(SF), u=view(SF)))
    refused(SHAPE, f, *call(u=view(SF, 5)))
    refused(SHAPE, f, *call(u=view(SF, 4, 1)))
    refused(SHAPE, f, *call(u=view(SF)))
    refused(ARGUMENT, f, *call(u=None))
    for t in (-0.5, nan):
        refused(ARGUMENT, f, *call(t=t))
    refused(ARGUMENT, f, *call(k=-1))
    for p in (-0.1, 1.1, nan):
        refused(ARGUMENT, f, *call(p=p))
        refused(ARGUMENT, f, *call(m=p))
    refused(TYPE, f, *call(ks=view(SF, 4)))
    refused(TYPE, f, *call(ts=view(I32, 4)))
    refused(SHAPE, f, *call(ps=view(SF, 3)))
    refused(SHAPE, f, *call(ms=view(DF, 4, 100)))
    refused(ARGUMENT, f, *call(x=view(SF, 4, 1 << 31)))
    refused(TYPE, f, *call(z=view(I64, 4)))
    refused(SHAPE, f, *call(z=view(I32, 5)))


def test_python_names():
    import cumo_amd as m
    assert m.Int8.type_code == 6 and m.Int8.elmsz == 1
    for bad in (lambda: m.Fused.rmsnorm([1.0]), lambda: m.Fused.sample(3, 4), lambda: m.Fused.recurrence(1, 2), lambda: m.Fused.dequantize(1, 2)):
        with pytest.raises(TypeError):
            bad()


def window(type_, ptr, shape, stride, offset=0):
    d = view(type_, *shape, ptr=ptr)
    d.offset = offset
    for k, s in enumerate(stride):
        d.stride[k] = s
    return d


def test_windows_of_one_array_that_share_elements():
    """Columns [0, 6) and [5, 11) of rows of 11; channels 0, 2, ... and 1, 2, 3, ...; a matrix and its transpose; one row of another."""
    f = L.cumo_hip_na_recurrence_grad
    at = 0x70000000
    cases = [((4, 6), (44, 4), 0, (44, 4), 20), ((4, 5), (88, 8), 0, (88, 4), 4), ((5, 5), (20, 4), 0, (4, 20), 0), ((1, 6), (24, 4), 48, (24, 4), 52),
             ((3, 4), (160, 40), 0, (40, 40), 80), ((3, 2, 3), (120, 40, 8), 4, (120, 20, 8), 24)]
    for shape, one, at_one, two, at_two in cases:
        g, a, h = (view(SF, *shape) for _ in range(3))
        refused(ARGUMENT, f, g, a, h, None, 0, window(SF, at, shape, one, at_one), window(SF, at, shape, two, at_two), None)
        refused(ARGUMENT, f, g, a, h, None, 0, window(SF, at, shape, two, at_two), window(SF, at, shape, one, at_one), None)

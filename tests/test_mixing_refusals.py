"""What products of 8-bit rows, rotary positions and linear attention refuse, without a GPU: the error's kind, nothing allocated, results left
as they came. Operands are made-up addresses; a refused call reads none of them."""
import pytest

from test_fused_refusals import ARGUMENT, BIT, DF, DIMENSION, I32, I8, L, SF, SHAPE, TYPE, host_pool, new, refused, view  # noqa: F401


def test_quantize():
    f = L.cumo_hip_na_quantize
    x = view(SF, 4, 8)
    refused(TYPE, f, view(I32, 4, 8), new(), new())
    refused(TYPE, f, view(I8, 4, 8), new(), new())
    refused(DIMENSION, f, view(SF), new(), new())
    refused(ARGUMENT, f, None, new(), new())
    refused(ARGUMENT, f, x, None, new())
    refused(ARGUMENT, f, x, new(), None)
    refused(TYPE, f, x, view(SF, 4, 8), new())
    refused(SHAPE, f, x, view(I8, 4, 7), new())
    refused(TYPE, f, x, new(), view(DF, 4, 1))
    refused(SHAPE, f, x, new(), view(SF, 4))
    q = view(I8, 4, 8)
    refused(ARGUMENT, f, x, q, view(SF, 4, 1, ptr=q.ptr + 16))


def test_matmul_q8():
    f = L.cumo_hip_na_matmul_q8
    x, xs, w, ws = view(I8, 4, 8), view(SF, 4, 1), view(I8, 5, 8), view(SF, 5, 1)
    refused(TYPE, f, view(SF, 4, 8), xs, w, ws, None, new())
    refused(TYPE, f, x, xs, view(BIT, 5, 8), ws, None, new())
    refused(TYPE, f, x, view(I32, 4, 1), w, ws, None, new())
    refused(TYPE, f, x, xs, w, view(DF, 5, 1), None, new())
    refused(TYPE, f, x, xs, w, ws, view(DF, 5), new())
    refused(DIMENSION, f, view(I8), view(SF), w, ws, None, new())
    refused(DIMENSION, f, x, xs, view(I8, 8), ws, None, new())
    refused(DIMENSION, f, x, xs, view(I8, 1, 5, 8), ws, None, new())
    refused(SHAPE, f, x, xs, view(I8, 5, 7), ws, None, new())
    refused(SHAPE, f, x, view(SF, 4), w, ws, None, new())
    refused(SHAPE, f, x, view(SF, 1, 1), w, ws, None, new())
    refused(SHAPE, f, x, xs, w, view(SF, 5), None, new())
    refused(SHAPE, f, x, xs, w, view(SF, 1, 5), None, new())
    refused(SHAPE, f, x, xs, w, ws, view(SF, 4), new())
    refused(SHAPE, f, x, xs, w, ws, view(SF, 5, 1), new())
    for k in range(4):
        args = [x, xs, w, ws, None, new()]
        args[k] = None
        refused(ARGUMENT, f, *args)
    refused(ARGUMENT, f, x, xs, w, ws, None, None)
    refused(ARGUMENT, f, view(I8, 4, 1 << 17), xs, view(I8, 5, 1 << 17), ws, None, new())
    refused(TYPE, f, x, xs, w, ws, None, view(DF, 4, 5))
    refused(SHAPE, f, x, xs, w, ws, None, view(SF, 5, 4))


def test_rotary():
    f = L.cumo_hip_na_rotary
    x, p, fr = view(SF, 2, 3, 4, 8), view(I32, 2, 3), view(DF, 4)
    refused(TYPE, f, view(I32, 2, 3, 4, 8), p, fr, 0, 0, 1.0, new())
    refused(TYPE, f, x, view(SF, 2, 3), fr, 0, 0, 1.0, new())
    refused(TYPE, f, x, p, view(SF, 4), 0, 0, 1.0, new())
    refused(DIMENSION, f, view(SF, 8), view(I32), fr, 0, 0, 1.0, new())
    refused(DIMENSION, f, x, p, view(DF, 1, 4), 0, 0, 1.0, new())
    refused(SHAPE, f, x, view(I32, 3), fr, 0, 0, 1.0, new())
    refused(SHAPE, f, x, view(I32, 2, 3, 1), fr, 0, 0, 1.0, new())
    refused(SHAPE, f, x, p, view(DF, 5), 0, 0, 1.0, new())
    refused(SHAPE, f, view(SF, 2, 3, 4, 9), p, view(DF, 5), 0, 0, 1.0, new())
    for amplitude in (float("nan"), float("inf")):
        refused(ARGUMENT, f, x, p, fr, 0, 0, amplitude, new())
    refused(ARGUMENT, f, None, p, fr, 0, 0, 1.0, new())
    refused(ARGUMENT, f, x, None, fr, 0, 0, 1.0, new())
    refused(ARGUMENT, f, x, p, None, 0, 0, 1.0, new())
    refused(ARGUMENT, f, x, p, fr, 0, 0, 1.0, None)
    refused(ARGUMENT, f, view(SF, 2, 3, 1 << 31, 8), p, fr, 0, 0, 1.0, new())
    refused(TYPE, f, x, p, fr, 0, 0, 1.0, view(DF, 2, 3, 4, 8))
    refused(SHAPE, f, x, p, fr, 0, 0, 1.0, view(SF, 6, 4, 8))


def test_linear_attention():
    f = L.cumo_hip_na_linear_attention

    def call(q=view(SF, 2, 9, 4, 8), k=view(SF, 2, 9, 2, 8), v=view(SF, 2, 9, 2, 6), a=view(SF, 4), s=None, n=None, scale=1.0, o=None, last=None):
        return q, k, v, a, s, n, scale, o or new(), last

    for name, bad in (("q", view(I32, 2, 9, 4, 8)), ("k", view(DF, 2, 9, 2, 8)), ("v", view(DF, 2, 9, 2, 6)), ("a", view(DF, 4)), ("s", view(DF, 2, 4, 8, 6)),
                      ("n", view(SF, 2)), ("o", view(DF, 2, 9, 4, 6)), ("last", view(DF, 2, 4, 8, 6))):
        refused(TYPE, f, *call(**{name: bad}))
    for name, bad in (("q", view(SF, 2, 4, 8)), ("k", view(SF, 2, 8)), ("v", view(SF, 1, 2, 9, 2, 6))):
        refused(DIMENSION, f, *call(**{name: bad}))
    for name, bad in (("k", view(SF, 2, 9, 2, 7)), ("k", view(SF, 2, 8, 2, 8)), ("k", view(SF, 1, 9, 2, 8)), ("v", view(SF, 2, 8, 2, 6)), ("v", view(SF, 2, 9, 1, 6)),
                      ("a", view(SF, 2)), ("a", view(SF, 4, 1)), ("s", view(SF, 2, 2, 8, 6)), ("s", view(SF, 2, 4, 6, 8)), ("n", view(I32, 9)), ("n", view(I32, 2, 1)),
                      ("o", view(SF, 2, 9, 4, 8)), ("last", view(SF, 2, 4, 6, 8))):
        refused(SHAPE, f, *call(**{name: bad}))
    refused(SHAPE, f, *call(k=view(SF, 2, 9, 3, 8), v=view(SF, 2, 9, 3, 6)))     # four heads for three
    refused(SHAPE, f, *call(k=view(SF, 2, 9, 0, 8), v=view(SF, 2, 9, 0, 6)))
    refused(ARGUMENT, f, *call(q=view(SF, 2, 9, 4, 257), k=view(SF, 2, 9, 2, 257)))
    refused(ARGUMENT, f, *call(v=view(SF, 2, 9, 2, 257)))
    for scale in (float("nan"), float("inf")):
        refused(ARGUMENT, f, *call(scale=scale))
    for k in range(4):
        args = list(call())
        args[k] = None
        refused(ARGUMENT, f, *args)
    refused(ARGUMENT, f, *call()[:7], None, None)
    o = view(SF, 2, 9, 4, 6)
    refused(ARGUMENT, f, *call(o=o, last=view(SF, 2, 4, 8, 6, ptr=o.ptr + 400)))
    big = 1 << 31
    refused(ARGUMENT, f, *call(q=view(SF, 2, big, 4, 8), k=view(SF, 2, big, 2, 8), v=view(SF, 2, big, 2, 6)))
    many = 1 << 20
    refused(ARGUMENT, f, *call(q=view(SF, many, 9, 4, 8), k=view(SF, many, 9, 2, 8), v=view(SF, many, 9, 2, 6)))


def test_linear_attention_grad():
    f = L.cumo_hip_na_linear_attention_grad

    def call(g=view(SF, 2, 9, 4, 6), q=view(SF, 2, 9, 4, 8), k=view(SF, 2, 9, 2, 8), v=view(SF, 2, 9, 2, 6), a=view(SF, 4), s=None, gl=None, n=None, scale=1.0, gq=None, gk=None,
             gv=None, gs=None):
        return g, q, k, v, a, s, gl, n, scale, gq or new(), gk or new(), gv or new(), gs

    for name, bad in (("g", view(DF, 2, 9, 4, 6)), ("k", view(DF, 2, 9, 2, 8)), ("gl", view(DF, 2, 4, 8, 6)), ("gq", view(DF, 2, 9, 4, 8)), ("n", view(DF, 2))):
        refused(TYPE, f, *call(**{name: bad}))
    for name, bad in (("g", view(SF, 2, 9, 2, 6)), ("g", view(SF, 2, 9, 4, 8)), ("g", view(SF, 2, 8, 4, 6)), ("gl", view(SF, 2, 2, 8, 6)), ("gq", view(SF, 2, 9, 2, 8)),
                      ("gk", view(SF, 2, 9, 4, 8)), ("gv", view(SF, 2, 9, 4, 6))):
        refused(SHAPE, f, *call(**{name: bad}))
    refused(DIMENSION, f, *call(g=view(SF, 2, 4, 6)))
    refused(ARGUMENT, f, *call(s=view(SF, 2, 4, 8, 6)))                    # a state without its gradient
    refused(ARGUMENT, f, *call(gs=new()))                                  # and the other way round
    refused(ARGUMENT, f, *call(scale=float("nan")))
    for k in range(5):
        args = list(call())
        args[k] = None
        refused(ARGUMENT, f, *args)
    for k in range(9, 12):
        args = list(call())
        args[k] = None
        refused(ARGUMENT, f, *args)
    gq = view(SF, 2, 9, 4, 8)
    refused(ARGUMENT, f, *call(gq=gq, gk=view(SF, 2, 9, 2, 8, ptr=gq.ptr)))


def test_python_names():
    import cumo_amd as m
    F = m.Fused
    for bad in (lambda: F.quantize([1.0]), lambda: F.matmul_q8(1, 2, 3, 4), lambda: F.rotary(1, 2, 3), lambda: F.linear_attention(1, 2, 3, 4),
                lambda: F.linear_attention_grad(1, 2, 3, 4, 5)):
        with pytest.raises(TypeError):
            bad()

"""Limits of the operators of a layer with a matrix state, without a GPU: what is beyond them is refused before anything is held for it."""
from test_fused_refusals import ARGUMENT, DF, I8, L, SF, host_pool, new, refused, view  # noqa: F401


def test_matmul_q8_of_too_many_rows_by_columns():
    f = L.cumo_hip_na_matmul_q8
    for rows, cols in ((1 << 30, 1), (1, 1 << 30), (1 << 31, 1), (1, 1 << 31), (1 << 20, 1 << 18)):
        refused(ARGUMENT, f, view(I8, rows, 1), view(SF, rows, 1), view(I8, cols, 1), view(SF, cols, 1), None, new())
    # none at all are not too many
    for rows, cols in ((1 << 31, 0), (0, 1 << 31)):
        z = new()
        assert f(view(I8, rows, 1), view(SF, rows, 1), view(I8, cols, 1), view(SF, cols, 1), None, z) == 0 and list(z.shape[:2]) == [rows, cols]


def test_linear_attention_of_sequences_by_heads_that_pass_64_bits():
    """Sequences of no steps take no memory, and their product with the heads is 0 modulo 2^64, or 1."""
    f, grad = L.cumo_hip_na_linear_attention, L.cumo_hip_na_linear_attention_grad
    for batch, heads in ((1 << 32, 1 << 32), (1 << 40, 1 << 24), (pow(12345679, -1, 1 << 64), 12345679)):
        q, kv, a = view(SF, batch, 0, heads, 4), view(SF, batch, 0, 1, 4), view(SF, heads)
        refused(ARGUMENT, f, q, kv, kv, a, None, None, 1.0, new(), new())
        refused(ARGUMENT, f, q, kv, kv, a, None, None, 1.0, new(), None)
        refused(ARGUMENT, grad, q, q, kv, kv, a, None, None, None, 1.0, new(), new(), new(), None)


def test_linear_attention_by_a_scale_that_its_type_does_not_reach():
    f, grad = L.cumo_hip_na_linear_attention, L.cumo_hip_na_linear_attention_grad
    q, kv, a, n = view(SF, 2, 0, 4, 4), view(SF, 2, 0, 1, 4), view(SF, 4), new
    for scale in (1e39, -1e300):
        refused(ARGUMENT, f, q, kv, kv, a, None, None, scale, n(), None)
        refused(ARGUMENT, grad, q, q, kv, kv, a, None, None, None, scale, n(), n(), n(), None)
    assert f(q, kv, kv, a, None, None, 3.4e38, n(), None) == 0
    q, kv, a = view(DF, 2, 0, 4, 4), view(DF, 2, 0, 1, 4), view(DF, 4)
    assert f(q, kv, kv, a, None, None, -1e300, n(), None) == 0

// The host layer's row operators and the recurrence: checks, layouts, results; the kernels are in rmsnorm.hip,
// recurrence.hip and sample.hip. (Library additions; the reference has no such methods.)
//
// No function here keeps a C++ object with a destructor alive across a call that may report an error: the installed
// handler may leave with longjmp.
#include <cmath>
#include <cstdint>
#include <cstring>

#include "ndloop_views.h"

using namespace cumo_hip;

namespace {

int check_float(const NA* a, const char* message) {
    const int rc = check_view(a, "operand");
    if (rc) return rc;
    return is_float(a->type) ? CUMO_HIP_OK : fail(CUMO_HIP_ERROR_TYPE, message);
}

bool same_shape(const NA* a, int ndim, const size_t* shape) {
    bool same = a->ndim == ndim;
    for (int d = 0; same && d < ndim; ++d) same = a->shape[d] == shape[d];
    return same;
}

// the same for one number a row (a state, a setting): where nothing is left of the shape, an array of one element will do
bool same_rows(const NA* a, int ndim, const size_t* shape) {
    return same_shape(a, ndim, shape) || (ndim == 0 && a->ndim == 1 && a->shape[0] == 1);
}

// the bytes from a view's first to behind its last element
void reach(const NA* a, uintptr_t* low, uintptr_t* high) {
    ssize_t lo = 0, hi = 0;
    for (int d = 0; d < a->ndim; ++d) {
        if (a->shape[d] == 0) {
            *low = *high = 0;
            return;
        }
        const ssize_t far = a->stride[d] * (ssize_t)(a->shape[d] - 1);
        (far < 0 ? lo : hi) += far;
    }
    const uintptr_t at = (uintptr_t)a->ptr + (uintptr_t)a->offset;
    *low = at + (uintptr_t)lo;
    *high = at + (uintptr_t)hi + (uintptr_t)kElmsz[a->type];
}

bool overlap(const NA* a, const NA* b) {
    uintptr_t al, ah, bl, bh;
    reach(a, &al, &ah);
    reach(b, &bl, &bh);
    return al < bh && bl < ah;
}

// the dimensions of a view that are in the mask: from its first byte to behind its last, counted from the element at no index
void span(const NA* a, unsigned mask, ssize_t* low, ssize_t* high) {
    *low = 0;
    *high = kElmsz[a->type];
    for (int d = 0; d < a->ndim; ++d) {
        if (!(mask >> d & 1)) continue;
        const ssize_t far = a->stride[d] * (ssize_t)(a->shape[d] - 1);
        *(far < 0 ? low : high) += far;
    }
}

// Whether two views can share a byte, b's element at no index lying `ahead` bytes behind a's. Windows of one array often reach across each
// other and share none (its left and its right columns, its even and its odd ones): bytes are compared by what is left of their
// places on division by a stride, to which dimensions of whole multiples of it add nothing. What that does not tell apart is taken to meet.
bool can_meet(const NA* a, unsigned in_a, const NA* b, unsigned in_b, ssize_t ahead, int depth) {
    ssize_t al, ah, bl, bh;
    span(a, in_a, &al, &ah);
    span(b, in_b, &bl, &bh);
    if (ahead + bh <= al || ah <= ahead + bl) return false;
    for (int k = 0; depth > 0 && k < 2 * kMaxDim; ++k) {
        const NA* of = k < kMaxDim ? a : b;
        const int d = k % kMaxDim;
        if (!((k < kMaxDim ? in_a : in_b) >> d & 1)) continue;
        const ssize_t m = of->stride[d] < 0 ? -of->stride[d] : of->stride[d];
        unsigned rest_a = in_a, rest_b = in_b;
        for (int e = 0; e < kMaxDim; ++e) {
            if ((in_a >> e & 1) && a->stride[e] % m == 0) rest_a &= ~(1u << e);
            if ((in_b >> e & 1) && b->stride[e] % m == 0) rest_b &= ~(1u << e);
        }
        span(a, rest_a, &al, &ah);
        span(b, rest_b, &bl, &bh);
        if (ah - al > m || bh - bl > m) continue;
        const ssize_t behind = ((ahead + bl - al) % m + m) % m;   // of b's first byte, from a's, or m less
        const bool here = behind < ah - al && can_meet(a, rest_a, b, rest_b, behind + al - bl, depth - 1);
        const bool there = behind - m + (bh - bl) > 0 && can_meet(a, rest_a, b, rest_b, behind - m + al - bl, depth - 1);
        if (!here && !there) return false;
    }
    return true;
}

bool share(const NA* a, const NA* b) {
    if (!overlap(a, b)) return false;
    unsigned in_a = 0, in_b = 0;   // (dimensions that have somewhere to go)
    for (int d = 0; d < a->ndim; ++d) in_a |= a->shape[d] > 1 && a->stride[d] ? 1u << d : 0;
    for (int d = 0; d < b->ndim; ++d) in_b |= b->shape[d] > 1 && b->stride[d] ? 1u << d : 0;
    return can_meet(a, in_a, b, in_b, (ssize_t)((uintptr_t)b->ptr + (uintptr_t)b->offset - (uintptr_t)a->ptr - (uintptr_t)a->offset), 3);
}

bool aligned(const NA* a) {
    uintptr_t bits = (uintptr_t)a->ptr + (uintptr_t)a->offset;
    for (int d = 0; d < a->ndim; ++d)
        if (a->shape[d] > 1) bits |= (uintptr_t)a->stride[d];
    return bits % (uintptr_t)kElmsz[a->type] == 0;
}

// Dimensions [lo, hi) as one with a single step: false when there is none. No element, or one: step 0.
bool one_step(const NA* a, int lo, int hi, ssize_t* step) {
    size_t n = 1;
    ssize_t st = 0;
    for (int d = hi - 1; d >= lo; --d) {
        if (a->shape[d] == 1) continue;
        if (n == 1) st = a->stride[d];
        else if (a->stride[d] != st * (ssize_t)n) return false;
        n *= a->shape[d];
    }
    *step = st;
    return true;
}

// What a call holds beside its operands and results, given up at its end.
struct Scratch {
    char* held[16];
    int n;
};
void let_go(Scratch* s) {
    for (int k = 0; k < s->n; ++k) scratch_free(s->held[k]);
    s->n = 0;
}

// Layouts: rows whose elements lie side by side, with one step from row to row; elements without gaps; outer x axis x inner
// with a step each.
enum Layout { ROWS, DENSE, AXIS };
bool laid_out(const NA* a, Layout l, int axis, ssize_t* step) {
    if (!aligned(a)) return false;
    if (l == DENSE) return is_contiguous(a);
    if (l == ROWS) return (a->shape[a->ndim - 1] == 1 || a->stride[a->ndim - 1] == kElmsz[a->type]) && one_step(a, 0, a->ndim - 1, step);
    step[1] = a->shape[axis] == 1 ? 0 : a->stride[axis];
    return one_step(a, 0, axis, step) && one_step(a, axis + 1, a->ndim, step + 2);
}

// an operand in the layout that the kernels take: itself, or a copy
struct Operand {
    NA tmp;
    const NA* use;
    const NA* given;
    ssize_t step[3];
    const char* at() const { return use->ptr + use->offset; }
};
int take(Operand* o, const NA* a, Layout l, int axis, Scratch* s) {
    o->given = o->use = a;
    o->step[0] = o->step[1] = o->step[2] = 0;
    if (laid_out(a, l, axis, o->step)) return CUMO_HIP_OK;
    o->tmp.ptr = NULL;
    const int rc = cumo_hip_na_copy(a, &o->tmp);
    if (o->tmp.ptr) s->held[s->n++] = o->tmp.ptr;
    if (rc) return rc;
    o->use = &o->tmp;
    laid_out(o->use, l, axis, o->step);
    return CUMO_HIP_OK;
}

// A result: new, given, or (where the kernels cannot write what is given as it lies) a new one that is copied at the end.
struct Result {
    NA tmp;
    NA* use;
    NA* z;
    bool fresh;
    ssize_t step[3];
    char* at() const { return use->ptr + use->offset; }
};
int check_result(const NA* z, int type, int ndim, const size_t* shape) {
    if (!z) return fail(CUMO_HIP_ERROR_ARGUMENT, "no result descriptor");
    if (!z->ptr) return CUMO_HIP_OK;
    const int rc = check_view(z, "result");
    if (rc) return rc;
    if (z->type != type) return fail(CUMO_HIP_ERROR_TYPE, "result array has the wrong element type");
    if (!same_shape(z, ndim, shape)) return fail(CUMO_HIP_ERROR_SHAPE, "result array has the wrong shape");
    return CUMO_HIP_OK;
}
int make(Result* r, NA* z, int type, int ndim, const size_t* shape, Layout l, int axis, const Operand* o, int n_operands, Scratch* s) {
    r->z = r->use = z;
    r->fresh = z->ptr == NULL;
    r->step[0] = r->step[1] = r->step[2] = 0;
    int rc = CUMO_HIP_OK;
    if (r->fresh) {
        rc = cumo_hip_na_alloc(z, type, ndim, shape);
    } else {
        bool as_given = laid_out(z, l, axis, r->step);
        for (int k = 0; as_given && k < n_operands; ++k) as_given = !o[k].given || !overlap(z, o[k].given);
        if (as_given) return CUMO_HIP_OK;
        rc = cumo_hip_na_alloc(&r->tmp, type, ndim, shape);
        if (r->tmp.ptr) s->held[s->n++] = r->tmp.ptr;
        r->use = &r->tmp;
    }
    if (!rc) laid_out(r->use, l, axis, r->step);
    return rc;
}
// what is left to do with the results once the kernels are queued, or could not be
int finish(int rc, Result* r, int n, Scratch* s) {
    for (int k = 0; !rc && k < n; ++k)
        if (r[k].use != r[k].z) rc = cumo_hip_na_copy(r[k].use, r[k].z);
    if (rc)
        for (int k = 0; k < n; ++k)
            if (r[k].fresh) free_tmp(r[k].z);
    let_go(s);
    return rc;
}

int results_apart(const NA* const* z, int n) {
    for (int a = 0; a < n; ++a)
        for (int b = a + 1; b < n; ++b)
            if (z[a] && z[b] && z[a]->ptr && z[b]->ptr && share(z[a], z[b])) return fail(CUMO_HIP_ERROR_ARGUMENT, "results overlap each other");
    return CUMO_HIP_OK;
}

const char kNormType[] = "rmsnorm: operands are SFloat or DFloat, all of one type";

int norm_operands(const NA* x, const NA* weight, const NA* residual, double eps) {
    int rc = check_float(x, kNormType);
    if (rc) return rc;
    if (x->ndim < 1) return fail(CUMO_HIP_ERROR_DIMENSION, "rmsnorm needs at least one dimension");
    if (!(eps >= 0.0) || std::isinf(eps)) return fail(CUMO_HIP_ERROR_ARGUMENT, "rmsnorm: eps must be a finite number of 0 or more");
    if (weight) {
        rc = check_float(weight, kNormType);
        if (rc) return rc;
        if (weight->type != x->type) return fail(CUMO_HIP_ERROR_TYPE, kNormType);
        if (weight->ndim != 1 || weight->shape[0] != x->shape[x->ndim - 1])
            return fail(CUMO_HIP_ERROR_SHAPE, "rmsnorm: weight must be one dimension, as long as a row");
    }
    if (residual) {
        rc = check_float(residual, kNormType);
        if (rc) return rc;
        if (residual->type != x->type) return fail(CUMO_HIP_ERROR_TYPE, kNormType);
        if (!same_shape(residual, x->ndim, x->shape)) return fail(CUMO_HIP_ERROR_SHAPE, "rmsnorm: residual must have the array's shape");
    }
    return CUMO_HIP_OK;
}

int norm(const NA* x, const NA* weight, const NA* residual, double eps, NA* y, NA* scale, NA* sum) {
    int rc = norm_operands(x, weight, residual, eps);
    if (rc) return rc;
    const int nd = x->ndim;
    const size_t n = x->shape[nd - 1];
    size_t scale_shape[kMaxDim];
    std::memcpy(scale_shape, x->shape, sizeof(size_t) * nd);
    scale_shape[nd - 1] = 1;
    if ((residual != NULL) != (sum != NULL)) return fail(CUMO_HIP_ERROR_ARGUMENT, "rmsnorm: sum is the result of adding a residual");
    rc = check_result(y, scale ? CUMO_HIP_INT8 : x->type, nd, x->shape);
    if (!rc && scale) rc = check_result(scale, x->type, nd, scale_shape);
    if (!rc && sum) rc = check_result(sum, x->type, nd, x->shape);
    const NA* const z[3] = {y, scale, sum};
    if (!rc) rc = results_apart(z, 3);
    if (rc) return rc;

    Scratch s;
    s.n = 0;
    Operand o[3];
    Result r[3];
    int nr = 0;
    o[1].given = o[2].given = NULL;
    rc = take(&o[0], x, ROWS, 0, &s);
    if (!rc && weight) rc = take(&o[1], weight, DENSE, 0, &s);
    if (!rc && residual) rc = take(&o[2], residual, ROWS, 0, &s);
    if (!rc) rc = make(&r[nr++], y, scale ? CUMO_HIP_INT8 : x->type, nd, x->shape, ROWS, 0, o, 3, &s);
    Result *rsum = NULL, *rscale = NULL;
    if (!rc && sum) {
        rsum = &r[nr++];
        rc = make(rsum, sum, x->type, nd, x->shape, ROWS, 0, o, 3, &s);
    }
    if (!rc && scale) {
        rscale = &r[nr++];
        rc = make(rscale, scale, x->type, nd, scale_shape, DENSE, 0, o, 3, &s);
    }
    if (!rc) {
        cumo_hip_rmsnorm_t d;
        std::memset(&d, 0, sizeof(d));
        d.n = n;
        d.rows = 1;
        for (int k = 0; k < nd - 1; ++k) d.rows *= x->shape[k];
        d.x = o[0].at();
        d.x_step = o[0].step[0];
        d.weight = weight ? o[1].at() : NULL;
        d.residual = residual ? o[2].at() : NULL;
        d.residual_step = residual ? o[2].step[0] : 0;
        d.y = r[0].at();
        d.y_step = r[0].step[0];
        if (rsum) {
            d.sum = rsum->at();
            d.sum_step = rsum->step[0];
        }
        if (rscale) d.scale = rscale->at();
        d.eps = eps;
        if (d.rows && n) cumo_hip_rmsnorm_kernel_launch(x->type, scale ? 1 : 0, &d);
        else if (d.rows && rscale) rc = cumo_hip_na_fill(rscale->use, 0.0);  // (rows of no elements still have a scale)
    }
    return finish(rc, r, nr, &s);
}

}  // namespace

extern "C" {

int cumo_hip_na_rmsnorm(const cumo_hip_narray_t* x, const cumo_hip_narray_t* weight, const cumo_hip_narray_t* residual, double eps,
                        cumo_hip_narray_t* y, cumo_hip_narray_t* sum) {
    return norm(x, weight, residual, eps, y, NULL, sum);
}

int cumo_hip_na_rmsnorm_q8(const cumo_hip_narray_t* x, const cumo_hip_narray_t* weight, const cumo_hip_narray_t* residual, double eps,
                           cumo_hip_narray_t* q, cumo_hip_narray_t* scale, cumo_hip_narray_t* sum) {
    if (!scale) return fail(CUMO_HIP_ERROR_ARGUMENT, "no result descriptor");
    return norm(x, weight, residual, eps, q, scale, sum);
}

int cumo_hip_na_dequantize(const cumo_hip_narray_t* q, const cumo_hip_narray_t* scale, cumo_hip_narray_t* y) {
    int rc = check_view(q, "operand");
    if (!rc) rc = check_float(scale, "dequantize: scale is SFloat or DFloat");
    if (rc) return rc;
    if (q->type != CUMO_HIP_INT8) return fail(CUMO_HIP_ERROR_TYPE, "dequantize: the array is not Int8");
    const int nd = q->ndim;
    if (nd < 1) return fail(CUMO_HIP_ERROR_DIMENSION, "dequantize needs at least one dimension");
    size_t want[kMaxDim];
    std::memcpy(want, q->shape, sizeof(size_t) * nd);
    want[nd - 1] = 1;
    if (!same_shape(scale, nd, want)) return fail(CUMO_HIP_ERROR_SHAPE, "dequantize: scale must have the array's shape with a last dimension of 1");
    rc = check_result(y, scale->type, nd, q->shape);
    if (rc) return rc;
    Scratch s;
    s.n = 0;
    Operand o[2];
    o[1].given = NULL;
    Result r;
    int nr = 0;
    rc = take(&o[0], q, ROWS, 0, &s);
    if (!rc) rc = take(&o[1], scale, DENSE, 0, &s);
    if (!rc) rc = make(&r, y, scale->type, nd, q->shape, ROWS, 0, o, 2, &s), nr = 1;
    if (!rc && total_of(q)) {
        cumo_hip_dequantize_t d;
        d.n = q->shape[nd - 1];
        d.rows = total_of(scale);
        d.q = o[0].at();
        d.q_step = o[0].step[0];
        d.scale = o[1].at();
        d.y = r.at();
        d.y_step = r.step[0];
        cumo_hip_dequantize_kernel_launch(scale->type, &d);
    }
    return finish(rc, &r, nr, &s);
}

int cumo_hip_na_rmsnorm_grad(const cumo_hip_narray_t* g, const cumo_hip_narray_t* s, const cumo_hip_narray_t* weight,
                             const cumo_hip_narray_t* gsum, double eps, cumo_hip_narray_t* gx, cumo_hip_narray_t* gweight) {
    int rc = norm_operands(g, weight, s, eps);
    if (rc) return rc;
    if (!s) return fail(CUMO_HIP_ERROR_ARGUMENT, "rmsnorm_grad: missing array argument");
    rc = norm_operands(g, NULL, gsum, eps);
    if (rc) return rc;
    if ((weight != NULL) != (gweight != NULL)) return fail(CUMO_HIP_ERROR_ARGUMENT, "rmsnorm_grad: gweight is the gradient of weight");
    const int nd = g->ndim;
    rc = check_result(gx, g->type, nd, g->shape);
    if (!rc && gweight) rc = check_result(gweight, g->type, 1, &g->shape[nd - 1]);
    const NA* const z[2] = {gx, gweight};
    if (!rc) rc = results_apart(z, 2);
    if (rc) return rc;

    Scratch sc;
    sc.n = 0;
    Operand o[4];
    o[1].given = o[2].given = o[3].given = NULL;
    Result r[2];
    int nr = 0;
    rc = take(&o[0], g, ROWS, 0, &sc);
    if (!rc) rc = take(&o[1], s, ROWS, 0, &sc);
    if (!rc && weight) rc = take(&o[2], weight, DENSE, 0, &sc);
    if (!rc && gsum) rc = take(&o[3], gsum, ROWS, 0, &sc);
    if (!rc) rc = make(&r[nr++], gx, g->type, nd, g->shape, ROWS, 0, o, 4, &sc);
    if (!rc && gweight) rc = make(&r[nr++], gweight, g->type, 1, &g->shape[nd - 1], DENSE, 0, o, 4, &sc);
    if (!rc && g->shape[nd - 1]) {
        cumo_hip_rmsnorm_grad_t d;
        std::memset(&d, 0, sizeof(d));
        d.n = g->shape[nd - 1];
        d.rows = 1;
        for (int k = 0; k < nd - 1; ++k) d.rows *= g->shape[k];
        d.g = o[0].at();
        d.g_step = o[0].step[0];
        d.s = o[1].at();
        d.s_step = o[1].step[0];
        d.weight = weight ? o[2].at() : NULL;
        d.gsum = gsum ? o[3].at() : NULL;
        d.gsum_step = gsum ? o[3].step[0] : 0;
        d.gx = r[0].at();
        d.gx_step = r[0].step[0];
        d.gweight = gweight ? r[1].at() : NULL;
        d.eps = eps;
        rc = cumo_hip_rmsnorm_grad_kernel_launch(g->type, &d);  // (no rows: the weight's gradient is 0)
    }
    return finish(rc, r, nr, &sc);
}

}  // extern "C"

namespace {

const char kRecurrenceType[] = "recurrence: operands are SFloat or DFloat, all of one type";

// a: any of the operands of the full shape; the others as the first says
int recurrence_operands(const NA* const* full, int n, const NA* h0, int axis, size_t* state_shape) {
    for (int k = 0; k < n; ++k) {
        const int rc = check_float(full[k], kRecurrenceType);
        if (rc) return rc;
        if (full[k]->type != full[0]->type) return fail(CUMO_HIP_ERROR_TYPE, kRecurrenceType);
        if (!same_shape(full[k], full[0]->ndim, full[0]->shape)) return fail(CUMO_HIP_ERROR_SHAPE, "recurrence: the arrays must have one shape");
    }
    const int nd = full[0]->ndim;
    if (axis < 0 || axis >= nd) return fail(CUMO_HIP_ERROR_DIMENSION, "dimension is out of range");
    for (int d = 0, k = 0; d < nd; ++d)
        if (d != axis) state_shape[k++] = full[0]->shape[d];
    if (h0) {
        const int rc = check_float(h0, kRecurrenceType);
        if (rc) return rc;
        if (h0->type != full[0]->type) return fail(CUMO_HIP_ERROR_TYPE, kRecurrenceType);
        if (!same_rows(h0, nd - 1, state_shape)) return fail(CUMO_HIP_ERROR_SHAPE, "recurrence: h0 must have the array's shape without the axis");
    }
    return CUMO_HIP_OK;
}

void axis_sizes(const NA* a, int axis, uint64_t* outer, uint64_t* time, uint64_t* inner) {
    *outer = *inner = 1;
    for (int d = 0; d < axis; ++d) *outer *= a->shape[d];
    for (int d = axis + 1; d < a->ndim; ++d) *inner *= a->shape[d];
    *time = a->shape[axis];
}

}  // namespace

extern "C" {

int cumo_hip_na_recurrence(const cumo_hip_narray_t* a, const cumo_hip_narray_t* b, const cumo_hip_narray_t* h0, int axis, cumo_hip_narray_t* h) {
    const NA* const full[2] = {a, b};
    size_t state_shape[kMaxDim];
    int rc = recurrence_operands(full, 2, h0, axis, state_shape);
    if (!rc) rc = check_result(h, a->type, a->ndim, a->shape);
    if (rc) return rc;
    Scratch s;
    s.n = 0;
    Operand o[3];
    o[1].given = o[2].given = NULL;
    Result r;
    int nr = 0;
    rc = take(&o[0], a, AXIS, axis, &s);
    if (!rc) rc = take(&o[1], b, AXIS, axis, &s);
    if (!rc && h0) rc = take(&o[2], h0, DENSE, 0, &s);
    if (!rc) rc = make(&r, h, a->type, a->ndim, a->shape, AXIS, axis, o, 3, &s), nr = 1;
    if (!rc && total_of(a)) {
        cumo_hip_recurrence_t d;
        axis_sizes(a, axis, &d.outer, &d.time, &d.inner);
        std::memcpy(d.a_step, o[0].step, sizeof(d.a_step));
        std::memcpy(d.b_step, o[1].step, sizeof(d.b_step));
        std::memcpy(d.h_step, r.step, sizeof(d.h_step));
        d.a = o[0].at();
        d.b = o[1].at();
        d.h0 = h0 ? o[2].at() : NULL;
        d.h = r.at();
        rc = cumo_hip_recurrence_kernel_launch(a->type, &d);
    }
    return finish(rc, &r, nr, &s);
}

int cumo_hip_na_recurrence_grad(const cumo_hip_narray_t* g, const cumo_hip_narray_t* a, const cumo_hip_narray_t* h,
                                const cumo_hip_narray_t* h0, int axis, cumo_hip_narray_t* ga, cumo_hip_narray_t* gb, cumo_hip_narray_t* gh0) {
    const NA* const full[3] = {g, a, h};
    size_t state_shape[kMaxDim];
    int rc = recurrence_operands(full, 3, h0, axis, state_shape);
    if (rc) return rc;
    if ((h0 != NULL) != (gh0 != NULL)) return fail(CUMO_HIP_ERROR_ARGUMENT, "recurrence_grad: gh0 is the gradient of h0");
    rc = check_result(ga, g->type, g->ndim, g->shape);
    if (!rc) rc = check_result(gb, g->type, g->ndim, g->shape);
    if (!rc && gh0) rc = check_result(gh0, g->type, h0->ndim, h0->shape);
    const NA* const z[3] = {ga, gb, gh0};
    if (!rc) rc = results_apart(z, 3);
    if (rc) return rc;
    Scratch s;
    s.n = 0;
    Operand o[4];
    o[1].given = o[2].given = o[3].given = NULL;
    Result r[3];
    int nr = 0;
    rc = take(&o[0], g, AXIS, axis, &s);
    if (!rc) rc = take(&o[1], a, AXIS, axis, &s);
    if (!rc) rc = take(&o[2], h, AXIS, axis, &s);
    if (!rc && h0) rc = take(&o[3], h0, DENSE, 0, &s);
    if (!rc) rc = make(&r[nr++], ga, g->type, g->ndim, g->shape, AXIS, axis, o, 4, &s);
    if (!rc) rc = make(&r[nr++], gb, g->type, g->ndim, g->shape, AXIS, axis, o, 4, &s);
    if (!rc && gh0) rc = make(&r[nr++], gh0, g->type, h0->ndim, h0->shape, DENSE, 0, o, 4, &s);
    if (!rc) {
        cumo_hip_recurrence_grad_t d;
        axis_sizes(g, axis, &d.outer, &d.time, &d.inner);
        std::memcpy(d.g_step, o[0].step, sizeof(d.g_step));
        std::memcpy(d.a_step, o[1].step, sizeof(d.a_step));
        std::memcpy(d.h_step, o[2].step, sizeof(d.h_step));
        std::memcpy(d.ga_step, r[0].step, sizeof(d.ga_step));
        std::memcpy(d.gb_step, r[1].step, sizeof(d.gb_step));
        d.g = o[0].at();
        d.a = o[1].at();
        d.h = o[2].at();
        d.h0 = h0 ? o[3].at() : NULL;
        d.ga = r[0].at();
        d.gb = r[1].at();
        d.gh0 = gh0 ? r[2].at() : NULL;
        if (total_of(g)) rc = cumo_hip_recurrence_grad_kernel_launch(g->type, &d);
        else if (gh0 && total_of(gh0)) rc = cumo_hip_na_fill(r[2].use, 0.0);  // (no steps: the state reaches nothing)
    }
    return finish(rc, r, nr, &s);
}

int cumo_hip_na_sample(const cumo_hip_narray_t* x, const cumo_hip_narray_t* u, double temperature, const cumo_hip_narray_t* temperatures,
                       ssize_t top_k, const cumo_hip_narray_t* top_ks, double top_p, const cumo_hip_narray_t* top_ps,
                       double min_p, const cumo_hip_narray_t* min_ps, cumo_hip_narray_t* z) {
    int rc = check_float(x, "sample: the logits are not SFloat or DFloat");
    if (!rc) rc = check_float(u, "sample: u is not SFloat or DFloat");
    if (rc) return rc;
    if (x->ndim < 1) return fail(CUMO_HIP_ERROR_DIMENSION, "sample needs at least one dimension");
    const int nd = x->ndim - 1;
    const NA* const each[5] = {u, temperatures, top_ks, top_ps, min_ps};
    for (int k = 0; k < 5; ++k) {
        if (!each[k]) continue;
        rc = check_view(each[k], "operand");
        if (rc) return rc;
        if (k == 2 ? each[k]->type != CUMO_HIP_INT32 : !is_float(each[k]->type))
            return fail(CUMO_HIP_ERROR_TYPE, "sample: settings of rows are SFloat or DFloat, top_k Int32");
        if (!same_rows(each[k], nd, x->shape)) return fail(CUMO_HIP_ERROR_SHAPE, "sample: u and settings of rows must have the logits' shape without the last dimension");
    }
    if (!temperatures && !(temperature >= 0.0)) return fail(CUMO_HIP_ERROR_ARGUMENT, "sample: temperature must be 0 or more");
    if (!top_ks && top_k < 0) return fail(CUMO_HIP_ERROR_ARGUMENT, "sample: top_k must be 0 or more");
    if (!top_ps && !(top_p >= 0.0 && top_p <= 1.0)) return fail(CUMO_HIP_ERROR_ARGUMENT, "sample: top_p must be from 0 to 1");
    if (!min_ps && !(min_p >= 0.0 && min_p <= 1.0)) return fail(CUMO_HIP_ERROR_ARGUMENT, "sample: min_p must be from 0 to 1");
    if (x->shape[nd] > (size_t)INT32_MAX) return fail(CUMO_HIP_ERROR_ARGUMENT, "sample: rows are too long for Int32 positions");
    rc = check_result(z, CUMO_HIP_INT32, nd, x->shape);
    if (rc) return rc;
    Scratch s;
    s.n = 0;
    Operand o[6];
    for (int k = 1; k < 6; ++k) o[k].given = NULL;
    Result r;
    int nr = 0;
    rc = take(&o[0], x, ROWS, 0, &s);
    for (int k = 0; !rc && k < 5; ++k)
        if (each[k]) rc = take(&o[1 + k], each[k], DENSE, 0, &s);
    if (!rc) rc = make(&r, z, CUMO_HIP_INT32, nd, x->shape, DENSE, 0, o, 6, &s), nr = 1;
    if (!rc) {
        cumo_hip_sample_t d;
        d.rows = total_of(r.use);
        d.n = x->shape[nd];
        d.x = o[0].at();
        d.x_step = o[0].step[0];
        cumo_hip_row_number_t* const to[5] = {&d.u, &d.temperature, &d.top_k, &d.top_p, &d.min_p};
        const double value[5] = {0.0, temperature, (double)top_k, top_p, min_p};
        for (int k = 0; k < 5; ++k) {
            to[k]->each = each[k] ? o[1 + k].at() : NULL;
            to[k]->type = each[k] ? each[k]->type : CUMO_HIP_DFLOAT;
            to[k]->value = value[k];
        }
        d.out = (int32_t*)r.at();
        if (d.rows) rc = cumo_hip_sample_kernel_launch(x->type, &d);
    }
    return finish(rc, &r, nr, &s);
}

}  // extern "C"

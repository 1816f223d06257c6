// Views as the host layer's functions look at them: element sizes, the checks that come first, temporaries.
#ifndef CUMO_HIP_NDLOOP_VIEWS_H
#define CUMO_HIP_NDLOOP_VIEWS_H

#include "common.h"
#include "cumo_hip_ndloop.h"

namespace cumo_hip {

typedef cumo_hip_narray_t NA;

static const int kElmsz[CUMO_HIP_N_TYPES] = {4, 8, 4, 8, 8, 0, 1};
static const int kMaxDim = CUMO_NA_MAX_DIMENSION;

inline int fail(int kind, const char* msg) {
    report_error(kind, 0, msg);
    return kind;
}

inline bool valid_type(int t) { return t >= 0 && t < CUMO_HIP_N_TYPES; }
inline bool is_arith(int t) { return t == CUMO_HIP_SFLOAT || t == CUMO_HIP_DFLOAT || t == CUMO_HIP_INT32; }
inline bool is_float(int t) { return t == CUMO_HIP_SFLOAT || t == CUMO_HIP_DFLOAT; }

inline size_t total_of(const NA* a) {
    size_t n = 1;
    for (int d = 0; d < a->ndim; d++) n *= a->shape[d];
    return n;
}

// a view whose elements sit in row-major order without gaps (any offset)
inline bool is_contiguous(const NA* a) {
    ssize_t unit = a->type == CUMO_HIP_BIT ? 1 : kElmsz[a->type];
    ssize_t s = unit;
    for (int d = a->ndim - 1; d >= 0; d--) {
        if (a->shape[d] != 1 && a->stride[d] != s) return false;
        s *= (ssize_t)a->shape[d];
    }
    return true;
}

inline int check_view(const NA* a, const char* what) {
    if (!a) return fail(CUMO_HIP_ERROR_ARGUMENT, "ndloop: missing array argument");
    if (!valid_type(a->type)) return fail(CUMO_HIP_ERROR_TYPE, "ndloop: unknown element type");
    if (a->ndim < 0 || a->ndim > kMaxDim) return fail(CUMO_HIP_ERROR_DIMENSION, "ndloop: too many dimensions");
    if (a->type == CUMO_HIP_BIT && a->offset < 0) return fail(CUMO_HIP_ERROR_ARGUMENT, "ndloop: negative bit offset");
    (void)what;
    return CUMO_HIP_OK;
}

inline void free_tmp(NA* t) {
    if (t->ptr) {
        cumo_cuda_runtime_free(t->ptr);
        t->ptr = NULL;
    }
}

}  // namespace cumo_hip

#endif

// Linear attention with a decay for each head, S[t] = a S[t-1] + k[t] (x) v[t], o[t] = scale (S[t] by q[t]), and its gradients.
//
// A walk is this: from q, k (of `dim` elements) and v, o (of `wide`), forwards or backwards in time. With G[t] what the loss has for S[t],
// G[t] = a G[t+1] + scale q[t] (x) g[t], the gradients are three walks more:
//   gq[t] = scale (S[t] by g[t]):  g in the place of q, v of k, k of v, the state transposed
//   gk[t] = G[t] by v[t]:          backwards, v in the place of q, scale g of k, q of v, the state transposed
//   gv[t] = G[t] by k[t]:          backwards, k in the place of q, scale q of k, g of v
// Backwards the state decays behind a step instead of before it (`late`): what is handed on is a G.
#include "common.h"

namespace cumo_hip {
namespace {

struct LaWalk {
    const char *q, *k, *v, *state;
    char *o, *last;                            // last: NULL, not wanted
    int64_t q_step[3], k_step[3], v_step[3], o_step[3];  // bytes: sequence, step, head
    uint32_t q_share, k_share, v_share;        // heads of the walk to one of the array
    uint32_t dim, wide;
    uint32_t state_row, state_col;             // elements from S's row to row (of dim), column to column
    double o_scale, k_scale;
    bool backwards;                            // and late
};
struct LaCommon {
    uint64_t batch, time, heads;
    const char* decay;
    const int32_t* lengths;
};

template <class T> __device__ __forceinline__ T la_fma(T a, T b, T c);
template <> __device__ __forceinline__ float la_fma(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
template <> __device__ __forceinline__ double la_fma(double a, double b, double c) { return __builtin_fma(a, b, c); }

__device__ __forceinline__ uint64_t la_length(const LaCommon& c, uint64_t b) {
    if (!c.lengths) return c.time;
    const int64_t n = c.lengths[b];
    return n < 0 ? 0 : (uint64_t)n < c.time ? (uint64_t)n : c.time;
}

// One step after the other. LPR lanes hold VE columns each of a row of S, the block's other lanes other rows; S goes through memory from
// step to step (`memory`: last, or scratch), which every lane reads as it wrote it.
constexpr int kLaStepBlock = 256;
template <class T, int VE, int LPR>
__global__ __launch_bounds__(kLaStepBlock) void la_step_kernel(LaWalk w, LaCommon c, char* memory, uint32_t slices) {
    constexpr int RG = kLaStepBlock / LPR;
    __shared__ T part[kLaStepBlock * VE];
    const uint64_t which = blockIdx.x / slices, b = which / c.heads, h = which - b * c.heads;
    const uint32_t lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
    const uint32_t e = ((uint32_t)(blockIdx.x % slices) * LPR + lane) * VE;
    const bool there = e < w.wide;
    const uint64_t length = la_length(c, b), size = (uint64_t)w.dim * w.wide;
    const T a = reinterpret_cast<const T*>(c.decay)[h];
    const T *from = w.state ? reinterpret_cast<const T*>(w.state) + which * size : nullptr;
    T* to = memory ? reinterpret_cast<T*>(memory) + which * size : nullptr;
    const char* q = w.q + (int64_t)b * w.q_step[0] + (int64_t)(h / w.q_share) * w.q_step[2];
    const char* k = w.k + (int64_t)b * w.k_step[0] + (int64_t)(h / w.k_share) * w.k_step[2];
    const char* v = w.v + (int64_t)b * w.v_step[0] + (int64_t)(h / w.v_share) * w.v_step[2];
    char* o = w.o + (int64_t)b * w.o_step[0] + (int64_t)h * w.o_step[2];
    for (uint64_t n = 0; n < length; ++n) {
        const uint64_t t = w.backwards ? length - 1 - n : n;
        const T* qt = reinterpret_cast<const T*>(q + (int64_t)t * w.q_step[1]);
        const T* kt = reinterpret_cast<const T*>(k + (int64_t)t * w.k_step[1]);
        const T* vt = reinterpret_cast<const T*>(v + (int64_t)t * w.v_step[1]);
        T sum[VE], vv[VE];
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            sum[j] = (T)0;
            vv[j] = there ? vt[e + j] : (T)0;
        }
        if (there) {
#pragma unroll 4
            for (uint32_t d = group; d < w.dim; d += RG) {
                const uint64_t at = (uint64_t)d * w.state_row + (uint64_t)e * w.state_col;
                const T kd = kt[d] * (T)w.k_scale, qd = qt[d];
#pragma unroll
                for (int j = 0; j < VE; ++j) {
                    const uint64_t here = at + (uint64_t)j * w.state_col;
                    T s = from ? from[here] : (T)0;
                    s = w.backwards ? la_fma(kd, vv[j], s) : la_fma(kd, vv[j], a * s);
                    sum[j] = la_fma(qd, s, sum[j]);
                    if (to) to[here] = w.backwards ? a * s : s;
                }
            }
        }
        from = to;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < VE; ++j) part[threadIdx.x * VE + j] = sum[j];
        __syncthreads();
        if (group == 0 && there) {
            T* ot = reinterpret_cast<T*>(o + (int64_t)t * w.o_step[1]);
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                T all = (T)0;
                for (int g = 0; g < RG; ++g) all += part[(g * LPR + lane) * VE + j];
                ot[e + j] = all * (T)w.o_scale;
            }
        }
    }
    if (length == 0 && to && there) {
        for (uint32_t d = group; d < w.dim; d += RG) {
            const uint64_t at = (uint64_t)d * w.state_row + (uint64_t)e * w.state_col;
            for (int j = 0; j < VE; ++j) to[at + (uint64_t)j * w.state_col] = from ? from[at + (uint64_t)j * w.state_col] : (T)0;
        }
    }
    if (there && group == 0)
        for (uint64_t t = length; t < c.time; ++t)
            for (int j = 0; j < VE; ++j) reinterpret_cast<T*>(o + (int64_t)t * w.o_step[1])[e + j] = (T)0;
}

template <class T, int VE, int LPR>
void la_step_one(const LaWalk& w, const LaCommon& c, char* memory, hipStream_t stream) {
    const uint32_t slices = (w.wide + LPR * VE - 1) / (LPR * VE);
    hipLaunchKernelGGL((la_step_kernel<T, VE, LPR>), dim3((unsigned)(c.batch * c.heads * slices)), dim3(kLaStepBlock), 0, stream, w, c, memory, slices);
}

template <class T>
void la_step(const LaWalk& w, const LaCommon& c, char* memory, hipStream_t stream) {
    constexpr int V = 16 / (int)sizeof(T);
    if (w.wide % V == 0) {
        if (w.wide <= 16 * V) la_step_one<T, V, 16>(w, c, memory, stream);
        else if (w.wide <= 32 * V) la_step_one<T, V, 32>(w, c, memory, stream);
        else la_step_one<T, V, 64>(w, c, memory, stream);
    } else {
        if (w.wide <= 16) la_step_one<T, 1, 16>(w, c, memory, stream);
        else la_step_one<T, 1, 64>(w, c, memory, stream);
    }
}

template <class T>
int la_walk(const LaWalk& w, const LaCommon& c, hipStream_t stream) {
    char* memory = w.last;
    char* scratch = nullptr;
    if (!memory && c.time > 1 && w.dim) {
        scratch = cumo_cuda_runtime_malloc(c.batch * c.heads * w.dim * w.wide * sizeof(T));
        if (!scratch) return CUMO_HIP_ERROR_OUT_OF_MEMORY;
        memory = scratch;
    }
    la_step<T>(w, c, memory, stream);
    cumo_cuda_runtime_check_kernel_launch();
    if (scratch) scratch_free(scratch);
    return CUMO_HIP_OK;
}

// [batch, time, shared, group, n] contiguous into [batch, time, shared, n] with steps: the heads that share an array's head, in their order
template <class T>
__global__ __launch_bounds__(256) void la_share_kernel(const T* x, char* y, uint64_t batch, uint64_t time, uint64_t shared, uint32_t group, uint32_t n, int64_t y0, int64_t y1,
                                                       int64_t y2) {
    const uint64_t total = batch * time * shared * n;
    for (uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x; at < total; at += (uint64_t)gridDim.x * 256) {
        const uint64_t row = at / n, i = at - row * n, bt = row / shared, h = row - bt * shared, b = bt / time, t = bt - b * time;
        const T* from = x + row * group * n + i;
        T sum = from[0];
        for (uint32_t g = 1; g < group; ++g) sum += from[(uint64_t)g * n];
        reinterpret_cast<T*>(y + (int64_t)b * y0 + (int64_t)t * y1 + (int64_t)h * y2)[i] = sum;
    }
}

void la_steps(int64_t* to, const ssize_t* from) {
    for (int k = 0; k < 3; ++k) to[k] = from[k];
}

template <class T>
int la_forward(const cumo_hip_linear_attention_t& d, hipStream_t stream) {
    LaCommon c = {d.batch, d.time, d.heads, d.decay, d.lengths};
    LaWalk w;
    const uint32_t share = (uint32_t)(d.heads / d.shared);
    w.q = d.q, w.k = d.k, w.v = d.v, w.state = d.state, w.o = d.o, w.last = d.last;
    la_steps(w.q_step, d.q_step), la_steps(w.k_step, d.k_step), la_steps(w.v_step, d.v_step), la_steps(w.o_step, d.o_step);
    w.q_share = 1, w.k_share = w.v_share = share;
    w.dim = (uint32_t)d.dim, w.wide = (uint32_t)d.wide;
    w.state_row = w.wide, w.state_col = 1;
    w.o_scale = d.scale, w.k_scale = 1.0;
    w.backwards = false;
    return la_walk<T>(w, c, stream);
}

template <class T>
int la_backward(const cumo_hip_linear_attention_grad_t& d, hipStream_t stream) {
    LaCommon c = {d.batch, d.time, d.heads, d.decay, d.lengths};
    const uint32_t share = (uint32_t)(d.heads / d.shared), dim = (uint32_t)d.dim, wide = (uint32_t)d.wide;
    const uint64_t rows = d.batch * d.time * d.heads;
    // gradients of heads that are shared, before their sum
    char* parts = nullptr;
    if (share > 1 && !(parts = cumo_cuda_runtime_malloc(rows * (dim + wide) * sizeof(T)))) return CUMO_HIP_ERROR_OUT_OF_MEMORY;
    char* const part_k = parts;
    char* const part_v = parts ? parts + rows * dim * sizeof(T) : nullptr;
    const int64_t e = sizeof(T), heads = (int64_t)d.heads, time = (int64_t)d.time;
    LaWalk w;
    int rc = CUMO_HIP_OK;
    if (dim) {
        // gq
        w.q = d.g, w.k = d.v, w.v = d.k, w.state = d.state, w.o = d.gq, w.last = nullptr;
        la_steps(w.q_step, d.g_step), la_steps(w.k_step, d.v_step), la_steps(w.v_step, d.k_step), la_steps(w.o_step, d.gq_step);
        w.q_share = 1, w.k_share = w.v_share = share;
        w.dim = wide, w.wide = dim, w.state_row = 1, w.state_col = wide;
        w.o_scale = d.scale, w.k_scale = 1.0, w.backwards = false;
        rc = la_walk<T>(w, c, stream);
        if (!rc) {
            // gk
            w.q = d.v, w.k = d.g, w.v = d.q, w.state = d.glast;
            la_steps(w.q_step, d.v_step), la_steps(w.k_step, d.g_step), la_steps(w.v_step, d.q_step), la_steps(w.o_step, d.gk_step);
            w.o = d.gk;
            if (parts) w.o = part_k, w.o_step[0] = time * heads * dim * e, w.o_step[1] = heads * dim * e, w.o_step[2] = dim * e;
            w.q_share = share, w.k_share = w.v_share = 1;
            w.o_scale = 1.0, w.k_scale = d.scale, w.backwards = true;
            rc = la_walk<T>(w, c, stream);
        }
    }
    if (!rc && wide) {
        // gv
        w.q = d.k, w.k = d.q, w.v = d.g, w.state = d.glast, w.last = d.gstate;
        la_steps(w.q_step, d.k_step), la_steps(w.k_step, d.q_step), la_steps(w.v_step, d.g_step), la_steps(w.o_step, d.gv_step);
        w.o = d.gv;
        if (parts) w.o = part_v, w.o_step[0] = time * heads * wide * e, w.o_step[1] = heads * wide * e, w.o_step[2] = wide * e;
        w.q_share = share, w.k_share = w.v_share = 1;
        w.dim = dim, w.wide = wide, w.state_row = wide, w.state_col = 1;
        w.o_scale = 1.0, w.k_scale = d.scale, w.backwards = true;
        rc = la_walk<T>(w, c, stream);
    }
    if (!rc && parts) {
        for (int k = 0; k < 2; ++k) {
            const uint32_t n = k ? wide : dim;
            const uint64_t blocks = (d.batch * d.time * d.shared * n + 255) / 256;
            const ssize_t* step = k ? d.gv_step : d.gk_step;
            if (blocks)
                hipLaunchKernelGGL((la_share_kernel<T>), dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, stream, reinterpret_cast<const T*>(k ? part_v : part_k),
                                   k ? d.gv : d.gk, d.batch, d.time, d.shared, share, n, step[0], step[1], step[2]);
        }
        cumo_cuda_runtime_check_kernel_launch();
    }
    if (parts) scratch_free(parts);
    return rc;
}

}  // namespace
}  // namespace cumo_hip

using namespace cumo_hip;

extern "C" int cumo_hip_linear_attention_kernel_launch(int type, const cumo_hip_linear_attention_t* d) {
    return type == 0 ? la_forward<float>(*d, current_stream()) : la_forward<double>(*d, current_stream());
}

extern "C" int cumo_hip_linear_attention_grad_kernel_launch(int type, const cumo_hip_linear_attention_grad_t* d) {
    return type == 0 ? la_backward<float>(*d, current_stream()) : la_backward<double>(*d, current_stream());
}

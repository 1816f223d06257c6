// Root-mean-square normalisation of rows, with the addition of a residual before it, an 8-bit form of the result and the
// gradients:
//   s = x + residual        r = 1 / sqrt(sum(s^2) / n + eps)        y = s r w
//   c = r^2 sum(g w s) / n  gx = r (g w - s c) + gsum               gw = sum over rows of g s r
// (gx: with u = s r the derivative of u_i by s_j is r (delta_ij - u_i u_j / n).)
#include "common.h"

namespace cumo_hip {
namespace {

constexpr int kRnBlock = 256;

__device__ __forceinline__ double rn_shfl_xor(double v, int m) { return __shfl_xor(v, m); }

template <class F>
__device__ __forceinline__ double rn_allreduce(double v, F f) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v = f(v, rn_shfl_xor(v, m));
    __shared__ double slot[kRnBlock / 64];
    __syncthreads();  // the slots may still be read from the previous use
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
    __syncthreads();
    v = slot[0];
#pragma unroll
    for (int w = 1; w < kRnBlock / 64; ++w) v = f(v, slot[w]);
    return v;
}
__device__ __forceinline__ double rn_add(double a, double b) { return a + b; }
__device__ __forceinline__ double rn_max_nan(double a, double b) { return (a != a) ? a : ((b != b) ? b : (a > b ? a : b)); }

template <class T, bool Q8>
__global__ __launch_bounds__(kRnBlock) void rmsnorm_kernel(cumo_hip_rmsnorm_t p) {
    for (uint64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = reinterpret_cast<const T*>(p.x + (int64_t)row * p.x_step);
        const T* res = p.residual ? reinterpret_cast<const T*>(p.residual + (int64_t)row * p.residual_step) : nullptr;
        const T* w = reinterpret_cast<const T*>(p.weight);
        T* sum = p.sum ? reinterpret_cast<T*>(p.sum + (int64_t)row * p.sum_step) : nullptr;
        double q = 0.0;
        for (uint64_t i = threadIdx.x; i < p.n; i += kRnBlock) {
            const T s = res ? x[i] + res[i] : x[i];
            if (sum) sum[i] = s;
            q = __builtin_fma((double)s, (double)s, q);
        }
        const double r = 1.0 / sqrt(rn_allreduce(q, rn_add) / (double)p.n + p.eps);
        const T* from = sum ? sum : x;
        auto value = [&](uint64_t i) { return (double)from[i] * r * (w ? (double)w[i] : 1.0); };
        if constexpr (Q8) {
            double most = 0.0;
            for (uint64_t i = threadIdx.x; i < p.n; i += kRnBlock) most = rn_max_nan(most, fabs(value(i)));
            most = rn_allreduce(most, rn_max_nan);
            const T scale = (T)(most / 127.0);
            if (threadIdx.x == 0) reinterpret_cast<T*>(p.scale)[row] = scale;
            int8_t* y = reinterpret_cast<int8_t*>(p.y + (int64_t)row * p.y_step);
            for (uint64_t i = threadIdx.x; i < p.n; i += kRnBlock) {
                const double z = rint(value(i) / (double)scale);
                y[i] = scale > (T)0 ? (int8_t)(z > 127.0 ? 127.0 : (z < -127.0 ? -127.0 : (z == z ? z : 0.0))) : (int8_t)0;
            }
        } else {
            T* y = reinterpret_cast<T*>(p.y + (int64_t)row * p.y_step);
            for (uint64_t i = threadIdx.x; i < p.n; i += kRnBlock) y[i] = (T)value(i);
        }
    }
}

template <class T>
__global__ __launch_bounds__(kRnBlock) void dequantize_kernel(cumo_hip_dequantize_t p) {
    const uint64_t total = p.rows * p.n;
    for (uint64_t at = (uint64_t)blockIdx.x * kRnBlock + threadIdx.x; at < total; at += (uint64_t)gridDim.x * kRnBlock) {
        const uint64_t row = at / p.n, i = at - row * p.n;
        reinterpret_cast<T*>(p.y + (int64_t)row * p.y_step)[i] =
            (T)reinterpret_cast<const int8_t*>(p.q + (int64_t)row * p.q_step)[i] * reinterpret_cast<const T*>(p.scale)[row];
    }
}

// the rows' gradients; r of each row is left for the weight's
template <class T>
__global__ __launch_bounds__(kRnBlock) void rmsnorm_grad_kernel(cumo_hip_rmsnorm_grad_t p, double* rs) {
    for (uint64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* g = reinterpret_cast<const T*>(p.g + (int64_t)row * p.g_step);
        const T* s = reinterpret_cast<const T*>(p.s + (int64_t)row * p.s_step);
        const T* gs = p.gsum ? reinterpret_cast<const T*>(p.gsum + (int64_t)row * p.gsum_step) : nullptr;
        const T* w = reinterpret_cast<const T*>(p.weight);
        T* gx = reinterpret_cast<T*>(p.gx + (int64_t)row * p.gx_step);
        double q = 0.0, c = 0.0;
        for (uint64_t i = threadIdx.x; i < p.n; i += kRnBlock) {
            const double si = (double)s[i], gw = (double)g[i] * (w ? (double)w[i] : 1.0);
            q = __builtin_fma(si, si, q);
            c = __builtin_fma(gw, si, c);
        }
        const double r = 1.0 / sqrt(rn_allreduce(q, rn_add) / (double)p.n + p.eps);
        c = r * r * rn_allreduce(c, rn_add) / (double)p.n;
        if (rs && threadIdx.x == 0) rs[row] = r;
        for (uint64_t i = threadIdx.x; i < p.n; i += kRnBlock) {
            const double gw = (double)g[i] * (w ? (double)w[i] : 1.0);
            gx[i] = (T)(r * (gw - (double)s[i] * c) + (gs ? (double)gs[i] : 0.0));
        }
    }
}

template <class T>
__global__ __launch_bounds__(kRnBlock) void rmsnorm_grad_weight_kernel(cumo_hip_rmsnorm_grad_t p, const double* rs) {
    const uint64_t i = (uint64_t)blockIdx.x * kRnBlock + threadIdx.x;
    if (i >= p.n) return;
    double sum = 0.0;
    for (uint64_t row = 0; row < p.rows; ++row)
        sum += (double)reinterpret_cast<const T*>(p.g + (int64_t)row * p.g_step)[i] * (double)reinterpret_cast<const T*>(p.s + (int64_t)row * p.s_step)[i] * rs[row];
    reinterpret_cast<T*>(p.gweight)[i] = (T)sum;
}

unsigned rn_grid(uint64_t blocks) { return (unsigned)(blocks < (1u << 20) ? blocks : (1u << 20)); }

template <class T>
int rn_grad(const cumo_hip_rmsnorm_grad_t& p, hipStream_t stream) {
    char* rs = nullptr;
    if (p.gweight && p.rows && !(rs = cumo_cuda_runtime_malloc(p.rows * sizeof(double)))) return CUMO_HIP_ERROR_OUT_OF_MEMORY;
    if (p.rows) hipLaunchKernelGGL((rmsnorm_grad_kernel<T>), dim3(rn_grid(p.rows)), dim3(kRnBlock), 0, stream, p, reinterpret_cast<double*>(rs));
    if (p.gweight)
        hipLaunchKernelGGL((rmsnorm_grad_weight_kernel<T>), dim3((unsigned)((p.n + kRnBlock - 1) / kRnBlock)), dim3(kRnBlock), 0, stream, p, reinterpret_cast<double*>(rs));
    cumo_cuda_runtime_check_kernel_launch();
    if (rs && !stream_under_capture()) cumo_cuda_runtime_free(rs);
    return CUMO_HIP_OK;
}

}  // namespace
}  // namespace cumo_hip

using namespace cumo_hip;

extern "C" void cumo_hip_rmsnorm_kernel_launch(int type, int quantised, const cumo_hip_rmsnorm_t* d) {
    hipStream_t stream = current_stream();
    const dim3 grid(rn_grid(d->rows)), block(kRnBlock);
    if (type == 0 && !quantised) hipLaunchKernelGGL((rmsnorm_kernel<float, false>), grid, block, 0, stream, *d);
    else if (type == 0) hipLaunchKernelGGL((rmsnorm_kernel<float, true>), grid, block, 0, stream, *d);
    else if (!quantised) hipLaunchKernelGGL((rmsnorm_kernel<double, false>), grid, block, 0, stream, *d);
    else hipLaunchKernelGGL((rmsnorm_kernel<double, true>), grid, block, 0, stream, *d);
    cumo_cuda_runtime_check_kernel_launch();
}

extern "C" void cumo_hip_dequantize_kernel_launch(int type, const cumo_hip_dequantize_t* d) {
    const dim3 grid(rn_grid((d->rows * d->n + kRnBlock - 1) / kRnBlock)), block(kRnBlock);
    if (type == 0) hipLaunchKernelGGL((dequantize_kernel<float>), grid, block, 0, current_stream(), *d);
    else hipLaunchKernelGGL((dequantize_kernel<double>), grid, block, 0, current_stream(), *d);
    cumo_cuda_runtime_check_kernel_launch();
}

extern "C" int cumo_hip_rmsnorm_grad_kernel_launch(int type, const cumo_hip_rmsnorm_grad_t* d) {
    return type == 0 ? rn_grad<float>(*d, current_stream()) : rn_grad<double>(*d, current_stream());
}

// The gated linear recurrence h[t] = a[t] h[t-1] + b[t] along one axis, and its gradients:
//   l[t] = g[t] + a[t+1] l[t+1] from the end;  gb = l;  ga[t] = l[t] h[t-1];  gh0 = a[0] l[0]
// Backwards what is carried from step to step is m[t] = a[t] l[t], so that a step needs its own elements alone:
//   l[t] = g[t] + m[t+1],  m[t] = a[t] l[t].
#include "common.h"

namespace cumo_hip {
namespace {

constexpr int kReBlock = 64;

template <class T>
__global__ __launch_bounds__(kReBlock) void recurrence_kernel(cumo_hip_recurrence_t p) {
    const uint64_t c = (uint64_t)blockIdx.x * kReBlock + threadIdx.x;
    if (c >= p.outer * p.inner) return;
    const int64_t o = (int64_t)(c / p.inner), i = (int64_t)(c % p.inner);
    const char* a = p.a + o * p.a_step[0] + i * p.a_step[2];
    const char* b = p.b + o * p.b_step[0] + i * p.b_step[2];
    char* h = p.h + o * p.h_step[0] + i * p.h_step[2];
    T state = p.h0 ? reinterpret_cast<const T*>(p.h0)[c] : (T)0;
    for (int64_t t = 0; t < (int64_t)p.time; ++t) {
        state = __builtin_elementwise_fma(*reinterpret_cast<const T*>(a + t * p.a_step[1]), state, *reinterpret_cast<const T*>(b + t * p.b_step[1]));
        *reinterpret_cast<T*>(h + t * p.h_step[1]) = state;
    }
}

template <class T>
__global__ __launch_bounds__(kReBlock) void recurrence_grad_kernel(cumo_hip_recurrence_grad_t p) {
    const uint64_t c = (uint64_t)blockIdx.x * kReBlock + threadIdx.x;
    if (c >= p.outer * p.inner) return;
    const int64_t o = (int64_t)(c / p.inner), i = (int64_t)(c % p.inner);
    const char* g = p.g + o * p.g_step[0] + i * p.g_step[2];
    const char* a = p.a + o * p.a_step[0] + i * p.a_step[2];
    const char* h = p.h + o * p.h_step[0] + i * p.h_step[2];
    char* ga = p.ga + o * p.ga_step[0] + i * p.ga_step[2];
    char* gb = p.gb + o * p.gb_step[0] + i * p.gb_step[2];
    T m = (T)0;
    for (int64_t t = (int64_t)p.time - 1; t >= 0; --t) {
        const T before = t > 0 ? *reinterpret_cast<const T*>(h + (t - 1) * p.h_step[1]) : (p.h0 ? reinterpret_cast<const T*>(p.h0)[c] : (T)0);
        const T l = *reinterpret_cast<const T*>(g + t * p.g_step[1]) + m;
        *reinterpret_cast<T*>(gb + t * p.gb_step[1]) = l;
        *reinterpret_cast<T*>(ga + t * p.ga_step[1]) = l * before;
        m = *reinterpret_cast<const T*>(a + t * p.a_step[1]) * l;
    }
    if (p.gh0) reinterpret_cast<T*>(p.gh0)[c] = m;
}

}  // namespace
}  // namespace cumo_hip

using namespace cumo_hip;

extern "C" int cumo_hip_recurrence_kernel_launch(int type, const cumo_hip_recurrence_t* d) {
    const dim3 grid((unsigned)((d->outer * d->inner + kReBlock - 1) / kReBlock)), block(kReBlock);
    if (type == 0) hipLaunchKernelGGL((recurrence_kernel<float>), grid, block, 0, current_stream(), *d);
    else hipLaunchKernelGGL((recurrence_kernel<double>), grid, block, 0, current_stream(), *d);
    cumo_cuda_runtime_check_kernel_launch();
    return CUMO_HIP_OK;
}

extern "C" int cumo_hip_recurrence_grad_kernel_launch(int type, const cumo_hip_recurrence_grad_t* d) {
    const dim3 grid((unsigned)((d->outer * d->inner + kReBlock - 1) / kReBlock)), block(kReBlock);
    if (type == 0) hipLaunchKernelGGL((recurrence_grad_kernel<float>), grid, block, 0, current_stream(), *d);
    else hipLaunchKernelGGL((recurrence_grad_kernel<double>), grid, block, 0, current_stream(), *d);
    cumo_cuda_runtime_check_kernel_launch();
    return CUMO_HIP_OK;
}

// The product of 8-bit rows by 8-bit rows, y[i][j] = (sum of x[i][k] w[j][k]) xscale[i] wscale[j] + bias[j].
#include "common.h"

namespace cumo_hip {
namespace {

// what a sum stands for, in double and rounded once
template <class T>
__device__ __forceinline__ T mq_value(int sum, double xs, double ws, double bias) { return (T)__builtin_fma((double)sum * xs, ws, bias); }

template <class T>
__global__ __launch_bounds__(256) void matmul_q8_kernel(cumo_hip_matmul_q8_t p) {
    const uint64_t total = p.rows * p.cols;
    for (uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x; at < total; at += (uint64_t)gridDim.x * 256) {
        const uint64_t i = at / p.cols, j = at - i * p.cols;
        const int8_t* x = reinterpret_cast<const int8_t*>(p.x + (int64_t)i * p.x_step);
        const int8_t* w = reinterpret_cast<const int8_t*>(p.w + (int64_t)j * p.w_step);
        int sum = 0;
        for (uint64_t k = 0; k < p.inner; ++k) sum += (int)x[k] * (int)w[k];
        const T* bias = reinterpret_cast<const T*>(p.bias);
        reinterpret_cast<T*>(p.y + (int64_t)i * p.y_step)[j] =
            mq_value<T>(sum, (double)reinterpret_cast<const T*>(p.xscale)[i], (double)reinterpret_cast<const T*>(p.wscale)[j], bias ? (double)bias[j] : 0.0);
    }
}

template <class T>
int mq_launch(const cumo_hip_matmul_q8_t& d, hipStream_t stream) {
    if (d.rows == 0 || d.cols == 0) return CUMO_HIP_OK;
    const uint64_t blocks = (d.rows * d.cols + 255) / 256;
    hipLaunchKernelGGL((matmul_q8_kernel<T>), dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, stream, d);
    cumo_cuda_runtime_check_kernel_launch();
    return CUMO_HIP_OK;
}

}  // namespace
}  // namespace cumo_hip

using namespace cumo_hip;

extern "C" int cumo_hip_matmul_q8_kernel_launch(int type, const cumo_hip_matmul_q8_t* d) {
    return type == 0 ? mq_launch<float>(*d, current_stream()) : mq_launch<double>(*d, current_stream());
}

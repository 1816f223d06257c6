// Linear attention of SFloat arrays, and the launchers (linear_attention.h).
#include "linear_attention.h"

namespace cumo_hip {
int la_forward_dfloat(const cumo_hip_linear_attention_t& d, hipStream_t stream);
int la_backward_dfloat(const cumo_hip_linear_attention_grad_t& d, hipStream_t stream);
}  // namespace cumo_hip

using namespace cumo_hip;

extern "C" int cumo_hip_linear_attention_kernel_launch(int type, const cumo_hip_linear_attention_t* d) {
    return type == 0 ? la_forward<float>(*d, current_stream()) : la_forward_dfloat(*d, current_stream());
}

extern "C" int cumo_hip_linear_attention_grad_kernel_launch(int type, const cumo_hip_linear_attention_grad_t* d) {
    return type == 0 ? la_backward<float>(*d, current_stream()) : la_backward_dfloat(*d, current_stream());
}

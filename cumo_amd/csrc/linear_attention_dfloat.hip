// Linear attention of DFloat arrays (linear_attention.h).
#include "linear_attention.h"

namespace cumo_hip {
int la_forward_dfloat(const cumo_hip_linear_attention_t& d, hipStream_t stream) { return la_forward<double>(d, stream); }
int la_backward_dfloat(const cumo_hip_linear_attention_grad_t& d, hipStream_t stream) { return la_backward<double>(d, stream); }
}  // namespace cumo_hip

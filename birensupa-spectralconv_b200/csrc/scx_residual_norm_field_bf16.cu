// The field kernels of the residual norm for __nv_bfloat16 (a file per type, so that they build at once).
#include "scx_residual_norm_field.cuh"

namespace scx_rn {
template cudaError_t field_forward<__nv_bfloat16>(const Problem&, cudaStream_t);
template cudaError_t field_backward<__nv_bfloat16>(Problem&, cudaStream_t);
}  // namespace scx_rn

// The field kernels of the residual norm for __half (a file per type, so that they build at once).
#include "scx_residual_norm_field.cuh"

namespace scx_rn {
template cudaError_t field_forward<__half>(const Problem&, cudaStream_t);
template cudaError_t field_backward<__half>(Problem&, cudaStream_t);
}  // namespace scx_rn

// The token kernels of the residual norm for float (a file per type, so that they build at once).
#include "scx_residual_norm_token.cuh"

namespace scx_rn {
template cudaError_t token_forward<float>(const Problem&, cudaStream_t);
template cudaError_t token_backward<float>(Problem&, cudaStream_t);
}  // namespace scx_rn

// The token kernels of the residual norm for __nv_bfloat16 (a file per type, so that they build at once).
#include "scx_residual_norm_token.cuh"

namespace scx_rn {
template cudaError_t token_forward<__nv_bfloat16>(const Problem&, cudaStream_t);
template cudaError_t token_backward<__nv_bfloat16>(Problem&, cudaStream_t);
}  // namespace scx_rn

// rows_bf16.cu -- the row operators on bf16 activations.
#include "rows_kernel.cuh"

namespace gcdr {
template cudaError_t rows_launch<__nv_bfloat16, true>(const RowArgs &, int, cudaStream_t);
template cudaError_t rows_launch<__nv_bfloat16, false>(const RowArgs &, int, cudaStream_t);
}  // namespace gcdr

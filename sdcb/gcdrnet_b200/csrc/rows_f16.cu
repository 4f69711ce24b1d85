// rows_f16.cu -- the row operators on fp16 activations.
#include "rows_kernel.cuh"

namespace gcdr {
template cudaError_t rows_launch<__half, true>(const RowArgs &, int, cudaStream_t);
template cudaError_t rows_launch<__half, false>(const RowArgs &, int, cudaStream_t);
}  // namespace gcdr

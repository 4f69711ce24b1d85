// rows_f32.cu -- the row operators on fp32 activations.
#include "rows_kernel.cuh"

namespace gcdr {
template cudaError_t rows_launch<float, true>(const RowArgs &, int, cudaStream_t);
template cudaError_t rows_launch<float, false>(const RowArgs &, int, cudaStream_t);
}  // namespace gcdr

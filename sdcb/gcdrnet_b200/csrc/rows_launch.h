// rows_launch.h -- a call of the row operators as their kernels take it, and the launches, one per type of the
// activations (rows_f16.cu, rows_bf16.cu, rows_f32.cu) and form (QUANT: the rounding alone).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace gcdr {

constexpr int kMaxRow = 32768;   // elements: 32 a thread of the largest block

struct RowArgs {
    int64_t rows;
    int C;
    float inv_C;
    const void *x;
    int64_t ldx;
    const void *f;
    int64_t ldf;
    int post;
    const float *g1, *b1;
    float eps1;
    const void *gate;
    int64_t ldg, gate_rows;
    uint32_t gate_mul;      // t / gate_rows = mulhi(t, gate_mul) >> gate_shift, exact for t < 2^31; 0: divide
    int gate_shift;
    float res_scale;
    void *r;
    int64_t ldr;
    int pre;
    const float *g2, *b2;
    float eps2;
    void *y;
    int64_t ldy;
    int8_t *q;
    int64_t ldq;
    float *qs;
};

// Aligned pieces that every row of every operand is made of: 16 bytes, 2 elements, or 0: single elements
template <class T, bool QUANT>
cudaError_t rows_launch(const RowArgs &a, int piece, cudaStream_t st);

}  // namespace gcdr

// int8.h -- the int8 token product (gcdr_k_i8_gemm): its arguments, its tensor-core kernel's launch, and the
// layer error word that capi.cu reads.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "gcdr_cuda.h"

namespace gcdr {

// The current device's layer error word, which the int8 product's kernels set (null: it cannot be had).
int *i8_error_word();

struct I8Args {
    int64_t M;
    int N, K;
    const int8_t *x;
    int64_t ldx;
    const float *xs;
    const int8_t *w;
    int64_t ldw;
    const float *ws, *bias;
    int relu, dtype;
    void *out;
    int64_t ldo;
    long long wait_cycles;
    int timeout_probe;
};

// The tensor-core kernel (int8_tc.cu); 0, or -1 and why not.
int i8_tc_launch(const I8Args &a, cudaStream_t st, std::string &err);

// The form that launch takes on a device of `sms` SMs (host only).
void i8_tc_form(const I8Args &a, int sms, gcdr_i8_form &f);

}  // namespace gcdr

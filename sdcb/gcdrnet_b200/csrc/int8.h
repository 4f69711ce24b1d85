// int8.h -- the int8 token product (gcdr_k_i8_gemm): its arguments, its tensor-core kernel's launch, and the
// status word that capi.cu reads.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "gcdr_cuda.h"

namespace gcdr {

constexpr int GCDR_ERR_FLAG_OTHER = 1 << 30;   // the status itself could not be read

// Reads and clears the current device's error word of the int8 product (GCDR_ERR_FLAG_*).
int i8_status_word();

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

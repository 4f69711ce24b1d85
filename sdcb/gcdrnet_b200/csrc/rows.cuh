// rows.cuh -- element types of the row operators (rows.cu) and of the int8 product (int8.cu):
// fp16, bf16 or fp32 in memory, fp32 in registers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <initializer_list>

#include "gcdr_cuda.h"

namespace gcdr {

inline int dtype_bytes(int dtype) {
    return dtype == GCDR_DTYPE_F32 ? 4 : (dtype == GCDR_DTYPE_F16 || dtype == GCDR_DTYPE_BF16) ? 2 : 0;
}

// One operand as the caller describes it, for the checks the operator entries share.
enum Role : int { kIn, kInPlace, kOut };   // kInPlace: an input that an output of its very layout may lie on
struct Operand {
    const char *name;
    const void *p;
    int64_t rows, cols, ld;   // ld in elements; rows x cols elements are read or written
    int size;                 // bytes per element
    Role role;
};

// Checks of one call's operands (int8.cu): pitches, extents that fit 63 bits, natural alignment, no
// output on top of another operand, and all of it memory of the current device.  Null operands are
// skipped.  Prints what is wrong to stderr and returns its GCDR_* status.
int check_operands(const char *who, std::initializer_list<Operand> ops);
int refuse(const char *who, int status, const char *what);

__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }

__device__ __forceinline__ void unpack2(uint32_t u, float *v, __half) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u));
    v[0] = f.x;
    v[1] = f.y;
}
__device__ __forceinline__ void unpack2(uint32_t u, float *v, __nv_bfloat16) {
    v[0] = __uint_as_float(u << 16);
    v[1] = __uint_as_float(u & 0xFFFF0000u);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// max(v, 0): a NaN stays, a zero has no sign
__device__ __forceinline__ float relu_f32(float v) {
    float m;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(m) : "f"(v));
    return m;
}

// One result of the int8 product: a rounding of the sum's (up to 31) bits to fp32 and two of the scaling.  The sum
// takes one scale, then the other: the product of the two alone could leave the normal numbers.
__device__ __forceinline__ float i8_result(int acc, float xs, float ws, float bias, bool relu) {
    const float v = fmaf((float)acc * xs, ws, bias);
    return relu ? relu_f32(v) : v;
}

}  // namespace gcdr

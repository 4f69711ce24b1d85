// int8.cu -- the int8 token product (gcdr_k_i8_gemm) and the operand checks it shares with rows.cu.
//
//   out[m][n] = xs[m] * ws[n] * sum_k x[m][k] w[n][k] + bias[n]   [relu]
//
// The sum is an int32: exact, so no split or order of it changes a result.  It is converted to fp32
// once (24 of its up to 31 bits, half a step of fp32) and scaled there.
#include <cstdio>

#include "common.cuh"
#include "int8.h"
#include "rows.cuh"

namespace gcdr {

int refuse(const char *who, int status, const char *what) {
    std::fprintf(stderr, "%s: %s\n", who, what);
    return status;
}

namespace {

struct Extent {
    uintptr_t begin, end;
    int64_t pitch, width;   // bytes
};

// Whether two strided operands share a byte.  At one pitch their columns decide (two slices of one
// buffer's columns are apart), at different pitches their ranges do.
bool overlap(const Extent &a, const Extent &b) {
    if (a.end <= b.begin || b.end <= a.begin) return false;
    if (a.pitch != b.pitch) return true;
    const uintptr_t P = (uintptr_t)a.pitch;
    const uintptr_t d = a.begin <= b.begin ? (b.begin - a.begin) % P : (P - (a.begin - b.begin) % P) % P;
    return !((int64_t)d >= a.width && (int64_t)d + b.width <= a.pitch);
}

}  // namespace

int check_operands(const char *who, std::initializer_list<Operand> ops) {
    Extent ext[16];
    const Operand *op[16];
    char msg[160];
    int n = 0;
    const auto bad = [&](int status, const Operand &o, const char *what) {
        std::snprintf(msg, sizeof msg, "%s %s", o.name, what);
        return refuse(who, status, msg);
    };
    for (const Operand &o : ops) {
        if (!o.p || o.rows < 1) continue;
        if (o.ld < o.cols) return bad(GCDR_ERR_RANGE, o, "has a pitch below its row length");
        int64_t pitch, last;
        if (__builtin_mul_overflow(o.ld, (int64_t)o.size, &pitch) || __builtin_mul_overflow(pitch, o.rows, &last) ||
            last > ((int64_t)1 << 60))
            return bad(GCDR_ERR_RANGE, o, "is too large");
        const uintptr_t at = reinterpret_cast<uintptr_t>(o.p);
        if (at % o.size) return bad(GCDR_ERR_ARG, o, "is not aligned to its elements");
        ext[n] = {at, at + (uintptr_t)(pitch * (o.rows - 1) + o.cols * o.size), pitch, o.cols * o.size};
        op[n++] = &o;
    }
    for (int i = 0; i < n; i++)
        for (int j = i + 1; j < n; j++) {
            if (op[i]->role != kOut && op[j]->role != kOut) continue;
            if (!overlap(ext[i], ext[j])) continue;
            const bool same = ext[i].begin == ext[j].begin && ext[i].pitch == ext[j].pitch && op[i]->rows == op[j]->rows &&
                              op[i]->cols == op[j]->cols && op[i]->size == op[j]->size;
            if (same && (op[i]->role == kInPlace || op[j]->role == kInPlace)) continue;
            std::snprintf(msg, sizeof msg, "%s and %s overlap", op[i]->name, op[j]->name);
            return refuse(who, GCDR_ERR_ARG, msg);
        }
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    for (int i = 0; i < n && e == cudaSuccess; i++) {
        cudaPointerAttributes at;
        e = cudaPointerGetAttributes(&at, op[i]->p);
        if (e == cudaSuccess && !(at.type == cudaMemoryTypeManaged || (at.type == cudaMemoryTypeDevice && at.device == dev)))
            return bad(GCDR_ERR_ARG, *op[i], "is not memory of the current device");
    }
    if (e != cudaSuccess) {
        cudaGetLastError();
        return refuse(who, GCDR_ERR_DEVICE, cudaGetErrorString(e));
    }
    return GCDR_OK;
}

namespace {

constexpr int kDotTokens = 4;

__device__ __forceinline__ float scaled(int acc, float xs, float ws, float bias, int relu) {
    const float v = fmaf((float)acc * xs, ws, bias);
    return relu && v < 0.f ? 0.f : v;   // (a NaN stays)
}

// 16 bytes of a row from k on, zeros past K (a row's tail is read byte by byte: nothing lies behind
// the last one)
__device__ __forceinline__ int4 load16(const int8_t *row, int k, int K) {
    if (k + 16 <= K) return *reinterpret_cast<const int4 *>(row + k);
    int w[4] = {0, 0, 0, 0};
    for (int i = 0; i < 16 && k + i < K; i++) w[i >> 2] |= (int)(uint8_t)row[k + i] << (8 * (i & 3));
    return make_int4(w[0], w[1], w[2], w[3]);
}

// A warp forms the products of one channel with MT tokens: the lanes take the row 16 bytes each.
template <class T, int MT>
__global__ void __launch_bounds__(256) i8_dot_kernel(const __grid_constant__ I8Args a) {
    const int lane = threadIdx.x & 31;
    const int64_t n = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    pdl_wait();
    if (n < a.N) {
        const int8_t *w = a.w + n * a.ldw;
        const float ws = a.ws[n], bias = a.bias ? a.bias[n] : 0.f;
        for (int64_t m0 = (int64_t)blockIdx.y * MT; m0 < a.M; m0 += (int64_t)gridDim.y * MT) {
            int acc[MT];
#pragma unroll
            for (int j = 0; j < MT; j++) acc[j] = 0;
            for (int k = lane * 16; k < a.K; k += 512) {
                const int4 b = load16(w, k, a.K);
#pragma unroll
                for (int j = 0; j < MT; j++) {
                    if (m0 + j >= a.M) break;
                    const int4 x = load16(a.x + (m0 + j) * a.ldx, k, a.K);
                    acc[j] = __dp4a(x.x, b.x, acc[j]);
                    acc[j] = __dp4a(x.y, b.y, acc[j]);
                    acc[j] = __dp4a(x.z, b.z, acc[j]);
                    acc[j] = __dp4a(x.w, b.w, acc[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < MT; j++) {
                if (m0 + j >= a.M) break;
                const int sum = __reduce_add_sync(0xFFFFFFFFu, acc[j]);
                if (lane == 0)
                    static_cast<T *>(a.out)[(m0 + j) * a.ldo + n] = from_f32<T>(scaled(sum, a.xs[m0 + j], ws, bias, a.relu));
            }
        }
    }
    pdl_trigger();
}

template <class T>
cudaError_t launch_dot(const I8Args &a, cudaStream_t st) {
    constexpr int MT = 4;
    const int64_t my = (a.M + MT - 1) / MT;
    const dim3 grid((unsigned)(((int64_t)a.N + 7) / 8), (unsigned)(my < 65535 ? my : 65535));
    return launch_pdl(i8_dot_kernel<T, MT>, grid, dim3(256), 0, st, a);
}

}  // namespace

}  // namespace gcdr

using namespace gcdr;

extern "C" int gcdr_k_i8_gemm(const gcdr_i8_gemm_desc *d, void *stream) {
    const char *who = "gcdr_k_i8_gemm";
    if (!d) return refuse(who, GCDR_ERR_ARG, "null descriptor");
    const int size = dtype_bytes(d->dtype);
    if (!size) return refuse(who, GCDR_ERR_ARG, "unknown dtype");
    if (d->M < 0 || d->M > 0x7FFFFFFF || d->N < 1 || d->K < 1 || d->K > 131071)
        return refuse(who, GCDR_ERR_RANGE, "M must be 0..2^31-1, N >= 1 and K 1..131071");
    if (d->wait_cycles < 0) return refuse(who, GCDR_ERR_RANGE, "wait_cycles must be >= 0");
    if (d->M == 0) return GCDR_OK;
    if (!d->x || !d->xs || !d->w || !d->ws || !d->out) return refuse(who, GCDR_ERR_ARG, "null operand");
    if (((uintptr_t)d->x | (uintptr_t)d->w) % 16 || d->ldx % 16 || d->ldw % 16)
        return refuse(who, GCDR_ERR_ARG, "x and w must be 16-byte aligned at pitches of a multiple of 16");
    const int rc = check_operands(who, {{"x", d->x, d->M, d->K, d->ldx, 1, kIn},
                                        {"xs", d->xs, 1, d->M, d->M, 4, kIn},
                                        {"w", d->w, d->N, d->K, d->ldw, 1, kIn},
                                        {"ws", d->ws, 1, d->N, d->N, 4, kIn},
                                        {"bias", d->bias, 1, d->N, d->N, 4, kIn},
                                        {"out", d->out, d->M, d->N, d->ldo, size, kOut}});
    if (rc) return rc;
    if (d->ldx >= (int64_t)1 << 40 || d->ldw >= (int64_t)1 << 40) return refuse(who, GCDR_ERR_RANGE, "a pitch of 2^40 or more");
    const I8Args a = {d->M, d->N, d->K, d->x, d->ldx, d->xs, d->w, d->ldw, d->ws, d->bias, d->relu, d->dtype, d->out, d->ldo,
                      d->wait_cycles, d->timeout_probe != 0};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a.M > kDotTokens || a.timeout_probe) {
        std::string err;
        return i8_tc_launch(a, st, err) ? refuse(who, GCDR_ERR_DEVICE, err.c_str()) : GCDR_OK;
    }
    const cudaError_t e = d->dtype == GCDR_DTYPE_F16    ? launch_dot<__half>(a, st)
                          : d->dtype == GCDR_DTYPE_BF16 ? launch_dot<__nv_bfloat16>(a, st)
                                                        : launch_dot<float>(a, st);
    if (e == cudaSuccess) return GCDR_OK;
    cudaGetLastError();
    return refuse(who, GCDR_ERR_DEVICE, cudaGetErrorString(e));
}

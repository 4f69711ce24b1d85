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

// 16 bytes of a row from k on, zeros past K (a row's tail is read byte by byte: nothing lies behind
// the last one)
__device__ __forceinline__ int4 load16(const int8_t *row, int k, int K) {
    if (k + 16 <= K) return *reinterpret_cast<const int4 *>(row + k);
    int w[4] = {0, 0, 0, 0};
    for (int i = 0; i < 16 && k + i < K; i++) w[i >> 2] |= (int)(uint8_t)row[k + i] << (8 * (i & 3));
    return make_int4(w[0], w[1], w[2], w[3]);
}

// A warp forms the products of R channels with MT tokens, the lanes 16 bytes of a row each: U pieces of every row
// are on their way at once, each token's piece serves R channels.
template <class T, int MT, int R, int U>
__global__ void __launch_bounds__(128) i8_dot_kernel(const __grid_constant__ I8Args a) {
    const int lane = threadIdx.x & 31;
    const int64_t n0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 5)) * R;
    pdl_wait();
    if (n0 < a.N) {
        int acc[R][MT];
        const int8_t *w[R], *x[MT];
#pragma unroll
        for (int r = 0; r < R; r++) w[r] = a.w + (n0 + r < a.N ? n0 + r : a.N - 1) * a.ldw;   // (a row twice, not past the last)
#pragma unroll
        for (int j = 0; j < MT; j++) x[j] = a.x + (j < a.M ? j : a.M - 1) * a.ldx;
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int j = 0; j < MT; j++) acc[r][j] = 0;
        const auto dot = [&](const int4 &p, const int4 &q, int &sum) {
            sum = __dp4a(p.x, q.x, sum);
            sum = __dp4a(p.y, q.y, sum);
            sum = __dp4a(p.z, q.z, sum);
            sum = __dp4a(p.w, q.w, sum);
        };
        int k = lane * 16;
        for (; k - lane * 16 + U * 512 <= a.K; k += U * 512) {
            int4 p[R][U], q[MT];
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int r = 0; r < R; r++) p[r][u] = __ldcs(reinterpret_cast<const int4 *>(w[r] + k + u * 512));
#pragma unroll
            for (int u = 0; u < U; u++) {
#pragma unroll
                for (int j = 0; j < MT; j++) q[j] = *reinterpret_cast<const int4 *>(x[j] + k + u * 512);
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int j = 0; j < MT; j++) dot(p[r][u], q[j], acc[r][j]);
            }
        }
        for (; k < a.K; k += 512) {
#pragma unroll
            for (int r = 0; r < R; r++) {
                const int4 p = load16(w[r], k, a.K);
#pragma unroll
                for (int j = 0; j < MT; j++) dot(p, load16(x[j], k, a.K), acc[r][j]);
            }
        }
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int j = 0; j < MT; j++) {
                const int sum = __reduce_add_sync(0xFFFFFFFFu, acc[r][j]);
                if (lane == 0 && j < a.M && n0 + r < a.N)
                    static_cast<T *>(a.out)[j * a.ldo + n0 + r] =
                        from_f32<T>(i8_result(sum, a.xs[j], a.ws[n0 + r], a.bias ? a.bias[n0 + r] : 0.f, a.relu));
            }
    }
    pdl_trigger();   // (earlier, the next kernel's blocks wait beside these: 8192 x 8192 12.7 us against 12.0)
}

template <class T, int MT, int R, int U>
cudaError_t launch_dot(const I8Args &a, cudaStream_t st) {
    return launch_pdl(i8_dot_kernel<T, MT, R, U>, dim3((unsigned)(((int64_t)a.N + 4 * R - 1) / (4 * R))), dim3(128), 0, st, a);
}

// Channels of a warp (few of them: a warp each, so that they spread over the GPU)
int dot_channels(const I8Args &a) { return a.N < 4096 ? 1 : 2; }

template <class T>
cudaError_t launch_dot(const I8Args &a, cudaStream_t st) {
    const bool few = dot_channels(a) == 1;
    if (a.M == 1) return few ? launch_dot<T, 1, 1, 4>(a, st) : launch_dot<T, 1, 2, 4>(a, st);
    if (a.M == 2) return few ? launch_dot<T, 2, 1, 4>(a, st) : launch_dot<T, 2, 2, 4>(a, st);
    return few ? launch_dot<T, 4, 1, 4>(a, st) : launch_dot<T, 4, 2, 4>(a, st);
}

}  // namespace

}  // namespace gcdr

using namespace gcdr;

namespace {

// What a descriptor may hold, as far as the host can tell without the device
int check_desc(const char *who, const gcdr_i8_gemm_desc *d) {
    if (!d) return refuse(who, GCDR_ERR_ARG, "null descriptor");
    if (!dtype_bytes(d->dtype)) return refuse(who, GCDR_ERR_ARG, "unknown dtype");
    if (d->M < 0 || d->M > 0x7FFFFFFF || d->N < 1 || d->K < 1 || d->K > 131071)
        return refuse(who, GCDR_ERR_RANGE, "M must be 0..2^31-1, N >= 1 and K 1..131071");
    if (d->wait_cycles < 0) return refuse(who, GCDR_ERR_RANGE, "wait_cycles must be >= 0");
    return GCDR_OK;
}

I8Args args_of(const gcdr_i8_gemm_desc *d) {
    return {d->M, d->N, d->K, d->x, d->ldx, d->xs, d->w, d->ldw, d->ws, d->bias, d->relu, d->dtype, d->out, d->ldo,
            d->wait_cycles, d->timeout_probe != 0};
}

bool by_dots(const I8Args &a) { return a.M <= kDotTokens && !a.timeout_probe; }

}  // namespace

extern "C" int gcdr_k_i8_gemm_form(const gcdr_i8_gemm_desc *d, int sms, gcdr_i8_form *form) {
    const char *who = "gcdr_k_i8_gemm_form";
    const int rc = check_desc(who, d);
    if (rc) return rc;
    if (!form) return refuse(who, GCDR_ERR_ARG, "null form");
    if (sms < 2 || sms > 4096) return refuse(who, GCDR_ERR_RANGE, "sms must be 2..4096");
    *form = {};
    const I8Args a = args_of(d);
    if (!a.M) return GCDR_OK;
    if (!by_dots(a)) {
        i8_tc_form(a, sms, *form);
        return GCDR_OK;
    }
    form->form = GCDR_I8_DOT;
    form->tile = dot_channels(a);
    form->units = ((int64_t)a.N + form->tile - 1) / form->tile;
    return GCDR_OK;
}

extern "C" int gcdr_k_i8_gemm(const gcdr_i8_gemm_desc *d, void *stream) {
    const char *who = "gcdr_k_i8_gemm";
    const int bad = check_desc(who, d);
    if (bad) return bad;
    const int size = dtype_bytes(d->dtype);
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
    const I8Args a = args_of(d);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!by_dots(a)) {
        try {
            std::string err;
            return i8_tc_launch(a, st, err) ? refuse(who, GCDR_ERR_DEVICE, err.c_str()) : GCDR_OK;
        } catch (...) {   // (of the message's memory: nothing leaves a C entry)
            return GCDR_ERR_OOM;
        }
    }
    const cudaError_t e = d->dtype == GCDR_DTYPE_F16    ? launch_dot<__half>(a, st)
                          : d->dtype == GCDR_DTYPE_BF16 ? launch_dot<__nv_bfloat16>(a, st)
                                                        : launch_dot<float>(a, st);
    if (e == cudaSuccess) return GCDR_OK;
    cudaGetLastError();
    return refuse(who, GCDR_ERR_DEVICE, cudaGetErrorString(e));
}

// rows.cu -- operators over rows (one token's channels, or one channel's weights):
//
//   quant_rows   s = max|x| / 127,  q = x * 127 / max|x| rounded to nearest even
//   block_norm   v = x + res_scale * gate . N1(f);  r = v;  h = N2(v) as y or as int8 rows
//                N = LayerNorm (u - mean) / sqrt(var + eps) * g + b, or RMS u / sqrt(mean u^2 + eps) * g + b
//
// Both are bound by memory: each element is read once into fp32 registers, every statistic is
// taken there (mean first, then the squares about it), and the row is written once.  A group of G
// threads holds a row, 8 * NCH elements a thread.  v stays in fp32 for the second norm: only what is
// stored is rounded to the activations' type.
#include <cstdio>

#include "common.cuh"
#include "rows.cuh"

namespace gcdr {
namespace {

struct RowArgs {
    int64_t rows;
    int C;
    const void *x;
    int64_t ldx;
    const void *f;
    int64_t ldf;
    int post;
    const float *g1, *b1;
    float eps1;
    const void *gate;
    int64_t ldg, gate_rows;
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

constexpr int kMaxRow = 32768;

// Group-wide reductions: shuffles inside a warp, one shared slot per warp beyond.  The slots
// alternate between two sets, so one barrier per reduction is enough.
template <int G>
struct Group {
    float *slots;
    int turn = 0;
    template <class Op>
    __device__ __forceinline__ float all(float v, Op op) {
#pragma unroll
        for (int o = (G < 32 ? G : 32) / 2; o; o >>= 1) v = op(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
        if (G > 32) {
            constexpr int W = G > 32 ? G / 32 : 1;
            float *s = slots + turn * W;
            turn ^= 1;
            if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
            __syncthreads();
            v = s[0];
#pragma unroll
            for (int w = 1; w < W; w++) v = op(v, s[w]);
        }
        return v;
    }
    __device__ __forceinline__ float sum(float v) {
        return all(v, [](float a, float b) { return a + b; });
    }
    // NaN when any is NaN (fmaxf would drop it)
    __device__ __forceinline__ float top(float v) {
        return all(v, [](float a, float b) {
            float m;
            asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
            return m;
        });
    }
};

// v * 127 / top to nearest even, exactly: the quotient is estimated with inv = 127 / top (off by less
// than 2e-5), and an estimate that close to a border k + 1/2 is decided by the sign of
// 127 v - (k + 1/2) top, whose two products and their rests are exact in fp32 (31 and 32 bits).
__device__ __forceinline__ int round_to(float v, float top, float inv) {
    const float t = v * inv;
    float q = rintf(t);
    if (fabsf(t - q) > 0.4999f) {
        const float k = floorf(t), h = k + 0.5f;
        const float p = __fmul_rn(127.f, v), pr = fmaf(127.f, v, -p);
        const float m = __fmul_rn(h, top), mr = fmaf(h, top, -m);
        const float d = (p - m) + (pr - mr);
        q = d > 0.f ? k + 1.f : d < 0.f ? k : 2.f * rintf(h * 0.5f);
    }
    return (int)q;
}

// Rows beyond these are scaled by a power of two first (exact), so that 127 / top and the
// products of round_to stay normal numbers.
__device__ __forceinline__ float row_lift(float top) {
    return top < 0x1p-60f ? 0x1p60f : top > 0x1p60f ? 0x1p-60f : 1.f;
}

template <class T, int G, int NCH, bool VEC, bool QUANT>
__global__ void __launch_bounds__(G > 32 ? G : 256) rows_kernel(const __grid_constant__ RowArgs a) {
    constexpr int RPB = G > 32 ? 1 : 256 / G;   // rows per block
    constexpr int E = 8 * NCH;
    __shared__ float slots[G > 32 ? 2 * (G / 32) : 1];
    Group<G> grp{slots};
    const int l = threadIdx.x % G, C = a.C;
    // element j of this thread: 8 neighbours a chunk, or G apart where rows are not aligned
    const auto at = [&](int j) { return VEC ? (l + G * (j / 8)) * 8 + j % 8 : l + G * j; };
    const auto load = [&](const auto *p, float *v, float fill) {
        using P = typename std::remove_cv<typename std::remove_pointer<decltype(p)>::type>::type;
        if (VEC) {
#pragma unroll
            for (int k = 0; k < NCH; k++) {
                if (at(8 * k) < C) load8<P>(p + at(8 * k), v + 8 * k);
                else
#pragma unroll
                    for (int e = 0; e < 8; e++) v[8 * k + e] = fill;
            }
        } else {
#pragma unroll
            for (int j = 0; j < E; j++) v[j] = at(j) < C ? to_f32(p[at(j)]) : fill;
        }
    };
    const auto store = [&](T *p, const float *v) {
        if (VEC) {
#pragma unroll
            for (int k = 0; k < NCH; k++)
                if (at(8 * k) < C) store8<T>(p + at(8 * k), v + 8 * k);
        } else {
#pragma unroll
            for (int j = 0; j < E; j++)
                if (at(j) < C) p[at(j)] = from_f32<T>(v[j]);
        }
    };
    const auto norm = [&](float *v, int kind, const float *g, const float *b, float eps) {
        float mean = 0.f;
        if (kind == GCDR_NORM_LAYER) {
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < E; j++) s += v[j];   // (elements past C are zero)
            mean = grp.sum(s) / C;
        }
        float q = 0.f;
#pragma unroll
        for (int j = 0; j < E; j++) {
            const float d = at(j) < C ? v[j] - mean : 0.f;
            v[j] = d;
            q += d * d;
        }
        const float rstd = 1.f / sqrtf(grp.sum(q) / C + eps);
        float t[E];
        if (g) {
            load(g, t, 0.f);
#pragma unroll
            for (int j = 0; j < E; j++) v[j] = v[j] * rstd * t[j];
        } else {
#pragma unroll
            for (int j = 0; j < E; j++) v[j] *= rstd;
        }
        if (b) {
            load(b, t, 0.f);
#pragma unroll
            for (int j = 0; j < E; j++) v[j] += t[j];
        }
    };

    pdl_wait();
    for (int64_t base = (int64_t)blockIdx.x * RPB; base < a.rows; base += (int64_t)gridDim.x * RPB) {
        const int64_t row = base + threadIdx.x / G;
        const bool valid = row < a.rows;          // idle groups still join the shuffles
        const int64_t rr = valid ? row : a.rows - 1;
        float v[E];
        if (QUANT) {
            load(static_cast<const T *>(a.x) + rr * a.ldx, v, 0.f);
        } else {
            if (a.f) {
                load(static_cast<const T *>(a.f) + rr * a.ldf, v, 0.f);
                if (a.post) norm(v, a.post, a.g1, a.b1, a.eps1);
                float t[E];
                if (a.gate) {
                    load(static_cast<const T *>(a.gate) + rr / a.gate_rows * a.ldg, t, 0.f);
#pragma unroll
                    for (int j = 0; j < E; j++) v[j] *= t[j];
                }
                if (a.x) {
                    load(static_cast<const T *>(a.x) + rr * a.ldx, t, 0.f);
#pragma unroll
                    for (int j = 0; j < E; j++) v[j] = fmaf(a.res_scale, v[j], t[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < E; j++) v[j] *= a.res_scale;
                }
            } else {
                load(static_cast<const T *>(a.x) + rr * a.ldx, v, 0.f);
            }
            if (a.r && valid) store(static_cast<T *>(a.r) + row * a.ldr, v);
            if (a.pre) norm(v, a.pre, a.g2, a.b2, a.eps2);
            if (a.y && valid) store(static_cast<T *>(a.y) + row * a.ldy, v);
        }
        if (QUANT || a.q) {
            float top = 0.f;
#pragma unroll
            for (int j = 0; j < E; j++) {
                const float m = fabsf(v[j]);
                asm("max.NaN.f32 %0, %1, %2;" : "=f"(top) : "f"(top), "f"(m));
            }
            top = grp.top(top);
            // an infinity or NaN anywhere in the row: the scale says so, the bytes are zero
            const bool fine = top < __int_as_float(0x7F800000);
            const float lift = row_lift(top), t2 = top * lift;
            const float inv = fine && top > 0.f ? 127.f / t2 : 0.f;
            if (valid) {
                if (l == 0) a.qs[row] = fine ? top / 127.f : __int_as_float(0x7FC00000);
                int8_t *p = a.q + row * a.ldq;
#pragma unroll
                for (int j = 0; j < E; j++) v[j] *= lift;
                if (VEC) {
#pragma unroll
                    for (int k = 0; k < NCH; k++) {
                        if (at(8 * k) >= C) continue;
                        uint32_t w[2] = {0, 0};
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            w[e / 4] |= (uint32_t)(inv > 0.f ? round_to(v[8 * k + e], t2, inv) & 0xFF : 0) << (8 * (e % 4));
                        *reinterpret_cast<uint2 *>(p + at(8 * k)) = make_uint2(w[0], w[1]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < E; j++)
                        if (at(j) < C) p[at(j)] = (int8_t)(inv > 0.f ? round_to(v[j], t2, inv) : 0);
                }
            }
        }
    }
    pdl_trigger();
}

template <class T, int G, int NCH, bool QUANT>
cudaError_t launch_rows(const RowArgs &a, bool vec, cudaStream_t st) {
    constexpr int T_ = G > 32 ? G : 256;
    constexpr int RPB = G > 32 ? 1 : 256 / G;
    const int64_t want = (a.rows + RPB - 1) / RPB;
    const unsigned grid = (unsigned)(want < (1 << 20) ? want : (1 << 20));
    return vec ? launch_pdl(rows_kernel<T, G, NCH, true, QUANT>, dim3(grid), dim3(T_), 0, st, a)
               : launch_pdl(rows_kernel<T, G, NCH, false, QUANT>, dim3(grid), dim3(T_), 0, st, a);
}

template <class T, bool QUANT>
cudaError_t launch_type(const RowArgs &a, bool vec, cudaStream_t st) {
    const int C = a.C;
    if (C <= 64) return launch_rows<T, 8, 1, QUANT>(a, vec, st);
    if (C <= 128) return launch_rows<T, 16, 1, QUANT>(a, vec, st);
    if (C <= 256) return launch_rows<T, 32, 1, QUANT>(a, vec, st);
    if (C <= 512) return launch_rows<T, 32, 2, QUANT>(a, vec, st);
    if (C <= 1024) return launch_rows<T, 64, 2, QUANT>(a, vec, st);
    if (C <= 2048) return launch_rows<T, 128, 2, QUANT>(a, vec, st);
    if (C <= 4096) return launch_rows<T, 256, 2, QUANT>(a, vec, st);
    if (C <= 8192) return launch_rows<T, 512, 2, QUANT>(a, vec, st);
    if (C <= 16384) return launch_rows<T, 1024, 2, QUANT>(a, vec, st);
    return launch_rows<T, 1024, 4, QUANT>(a, vec, st);
}

template <bool QUANT>
int launch(const char *who, const RowArgs &a, int dtype, bool vec, cudaStream_t st) {
    const cudaError_t e = dtype == GCDR_DTYPE_F16    ? launch_type<__half, QUANT>(a, vec, st)
                          : dtype == GCDR_DTYPE_BF16 ? launch_type<__nv_bfloat16, QUANT>(a, vec, st)
                                                     : launch_type<float, QUANT>(a, vec, st);
    if (e == cudaSuccess) return GCDR_OK;
    cudaGetLastError();
    return refuse(who, GCDR_ERR_DEVICE, cudaGetErrorString(e));
}

// 16-byte vectors of an activation row, 8-byte ones of an int8 row
bool aligned(const void *p, int64_t ld_bytes, int n) {
    return !p || (reinterpret_cast<uintptr_t>(p) % n == 0 && ld_bytes % n == 0);
}

}  // namespace
}  // namespace gcdr

using namespace gcdr;

extern "C" int gcdr_k_quant_rows(const void *x, int dtype, int64_t rows, int C, int64_t ldx, int8_t *q, int64_t ldq,
                                 float *scale, void *stream) {
    const char *who = "gcdr_k_quant_rows";
    const int size = dtype_bytes(dtype);
    if (!size) return refuse(who, GCDR_ERR_ARG, "unknown dtype");
    if (rows < 0 || C < 1 || C > kMaxRow) return refuse(who, GCDR_ERR_RANGE, "rows must be >= 0 and C 1..32768");
    if (rows == 0) return GCDR_OK;
    if (!x || !q || !scale) return refuse(who, GCDR_ERR_ARG, "null operand");
    const int rc = check_operands(who, {{"x", x, rows, C, ldx, size, kIn},
                                        {"q", q, rows, C, ldq, 1, kOut},
                                        {"scale", scale, 1, rows, rows, 4, kOut}});
    if (rc) return rc;
    RowArgs a = {};
    a.rows = rows;
    a.C = C;
    a.x = x;
    a.ldx = ldx;
    a.q = q;
    a.ldq = ldq;
    a.qs = scale;
    const bool vec = C % 8 == 0 && aligned(x, ldx * size, 16) && aligned(q, ldq, 8);
    return launch<true>(who, a, dtype, vec, static_cast<cudaStream_t>(stream));
}

extern "C" int gcdr_k_block_norm(const gcdr_block_norm_desc *d, void *stream) {
    const char *who = "gcdr_k_block_norm";
    if (!d) return refuse(who, GCDR_ERR_ARG, "null descriptor");
    const int size = dtype_bytes(d->dtype);
    if (!size) return refuse(who, GCDR_ERR_ARG, "unknown dtype");
    if (d->rows < 0 || d->C < 1 || d->C > kMaxRow) return refuse(who, GCDR_ERR_RANGE, "rows must be >= 0 and C 1..32768");
    if (d->post < 0 || d->post > GCDR_NORM_RMS || d->pre < 0 || d->pre > GCDR_NORM_RMS)
        return refuse(who, GCDR_ERR_ARG, "unknown norm");
    if (!(d->eps1 >= 0.f) || !(d->eps2 >= 0.f)) return refuse(who, GCDR_ERR_ARG, "eps must be >= 0");
    if (d->gate && d->gate_rows < 1) return refuse(who, GCDR_ERR_RANGE, "gate_rows must be >= 1");
    if (d->rows == 0) return GCDR_OK;
    if (!d->x && !d->f) return refuse(who, GCDR_ERR_ARG, "neither x nor f");
    if (!d->f && (d->post || d->gate)) return refuse(who, GCDR_ERR_ARG, "a norm or gate of f, but no f");
    if (!d->r && !d->y && !d->q) return refuse(who, GCDR_ERR_ARG, "no output");
    if (!d->q != !d->qs) return refuse(who, GCDR_ERR_ARG, "q and qs come together");
    const int64_t n = d->rows;
    const int C = d->C;
    // a gain or shift without its norm is not read
    const float *g1 = d->post ? d->g1 : nullptr, *b1 = d->post ? d->b1 : nullptr;
    const float *g2 = d->pre ? d->g2 : nullptr, *b2 = d->pre ? d->b2 : nullptr;
    const int rc = check_operands(who, {{"x", d->x, n, C, d->ldx, size, kInPlace},
                                        {"f", d->f, n, C, d->ldf, size, kInPlace},
                                        {"gate", d->gate, d->gate ? (n - 1) / d->gate_rows + 1 : 0, C, d->ldg, size, kIn},
                                        {"g1", g1, 1, C, C, 4, kIn},
                                        {"b1", b1, 1, C, C, 4, kIn},
                                        {"g2", g2, 1, C, C, 4, kIn},
                                        {"b2", b2, 1, C, C, 4, kIn},
                                        {"r", d->r, n, C, d->ldr, size, kOut},
                                        {"y", d->y, n, C, d->ldy, size, kOut},
                                        {"q", d->q, n, C, d->ldq, 1, kOut},
                                        {"qs", d->qs, 1, n, n, 4, kOut}});
    if (rc) return rc;
    RowArgs a = {};
    a.rows = n;
    a.C = C;
    a.x = d->x;
    a.ldx = d->ldx;
    a.f = d->f;
    a.ldf = d->ldf;
    a.post = d->post;
    a.g1 = g1;
    a.b1 = b1;
    a.eps1 = d->eps1;
    a.gate = d->gate;
    a.ldg = d->ldg;
    a.gate_rows = d->gate_rows;
    a.res_scale = d->res_scale;
    a.r = d->r;
    a.ldr = d->ldr;
    a.pre = d->pre;
    a.g2 = g2;
    a.b2 = b2;
    a.eps2 = d->eps2;
    a.y = d->y;
    a.ldy = d->ldy;
    a.q = d->q;
    a.ldq = d->ldq;
    a.qs = d->qs;
    const bool vec = C % 8 == 0 && aligned(d->x, d->ldx * size, 16) && aligned(d->f, d->ldf * size, 16) &&
                     aligned(d->gate, d->ldg * size, 16) && aligned(d->r, d->ldr * size, 16) &&
                     aligned(d->y, d->ldy * size, 16) && aligned(d->q, d->ldq, 8) && aligned(g1, 16, 16) &&
                     aligned(b1, 16, 16) && aligned(g2, 16, 16) && aligned(b2, 16, 16);
    return launch<false>(who, a, d->dtype, vec, static_cast<cudaStream_t>(stream));
}

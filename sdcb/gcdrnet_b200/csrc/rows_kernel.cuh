// rows_kernel.cuh -- operators over rows (one token's channels, or one channel's weights):
//
//   quant_rows   s = max|x| / 127,  q = x * 127 / max|x| rounded to nearest even
//   block_norm   v = x + res_scale * gate . N1(f);  r = v;  h = N2(v) as y or as int8 rows
//                N = LayerNorm (u - mean) / sqrt(var + eps) * g + b, or RMS u / sqrt(mean u^2 + eps) * g + b
//
// Both are bound by memory: each element is read once into registers (rows too long for them: see rows_launch), every
// statistic is taken there in fp32 (the mean first, then the squares about it), and the row is written once.  v stays in
// fp32 for the second norm: only what is stored is rounded to the activations' type.
//
// A group of G threads holds a row, 8 * NCH elements a thread, and walks the rows with the resident blocks of the
// whole GPU; an operand's next row is on its way as soon as this one's registers are free.
#pragma once
#include "common.cuh"
#include "rows.cuh"
#include "rows_launch.h"

namespace gcdr {
namespace {

__device__ __forceinline__ float nan_max(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

// Group-wide reductions: shuffles inside a warp, one shared slot per warp beyond.  The slots
// alternate between two sets, so one barrier per reduction is enough.
template <int G>
struct Group {
    float *slots;
    int turn = 0;
    // every warp's value, one a lane (lanes beyond the warps repeat them)
    __device__ __forceinline__ float exchange(float v) {
        constexpr int W = G > 32 ? G / 32 : 1;
        float *s = slots + turn * W;
        turn ^= 1;
        if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
        __syncthreads();
        return s[threadIdx.x % W];
    }
    template <int N>
    static __device__ __forceinline__ float sum_lanes(float v) {
#pragma unroll
        for (int o = N / 2; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
        return v;
    }
    __device__ __forceinline__ float sum(float v) {
        v = sum_lanes<(G < 32 ? G : 32)>(v);
        if (G > 32) v = sum_lanes<(G > 32 ? G / 32 : 1)>(exchange(v));
        return v;
    }
    // of magnitudes; NaN when any is NaN (their bits order as the numbers do, NaN last)
    __device__ __forceinline__ float top(float v) {
        if (G < 32) {
#pragma unroll
            for (int o = G / 2; o; o >>= 1) v = nan_max(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
            return v;
        }
        v = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(v)));
        return G > 32 ? __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(exchange(v)))) : v;
    }
};

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Four values as int8, in order: v * 127 / top to nearest even, exactly.  inv estimates 127 / top to 2^-22, so the quotient
// t lies between the products with lo = inv (1 - 2^-21) and hi = inv (1 + 2^-21); both are rounded by the addition of
// 1.5 * 2^23.  Where they differ, a border k + 1/2 lies between.
//   SHORT: v and top have 11 bits or fewer.  A quotient of theirs that is no border is at least t 2^-20 from one
//     (254 v - (2 k + 1) top is a whole number of v's last places, each t / 254 of top's or more), further than
//     lo and hi reach: t IS the border, and of k and k + 1 the even one is wanted.  Their sum, at twice the size,
//     rounds to exactly that.  (Borders are common then: a bf16 row whose largest mantissa is 254 / 256 has half of
//     its values on one.)
//   else the sign of 127 v - (k + 1/2) top decides, whose two products and their rests are exact in fp32 (31 and 32
//     bits).
template <bool SHORT>
__device__ __forceinline__ uint32_t round4(const float2 *v, float top, float lo, float hi) {
    constexpr float kMagic = 12582912.f;
    uint32_t a[4];
    if constexpr (SHORT) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float2 s = __fadd2_rn(__ffma2_rn(v[i], both(lo), both(kMagic)), __ffma2_rn(v[i], both(hi), both(kMagic)));
            a[2 * i] = __float_as_uint(s.x);
            a[2 * i + 1] = __float_as_uint(s.y);
        }
    } else {
        uint32_t c[4];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float2 p = __ffma2_rn(v[i], both(lo), both(kMagic)), q = __ffma2_rn(v[i], both(hi), both(kMagic));
            a[2 * i] = __float_as_uint(p.x);
            a[2 * i + 1] = __float_as_uint(p.y);
            c[2 * i] = a[2 * i] ^ __float_as_uint(q.x);
            c[2 * i + 1] = a[2 * i + 1] ^ __float_as_uint(q.y);
        }
        if (c[0] | c[1] | c[2] | c[3]) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float x = i & 1 ? v[i / 2].y : v[i / 2].x;
                const float k = floorf(x * lo), h = k + 0.5f;
                const float p = __fmul_rn(127.f, x), m = __fmul_rn(h, top);
                const float d = (p - m) + (fmaf(127.f, x, -p) - fmaf(h, top, -m));
                const float q = d > 0.f ? k + 1.f : d < 0.f ? k : 2.f * rintf(h * 0.5f);
                a[i] = c[i] ? __float_as_uint(q + kMagic) : a[i];
            }
        }
    }
    return __byte_perm(__byte_perm(a[0], a[1], 0x0040), __byte_perm(a[2], a[3], 0x0040), 0x5410);
}

// Rows beyond these are scaled by a power of two first (exact), so that 127 / top and the
// products of round4 stay normal numbers.
__device__ __forceinline__ float row_lift(float top) {
    return top < 0x1p-60f ? 0x1p60f : top > 0x1p60f ? 0x1p-60f : 1.f;
}

// top / 127, correctly rounded: a quotient by the rounded 1 / 127 and one correction from its exact rest (Markstein,
// IBM J. Res. Dev. 34, 1990); the plain division where the rest could be lost below the normal numbers
__device__ __forceinline__ float row_scale(float top) {
    constexpr float r = 1.f / 127.f;
    const float q = top * r;
    return top > 0x1p-90f ? fmaf(fmaf(-q, 127.f, top), r, q) : top / 127.f;
}

// 1 / sqrt(a): rsqrtf and a step of Newton's iteration (0 for an infinite a)
__device__ __forceinline__ float inv_sqrt(float a) {
    const float r = rsqrtf(a);
    return isinf(a) ? 0.f : fmaf(0.5f * r, fmaf(-a * r, r, 1.f), r);
}

// What a thread holds of a row: 8 * NCH elements, in 16-byte pieces of neighbours G pieces apart, or, where
// rows are not aligned, pairs or single ones G apart.  `raw` keeps them as they lie in memory.  Pointers are those of the
// thread's first element, `left` what the row has from there on.
// FIT: kOdd rows start anywhere, kPair rows are whole pairs of elements (8192 x 2046 fp16, both LayerNorm and a gate: 33 us
// against 44 by single elements; to int8 9.9 and 13.1; fp32 norm 51 and 53), kVec rows whole 16-byte pieces, kFull rows
// too and fill their group (nothing lies past the end).
enum Fit : int { kOdd, kPair, kVec, kFull };
template <class T, int G, int NCH, Fit FIT>
struct RowPart {
    static constexpr bool VEC = FIT >= kVec;
    static constexpr int E = 8 * NCH;
    static constexpr int P = VEC ? 16 / (int)sizeof(T) : FIT == kPair ? 2 : 1;        // elements of a piece
    using Pair = typename std::conditional<sizeof(T) == 4, uint2, uint32_t>::type;
    using Raw = typename std::conditional<VEC, uint4, typename std::conditional<FIT == kPair, Pair, T>::type>::type;
    Raw raw[E / P];
    static __device__ __forceinline__ constexpr int at(int j) { return j / P * G * P + j % P; }
    static __device__ __forceinline__ bool in(int j, int left) { return FIT == kFull || at(j) < left; }
    __device__ __forceinline__ void load(const T *p, int left) {
#pragma unroll
        for (int i = 0; i < E / P; i++) {
            if (in(i * P, left)) raw[i] = *reinterpret_cast<const Raw *>(p + at(i * P));
            else if constexpr (P > 1) raw[i] = Raw();
            else raw[i] = from_f32<T>(0.f);
        }
    }
    __device__ __forceinline__ void get(float2 *v) const {
#pragma unroll
        for (int i = 0; i < E / P; i++) {
            if constexpr (P == 1) {
                (i & 1 ? v[i / 2].y : v[i / 2].x) = to_f32(raw[i]);
            } else if constexpr (!VEC && sizeof(T) == 4) {
                v[i] = make_float2(__uint_as_float(raw[i].x), __uint_as_float(raw[i].y));
            } else if constexpr (!VEC) {
                unpack2(raw[i], &v[i].x, T());
            } else if constexpr (sizeof(T) == 4) {
                v[2 * i] = make_float2(__uint_as_float(raw[i].x), __uint_as_float(raw[i].y));
                v[2 * i + 1] = make_float2(__uint_as_float(raw[i].z), __uint_as_float(raw[i].w));
            } else {
                unpack2(raw[i].x, &v[4 * i].x, T());
                unpack2(raw[i].y, &v[4 * i + 1].x, T());
                unpack2(raw[i].z, &v[4 * i + 2].x, T());
                unpack2(raw[i].w, &v[4 * i + 3].x, T());
            }
        }
    }
    static __device__ __forceinline__ void store(T *p, int left, const float2 *v) {
#pragma unroll
        for (int i = 0; i < E / P; i++) {
            if (!in(i * P, left)) continue;
            if constexpr (P == 1) {
                p[at(i)] = from_f32<T>(i & 1 ? v[i / 2].y : v[i / 2].x);
            } else if constexpr (!VEC && sizeof(T) == 4) {
                *reinterpret_cast<float2 *>(p + at(2 * i)) = v[i];
            } else if constexpr (!VEC) {
                *reinterpret_cast<uint32_t *>(p + at(2 * i)) = pack2(v[i].x, v[i].y, T());
            } else if constexpr (sizeof(T) == 4) {
                *reinterpret_cast<float4 *>(p + at(4 * i)) = make_float4(v[2 * i].x, v[2 * i].y, v[2 * i + 1].x, v[2 * i + 1].y);
            } else {
                *reinterpret_cast<uint4 *>(p + at(8 * i)) =
                    make_uint4(pack2(v[4 * i].x, v[4 * i].y, T()), pack2(v[4 * i + 1].x, v[4 * i + 1].y, T()),
                               pack2(v[4 * i + 2].x, v[4 * i + 2].y, T()), pack2(v[4 * i + 3].x, v[4 * i + 3].y, T()));
            }
        }
    }
    // elements 4 k .. 4 k + 3 of a gain or shift, `fill` where there is none
    static __device__ __forceinline__ void param4(const float *p, int left, int k, float fill, float2 *v) {
        if constexpr (VEC) {
            const float4 t = in(4 * k, left) ? *reinterpret_cast<const float4 *>(p + at(4 * k)) : make_float4(fill, fill, fill, fill);
            v[0] = make_float2(t.x, t.y);
            v[1] = make_float2(t.z, t.w);
        } else if constexpr (P == 2) {
#pragma unroll
            for (int e = 0; e < 2; e++)
                v[e] = in(4 * k + 2 * e, left) ? *reinterpret_cast<const float2 *>(p + at(4 * k + 2 * e)) : both(fill);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float t = in(4 * k + e, left) ? p[at(4 * k + e)] : fill;
                (e & 1 ? v[e / 2].y : v[e / 2].x) = t;
            }
        }
    }
    // elements 8 k .. 8 k + 7 of 16-bit rows in one load of 32 bytes (two of 16 take twice the passes over the lines)
    static __device__ __forceinline__ void param8(const float *p, int left, int k, float fill, float2 *v) {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = make_float2(fill, fill);
        if (in(8 * k, left))
            asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=f"(v[0].x), "=f"(v[0].y), "=f"(v[1].x), "=f"(v[1].y), "=f"(v[2].x), "=f"(v[2].y), "=f"(v[3].x), "=f"(v[3].y)
                         : "l"(p + at(8 * k))
                         : "memory");
    }
    // the same from a table in shared memory that fills the whole group: four elements of each thread after the other
    // threads' four, so that a load's 16-byte pieces are neighbours
    static __device__ __forceinline__ void table4(uint32_t p, int k, float2 *v) {
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0].x), "=f"(v[0].y), "=f"(v[1].x), "=f"(v[1].y) : "r"(p + 16u * (G * k)) : "memory");
    }
    // the row's element at place i of the table
    static __device__ __forceinline__ int table_at(int i) { return i / 4 % G * P + at(i / (4 * G) * 4 + i % 4); }
};

// The arithmetic of a row once its group holds it: 8 * NCH elements a thread, zeros past its end (and zeros they
// stay: the mean is not taken from them, a gain and shift past the row are 1 and 0).
template <class T, int G, int NCH, Fit FIT, bool QUANT>
struct RowMath {
    using Part = RowPart<T, G, NCH, FIT>;
    static constexpr bool VEC = FIT >= kVec;
    static constexpr int E = 8 * NCH;
    // 16-bit rows of a warp or less keep the gains and shifts in shared memory, 1 and 0 past the row and where there
    // are none (57600 rows of 256 fp16, both LayerNorm: 22 us against 27 from L1, where the rows pass through and the 32 bytes
    // of a thread's eight elements take two passes; fp32 rows lose 3 % by it).
    static constexpr bool TABLE = G <= 32 && !QUANT && sizeof(T) == 2;
    static constexpr int W = G * E;         // floats of one of its four rows: g1, b1, g2, b2
    uint32_t table = 0;                     // this thread's first four elements of g1
    const RowArgs &a;
    Group<G> grp;
    const int first, left;                  // this thread's first element, and how many the row has from there
    const float *g1, *b1, *g2, *b2;

    __device__ __forceinline__ RowMath(const RowArgs &a_, float *slots, int l)
        : a(a_), grp{slots}, first(l * Part::P), left(a_.C - l * Part::P), g1(at(a_.g1)), b1(at(a_.b1)), g2(at(a_.g2)), b2(at(a_.b2)) {}
    __device__ __forceinline__ const float *at(const float *p) const { return p ? p + first : p; }
    __device__ __forceinline__ void norm(float2 *v, bool second) {
        const int kind = second ? a.pre : a.post;
        const float *g = second ? g2 : g1, *b = second ? b2 : b1;
        const float eps = second ? a.eps2 : a.eps1;
        if (kind == GCDR_NORM_LAYER) {
            float2 s = both(0.f);
#pragma unroll
            for (int i = 0; i < E / 2; i++) s = __fadd2_rn(s, v[i]);
            const float mean = grp.sum(s.x + s.y) * a.inv_C;
#pragma unroll
            for (int i = 0; i < E / 2; i++) {
                const float mx = Part::in(2 * i, left) ? -mean : 0.f, my = Part::in(2 * i + 1, left) ? -mean : 0.f;
                v[i] = __fadd2_rn(v[i], make_float2(mx, my));
            }
        }
        float2 q = both(0.f);
#pragma unroll
        for (int i = 0; i < E / 2; i++) q = __ffma2_rn(v[i], v[i], q);
        const float2 rstd = both(inv_sqrt(fmaf(grp.sum(q.x + q.y), a.inv_C, eps)));
        if constexpr (TABLE) {
            const uint32_t t = table + (second ? 8u * W : 0u);
            if (b) from_table<true>(v, rstd, t);
            else from_table<false>(v, rstd, t);
            return;
        }
        if (g && b) affine<true, true>(v, rstd, g, b);
        else if (g) affine<true, false>(v, rstd, g, b);
        else if (b) affine<false, true>(v, rstd, g, b);
        else affine<false, false>(v, rstd, g, b);
    }
    template <bool SHIFT>
    __device__ __forceinline__ void from_table(float2 *v, float2 rstd, uint32_t p) const {
#pragma unroll
        for (int k = 0; k < E / 4; k++) {
            float2 g[2], b[2];
            Part::table4(p, k, g);
            if (SHIFT) Part::table4(p + 4u * W, k, b);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float2 &x = v[2 * k + i];
                x = __fmul2_rn(x, rstd);
                x = SHIFT ? __ffma2_rn(x, g[i], b[i]) : __fmul2_rn(x, g[i]);
            }
        }
    }
    // fills the table: every thread of the block, before the first norm
    __device__ __forceinline__ void fill(float *t) {
        for (int i = threadIdx.x; i < 4 * W; i += blockDim.x) {
            const int row = i / W, c = Part::table_at(i - row * W);
            const float *p = row == 0 ? a.g1 : row == 1 ? a.b1 : row == 2 ? a.g2 : a.b2;
            t[i] = p && c < a.C ? p[c] : row & 1 ? 0.f : 1.f;
        }
        table = (uint32_t)__cvta_generic_to_shared(t) + 16u * (first / Part::P);
        __syncthreads();
    }
    template <bool GAIN, bool SHIFT>
    __device__ __forceinline__ void affine(float2 *v, float2 rstd, const float *g, const float *b) const {
        constexpr int S = VEC && sizeof(T) == 2 ? 8 : 4;      // elements of a load
#pragma unroll
        for (int k = 0; k < E / S; k++) {
            float2 tg[S / 2], tb[S / 2];
            if constexpr (S == 8) {
                if (GAIN) Part::param8(g, left, k, 1.f, tg);
                if (SHIFT) Part::param8(b, left, k, 0.f, tb);
            } else {
                if (GAIN) Part::param4(g, left, k, 1.f, tg);
                if (SHIFT) Part::param4(b, left, k, 0.f, tb);
            }
#pragma unroll
            for (int i = 0; i < S / 2; i++) {
                float2 &x = v[S / 2 * k + i];
                x = __fmul2_rn(x, rstd);
                x = GAIN && SHIFT ? __ffma2_rn(x, tg[i], tb[i]) : GAIN ? __fmul2_rn(x, tg[i]) : SHIFT ? __fadd2_rn(x, tb[i]) : x;
            }
        }
    }

    // v = N1(v), then v = x + res_scale * gate . v
    __device__ __forceinline__ void join(float2 *v, const Part &gate, const Part &x) {
        if (a.post) norm(v, false);
        float2 t[E / 2];
        if (a.gate) {
            gate.get(t);
#pragma unroll
            for (int i = 0; i < E / 2; i++) v[i] = __fmul2_rn(v[i], t[i]);
        }
        if (a.x) {
            x.get(t);
#pragma unroll
            for (int i = 0; i < E / 2; i++) v[i] = __ffma2_rn(both(a.res_scale), v[i], t[i]);
        } else {
#pragma unroll
            for (int i = 0; i < E / 2; i++) v[i] = __fmul2_rn(both(a.res_scale), v[i]);
        }
    }
    // r, N2, y and the int8 row of v (not valid: an idle group, which joins the reductions and stores nothing)
    __device__ __forceinline__ void finish(float2 *v, int64_t row, bool valid) {
        const int n = left;
        if (!QUANT) {
            if (a.r && valid) Part::store(static_cast<T *>(a.r) + row * a.ldr + first, n, v);
            if (a.pre) norm(v, true);
            if (a.y && valid) Part::store(static_cast<T *>(a.y) + row * a.ldy + first, n, v);
        }
        if (QUANT || a.q) quant(v, row, valid);
    }
    __device__ __forceinline__ void quant(float2 *v, int64_t row, bool valid) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < E / 2; i++) top = nan_max(top, nan_max(fabsf(v[i].x), fabsf(v[i].y)));
        top = grp.top(top);
        // an infinity or NaN anywhere in the row: the scale says so, the bytes are zero
        const bool fine = top < __int_as_float(0x7F800000), some = fine && top > 0.f;
        const float lift = row_lift(top);
        if (first == 0 && valid) a.qs[row] = fine ? row_scale(top) : __int_as_float(0x7FC00000);
        if (lift != 1.f || !some) {
#pragma unroll
            for (int i = 0; i < E / 2; i++) v[i] = some ? __fmul2_rn(v[i], both(lift)) : both(0.f);
        }
        top *= lift;
        const float inv = some ? __fdividef(127.f, top) : 0.f, lo = inv * (1.f - 0x1p-21f), hi = inv * (1.f + 0x1p-21f);
        if (!valid) return;
        int8_t *p = a.q + row * a.ldq + first;
        const int n = left;
        uint32_t last = 0;
#pragma unroll
        for (int i = 0; i < E / 4; i++) {
            const uint32_t w = round4<QUANT && sizeof(T) == 2>(v + 2 * i, top, lo, hi);
            if constexpr (FIT == kPair) {
#pragma unroll
                for (int e = 0; e < 2; e++)
                    if (Part::in(4 * i + 2 * e, n)) *reinterpret_cast<uint16_t *>(p + Part::at(4 * i + 2 * e)) = (uint16_t)(w >> (16 * e));
            } else if constexpr (!VEC) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (Part::in(4 * i + e, n)) p[Part::at(4 * i + e)] = (int8_t)(w >> (8 * e));
            } else if constexpr (sizeof(T) == 4) {
                if (Part::in(4 * i, n)) *reinterpret_cast<uint32_t *>(p + Part::at(4 * i)) = w;
            } else if (i & 1) {
                if (Part::in(4 * i - 4, n)) *reinterpret_cast<uint2 *>(p + Part::at(4 * i - 4)) = make_uint2(last, w);
            }
            last = w;
        }
    }

    // the gate's row of token t
    __device__ __forceinline__ const T *gate_row(int64_t t) const {
        const int64_t g = a.gate_mul ? (int64_t)(__umulhi((uint32_t)t, a.gate_mul) >> a.gate_shift) : t / a.gate_rows;
        return static_cast<const T *>(a.gate) + g * a.ldg + first;
    }
};

template <class T, int G, int NCH, Fit FIT, bool QUANT>
__global__ void __launch_bounds__(G > 32 ? G : 256) rows_kernel(const __grid_constant__ RowArgs a) {
    constexpr int RPB = G > 32 ? 1 : 256 / G;   // rows per block
    using Math = RowMath<T, G, NCH, FIT, QUANT>;
    __shared__ float slots[G > 32 ? 2 * (G / 32) : 1];
    Math m(a, slots, threadIdx.x % G);
    const bool has_x = QUANT || a.x, has_f = !QUANT && a.f, has_gate = has_f && a.gate;
    const int64_t stride = (int64_t)gridDim.x * RPB;
    const int g = threadIdx.x / G;
    typename Math::Part x, f, gate;
    // each operand's next row is loaded as soon as this one's is used up
    const auto load_x = [&](int64_t row) { x.load(static_cast<const T *>(a.x) + row * a.ldx + m.first, m.left); };
    const auto load_f = [&](int64_t row) { f.load(static_cast<const T *>(a.f) + row * a.ldf + m.first, m.left); };
    const auto clip = [&](int64_t row) { return row < a.rows ? row : a.rows - 1; };   // idle groups join the shuffles
    int64_t base = (int64_t)blockIdx.x * RPB;
    pdl_trigger();   // (every block is resident: the next kernel sets itself up meanwhile, 89.7 us a launch against 94.8)
    pdl_wait();
    if (has_f) load_f(clip(base + g));
    if (has_gate) gate.load(m.gate_row(clip(base + g)), m.left);
    if (has_x) load_x(clip(base + g));
    if constexpr (Math::TABLE) {
        __shared__ float table[4 * Math::W];
        m.fill(table);
    }
    for (; base < a.rows; base += stride) {
        const int64_t row = base + g, next = clip(row + stride);
        const bool more = base + stride < a.rows;
        float2 v[Math::E / 2];
        if (has_f) {
            f.get(v);
            if (more) load_f(next);
            m.join(v, gate, x);
            if (more && has_gate) gate.load(m.gate_row(next), m.left);
        } else {
            x.get(v);
        }
        if (more && has_x) load_x(next);
        m.finish(v, clip(row), row < a.rows);
    }
}

int sm_count() {
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms;
}

// Blocks of a kernel that an SM holds at once (asked once per kernel: the grid is a multiple of the resident blocks)
template <class K>
int resident(K k, int threads) {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k, threads, 0) != cudaSuccess || n < 1) n = 1;
    return n;
}

template <class T, int G, int NCH, Fit FIT, bool QUANT>
cudaError_t launch_rows(const RowArgs &a, cudaStream_t st) {
    constexpr int T_ = G > 32 ? G : 256;
    constexpr int RPB = G > 32 ? 1 : 256 / G;
    auto k = rows_kernel<T, G, NCH, FIT, QUANT>;
    static const int blocks = resident(k, T_);
    const int64_t want = (a.rows + RPB - 1) / RPB, most = (int64_t)sm_count() * blocks;
    return launch_pdl(k, dim3((unsigned)(want < most ? want : most)), dim3(T_), 0, st, a);
}

template <class T, int G, int NCH, bool QUANT>
cudaError_t launch_rows(const RowArgs &a, int piece, cudaStream_t st) {
    if (piece < 16) return piece ? launch_rows<T, G, NCH, kPair, QUANT>(a, st) : launch_rows<T, G, NCH, kOdd, QUANT>(a, st);
    return a.C == 8 * G * NCH ? launch_rows<T, G, NCH, kFull, QUANT>(a, st) : launch_rows<T, G, NCH, kVec, QUANT>(a, st);
}

}  // namespace

// G and NCH by the row's length: 16 elements a thread, 24 where that leaves fewer threads idle (4099 rows of 1037 fp32
// elements to int8: 64 x 24 4.7 us, 128 x 16 5.7).  The norms of long 16-bit rows, whose reductions cost as much as their
// bytes, take 32 in half the threads (both LayerNorm, bf16: 16384 rows of 4096 128 x 32 95 us, 256 x 16 108; 8192 of 8192
// 256 x 32 107, 512 x 16 143; 16384 of 2048 64 x 32 48, 128 x 16 54); shorter rows, fp32 rows and the rounding alone do
// not (1024 bf16 64 x 16 51 us, 32 x 32 50, RMS 46 and 49; 8192 to int8 512 x 16 40, 256 x 32 45).  Beyond 8192 the
// registers of larger blocks decide (4096 rows of 16384 bf16, RMS: 512 x 32 97 us, 1024 x 16 147; to int8 46 and 41).
// Past 8192 elements in fp32, and past 12288 (odd places) or 16384 in 16 bits, these blocks' registers do not hold a row beside
// the next one's operands: part of them lies in local memory (fp32 norms 60 bytes a thread up to 12288 elements, 0.4 KB up to
// 16384, 1.7 to 4.2 KB at 32768; both LayerNorm with a gate, over the floor of their bytes: fp32 12288 1.2, 16384 1.6, 24576
// 2.9, 32768 7.3 times; fp16 16384 1.5, 24576 2.4, 32768 2.9).
template <class T, bool QUANT>
cudaError_t rows_launch(const RowArgs &a, int piece, cudaStream_t st) {
    const auto fits = [&](int g, int nch) { return a.C <= 8 * g * nch; };
    constexpr bool LONG = !QUANT && sizeof(T) == 2;
    if (fits(8, 1)) return launch_rows<T, 8, 1, QUANT>(a, piece, st);
    if (fits(8, 2)) return launch_rows<T, 8, 2, QUANT>(a, piece, st);
    if (fits(8, 3)) return launch_rows<T, 8, 3, QUANT>(a, piece, st);
    if (fits(16, 2)) return launch_rows<T, 16, 2, QUANT>(a, piece, st);
    if (fits(16, 3)) return launch_rows<T, 16, 3, QUANT>(a, piece, st);
    if (fits(32, 2)) return launch_rows<T, 32, 2, QUANT>(a, piece, st);
    if (fits(32, 3)) return launch_rows<T, 32, 3, QUANT>(a, piece, st);
    if (fits(64, 2)) return launch_rows<T, 64, 2, QUANT>(a, piece, st);
    if (fits(64, 3)) return launch_rows<T, 64, 3, QUANT>(a, piece, st);
    if (fits(64, 4)) return launch_rows<T, LONG ? 64 : 128, LONG ? 4 : 2, QUANT>(a, piece, st);
    if (fits(128, 3)) return launch_rows<T, 128, 3, QUANT>(a, piece, st);
    if (fits(128, 4)) return launch_rows<T, LONG ? 128 : 256, LONG ? 4 : 2, QUANT>(a, piece, st);
    if (fits(256, 3)) return launch_rows<T, 256, 3, QUANT>(a, piece, st);
    if (fits(256, 4)) return launch_rows<T, LONG ? 256 : 512, LONG ? 4 : 2, QUANT>(a, piece, st);
    if (!QUANT && fits(512, 3)) return launch_rows<T, 512, 3, QUANT>(a, piece, st);
    if (fits(512, 4)) return launch_rows<T, QUANT ? 1024 : 512, QUANT ? 2 : 4, QUANT>(a, piece, st);
    if (fits(1024, 3)) return launch_rows<T, 1024, 3, QUANT>(a, piece, st);
    return launch_rows<T, 1024, 4, QUANT>(a, piece, st);
}

}  // namespace gcdr

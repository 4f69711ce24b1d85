// rows.cu -- the entries of the row operators (gcdr_k_quant_rows, gcdr_k_block_norm): checks and dispatch; the
// kernels are in rows_kernel.cuh.
#include <cstdio>

#include "rows.cuh"
#include "rows_launch.h"

namespace gcdr {
namespace {

template <bool QUANT>
int launch(const char *who, const RowArgs &a, int dtype, int piece, cudaStream_t st) {
    const cudaError_t e = dtype == GCDR_DTYPE_F16    ? rows_launch<__half, QUANT>(a, piece, st)
                          : dtype == GCDR_DTYPE_BF16 ? rows_launch<__nv_bfloat16, QUANT>(a, piece, st)
                                                     : rows_launch<float, QUANT>(a, piece, st);
    if (e == cudaSuccess) return GCDR_OK;
    cudaGetLastError();
    return refuse(who, GCDR_ERR_DEVICE, cudaGetErrorString(e));
}

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
    a.inv_C = 1.f / C;
    a.x = x;
    a.ldx = ldx;
    a.q = q;
    a.ldq = ldq;
    a.qs = scale;
    // n elements at a time: pieces of an activation's row and of an int8 row
    const auto whole = [&](int n, int bytes) { return C % n == 0 && aligned(x, ldx * size, bytes) && aligned(q, ldq, n); };
    return launch<true>(who, a, dtype, whole(8, 16) ? 16 : whole(2, 2 * size) ? 2 : 0, static_cast<cudaStream_t>(stream));
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
    a.inv_C = 1.f / C;
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
    if (d->gate && d->gate_rows > 1 && n < (int64_t)1 << 31) {
        // m = ceil(2^(32 + s) / d) with 2^s >= d / 2: t m / 2^(32 + s) exceeds t / d by less than 1 / d for t < 2^31
        const uint64_t per = (uint64_t)(d->gate_rows < n ? d->gate_rows : n);
        while (((uint64_t)2 << a.gate_shift) < per) a.gate_shift++;
        a.gate_mul = (uint32_t)((((uint64_t)1 << (32 + a.gate_shift)) + per - 1) / per);
    }
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
    // n elements at a time: pieces of the activations' rows, of an int8 row and of the gains and shifts
    const auto whole = [&](int n, int bytes) {
        return C % n == 0 && aligned(d->x, d->ldx * size, bytes) && aligned(d->f, d->ldf * size, bytes) &&
               aligned(d->gate, d->ldg * size, bytes) && aligned(d->r, d->ldr * size, bytes) && aligned(d->y, d->ldy * size, bytes) &&
               aligned(d->q, d->ldq, n) && aligned(g1, 0, 4 * n) && aligned(b1, 0, 4 * n) && aligned(g2, 0, 4 * n) && aligned(b2, 0, 4 * n);
    };
    return launch<false>(who, a, d->dtype, whole(8, 16) ? 16 : whole(2, 2 * size) ? 2 : 0, static_cast<cudaStream_t>(stream));
}

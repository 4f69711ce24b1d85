// int8_tc.cu -- the int8 token product on the 5th-generation tensor cores (sm_100a).
//
// tcgen05.mma.kind::i8 multiplies int8 tiles into int32 accumulators in TMEM: exact sums, whatever
// the order.  A unit of work is a tile of 128 rows of one operand ("P", the MMA's M) times bn rows of
// the other ("Q", its N), K in blocks of 128 bytes:
//
//   wide form     P = tokens, Q = channels.  A thread of the epilogue holds a token's results in a row;
//                 they go through a per-warp stage in shared memory, so that a store instruction writes
//                 64 neighbouring bytes of eight tokens instead of 16 bytes of 32.
//   narrow form   P = channels, Q = tokens (few of them): the weights' rows fill the 128 MMA rows that
//                 few tokens would leave empty, and a warp's 32 channels are neighbours in the result.
//                 K is split over the CTAs of a cluster when the tiles do not fill the GPU: their int32
//                 sums are joined through distributed shared memory, each CTA finishing a share of the
//                 tokens.  (Integers: the join is exact and the same at any split.)
//
// 12 warps: TMA producer, MMA issuer, TMEM allocation, one idle, 8 epilogue warps (two per TMEM lane
// quadrant).  Accumulators are double-buffered in TMEM: a unit's epilogue runs under the next one's MMAs.
// The tail of K and rows past an operand's end arrive as zeros (TMA fill).  Every mbarrier wait is
// bounded, as in conv_tc.cu.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <cstdio>
#include <string>

#include "conv_launch.h"
#include "int8.h"
#include "rows.cuh"
#include "tc_util.cuh"

namespace gcdr {
namespace {

__device__ int g_i8_err;   // set by a kernel whose bounded wait ran out (GCDR_ERR_FLAG_*)

constexpr int kEpiWarps = 8;
constexpr int kFirstEpi = 4;
constexpr int kThreads = (kFirstEpi + kEpiWarps) * 32;
constexpr int kBlockK = 128;                       // bytes of K per ring stage (one 128-byte swizzle row)
constexpr int kRingStages = 12;
constexpr int kPBytes = 128 * kBlockK;
constexpr int kStageBytes = 2048;                  // an epilogue warp's store stage: 32 rows of 64 bytes
constexpr int kSmemCap = 227 * 1024;
constexpr int kXchPitch = 129;                     // int32 words per column of the split's exchange (odd: no bank conflicts)

struct I8Plan {
    int narrow;          // P = channels
    int bn;              // rows of Q per unit
    int split;           // CTAs per cluster, each a share of K (narrow form)
    int stages;
    int kblocks;
    int tiles_p, tiles_q;
    int group;           // P tiles walked per Q tile: their operands stay in L2
    int extra_bytes;     // store stages and scales (wide), exchange (split)
};

struct I8Shared {
    uint64_t full[kRingStages], empty[kRingStages], tfull[2], tempty[2], mdone;
    uint32_t tmem_base;
    int abort_flag, peer_abort;
    int issued, consumed;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_to(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, int v) {
    asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// D = int32, A and B signed int8, both K-major, N >> 3 at [17, 23), M >> 4 at [24, 29)
__device__ __forceinline__ uint32_t idesc_i8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void mma_i8(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(idesc), "r"(accum));
}

__device__ __forceinline__ float scaled(int acc, float xs, float ws, float bias, int relu) {
    const float v = fmaf((float)acc * xs, ws, bias);
    return relu && v < 0.f ? 0.f : v;   // (a NaN stays)
}

// Unit u -> its P and Q tiles: `group` P tiles per Q tile, then the next Q tile.
__device__ __forceinline__ void unit_tiles(const I8Plan &pl, int u, int &pt, int &qt) {
    const int per = pl.group * pl.tiles_q;
    const int g = u / per, r = u - g * per;
    const int left = pl.tiles_p - g * pl.group;
    const int n = left < pl.group ? left : pl.group;
    qt = r / n;
    pt = g * pl.group + r - qt * n;
}

template <class T, bool NARROW>
__global__ void __launch_bounds__(kThreads, 1)
    i8_tc_kernel(const __grid_constant__ CUtensorMap tmP, const __grid_constant__ CUtensorMap tmQ,
                 const __grid_constant__ I8Args a, const __grid_constant__ I8Plan pl) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int bn = pl.bn;
    const int stage_bytes = kPBytes + bn * kBlockK;
    uint8_t *extra = ring + (size_t)pl.stages * stage_bytes;
    I8Shared *sh = reinterpret_cast<I8Shared *>(extra + pl.extra_bytes);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = NARROW ? pl.split : 1;
    const uint32_t rank = split > 1 ? cluster_rank() : 0;
    const int first = blockIdx.x / split, stride = gridDim.x / split;
    const int units = pl.tiles_p * pl.tiles_q;
    const int kb0 = (int)((long long)pl.kblocks * rank / split), kb1 = (int)((long long)pl.kblocks * (rank + 1) / split);
    const uint32_t tmem_cols = 2u * bn;

    if (threadIdx.x == 0) {
        for (int s = 0; s < pl.stages; s++) {
            mbar_init(&sh->full[s], 1);
            mbar_init(&sh->empty[s], 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&sh->tfull[b], 1);
            mbar_init(&sh->tempty[b], kEpiWarps);
        }
        mbar_init(&sh->mdone, 1);
        sh->abort_flag = sh->peer_abort = 0;
        sh->issued = sh->consumed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        __syncwarp();
        tmem_alloc(&sh->tmem_base, tmem_cols);
    }
    tc_fence_before();
    __syncthreads();
    if (split > 1) cluster_sync();       // the other CTAs run: their shared memory may be written
    tc_fence_after();
    const uint32_t tmem_base = sh->tmem_base;
    volatile int *abort_flag = &sh->abort_flag;
    const long long budget = a.wait_cycles > 0 ? a.wait_cycles : kWaitCycles;
    pdl_trigger();
    pdl_wait();

    if (warp == 0) {
        if (lane == 0 && !a.timeout_probe) {   // (the probe issues nothing: the other roles' waits run out)
            int s = 0, issued = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int u = first; u < units && ok; u += stride) {
                int pt, qt;
                unit_tiles(pl, u, pt, qt);
                for (int kb = kb0; kb < kb1; kb++) {
                    if (!mbar_wait(&sh->empty[s], ph ^ 1u, abort_flag, &g_i8_err, budget)) { ok = false; break; }
                    uint8_t *st = ring + (size_t)s * stage_bytes;
                    mbar_expect_tx(&sh->full[s], (uint32_t)stage_bytes);
                    tma_load_2d(st, &tmP, kb * kBlockK, pt * 128, &sh->full[s]);
                    tma_load_2d(st + kPBytes, &tmQ, kb * kBlockK, qt * bn, &sh->full[s]);
                    issued++;
                    if (++s == pl.stages) { s = 0; ph ^= 1u; }
                }
            }
            sh->issued = issued;
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint64_t desc0 = sdesc(0, 8 * kBlockK, 2);
            const uint32_t idesc = idesc_i8(128, bn);
            int s = 0, t = 0, consumed = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int u = first; u < units && ok; u += stride, t++) {
                const int ab = t & 1;
                if (!mbar_wait(&sh->tempty[ab], (uint32_t)((t >> 1) & 1) ^ 1u, abort_flag, &g_i8_err, budget)) break;
                tc_fence_after();
                const uint32_t d = tmem_base + (uint32_t)(ab * bn);
                for (int kb = kb0; kb < kb1; kb++) {
                    if (!mbar_wait(&sh->full[s], ph, abort_flag, &g_i8_err, budget)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t st = smem_u32(ring + (size_t)s * stage_bytes);
                    const uint64_t ad = desc0 | (uint64_t)((st & 0x3FFFFu) >> 4);
                    const uint64_t bd = desc0 | (uint64_t)(((st + kPBytes) & 0x3FFFFu) >> 4);
#pragma unroll
                    for (int k = 0; k < kBlockK / 32; k++)
                        mma_i8(d, ad + (uint64_t)(k * 2), bd + (uint64_t)(k * 2), idesc, (kb > kb0 || k) ? 1u : 0u);
                    mma_commit(&sh->empty[s]);
                    consumed++;
                    if (++s == pl.stages) { s = 0; ph ^= 1u; }
                }
                if (ok) mma_commit(&sh->tfull[ab]);
            }
            sh->consumed = consumed;
            if (*abort_flag) {   // every MMA issued is done (bounded) before TMEM is freed
                mma_commit(&sh->mdone);
                const long long t0 = clock64();
                while (!mbar_try(&sh->mdone, 0) && clock64() - t0 < kWaitCycles) {}
            }
        }
    } else if (warp >= kFirstEpi) {
        const int e = warp - kFirstEpi, quad = warp & 3, part = e >> 2;
        const int row = quad * 32 + lane;
        const uint32_t lane_base = tmem_base + ((uint32_t)(quad * 32) << 16);
        int t = 0;
        for (int u = first; u < units; u += stride, t++) {
            int pt, qt;
            unit_tiles(pl, u, pt, qt);
            const int ab = t & 1;
            const int64_t n0 = NARROW ? (int64_t)pt * 128 : (int64_t)qt * bn;
            const int64_t m0 = NARROW ? (int64_t)qt * bn : (int64_t)pt * 128;
            // the tile's channel scales and biases, before its sums arrive
            float *sc = reinterpret_cast<float *>(extra + kEpiWarps * kStageBytes) + ab * 512;
            float rs = 0.f, rb = 0.f;
            if (NARROW) {
                if (n0 + row < a.N) {
                    rs = a.ws[n0 + row];
                    rb = a.bias ? a.bias[n0 + row] : 0.f;
                }
            } else {
                const int i = threadIdx.x - kFirstEpi * 32;
                if (i < bn) {
                    const bool in = n0 + i < a.N;
                    sc[i] = in ? a.ws[n0 + i] : 0.f;
                    sc[256 + i] = in && a.bias ? a.bias[n0 + i] : 0.f;
                }
                if (m0 + row < a.M) rs = a.xs[m0 + row];
            }
            const bool ok = mbar_wait(&sh->tfull[ab], (uint32_t)((t >> 1) & 1), abort_flag, &g_i8_err, budget);
            // the epilogue warps go on or leave together
            uint32_t bad;
            asm volatile(
                "{\n\t.reg .pred p, q;\n\t"
                "setp.eq.u32 p, %1, 0;\n\t"
                "bar.red.or.pred q, 1, %2, p;\n\t"
                "selp.u32 %0, 1, 0, q;\n\t}"
                : "=r"(bad)
                : "r"((uint32_t)ok), "n"(kEpiWarps * 32)
                : "memory");
            if (bad) break;
            tc_fence_after();
            TmemLoader ld{lane_base + (uint32_t)(ab * bn)};
            if (NARROW && split > 1) {
                // to the CTA that finishes these tokens: its slot of this CTA, [token][channel]
                const uint32_t own = smem_u32(extra);
                const int cols = (bn + split - 1) / split;
                for (int c0 = part * 16; c0 < bn && m0 + c0 < a.M; c0 += 32) {
                    uint32_t r[16];
                    ld.load16_nw(r, c0);
                    TmemLoader::wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        const int c = c0 + j;
                        if (m0 + c >= a.M) break;
                        const int to = c % split, at = c / split;
                        st_cluster(map_to(own + (uint32_t)(((rank * cols + at) * kXchPitch + row) * 4), to), (int)r[j]);
                    }
                }
            } else if (NARROW) {
                T *out = static_cast<T *>(a.out);
                for (int c0 = part * 16; c0 < bn && m0 + c0 < a.M; c0 += 32) {
                    uint32_t r[16];
                    ld.load16_nw(r, c0);
                    TmemLoader::wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        const int64_t m = m0 + c0 + j;
                        if (m >= a.M) break;
                        const float v = scaled((int)r[j], a.xs[m], rs, rb, a.relu);
                        if (n0 + row < a.N) out[m * a.ldo + n0 + row] = from_f32<T>(v);
                    }
                }
            } else {
                constexpr int CW = 64 / (int)sizeof(T);       // columns of a store stage
                constexpr int E = 16 / (int)sizeof(T);        // elements of a 16-byte store
                uint8_t *stg = extra + e * kStageBytes;
                T *out = static_cast<T *>(a.out);
                const bool vec = ((reinterpret_cast<uintptr_t>(out) | (uintptr_t)(a.ldo * (int64_t)sizeof(T))) & 15) == 0;
                const int64_t mb = m0 + quad * 32;
                for (int c0 = part * CW; c0 < bn && n0 + c0 < a.N; c0 += 2 * CW) {
                    uint32_t r[CW];
                    ld.taddr = lane_base + (uint32_t)(ab * bn + c0);
                    if constexpr (CW == 32) ld.load32_nw(r);
                    else ld.load16_nw(r);
                    TmemLoader::wait_ld();
                    const float *ws = sc + c0, *bs = ws + 256;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        float v[E];
#pragma unroll
                        for (int i = 0; i < E; i++) v[i] = scaled((int)r[k * E + i], rs, ws[k * E + i], bs[k * E + i], a.relu);
                        // 16-byte pieces are stored crosswise: neither the writes (a row a lane) nor the
                        // reads (a row per four lanes) meet in a bank
                        uint4 *to = reinterpret_cast<uint4 *>(stg + lane * 64 + ((k ^ ((lane >> 1) & 3)) * 16));
                        if constexpr (sizeof(T) == 4)
                            *to = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
                        else
                            *to = make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()), pack2(v[6], v[7], T()));
                    }
                    __syncwarp();
                    const int64_t nb = n0 + c0;
                    if (vec) {
                        const int64_t n = nb + (lane & 3) * E;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int r8 = i * 8 + (lane >> 2);
                            const uint8_t *from = stg + r8 * 64 + (((lane & 3) ^ ((r8 >> 1) & 3)) * 16);
                            if (mb + r8 < a.M) {
                                T *to = out + (mb + r8) * a.ldo + n;
                                if (n + E <= a.N) *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(from);
                                else
                                    for (int k = 0; k < E && n + k < a.N; k++) to[k] = reinterpret_cast<const T *>(from)[k];
                            }
                        }
                    } else {
                        constexpr int RI = 32 / CW;           // rows per instruction
                        const int c = lane % CW;
                        for (int r0 = lane / CW; r0 < 32; r0 += RI)
                            if (mb + r0 < a.M && nb + c < a.N)
                                out[(mb + r0) * a.ldo + nb + c] = *reinterpret_cast<const T *>(
                                    stg + r0 * 64 + (((c / E) ^ ((r0 >> 1) & 3)) * 16) + (c % E) * sizeof(T));
                    }
                    __syncwarp();
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->tempty[ab]);
        }
    }

    __syncthreads();
    if (NARROW && split > 1) {
        // join: a CTA that gave up says so to all, the sums of the others are then not used
        if (threadIdx.x < split && *abort_flag) st_cluster(map_to(smem_u32(&sh->peer_abort), threadIdx.x), 1);
        cluster_sync();
        if (first < units && !*const_cast<volatile int *>(&sh->peer_abort)) {
            int pt, qt;
            unit_tiles(pl, first, pt, qt);
            const int *xch = reinterpret_cast<const int *>(extra);
            const int cols = (bn + split - 1) / split;
            const int row = threadIdx.x & 127;
            const int64_t n = (int64_t)pt * 128 + row, m0 = (int64_t)qt * bn;
            if (n < a.N) {
                const float ws = a.ws[n], bs = a.bias ? a.bias[n] : 0.f;
                for (int at = threadIdx.x >> 7; at < cols; at += kThreads / 128) {
                    const int64_t m = m0 + at * split + rank;
                    if (at * split + (int)rank >= bn || m >= a.M) break;
                    int sum = 0;
                    for (int r = 0; r < split; r++) sum += xch[(r * cols + at) * kXchPitch + row];
                    static_cast<T *>(a.out)[m * a.ldo + n] = from_f32<T>(scaled(sum, a.xs[m], ws, bs, a.relu));
                }
            }
        }
    }
    if (threadIdx.x == 0) {
        // copies issued but never consumed (only after an abort), then the arrivals of the last commits
        for (int g = sh->consumed; g < sh->issued; g++) {
            const long long t0 = clock64();
            while (!mbar_try(&sh->full[g % pl.stages], (uint32_t)((g / pl.stages) & 1)) && clock64() - t0 < kWaitCycles) {}
        }
        if (sh->consumed > 0) {
            const int g = sh->consumed - 1;
            const long long t0 = clock64();
            while (!mbar_try(&sh->empty[g % pl.stages], (uint32_t)((g / pl.stages) & 1)) && clock64() - t0 < kWaitCycles) {}
        }
    }
    __syncthreads();
    if (warp == 2) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem_base, tmem_cols);
    }
}

int pow2_at_least(int64_t v) {
    int p = 1;
    while (p < v) p <<= 1;
    return p;
}

I8Plan plan_for(const I8Args &a, int sms) {
    I8Plan pl = {};
    pl.kblocks = (a.K + kBlockK - 1) / kBlockK;
    pl.split = 1;
    const auto div = [](int64_t v, int d) { return (int)((v + d - 1) / d); };
    if (a.M <= 64) {
        pl.narrow = 1;
        pl.bn = a.M <= 16 ? 16 : pow2_at_least(a.M);
        pl.tiles_p = div(a.N, 128);
        pl.tiles_q = div(a.M, pl.bn);
        while (pl.split < 8 && 2 * pl.split <= pl.kblocks && (int64_t)pl.tiles_p * pl.tiles_q * pl.split * 2 <= sms) pl.split *= 2;
    } else {
        // the widest tile that still gives every SM one; 64 columns at least
        pl.bn = 256;
        while (pl.bn > 64 && ((int64_t)div(a.M, 128) * div(a.N, pl.bn) < sms || a.N <= pl.bn / 2)) pl.bn /= 2;
        pl.tiles_p = div(a.M, 128);
        pl.tiles_q = div(a.N, pl.bn);
    }
    pl.group = pl.tiles_p < 16 ? pl.tiles_p : 16;
    pl.extra_bytes = pl.narrow ? (pl.split > 1 ? (pl.bn + pl.split) * kXchPitch * 4 : 0) : kEpiWarps * kStageBytes + 2 * 512 * 4;
    pl.extra_bytes = (pl.extra_bytes + 15) & ~15;
    const int room = kSmemCap - 1024 - pl.extra_bytes - (int)sizeof(I8Shared);
    pl.stages = room / (kPBytes + pl.bn * kBlockK);
    if (pl.stages > kRingStages) pl.stages = kRingStages;
    return pl;
}

template <class T, bool NARROW>
cudaError_t launch(const I8Args &a, const I8Plan &pl, const CUtensorMap &tp, const CUtensorMap &tq, int sms, cudaStream_t st) {
    auto k = i8_tc_kernel<T, NARROW>;
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemCap);
    if (e != cudaSuccess) return e;
    const int64_t units = (int64_t)pl.tiles_p * pl.tiles_q;
    cudaLaunchConfig_t cfg = {};
    // a split unit has a cluster of its own; else persistent CTAs walk the units
    cfg.gridDim = dim3((unsigned)(pl.split > 1 ? units * pl.split : units < sms ? units : sms));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = 1024 + (size_t)pl.stages * (kPBytes + pl.bn * kBlockK) + pl.extra_bytes + sizeof(I8Shared);
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    int n = 0;
    if (pdl_enabled()) {
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (pl.split > 1) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = pl.split;
        at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
        n++;
    }
    cfg.attrs = at;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, k, tp, tq, a, pl);
}

}  // namespace

int i8_tc_launch(const I8Args &a, cudaStream_t st, std::string &err) {
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) { err = cudaGetErrorString(e); return -1; }
    const I8Plan pl = plan_for(a, sms);
    const int64_t units = (int64_t)pl.tiles_p * pl.tiles_q;
    if (units > (1 << 30)) { err = "too many tiles"; return -1; }
    CUtensorMap tx, tw;
    if (!tma_encode_i8(&tx, a.x, a.K, a.M, a.ldx, pl.narrow ? pl.bn : 128, err) ||
        !tma_encode_i8(&tw, a.w, a.K, a.N, a.ldw, pl.narrow ? 128 : pl.bn, err))
        return -1;
    const CUtensorMap &tp = pl.narrow ? tw : tx, &tq = pl.narrow ? tx : tw;
    const auto go = [&](auto type) {
        using T = decltype(type);
        return pl.narrow ? launch<T, true>(a, pl, tp, tq, sms, st) : launch<T, false>(a, pl, tp, tq, sms, st);
    };
    e = a.dtype == GCDR_DTYPE_F16 ? go(__half()) : a.dtype == GCDR_DTYPE_BF16 ? go(__nv_bfloat16()) : go(0.f);
    if (e != cudaSuccess) {
        cudaGetLastError();
        err = cudaGetErrorString(e);
        return -1;
    }
    return 0;
}

int i8_status_word() {
    int h = 0;
    const int zero = 0;
    if (cudaMemcpyFromSymbol(&h, g_i8_err, sizeof h) != cudaSuccess ||
        (h && cudaMemcpyToSymbol(g_i8_err, &zero, sizeof zero) != cudaSuccess)) {
        cudaGetLastError();
        return GCDR_ERR_FLAG_OTHER;
    }
    return h;
}

}  // namespace gcdr

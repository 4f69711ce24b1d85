// int8_tc.cu -- the int8 token product on the 5th-generation tensor cores (sm_100a).
//
// tcgen05.mma.kind::i8 multiplies int8 tiles into int32 accumulators in TMEM: exact sums, whatever
// the order.  A unit of work is a tile of 128 or 256 rows of one operand ("P", the MMA's M) times bn rows of
// the other ("Q", its N), K in blocks of 128 bytes:
//
//   wide form     P = tokens, Q = channels.  A thread of the epilogue holds a token's results in a row;
//                 they go through a per-warp stage in shared memory, so that a tensor store or the warp's
//                 own store instructions write whole lines or halves.  Units of 256 rows are shared by the two CTAs of a cluster
//                 (cta_group::2): each loads 128 rows of P and half of Q, one issues the MMAs for both.
//   narrow form   P = channels, Q = tokens (few of them): the weights' rows fill the 128 MMA rows that
//                 few tokens would leave empty, and a warp's 32 channels are neighbours in the result.
//                 K is split over the CTAs of a cluster when the tiles do not fill the GPU: their int32
//                 sums are joined through distributed shared memory, each CTA finishing a share of the
//                 tokens.  (Integers: the join is exact and the same at any split.)
//
// 4 + EPI warps: TMA producer, MMA issuer, TMEM allocation, one idle, and the epilogue warps, which read the TMEM lane
// quadrant of their number.  Producer and issuer are one elected lane (elect.sync): the compiler then knows that one
// thread is active; under a test of the lane's number a stage's two copies cost 420 cycles instead of 240 and a block's
// four MMAs 560 instead of 260.  TMEM holds up to four accumulators; in the wide form each has its own group of epilogue
// warps, so that several units' epilogues, whose latencies add up to more than a unit's MMAs, run side by side.
// The tail of K and rows past an operand's end arrive as zeros (TMA fill).  Every mbarrier wait is
// bounded, as in conv_tc.cu.
#include <cuda.h>
#include <cuda_runtime.h>

#include <string>
#include <type_traits>

#include "conv_launch.h"
#include "int8.h"
#include "rows.cuh"
#include "tc_util.cuh"

namespace gcdr {
namespace {

__device__ int g_i8_err;   // the device's layer error word (GCDR_ERR_FLAG_*): a kernel's bounded wait ran out

constexpr int kFirstEpi = 4;
constexpr int kBlockK = 128;                       // bytes of K per ring stage (one 128-byte swizzle row)
constexpr int kRingStages = 12;
constexpr int kMaxBufs = 4;                        // accumulators in TMEM
constexpr int kPBytes = 128 * kBlockK;
// An epilogue warp's store stage: 32 rows of a 128-byte line where the stores bound the launch (16 warps), of half of
// it where a unit's latency counts (8 warps: more of them share a unit's columns).
__host__ __device__ constexpr int row_bytes(int epi) { return epi == 16 ? 128 : 64; }
constexpr int kScaleBytes = 8192;                  // channel scales and biases: two sets per accumulator
constexpr int kSmemCap = 227 * 1024;
constexpr int kXchPitch = 129;                     // int32 words per column of the split's exchange (odd: no bank conflicts)

struct I8Plan {
    int narrow;          // P = channels
    int pair;            // units of 256 rows, two CTAs each (wide form)
    int epi;             // epilogue warps: 8 or 16
    int bn;              // rows of Q per unit
    int bufs;            // accumulators
    int split;           // CTAs per cluster, each a share of K (narrow form)
    int stages;
    int kblocks;
    int tiles_p, tiles_q;
    int group;           // P tiles walked per Q tile: their operands stay in L2
    int tma_out;         // results leave by tensor store (wide form)
    int extra_bytes;     // store stages and scales (wide), exchange (split)
};

struct I8Shared {
    uint64_t full[kRingStages], empty[kRingStages], tfull[kMaxBufs], tempty[kMaxBufs], mdone;
    uint32_t tmem_base;
    int abort_flag, peer_abort;
    int issued, consumed;
    int peer_count;          // of a pair's other CTA, if it gave up: stages issued (told to the leader) or consumed
};

// One lane of the (converged) warp
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xFFFFFFFF;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(p));
    return p != 0;
}
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

__device__ __forceinline__ void prefetch_map(const CUtensorMap *m) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
}

// A box from shared memory (its own bulk group), and the waits of the lane that issued it
__device__ __forceinline__ void tma_store_2d(const CUtensorMap *map, uint32_t src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];\n\tcp.async.bulk.commit_group;" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(c0), "r"(c1), "r"(src)
                 : "memory");
}
__device__ __forceinline__ void store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void store_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// D = int32, A and B signed int8, both K-major, N >> 3 at [17, 23), M >> 4 at [24, 29)
__device__ __forceinline__ uint32_t idesc_i8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

template <int CG>
__device__ __forceinline__ void mma_i8(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
    if constexpr (CG == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
            "l"(a), "l"(b), "r"(idesc), "r"(accum));
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
            "l"(a), "l"(b), "r"(idesc), "r"(accum));
}

// The MMAs issued so far arrive on `bar` when they are done: in the pair form on that barrier of both CTAs.
template <int CG>
__device__ __forceinline__ void commit(uint64_t *bar) {
    if constexpr (CG == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                         smem_u32(bar)),
                     "h"((uint16_t)3)
                     : "memory");
    else
        mma_commit(bar);
}

// The same on this CTA's barrier alone: the other CTA of a pair does not wait for it, and could be gone when it arrives.
template <int CG>
__device__ __forceinline__ void commit_own(uint64_t *bar) {
    if constexpr (CG == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
    else
        mma_commit(bar);
}

// A box of one of the pair's CTAs, counted by the leader's barrier (`bar`: its shared::cluster address)
__device__ __forceinline__ void tma_load_pair(void *dst, const CUtensorMap *map, int c0, int c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Takes bytes that no copy will bring off a phase's count
__device__ __forceinline__ void mbar_complete_tx(uint64_t *bar, uint32_t bytes) {
    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void fence_acquire_cluster() { asm volatile("fence.acq_rel.cluster;" ::: "memory"); }

template <int CG>
__device__ __forceinline__ void alloc_tmem(uint32_t *slot, uint32_t cols) {
    if constexpr (CG == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        tmem_alloc(slot, cols);
    }
}
template <int CG>
__device__ __forceinline__ void free_tmem(uint32_t base, uint32_t cols) {
    if constexpr (CG == 2)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
    else
        tmem_dealloc(base, cols);
}

// relu_f32 of two packed results
__device__ __forceinline__ uint32_t relu2(uint32_t v, __half) {
    const __half2 h = __hmax2_nan(*reinterpret_cast<const __half2 *>(&v), __half2half2(__ushort_as_half(0)));
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t relu2(uint32_t v, __nv_bfloat16) {
    const __nv_bfloat162 h = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162 *>(&v), __bfloat162bfloat162(__ushort_as_bfloat16(0)));
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float4 ld_shared(uint32_t p) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(p) : "memory");
    return v;
}
__device__ __forceinline__ void st_shared(uint32_t p, const uint32_t *v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}

__device__ __forceinline__ uint16_t ld_shared(uint32_t p, uint16_t) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(p) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t ld_shared(uint32_t p, uint32_t) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(p) : "memory");
    return v;
}
__device__ __forceinline__ uint2 ld_shared(uint32_t p, uint2) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(p) : "memory");
    return v;
}

// A store stage's rows of RB bytes to rows at any element, V at a time; what is left of `cols` behind the last whole V
// goes element by element (U: one as its bits)
template <class V, class U, int RB>
__device__ __forceinline__ void store_rows(uint32_t from, U *to, int64_t ldo, int rows, int cols, int lane) {
    constexpr int E = sizeof(V) / sizeof(U), LR = RB / (int)sizeof(V), CL = LR < 32 ? LR : 32, RO = 32 / CL, PC = RB / 16;
    const auto at = [&](int r, int byte) { return from + (uint32_t)(r * RB + (byte ^ (PC == 8 ? r & 7 : (r >> 1) & 3) << 4)); };
    const int c = lane % CL, r0 = lane / CL, whole = cols / E;
    U *q = to + r0 * ldo + c * E;
    const int64_t step = RO * ldo;
#pragma unroll 8
    for (int i = 0; i < CL; i++, q += step) {
#pragma unroll
        for (int k = 0; k < LR; k += CL) {
            const V v = ld_shared(at(r0 + i * RO, (c + k) * (int)sizeof(V)), V());
            if (r0 + i * RO < rows && c + k < whole) *reinterpret_cast<V *>(q + k * E) = v;
        }
    }
    if (E > 1 && lane < rows)
        for (int k = whole * E; k < cols; k++) to[lane * ldo + k] = ld_shared(at(lane, k * (int)sizeof(U)), U());
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

// The result's map, a parameter of the kernels that store by it alone.
template <bool STORE> struct OutMap { CUtensorMap map; };
template <> struct OutMap<false> {};

// CG: CTAs per unit.  EPI: epilogue warps.  STORE: results leave by tensor store.
template <class T, bool NARROW, int CG, int EPI, bool STORE>
__global__ void __launch_bounds__((kFirstEpi + EPI) * 32, 1)
    i8_tc_kernel(const __grid_constant__ CUtensorMap tmP, const __grid_constant__ CUtensorMap tmQ,
                 const __grid_constant__ OutMap<STORE> out_map, const __grid_constant__ I8Args a, const __grid_constant__ I8Plan pl) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int bn = pl.bn;
    const int stage_bytes = kPBytes + bn / CG * kBlockK;
    uint8_t *extra = ring + (size_t)pl.stages * stage_bytes;
    I8Shared *sh = reinterpret_cast<I8Shared *>(extra + pl.extra_bytes);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = NARROW ? pl.split : 1;
    const int cluster = CG == 2 ? 2 : split;
    const uint32_t rank = cluster > 1 ? cluster_rank() : 0;
    const int first = blockIdx.x / cluster, stride = gridDim.x / cluster;
    const int units = pl.tiles_p * pl.tiles_q;
    const int kb0 = NARROW ? (int)((long long)pl.kblocks * rank / split) : 0;
    const int kb1 = NARROW ? (int)((long long)pl.kblocks * (rank + 1) / split) : pl.kblocks;
    const uint32_t tmem_cols = (uint32_t)(pl.bufs * bn);
    // epilogue warps of an accumulator: all of them in the narrow form, else a group of its own
    const int per_buf = NARROW ? EPI : EPI / pl.bufs;

    if (threadIdx.x == 32) {             // the tensor maps are on their way while the previous kernel ends
        prefetch_map(&tmP);
        prefetch_map(&tmQ);
        if constexpr (STORE) prefetch_map(&out_map.map);
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < pl.stages; s++) {
            mbar_init(&sh->full[s], 1);
            mbar_init(&sh->empty[s], 1);
        }
        for (int b = 0; b < pl.bufs; b++) {
            mbar_init(&sh->tfull[b], 1);
            mbar_init(&sh->tempty[b], (uint32_t)(per_buf * CG));
        }
        mbar_init(&sh->mdone, 1);
        sh->abort_flag = sh->peer_abort = 0;
        sh->issued = sh->consumed = sh->peer_count = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        __syncwarp();
        alloc_tmem<CG>(&sh->tmem_base, tmem_cols);
    }
    tc_fence_before();
    __syncthreads();
    if (cluster > 1) cluster_sync();     // the other CTAs run and have their barriers: they may be written to
    tc_fence_after();
    const uint32_t tmem_base = sh->tmem_base;
    volatile int *abort_flag = &sh->abort_flag;
    const long long budget = a.wait_cycles > 0 ? a.wait_cycles : kWaitCycles;
    pdl_trigger();
    pdl_wait();

    if (warp == 0) {
        if (elect_one() && !a.timeout_probe) {   // (the probe issues nothing: the other roles' waits run out)
            int s = 0, issued = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int u = first; u < units && ok; u += stride) {
                int pt, qt;
                unit_tiles(pl, u, pt, qt);
                for (int kb = kb0; kb < kb1; kb++) {
                    if (!mbar_wait(&sh->empty[s], ph ^ 1u, abort_flag, &g_i8_err, budget)) { ok = false; break; }
                    uint8_t *st = ring + (size_t)s * stage_bytes;
                    if constexpr (CG == 2) {
                        const uint32_t bar = map_to(smem_u32(&sh->full[s]), 0);
                        if (rank == 0) mbar_expect_tx(&sh->full[s], 2u * (uint32_t)stage_bytes);
                        tma_load_pair(st, &tmP, kb * kBlockK, pt * 256 + (int)rank * 128, bar);
                        tma_load_pair(st + kPBytes, &tmQ, kb * kBlockK, qt * bn + (int)rank * (bn / 2), bar);
                    } else {
                        mbar_expect_tx(&sh->full[s], (uint32_t)stage_bytes);
                        tma_load_2d(st, &tmP, kb * kBlockK, pt * 128, &sh->full[s]);
                        tma_load_2d(st + kPBytes, &tmQ, kb * kBlockK, qt * bn, &sh->full[s]);
                    }
                    issued++;
                    if (++s == pl.stages) { s = 0; ph ^= 1u; }
                }
            }
            sh->issued = issued;
        }
    } else if (warp == 1) {
        if (elect_one() && (CG == 1 || rank == 0)) {
            const uint64_t desc0 = sdesc(0, 8 * kBlockK, 2);
            const uint32_t idesc = idesc_i8(128 * CG, bn);
            int s = 0, ab = 0, consumed = 0;
            uint32_t ph = 0, aph = 0;
            bool ok = true;
            for (int u = first; u < units && ok; u += stride) {
                if (!mbar_wait(&sh->tempty[ab], aph ^ 1u, abort_flag, &g_i8_err, budget)) break;
                if (CG == 2) fence_acquire_cluster();    // the other CTA's epilogue has read its half
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
                        mma_i8<CG>(d, ad + (uint64_t)(k * 2), bd + (uint64_t)(k * 2), idesc, (kb > kb0 || k) ? 1u : 0u);
                    commit<CG>(&sh->empty[s]);
                    consumed++;
                    if (++s == pl.stages) { s = 0; ph ^= 1u; }
                }
                if (ok) commit<CG>(&sh->tfull[ab]);
                if (++ab == pl.bufs) { ab = 0; aph ^= 1u; }
            }
            sh->consumed = consumed;
            if (*abort_flag) {   // every MMA issued is done (bounded) before TMEM is freed
                commit_own<CG>(&sh->mdone);
                const long long t0 = clock64();
                while (!mbar_try(&sh->mdone, 0) && clock64() - t0 < kWaitCycles) {}
            }
        }
    } else if (warp >= kFirstEpi) {
        const int e = warp - kFirstEpi, quad = warp & 3;
        const int group = NARROW ? 0 : e / per_buf, parts = per_buf / 4, part = (e - group * per_buf) >> 2;
        const int gi = (int)threadIdx.x - (kFirstEpi + group * per_buf) * 32;   // thread of the group
        const int row = quad * 32 + lane;
        const uint32_t lane_base = tmem_base + ((uint32_t)(quad * 32) << 16);
        float *scales = reinterpret_cast<float *>(extra + EPI * 32 * row_bytes(EPI)) + group * 4 * bn;
        // a unit's scales: of this thread's row, and (wide) of one or two channels for the group; those of the group's
        // next unit are fetched while this one is finished
        constexpr int CH = NARROW || EPI == 16 ? 1 : 2;
        float rs = 0.f, rb = 0.f, cs[CH], cb[CH];
        const auto fetch_scales = [&](int u) {
            int pt, qt;
            unit_tiles(pl, u, pt, qt);
            if (NARROW) {
                const int64_t n = (int64_t)pt * 128 + row;
                rs = n < a.N ? a.ws[n] : 0.f;
                rb = n < a.N && a.bias ? a.bias[n] : 0.f;
            } else {
                const int64_t m = ((int64_t)pt * CG + rank) * 128 + row;
                rs = m < a.M ? a.xs[m] : 0.f;
#pragma unroll
                for (int i = 0; i < CH; i++) {
                    const int c = gi + i * per_buf * 32;
                    const int64_t n = (int64_t)qt * bn + c;
                    cs[i] = c < bn && n < a.N ? a.ws[n] : 0.f;
                    cb[i] = c < bn && n < a.N && a.bias ? a.bias[n] : 0.f;
                }
            }
        };
        const int step = NARROW ? 1 : pl.bufs;
        int ab = group, odd = 0;
        uint32_t aph = 0;
        if (first + group * stride < units) fetch_scales(first + group * stride);
        for (int u = first + group * stride; u < units; u += step * stride) {
            int pt, qt;
            unit_tiles(pl, u, pt, qt);
            const int64_t n0 = NARROW ? (int64_t)pt * 128 : (int64_t)qt * bn;
            const int64_t m0 = NARROW ? (int64_t)qt * bn : ((int64_t)pt * CG + rank) * 128;
            float *sc = scales + odd * 2 * bn;     // (the other set may still be read)
            odd ^= 1;
            const float row_s = rs, row_b = rb;
#pragma unroll
            for (int i = 0; !NARROW && i < CH; i++) {
                const int c = gi + i * per_buf * 32;
                if (c < bn) {
                    sc[c] = cs[i];
                    sc[bn + c] = cb[i];
                }
            }
            if (u + step * stride < units) fetch_scales(u + step * stride);
            const bool ok = mbar_wait(&sh->tfull[ab], aph, abort_flag, &g_i8_err, budget);
            // the accumulator's warps go on or leave together
            uint32_t bad;
            asm volatile(
                "{\n\t.reg .pred p, q;\n\t"
                "setp.eq.u32 p, %1, 0;\n\t"
                "bar.red.or.pred q, %2, %3, p;\n\t"
                "selp.u32 %0, 1, 0, q;\n\t}"
                : "=r"(bad)
                : "r"((uint32_t)ok), "r"(1 + group), "r"(per_buf * 32)
                : "memory");
            if (bad) break;
            tc_fence_after();
            TmemLoader ld{lane_base + (uint32_t)(ab * bn)};
            if (NARROW && split > 1) {
                // to the CTA that finishes these tokens: its slot of this CTA, [token][channel]
                const uint32_t own = smem_u32(extra);
                const int cols = (bn + split - 1) / split;
                for (int c0 = part * 16; c0 < bn && m0 + c0 < a.M; c0 += parts * 16) {
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
                for (int c0 = part * 16; c0 < bn && m0 + c0 < a.M; c0 += parts * 16) {
                    uint32_t r[16];
                    ld.load16_nw(r, c0);
                    TmemLoader::wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        const int64_t m = m0 + c0 + j;
                        if (m >= a.M) break;
                        const float v = i8_result((int)r[j], a.xs[m], row_s, row_b, a.relu);
                        if (n0 + row < a.N) out[m * a.ldo + n0 + row] = from_f32<T>(v);
                    }
                }
            } else {
                constexpr int E = 16 / (int)sizeof(T);        // elements of a 16-byte piece
                constexpr int RB = row_bytes(EPI), PC = RB / 16;   // bytes and pieces of a stage's row
                constexpr int CW = PC * E, LW = CW < 32 ? CW : 32;  // its columns, those of one TMEM load
                constexpr int RI = 32 / PC;                   // rows of one store instruction
                // Piece k of row r lies at r * RB + (k ^ x(r)) * 16, x = r % 8 or r / 2 % 4: neither the writes (a row a
                // lane) nor the reads (a row per PC lanes) meet in a bank.  The same x in every RI-th row but for its
                // highest bit (PC 8).
                const uint32_t stg = smem_u32(extra) + (uint32_t)(e * 32 * RB);
                const uint32_t put = stg + (uint32_t)(lane * RB + (PC == 8 ? lane & 7 : (lane >> 1) & 3) * 16);
                const uint32_t take = stg + (uint32_t)(lane / PC * RB + (lane % PC ^ (lane >> 3)) * 16);
                const int64_t mb = m0 + quad * 32, left = a.M - mb - lane / PC, step8 = RI * a.ldo;
                T *out = static_cast<T *>(a.out) + (mb + lane / PC) * a.ldo + n0 + lane % PC * E;
                const bool vec = ((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.ldo * (int64_t)sizeof(T))) & 15) == 0;
                const float2 rs2 = make_float2(row_s, row_s);
                const int c_end = a.N - n0 < bn ? (int)(a.N - n0) : bn;
                const uint32_t scale = smem_u32(sc);
                for (int c0 = part * CW; c0 < c_end; c0 += parts * CW) {
                    if (STORE) {                              // the last piece has left the stage
                        if (elect_one()) store_wait_read();
                        __syncwarp();
                    }
#pragma unroll
                    for (int h = 0; h < CW / LW; h++) {
                        uint32_t r[LW];
                        ld.taddr = lane_base + (uint32_t)(ab * bn + c0 + LW * h);
                        if constexpr (LW == 32) ld.load32_nw(r);
                        else ld.load16_nw(r);
                        TmemLoader::wait_ld();
                        const uint32_t ws = scale + (uint32_t)(c0 + LW * h) * 4u, bs = ws + (uint32_t)bn * 4u;
#pragma unroll
                        for (int k = 0; k < LW / E; k++) {
                            uint32_t p[4];
#pragma unroll
                            for (int i = 0; i < E / 4; i++) {
                                const float4 w = ld_shared(ws + (uint32_t)(k * E + 4 * i) * 4u), c = ld_shared(bs + (uint32_t)(k * E + 4 * i) * 4u);
                                const int *q = reinterpret_cast<const int *>(r) + k * E + 4 * i;
                                const float2 v0 = __ffma2_rn(__fmul2_rn(make_float2((float)q[0], (float)q[1]), rs2), make_float2(w.x, w.y), make_float2(c.x, c.y));
                                const float2 v1 = __ffma2_rn(__fmul2_rn(make_float2((float)q[2], (float)q[3]), rs2), make_float2(w.z, w.w), make_float2(c.z, c.w));
                                if constexpr (sizeof(T) == 4) {
                                    p[0] = __float_as_uint(a.relu ? relu_f32(v0.x) : v0.x);
                                    p[1] = __float_as_uint(a.relu ? relu_f32(v0.y) : v0.y);
                                    p[2] = __float_as_uint(a.relu ? relu_f32(v1.x) : v1.x);
                                    p[3] = __float_as_uint(a.relu ? relu_f32(v1.y) : v1.y);
                                } else {
                                    p[2 * i] = pack2(v0.x, v0.y, T());
                                    p[2 * i + 1] = pack2(v1.x, v1.y, T());
                                    if (a.relu) {             // (the same once rounded)
                                        p[2 * i] = relu2(p[2 * i], T());
                                        p[2 * i + 1] = relu2(p[2 * i + 1], T());
                                    }
                                }
                            }
                            st_shared(put ^ (uint32_t)((h * (LW / E) + k) * 16), p);
                        }
                    }
                    if constexpr (STORE) {
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (mb < a.M && elect_one()) tma_store_2d(&out_map.map, stg, (int)(n0 + c0), (int)mb);
                        continue;
                    }
                    __syncwarp();
                    if (vec && (a.N % E == 0 || c0 + CW <= c_end)) {
                        T *to = out + c0;
                        const bool in = c0 + lane % PC * E < c_end;
#pragma unroll
                        for (int i = 0; i < PC; i++, to += step8) {
                            const float4 v = ld_shared((PC == 8 && (i & 1) ? take ^ 64u : take) + (uint32_t)(i * RI * RB));
                            if (in && i * RI < left) *reinterpret_cast<float4 *>(to) = v;
                        }
                    } else {
                        // results at odd places, or a row's last piece cut short
                        const unsigned odd = (unsigned)(reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.ldo * (int64_t)sizeof(T))) & 15u;
                        using U = typename std::conditional<sizeof(T) == 2, uint16_t, uint32_t>::type;
                        U *to = static_cast<U *>(a.out) + mb * a.ldo + n0 + c0;
                        const int rows = a.M - mb < 32 ? (int)(a.M - mb) : 32, cols = c_end - c0 < CW ? c_end - c0 : CW;
                        if (odd % 8 == 0) store_rows<uint2, U, RB>(stg, to, a.ldo, rows, cols, lane);
                        else if (sizeof(T) == 4 || odd % 4 == 0) store_rows<uint32_t, U, RB>(stg, to, a.ldo, rows, cols, lane);
                        else store_rows<U, U, RB>(stg, to, a.ldo, rows, cols, lane);
                    }
                    __syncwarp();
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (CG == 2) arrive_cluster(map_to(smem_u32(&sh->tempty[ab]), 0));
                else mbar_arrive(&sh->tempty[ab]);
            }
            if (!NARROW || ++ab == pl.bufs) {
                if (NARROW) ab = 0;
                aph ^= 1u;
            }
        }
        if (STORE) {
            __syncwarp();
            if (elect_one()) store_wait_all();
        }
    }

    __syncthreads();
    if (NARROW && split > 1) {
        // join: a CTA that gave up says so to all, the sums of the others are then not used
        if (threadIdx.x < split && *abort_flag) st_cluster(map_to(smem_u32(&sh->peer_abort), threadIdx.x), 1);
        __syncwarp();
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
                for (int at = threadIdx.x >> 7; at < cols; at += (kFirstEpi + EPI) / 4) {
                    const int64_t m = m0 + at * split + rank;
                    if (at * split + (int)rank >= bn || m >= a.M) break;
                    int sum = 0;
                    for (int r = 0; r < split; r++) sum += xch[(r * cols + at) * kXchPitch + row];
                    static_cast<T *>(a.out)[m * a.ldo + n] = from_f32<T>(i8_result(sum, a.xs[m], ws, bs, a.relu));
                }
            }
        }
    }
    const auto done = [&](uint64_t *bars, int use) {    // the use-th phase of a ring's barriers (counted from 0)
        const long long t0 = clock64();
        while (!mbar_try(&bars[use % pl.stages], (uint32_t)((use / pl.stages) & 1)) && clock64() - t0 < kWaitCycles) {}
    };
    if (threadIdx.x == 0) {
        if (CG == 2 && *abort_flag) {    // the other CTA hears of it, and how far this one came
            st_cluster(map_to(smem_u32(&sh->peer_count), rank ^ 1), rank ? sh->issued : sh->consumed);
            st_cluster(map_to(smem_u32(&sh->peer_abort), rank ^ 1), 1);
        } else {
            // copies issued but never consumed (only after an abort), then the arrivals of the last commits (a CTA of a
            // pair that did not give up has seen all its units through: what it has issued is consumed)
            for (int g = sh->consumed; CG == 1 && g < sh->issued; g++) done(sh->full, g);
            const int last = CG == 2 ? sh->issued : sh->consumed;
            if (last > 0) done(sh->empty, last - 1);
        }
    }
    __syncthreads();
    if (CG == 2) {
        cluster_sync();                  // neither CTA's memory goes while the other's MMAs or arrivals may use it
        const bool peer = *const_cast<volatile int *>(&sh->peer_abort);
        if (peer || *abort_flag) {
            if (threadIdx.x == 0) {
                const int count = *const_cast<volatile int *>(&sh->peer_count);
                const int consumed = rank == 0 ? sh->consumed : peer ? count : sh->issued;
                const int other = rank == 0 && peer ? count : consumed;      // (issued by the other CTA)
                // Copies never consumed.  The leader's barriers count those of both CTAs; a stage that one of the two
                // has issued alone is waited for by that one's bytes.
                for (int g = consumed; rank == 0 && (g < sh->issued || g < other); g++) {
                    uint64_t *bar = &sh->full[g % pl.stages];
                    if (g >= other) mbar_complete_tx(bar, (uint32_t)stage_bytes);
                    if (g >= sh->issued) mbar_expect_tx(bar, (uint32_t)stage_bytes);
                    done(sh->full, g);
                }
                if (consumed > 0) done(sh->empty, consumed - 1);
            }
            __syncwarp();
            cluster_sync();
        }
    }
    if (warp == 2) {
        __syncwarp();
        tc_fence_after();
        free_tmem<CG>(tmem_base, tmem_cols);
    }
}

uintptr_t result_place(const I8Args &a) {   // what the starts of the result's rows are multiples of
    return reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.ldo * dtype_bytes(a.dtype));
}

// Picks form and tile by an estimate in SM cycles, fitted to measured sweeps on a B200.  Against every form forced in turn:
// 93 % of random sizes are within 15 % of the best one (K 256 to 8192, 16 to 57600 tokens, 160 to 8192 channels; and as many
// of smaller K and N), the worst 2.1 times (2.5) as slow: splits of four at 34 to 37 units, which take a second round
// (33 clusters of four fit 148 SMs), and 260 to 512 tokens with K up to 300 against thousands of channels.
//   a k-block step     what its loads and MMAs take together (a pair's for twice the rows; the second figures where
//                      rows do not start on a line: each 128 bytes are then two requests); 16 epilogue warps leave a
//                      ring stage less
//   a unit's results   at 12 bytes per cycle with 8 epilogue warps (64-byte stores), 16 with 16 of them; rows that start
//                      at multiples of 8 bytes only 10 (a pair 8) and 13, at any element 8 (6) and 11
//   a round            700 between units; the last one's results and the start are not hidden (nor, of two units, the
//                      second half of the warps)
//   a split of K       the join's words through distributed shared memory; clusters of eight fit 148 SMs 12 times
// E.g. 57600 x 256 x 256 fp16: wide 128, 16 warps 11.7 us, 8 warps 14.5, wide 256 13.0; 1213 x 1040 x 1000 fp32: wide 128
// 7.4 us, 64 8.8, 256 10.5; 128 x 8192 x 8192: wide 64 16.9 us, 128 20.1; 4096^3: pair 48 us, wide 256 53, 128 56;
// 128 x 1024 x 8192: narrow 32 split 4 9.0 us, wide 64 11.1; 16 x 1024 x 8192: split 8 6.4 us, 4 7.1, 2 9.3, none 11.3.
I8Plan plan_for(const I8Args &a, int sms) {
    const auto div = [](int64_t v, int64_t d) { return (v + d - 1) / d; };
    const int64_t kb = div(a.K, kBlockK);
    const int size = dtype_bytes(a.dtype);
    I8Plan pl = {};
    int64_t best = INT64_MAX;
    const auto offer = [&](int64_t cost, int narrow, int pair, int epi, int bn, int split) {
        if (cost >= best) return;
        best = cost;
        pl.narrow = narrow;
        pl.pair = pair;
        pl.epi = epi;
        pl.bn = bn;
        pl.split = split;
    };
    const bool cut = (a.ldx | a.ldw) % 128 != 0;   // a box's 128 bytes lie in two lines each
    const int64_t m128 = div(a.M, 128);
    const uintptr_t odd = result_place(a);
    const int e8 = odd % 16 == 0 ? 12 : odd % 8 == 0 ? 10 : 8, pair8 = odd % 16 == 0 ? 12 : odd % 8 == 0 ? 8 : 6;
    for (int bn = 64; bn <= 256; bn *= 2) {
        const int64_t tq = div(a.N, bn), units = m128 * tq, rounds = div(units, sms);
        const int64_t work = kb * (cut ? (bn == 256 ? 1300 : bn == 128 ? 950 : 670) : bn == 256 ? 740 : bn == 128 ? 430 : 300), bytes = 128 * div(a.N, tq) * size;
        const int e16 = odd % 16 == 0 ? 16 : odd % 8 == 0 ? (bn == 256 ? 11 : 13) : bn == 256 ? 10 : 11;
        const auto cost = [](int64_t r, int64_t w, int64_t e) { return r * ((w > e ? w : e) + 700) + (w > e ? e : w) + (r == 2 ? e : 0); };
        offer(cost(rounds, work, bytes / e8) + 1500, 0, 0, 8, bn, 1);
        if (rounds > 2) offer(cost(rounds, work * 11 / 10, bytes / e16) + 2000, 0, 0, 16, bn, 1);
        if (bn == 256 && a.M > 128) offer(cost(div(div(a.M, 256) * tq, sms / 2), kb * (cut ? 1000 : 650), bytes / pair8) + 5500, 0, 1, 8, bn, 1);
        if (a.N <= bn) break;
    }
    const int64_t n128 = div(a.N, 128);
    for (int bn = 16; a.M <= 512 && bn <= 128; bn *= 2) {
        const int64_t tiles = n128 * div(a.M, bn), step = (bn == 128 ? 430 : bn == 64 ? 330 : 270) * (cut ? 2 : 1);
        for (int split = 1; split <= 8 && split <= kb; split *= 2) {
            const int64_t rounds = div(tiles * split, split == 8 ? 96 : sms);
            offer(rounds * (div(kb, split) * step + (split > 1 ? 1500 + bn * 100 : 0)) + 3300 + bn * 50, 1, 0, 8, bn, split);
        }
        if (a.M <= bn) break;
    }
    pl.kblocks = (int)kb;
    pl.tiles_p = (int)(pl.narrow ? n128 : div(a.M, pl.pair ? 256 : 128));
    pl.tiles_q = (int)div(pl.narrow ? a.M : a.N, pl.bn);
    pl.group = pl.tiles_p < 16 ? pl.tiles_p : 16;
    // no more accumulators than a CTA has units: the fewer share the epilogue warps
    const int64_t each = div((int64_t)pl.tiles_p * pl.tiles_q, pl.pair ? sms / 2 : sms);
    pl.bufs = pl.narrow ? 2 : 512 / pl.bn < pl.epi / 4 ? 512 / pl.bn : pl.epi / 4;
    while (!pl.narrow && pl.bufs > 1 && pl.bufs / 2 >= each) pl.bufs /= 2;
    pl.extra_bytes = !pl.narrow ? pl.epi * 32 * row_bytes(pl.epi) + kScaleBytes : pl.split > 1 ? (pl.bn + pl.split) * kXchPitch * 4 : 0;
    pl.extra_bytes = (pl.extra_bytes + 15) & ~15;
    const int room = kSmemCap - 1024 - pl.extra_bytes - (int)sizeof(I8Shared);
    pl.stages = room / (kPBytes + pl.bn / (pl.pair ? 2 : 1) * kBlockK);
    if (pl.stages > kRingStages) pl.stages = kRingStages;
    // Several units a CTA: their results leave by tensor store (57600 x 512 x 512 fp16 21.8 us, 23.0 by the warps; a
    // single unit gains nothing by it, and its caller waits for the map).  A tensor store writes whole 16-byte pieces:
    // a row that ended inside one would spill into the space behind it.
    pl.tma_out = !pl.narrow && (int64_t)pl.tiles_p * pl.tiles_q > (pl.pair ? sms / 2 : sms) &&
                 (odd | (uintptr_t)((int64_t)a.N * size)) % 16 == 0 && a.ldo < (int64_t)1 << 36;
    return pl;
}

template <class T, bool NARROW, int CG, int EPI, bool STORE>
cudaError_t launch(const I8Args &a, const I8Plan &pl, const CUtensorMap &tp, const CUtensorMap &tq, const CUtensorMap &to, int sms,
                   cudaStream_t st) {
    auto k = i8_tc_kernel<T, NARROW, CG, EPI, STORE>;
    OutMap<STORE> out;
    if constexpr (STORE) out.map = to;
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemCap);
    if (e != cudaSuccess) return e;
    const int64_t units = (int64_t)pl.tiles_p * pl.tiles_q;
    const int cluster = CG == 2 ? 2 : pl.split;
    cudaLaunchConfig_t cfg = {};
    // a split unit has a cluster of its own; else persistent CTAs (or pairs of them) walk the units
    cfg.gridDim = dim3((unsigned)((pl.split > 1 || units < sms / CG ? units : sms / CG) * cluster));
    cfg.blockDim = dim3((kFirstEpi + EPI) * 32);
    cfg.dynamicSmemBytes = 1024 + (size_t)pl.stages * (kPBytes + pl.bn / CG * kBlockK) + pl.extra_bytes + sizeof(I8Shared);
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    int n = 0;
    if (pdl_enabled()) {
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = cluster;
        at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
        n++;
    }
    cfg.attrs = at;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, k, tp, tq, out, a, pl);
}

template <class T, bool STORE>
cudaError_t launch_wide(const I8Args &a, const I8Plan &pl, const CUtensorMap &tp, const CUtensorMap &tq, const CUtensorMap &to,
                        int sms, cudaStream_t st) {
    if (pl.pair) return launch<T, false, 2, 8, STORE>(a, pl, tp, tq, to, sms, st);
    return pl.epi == 16 ? launch<T, false, 1, 16, STORE>(a, pl, tp, tq, to, sms, st)
                        : launch<T, false, 1, 8, STORE>(a, pl, tp, tq, to, sms, st);
}

template <class T>
cudaError_t launch_form(const I8Args &a, const I8Plan &pl, const CUtensorMap &tp, const CUtensorMap &tq, const CUtensorMap &to,
                        int sms, cudaStream_t st) {
    if (pl.narrow) return launch<T, true, 1, 8, false>(a, pl, tp, tq, to, sms, st);
    return pl.tma_out ? launch_wide<T, true>(a, pl, tp, tq, to, sms, st) : launch_wide<T, false>(a, pl, tp, tq, to, sms, st);
}

}  // namespace

int i8_tc_launch(const I8Args &a, cudaStream_t st, std::string &err) {
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) { err = cudaGetErrorString(e); return -1; }
    I8Plan pl = plan_for(a, sms);
    const int64_t units = (int64_t)pl.tiles_p * pl.tiles_q;
    if (units > (1 << 30)) { err = "too many tiles"; return -1; }
    CUtensorMap tx, tw, to;
    const int q_box = pl.bn / (pl.pair ? 2 : 1);
    if (!tma_encode_rows(&tx, a.x, 1, a.K, a.M, a.ldx, kBlockK, pl.narrow ? q_box : 128, err) ||
        !tma_encode_rows(&tw, a.w, 1, a.K, a.N, a.ldw, kBlockK, pl.narrow ? 128 : q_box, err))
        return -1;
    const int size = dtype_bytes(a.dtype);
    if (pl.tma_out && !tma_encode_rows(&to, a.out, size, a.N, a.M, a.ldo * size, row_bytes(pl.epi), 32, err)) return -1;
    const CUtensorMap &tp = pl.narrow ? tw : tx, &tq = pl.narrow ? tx : tw;
    e = a.dtype == GCDR_DTYPE_F16    ? launch_form<__half>(a, pl, tp, tq, to, sms, st)
        : a.dtype == GCDR_DTYPE_BF16 ? launch_form<__nv_bfloat16>(a, pl, tp, tq, to, sms, st)
                                     : launch_form<float>(a, pl, tp, tq, to, sms, st);
    if (e != cudaSuccess) {
        cudaGetLastError();
        err = cudaGetErrorString(e);
        return -1;
    }
    return 0;
}

void i8_tc_form(const I8Args &a, int sms, gcdr_i8_form &f) {
    const I8Plan pl = plan_for(a, sms);
    f.form = pl.narrow ? GCDR_I8_NARROW : pl.pair ? GCDR_I8_PAIR : GCDR_I8_WIDE;
    f.tile = pl.bn;
    f.split = pl.split;
    f.epilogue_warps = pl.epi;
    f.accumulators = pl.bufs;
    f.tensor_store = pl.tma_out;
    f.stages = pl.stages;
    f.units = (int64_t)pl.tiles_p * pl.tiles_q;
}

int *i8_error_word() {
    void *p = nullptr;
    if (cudaGetSymbolAddress(&p, g_i8_err) == cudaSuccess) return static_cast<int *>(p);
    cudaGetLastError();
    return nullptr;
}

}  // namespace gcdr

// fp4_gemm_sm100.cu -- products of microscaled 4-bit matrices on sm_100a:
//     out[m, n] = round16( sum_k a[m, k] b[n, k]  [* ga[m] * gb[n]] )
// with a and b as codes, block scales and (NV) row scales of fp4_rows_sm100.cu, and the gated form
//     out = round16( silu(a gate^T) * (a up^T) ).
//
// The tensor cores take the codes as they are stored and apply the block scales themselves
// (tcgen05.mma .block_scale, kind mxf4 and mxf4nvf4: 64 values of K per instruction, f32 accumulators in tensor
// memory), so nothing is decoded on the way: TMA brings 128-byte-swizzled blocks of 256 values of K per row and the scale tiles that
// belong to them, and tcgen05.cp moves those to tensor memory, where the instruction reads them. Row scales are applied to the
// accumulators (scale_rows); the quantiser's are powers of two, for which that is exact.
//
// Three forms, by what bounds them (gemm_fp4_dispatch chooses):
//   split      few rows or few tiles: latency, and reading the weights. One tile per CTA, K split over a cluster.
//   resident   many tiles, K <= 1024: writing the output (gated: the epilogue's SiLU). Pairs of SMs, the weight's rows stay on chip.
//   pair       many tiles, longer K: the MMAs, under the power limit. Pairs of SMs, both operands stream.
// In each warp 0 loads (one thread), warp 1 owns tensor memory and issues scale copies and MMAs, warps 2-3 are idle and the others are the
// epilogue. An MMA of 128 (pair: 256) x 256 x 64 takes 128 cycles, one of half the columns 64, with or without the scale copies
// between them; the first result comes some 450 cycles after the first instruction.
//
// The scale tiles of a stage have tensor-memory columns of their own: they are overwritten when the stage is filled
// again, which the MMAs that read them have announced (resident: see its layout).

#include "kept.h"

namespace fluke_sm100 {
namespace {

constexpr int kFp4Threads = 384;
constexpr int kFp4StageK = 256;       // values of K per stage: 128 bytes per row

// The issuing warps run their loops as a whole, with one elected lane at the instructions themselves: like this descriptors, stages and
// addresses are uniform values, and an MMA costs some 30 cycles to issue. Inside an elected branch each operand was
// moved over on its own.
//
// Of a descriptor only the low word changes (the address, 14 bits of 16-byte units). Scale tiles: 32 rows of 16 bytes without
// swizzle, 8 rows 128 bytes apart.
constexpr uint32_t kDescHiSw128 = (1024u >> 4) | (1u << 14) | (2u << 29), kDescHiScales = (128u >> 4) | (1u << 14);
__device__ __forceinline__ uint32_t desc_lo(uint32_t byte_addr) { return ((byte_addr & 0x3FFFFu) >> 4) | (1u << 16); }

// D (+)= A B^T over 64 values of K: GROUP 1, or 2 for a pair of CTAs.
template <int FMT, int GROUP>
__device__ __forceinline__ void tc_mma_fp4(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
#define FLUKE_FP4_MMA(GROUP_, KIND_)                                                                                        \
    asm volatile(                                                                                                           \
        "{\n.reg .pred P;\n.reg .b64 A, B;\nsetp.ne.b32 P, %6, 0;\nmov.b64 A, {%1, %7};\nmov.b64 B, {%2, %7};\n"             \
        "tcgen05.mma.cta_group::" GROUP_ "." KIND_ " [%0], A, B, %3, [%4], [%5], P;\n}\n"                                   \
        ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(kDescHiSw128)                  \
        : "memory")
    if constexpr (FMT == FLUKE_SM100_FP4_MX && GROUP == 1) FLUKE_FP4_MMA("1", "kind::mxf4.block_scale.scale_vec::2X");
    else if constexpr (FMT == FLUKE_SM100_FP4_MX) FLUKE_FP4_MMA("2", "kind::mxf4.block_scale.scale_vec::2X");
    else if constexpr (GROUP == 1) FLUKE_FP4_MMA("1", "kind::mxf4nvf4.block_scale.scale_vec::4X");
    else FLUKE_FP4_MMA("2", "kind::mxf4nvf4.block_scale.scale_vec::4X");
#undef FLUKE_FP4_MMA
}
// A scale tile from shared memory to four tensor-memory columns, the same in all four lane quadrants. GROUP 2: in both CTAs, each
// from its own shared memory to its own tensor memory.
template <int GROUP>
__device__ __forceinline__ void tc_copy_scales(uint32_t taddr, uint32_t lo) {
    if constexpr (GROUP == 1)
        asm volatile("{\n.reg .b64 D;\nmov.b64 D, {%1, %2};\ntcgen05.cp.cta_group::1.32x128b.warpx4 [%0], D;\n}\n"
                     ::"r"(taddr), "r"(lo), "r"(kDescHiScales) : "memory");
    else
        asm volatile("{\n.reg .b64 D;\nmov.b64 D, {%1, %2};\ntcgen05.cp.cta_group::2.32x128b.warpx4 [%0], D;\n}\n"
                     ::"r"(taddr), "r"(lo), "r"(kDescHiScales) : "memory");
}
// Whether the phase has completed, without waiting.
__device__ __forceinline__ bool mbar_test(uint64_t *bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n.reg .pred P;\nmbarrier.test_wait.parity.shared::cta.b64 P, [%1], %2;\nselp.u32 %0, 1, 0, P;\n}\n"
        : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return done != 0;
}
// mbar_wait() of a whole warp, with the same answer for every lane: where one lane gives up, no other goes on to an instruction that takes the warp.
__device__ __forceinline__ bool mbar_wait_warp(uint64_t *bar, uint32_t parity, volatile int *abort_flag, unsigned int site) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, site));
}
// Untiled copy; both addresses and the size are multiples of 16 bytes.
__device__ __forceinline__ void bulk_load(void *smem_dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(smem_dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

// Block-scaled MMA, E2M1 x E2M1, both K-major: bits [4,6) / [29,31) which part of a 32-bit scale cell is B's / A's, [7,10) and
// [10,13) the formats, [17,23) N/8, 23 the scale's type (1 e8m0), [24,29) M/16.
template <int FMT>
__host__ __device__ constexpr uint32_t make_idesc_fp4(int M, int N, int part) {
    return (uint32_t(part) << 4) | (1u << 7) | (1u << 10) | (uint32_t(N >> 3) << 17) | (FMT == FLUKE_SM100_FP4_MX ? 1u << 23 : 0u) |
           (uint32_t(M >> 4) << 24) | (uint32_t(part) << 29);
}


// The address, in the cluster's shared window, of this CTA's shared address `local` in CTA `rank`.
__device__ __forceinline__ uint32_t cluster_address(uint32_t local, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
    return r;
}
// Every thread of the cluster has come here.
__device__ __forceinline__ void cluster_sync_threads() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The two halves of it; without ordering memory.
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
// acc * ga * gb for two columns of a row (NV), in an order that leaves f32 only where the result does: ga is given as low * high, min(ga, 1) and max(ga, 1).
// A sum that is not zero is a multiple of 2^-20 and the quantiser's scales are at least 2^-100, so acc * low is exact; and where high is above one (low is one),
// a product with gb that overflows does so for good. With ga as one factor a row of 1e36 times weights of 0.01 overflowed at acc * ga. The resident form, bound
// by its epilogue, leaves the third product out where no row of a warp has a scale above one (amax above 2688): always : where needed [32000, 512] x [1536, 512] 31.1 : 28.3 us,
// gated with 2 [2048, 512] 70 : 60.
struct RowScale {
    float2 low, high;
    __device__ __forceinline__ explicit RowScale(float ga) {
        const bool small = ga < 1.f;   // a NaN is high
        low = small ? make_float2(ga, ga) : make_float2(1.f, 1.f);
        high = small ? make_float2(1.f, 1.f) : make_float2(ga, ga);
    }
};
template <bool HIGH = true>   // false: high is one
__device__ __forceinline__ float2 scale_rows(float2 acc, const RowScale &ga, float2 gb) {
    const float2 v = mul2(mul2(acc, ga.low), gb);
    return HIGH ? mul2(v, ga.high) : v;
}

__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// silu(g) * u = g / (1 + exp(-g)) * u, which cancels for no gate (h + h tanh(h), h = g / 2, does for a negative one, and the hardware's tanh has 11 bits: at a
// gate of -8 it was off by up to 70 %). Relative error below (|g| + 5) 2^-23: ex2.approx 2^-22, its argument 2^-23 of itself, rcp.approx 2^-23, the other
// operations 2^-24 each. Below a gate of -87 silu, less than 2^-119 there, is zero. Two operations of the special-function unit per value instead of one: gated
// [32000, 512] x 2 [2048, 512] mx 34.9 -> 43.8 us, nv 50.5 -> 55.6, [1803, 2048] x 2 [4096, 2048] nv 17.3 -> 17.6, mx [300, 512] 5.8 -> 6.0, few rows as before.
// Where this form took 48.0 (mx) and 61.9 (nv), before the epilogue's waits were made uniform: a reciprocal for two values, where no gate of a lane's 32 is
// below -43 (a product of two of 1 + exp(-g) overflows otherwise), 44.7 and 65.8, whose registers do not hold the test; for four values 45.9 and 68.9; every
// second exp(-g) as a polynomial 49.3 and 76.8.
__device__ __forceinline__ float2 silu_times(float2 g, float2 u) {
    const float2 t = mul2(g, make_float2(-1.44269504f, -1.44269504f));
    const float2 d = add2(make_float2(ex2_approx(t.x), ex2_approx(t.y)), make_float2(1.f, 1.f));
    return mul2(mul2(g, make_float2(rcp_approx(d.x), rcp_approx(d.y))), u);
}

// ---- few tiles: weights as the first operand, K split over a cluster --------------------------------
// A tile is 128 rows of the weight x up to 128 rows of a (gated: 128 rows of gate and 128 of up x up to 64), with the weight as the MMA's first
// operand: the accumulators are [weight row, row of a], so a few rows of a cost a few columns (N = 16) and the weight's rows fill the
// lanes. With few tiles a tile is given to a cluster of up to 8 CTAs, each of which takes a run of K; they leave their f32 sums in
// their own shared memory, and every CTA then adds up a share of the tile from all of them, in the order of the ranks. What bounds it
// is latency (launch, loads, hand-over) and, for one or a few rows, reading the weights: all of a CTA's loads are in flight at once
// where the ring holds them.
//
// A CTA takes less than half of an SM's shared memory and half of its tensor memory, so that the next kernel's CTAs are set
// up beside it; and more than a third of the shared memory, so that no more than two CTAs of a cluster, which wait for each other,
// share an SM's tensor memory.
constexpr int kFp4SplitSmem = 104 * 1024, kFp4SplitMinSmem = 78 * 1024, kFp4SplitDeep = 152 * 1024, kFp4SplitMaxSmem = 160 * 1024;
constexpr int kFp4SplitStages = 8, kFp4SplitCols = 256;
constexpr int kFp4SumPitch = 132;              // floats between rows of the sums

struct Fp4SplitDev {
    int M, N, K;
    int n_tiles, stages_k, split;     // tiles along N; ring stages of all of K; CTAs per tile
    int sf_tiles, last_steps;         // 512-byte scale tiles per 128 rows; MMAs of the last stage
    int a_rows, stages;               // rows of a per tile (a multiple of 16), ring stages
    int sums_at;                      // byte offset of the sums in shared memory
    int acc_cols;                     // tensor-memory columns per weight
    const uint8_t *sfa, *sfb, *sfb2;
    const float *ga, *gb, *gb2;
    void *out;
};

// Copies `bytes` (a multiple of 16) from this CTA's shared memory to a CTA of the cluster and counts them on its barrier.
__device__ __forceinline__ void bulk_send(uint32_t dst_cluster, const void *src, uint32_t bytes, uint32_t bar_cluster) {
    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst_cluster), "r"(smem_u32(src)), "r"(bytes), "r"(bar_cluster) : "memory");
}

template <int FMT, bool GATED, typename T>
__global__ void __launch_bounds__(kFp4Threads, 2)
gemm_fp4_split_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_b2,
                      const Fp4SplitDev p) {
    constexpr int kAtoms = kFp4StageK / (4 * (FMT == FLUKE_SM100_FP4_MX ? 32 : 16)), kSf = kAtoms * 512;
    constexpr int kWeights = GATED ? 2 : 1, kBBytes = 128 * 128, kSfBytes = kSf * (kWeights + 1), kSfCols = kAtoms * 4 * (kWeights + 1);
    extern __shared__ uint8_t smem_raw[];
    // every CTA of the cluster computes the same offset
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t full_bar[kFp4SplitStages], empty_bar[kFp4SplitStages], done_bar, sums_bar;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    volatile int *abort_flag = &abort_word;
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
    const int rank = int(blockIdx.x) % p.split, tile = int(blockIdx.x) / p.split;
    const int m_tile = tile / p.n_tiles, m0 = m_tile * p.a_rows, n_tile = tile - m_tile * p.n_tiles, n0 = n_tile * 128;
    const int ks0 = p.stages_k * rank / p.split, ks1 = p.stages_k * (rank + 1) / p.split;
    // per stage the weight's rows, then a's; the scales of all stages behind
    const int slot = kWeights * kBBytes + p.a_rows * 128;
    uint8_t *sf = smem + p.stages * slot;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        mbar_init(&done_bar, 1);
        mbar_init(&sums_bar, 1);
        abort_word = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tm_a);
        tma_prefetch_desc(&tm_b);
        if (GATED) tma_prefetch_desc(&tm_b2);
    }
    if (warp == 1) {
        tmem_alloc(&tmem_slot, kFp4SplitCols);
        dependency_trigger();
    }
    tc_fence_before_sync();
    __syncthreads();
    if (p.split > 1) cluster_arrive_relaxed();  // (1) this CTA's barriers are set up; awaited before sums are sent
    tc_fence_after_sync();
    const uint32_t tmem = tmem_slot;
    dependency_wait();

    if (warp == 0) {
        if (elect_one()) {
            const uint8_t *sfa = p.sfa + int64_t(m0 >> 7) * p.sf_tiles * 512;
            const uint8_t *sfb = p.sfb + int64_t(n_tile) * p.sf_tiles * 512;
            const uint8_t *sfb2 = GATED ? p.sfb2 + int64_t(n_tile) * p.sf_tiles * 512 : nullptr;
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int ks = ks0; ks < ks1; ++ks) {
                ok = mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, 120);
                if (!ok) break;
                const uint32_t sf_bytes = min(kAtoms, p.sf_tiles - ks * kAtoms) * 512;
                uint8_t *sb = smem + stage * slot, *ss = sf + stage * kSfBytes;
                mbar_arrive_expect_tx(&full_bar[stage], slot + sf_bytes * (kWeights + 1));
                tma_load_2d(sb, &tm_b, &full_bar[stage], ks * 128, n0);
                if constexpr (GATED) tma_load_2d(sb + kBBytes, &tm_b2, &full_bar[stage], ks * 128, n0);
                bulk_load(ss, sfb + int64_t(ks) * kSf, sf_bytes, &full_bar[stage]);
                if constexpr (GATED) bulk_load(ss + kSf, sfb2 + int64_t(ks) * kSf, sf_bytes, &full_bar[stage]);
                tma_load_2d(sb + kWeights * kBBytes, &tm_a, &full_bar[stage], ks * 128, m0);
                bulk_load(ss + kWeights * kSf, sfa + int64_t(ks) * kSf, sf_bytes, &full_bar[stage]);
                if (++stage == p.stages) { stage = 0; phase ^= 1u; }
            }
            if (!ok) {
                // loads in flight get a bounded chance to land before the shared memory is released
                const long long t0 = clock64();
                while (clock64() - t0 < (1ll << 22)) { }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        const bool leader = elect_one();
        const uint32_t b_lo0 = desc_lo(smem_u32(smem)), s_lo0 = desc_lo(smem_u32(sf));
        const uint32_t shape = uint32_t(p.a_rows >> 3) << 17, first = uint32_t(m0 & 64) >> 5;  // where a tile of 64 begins in a scale tile (32 rows per column; odd columns cannot be addressed)
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int ks = ks0; ks < ks1; ++ks) {
            ok = mbar_wait_warp(&full_bar[stage], phase, abort_flag, 122);
            if (!ok) break;
            tc_fence_after_sync();
            const uint32_t b_lo = b_lo0 + stage * (slot >> 4), a_lo = b_lo + (kWeights * kBBytes >> 4), s_lo = s_lo0 + stage * (kSfBytes >> 4);
            const uint32_t ts = tmem + kWeights * p.acc_cols + stage * kSfCols, tsa = ts + kWeights * kAtoms * 4 + first;
            const int steps = ks == p.stages_k - 1 ? p.last_steps : 4;
            if (leader) {
#pragma unroll
                for (int i = 0; i < kAtoms * (kWeights + 1); ++i) tc_copy_scales<1>(ts + i * 4, s_lo + i * 32);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    constexpr bool mx = FMT == FLUKE_SM100_FP4_MX;
                    const int atom = mx ? k / 2 : k, part = mx ? (k & 1) * 2 : 0;
                    if (k >= steps) break;
#pragma unroll
                    for (int w = 0; w < kWeights; ++w)
                        tc_mma_fp4<FMT, 1>(tmem + w * p.acc_cols, b_lo + w * (kBBytes >> 4) + 2 * k, a_lo + 2 * k, make_idesc_fp4<FMT>(128, 0, part) | shape,
                                           ts + (w * kAtoms + atom) * 4, tsa + atom * 4, ks > ks0 || k > 0);
                }
                tc_commit(&empty_bar[stage]);
                if (ks == ks1 - 1) tc_commit(&done_bar);
            }
            if (++stage == p.stages) { stage = 0; phase ^= 1u; }
        }
        __syncwarp();
    }

    // The sums as [weight, row of a, weight row], gate before up, behind the ring; and in front of it, where the first loads went (all of them have
    // been used by then everywhere: (2)), what the ranks send of this CTA's share of the rows, [rank, weight, row, weight row].
    const int rows = min(p.a_rows, p.M - m0);
    const int share = (rows + p.split - 1) / p.split, row0 = min(rank * share, rows), mine = min(share, rows - row0);
    float *sums = reinterpret_cast<float *>(smem + p.sums_at);
    bool ok = true;
    if (warp >= 4) {
        const int q = warp & 3, half = (warp - 4) >> 2;
        ok = mbar_wait_warp(&done_bar, 0, abort_flag, 123);
        if (ok) {
            tc_fence_after_sync();
            // eight columns per turn: this code runs once, and more of it would cost more to fetch than to execute
            for (int c0 = half * 8; c0 < rows; c0 += 16) {
#pragma unroll
                for (int w = 0; w < kWeights; ++w) {
                    uint32_t a[8];
                    tmem_ld_32x8(tmem + (uint32_t(q * 32) << 16) + w * p.acc_cols + c0, a);
                    tmem_ld_wait();
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        if (c0 + c < rows) sums[(w * p.a_rows + c0 + c) * kFp4SumPitch + q * 32 + lane] = __uint_as_float(a[c]);
                }
            }
        }
        fence_proxy_async_smem();
        __syncwarp();
    }
    if (p.split > 1) {
        cluster_wait();                 // (1)
        cluster_arrive_relaxed();       // (2) this CTA's loads and MMAs have finished
        cluster_wait();
    }
    __syncthreads();
    const float *parts = sums + row0 * kFp4SumPitch;
    int part_pitch = p.a_rows * kFp4SumPitch, rank_pitch = 0;   // floats between the weights and between the ranks
    if (p.split > 1) {
        parts = reinterpret_cast<const float *>(smem);
        part_pitch = share * kFp4SumPitch;
        rank_pitch = kWeights * part_pitch;
        if (warp == 0 && ok) {
            if (lane == 0 && mine > 0) mbar_arrive_expect_tx(&sums_bar, p.split * kWeights * mine * kFp4SumPitch * 4);
            // lane = rank that a share goes to
            const int theirs = min(share, rows - min(lane * share, rows));
            if (lane < p.split && theirs > 0)
#pragma unroll
                for (int w = 0; w < kWeights; ++w)
                    bulk_send(cluster_address(smem_u32(smem) + (rank * rank_pitch + w * part_pitch) * 4, lane),
                              sums + (w * p.a_rows + lane * share) * kFp4SumPitch, theirs * kFp4SumPitch * 4,
                              cluster_address(smem_u32(&sums_bar), lane));
        }
        if (warp >= 4 && ok && mine > 0) ok = mbar_wait_warp(&sums_bar, 0, abort_flag, 124);
    }
    if (warp >= 4 && ok) {
        // eight output columns of a row per turn
        for (int g = int(threadIdx.x) - 128; g < mine * 16; g += 256) {
            const int row = g >> 4, c = (g & 15) * 8, col = n0 + c;
            if (col >= p.N) continue;
            float v[kWeights][8] = {};
#pragma unroll 2
            for (int r = 0; r < p.split; ++r)
#pragma unroll
                for (int i = 0; i < 2 * kWeights; ++i) {
                    const float4 x = *reinterpret_cast<const float4 *>(parts + r * rank_pitch + (i >> 1) * part_pitch + row * kFp4SumPitch + c + (i & 1) * 4);
                    v[i >> 1][(i & 1) * 4] += x.x;
                    v[i >> 1][(i & 1) * 4 + 1] += x.y;
                    v[i >> 1][(i & 1) * 4 + 2] += x.z;
                    v[i >> 1][(i & 1) * 4 + 3] += x.w;
                }
            const int out_row = m0 + row0 + row;
            const RowScale ga(FMT == FLUKE_SM100_FP4_NV ? p.ga[out_row] : 1.f);
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float2 y = make_float2(v[0][2 * i], v[0][2 * i + 1]), u = make_float2(v[kWeights - 1][2 * i], v[kWeights - 1][2 * i + 1]);
                if constexpr (FMT == FLUKE_SM100_FP4_NV) {
                    y = scale_rows(y, ga, *reinterpret_cast<const float2 *>(p.gb + col + 2 * i));
                    if constexpr (GATED) u = scale_rows(u, ga, *reinterpret_cast<const float2 *>(p.gb2 + col + 2 * i));
                }
                if constexpr (GATED) y = silu_times(y, u);
                w[i] = pack2(y, T());
            }
            *reinterpret_cast<uint4 *>(static_cast<T *>(p.out) + int64_t(out_row) * p.N + col) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    __syncwarp();
    tc_fence_before_sync();
    if (p.split > 1) {
        // (3) every share has arrived, so nothing is read from this CTA any more. Relaxed: a release would wait for the output.
        cluster_arrive_relaxed();
        cluster_wait();
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, kFp4SplitCols);
    }
}

// ---- pairs of SMs -------------------------------------------------------------------------------
// Many tiles: a pair of CTAs (cluster of 2) works on 256 x 256 accumulators (gated: 256 rows x 128 gate and 128 up columns) with
// tcgen05 cta_group::2. Each CTA loads its own 128 rows of A and half of the rows of B, and holds its 128 rows of the
// accumulators; the first CTA issues for both. Per 128 cycles of MMA an SM takes in 8 KB of operands instead of the 12 KB that it
// would need on its own, which is what bounds large products (L2 to SM).
//
// The accumulators take 256 of the 512 tensor-memory columns, the scales most of the others, so there is no second
// buffer: the epilogue warps take all of their part into registers (some 150 cycles; 128 of them, for which the compiler spills 12 at most), hand the columns back
// and do the arithmetic and the stores while the MMAs of the next tile run.
//
// A pair works through a contiguous run of the tiles in n-major order.
template <int FMT>
struct Fp4PairLayout {
    static constexpr int kBlock = FMT == FLUKE_SM100_FP4_MX ? 32 : 16;
    static constexpr int kAtoms = kFp4StageK / (4 * kBlock);   // scale tiles per stage and 128 rows
    static constexpr int kOperand = 128 * 128;                 // 128 rows of a stage
    static constexpr int kSfA = kAtoms * 512, kSfB = 2 * kSfA;
    static constexpr int kStages = 5;
    static constexpr int kSlot = 2 * kOperand, kSfSlot = kSfA + kSfB;
    static constexpr int kOffSf = kStages * kSlot;
    static constexpr int kOffStaging = kOffSf + kStages * kSfSlot;
    static constexpr int kOffBars = kOffStaging + 8 * 32 * 128;
    static constexpr int kBars = 2 * kStages + 2;
    static constexpr int kDynamic = kOffBars + kBars * 8 + 16 + 1024;
    static constexpr int kColsSfB = 256 + kStages * kAtoms * 4;   // tensor memory: accumulators, scales of A, scales of B
    static_assert(kOffStaging % 1024 == 0 && kDynamic <= 232448, "shared memory");
    static_assert(kColsSfB + kStages * kAtoms * 8 <= 512, "tensor memory");
};

struct Fp4PairDev {
    int M, N, K;
    int m_tiles, tiles, stages_k;     // pairs of row tiles, tiles in all, stages per tile
    int last_steps;                   // MMAs of the last stage
    const float *ga, *gb, *gb2;
    int passes_by;                    // the output is larger than what L2 can keep, its lines go first
};

// A load into this CTA's shared memory that completes on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_2d_pair(void *smem_dst, const CUtensorMap *m, uint32_t bar_cluster, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2"
        " [%0], [%1, {%3, %4}], [%2];"
        ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar_cluster), "r"(c0), "r"(c1)
        : "memory");
}
// Arrives on the barrier at this offset in both CTAs when the pair's MMAs so far have finished.
__device__ __forceinline__ void tc_commit_pair(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"(uint16_t(3)) : "memory");
}
// Arrives on a barrier of either CTA. What it announces are reads of tensor memory, which tcgen05.fence orders: no wider scope than
// the default is asked for (with release.cluster the arrival waited for the warp's stores as well, some 1300 cycles per tile).
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar_cluster) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster) : "memory");
}

// Walks the run of tiles of a pair. The position is advanced, not recomputed: a division per tile in the issuing warp costs as much as
// several MMAs.
struct PairRun {
    int left, n, m;   // tiles still to do, this one included; its position
    __device__ __forceinline__ PairRun(const Fp4PairDev &p) {
        const int pairs = int(gridDim.x) >> 1, pair = int(blockIdx.x) >> 1;
        const int first = int(int64_t(p.tiles) * pair / pairs);
        left = int(int64_t(p.tiles) * (pair + 1) / pairs) - first;
        n = first / p.m_tiles;
        m = first - n * p.m_tiles;
    }
    __device__ __forceinline__ bool last_of_n(const Fp4PairDev &p) const { return m + 1 == p.m_tiles; }
    __device__ __forceinline__ void next(const Fp4PairDev &p) {
        --left;
        if (++m == p.m_tiles) {
            m = 0;
            ++n;
        }
    }
};

template <int FMT, bool GATED, typename T>
__global__ void __launch_bounds__(kFp4Threads, 1)
gemm_fp4_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_b2,
                     const __grid_constant__ CUtensorMap tm_sfa, const __grid_constant__ CUtensorMap tm_sfb,
                     const __grid_constant__ CUtensorMap tm_sfb2, const __grid_constant__ CUtensorMap tm_out, const Fp4PairDev p) {
    using L = Fp4PairLayout<FMT>;
    constexpr int STAGES = L::kStages, BN_OUT = GATED ? 128 : 256;
    extern __shared__ uint8_t smem_raw[];
    // both CTAs compute the same offset
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kOffBars);
    uint64_t *full_bar = bars, *empty_bar = bars + STAGES, *tfull_bar = bars + 2 * STAGES, *tempty_bar = tfull_bar + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + L::kBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
    const int rank = int(blockIdx.x & 1);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        mbar_init(tfull_bar, 1);
        mbar_init(tempty_bar, 16);
        *abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tm_a);
        tma_prefetch_desc(&tm_b);
        tma_prefetch_desc(&tm_sfa);
        tma_prefetch_desc(&tm_sfb);
        tma_prefetch_desc(&tm_out);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512, PairTag());
        dependency_trigger();
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_threads();  // the partner's barriers are set up, its tensor memory is there
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    dependency_wait();

    PairRun run(p);
    if (warp < 4) reg_dealloc<kRegsLight>();
    if (warp == 0) {
        if (elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            const CUtensorMap *b = GATED && rank ? &tm_b2 : &tm_b;
            for (; run.left > 0 && ok; run.next(p)) {
                const int n = run.n, m0 = run.m * 256 + rank * 128, n0 = n * BN_OUT;
                const int b_row = GATED ? n0 : n0 + rank * 128;
                for (int ks = 0; ks < p.stages_k; ++ks) {
                    ok = mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, 131);
                    if (!ok) break;
                    uint8_t *sa = smem + stage * L::kSlot, *sb = sa + L::kOperand;
                    uint8_t *ssa = smem + L::kOffSf + stage * L::kSfSlot, *ssb = ssa + L::kSfA;
                    const uint32_t bar = cluster_address(smem_u32(&full_bar[stage]), 0);
                    if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * (L::kSlot + L::kSfSlot));
                    tma_load_2d_pair(sa, &tm_a, bar, ks * 128, m0);
                    tma_load_2d_pair(ssa, &tm_sfa, bar, ks * L::kSfA / 8, m0 >> 7);
                    tma_load_2d_pair(sb, b, bar, ks * 128, b_row);
                    tma_load_2d_pair(ssb, &tm_sfb, bar, ks * L::kSfA / 8, n0 >> 7);
                    if constexpr (GATED) tma_load_2d_pair(ssb + L::kSfA, &tm_sfb2, bar, ks * L::kSfA / 8, n0 >> 7);
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                }
            }
            if (!ok) {
                // loads in flight get a bounded chance to land before the shared memory is released
                const long long t0 = clock64();
                while (clock64() - t0 < (1ll << 22)) { }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            const bool leader = elect_one();
            int stage = 0;
            uint32_t phase = 0, t_phase = 0;
            bool ok = true, ready = false;
            const uint32_t base_lo = desc_lo(smem_u32(smem)), sf_lo = desc_lo(smem_u32(smem) + L::kOffSf);
            for (; run.left > 0 && ok; run.next(p), t_phase ^= 1u) {
                ok = mbar_wait_warp(tempty_bar, t_phase ^ 1u, abort_flag, 132);
                if (!ok) break;
                tc_fence_after_sync();
                for (int ks = 0; ks < p.stages_k; ++ks) {
                    if (!ready) ok = mbar_wait_warp(&full_bar[stage], phase, abort_flag, 134);
                    if (!ok) break;
                    tc_fence_after_sync();
                    // The next stage is asked about here and the answer is looked at behind this stage's MMAs.
                    const bool wraps = stage + 1 == STAGES;
                    const bool next = mbar_test(&full_bar[wraps ? 0 : stage + 1], wraps ? phase ^ 1u : phase);
                    const uint32_t a_lo = base_lo + stage * (L::kSlot >> 4), s_lo = sf_lo + stage * (L::kSfSlot >> 4);
                    const uint32_t tsa = tmem + 256 + stage * L::kAtoms * 4, tsb = tmem + L::kColsSfB + stage * L::kAtoms * 8;
                    const int steps = ks == p.stages_k - 1 ? p.last_steps : 4;
                    if (leader) {
#pragma unroll
                        for (int i = 0; i < L::kAtoms; ++i) {
                            tc_copy_scales<2>(tsa + i * 4, s_lo + i * 32);
#pragma unroll
                            for (int t = 0; t < 2; ++t) tc_copy_scales<2>(tsb + (2 * i + t) * 4, s_lo + (L::kSfA >> 4) + (t * L::kAtoms + i) * 32);
                        }
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            constexpr bool mx = FMT == FLUKE_SM100_FP4_MX;
                            const int atom = mx ? k / 2 : k, part = mx ? (k & 1) * 2 : 0;
                            if (k < steps)
                                tc_mma_fp4<FMT, 2>(tmem, a_lo + 2 * k, a_lo + (L::kOperand >> 4) + 2 * k, make_idesc_fp4<FMT>(256, 256, part),
                                                     tsa + atom * 4, tsb + atom * 8, (ks | k) != 0);
                        }
                        tc_commit_pair(&empty_bar[stage]);
                        if (ks == p.stages_k - 1) tc_commit_pair(tfull_bar);
                    }
                    ready = __all_sync(0xffffffffu, next);
                    stage = wraps ? 0 : stage + 1;
                    phase ^= wraps;
                }
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        reg_alloc<kRegsEpilogue>();
        const int q = warp & 3, half = (warp - 4) >> 2;
        uint8_t *staging = smem + L::kOffStaging + (warp - 4) * (32 * 128);
        const uint32_t tempty = cluster_address(smem_u32(tempty_bar), 0);
        uint32_t t_phase = 0;
        bool ok = true;
        for (; run.left > 0 && ok; run.next(p), t_phase ^= 1u) {
            const int n = run.n, m0 = run.m * 256 + rank * 128 + q * 32, n0 = n * BN_OUT;
            float ga = 1.f;
            if (FMT == FLUKE_SM100_FP4_NV && m0 + lane < p.M) ga = p.ga[m0 + lane];
            ok = mbar_wait_warp(tfull_bar, t_phase, abort_flag, 135);
            if (!ok) break;
            tc_fence_after_sync();
            const uint32_t t_row = tmem + (uint32_t(q * 32) << 16);
            // plain: columns 128 half .. + 127; gated: gate columns 64 half .. + 63 and the up columns 128 further
            uint32_t a[4][32];
#pragma unroll
            for (int j = 0; j < 4; ++j) tmem_ld_32x32(t_row + (GATED ? half * 64 + (j >> 1) * 128 + (j & 1) * 32 : half * 128 + j * 32), a[j]);
            tmem_ld_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(tempty);
            if (m0 >= p.M) continue;
            const RowScale ga2(ga);
#pragma unroll
            for (int g = 0; g < (GATED ? 1 : 2); ++g) {
                const int c0 = n0 + (GATED ? half * 64 : half * 128 + g * 64);
                if (c0 >= p.N) break;
                if (lane == 0) tma_store_wait_read<0>();
                __syncwarp();
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t w[16];
#pragma unroll
                    for (int c = 0; c < 32; c += 4) {
                        const int j = 2 * g + h;
                        float2 v[2] = {make_float2(__uint_as_float(a[j][c]), __uint_as_float(a[j][c + 1])),
                                       make_float2(__uint_as_float(a[j][c + 2]), __uint_as_float(a[j][c + 3]))};
                        float2 u[2];
                        if constexpr (GATED) {
                            u[0] = make_float2(__uint_as_float(a[2 + h][c]), __uint_as_float(a[2 + h][c + 1]));
                            u[1] = make_float2(__uint_as_float(a[2 + h][c + 2]), __uint_as_float(a[2 + h][c + 3]));
                        }
                        if constexpr (FMT == FLUKE_SM100_FP4_NV) {
                            const int col = c0 + 32 * h + c;
                            float4 gb = make_float4(0.f, 0.f, 0.f, 0.f), gu = gb;
                            if (col < p.N) {
                                gb = *reinterpret_cast<const float4 *>(p.gb + col);
                                if (GATED) gu = *reinterpret_cast<const float4 *>(p.gb2 + col);
                            }
                            v[0] = scale_rows(v[0], ga2, make_float2(gb.x, gb.y));
                            v[1] = scale_rows(v[1], ga2, make_float2(gb.z, gb.w));
                            if constexpr (GATED) {
                                u[0] = scale_rows(u[0], ga2, make_float2(gu.x, gu.y));
                                u[1] = scale_rows(u[1], ga2, make_float2(gu.z, gu.w));
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            if constexpr (GATED) v[i] = silu_times(v[i], u[i]);
                            w[c / 2 + i] = pack2(v[i], T());
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        *reinterpret_cast<uint4 *>(staging + sw128_offset(lane, 4 * h + j)) =
                            make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    if (p.passes_by) tma_store_2d(&tm_out, staging, c0, m0, l2_evict_first());
                    else tma_store_2d(&tm_out, staging, c0, m0);
                    tma_store_commit();
                }
            }
        }
        if (lane == 0) tma_store_wait_all<0>();
        __syncwarp();
    }

    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_threads();  // nothing of the partner still arrives here or reads this CTA's operands
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512, PairTag());
    }
}

// ---- pairs of SMs, resident rows of B -------------------------------------------------------------
// K <= 1024: the pair's rows of B stay in shared memory and their scales in tensor memory for as long as the pair works on the same
// columns; only A streams. With so few instructions per tile (8 of 128 cycles at K = 512) what lies between two tiles counts: an
// MMA chain takes some 450 cycles from its first instruction to its first result, and the hand-over of a buffer as long again. So a
// tile is two halves of 128 columns (gated: gate and up) with a buffer each out of a ring of three (two where the scales need
// the room), and the chain does not stop. The issuing warp has some 1000 cycles for a tile: its loops are unrolled, and A comes in
// slots of 512 values of K with one barrier each. 16 epilogue warps, each 32 rows x 32 columns of a buffer.
template <int FMT, int KMAX>   // KMAX: stages of K that B may have (2 or 4)
struct Fp4ResidentLayout {
    static constexpr int kBlock = FMT == FLUKE_SM100_FP4_MX ? 32 : 16;
    static constexpr int kAtoms = kFp4StageK / (4 * kBlock);
    static constexpr int kOperand = 128 * 128;
    static constexpr int kSf = kAtoms * 512;                   // scales of 128 rows of a stage
    static constexpr bool kRoom = FMT == FLUKE_SM100_FP4_MX || KMAX == 2;
    static constexpr int kAccs = kRoom ? 3 : 2;
    static constexpr int kSlots = KMAX == 2 ? 4 : 3;           // of two stages of A
    static constexpr int kOffB = kSlots * 2 * kOperand;
    static constexpr int kOffSf = kOffB + KMAX * kOperand;
    static constexpr int kOffSfB = kOffSf + kSlots * 2 * kSf;
    static constexpr int kOffStaging = kOffSfB + KMAX * 2 * kSf;
    static constexpr int kOffBars = kOffStaging + 16 * 32 * 64;
    static constexpr int kBars = 2 * kSlots + KMAX + 1 + 2 * kAccs;
    static constexpr int kDynamic = kOffBars + kBars * 8 + 16 + 1024;
    // Tensor memory: accumulators; the scales of A, of two tiles in turns (a tile begins when the buffer that the half three, or two, before its
    // first one filled has been read, so the MMAs of the tile before the last have finished); the scales of B.
    static constexpr int kColsSfA = kAccs * 128, kSetCols = KMAX * kAtoms * 4, kColsSfB = kColsSfA + 2 * kSetCols;
    static_assert(kOffStaging % 1024 == 0 && kDynamic <= 232448, "shared memory");
    static_assert(kColsSfB + KMAX * kAtoms * 8 <= 512, "tensor memory");
};

constexpr int kFp4ResidentThreads = 640;

template <int FMT, bool GATED, int KMAX, typename T>
__global__ void __launch_bounds__(kFp4ResidentThreads, 1)
gemm_fp4_resident_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                         const __grid_constant__ CUtensorMap tm_b2, const __grid_constant__ CUtensorMap tm_sfa,
                         const __grid_constant__ CUtensorMap tm_sfb, const __grid_constant__ CUtensorMap tm_sfb2,
                         const __grid_constant__ CUtensorMap tm_out, const Fp4PairDev p) {
    using L = Fp4ResidentLayout<FMT, KMAX>;
    constexpr int SLOTS = L::kSlots, ACCS = L::kAccs, BN_OUT = GATED ? 128 : 256;
    extern __shared__ uint8_t smem_raw[];
    // both CTAs compute the same offset
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kOffBars);
    uint64_t *full_bar = bars, *empty_bar = bars + SLOTS, *bfull_bar = bars + 2 * SLOTS, *bempty_bar = bfull_bar + KMAX;
    uint64_t *tfull_bar = bempty_bar + 1, *tempty_bar = tfull_bar + ACCS;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + L::kBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
    const int rank = int(blockIdx.x & 1);

    if (threadIdx.x == 0) {
        for (int s = 0; s < SLOTS; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int s = 0; s < KMAX; ++s) mbar_init(&bfull_bar[s], 1);
        mbar_init(bempty_bar, 1);
        for (int s = 0; s < ACCS; ++s) {
            mbar_init(&tfull_bar[s], 1);
            mbar_init(&tempty_bar[s], 32);
        }
        *abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tm_a);
        tma_prefetch_desc(&tm_b);
        tma_prefetch_desc(&tm_sfa);
        tma_prefetch_desc(&tm_sfb);
        tma_prefetch_desc(&tm_out);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512, PairTag());
        dependency_trigger();
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_threads();  // the partner's barriers are set up, its tensor memory is there
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    dependency_wait();

    PairRun run(p);
    if (warp == 0) {
        if (elect_one()) {
            int slot = 0, cur_n = -1, loads_b = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (; run.left > 0 && ok; run.next(p)) {
                const int n = run.n, m0 = run.m * 256 + rank * 128, n0 = n * BN_OUT;
                const bool load_b = n != cur_n;
                if (load_b) {
                    // the MMAs that read the rows of B before these
                    if (loads_b > 0) ok = mbar_wait(bempty_bar, (loads_b - 1) & 1, abort_flag, 140);
                    if (!ok) break;
                    cur_n = n;
                    ++loads_b;
                }
                for (int ks = 0; ks < p.stages_k; ++ks) {
                    if (load_b) {
                        // this CTA's 64 rows of either half
                        const uint32_t bar = cluster_address(smem_u32(&bfull_bar[ks]), 0);
                        uint8_t *sb = smem + L::kOffB + ks * L::kOperand, *ssb = smem + L::kOffSfB + ks * 2 * L::kSf;
                        if (rank == 0) mbar_arrive_expect_tx(&bfull_bar[ks], 2 * (L::kOperand + 2 * L::kSf));
                        tma_load_2d_pair(sb, &tm_b, bar, ks * 128, n0 + 64 * rank);
                        tma_load_2d_pair(sb + L::kOperand / 2, GATED ? &tm_b2 : &tm_b, bar, ks * 128, (GATED ? n0 : n0 + 128) + 64 * rank);
                        tma_load_2d_pair(ssb, &tm_sfb, bar, ks * L::kSf / 8, n0 >> 7);
                        if constexpr (GATED) tma_load_2d_pair(ssb + L::kSf, &tm_sfb2, bar, ks * L::kSf / 8, n0 >> 7);
                    }
                    const int part = ks & 1;
                    if (part == 0) {
                        ok = mbar_wait(&empty_bar[slot], phase ^ 1u, abort_flag, 141);
                        if (!ok) break;
                        if (rank == 0) mbar_arrive_expect_tx(&full_bar[slot], (ks + 1 < p.stages_k ? 4 : 2) * (L::kOperand + L::kSf));
                    }
                    const uint32_t bar = cluster_address(smem_u32(&full_bar[slot]), 0);
                    tma_load_2d_pair(smem + (2 * slot + part) * L::kOperand, &tm_a, bar, ks * 128, m0);
                    tma_load_2d_pair(smem + L::kOffSf + (2 * slot + part) * L::kSf, &tm_sfa, bar, ks * L::kSf / 8, m0 >> 7);
                    if (part == 1 || ks + 1 == p.stages_k)
                        if (++slot == SLOTS) { slot = 0; phase ^= 1u; }
                }
            }
            if (!ok) {
                // loads in flight get a bounded chance to land before the shared memory is released
                const long long t0 = clock64();
                while (clock64() - t0 < (1ll << 22)) { }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            const bool leader = elect_one();
            int slot = 0, cur_n = -1, acc = 0;
            uint32_t phase = 0, t_phase = 0, b_phase = 1, set = 0;   // of the slots, the buffers, the rows of B; scales of A
            bool ok = true;
            const uint32_t a_lo0 = desc_lo(smem_u32(smem)), b_lo0 = desc_lo(smem_u32(smem) + L::kOffB);
            const uint32_t sa_lo0 = desc_lo(smem_u32(smem) + L::kOffSf), sb_lo0 = desc_lo(smem_u32(smem) + L::kOffSfB);
            const int mmas = (p.stages_k - 1) * 4 + p.last_steps, stages_k = p.stages_k;
            for (; run.left > 0 && ok; run.next(p)) {
                const bool first_of_n = run.n != cur_n;
                if (first_of_n) {
                    cur_n = run.n;
                    b_phase ^= 1u;
                }
                const uint32_t tsa = tmem + L::kColsSfA + set;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    ok = ok && mbar_wait_warp(&tempty_bar[acc], t_phase ^ 1u, abort_flag, 142);
                    if (!ok) break;
                    tc_fence_after_sync();
                    const uint32_t d = tmem + acc * 128;
                    int sl = slot;
                    uint32_t sl_phase = phase;
#pragma unroll
                    for (int pair = 0; pair < KMAX / 2; ++pair) {
                        if (2 * pair >= stages_k) break;
                        const uint32_t a_lo = a_lo0 + sl * (2 * L::kOperand >> 4), sa_lo = sa_lo0 + sl * (2 * L::kSf >> 4);
                        if (half == 0) {
                            if (first_of_n) {
                                ok = mbar_wait_warp(&bfull_bar[2 * pair], b_phase, abort_flag, 143);
                                if (2 * pair + 1 < stages_k) ok = ok && mbar_wait_warp(&bfull_bar[2 * pair + 1], b_phase, abort_flag, 143);
                            }
                            ok = ok && mbar_wait_warp(&full_bar[sl], sl_phase, abort_flag, 144);
                            if (!ok) break;
                            tc_fence_after_sync();
                            if (leader) {
#pragma unroll
                                for (int i = 0; i < 2 * L::kAtoms; ++i)
                                    if (2 * pair + i / L::kAtoms < stages_k) tc_copy_scales<2>(tsa + (2 * pair * L::kAtoms + i) * 4, sa_lo + i * 32);
                                if (first_of_n)
#pragma unroll
                                    for (int i = 0; i < 4 * L::kAtoms; ++i)
                                        if (2 * pair + i / (2 * L::kAtoms) < stages_k)
                                            tc_copy_scales<2>(tmem + L::kColsSfB + (4 * pair * L::kAtoms + i) * 4, sb_lo0 + (4 * pair * L::kAtoms + i) * 32);
                            }
                        }
                        if (leader) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                constexpr bool mx = FMT == FLUKE_SM100_FP4_MX;
                                const int ks = 2 * pair + i / 4, k = i % 4, atom = mx ? k / 2 : k, part = mx ? (k & 1) * 2 : 0;
                                if (8 * pair + i < mmas)
                                    tc_mma_fp4<FMT, 2>(d, a_lo + (i / 4) * (L::kOperand >> 4) + 2 * k,
                                                       b_lo0 + ks * (L::kOperand >> 4) + half * (L::kOperand >> 5) + 2 * k,
                                                       make_idesc_fp4<FMT>(256, 128, part), tsa + (ks * L::kAtoms + atom) * 4,
                                                       tmem + L::kColsSfB + (ks * 2 * L::kAtoms + half * L::kAtoms + atom) * 4, (pair | i) != 0);
                            }
                            if (half == 1) tc_commit_pair(&empty_bar[sl]);
                        }
                        if (++sl == SLOTS) { sl = 0; sl_phase ^= 1u; }
                    }
                    if (!ok) break;
                    if (leader) tc_commit_pair(&tfull_bar[acc]);
                    if (++acc == ACCS) { acc = 0; t_phase ^= 1u; }
                    if (half == 1) {
                        slot = sl;
                        phase = sl_phase;
                    }
                }
                set ^= L::kSetCols;
                if (ok && leader && run.left > 1 && run.last_of_n(p)) tc_commit_pair(bempty_bar);
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        const int q = warp & 3, slice = (warp - 4) >> 2;
        uint8_t *staging = smem + L::kOffStaging + (warp - 4) * (32 * 64);
        const uint32_t tempty = cluster_address(smem_u32(tempty_bar), 0);
        const uint32_t t_row = tmem + (uint32_t(q * 32) << 16) + slice * 32;
        int acc = 0;
        uint32_t t_phase = 0;
        bool ok = true;
        const uint64_t evict_first = l2_evict_first();
        // The warp's 32 x 32 cells of the next buffer, which is handed back.
        auto take = [&](uint32_t (&a)[32]) {
            if (!mbar_wait_warp(&tfull_bar[acc], t_phase, abort_flag, 145)) return false;
            tc_fence_after_sync();
            tmem_ld_32x32(t_row + acc * 128, a);
            tmem_ld_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(tempty + acc * 8);
            if (++acc == ACCS) { acc = 0; t_phase ^= 1u; }
            return true;
        };
        for (; run.left > 0 && ok; run.next(p)) {
            const int n = run.n, m0 = run.m * 256 + rank * 128 + q * 32, n0 = n * BN_OUT;
            float ga = 1.f;
            if (FMT == FLUKE_SM100_FP4_NV && m0 + lane < p.M) ga = p.ga[m0 + lane];
#pragma unroll 1
            for (int half = 0; half < (GATED ? 1 : 2) && ok; ++half) {
                uint32_t a[32], u[GATED ? 32 : 1];
                ok = take(a);
                if constexpr (GATED) ok = ok && take(u);
                if (!ok) break;
                const int c0 = n0 + half * 128 + slice * 32;
                if (m0 >= p.M || c0 >= p.N) continue;
                if (lane == 0) tma_store_wait_read<0>();
                __syncwarp();
                const RowScale ga2(ga);
                auto finish = [&](auto high) {   // high: some row of the warp has a scale above one
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float2 v[4];
                        [[maybe_unused]] float2 up[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            v[i] = make_float2(__uint_as_float(a[8 * j + 2 * i]), __uint_as_float(a[8 * j + 2 * i + 1]));
                            if constexpr (GATED) up[i] = make_float2(__uint_as_float(u[8 * j + 2 * i]), __uint_as_float(u[8 * j + 2 * i + 1]));
                        }
                        auto scale = [&](float2 (&x)[4], const float *g) {   // eight columns; N is a multiple of eight
                            float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
                            if (c0 + 8 * j < p.N) {
                                lo = *reinterpret_cast<const float4 *>(g + c0 + 8 * j);
                                hi = *reinterpret_cast<const float4 *>(g + c0 + 8 * j + 4);
                            }
                            x[0] = scale_rows<high>(x[0], ga2, make_float2(lo.x, lo.y));
                            x[1] = scale_rows<high>(x[1], ga2, make_float2(lo.z, lo.w));
                            x[2] = scale_rows<high>(x[2], ga2, make_float2(hi.x, hi.y));
                            x[3] = scale_rows<high>(x[3], ga2, make_float2(hi.z, hi.w));
                        };
                        if constexpr (FMT == FLUKE_SM100_FP4_NV) {
                            scale(v, p.gb);
                            if constexpr (GATED) scale(up, p.gb2);
                        }
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if constexpr (GATED) v[i] = silu_times(v[i], up[i]);
                            w[i] = pack2(v[i], T());
                        }
                        *reinterpret_cast<uint4 *>(staging + tile_offset<32>(lane, j)) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                };
                if (FMT == FLUKE_SM100_FP4_NV && __any_sync(0xffffffffu, !(ga <= 1.f))) finish(std::true_type());
                else finish(std::false_type());
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    if (p.passes_by) tma_store_2d(&tm_out, staging, c0, m0, evict_first);
                    else tma_store_2d(&tm_out, staging, c0, m0);
                    tma_store_commit();
                }
            }
        }
        if (lane == 0) tma_store_wait_all<0>();
        __syncwarp();
    }

    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_threads();  // nothing of the partner still arrives here or reads this CTA's operands
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512, PairTag());
    }
}

// Launches clusters of `cluster` CTAs that wait for their predecessors themselves.
template <typename... P, typename... A>
int launch_dependent_clusters(void (*kernel)(P...), int cluster, dim3 grid, int block, size_t smem, cudaStream_t stream, A &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    if (e != cudaSuccess) cudaGetLastError();
    return (int)e;
}

// Clusters of `size` CTAs of KERNEL that run at once with `smem` bytes each; 0 where they cannot or the device does not say. A GPC's SMs bound it as
// well as their number: 16 clusters of 8 CTAs, one per SM, ran in two rounds.
template <auto KERNEL>
int cluster_capacity(int size, int threads, int smem) {
    static std::atomic<int> cached[64][9];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) dev = 0;
    return kept(cached[dev][size], [&] {
        int n = 0;
        bool ok = configure_smem<KERNEL>(smem) == 0;
        if (ok) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(size);
            cfg.blockDim = dim3(threads);
            cfg.dynamicSmemBytes = smem;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = size;
            attr[0].val.clusterDim.y = 1;
            attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            ok = cudaOccupancyMaxActiveClusters(&n, reinterpret_cast<const void *>(KERNEL), &cfg) == cudaSuccess;
        }
        cudaGetLastError();
        return ok ? n : 0;
    });
}

// KMAX: 0 streams B, else the resident form with that many stages.
template <int FMT, bool GATED, int KMAX, typename T>
int gemm_fp4_pair_launch(const fluke_sm100_gemm_fp4_t *g, cudaStream_t stream) {
    constexpr int BN_OUT = GATED ? 128 : 256, kThreads = KMAX ? kFp4ResidentThreads : kFp4Threads;
    constexpr int kSmem = KMAX ? Fp4ResidentLayout<FMT, KMAX ? KMAX : 2>::kDynamic : Fp4PairLayout<FMT>::kDynamic;
    constexpr int kSf = Fp4PairLayout<FMT>::kSfA;
    constexpr auto kernel = [] {
        if constexpr (KMAX == 0) return gemm_fp4_pair_kernel<FMT, GATED, T>;
        else return gemm_fp4_resident_kernel<FMT, GATED, KMAX, T>;
    }();
    const int capacity = cluster_capacity<kernel>(2, kThreads, kSmem);
    if (capacity < 1) return (int)cudaErrorNotSupported;
    Fp4PairDev p;
    p.M = g->M; p.N = g->N; p.K = g->K;
    p.m_tiles = (g->M + 255) / 256;
    const int64_t tiles = int64_t(p.m_tiles) * ((g->N + BN_OUT - 1) / BN_OUT);
    if (tiles > INT32_MAX - 1024) return (int)cudaErrorInvalidValue;
    p.tiles = int(tiles);
    p.stages_k = (g->K + kFp4StageK - 1) / kFp4StageK;
    p.last_steps = (g->K - (p.stages_k - 1) * kFp4StageK + 63) / 64;
    p.ga = g->a_row; p.gb = g->b_row; p.gb2 = g->b2_row;
    // such lines drive out what the next kernels read: gated [32000, 512] x 2 [2048, 512] (131 MB) 48.9 : 47.8 us, in a long loop 50.6 : 49.6;
    // streamed [8192, 4096] x [8192, 4096] (134 MB) 106.6 : 106.3
    p.passes_by = int64_t(g->M) * g->N * 2 > int64_t(device_l2_bytes()) / 8 * 7;
    CUtensorMap tm_a, tm_b, tm_b2, tm_sfa, tm_sfb, tm_sfb2, tm_out;
    const uint64_t pitch = uint64_t(g->K) / 2, sf_words = uint64_t(fp4_tiles(g->K, FMT)) * 64;
    auto operand = [&](CUtensorMap *m, const void *base, int rows, int box_rows) {
        return make_tmap_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, base, rows, pitch, pitch, box_rows, 128, true);
    };
    // scale tiles of 128 rows as a row of 8-byte words
    auto scales = [&](CUtensorMap *m, const void *base, int rows, int box_rows) {
        return make_tmap_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT64, 8, base, (rows + 127) / 128, sf_words, sf_words * 8, box_rows, kSf / 8, false);
    };
    int rc = operand(&tm_a, g->a, g->M, 128);
    if (!rc) rc = operand(&tm_b, g->b, g->N, KMAX ? 64 : 128);
    if (!rc) rc = scales(&tm_sfa, g->a_scale, g->M, 1);
    if (!rc) rc = scales(&tm_sfb, g->b_scale, g->N, GATED ? 1 : 2);
    if (!rc)
        rc = make_tmap_2d_sw(&tm_out, CU_TENSOR_MAP_DATA_TYPE_UINT16, g->out, g->M, g->N, uint64_t(g->N) * 2, 32, KMAX ? 32 : 64,
                             KMAX ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
    tm_b2 = tm_b;
    tm_sfb2 = tm_sfb;
    if (GATED && !rc) rc = operand(&tm_b2, g->b2, g->N, KMAX ? 64 : 128);
    if (GATED && !rc) rc = scales(&tm_sfb2, g->b2_scale, g->N, 1);
    if (rc) return rc;
    const int pairs = p.tiles < capacity ? p.tiles : capacity;
    return launch_dependent_clusters(kernel, 2, pairs * 2, kThreads, kSmem, stream, tm_a, tm_b, tm_b2, tm_sfa, tm_sfb, tm_sfb2, tm_out, p);
}

// Rows of a per tile of the split form: 64 while those tiles are all resident at once, else 128 (plain form; the gated one keeps to
// 64); what there is of them, if less.
template <bool GATED>
int split_rows(const fluke_sm100_gemm_fp4_t *g) {
    if (g->M <= 32) return g->M <= 16 ? 16 : 32;
    return GATED || int64_t((g->M + 63) / 64) * ((g->N + 127) / 128) <= device_sm_count() ? 64 : 128;
}
template <bool GATED>
int64_t split_tiles(const fluke_sm100_gemm_fp4_t *g) {
    const int rows = split_rows<GATED>(g);
    return int64_t((g->M + rows - 1) / rows) * ((g->N + 127) / 128);
}

template <int FMT, bool GATED, typename T>
int gemm_fp4_split_launch(const fluke_sm100_gemm_fp4_t *g, cudaStream_t stream) {
    constexpr int kAtoms = kFp4StageK / (4 * (FMT == FLUKE_SM100_FP4_MX ? 32 : 16)), kSf = kAtoms * 512, kWeights = GATED ? 2 : 1;
    constexpr auto kernel = gemm_fp4_split_kernel<FMT, GATED, T>;
    Fp4SplitDev p;
    p.M = g->M; p.N = g->N; p.K = g->K;
    p.n_tiles = (g->N + 127) / 128;
    p.stages_k = (g->K + kFp4StageK - 1) / kFp4StageK;
    p.last_steps = (g->K - (p.stages_k - 1) * kFp4StageK + 63) / 64;
    p.sf_tiles = fp4_tiles(g->K, FMT);
    p.sfa = static_cast<const uint8_t *>(g->a_scale);
    p.sfb = static_cast<const uint8_t *>(g->b_scale);
    p.sfb2 = static_cast<const uint8_t *>(g->b2_scale);
    p.ga = g->a_row; p.gb = g->b_row; p.gb2 = g->b2_row;
    p.out = g->out;
    const int rows = p.a_rows = split_rows<GATED>(g), sms = device_sm_count();
    const int64_t tiles = split_tiles<GATED>(g);
    if (tiles > (INT32_MAX >> 3) - 1024) return (int)cudaErrorInvalidValue;
    // CTAs per tile, while all of them run at once and each has a stage of K at least: the number with the shortest time by what a stage takes
    // (0.2 us, 0.35 with two weights) and what a hand-over of the tile's rows does (0.6 us, and 18 ns per row and weight). Us per call, 1 : 2 : 4
    // CTAs per tile: [1, 4096] x [4096, 4096] 6.6 : 5.1 : 4.5, [333, 2048] x [2048, 512] (24 tiles of 64 rows) 5.1 : 5.7 : 5.6.
    const int most = g->M < rows ? g->M : rows;
    int each = p.stages_k;
    float best = 0.f;
    for (int c = 1; c <= 8 && c <= p.stages_k && (c == 1 || tiles * c <= sms); ++c) {
        const int n = (p.stages_k + c - 1) / c;
        const float us = n * (GATED ? 0.35f : 0.2f) + (c > 1 ? 0.6f + 0.018f * kWeights * most : 0.f);
        if (c > 1 && (us >= best || tiles > cluster_capacity<kernel>(c, kFp4Threads, kFp4SplitMaxSmem + 1024))) continue;
        best = us;
        each = n;
    }
    const int split = p.split = (p.stages_k + each - 1) / each;
    p.acc_cols = rows < 32 ? 32 : rows;
    const int stage_bytes = p.a_rows * 128 + kWeights * 128 * 128 + kSf * (kWeights + 1);
    // A longer run of K than the ring holds streams through a deeper one, where an SM has no second CTA to run: [5, 4096] gated with
    // [8192, 4096] twice 10.2 us at 104 KB, 8.2 at 150.
    p.stages = (each * stage_bytes > kFp4SplitSmem && tiles * split <= sms ? kFp4SplitDeep : kFp4SplitSmem) / stage_bytes;
    const int scale_stages = (kFp4SplitCols - kWeights * p.acc_cols) / (kAtoms * 4 * (kWeights + 1));   // what tensor memory holds
    if (p.stages > kFp4SplitStages) p.stages = kFp4SplitStages;
    if (p.stages > scale_stages) p.stages = scale_stages;
    if (p.stages > each) p.stages = each;
    // the sums, and with a split what is received (of one share from every rank) in front of them
    const int sums = kWeights * rows * kFp4SumPitch * 4;
    p.sums_at = split > 1 ? (split * kWeights * ((most + split - 1) / split) * kFp4SumPitch * 4 + 1023) / 1024 * 1024 : 0;
    int smem = p.stages * stage_bytes;
    if (smem < p.sums_at + sums) smem = p.sums_at + sums;
    if (smem < kFp4SplitMinSmem) smem = kFp4SplitMinSmem;
    if (smem > kFp4SplitMaxSmem) return (int)cudaErrorInvalidValue;   // gated, 64 rows, split: 136 KB
    CUtensorMap tm_a, tm_b, tm_b2;
    const uint64_t pitch = uint64_t(g->K) / 2;
    int rc = make_tmap_2d(&tm_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g->a, g->M, pitch, pitch, p.a_rows, 128, true);
    if (!rc) rc = make_tmap_2d(&tm_b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g->b, g->N, pitch, pitch, 128, 128, true);
    tm_b2 = tm_b;
    if (GATED && !rc) rc = make_tmap_2d(&tm_b2, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g->b2, g->N, pitch, pitch, 128, 128, true);
    if (!rc) rc = configure_smem<kernel>(kFp4SplitMaxSmem + 1024);
    if (rc) return rc;
    return launch_dependent_clusters(kernel, split, dim3(int(tiles) * split), kFp4Threads, smem + 1024, stream, tm_a,
                                     tm_b, tm_b2, p);
}

// The split form for few rows and for products whose tiles it holds all at once, pairs of SMs for the others. MX, us per call, pairs : split:
// plain, N = 2048: 512 rows K = 512 5.2 : 4.0, K = 2048 7.1 : 5.7, 3000 rows 7.5 : 10.6, 11.4 : 19.1; gated, N = 2048, 256 rows (64 tiles) K = 1024 6.3 :
// 5.7, 384 rows (96) 6.5 : 5.8, 512 rows (128) K = 512 5.8 : 6.4, K = 2048 7.4 : 7.5.
template <int FMT, bool GATED, typename T>
int gemm_fp4_dispatch(const fluke_sm100_gemm_fp4_t *g, cudaStream_t stream) {
    if (g->M <= 64 || split_tiles<GATED>(g) <= (GATED ? 100 : device_sm_count())) return gemm_fp4_split_launch<FMT, GATED, T>(g, stream);
    if (g->K <= 512) return gemm_fp4_pair_launch<FMT, GATED, 2, T>(g, stream);
    if (g->K <= 1024) return gemm_fp4_pair_launch<FMT, GATED, 4, T>(g, stream);
    return gemm_fp4_pair_launch<FMT, GATED, 0, T>(g, stream);
}
template <int FMT, typename T>
int gemm_fp4_dispatch(const fluke_sm100_gemm_fp4_t *g, cudaStream_t stream) {
    return g->b2 ? gemm_fp4_dispatch<FMT, true, T>(g, stream) : gemm_fp4_dispatch<FMT, false, T>(g, stream);
}

}  // namespace
}  // namespace fluke_sm100

extern "C" int fluke_sm100_gemm_fp4(const fluke_sm100_gemm_fp4_t *g, void *stream) {
    using namespace fluke_sm100;
    if (!g || !fp4_shape_ok(g->M, g->K) || g->N <= 0 || g->N > kFp4MaxSize || g->N % 8 != 0) return (int)cudaErrorInvalidValue;
    if (g->format != FLUKE_SM100_FP4_MX && g->format != FLUKE_SM100_FP4_NV) return (int)cudaErrorInvalidValue;
    if (g->M == 0) return 0;
    const bool nv = g->format == FLUKE_SM100_FP4_NV;
    if (!g->a || !g->a_scale || !g->b || !g->b_scale || !g->out || (g->b2 && !g->b2_scale)) return (int)cudaErrorInvalidValue;
    if (nv && (!g->a_row || !g->b_row || (g->b2 && !g->b2_row))) return (int)cudaErrorInvalidValue;
    if (!aligned16(g->a) || !aligned16(g->a_scale) || !aligned16(g->b) || !aligned16(g->b_scale) || !aligned16(g->b2) || !aligned16(g->b2_scale) ||
        !aligned16(g->out) || (nv && (!aligned4(g->a_row) || !aligned16(g->b_row) || !aligned16(g->b2_row))))
        return (int)cudaErrorMisalignedAddress;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (nv) return g->bf16 ? gemm_fp4_dispatch<FLUKE_SM100_FP4_NV, __nv_bfloat16>(g, s) : gemm_fp4_dispatch<FLUKE_SM100_FP4_NV, __half>(g, s);
    return g->bf16 ? gemm_fp4_dispatch<FLUKE_SM100_FP4_MX, __nv_bfloat16>(g, s) : gemm_fp4_dispatch<FLUKE_SM100_FP4_MX, __half>(g, s);
}

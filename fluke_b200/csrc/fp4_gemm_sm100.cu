// fp4_gemm_sm100.cu -- products of microscaled 4-bit matrices on sm_100a:
//     out[m, n] = round16( sum_k a[m, k] b[n, k]  [* ga[m] * gb[n]] )
// with a and b as codes, block scales and (NV) row scales of fp4_rows_sm100.cu, and the gated form
//     out = round16( silu(a gate^T) * (a up^T) ).
//
// The tensor cores take the codes as they are stored and apply the block scales themselves
// (tcgen05.mma .block_scale, kind mxf4 and mxf4nvf4: 64 values of K per instruction, f32 accumulators in tensor
// memory), so nothing is decoded on the way: TMA brings 128-byte-swizzled blocks of 256 values of K per row into a ring of
// stages, bulk copies bring the stage's scale tiles, and tcgen05.cp moves those to tensor memory, where the instruction reads
// them. Row scales are powers of two and are applied to the accumulators, which is exact.
//
//   warp 0      loader (one thread)
//   warp 1      tensor memory, scale copies and MMAs (one thread)
//   warps 2-3   idle
//   warps 4-11  epilogue: two warps per quadrant of tensor-memory lanes, thread = row
//
// The scale tiles of a stage have tensor-memory columns of their own: they are overwritten when the stage is filled
// again, which the MMAs that read them have announced.

namespace fluke_sm100 {
namespace {

constexpr int kFp4Threads = 384;
constexpr int kFp4StageK = 256;       // values of K per stage: 128 bytes per row

struct Fp4GemmDev {
    int M, N, K;
    int n_tiles, tiles, stages_k;     // output tiles along N, in all; ring stages per tile
    int sf_tiles;                     // 512-byte scale tiles per 128 rows
    const uint8_t *sfa, *sfb, *sfb2;
    const float *ga, *gb, *gb2;
};

template <int FMT>
__device__ __forceinline__ void tc_mma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if constexpr (FMT == FLUKE_SM100_FP4_MX)
        asm volatile(
            "{\n.reg .pred P;\nsetp.ne.b32 P, %6, 0;\n"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], P;\n}\n"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n.reg .pred P;\nsetp.ne.b32 P, %6, 0;\n"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], P;\n}\n"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
}
// 32 rows of 16 bytes from shared memory to four tensor-memory columns, the same in all four lane quadrants.
__device__ __forceinline__ void tc_copy_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// Descriptor of a scale tile: 32 rows of 16 bytes without swizzle, 8 rows 128 bytes apart.
__device__ __forceinline__ uint64_t make_smem_desc_scales(uint32_t byte_addr) {
    return uint64_t((byte_addr & 0x3FFFFu) >> 4) | uint64_t(128 >> 4) << 32 | uint64_t(1) << 46;
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

template <int FMT, bool GATED, int BN>
struct Fp4Layout {
    static constexpr int kBlock = FMT == FLUKE_SM100_FP4_MX ? 32 : 16;
    static constexpr int kAtoms = kFp4StageK / (4 * kBlock);         // scale tiles per stage and 128 rows
    static constexpr int kBTiles = (BN + 127) / 128;                 // of B (gated: one each of gate and up)
    static constexpr int kABytes = 128 * 128, kBBytes = BN * 128;
    static constexpr int kSfA = kAtoms * 512, kSfB = kBTiles * kAtoms * 512;
    static constexpr int kStageBytes = kABytes + kBBytes + kSfA + kSfB;
    static constexpr int kStaging = 8 * 32 * 128;
    static constexpr int kStages = (226 * 1024 - kStaging - 1024 - 512) / kStageBytes < 6 ? (226 * 1024 - kStaging - 1024 - 512) / kStageBytes : 6;
    static constexpr int kSfCols = kAtoms * 4 * (1 + kBTiles);       // tensor-memory columns of a stage's scales
    static constexpr int kAccs = 2 * BN + kStages * kSfCols <= 512 ? 2 : 1;
    static_assert(kAccs * BN + kStages * kSfCols <= 512, "tensor memory");
    // the stages' operands first (1024-byte aligned), then their scales
    static constexpr int kOffSf = kStages * (kABytes + kBBytes);
    static constexpr int kOffStaging = kStages * kStageBytes;
    static constexpr int kOffBars = kOffStaging + kStaging;
    static constexpr int kDynamic = kOffBars + (2 * kStages + 4) * 8 + 16 + 1024;
    static_assert(kOffStaging % 1024 == 0 && kDynamic <= 232448, "shared memory");
};

template <int FMT, bool GATED, int BN, typename T>
__global__ void __launch_bounds__(kFp4Threads, 1)
gemm_fp4_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_b2,
                const __grid_constant__ CUtensorMap tm_out, const Fp4GemmDev p) {
    using L = Fp4Layout<FMT, GATED, BN>;
    constexpr int STAGES = L::kStages, ACCS = L::kAccs;
    constexpr int BN_OUT = GATED ? BN / 2 : BN;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kOffBars);
    uint64_t *full_bar = bars, *empty_bar = bars + STAGES, *tfull_bar = bars + 2 * STAGES, *tempty_bar = tfull_bar + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * STAGES + 4);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&tfull_bar[s], 1);
            mbar_init(&tempty_bar[s], 8);
        }
        *abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tm_a);
        tma_prefetch_desc(&tm_b);
        if (GATED) tma_prefetch_desc(&tm_b2);
        tma_prefetch_desc(&tm_out);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        dependency_trigger();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    dependency_wait();

    if (warp == 0) {
        if (elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x) {
                const int m_tile = tile / p.n_tiles, m0 = m_tile * 128, n0 = (tile - m_tile * p.n_tiles) * BN_OUT;
                const uint8_t *sfa = p.sfa + int64_t(m_tile) * p.sf_tiles * 512;
                const uint8_t *sfb = p.sfb + int64_t(n0 >> 7) * p.sf_tiles * 512;
                // the second 128 rows of B, where there are any
                const uint8_t *sfb2 = GATED ? p.sfb2 + int64_t(n0 >> 7) * p.sf_tiles * 512 : sfb + int64_t(p.sf_tiles) * 512;
                const bool second = GATED || (L::kBTiles == 2 && n0 + 128 < p.N);
                for (int ks = 0; ks < p.stages_k; ++ks) {
                    ok = mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, 120);
                    if (!ok) break;
                    const uint32_t sf_bytes = min(L::kAtoms, p.sf_tiles - ks * L::kAtoms) * 512;
                    uint8_t *sa = smem + stage * (L::kABytes + L::kBBytes), *sb = sa + L::kABytes;
                    uint8_t *ssa = smem + L::kOffSf + stage * (L::kSfA + L::kSfB), *ssb = ssa + L::kSfA;
                    mbar_arrive_expect_tx(&full_bar[stage], L::kABytes + L::kBBytes + sf_bytes * (second ? 3 : 2));
                    tma_load_2d(sa, &tm_a, &full_bar[stage], ks * 128, m0);
                    tma_load_2d(sb, &tm_b, &full_bar[stage], ks * 128, n0);
                    if constexpr (GATED) tma_load_2d(sb + L::kBBytes / 2, &tm_b2, &full_bar[stage], ks * 128, n0);
                    bulk_load(ssa, sfa + int64_t(ks) * L::kSfA, sf_bytes, &full_bar[stage]);
                    bulk_load(ssb, sfb + int64_t(ks) * L::kSfA, sf_bytes, &full_bar[stage]);
                    if (second) bulk_load(ssb + L::kSfA, sfb2 + int64_t(ks) * L::kSfA, sf_bytes, &full_bar[stage]);
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
        if (elect_one()) {
            int stage = 0, local = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x, ++local) {
                const int acc = local % ACCS;
                ok = mbar_wait(&tempty_bar[acc], ((local / ACCS) & 1) ^ 1u, abort_flag, 121);
                if (!ok) break;
                tc_fence_after_sync();
                for (int ks = 0; ks < p.stages_k; ++ks) {
                    ok = mbar_wait(&full_bar[stage], phase, abort_flag, 122);
                    if (!ok) break;
                    tc_fence_after_sync();
                    const uint32_t sa = smem_u32(smem) + stage * (L::kABytes + L::kBBytes);
                    const uint32_t ssa = smem_u32(smem) + L::kOffSf + stage * (L::kSfA + L::kSfB);
                    const uint32_t tsa = tmem + ACCS * BN + stage * L::kSfCols, tsb = tsa + L::kAtoms * 4;
#pragma unroll
                    for (int i = 0; i < L::kAtoms; ++i) {
                        tc_copy_scales(tsa + i * 4, make_smem_desc_scales(ssa + i * 512));
#pragma unroll
                        for (int t = 0; t < L::kBTiles; ++t)
                            tc_copy_scales(tsb + (i * L::kBTiles + t) * 4, make_smem_desc_scales(ssa + L::kSfA + (t * L::kAtoms + i) * 512));
                    }
                    const uint64_t ad = make_smem_desc_sw128(sa), bd = make_smem_desc_sw128(sa + L::kABytes);
                    const int steps = min(4, (p.K - ks * kFp4StageK + 63) / 64);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (k >= steps) break;
                        // 64 values: two scales of a cell (MX: halves of it in turns), or all four
                        constexpr bool mx = FMT == FLUKE_SM100_FP4_MX;
                        const int atom = mx ? k / 2 : k, part = mx ? (k & 1) * 2 : 0;
                        tc_mma_fp4<FMT>(tmem + acc * BN, ad + uint64_t(2 * k), bd + uint64_t(2 * k), make_idesc_fp4<FMT>(128, BN, part),
                                        tsa + atom * 4, tsb + atom * L::kBTiles * 4, (ks | k) != 0);
                    }
                    tc_commit(&empty_bar[stage]);
                    if (ks == p.stages_k - 1) tc_commit(&tfull_bar[acc]);
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                }
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        const int q = warp & 3, half = (warp - 4) >> 2;
        uint8_t *staging = smem + L::kOffStaging + (warp - 4) * (32 * 128);
        int local = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x, ++local) {
            const int m_tile = tile / p.n_tiles, m0 = m_tile * 128, n0 = (tile - m_tile * p.n_tiles) * BN_OUT;
            const int acc = local % ACCS, row = m0 + q * 32 + lane;
            float ga = 1.f;
            if (FMT == FLUKE_SM100_FP4_NV && row < p.M) ga = p.ga[row];
            ok = mbar_wait(&tfull_bar[acc], (local / ACCS) & 1, abort_flag, 123);
            if (!ok) break;
            tc_fence_after_sync();
            const uint32_t t_row = tmem + (uint32_t(q * 32) << 16) + acc * BN;
            constexpr int kGroups = BN_OUT / 128;  // of 64 columns, per warp
#pragma unroll 1
            for (int c64 = 0; c64 < kGroups; ++c64) {
                const int c0 = (half * kGroups + c64) * 64;
                if (n0 + c0 < p.N) {
                    if (lane == 0) tma_store_wait_read<0>();
                    __syncwarp();
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
                        uint32_t a[32], u[GATED ? 32 : 1], w[16];
                        tmem_ld_32x32(t_row + c0 + 32 * h, a);
                        if constexpr (GATED) tmem_ld_32x32(t_row + BN_OUT + c0 + 32 * h, u);
                        tmem_ld_wait();
#pragma unroll
                        for (int c = 0; c < 32; c += 4) {
                            float4 gb = make_float4(1.f, 1.f, 1.f, 1.f), gu = gb;
                            const int col = n0 + c0 + 32 * h + c;
                            if (FMT == FLUKE_SM100_FP4_NV && col < p.N) {
                                gb = *reinterpret_cast<const float4 *>(p.gb + col);
                                if (GATED) gu = *reinterpret_cast<const float4 *>(p.gb2 + col);
                            }
                            float o[4];
                            const float sb[4] = {gb.x, gb.y, gb.z, gb.w}, su[4] = {gu.x, gu.y, gu.z, gu.w};
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                float v = __uint_as_float(a[c + i]);
                                if (FMT == FLUKE_SM100_FP4_NV) v = (v * ga) * sb[i];
                                if constexpr (GATED) {
                                    float up = __uint_as_float(u[c + i]);
                                    if (FMT == FLUKE_SM100_FP4_NV) up = (up * ga) * su[i];
                                    const float hg = 0.5f * v;
                                    v = fmaf(hg, tanh_approx(hg), hg) * up;
                                }
                                o[i] = v;
                            }
                            w[c / 2] = pack2(make_float2(o[0], o[1]), T());
                            w[c / 2 + 1] = pack2(make_float2(o[2], o[3]), T());
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            *reinterpret_cast<uint4 *>(staging + sw128_offset(lane, 4 * h + j)) =
                                make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&tm_out, staging, n0 + c0, m0 + q * 32);
                        tma_store_commit();
                    }
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tempty_bar[acc]);
        }
        if (lane == 0) tma_store_wait_all<0>();
        __syncwarp();
    }

    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
}

template <int FMT, bool GATED, int BN, typename T>
int gemm_fp4_launch(const fluke_sm100_gemm_fp4_t *g, cudaStream_t stream) {
    using L = Fp4Layout<FMT, GATED, BN>;
    constexpr int BN_OUT = GATED ? BN / 2 : BN;
    Fp4GemmDev p;
    p.M = g->M; p.N = g->N; p.K = g->K;
    p.n_tiles = (g->N + BN_OUT - 1) / BN_OUT;
    const int64_t tiles = int64_t((g->M + 127) / 128) * p.n_tiles;
    if (tiles > INT32_MAX - 1024) return (int)cudaErrorInvalidValue;
    p.tiles = int(tiles);
    p.stages_k = (g->K + kFp4StageK - 1) / kFp4StageK;
    p.sf_tiles = fp4_tiles(g->K, FMT);
    p.sfa = static_cast<const uint8_t *>(g->a_scale);
    p.sfb = static_cast<const uint8_t *>(g->b_scale);
    p.sfb2 = static_cast<const uint8_t *>(g->b2_scale);
    p.ga = g->a_row; p.gb = g->b_row; p.gb2 = g->b2_row;
    CUtensorMap tm_a, tm_b, tm_b2, tm_out;
    const uint64_t pitch = uint64_t(g->K) / 2;
    int rc = make_tmap_2d(&tm_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g->a, g->M, pitch, pitch, 128, 128, true);
    if (rc) return rc;
    rc = make_tmap_2d(&tm_b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g->b, g->N, pitch, pitch, BN_OUT, 128, true);
    if (rc) return rc;
    tm_b2 = tm_b;
    if (GATED) {
        rc = make_tmap_2d(&tm_b2, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g->b2, g->N, pitch, pitch, BN_OUT, 128, true);
        if (rc) return rc;
    }
    rc = make_tmap_2d(&tm_out, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, g->out, g->M, g->N, uint64_t(g->N) * 2, 32, 64, true);
    if (rc) return rc;
    rc = configure_smem<gemm_fp4_kernel<FMT, GATED, BN, T>>(L::kDynamic);
    if (rc) return rc;
    const int grid = p.tiles < device_sm_count() ? p.tiles : device_sm_count();
    return launch_dependent(gemm_fp4_kernel<FMT, GATED, BN, T>, grid, kFp4Threads, L::kDynamic, stream, tm_a, tm_b, tm_b2, tm_out, p);
}

template <int FMT, typename T>
int gemm_fp4_dispatch(const fluke_sm100_gemm_fp4_t *g, cudaStream_t stream) {
    if (g->b2) return gemm_fp4_launch<FMT, true, 256, T>(g, stream);
    return gemm_fp4_launch<FMT, false, 128, T>(g, stream);
}

}  // namespace
}  // namespace fluke_sm100

extern "C" int fluke_sm100_gemm_fp4(const fluke_sm100_gemm_fp4_t *g, void *stream) {
    using namespace fluke_sm100;
    if (!g || !fp4_shape_ok(g->M, g->K) || g->N <= 0 || g->N % 8 != 0) return (int)cudaErrorInvalidValue;
    if (g->format != FLUKE_SM100_FP4_MX && g->format != FLUKE_SM100_FP4_NV) return (int)cudaErrorInvalidValue;
    if (g->M == 0) return 0;
    const bool nv = g->format == FLUKE_SM100_FP4_NV;
    if (!g->a || !g->a_scale || !g->b || !g->b_scale || !g->out || (g->b2 && !g->b2_scale)) return (int)cudaErrorInvalidValue;
    if (nv && (!g->a_row || !g->b_row || (g->b2 && !g->b2_row))) return (int)cudaErrorInvalidValue;
    if (!aligned16(g->a) || !aligned16(g->a_scale) || !aligned16(g->b) || !aligned16(g->b_scale) || !aligned16(g->b2) || !aligned16(g->b2_scale) ||
        !aligned16(g->out) || (nv && (!aligned16(g->b_row) || !aligned16(g->b2_row))))
        return (int)cudaErrorMisalignedAddress;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (nv) return g->bf16 ? gemm_fp4_dispatch<FLUKE_SM100_FP4_NV, __nv_bfloat16>(g, s) : gemm_fp4_dispatch<FLUKE_SM100_FP4_NV, __half>(g, s);
    return g->bf16 ? gemm_fp4_dispatch<FLUKE_SM100_FP4_MX, __nv_bfloat16>(g, s) : gemm_fp4_dispatch<FLUKE_SM100_FP4_MX, __half>(g, s);
}

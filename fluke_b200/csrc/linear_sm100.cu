// linear_sm100.cu -- products of 16-bit matrices with an epilogue on sm_100a:
//     out[m, n] = round16( act( sum_k x[m, k] w[n, k] + bias[n] ) + alpha residual[m, n] )
// with x [M, K], w [N, K], residual and out [M, N] in f16 or bf16, sums and everything behind them in f32.
//
// TMA brings 128-byte-swizzled blocks of 64 values of K per row, tcgen05.mma (kind f16, 16 values of K per instruction) sums them
// up in tensor memory, and the epilogue takes the sums through registers, where bias, activation and residual cost no pass over memory.
//
// Two forms (linear_dispatch chooses): few tiles with K split over a cluster, bound by latency or by reading the weight ([1, 4096] x [4096, 4096] 8.8 us, of which
// the loads take 5.1 at 6.5 TB/s; [333, 512] x [1536, 512] 5.0), and pairs of SMs, bound by memory at small K ([32000, 512] x [512, 512] with bias and residual 27.9 us, 99 MB) and by the MMAs
// at the power limit at large ([8192, 4096] x [8192, 4096] 413 us, 1.33 PFLOP/s).

namespace fluke_sm100 {
namespace {

constexpr int kLinThreads = 384;
constexpr int kLinStageK = 64;        // values of K per stage: 128 bytes per row

// The low word of a 128-byte-swizzled operand's descriptor changes, the high word is kDescHiSw128.
template <int GROUP>
__device__ __forceinline__ void tc_mma_f16(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    if constexpr (GROUP == 1)
        asm volatile(
            "{\n.reg .pred P;\n.reg .b64 A, B;\nsetp.ne.b32 P, %4, 0;\nmov.b64 A, {%1, %5};\nmov.b64 B, {%2, %5};\n"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], A, B, %3, P;\n}\n"
            ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHiSw128) : "memory");
    else
        asm volatile(
            "{\n.reg .pred P;\n.reg .b64 A, B;\nsetp.ne.b32 P, %4, 0;\nmov.b64 A, {%1, %5};\nmov.b64 B, {%2, %5};\n"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], A, B, %3, P;\n}\n"
            ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHiSw128) : "memory");
}
// f32 sums of two f16 or two bf16 matrices, both K-major (the fields are those of make_idesc).
template <typename T>
__host__ __device__ constexpr uint32_t make_idesc_16(int M, int N) {
    const uint32_t fmt = std::is_same_v<T, __nv_bfloat16> ? 1u : 0u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}

// ---- activations ------------------------------------------------------------------------------
// In f32, with an error small against the 2^-12 of the last rounding (f16). ex2.approx and rcp.approx are 2^-22 and 2^-23 off, an
// exponent's argument 2^-24 of itself.
//   sigmoid, silu  1 / (1 + exp(-v)): nothing cancels.
//   tanh           (1 - t) / (1 + t) with t = exp(-2 |v|), whose numerator keeps 2^-17 at the |v| of 1/64 below which v - v^3 / 3 is used (the
//                  next term, 2/15 v^4 of it, is 2^-26).
//   gelu           v Phi(v), Phi the normal distribution: Phi(-a) = exp(-a^2 / 2) t P(t) with t = 1 / (1 + 0.31 a), P of degree five fitted to
//                  erfcx(a / sqrt(2)) / 2 with 4.7e-6 of it at most for 0 <= a <= 14; 1 - Phi(-a) for v >= 0.
// An infinity gives the limit and a NaN a NaN, except that v sigmoid(v) and v Phi(v) of -inf are NaN (inf * 0), as the formulas say.
enum LinAct { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActTanh = 4, kActSigmoid = 5 };

template <int ACT>
__device__ __forceinline__ float2 activate(float2 v) {
    const auto one = [](float x) { return make_float2(x, x); };
    const auto exp2_of = [](float2 x) { return make_float2(ex2_approx(x.x), ex2_approx(x.y)); };
    const auto rcp_of = [](float2 x) { return make_float2(rcp_approx(x.x), rcp_approx(x.y)); };
    if constexpr (ACT == kActRelu) return make_float2(v.x < 0.f ? 0.f : v.x, v.y < 0.f ? 0.f : v.y);
    if constexpr (ACT == kActSilu || ACT == kActSigmoid) {
        const float2 s = rcp_of(add2(exp2_of(mul2(v, one(-1.44269504f))), one(1.f)));
        return ACT == kActSilu ? mul2(v, s) : s;
    }
    if constexpr (ACT == kActTanh) {
        const float2 a = make_float2(fabsf(v.x), fabsf(v.y)), t = exp2_of(mul2(a, one(-2.88539008f)));
        const float2 big = mul2(fma2(t, one(-1.f), one(1.f)), rcp_of(add2(t, one(1.f))));
        const float2 small = fma2(mul2(mul2(v, v), v), one(-0.333333333f), v);
        return make_float2(a.x < 0.015625f ? small.x : copysignf(big.x, v.x), a.y < 0.015625f ? small.y : copysignf(big.y, v.y));
    }
    if constexpr (ACT == kActGelu) {
        const float2 a = make_float2(fabsf(v.x), fabsf(v.y)), t = rcp_of(fma2(a, one(0.31f), one(1.f)));
        float2 q = fma2(t, one(-0.0739276186f), one(0.180445790f));
        q = fma2(q, t, one(0.0157500077f));
        q = fma2(q, t, one(0.133426800f));
        q = fma2(q, t, one(0.120442092f));
        q = fma2(q, t, one(0.123860620f));
        const float2 h = mul2(mul2(q, t), exp2_of(mul2(mul2(a, a), one(-0.721347520f)))), rest = fma2(h, one(-1.f), one(1.f));
        return mul2(v, make_float2(v.x < 0.f ? h.x : rest.x, v.y < 0.f ? h.y : rest.y));
    }
    return v;
}

// What a product adds to its sums.
struct LinEpilogue {
    const void *bias, *residual;      // or null
    void *out;
    int64_t ld_residual, ld_out;
    float alpha;
};

// Eight columns of a row: sums plus bias through the activation, plus alpha times the residual, as 16 bits.
template <typename T, int ACT>
__device__ __forceinline__ uint4 finish8(const float (&sum)[8], const uint4 *bias, const uint4 *residual, float alpha) {
    uint32_t w[4];
    const uint32_t *b = reinterpret_cast<const uint32_t *>(bias), *r = reinterpret_cast<const uint32_t *>(residual);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float2 v = make_float2(sum[2 * i], sum[2 * i + 1]);
        if (bias) v = add2(v, unpack2(b[i], T()));
        v = activate<ACT>(v);
        if (residual) v = fma2(make_float2(alpha, alpha), unpack2(r[i], T()), v);
        w[i] = pack2(v, T());
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// ---- few tiles: weights as the first operand, K split over a cluster --------------------------------
// A tile is 128 rows of the weight x up to 128 rows of x, with the weight as the MMA's first operand: a few rows of x cost a few
// columns of tensor memory and of time, and the weight's rows fill the lanes. With few tiles a tile is given to a cluster of up
// to 8 CTAs, each of which takes a run of K; they leave their f32 sums in their own shared memory, and every CTA then adds
// up a share of the tile from all of them, in the order of the ranks. What bounds it is latency, and for one or a few rows
// reading the weights.
//
// A CTA takes 128 of an SM's 512 tensor-memory columns, and less than half of its shared memory (a ring of up to 104 KB; the sums and the shares of tiles
// of up to 64 rows are less), so that the next kernel's CTAs are set up beside it. Two kinds of launches take more and leave no room for them: the deep ring, 152 KB, for a run of
// K that a smaller one does not hold, and split tiles of 128 rows, up to 135 KB of sums and shares.
constexpr int kLinSplitSmem = 104 * 1024, kLinSplitMinSmem = 78 * 1024, kLinSplitDeep = 152 * 1024, kLinSplitMaxSmem = 160 * 1024;
constexpr int kLinSplitStages = 8, kLinSplitCols = 128;
constexpr int kLinSumPitch = 132;              // floats between rows of the sums

struct LinSplitDev {
    int M, N;
    int n_tiles, stages_k, split;     // tiles along N; ring stages of all of K; CTAs per tile
    int last_steps;                   // MMAs of the last stage
    int rows, stages;                 // rows of x per tile (a multiple of 16), ring stages
    int sums_at;                      // byte offset of the sums in shared memory
    LinEpilogue e;
};

template <typename T, int ACT>
__global__ void __launch_bounds__(kLinThreads, 2)
linear_split_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const LinSplitDev p) {
    constexpr int kWBytes = 128 * 128;
    extern __shared__ uint8_t smem_raw[];
    // every CTA of the cluster computes the same offset
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t full_bar[kLinSplitStages], empty_bar[kLinSplitStages], done_bar, sums_bar;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    volatile int *abort_flag = &abort_word;
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
    const int rank = int(blockIdx.x) % p.split, tile = int(blockIdx.x) / p.split;
    const int m_tile = tile / p.n_tiles, m0 = m_tile * p.rows, n0 = (tile - m_tile * p.n_tiles) * 128;
    const int ks0 = p.stages_k * rank / p.split, ks1 = p.stages_k * (rank + 1) / p.split;
    const int slot = kWBytes + p.rows * 128;   // per stage the weight's rows, then those of x

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        mbar_init(&done_bar, 1);
        mbar_init(&sums_bar, 1);
        abort_word = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tm_x);
        tma_prefetch_desc(&tm_w);
    }
    if (warp == 1) {
        tmem_alloc(&tmem_slot, kLinSplitCols);
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
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int ks = ks0; ks < ks1; ++ks) {
                ok = mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, 150);
                if (!ok) break;
                uint8_t *sw = smem + stage * slot;
                mbar_arrive_expect_tx(&full_bar[stage], slot);
                tma_load_2d(sw, &tm_w, &full_bar[stage], ks * kLinStageK, n0);
                tma_load_2d(sw + kWBytes, &tm_x, &full_bar[stage], ks * kLinStageK, m0);
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
        const uint32_t w_lo0 = desc_lo(smem_u32(smem)), idesc = make_idesc_16<T>(128, 0) | (uint32_t(p.rows >> 3) << 17);
        int stage = 0;
        uint32_t phase = 0;
        for (int ks = ks0; ks < ks1; ++ks) {
            if (!mbar_wait_warp(&full_bar[stage], phase, abort_flag, 151)) break;
            tc_fence_after_sync();
            const uint32_t w_lo = w_lo0 + stage * (slot >> 4), x_lo = w_lo + (kWBytes >> 4);
            const int steps = ks == p.stages_k - 1 ? p.last_steps : 4;
            if (leader) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (k < steps) tc_mma_f16<1>(tmem, w_lo + 2 * k, x_lo + 2 * k, idesc, ks > ks0 || k > 0);
                tc_commit(&empty_bar[stage]);
                if (ks == ks1 - 1) tc_commit(&done_bar);
            }
            if (++stage == p.stages) { stage = 0; phase ^= 1u; }
        }
        __syncwarp();
    }

    // The sums as [row of x, weight row] behind the ring; and in front of it, where the first loads went (all of them have been used by then
    // everywhere: (2)), what the ranks send of this CTA's share of the rows, [rank, row, weight row].
    const int rows = min(p.rows, p.M - m0);
    const int share = (rows + p.split - 1) / p.split, row0 = min(rank * share, rows), mine = min(share, rows - row0);
    float *sums = reinterpret_cast<float *>(smem + p.sums_at);
    bool ok = true;
    if (warp >= 4) {
        const int q = warp & 3, half = (warp - 4) >> 2;
        ok = mbar_wait_warp(&done_bar, 0, abort_flag, 152);
        if (ok) {
            tc_fence_after_sync();
            for (int c0 = half * 8; c0 < rows; c0 += 16) {
                uint32_t a[8];
                tmem_ld_32x8(tmem + (uint32_t(q * 32) << 16) + c0, a);
                tmem_ld_wait();
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    if (c0 + c < rows) sums[(c0 + c) * kLinSumPitch + q * 32 + lane] = __uint_as_float(a[c]);
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
    const float *parts = sums + row0 * kLinSumPitch;
    int rank_pitch = 0;                 // floats between the ranks
    if (p.split > 1) {
        parts = reinterpret_cast<const float *>(smem);
        rank_pitch = share * kLinSumPitch;
        if (warp == 0 && ok) {
            if (lane == 0 && mine > 0) mbar_arrive_expect_tx(&sums_bar, p.split * mine * kLinSumPitch * 4);
            // lane = rank that a share goes to
            const int theirs = min(share, rows - min(lane * share, rows));
            if (lane < p.split && theirs > 0)
                bulk_send(cluster_address(smem_u32(smem) + rank * rank_pitch * 4, lane), sums + lane * share * kLinSumPitch, theirs * kLinSumPitch * 4,
                          cluster_address(smem_u32(&sums_bar), lane));
        }
        if (warp >= 4 && ok && mine > 0) ok = mbar_wait_warp(&sums_bar, 0, abort_flag, 153);
    }
    if (warp >= 4 && ok) {
        // eight output columns of a row per turn
        for (int g = int(threadIdx.x) - 128; g < mine * 16; g += 256) {
            const int row = g >> 4, c = (g & 15) * 8, col = n0 + c;
            if (col >= p.N) continue;
            const int64_t out_row = m0 + row0 + row;
            uint4 bias, residual;
            if (p.e.bias) bias = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.e.bias) + col);
            if (p.e.residual) residual = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.e.residual) + out_row * p.e.ld_residual + col);
            float v[8] = {};
#pragma unroll 2
            for (int r = 0; r < p.split; ++r)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float4 x = *reinterpret_cast<const float4 *>(parts + r * rank_pitch + row * kLinSumPitch + c + i * 4);
                    v[i * 4] += x.x;
                    v[i * 4 + 1] += x.y;
                    v[i * 4 + 2] += x.z;
                    v[i * 4 + 3] += x.w;
                }
            *reinterpret_cast<uint4 *>(static_cast<T *>(p.e.out) + out_row * p.e.ld_out + col) =
                finish8<T, ACT>(v, p.e.bias ? &bias : nullptr, p.e.residual ? &residual : nullptr, p.e.alpha);
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
        tmem_dealloc(tmem, kLinSplitCols);
    }
}

// ---- many tiles: pairs of SMs -------------------------------------------------------------------
// A pair of CTAs (cluster of 2) works on tiles of 256 rows of x by BN columns with tcgen05 cta_group::2. Each CTA loads its own 128
// rows of x and half of the weight's rows and holds its 128 rows of the sums; the first CTA issues for both. The sums have two
// buffers in tensor memory, so that the epilogue of a tile runs under the MMAs of the next. The tiles of a residual come by TMA into the
// staging that the output leaves from, ahead of the sums.
//
// In each CTA warp 0 loads (one thread), warp 1 owns tensor memory and (first CTA) issues MMAs, warps 2-3 are idle and the others are
// the epilogue, 32 rows x 64 columns each: with half as many, of 128 columns, a tile with bias and residual took its warps 9000 cycles and its MMAs at
// K = 512 4000, most of it latency (loads of the bias and of the staging behind stores that may be to the same place; a proxy fence and a store per group).
//
// Pairs take tiles in turns, and the tiles are ordered in bands of kLinBand rows of tiles, column by column: what runs at the same time shares
// rows of x and of the weight in L2.
constexpr int kLinBand = 8;
template <int BN>
struct LinPairLayout {
    static constexpr int kOperandX = 128 * 128, kOperandW = BN / 2 * 128, kSlot = kOperandX + kOperandW;
    static constexpr int kEpilogueWarps = BN / 16, kThreads = 128 + kEpilogueWarps * 32;
    static constexpr int kStages = BN == 256 ? 5 : 7;
    static constexpr int kOffStaging = kStages * kSlot;        // per epilogue warp 32 rows x 64 columns
    static constexpr int kOffBars = kOffStaging + kEpilogueWarps * 32 * 128;
    static constexpr int kBars = 2 * kStages + 4 + kEpilogueWarps;
    static constexpr int kDynamic = kOffBars + kBars * 8 + 16 + 1024;
    static_assert(kOffStaging % 1024 == 0 && kDynamic <= 232448, "shared memory");
};

struct LinPairDev {
    int M, N;
    int m_tiles, n_tiles, tiles, stages_k;
    int last_steps;                   // MMAs of the last stage
    int passes_by;                    // the output is larger than what L2 can keep, its lines go first
    const void *bias;
    int residual;
    float alpha;
};

// The tiles of a pair, one after the other.
struct LinRun {
    int tile, m, n;
    __device__ __forceinline__ explicit LinRun(const LinPairDev &p) : tile(int(blockIdx.x) >> 1) { place(p); }
    __device__ __forceinline__ bool left(const LinPairDev &p) const { return tile < p.tiles; }
    __device__ __forceinline__ void next(const LinPairDev &p) {
        tile += int(gridDim.x) >> 1;
        if (left(p)) place(p);
    }
    __device__ __forceinline__ void place(const LinPairDev &p) {
        const int band = tile / (kLinBand * p.n_tiles), at = tile - band * kLinBand * p.n_tiles, rows = min(kLinBand, p.m_tiles - band * kLinBand);
        n = at / rows;
        m = band * kLinBand + at - n * rows;
    }
};

template <typename T, int ACT, int BN>
__global__ void __launch_bounds__(LinPairLayout<BN>::kThreads, 1)
linear_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_res,
                   const __grid_constant__ CUtensorMap tm_out, const LinPairDev p) {
    using L = LinPairLayout<BN>;
    constexpr int STAGES = L::kStages;
    extern __shared__ uint8_t smem_raw[];
    // both CTAs compute the same offset
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kOffBars);
    uint64_t *full_bar = bars, *empty_bar = bars + STAGES, *tfull_bar = bars + 2 * STAGES, *tempty_bar = tfull_bar + 2, *res_bar = tempty_bar + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + L::kBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
    const int rank = int(blockIdx.x & 1);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&tfull_bar[s], 1);
            mbar_init(&tempty_bar[s], 2 * L::kEpilogueWarps);
        }
        for (int s = 0; s < L::kEpilogueWarps; ++s) mbar_init(&res_bar[s], 1);
        *abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tm_x);
        tma_prefetch_desc(&tm_w);
        tma_prefetch_desc(&tm_out);
        if (p.residual) tma_prefetch_desc(&tm_res);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 2 * BN, PairTag());
        dependency_trigger();
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_threads();  // the partner's barriers are set up, its tensor memory is there
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    dependency_wait();

    LinRun run(p);
    bool ok = true;
    if (warp == 0) {
        if (elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            for (; run.left(p) && ok; run.next(p)) {
                const int m0 = run.m * 256 + rank * 128, n0 = run.n * BN + rank * (BN / 2);
                for (int ks = 0; ks < p.stages_k; ++ks) {
                    ok = mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, 160);
                    if (!ok) break;
                    uint8_t *sx = smem + stage * L::kSlot;
                    const uint32_t bar = cluster_address(smem_u32(&full_bar[stage]), 0);
                    if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * L::kSlot);
                    tma_load_2d_pair(sx, &tm_x, bar, ks * kLinStageK, m0);
                    tma_load_2d_pair(sx + L::kOperandX, &tm_w, bar, ks * kLinStageK, n0);
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            const bool leader = elect_one();
            int stage = 0;
            uint32_t phase = 0, buf = 0, t_phase = 0;
            bool ready = false;
            const uint32_t base_lo = desc_lo(smem_u32(smem));
            for (; run.left(p) && ok; run.next(p)) {
                ok = mbar_wait_warp(&tempty_bar[buf], t_phase ^ 1u, abort_flag, 161);
                if (!ok) break;
                tc_fence_after_sync();
                const uint32_t d = tmem + buf * BN;
                for (int ks = 0; ks < p.stages_k; ++ks) {
                    if (!ready) ok = mbar_wait_warp(&full_bar[stage], phase, abort_flag, 162);
                    if (!ok) break;
                    tc_fence_after_sync();
                    // The next stage is asked about here and the answer is looked at behind this stage's MMAs.
                    const bool wraps = stage + 1 == STAGES;
                    const bool next = mbar_test(&full_bar[wraps ? 0 : stage + 1], wraps ? phase ^ 1u : phase);
                    const uint32_t x_lo = base_lo + stage * (L::kSlot >> 4);
                    const int steps = ks == p.stages_k - 1 ? p.last_steps : 4;
                    if (leader) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (k < steps) tc_mma_f16<2>(d, x_lo + 2 * k, x_lo + (L::kOperandX >> 4) + 2 * k, make_idesc_16<T>(256, BN), (ks | k) != 0);
                        tc_commit_pair(&empty_bar[stage]);
                        if (ks == p.stages_k - 1) tc_commit_pair(&tfull_bar[buf]);
                    }
                    ready = __all_sync(0xffffffffu, next);
                    stage = wraps ? 0 : stage + 1;
                    phase ^= wraps;
                }
                buf ^= 1u;
                t_phase ^= buf ^ 1u;   // a buffer's phase advances when both have been used
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        const int q = warp & 3, part = (warp - 4) >> 2;
        uint8_t *staging = smem + L::kOffStaging + (warp - 4) * (32 * 128);
        const T *bias_at = static_cast<const T *>(p.bias);
        uint64_t *loaded = res_bar + (warp - 4);
        const uint32_t tempty = cluster_address(smem_u32(tempty_bar), 0);
        uint32_t buf = 0, t_phase = 0, res_phase = 0;
        for (; run.left(p) && ok; run.next(p)) {
            const int m0 = run.m * 256 + rank * 128 + q * 32, c0 = run.n * BN + part * 64;
            const bool live = m0 < p.M && c0 < p.N;
            if (live) {
                if (lane == 0) {
                    tma_store_wait_read<0>();   // the staging is free
                    if (p.residual) {
                        mbar_arrive_expect_tx(loaded, 32 * 128);
                        tma_load_2d(staging, &tm_res, loaded, c0, m0);
                    }
                }
                __syncwarp();
            }
            ok = mbar_wait_warp(&tfull_bar[buf], t_phase, abort_flag, 163);
            if (!ok) break;
            tc_fence_after_sync();
            const uint32_t t_row = tmem + (uint32_t(q * 32) << 16) + buf * BN + part * 64;
            if (live && p.residual) {
                ok = mbar_wait_warp(loaded, res_phase, abort_flag, 164);
                if (!ok) break;
                res_phase ^= 1u;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t a[32];
                tmem_ld_32x32(t_row + h * 32, a);
                // everything is read before anything is written: to the compiler these may be the same places
                uint4 bias[4], res[4];
                if (p.bias)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int c = c0 + 32 * h + 8 * j;
                        bias[j] = c < p.N ? *reinterpret_cast<const uint4 *>(bias_at + c) : make_uint4(0, 0, 0, 0);
                    }
                if (p.residual)
#pragma unroll
                    for (int j = 0; j < 4; ++j) res[j] = *reinterpret_cast<const uint4 *>(staging + sw128_offset(lane, 4 * h + j));
                tmem_ld_wait();
                if (h == 1) {
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(tempty + buf * 8);
                }
                if (!live) continue;
                uint4 out[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float v[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(a[8 * j + i]);
                    out[j] = finish8<T, ACT>(v, p.bias ? &bias[j] : nullptr, p.residual ? &res[j] : nullptr, p.alpha);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4 *>(staging + sw128_offset(lane, 4 * h + j)) = out[j];
            }
            if (live) {
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    if (p.passes_by) tma_store_2d(&tm_out, staging, c0, m0, l2_evict_first());
                    else tma_store_2d(&tm_out, staging, c0, m0);
                    tma_store_commit();
                }
            }
            buf ^= 1u;
            t_phase ^= buf ^ 1u;
        }
        if (lane == 0) tma_store_wait_all<0>();
        __syncwarp();
    }
    if (!ok) {
        // loads in flight get a bounded chance to land before the shared memory is released
        const long long t0 = clock64();
        while (clock64() - t0 < (1ll << 22)) { }
    }

    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_threads();  // nothing of the partner still arrives here or reads this CTA's operands
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 2 * BN, PairTag());
    }
}

inline LinEpilogue lin_epilogue(const fluke_sm100_linear_t *g) {
    return {g->bias, g->residual, g->out, g->ld_residual, g->ld_out, g->alpha};
}
inline int lin_operand(CUtensorMap *m, const void *base, int rows, int cols, int64_t ld, int box_rows) {
    return make_tmap_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, base, rows, cols, uint64_t(ld) * 2, box_rows, kLinStageK, true);
}

template <typename T, int ACT>
int linear_split_launch(const fluke_sm100_linear_t *g, cudaStream_t stream) {
    constexpr auto kernel = linear_split_kernel<T, ACT>;
    LinSplitDev p;
    p.M = g->M; p.N = g->N;
    p.n_tiles = (g->N + 127) / 128;
    p.stages_k = (g->K + kLinStageK - 1) / kLinStageK;
    p.last_steps = (g->K - (p.stages_k - 1) * kLinStageK + 15) / 16;
    p.e = lin_epilogue(g);
    // Rows of x per tile, and CTAs per tile while all of them run at once and each has a stage of K at least: those with the shortest time by what a stage takes
    // (0.2 us), the epilogue (18 ns per row), and a hand-over of the tile's rows (0.6 us, and 18 ns per row). Us per call, tiles of 16 : 32 : 64 : 128 rows:
    // [333, 512] x [1536, 512] 5.5 : 5.0 : 6.1 : 8.1, [64, 4096] x [4096, 4096] 17.6 : 11.9 : 10.9 : 11.7, [512, 2048] x [512, 2048] 9.7 : 7.5 : 7.3 : 10.2.
    const int sms = device_sm_count();
    int rows = 0, each = p.stages_k;
    float best = 0.f;
    for (int r = 16; r <= 128; r *= 2) {
        const int64_t tiles = (int64_t(g->M) + r - 1) / r * p.n_tiles;
        const int filled = g->M < r ? g->M : r;
        for (int c = 1; c <= 8 && c <= p.stages_k && (c == 1 || tiles * c <= sms); ++c) {
            const int n = (p.stages_k + c - 1) / c;
            const float us = (n * 0.2f + 0.018f * filled) * float((tiles + sms - 1) / sms) + (c > 1 ? 0.6f + 0.018f * filled : 0.f);
            if (rows && us >= best) continue;
            if (c > 1 && tiles > cluster_capacity<kernel>(c, kLinThreads, kLinSplitMaxSmem + 1024)) continue;
            best = us;
            each = n;
            rows = r;
        }
        if (r >= g->M) break;
    }
    const int64_t tiles = (int64_t(g->M) + rows - 1) / rows * p.n_tiles;
    if (tiles > (INT32_MAX >> 3) - 1024) return (int)cudaErrorInvalidValue;
    const int most = g->M < rows ? g->M : rows;
    p.rows = rows;
    const int split = p.split = (p.stages_k + each - 1) / each;
    const int stage_bytes = rows * 128 + 128 * 128;
    // a longer run of K than the ring holds streams through a deeper one, where an SM has no second CTA to run
    p.stages = (each * stage_bytes > kLinSplitSmem && tiles * split <= sms ? kLinSplitDeep : kLinSplitSmem) / stage_bytes;
    if (p.stages > kLinSplitStages) p.stages = kLinSplitStages;
    if (p.stages > each) p.stages = each;
    // the sums, and with a split what is received (of one share from every rank) in front of them
    const int sums = rows * kLinSumPitch * 4;
    p.sums_at = split > 1 ? (split * ((most + split - 1) / split) * kLinSumPitch * 4 + 1023) / 1024 * 1024 : 0;
    int smem = p.stages * stage_bytes;
    if (smem < p.sums_at + sums) smem = p.sums_at + sums;
    if (smem < kLinSplitMinSmem) smem = kLinSplitMinSmem;
    if (smem > kLinSplitMaxSmem) return (int)cudaErrorInvalidValue;   // 128 rows, split: 135 KB at most (6 or 7 CTAs per tile)
    CUtensorMap tm_x, tm_w;
    int rc = lin_operand(&tm_x, g->x, g->M, g->K, g->ld_x, rows);
    if (!rc) rc = lin_operand(&tm_w, g->w, g->N, g->K, g->K, 128);
    if (!rc) rc = configure_smem<kernel>(kLinSplitMaxSmem + 1024);
    if (rc) return rc;
    return launch_dependent_clusters(kernel, split, dim3(int(tiles) * split), kLinThreads, smem + 1024, stream, tm_x, tm_w, p);
}

template <typename T, int ACT, int BN>
int linear_pair_launch(const fluke_sm100_linear_t *g, cudaStream_t stream) {
    using L = LinPairLayout<BN>;
    constexpr auto kernel = linear_pair_kernel<T, ACT, BN>;
    const int capacity = cluster_capacity<kernel>(2, L::kThreads, L::kDynamic);
    if (capacity < 1) return (int)cudaErrorNotSupported;
    LinPairDev p;
    p.M = g->M; p.N = g->N;
    p.m_tiles = (g->M + 255) / 256;
    p.n_tiles = (g->N + BN - 1) / BN;
    const int64_t tiles = int64_t(p.m_tiles) * p.n_tiles;
    if (tiles > INT32_MAX - 1024 || int64_t(kLinBand) * p.n_tiles > INT32_MAX) return (int)cudaErrorInvalidValue;
    p.tiles = int(tiles);
    p.stages_k = (g->K + kLinStageK - 1) / kLinStageK;
    p.last_steps = (g->K - (p.stages_k - 1) * kLinStageK + 15) / 16;
    p.passes_by = int64_t(g->M) * g->N * 2 > int64_t(device_l2_bytes()) / 8 * 7;
    p.bias = g->bias;
    p.residual = g->residual != nullptr;
    p.alpha = g->alpha;
    CUtensorMap tm_x, tm_w, tm_res, tm_out;
    int rc = lin_operand(&tm_x, g->x, g->M, g->K, g->ld_x, 128);
    if (!rc) rc = lin_operand(&tm_w, g->w, g->N, g->K, g->K, BN / 2);
    if (!rc) rc = lin_operand(&tm_out, g->out, g->M, g->N, g->ld_out, 32);
    tm_res = tm_out;
    if (!rc && g->residual) rc = lin_operand(&tm_res, g->residual, g->M, g->N, g->ld_residual, 32);
    if (rc) return rc;
    const int pairs = p.tiles < capacity ? p.tiles : capacity;
    return launch_dependent_clusters(kernel, 2, pairs * 2, L::kThreads, L::kDynamic, stream, tm_x, tm_w, tm_res, tm_out, p);
}

template <typename T, int ACT>
int linear_dispatch(const fluke_sm100_linear_t *g, cudaStream_t stream) {
    // Us per call, split : pairs, 128 columns : pairs, 256 columns: [1000, 512] x [512, 512] 4.6 : 6.0 : 7.6, [700, 512] x [2048, 512] 6.7 : 6.1 : 7.7, [1500, 1024] x [1024, 1024] 9.1 : 7.8 : 9.9,
    // [3000, 512] x [2048, 512] 14.7 : 9.9 : 10.7, [9331, 512] x [1536, 512] 27.8 : 19.9 : 17.6. A tile of half the columns takes 0.6 of the time.
    const int64_t m_tiles = (int64_t(g->M) + 255) / 256, pairs = device_sm_count() / 2;
    if (g->M <= 64 || (int64_t(g->M) + 63) / 64 * ((g->N + 127) / 128) <= device_sm_count()) return linear_split_launch<T, ACT>(g, stream);
    const int64_t wide = (m_tiles * ((g->N + 255) / 256) + pairs - 1) / pairs, narrow = (m_tiles * ((g->N + 127) / 128) + pairs - 1) / pairs;
    if (5 * wide > 3 * narrow) return linear_pair_launch<T, ACT, 128>(g, stream);
    return linear_pair_launch<T, ACT, 256>(g, stream);
}
template <typename T>
int linear_dispatch(const fluke_sm100_linear_t *g, cudaStream_t stream) {
    switch (g->activation) {
        case kActNone: return linear_dispatch<T, kActNone>(g, stream);
        case kActRelu: return linear_dispatch<T, kActRelu>(g, stream);
        case kActSilu: return linear_dispatch<T, kActSilu>(g, stream);
        case kActGelu: return linear_dispatch<T, kActGelu>(g, stream);
        case kActTanh: return linear_dispatch<T, kActTanh>(g, stream);
        default: return linear_dispatch<T, kActSigmoid>(g, stream);
    }
}

// Rows of `cols` 16-bit values, `ld` apart.
struct LinRegion {
    const void *at;
    int64_t rows, cols, ld;
    uint64_t bytes() const { return at && rows > 0 ? (uint64_t(rows - 1) * ld + cols) * 2 : 0; }
};
// Whether two regions share no byte. Interleaved ones are told apart where their rows have the same distance (columns of one wider tensor).
inline bool regions_apart(const LinRegion &a, const LinRegion &b) {
    const uint64_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
    if (!a.bytes() || !b.bytes() || x + a.bytes() <= y || y + b.bytes() <= x) return true;
    if (a.ld != b.ld) return false;
    const uint64_t pitch = uint64_t(a.ld) * 2, wa = uint64_t(a.cols) * 2, wb = uint64_t(b.cols) * 2;
    const uint64_t ahead = (y + pitch - x % pitch) % pitch;   // where b's columns begin behind a's
    return ahead >= wa && ahead + wb <= pitch;
}

}  // namespace
}  // namespace fluke_sm100

extern "C" int fluke_sm100_linear(const fluke_sm100_linear_t *g, void *stream) {
    using namespace fluke_sm100;
    // sizes within 2^20 of the largest int: the next tile's end still fits 32 bits
    constexpr int kMost = INT32_MAX - (1 << 20);
    if (!g || g->M < 0 || g->M > kMost || g->N <= 0 || g->N > kMost || g->N % 8 != 0 || g->K <= 0 || g->K > kMost || g->K % 8 != 0) return (int)cudaErrorInvalidValue;
    if (g->activation < kActNone || g->activation > kActSigmoid) return (int)cudaErrorInvalidValue;
    if (g->M == 0) return 0;
    if (!g->x || !g->w || !g->out) return (int)cudaErrorInvalidValue;
    auto pitch_ok = [](int64_t ld, int cols) { return ld >= cols && ld % 8 == 0 && ld < (int64_t(1) << 38); };
    if (!pitch_ok(g->ld_x, g->K) || !pitch_ok(g->ld_out, g->N) || (g->residual && !pitch_ok(g->ld_residual, g->N))) return (int)cudaErrorInvalidValue;
    if (!aligned16(g->x) || !aligned16(g->w) || !aligned16(g->bias) || !aligned16(g->residual) || !aligned16(g->out)) return (int)cudaErrorMisalignedAddress;
    // A tile is written while others are still computed: the output lies apart from everything but a residual in the same place.
    const LinRegion out = {g->out, g->M, g->N, g->ld_out};
    const bool in_place = g->residual == g->out && g->ld_residual == g->ld_out;
    if (!regions_apart(out, {g->x, g->M, g->K, g->ld_x}) || !regions_apart(out, {g->w, g->N, g->K, g->K}) || !regions_apart(out, {g->bias, 1, g->N, g->N}) ||
        (!in_place && !regions_apart(out, {g->residual, g->M, g->N, g->ld_residual})))
        return (int)cudaErrorInvalidValue;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return g->bf16 ? linear_dispatch<__nv_bfloat16>(g, s) : linear_dispatch<__half>(g, s);
}

// linear_sm100.cu -- products of 16-bit matrices with an epilogue on sm_100a:
//     out[m, n] = round16( act( sum_k x[m, k] w[n, k] + bias[n] ) + alpha residual[m, n] )
// with x [M, K], w [N, K], residual and out [M, N] in f16 or bf16, sums and everything behind them in f32.
//
// TMA brings 128-byte-swizzled blocks of 64 values of K per row, tcgen05.mma (kind f16, 16 values of K per instruction) sums them
// up in tensor memory, and the epilogue takes the sums through registers, where bias, activation and residual cost no pass over memory.

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
__device__ __forceinline__ float activate(float v) {
    if constexpr (ACT == kActRelu) return v < 0.f ? 0.f : v;
    if constexpr (ACT == kActSilu || ACT == kActSigmoid) {
        const float s = rcp_approx(1.f + ex2_approx(-1.44269504f * v));
        return ACT == kActSilu ? v * s : s;
    }
    if constexpr (ACT == kActTanh) {
        const float t = ex2_approx(-2.88539008f * fabsf(v));
        const float big = copysignf((1.f - t) * rcp_approx(1.f + t), v);
        return fabsf(v) < 0.015625f ? fmaf(v * v * v, -0.333333333f, v) : big;
    }
    if constexpr (ACT == kActGelu) {
        const float a = fabsf(v), t = rcp_approx(fmaf(0.31f, a, 1.f));
        float p = -0.0739276186f;
        p = fmaf(p, t, 0.180445790f);
        p = fmaf(p, t, 0.0157500077f);
        p = fmaf(p, t, 0.133426800f);
        p = fmaf(p, t, 0.120442092f);
        p = fmaf(p, t, 0.123860620f);
        const float h = p * t * ex2_approx(-0.721347520f * (a * a));
        return v * (v < 0.f ? h : 1.f - h);
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
        v = make_float2(activate<ACT>(v.x), activate<ACT>(v.y));
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
// A CTA takes less than half of an SM's shared memory, so that the next kernel's CTAs are set up beside it, and 128 of its 512
// tensor-memory columns.
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

inline LinEpilogue lin_epilogue(const fluke_sm100_linear_t *g) {
    return {g->bias, g->residual, g->out, g->ld_residual, g->ld_out, g->alpha};
}
inline int lin_operand(CUtensorMap *m, const void *base, int rows, int cols, int64_t ld, int box_rows) {
    return make_tmap_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, base, rows, cols, uint64_t(ld) * 2, box_rows, kLinStageK, true);
}

// Rows of x per tile of the split form: 64 while those tiles are all resident at once, else 128; what there is of them, if less.
inline int lin_split_rows(const fluke_sm100_linear_t *g) {
    if (g->M <= 32) return g->M <= 16 ? 16 : 32;
    return int64_t((g->M + 63) / 64) * ((g->N + 127) / 128) <= device_sm_count() ? 64 : 128;
}
inline int64_t lin_split_tiles(const fluke_sm100_linear_t *g) {
    const int rows = lin_split_rows(g);
    return int64_t((g->M + rows - 1) / rows) * ((g->N + 127) / 128);
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
    const int rows = p.rows = lin_split_rows(g), sms = device_sm_count();
    const int64_t tiles = lin_split_tiles(g);
    if (tiles > (INT32_MAX >> 3) - 1024) return (int)cudaErrorInvalidValue;
    // CTAs per tile, while all of them run at once and each has a stage of K at least: the number with the shortest time by what a stage takes
    // (0.2 us) and what a hand-over of the tile's rows does (0.6 us, and 18 ns per row).
    const int most = g->M < rows ? g->M : rows;
    int each = p.stages_k;
    float best = 0.f;
    for (int c = 1; c <= 8 && c <= p.stages_k && (c == 1 || tiles * c <= sms); ++c) {
        const int n = (p.stages_k + c - 1) / c;
        const float us = n * 0.2f + (c > 1 ? 0.6f + 0.018f * most : 0.f);
        if (c > 1 && (us >= best || tiles > cluster_capacity<kernel>(c, kLinThreads, kLinSplitMaxSmem + 1024))) continue;
        best = us;
        each = n;
    }
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
    if (smem > kLinSplitMaxSmem) return (int)cudaErrorInvalidValue;   // 128 rows, split: 133 KB
    CUtensorMap tm_x, tm_w;
    int rc = lin_operand(&tm_x, g->x, g->M, g->K, g->ld_x, rows);
    if (!rc) rc = lin_operand(&tm_w, g->w, g->N, g->K, g->K, 128);
    if (!rc) rc = configure_smem<kernel>(kLinSplitMaxSmem + 1024);
    if (rc) return rc;
    return launch_dependent_clusters(kernel, split, dim3(int(tiles) * split), kLinThreads, smem + 1024, stream, tm_x, tm_w, p);
}

template <typename T, int ACT>
int linear_dispatch(const fluke_sm100_linear_t *g, cudaStream_t stream) {
    return linear_split_launch<T, ACT>(g, stream);
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

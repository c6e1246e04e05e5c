// recurrence_sm100.cu -- gated linear recurrence over time and its gradients on sm_100a:
//     h_t = f_t h_{t-1} + (1 - f_t) v_t,    f_t = sigmoid(g_t),    per chunk and channel.
// Gates do not depend on the state, so any run of steps acts on the state in front of it as one step does:
//     h_out = h_in + (V - C h_in)
// with C = 1 - prod f and V the state that the run leaves of zero. Runs are computed side by side and joined. One minus the
// product is carried, not the product: a step is h += c (v - h) with c = 1 - f = 1 / (1 + exp(g)), and a run of gates
// near one (a channel that remembers for thousands of steps) keeps the digits of its small c, where f rounded to f32 would
// be off by 2^-25 per step.
//
// Backwards, with e_t the gradient of h_t and x_t what reaches step t from the steps behind it:
//     e_t = dy_t + x_t,    x_{t-1} = e_t - c_t e_t,    dv_t = c_t e_t,    dg_t = e_t (h_{t-1} - v_t) f_t c_t
// a run of steps acts on x as x_out = x_in + (D - C x_in), C as above. The states h_{t-1} are computed again, from those that the forward
// pass keeps of every 64th step (4 bytes per 64 values): that reads 6 and writes 4 bytes per value, where states kept in full would be read as well, and rounded.
//
// Both are bound by memory: a lane holds two channels of eight steps in registers, a warp reads rows of 64 channels (128 bytes)
// or two runs of 32, all of a tile's loads are asked for a tile ahead, and what joins the runs goes through shared memory. Where chunks
// and channels fill too few SMs, the tiles of a chunk are spread over a cluster, whose CTAs tell each other what their runs do.

namespace fluke_sm100 {
namespace {

constexpr int kRecSteps = 8;          // of a lane
constexpr int kRecKept = FLUKE_SM100_RECURRENCE_KEPT;   // steps between kept states
constexpr int kRecMostCluster = 8;

struct RecIn {
    const void *at;
    int64_t step, chunk;              // values between steps and between chunks
};
struct RecOut {
    void *at;
    int64_t step, chunk;
};
struct RecDev {
    int T, B, H;
    int reverse, split, rounds;       // CTAs of a cluster; tiles of each
    int slabs;                        // runs of channels per chunk
    const int *lengths;
    RecIn gate, value, grad;          // grad: backwards
    RecOut out, grad_gate, grad_value;
    const float *h0, *grad_last;      // or null: zeros
    float *h_last, *grad_h0;          // or null
    float *states;                    // written forwards (or null), read backwards
};

__device__ __forceinline__ uint32_t ld_pair(const void *p, int64_t at) {
    uint32_t v;
    asm volatile("ld.global.L1::no_allocate.b32 %0, [%1];" : "=r"(v) : "l"(static_cast<const uint16_t *>(p) + at) : "memory");
    return v;
}
__device__ __forceinline__ void st_pair(void *p, int64_t at, uint32_t v) {
    *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(p) + at) = v;
}
// 1 / (1 + exp(g)): relative error below 2^-21 and, of the argument's rounding, |g| 2^-24; zero above 87, where it is below 2^-125.
__device__ __forceinline__ float2 one_minus_gate(float2 g) {
    const float2 a = mul2(g, make_float2(1.44269504f, 1.44269504f));
    const float2 d = add2(make_float2(ex2_approx(a.x), ex2_approx(a.y)), make_float2(1.f, 1.f));
    return make_float2(rcp_approx(d.x), rcp_approx(d.y));
}
// a + c (b - a)
__device__ __forceinline__ float2 towards(float2 a, float2 c, float2 b) { return fma2(c, fma2(a, make_float2(-1.f, -1.f), b), a); }
// a - c a
__device__ __forceinline__ float2 less(float2 a, float2 c) { return fma2(make_float2(-c.x, -c.y), a, a); }
// a + (b - c a): what a run (c, b) makes of a
__device__ __forceinline__ float2 through(float2 a, float2 c, float2 b) { return add2(a, fma2(make_float2(-c.x, -c.y), a, b)); }

// Where a thread works: its chunk, its two channels and which run of a tile it holds.
template <int LANES>
struct RecPlace {
    int b, rank, channel, lane, run, runs;
    bool in;                          // the channels exist
    __device__ __forceinline__ explicit RecPlace(const RecDev &p) {
        constexpr int kPerWarp = 32 / LANES;
        const int slab = int(blockIdx.x) / p.split;
        rank = int(blockIdx.x) - slab * p.split;
        b = slab / p.slabs;
        lane = threadIdx.x & (LANES - 1);
        channel = (slab - b * p.slabs) * (2 * LANES) + 2 * lane;
        run = int(threadIdx.x) / LANES;
        runs = int(blockDim.x) / LANES;
        (void)kPerWarp;
        in = channel < p.H;
    }
};
__device__ __forceinline__ int rec_length(const RecDev &p, int b) {
    return p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
}
__device__ __forceinline__ float2 ld_state(const float *s, int64_t at, bool in) {
    return s && in ? *reinterpret_cast<const float2 *>(s + at) : make_float2(0.f, 0.f);
}

// Forwards. LANES: lanes that share a run, with two channels each.
template <typename T, int LANES>
__global__ void __launch_bounds__(512)
recurrence_kernel(const RecDev p) {
    __shared__ float4 run_of[2][512 / LANES][LANES];            // C and V of every run of the tile
    __shared__ float4 tile_of[2][kRecMostCluster][LANES];       // of every CTA's tile
    const RecPlace<LANES> w(p);
    dependency_wait();
    const int length = rec_length(p, w.b), tile = w.runs * kRecSteps;
    const int64_t state_at = int64_t(w.b) * p.H + w.channel;
    float2 carry = ld_state(p.h0, state_at, w.in);
    // A step's place: processing goes through s = 0, 1, ..., time through s or T - 1 - s.
    auto time_of = [&](int s) { return p.reverse ? p.T - 1 - s : s; };
    const int64_t gate0 = w.b * p.gate.chunk + w.channel, value0 = w.b * p.value.chunk + w.channel, out0 = w.b * p.out.chunk + w.channel;
    uint32_t g[kRecSteps], v[kRecSteps];
    auto load = [&](int s0) {
#pragma unroll
        for (int k = 0; k < kRecSteps; ++k) {
            const int t = time_of(s0 + k);
            const bool ask = w.in && s0 + k < p.T;
            g[k] = ask ? ld_pair(p.gate.at, gate0 + t * p.gate.step) : 0;
            v[k] = ask ? ld_pair(p.value.at, value0 + t * p.value.step) : 0;
        }
    };
    int s0 = w.rank * tile + w.run * kRecSteps;
    load(s0);
    for (int round = 0; round < p.rounds; ++round, s0 += p.split * tile) {
        const int par = round & 1;
        float2 c[kRecSteps], x[kRecSteps], C = make_float2(0.f, 0.f), V = C;
#pragma unroll
        for (int k = 0; k < kRecSteps; ++k) {
            // behind a chunk's end nothing changes, whatever stands there
            const bool live = s0 + k < p.T && time_of(s0 + k) < length;
            c[k] = one_minus_gate(unpack2(g[k], T()));
            x[k] = unpack2(v[k], T());
            if (!live) c[k] = x[k] = make_float2(0.f, 0.f);
            V = towards(V, c[k], x[k]);
            C = towards(C, c[k], make_float2(1.f, 1.f));
        }
        load(s0 + p.split * tile);
        run_of[par][w.run][w.lane] = make_float4(C.x, C.y, V.x, V.y);
        __syncthreads();
        float2 h;
        if (p.split == 1) {
            h = carry;
            for (int r = 0; r < w.runs; ++r) {
                if (r == w.run) h = carry;
                const float4 q = run_of[par][r][w.lane];
                carry = through(carry, make_float2(q.x, q.y), make_float2(q.z, q.w));
            }
        } else {
            float2 before_c = make_float2(0.f, 0.f), before_v = before_c;
            C = V = before_c;
            for (int r = 0; r < w.runs; ++r) {
                if (r == w.run) {
                    before_c = C;
                    before_v = V;
                }
                const float4 q = run_of[par][r][w.lane];
                V = through(V, make_float2(q.x, q.y), make_float2(q.z, q.w));
                C = towards(C, make_float2(q.x, q.y), make_float2(1.f, 1.f));
            }
            // every CTA is told by as many threads as it has lanes of a run
            if (w.run < p.split) {
                const uint32_t to = cluster_address(smem_u32(&tile_of[par][w.rank][w.lane]), w.run);
                asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(C.x), "f"(C.y), "f"(V.x), "f"(V.y) : "memory");
            }
            cluster_sync_threads();
            h = carry;
            for (int r = 0; r < p.split; ++r) {
                if (r == w.rank) h = carry;
                const float4 q = tile_of[par][r][w.lane];
                carry = through(carry, make_float2(q.x, q.y), make_float2(q.z, q.w));
            }
            h = through(h, before_c, before_v);
        }
        if (w.in && s0 < p.T && p.states && s0 % kRecKept == 0)
            *reinterpret_cast<float2 *>(p.states + int64_t(s0 / kRecKept) * p.B * p.H + state_at) = h;
#pragma unroll
        for (int k = 0; k < kRecSteps; ++k) {
            h = towards(h, c[k], x[k]);
            const int t = time_of(s0 + k);
            if (w.in && s0 + k < p.T) st_pair(p.out.at, out0 + t * p.out.step, t < length ? pack2(h, T()) : 0);
        }
    }
    // every thread of the cluster has read h0, which may be the same, in front of the last barrier
    if (w.rank == 0 && w.run == 0 && w.in && p.h_last) *reinterpret_cast<float2 *>(p.h_last + state_at) = carry;
}

// Backwards: tiles, and the runs of a tile, are joined from the last to the first.
template <typename T, int LANES>
__global__ void __launch_bounds__(512)
recurrence_backward_kernel(const RecDev p) {
    __shared__ float4 run_of[2][512 / LANES][LANES];            // C and V of every run of the tile
    __shared__ float2 run_back[2][512 / LANES][LANES];          // D
    __shared__ float4 tile_of[2][kRecMostCluster][LANES];       // C and D of every CTA's tile
    const RecPlace<LANES> w(p);
    dependency_wait();
    const int length = rec_length(p, w.b), tile = w.runs * kRecSteps;
    const int64_t state_at = int64_t(w.b) * p.H + w.channel;
    float2 carry = ld_state(p.grad_last, state_at, w.in);
    auto time_of = [&](int s) { return p.reverse ? p.T - 1 - s : s; };
    const int64_t gate0 = w.b * p.gate.chunk + w.channel, value0 = w.b * p.value.chunk + w.channel, grad0 = w.b * p.grad.chunk + w.channel;
    const int64_t dg0 = w.b * p.grad_gate.chunk + w.channel, dv0 = w.b * p.grad_value.chunk + w.channel;
    uint32_t g[kRecSteps], v[kRecSteps], dy[kRecSteps];
    float2 kept;                                                // the state in front of the tile
    auto load = [&](int s0) {
#pragma unroll
        for (int k = 0; k < kRecSteps; ++k) {
            const int t = time_of(s0 + k);
            const bool ask = w.in && s0 >= 0 && s0 + k < p.T;
            g[k] = ask ? ld_pair(p.gate.at, gate0 + t * p.gate.step) : 0;
            v[k] = ask ? ld_pair(p.value.at, value0 + t * p.value.step) : 0;
            dy[k] = ask ? ld_pair(p.grad.at, grad0 + t * p.grad.step) : 0;
        }
        const int first = s0 - w.run * kRecSteps;
        kept = ld_state(p.states, int64_t(first / kRecKept) * p.B * p.H + state_at, w.in && first >= 0 && first < p.T);
    };
    int s0 = ((p.rounds - 1) * p.split + w.rank) * tile + w.run * kRecSteps;
    load(s0);
    for (int round = p.rounds - 1; round >= 0; --round, s0 -= p.split * tile) {
        const int par = round & 1;
        float2 c[kRecSteps], C = make_float2(0.f, 0.f), V = C, D = C, h = kept;
        uint32_t gate[kRecSteps], value[kRecSteps], grad[kRecSteps];
#pragma unroll
        for (int k = 0; k < kRecSteps; ++k) {
            const bool live = s0 + k < p.T && time_of(s0 + k) < length;
            gate[k] = g[k];
            value[k] = live ? v[k] : 0;
            grad[k] = live ? dy[k] : 0;
            c[k] = one_minus_gate(unpack2(g[k], T()));
            if (!live) c[k] = make_float2(0.f, 0.f);
            V = towards(V, c[k], unpack2(value[k], T()));
            C = towards(C, c[k], make_float2(1.f, 1.f));
        }
#pragma unroll
        for (int k = kRecSteps - 1; k >= 0; --k) D = less(add2(D, unpack2(grad[k], T())), c[k]);
        load(s0 - p.split * tile);
        run_of[par][w.run][w.lane] = make_float4(C.x, C.y, V.x, V.y);
        run_back[par][w.run][w.lane] = D;
        __syncthreads();
        for (int r = 0; r < w.run; ++r) {
            const float4 q = run_of[par][r][w.lane];
            h = through(h, make_float2(q.x, q.y), make_float2(q.z, q.w));
        }
        float2 x;
        if (p.split == 1) {
            x = carry;
            for (int r = w.runs - 1; r >= 0; --r) {
                if (r == w.run) x = carry;
                const float2 q = *reinterpret_cast<const float2 *>(&run_of[par][r][w.lane]);
                carry = through(carry, q, run_back[par][r][w.lane]);
            }
        } else {
            float2 behind_c = make_float2(0.f, 0.f), behind_d = behind_c;
            C = D = behind_c;
            for (int r = w.runs - 1; r >= 0; --r) {
                if (r == w.run) {
                    behind_c = C;
                    behind_d = D;
                }
                const float2 q = *reinterpret_cast<const float2 *>(&run_of[par][r][w.lane]);
                D = through(D, q, run_back[par][r][w.lane]);
                C = towards(C, q, make_float2(1.f, 1.f));
            }
            if (w.run < p.split) {
                const uint32_t to = cluster_address(smem_u32(&tile_of[par][w.rank][w.lane]), w.run);
                asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(C.x), "f"(C.y), "f"(D.x), "f"(D.y) : "memory");
            }
            cluster_sync_threads();
            x = carry;
            for (int r = p.split - 1; r >= 0; --r) {
                if (r == w.rank) x = carry;
                const float4 q = tile_of[par][r][w.lane];
                carry = through(carry, make_float2(q.x, q.y), make_float2(q.z, q.w));
            }
            x = through(x, behind_c, behind_d);
        }
        float2 before[kRecSteps];                               // h - v in front of each step
#pragma unroll
        for (int k = 0; k < kRecSteps; ++k) {
            const float2 u = unpack2(value[k], T());
            before[k] = fma2(u, make_float2(-1.f, -1.f), h);
            h = towards(h, c[k], u);
        }
#pragma unroll
        for (int k = kRecSteps - 1; k >= 0; --k) {
            const float2 e = add2(x, unpack2(grad[k], T())), ce = mul2(c[k], e);
            // f by itself: one minus c has no digits left where c is near one
            const float2 raw = unpack2(gate[k], T()), f = one_minus_gate(make_float2(-raw.x, -raw.y));
            x = less(e, c[k]);
            const bool live = s0 + k < p.T && time_of(s0 + k) < length;
            const float2 dg = mul2(mul2(ce, before[k]), f);
            const int t = time_of(s0 + k);
            if (w.in && s0 + k < p.T) {
                st_pair(p.grad_gate.at, dg0 + t * p.grad_gate.step, live ? pack2(dg, T()) : 0);
                st_pair(p.grad_value.at, dv0 + t * p.grad_value.step, live ? pack2(ce, T()) : 0);
            }
        }
    }
    if (w.rank == 0 && w.run == 0 && w.in && p.grad_h0) *reinterpret_cast<float2 *>(p.grad_h0 + state_at) = carry;
}

// How a call is spread: lanes per run, threads per CTA, CTAs per cluster.
struct RecPlan {
    int lanes, threads, split, blocks;
};
// Returns false for more CTAs than a grid has.
inline bool rec_plan(RecDev *p, RecPlan *plan) {
    plan->lanes = p->H <= 32 ? 16 : 32;
    const int per_warp = 32 / plan->lanes;
    // no more warps than the steps fill
    int warps = 8;
    while (warps > 1 && (warps / 2) * per_warp * kRecSteps >= p->T) warps /= 2;
    plan->threads = warps * 32;
    plan->split = 1;
    const int tile = warps * per_warp * kRecSteps;
    p->slabs = (p->H + 2 * plan->lanes - 1) / (2 * plan->lanes);
    p->split = plan->split;
    const int64_t tiles = (int64_t(p->T) + tile - 1) / tile, blocks = int64_t(p->B) * p->slabs * plan->split;
    p->rounds = int((tiles + plan->split - 1) / plan->split);
    plan->blocks = int(blocks);
    return blocks <= INT32_MAX;
}

template <typename T>
int recurrence_launch(RecDev p, bool backward, cudaStream_t stream) {
    RecPlan plan;
    if (!rec_plan(&p, &plan)) return (int)cudaErrorInvalidValue;
    auto kernel = plan.lanes == 16 ? (backward ? recurrence_backward_kernel<T, 16> : recurrence_kernel<T, 16>)
                                   : (backward ? recurrence_backward_kernel<T, 32> : recurrence_kernel<T, 32>);
    return launch_dependent_clusters(kernel, plan.split, dim3(plan.blocks), plan.threads, 0, stream, p);
}

// A tensor [T, B, H] by its strides: rows of H values that begin on 4 bytes.
inline bool rec_strides_ok(const void *at, int64_t step, int64_t chunk, const RecDev &p) {
    const int64_t most = int64_t(1) << 44;
    if (!at || (reinterpret_cast<uintptr_t>(at) & 3u)) return false;
    return (p.T <= 1 || (step >= p.H && step % 2 == 0 && step < most)) && (p.B <= 1 || (chunk >= p.H && chunk % 2 == 0 && chunk < most));
}
struct RecRange {
    uint64_t at, bytes;
    int64_t step, chunk;
    int T, B, H;
};
inline RecRange rec_range(const void *at, int64_t step, int64_t chunk, const RecDev &p) {
    const uint64_t last = uint64_t(p.T > 1 ? (p.T - 1) * step : 0) + uint64_t(p.B > 1 ? (p.B - 1) * chunk : 0);
    return {reinterpret_cast<uintptr_t>(at), at ? (last + p.H) * 2 : 0, step, chunk, p.T, p.B, p.H};
}
inline RecRange rec_flat(const void *at, uint64_t bytes) { return {reinterpret_cast<uintptr_t>(at), at ? bytes : 0, 0, 0, 0, 0, 0}; }
// Whether two tensors share no byte: one lies behind the other, or both are columns of the same wider rows.
inline bool rec_apart(const RecRange &a, const RecRange &b) {
    if (!a.bytes || !b.bytes || a.at + a.bytes <= b.at || b.at + b.bytes <= a.at) return true;
    if (!a.H || !b.H) return false;
    const int64_t sa = a.T > 1 ? a.step : a.chunk, sb = b.T > 1 ? b.step : b.chunk;
    const int64_t ca = a.B > 1 ? a.chunk : sa, cb = b.B > 1 ? b.chunk : sb;
    if (sa != sb || ca != cb || (a.T <= 1 && a.B <= 1)) return false;
    const int64_t row = sa < ca ? sa : ca, other = sa < ca ? ca : sa;
    if (other % row != 0) return false;
    const uint64_t pitch = uint64_t(row) * 2, width = uint64_t(a.H) * 2;
    const uint64_t ahead = (b.at % pitch + pitch - a.at % pitch) % pitch;
    return ahead >= width && ahead + width <= pitch;
}
// Whether no two rows of an output share a byte: time- or batch-major, in rows of any distance.
inline bool rec_rows_apart(const RecRange &r) {
    if (r.T <= 1 || r.B <= 1) return true;   // the strides are at least H
    return r.step < r.chunk ? r.chunk >= r.step * (r.T - 1) + r.H : r.step >= r.chunk * (r.B - 1) + r.H;
}

}  // namespace
}  // namespace fluke_sm100

extern "C" int fluke_sm100_recurrence(const fluke_sm100_recurrence_t *r, int backward, void *stream) {
    using namespace fluke_sm100;
    // sizes within 2^20 of the largest int: the next tile's end still fits 32 bits
    constexpr int kMost = INT32_MAX - (1 << 20);
    if (!r || r->T < 0 || r->T > kMost || r->B < 0 || r->H < 0 || r->H > kMost || r->H % 2 != 0) return (int)cudaErrorInvalidValue;
    if (r->B == 0 || r->H == 0) return 0;
    RecDev p = {};
    p.T = r->T; p.B = r->B; p.H = r->H; p.reverse = r->reverse != 0;
    p.lengths = r->lengths;
    p.gate = {r->gate, r->gate_step, r->gate_chunk};
    p.value = {r->value, r->value_step, r->value_chunk};
    p.out = {r->out, r->out_step, r->out_chunk};
    p.grad = {r->grad, r->grad_step, r->grad_chunk};
    p.grad_gate = {r->grad_gate, r->grad_gate_step, r->grad_gate_chunk};
    p.grad_value = {r->grad_value, r->grad_value_step, r->grad_value_chunk};
    p.h0 = r->h0; p.h_last = r->h_last; p.states = r->states; p.grad_last = r->grad_last; p.grad_h0 = r->grad_h0;
    auto aligned = [](const void *q, unsigned n) { return (reinterpret_cast<uintptr_t>(q) & (n - 1)) == 0; };
    if (!aligned(p.lengths, 4) || !aligned(p.h0, 8) || !aligned(p.h_last, 8) || !aligned(p.states, 8) || !aligned(p.grad_last, 8) || !aligned(p.grad_h0, 8))
        return (int)cudaErrorMisalignedAddress;
    if (p.T > 0) {
        if (!rec_strides_ok(p.gate.at, p.gate.step, p.gate.chunk, p) || !rec_strides_ok(p.value.at, p.value.step, p.value.chunk, p)) return (int)cudaErrorInvalidValue;
        if (backward && (!p.states || !rec_strides_ok(p.grad.at, p.grad.step, p.grad.chunk, p) || !rec_strides_ok(p.grad_gate.at, p.grad_gate.step, p.grad_gate.chunk, p) ||
                         !rec_strides_ok(p.grad_value.at, p.grad_value.step, p.grad_value.chunk, p)))
            return (int)cudaErrorInvalidValue;
        if (!backward && !rec_strides_ok(p.out.at, p.out.step, p.out.chunk, p)) return (int)cudaErrorInvalidValue;
    }
    // Tiles are written while others are still read, so outputs lie apart from inputs and from each other; the last state may replace the first.
    auto range = [&](const auto &t) { return rec_range(t.at, t.step, t.chunk, p); };
    const uint64_t state = uint64_t(p.B) * p.H * 4, kept = (uint64_t(p.T) + kRecKept - 1) / kRecKept * state;
    const RecRange none = rec_flat(nullptr, 0);
    const RecRange in[] = {range(p.gate), range(p.value), backward ? range(p.grad) : none, rec_flat(p.lengths, uint64_t(p.B) * 4),
                           backward ? rec_flat(p.states, kept) : none, backward ? none : rec_flat(p.h0, state), backward ? rec_flat(p.grad_last, state) : none};
    const RecRange out[] = {backward ? range(p.grad_gate) : range(p.out), backward ? range(p.grad_value) : none, backward ? none : rec_flat(p.states, kept),
                            backward ? rec_flat(p.grad_h0, state) : rec_flat(p.h_last, state)};
    for (int o = 0; o < 4; ++o) {
        for (int i = 0; i < 7; ++i) {
            const bool in_place = o == 3 && i >= 5 && out[o].at == in[i].at;
            if (p.T > 0 && !in_place && !rec_apart(out[o], in[i])) return (int)cudaErrorInvalidValue;
        }
        for (int other = 0; other < o; ++other)
            if (p.T > 0 && !rec_apart(out[o], out[other])) return (int)cudaErrorInvalidValue;
        if (p.T > 0 && out[o].H && !rec_rows_apart(out[o])) return (int)cudaErrorInvalidValue;
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return r->bf16 ? recurrence_launch<__nv_bfloat16>(p, backward != 0, s) : recurrence_launch<__half>(p, backward != 0, s);
}

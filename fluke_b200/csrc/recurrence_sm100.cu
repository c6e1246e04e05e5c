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
constexpr int kRecThreads = 256;       // at most; fewer for a few steps
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

__device__ __forceinline__ uint32_t ld_pair(const char *p) {
    uint32_t v;
    asm volatile("ld.global.L1::no_allocate.b32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
// -1 / (1 + exp(g)): relative error below 2^-21 and, of the argument's rounding, |g| 2^-24; zero above 87, where it is below 2^-125. Its sign
// saves the negations: packed operations have none.
__device__ __forceinline__ float2 gate_less_one(float2 g) {
    const float2 a = mul2(g, make_float2(1.44269504f, 1.44269504f)), one = make_float2(-1.f, -1.f);
    const float2 d = fma2(make_float2(ex2_approx(a.x), ex2_approx(a.y)), one, one);
    return make_float2(rcp_approx(d.x), rcp_approx(d.y));
}
// 1 / (1 + exp(-g)), alike.
__device__ __forceinline__ float2 gate_of(float2 g) {
    const float2 a = mul2(g, make_float2(-1.44269504f, -1.44269504f));
    const float2 d = add2(make_float2(ex2_approx(a.x), ex2_approx(a.y)), make_float2(1.f, 1.f));
    return make_float2(rcp_approx(d.x), rcp_approx(d.y));
}
// With m = -c: a + c (b - a), and a - c a.
__device__ __forceinline__ float2 towards(float2 a, float2 m, float2 b) { return fma2(m, fma2(b, make_float2(-1.f, -1.f), a), a); }
__device__ __forceinline__ float2 less(float2 a, float2 m) { return fma2(m, a, a); }
// C of a run and one more step; a run's C is kept as its negative as well.
__device__ __forceinline__ float2 longer(float2 M, float2 m) { return fma2(m, add2(M, make_float2(1.f, 1.f)), M); }
// a + (b - C a): what a run makes of a
__device__ __forceinline__ float2 through(float2 a, float2 M, float2 b) { return add2(a, fma2(M, a, b)); }
__device__ __forceinline__ float2 low(float4 q) { return make_float2(q.x, q.y); }
__device__ __forceinline__ float2 high(float4 q) { return make_float2(q.z, q.w); }
__device__ __forceinline__ float4 both(float2 a, float2 b) { return make_float4(a.x, a.y, b.x, b.y); }
// Stores into the shared memory of a CTA of the cluster.
__device__ __forceinline__ void tell(const float4 *to, int rank, float2 a, float2 b) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(cluster_address(smem_u32(to), rank)), "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y) : "memory");
}

// Where a thread works. Processing goes through steps s = 0 .. T-1, time through s or T - 1 - s; a tensor is walked from its first step in
// processing order. What lies in [from, to) is inside the chunk.
template <int LANES>
struct RecPlace {
    int b, rank, channel, lane, run, runs, from, to;
    bool in;                          // the channels exist (else the last two are read, and nothing is written)
    int64_t state;
    __device__ __forceinline__ explicit RecPlace(const RecDev &p) {
        const int slab = int(blockIdx.x) / p.split;
        rank = int(blockIdx.x) - slab * p.split;
        b = slab / p.slabs;
        lane = threadIdx.x & (LANES - 1);
        channel = (slab - b * p.slabs) * (2 * LANES) + 2 * lane;
        in = channel < p.H;
        channel = min(channel, p.H - 2);
        run = int(threadIdx.x) / LANES;
        runs = int(blockDim.x) / LANES;
        state = int64_t(b) * p.H + channel;
    }
    __device__ __forceinline__ void measure(const RecDev &p) {   // reads global memory
        const int length = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
        from = p.reverse ? p.T - length : 0;
        to = p.reverse ? p.T : length;
    }
};
// A tensor from step s on: bytes between steps, in processing order.
struct RecWalk {
    const char *at;
    int64_t step;
    template <int LANES, typename X>
    __device__ __forceinline__ RecWalk(const RecDev &p, const X &x, const RecPlace<LANES> &w, int s) {
        step = (p.reverse ? -x.step : x.step) * 2;
        at = static_cast<const char *>(x.at) + (w.b * x.chunk + w.channel + (p.reverse ? p.T - 1 : 0) * x.step) * 2 + s * step;
    }
    __device__ __forceinline__ const char *operator[](int k) const { return at + k * step; }
    __device__ __forceinline__ char *out(int k) const { return const_cast<char *>(at + k * step); }
};
__device__ __forceinline__ float2 ld_state(const float *s, int64_t at) {
    return s ? *reinterpret_cast<const float2 *>(s + at) : make_float2(0.f, 0.f);
}
__device__ __forceinline__ void st_state(float *s, int64_t at, float2 v) { *reinterpret_cast<float2 *>(s + at) = v; }

// Forwards. LANES: lanes that share a run, with two channels each.
template <typename T, int LANES, bool CLUSTER>
__global__ void __launch_bounds__(kRecThreads, 3)
recurrence_kernel(const RecDev p) {
    constexpr int kRuns = kRecThreads / LANES;
    __shared__ float4 run_of[2][kRuns][LANES];                             // -C and V of every run of the tile
    __shared__ float4 tile_of[2][CLUSTER ? kRecMostCluster : 1][LANES];    // of every CTA's tile
    __shared__ float2 carried[2][LANES];                                   // the state in front of the tile
    RecPlace<LANES> w(p);
    const bool last_run = w.run == w.runs - 1;
    int s0 = (w.rank * w.runs + w.run) * kRecSteps;
    const int stride = p.split * w.runs * kRecSteps;                       // steps of a round
    RecWalk gate(p, p.gate, w, s0), value(p, p.value, w, s0), out(p, p.out, w, s0);
    if (CLUSTER) cluster_arrive_relaxed();   // this CTA runs: awaited before others are told anything
    dependency_wait();
    w.measure(p);
    float2 h = ld_state(p.h0, w.state), carry = h;
    uint32_t g[kRecSteps], v[kRecSteps];
    auto load = [&](int s) {
        if (s + kRecSteps <= p.T) {
#pragma unroll
            for (int k = 0; k < kRecSteps; ++k) {
                g[k] = ld_pair(gate[k]);
                v[k] = ld_pair(value[k]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < kRecSteps; ++k) {
                g[k] = s + k < p.T ? ld_pair(gate[k]) : 0;
                v[k] = s + k < p.T ? ld_pair(value[k]) : 0;
            }
        }
        gate.at += stride * gate.step;
        value.at += stride * value.step;
    };
    load(s0);
    if (CLUSTER) cluster_wait();
    if (!CLUSTER && last_run) carried[0][w.lane] = h;
    for (int round = 0; round < p.rounds; ++round, s0 += stride) {
        const int par = round & 1;
        const bool all = s0 >= w.from && s0 + kRecSteps <= w.to;           // of the run's steps lie inside the chunk
        float2 m[kRecSteps], M = make_float2(0.f, 0.f), V = M;
        uint32_t values[kRecSteps];
#pragma unroll
        for (int k = 0; k < kRecSteps; ++k) {
            m[k] = gate_less_one(unpack2(g[k], T()));
            values[k] = v[k];
        }
        if (!all)
            // behind a chunk's end nothing changes, whatever stands there
#pragma unroll
            for (int k = 0; k < kRecSteps; ++k)
                if (s0 + k < w.from || s0 + k >= w.to) {
                    m[k] = make_float2(0.f, 0.f);
                    values[k] = 0;
                }
        if (round + 1 < p.rounds) load(s0 + stride);
#pragma unroll
        for (int k = 0; k < kRecSteps; ++k) {
            V = towards(V, m[k], unpack2(values[k], T()));
            M = longer(M, m[k]);
        }
        if (!CLUSTER) {
            run_of[par][w.run][w.lane] = both(M, V);
            __syncthreads();
            h = carried[par][w.lane];
            for (int r = 0; r < w.run; ++r) {
                const float4 q = run_of[par][r][w.lane];
                h = through(h, low(q), high(q));
            }
        } else {
            run_of[par][w.run][w.lane] = both(M, V);
            __syncthreads();
            float2 before_m = make_float2(0.f, 0.f), before_v = before_m;
            for (int r = 0; r < w.run; ++r) {
                const float4 q = run_of[par][r][w.lane];
                before_v = through(before_v, low(q), high(q));
                before_m = longer(before_m, low(q));
            }
            if (last_run)
                for (int r = 0; r < p.split; ++r) tell(&tile_of[par][w.rank][w.lane], r, longer(before_m, M), through(before_v, M, V));
            cluster_sync_threads();
            for (int r = 0; r < p.split; ++r) {
                const float4 q = tile_of[par][r][w.lane];
                if (r == w.rank) h = carry;
                carry = through(carry, low(q), high(q));
            }
            h = through(h, before_m, before_v);
        }
        if (p.states && s0 % kRecKept == 0 && w.in && s0 < p.T) st_state(p.states, int64_t(s0 / kRecKept) * p.B * p.H + w.state, h);
        if (all) {
#pragma unroll
            for (int k = 0; k < kRecSteps; ++k) {
                h = towards(h, m[k], unpack2(values[k], T()));
                if (w.in) *reinterpret_cast<uint32_t *>(out.out(k)) = pack2(h, T());
            }
        } else {
#pragma unroll
            for (int k = 0; k < kRecSteps; ++k) {
                h = towards(h, m[k], unpack2(values[k], T()));
                if (w.in && s0 + k < p.T) *reinterpret_cast<uint32_t *>(out.out(k)) = s0 + k >= w.from && s0 + k < w.to ? pack2(h, T()) : 0;
            }
        }
        out.at += stride * out.step;
        if (!CLUSTER && last_run) carried[par ^ 1][w.lane] = h;
    }
    // Only threads that have read h0 themselves, or are behind a barrier that all who do have passed, write what may lie in its place.
    if (p.h_last && w.in && (CLUSTER ? w.rank == 0 && w.run == 0 : last_run)) st_state(p.h_last, w.state, CLUSTER ? carry : h);
}

// Backwards: tiles, and the runs of a tile, are joined from the last to the first.
template <typename T, int LANES, bool CLUSTER>
__global__ void __launch_bounds__(kRecThreads, 2)
recurrence_backward_kernel(const RecDev p) {
    constexpr int kRuns = kRecThreads / LANES;
    __shared__ float4 run_of[2][kRuns][LANES];                             // -C and V of every run of the tile
    __shared__ float2 run_back[2][kRuns][LANES];                           // D
    __shared__ float4 tile_of[2][CLUSTER ? kRecMostCluster : 1][LANES];    // -C and D of every CTA's tile
    __shared__ float2 carried[2][LANES];                                   // what reaches the tile from the steps behind it
    RecPlace<LANES> w(p);
    const bool first_run = w.run == 0;
    const int stride = p.split * w.runs * kRecSteps;                       // steps of a round
    int tile0 = ((p.rounds - 1) * p.split + w.rank) * w.runs * kRecSteps, s0 = tile0 + w.run * kRecSteps;
    RecWalk gate(p, p.gate, w, s0), value(p, p.value, w, s0), grad(p, p.grad, w, s0), dgate(p, p.grad_gate, w, s0), dvalue(p, p.grad_value, w, s0);
    if (CLUSTER) cluster_arrive_relaxed();   // this CTA runs: awaited before others are told anything
    dependency_wait();
    w.measure(p);
    float2 x = ld_state(p.grad_last, w.state), carry = x, kept;
    uint32_t g[kRecSteps], v[kRecSteps], dy[kRecSteps];
    auto load = [&](int s, int tile) {
        if (s + kRecSteps <= p.T) {
#pragma unroll
            for (int k = 0; k < kRecSteps; ++k) {
                g[k] = ld_pair(gate[k]);
                v[k] = ld_pair(value[k]);
                dy[k] = ld_pair(grad[k]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < kRecSteps; ++k) {
                g[k] = s + k < p.T ? ld_pair(gate[k]) : 0;
                v[k] = s + k < p.T ? ld_pair(value[k]) : 0;
                dy[k] = s + k < p.T ? ld_pair(grad[k]) : 0;
            }
        }
        // the state in front of the tile
        kept = tile < p.T ? ld_state(p.states, int64_t(tile / kRecKept) * p.B * p.H + w.state) : make_float2(0.f, 0.f);
        gate.at -= stride * gate.step;
        value.at -= stride * value.step;
        grad.at -= stride * grad.step;
    };
    if (p.rounds > 0) load(s0, tile0);
    if (CLUSTER) cluster_wait();
    if (!CLUSTER && first_run) carried[(p.rounds - 1) & 1][w.lane] = x;
    for (int round = p.rounds - 1; round >= 0; --round, s0 -= stride, tile0 -= stride) {
        const int par = round & 1;
        const bool all = s0 >= w.from && s0 + kRecSteps <= w.to;
        float2 m[kRecSteps], M = make_float2(0.f, 0.f), V = M, D = M, h = kept;
        uint32_t gates[kRecSteps], values[kRecSteps], grads[kRecSteps];
#pragma unroll
        for (int k = 0; k < kRecSteps; ++k) {
            gates[k] = g[k];
            values[k] = v[k];
            grads[k] = dy[k];
            m[k] = gate_less_one(unpack2(g[k], T()));
        }
        if (!all)
#pragma unroll
            for (int k = 0; k < kRecSteps; ++k)
                if (s0 + k < w.from || s0 + k >= w.to) {
                    m[k] = make_float2(0.f, 0.f);
                    gates[k] = values[k] = grads[k] = 0;
                }
        if (round > 0) load(s0 - stride, tile0 - stride);
#pragma unroll
        for (int k = 0; k < kRecSteps; ++k) {
            V = towards(V, m[k], unpack2(values[k], T()));
            M = longer(M, m[k]);
        }
#pragma unroll
        for (int k = kRecSteps - 1; k >= 0; --k) D = less(add2(D, unpack2(grads[k], T())), m[k]);
        run_of[par][w.run][w.lane] = both(M, V);
        run_back[par][w.run][w.lane] = D;
        __syncthreads();
        for (int r = 0; r < w.run; ++r) {
            const float4 q = run_of[par][r][w.lane];
            h = through(h, low(q), high(q));
        }
        if (!CLUSTER) {
            x = carried[par][w.lane];
            for (int r = w.runs - 1; r > w.run; --r) x = through(x, low(run_of[par][r][w.lane]), run_back[par][r][w.lane]);
        } else {
            float2 behind_m = make_float2(0.f, 0.f), behind_d = behind_m;
            for (int r = w.runs - 1; r > w.run; --r) {
                const float2 q = low(run_of[par][r][w.lane]);
                behind_d = through(behind_d, q, run_back[par][r][w.lane]);
                behind_m = longer(behind_m, q);
            }
            if (first_run)
                for (int r = 0; r < p.split; ++r) tell(&tile_of[par][w.rank][w.lane], r, longer(behind_m, M), through(behind_d, M, D));
            cluster_sync_threads();
            for (int r = p.split - 1; r >= 0; --r) {
                const float4 q = tile_of[par][r][w.lane];
                if (r == w.rank) x = carry;
                carry = through(carry, low(q), high(q));
            }
            x = through(x, behind_m, behind_d);
        }
        float2 before[kRecSteps];                               // v - h in front of each step
#pragma unroll
        for (int k = 0; k < kRecSteps; ++k) {
            const float2 u = unpack2(values[k], T());
            before[k] = fma2(h, make_float2(-1.f, -1.f), u);
            h = towards(h, m[k], u);
        }
#pragma unroll
        for (int k = kRecSteps - 1; k >= 0; --k) {
            const float2 e = add2(x, unpack2(grads[k], T())), ce = mul2(m[k], e);   // -c e
            x = add2(e, ce);
            // f by itself: one minus c has no digits left where c is near one
            const uint32_t dg = pack2(mul2(mul2(ce, before[k]), gate_of(unpack2(gates[k], T()))), T()), dv = pack2(ce, T()) ^ 0x80008000u;
            if (all) {
                if (w.in) {
                    *reinterpret_cast<uint32_t *>(dgate.out(k)) = dg;
                    *reinterpret_cast<uint32_t *>(dvalue.out(k)) = dv;
                }
            } else {
                const bool live = s0 + k >= w.from && s0 + k < w.to;
                if (w.in && s0 + k < p.T) {
                    *reinterpret_cast<uint32_t *>(dgate.out(k)) = live ? dg : 0;
                    *reinterpret_cast<uint32_t *>(dvalue.out(k)) = live ? dv : 0;
                }
            }
        }
        dgate.at -= stride * dgate.step;
        dvalue.at -= stride * dvalue.step;
        if (!CLUSTER && first_run) carried[par ^ 1][w.lane] = x;
    }
    if (p.grad_h0 && w.in && (CLUSTER ? w.rank == 0 : true) && first_run) st_state(p.grad_h0, w.state, CLUSTER ? carry : x);
}

// How a call is spread: lanes per run, threads per CTA, CTAs per cluster.
struct RecPlan {
    int lanes, threads, split, blocks;
};
// Returns false for more CTAs than a grid has.
inline bool rec_plan(RecDev *p, RecPlan *plan) {
    plan->lanes = p->H <= 32 ? 16 : 32;
    // no more warps than the steps fill
    int warps = kRecThreads / 32;
    while (warps > 1 && (warps / 2) * (32 / plan->lanes) * kRecSteps >= p->T) warps /= 2;
    plan->threads = warps * 32;
    plan->split = 1;
    const int tile = plan->threads / plan->lanes * kRecSteps;
    p->slabs = (p->H + 2 * plan->lanes - 1) / (2 * plan->lanes);
    p->split = plan->split;
    const int64_t tiles = (int64_t(p->T) + tile - 1) / tile, blocks = int64_t(p->B) * p->slabs * plan->split;
    p->rounds = int((tiles + plan->split - 1) / plan->split);
    plan->blocks = int(blocks);
    return blocks <= INT32_MAX;
}

template <typename T, int LANES, bool CLUSTER>
int recurrence_launch(const RecDev &p, const RecPlan &plan, bool backward, cudaStream_t stream) {
    return launch_dependent_clusters(backward ? recurrence_backward_kernel<T, LANES, CLUSTER> : recurrence_kernel<T, LANES, CLUSTER>, plan.split, dim3(plan.blocks),
                                     plan.threads, 0, stream, p);
}
template <typename T>
int recurrence_launch(RecDev p, bool backward, cudaStream_t stream) {
    RecPlan plan;
    if (!rec_plan(&p, &plan)) return (int)cudaErrorInvalidValue;
    if (plan.split > 1) return plan.lanes == 16 ? recurrence_launch<T, 16, true>(p, plan, backward, stream) : recurrence_launch<T, 32, true>(p, plan, backward, stream);
    return plan.lanes == 16 ? recurrence_launch<T, 16, false>(p, plan, backward, stream) : recurrence_launch<T, 32, false>(p, plan, backward, stream);
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

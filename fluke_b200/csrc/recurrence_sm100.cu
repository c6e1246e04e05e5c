// recurrence_sm100.cu -- gated linear recurrence over time and its gradients on sm_100a:
//     h_t = f_t h_{t-1} + c_t v_t,    f_t = sigmoid(g_t),    c_t = 1 - f_t,    per chunk and channel.
// A step goes from the nearer end, by the smaller of f and c, which is 1 / (1 + exp |g|):
//     h += c (v - h) for g >= 0,    h = v + f (h - v) for g < 0.
// A run of gates near one (a channel that remembers for thousands of steps) keeps the digits of its small c so, where f rounded to f32 would be
// off by 2^-25 per step, and a gate that closes those of what it lets through, where 1 - c has 2^-24 / f of its value left: of a state of 100 behind a
// gate of -12 the form h + c (v - h) alone kept 0.9 % wrong, and a small value behind a large state lost digits to it.
//
// Gates do not depend on the state, so any run of steps acts on the state in front of it as one step does:
//     h_out = P h_in + V
// with P = prod f and V the state that the run leaves of zero. Runs are computed side by side and joined. Beside P the runs carry M = P - 1, summed up by
// itself: where P is above 1/2, which no gate below zero has then been part of, a run is h + (V + M h), for the same reason as a step.
//
// Differences are no use of infinities and of the largest bf16 values: h - v is then infinite or NaN, and the state stays one of them through any further
// steps. Steps that a state has not come out of finite are therefore taken once more, one by one, by f h + c v itself where one is not finite.
//
// Backwards, with e_t the gradient of h_t and x_t what reaches step t from the steps behind it:
//     e_t = dy_t + x_t,    x_{t-1} = f_t e_t,    dv_t = c_t e_t,    dg_t = e_t (h_{t-1} - v_t) f_t c_t
// a run of steps acts on x as x_out = P x_in + D. The states h_{t-1} are computed again, from those that the forward
// pass keeps of every 16th step (4 bytes per 16 values): that reads 6 and writes 4 bytes per value, where states kept in full would be read as well, and rounded.
//
// Both are bound by memory where chunks and channels fill the device ([1000, 256, 768] f16: forward 208 us, 0.87 of the measured copy rate, gradients 371, 0.83), else by what a warp
// issues one after the other. Four forms (recurrence_launch chooses): up to 8 steps in a thread; a warp per 64 channels of a chunk, through all steps; the same with the steps in
// segments, for few chunks; and through registers, for rows that copies of 16 bytes do not take.

namespace fluke_sm100 {
namespace {

constexpr int kRecSteps = 8;          // of a lane
constexpr int kRecKept = FLUKE_SM100_RECURRENCE_KEPT;   // steps between kept states
constexpr int kRecThreads = 256;      // of the form that goes through registers
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
    int reverse;
    int slabs;                        // runs of channels per chunk, a warp's each
    int split, segment;               // CTAs of a cluster; steps of a warp
    int rounds, runs;                 // (through registers) tiles, and warps per tile
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
__device__ __forceinline__ float plus(float a, float b) { return a + b; }
__device__ __forceinline__ float minus(float a, float b) { return a - b; }
__device__ __forceinline__ float times(float a, float b) { return a * b; }
__device__ __forceinline__ float add_times(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float2 plus(float2 a, float2 b) { return add2(a, b); }
__device__ __forceinline__ float2 minus(float2 a, float2 b) { return fma2(b, make_float2(-1.f, -1.f), a); }
__device__ __forceinline__ float2 times(float2 a, float2 b) { return mul2(a, b); }
__device__ __forceinline__ float2 add_times(float2 a, float2 b, float2 c) { return fma2(a, b, c); }
template <typename F> __device__ __forceinline__ F zero_of();
template <> __device__ __forceinline__ float zero_of<float>() { return 0.f; }
template <> __device__ __forceinline__ float2 zero_of<float2>() { return make_float2(0.f, 0.f); }
template <typename F> __device__ __forceinline__ F one_of();
template <> __device__ __forceinline__ float one_of<float>() { return 1.f; }
template <> __device__ __forceinline__ float2 one_of<float2>() { return make_float2(1.f, 1.f); }
// A step as one number q: -c where the gate keeps more than half (g >= 0), else +f; -0 is a step that changes nothing, +0 one that keeps nothing. Relative
// error below 2^-21 and, of the argument's rounding and the constant's, |g| 2^-23; zero above |g| = 87, where it is below 2^-125.
__device__ __forceinline__ float signed_share(float share, float g) { return __uint_as_float(__float_as_uint(share) ^ (~__float_as_uint(g) & 0x80000000u)); }
__device__ __forceinline__ float gate_step(float g) { return signed_share(rcp_approx(1.f + ex2_approx(fabsf(g * 1.44269504f))), g); }
__device__ __forceinline__ float2 gate_step(float2 g) {
    const float2 a = mul2(g, make_float2(1.44269504f, 1.44269504f));
    const float2 d = add2(make_float2(ex2_approx(fabsf(a.x)), ex2_approx(fabsf(a.y))), make_float2(1.f, 1.f));
    return make_float2(signed_share(rcp_approx(d.x), g.x), signed_share(rcp_approx(d.y), g.y));
}
__device__ __forceinline__ float keeps_or(float q, float a, float b) { return __float_as_int(q) < 0 ? a : b; }
__device__ __forceinline__ float2 keeps_or(float2 q, float2 a, float2 b) { return make_float2(keeps_or(q.x, a.x, b.x), keeps_or(q.y, a.y, b.y)); }
// f a + c b; f a
template <typename F> __device__ __forceinline__ F towards(F a, F q, F b) { return add_times(q, minus(a, b), keeps_or(q, a, b)); }
template <typename F> __device__ __forceinline__ F let_through(F a, F q) { return add_times(q, a, keeps_or(q, a, zero_of<F>())); }
// c a = a - f a
template <typename F> __device__ __forceinline__ F let_in(F a, F q) { return minus(minus(a, keeps_or(q, a, zero_of<F>())), times(q, a)); }
// f c = |q| (1 - |q|)
__device__ __forceinline__ float gate_slope(float q) { return fmaf(-fabsf(q), fabsf(q), fabsf(q)); }
__device__ __forceinline__ float2 gate_slope(float2 q) { return make_float2(gate_slope(q.x), gate_slope(q.y)); }
// The same where a value may be infinite, or a difference too large. A state that is not finite stays, whatever the gate.
__device__ __forceinline__ bool finite(float a) { return fabsf(a) <= 3.402823466e38f; }
// Whether steps from `start`, which a NaN would be right for, have left something that is not finite.
__device__ __forceinline__ bool broke(float start, float end) { return start == start && !finite(end); }
__device__ __forceinline__ bool broke(float2 start, float2 end) { return broke(start.x, end.x) || broke(start.y, end.y); }
__device__ __forceinline__ float share_of_state(float q) { return keeps_or(q, 1.f - fabsf(q), fabsf(q)); }
__device__ __forceinline__ float share_of_value(float q) { return keeps_or(q, fabsf(q), 1.f - fabsf(q)); }
__device__ __forceinline__ float towards_any(float a, float q, float b) {
    const float r = towards(a, q, b);
    return finite(r) ? r : finite(a) ? fmaf(share_of_state(q), a, share_of_value(q) * b) : a + share_of_value(q) * b;
}
__device__ __forceinline__ float let_through_any(float a, float q) { return finite(a) ? let_through(a, q) : a; }
__device__ __forceinline__ float let_in_any(float a, float q) { return finite(a) ? let_in(a, q) : share_of_value(q) * a; }
__device__ __forceinline__ float slope_any(float a, float q, float b) {   // (a - b) f c
    const float k = gate_slope(q), d = a - b;
    return finite(d) ? d * k : fmaf(a, k, -(b * k));
}
__device__ __forceinline__ float2 towards_any(float2 a, float2 q, float2 b) { return make_float2(towards_any(a.x, q.x, b.x), towards_any(a.y, q.y, b.y)); }
__device__ __forceinline__ float2 let_through_any(float2 a, float2 q) { return make_float2(let_through_any(a.x, q.x), let_through_any(a.y, q.y)); }
__device__ __forceinline__ float2 let_in_any(float2 a, float2 q) { return make_float2(let_in_any(a.x, q.x), let_in_any(a.y, q.y)); }
__device__ __forceinline__ float2 slope_any(float2 a, float2 q, float2 b) { return make_float2(slope_any(a.x, q.x, b.x), slope_any(a.y, q.y, b.y)); }
// What a run does: P, and M = P - 1, which is right where P is above 1/2.
template <typename F> struct RecRun { F P, M; };
template <typename F> __device__ __forceinline__ RecRun<F> no_run() { return {one_of<F>(), zero_of<F>()}; }
template <typename F> __device__ __forceinline__ void lengthen(RecRun<F> &r, F q) {
    r.M = add_times(q, r.P, r.M);
    r.P = let_through(r.P, q);
}
template <typename F> __device__ __forceinline__ RecRun<F> joined(const RecRun<F> &a, const RecRun<F> &b) { return {times(a.P, b.P), add_times(b.M, a.P, a.M)}; }
// P a + b: what a run makes of a
__device__ __forceinline__ float through(float a, const RecRun<float> &r, float b) {
    const float near = a + fmaf(r.M, a, b), far = fmaf(r.P, a, b);
    return !finite(a) ? a + b : r.P > 0.5f ? near : far;
}
__device__ __forceinline__ float2 through(float2 a, const RecRun<float2> &r, float2 b) {
    return make_float2(through(a.x, RecRun<float>{r.P.x, r.M.x}, b.x), through(a.y, RecRun<float>{r.P.y, r.M.y}, b.y));
}
__device__ __forceinline__ float2 low(float4 q) { return make_float2(q.x, q.y); }
__device__ __forceinline__ float2 high(float4 q) { return make_float2(q.z, q.w); }
__device__ __forceinline__ float4 both(float2 a, float2 b) { return make_float4(a.x, a.y, b.x, b.y); }
// Stores into the shared memory of a CTA of the cluster.
__device__ __forceinline__ void tell(const float2 *to, int rank, float2 a) {
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(cluster_address(smem_u32(to), rank)), "f"(a.x), "f"(a.y) : "memory");
}
__device__ __forceinline__ void tell(const float *to, int rank, float a) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_address(smem_u32(to), rank)), "f"(a) : "memory");
}
// 16-bit values of a lane, one or two.
template <typename T> __device__ __forceinline__ float2 widen(uint32_t v) { return unpack2(v, T()); }
template <typename T> __device__ __forceinline__ float widen(uint16_t v) { return unpack2(v, T()).x; }
template <typename T> __device__ __forceinline__ uint32_t narrow(float2 v) { return pack2(v, T()); }
template <typename T> __device__ __forceinline__ uint16_t narrow(float v) { return uint16_t(pack2(make_float2(v, 0.f), T())); }
// Gates of plus infinity: a step that changes nothing.
template <typename Raw> __device__ __forceinline__ Raw closed_gates(__half) { return Raw(0x7C007C00u); }
template <typename Raw> __device__ __forceinline__ Raw closed_gates(__nv_bfloat16) { return Raw(0x7F807F80u); }

template <int CH = 2> struct RecLane;
template <> struct RecLane<1> { typedef float F; typedef uint16_t Raw; };
template <> struct RecLane<2> { typedef float2 F; typedef uint32_t Raw; };

// A lane's channels of a chunk through steps s .. end - 1 again, from memory, where infinities or differences that are too large came up. What the steps had
// written is written over, by the same thread. Eight steps' loads (backwards four) are asked for at once: one by one they took 2.7 us a step.
template <typename T, int CH = 2>
struct RecAgain {
    using F = typename RecLane<CH>::F;
    using Raw = typename RecLane<CH>::Raw;
    const RecDev &p;
    int b, channel, from, to;
    template <typename X>
    __device__ __forceinline__ Raw *at(const X &x, int s) const {
        const uint16_t *row = static_cast<const uint16_t *>(x.at) + b * x.chunk + int64_t(p.reverse ? p.T - 1 - s : s) * x.step + channel;
        return reinterpret_cast<Raw *>(const_cast<uint16_t *>(row));
    }
    template <int N, typename X>
    __device__ __forceinline__ void read(Raw (&to_lane)[N], const X &x, int s, int end) const {
#pragma unroll
        for (int k = 0; k < N; ++k) to_lane[k] = s + k < end && live(s + k) ? *at(x, s + k) : Raw(0);
    }
    __device__ __forceinline__ F *kept(int s) const { return reinterpret_cast<F *>(p.states + (int64_t(s / kRecKept) * p.B + b) * p.H + channel); }
    __device__ __forceinline__ bool live(int s) const { return s >= from && s < to; }
    __device__ __forceinline__ F forward(int s, int end, F h, bool store) const {
#pragma unroll 1
        for (; s < end; s += kRecSteps) {
            Raw g[kRecSteps], v[kRecSteps];
            read(g, p.gate, s, end);
            read(v, p.value, s, end);
#pragma unroll
            for (int k = 0; k < kRecSteps; ++k)
                if (s + k < end) {
                    if (store && p.states && (s + k) % kRecKept == 0) *kept(s + k) = h;
                    if (!live(s + k)) continue;
                    h = towards_any(h, gate_step(widen<T>(g[k])), widen<T>(v[k]));
                    if (store) *at(p.out, s + k) = narrow<T>(h);
                }
        }
        return h;
    }
    // a run's D
    __device__ __forceinline__ F run_back(int s, int end, F d) const {
#pragma unroll 1
        for (int first = s + (end - s - 1) / kRecSteps * kRecSteps; end > s; end = first, first -= kRecSteps) {
            Raw g[kRecSteps], dy[kRecSteps];
            read(g, p.gate, first, end);
            read(dy, p.grad, first, end);
#pragma unroll
            for (int k = kRecSteps - 1; k >= 0; --k)
                if (first + k < end && live(first + k)) d = let_through_any(plus(d, widen<T>(dy[k])), gate_step(widen<T>(g[k])));
        }
        return d;
    }
    // steps from a kept state on
    static constexpr int kBack = 4;
    __device__ __forceinline__ F backward(int s, int end, F x) const {
#pragma unroll 1
        for (int first = s + (end - s - 1) / kRecKept * kRecKept; end > s; end = first, first -= kRecKept) {
            F h = *kept(first), u[kRecKept];
#pragma unroll 1
            for (int at0 = 0; at0 < kRecKept; at0 += kBack) {
                Raw g[kBack], v[kBack];
                read(g, p.gate, first + at0, end);
                read(v, p.value, first + at0, end);
#pragma unroll
                for (int k = 0; k < kBack; ++k)
                    if (first + at0 + k < end && live(first + at0 + k)) {
                        const F q = gate_step(widen<T>(g[k])), now = widen<T>(v[k]);
                        u[at0 + k] = slope_any(h, q, now);
                        h = towards_any(h, q, now);
                    }
            }
#pragma unroll 1
            for (int at0 = kRecKept - kBack; at0 >= 0; at0 -= kBack) {
                Raw g[kBack], dy[kBack];
                read(g, p.gate, first + at0, end);
                read(dy, p.grad, first + at0, end);
#pragma unroll
                for (int k = kBack - 1; k >= 0; --k)
                    if (first + at0 + k < end && live(first + at0 + k)) {
                        const F q = gate_step(widen<T>(g[k])), e = plus(x, widen<T>(dy[k]));
                        *at(p.grad_gate, first + at0 + k) = narrow<T>(times(e, u[at0 + k]));
                        *at(p.grad_value, first + at0 + k) = narrow<T>(let_in_any(e, q));
                        x = let_through_any(e, q);
                    }
            }
        }
        return x;
    }
};

// Where a warp works: 64 channels of a chunk, and of them the steps of one run of each tile. Processing goes through steps s = 0 .. T-1, time through s
// or T - 1 - s; a tensor is walked in processing order. What lies in [from, to) is inside the chunk.
struct RecPlace {
    int b, channel, lane, from, to;
    bool in;                          // the channels exist (else the last two are read, and nothing is written)
    int64_t state;
    __device__ __forceinline__ RecPlace(const RecDev &p, int slab) {
        b = slab / p.slabs;
        in = b < p.B;
        b = min(b, p.B - 1);
        lane = threadIdx.x & 31;
        channel = (slab % p.slabs) * 64 + 2 * lane;
        in = in && channel < p.H;
        channel = min(channel, p.H - 2);
        state = int64_t(b) * p.H + channel;
    }
    __device__ __forceinline__ void measure(const RecDev &p) {   // reads global memory
        const int length = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
        from = p.reverse ? p.T - length : 0;
        to = p.reverse ? p.T : length;
    }
    __device__ __forceinline__ bool inside(int s) const { return s >= from && s < to; }
};
// A tensor from step s on: bytes between steps, in processing order.
struct RecWalk {
    char *at;
    int64_t step;
    template <typename X>
    __device__ __forceinline__ RecWalk(const RecDev &p, const X &x, const RecPlace &w, int s) {
        step = (p.reverse ? -x.step : x.step) * 2;
        at = const_cast<char *>(static_cast<const char *>(x.at)) + (w.b * x.chunk + w.channel + (p.reverse ? p.T - 1 : 0) * x.step) * 2 + s * step;
    }
    __device__ __forceinline__ char *operator[](int k) const { return at + k * step; }
};
__device__ __forceinline__ void st_pair(char *p, uint32_t v) { *reinterpret_cast<uint32_t *>(p) = v; }
template <int CH = 2>
__device__ __forceinline__ typename RecLane<CH>::F ld_state(const float *s, int64_t at) {
    using F = typename RecLane<CH>::F;
    return s ? *reinterpret_cast<const F *>(s + at) : zero_of<F>();
}
template <typename F>
__device__ __forceinline__ void st_state(float *s, int64_t at, F v) { *reinterpret_cast<F *>(s + at) = v; }

// ---- a few steps ------------------------------------------------------------------------------------
// A thread has two channels of a chunk and takes them through all of up to STEPS steps, whose loads are asked for at once: what a stream's single steps cost is a
// launch and one trip to memory: [1, 1024, 768] 4.7 us (15.2 through the form below, whose registers hold a tile of runs).
template <typename T, int STEPS, bool BACKWARD>
__global__ void __launch_bounds__(256)
recurrence_steps_kernel(const RecDev p, const uint32_t pairs) {   // pairs of channels of all chunks
    const uint32_t i = blockIdx.x * 256u + threadIdx.x, row = uint32_t(p.H) / 2;
    dependency_wait();
    if (i >= pairs) return;
    const int b = int(i / row), channel = int(i - b * row) * 2;
    const int64_t state = int64_t(i) * 2;
    int from = 0, to = p.T;
    if (p.lengths) {
        const int length = min(max(p.lengths[b], 0), p.T);
        from = p.reverse ? p.T - length : 0;
        to = p.reverse ? p.T : length;
    }
    auto place = [&](const auto &x, int k) { return static_cast<const char *>(x.at) + (b * x.chunk + (p.reverse ? p.T - 1 - k : k) * x.step + channel) * 2; };
    const float2 h0 = ld_state(BACKWARD ? p.states : p.h0, state), x0 = BACKWARD ? ld_state(p.grad_last, state) : make_float2(0.f, 0.f);
    uint32_t g[STEPS], v[STEPS], dy[STEPS];
#pragma unroll
    for (int k = 0; k < STEPS; ++k)
        if (k < p.T) {
            g[k] = ld_pair(place(p.gate, k));
            v[k] = ld_pair(place(p.value, k));
            if (BACKWARD) dy[k] = ld_pair(place(p.grad, k));
        }
    if (!BACKWARD && p.states) st_state(p.states, state, h0);
    float2 q[STEPS], u[STEPS], h = h0;
    // behind a chunk's end nothing changes, whatever stands there
    auto live = [&](int k) { return k >= from && k < to; };
#pragma unroll
    for (int k = 0; k < STEPS; ++k)
        if (k < p.T) {
            const float2 now = unpack2(v[k], T());
            q[k] = gate_step(unpack2(g[k], T()));
            if (BACKWARD) u[k] = times(minus(h, now), gate_slope(q[k]));
            if (live(k)) h = towards(h, q[k], now);
            if (!BACKWARD) st_pair(const_cast<char *>(place(p.out, k)), live(k) ? pack2(h, T()) : 0);
        }
    const bool broken = broke(h0, h);
    // Again, from the registers; eight steps' gradients from memory: 80 registers instead of 86, of which an SM has three blocks instead of two (19.8 us : 24.1 at [8, 1024, 768])
    constexpr bool kFromMemory = BACKWARD && STEPS > 4;
    if (!kFromMemory && broken) {
        h = h0;
#pragma unroll
        for (int k = 0; k < STEPS; ++k)
            if (k < p.T && live(k)) {
                const float2 now = unpack2(v[k], T());
                if (BACKWARD) u[k] = slope_any(h, q[k], now);
                h = towards_any(h, q[k], now);
                if (!BACKWARD) st_pair(const_cast<char *>(place(p.out, k)), pack2(h, T()));
            }
    }
    if constexpr (!BACKWARD) {
        if (p.h_last) st_state(p.h_last, state, h);
    } else {
        float2 x = x0;
#pragma unroll
        for (int k = STEPS - 1; k >= 0; --k)
            if (k < p.T) {
                const float2 e = add2(x, unpack2(dy[k], T()));
                st_pair(const_cast<char *>(place(p.grad_gate, k)), live(k) ? pack2(mul2(e, u[k]), T()) : 0);
                st_pair(const_cast<char *>(place(p.grad_value, k)), live(k) ? pack2(let_in(e, q[k]), T()) : 0);
                if (live(k)) x = let_through(e, q[k]);
            }
        if constexpr (kFromMemory) {
            if (broken || broke(x0, x)) x = RecAgain<T>{p, b, channel, from, to}.backward(0, p.T, x0);
        } else if (broke(x0, x)) {
            x = x0;
#pragma unroll
            for (int k = STEPS - 1; k >= 0; --k)
                if (k < p.T && live(k)) {
                    const float2 e = add2(x, unpack2(dy[k], T()));
                    st_pair(const_cast<char *>(place(p.grad_gate, k)), pack2(mul2(e, u[k]), T()));
                    st_pair(const_cast<char *>(place(p.grad_value, k)), pack2(let_in_any(e, q[k]), T()));
                    x = let_through_any(e, q[k]);
                }
        }
        if (p.grad_h0) st_state(p.grad_h0, state, x);
    }
}

// ---- through registers ----------------------------------------------------------------------------
// For strides or addresses that copies of 16 bytes do not take (rows of 514 values, a view that starts on an odd multiple of two). Time is not spread over CTAs here, and a tile of 64 steps
// ends with a barrier: [1000, 32, 514] 34 us and 61 (gradients) where [1000, 32, 512] takes 33 and 42, but [65536, 1, 514] 1560 and 2520 where [65536, 1, 512] takes 90 and 130. A CTA's warps are runs of a tile (p.runs of them) of as many chunks or
// channels as that leaves; the next tile's loads are asked for while this one is computed.
template <typename T>
__global__ void __launch_bounds__(kRecThreads, 2)
recurrence_direct_kernel(const RecDev p) {
    __shared__ float4 run_of[2][kRecThreads / 32][32];                     // P and M of every run
    __shared__ float2 left_by[2][kRecThreads / 32][32];                    // V
    __shared__ float2 carried[2][kRecThreads / 32][32];                    // the state in front of the tile, by the last run's warp
    const int warp = threadIdx.x >> 5, run = warp & (p.runs - 1), first = warp - run, last = first + p.runs - 1;
    RecPlace w(p, int(blockIdx.x) * (kRecThreads / 32 / p.runs) + warp / p.runs);
    const int stride = p.runs * kRecSteps;
    int s0 = run * kRecSteps;
    RecWalk gate(p, p.gate, w, s0), value(p, p.value, w, s0), out(p, p.out, w, s0);
    dependency_wait();
    w.measure(p);
    float2 h = ld_state(p.h0, w.state);
    uint32_t g[kRecSteps], v[kRecSteps];
    auto load = [&](int s) {
#pragma unroll
        for (int k = 0; k < kRecSteps; ++k) {
            g[k] = s + k < p.T ? ld_pair(gate[k]) : 0;
            v[k] = s + k < p.T ? ld_pair(value[k]) : 0;
        }
        gate.at += stride * gate.step;
        value.at += stride * value.step;
    };
    load(s0);
    if (warp == last) carried[0][warp][w.lane] = h;
    for (int round = 0; round < p.rounds; ++round, s0 += stride) {
        const int par = round & 1;
        float2 q[kRecSteps], V = make_float2(0.f, 0.f);
        RecRun<float2> own = no_run<float2>();
        uint32_t values[kRecSteps];
#pragma unroll
        for (int k = 0; k < kRecSteps; ++k) {
            // behind a chunk's end nothing changes, whatever stands there
            const bool live = w.inside(s0 + k);
            q[k] = live ? gate_step(unpack2(g[k], T())) : make_float2(-0.f, -0.f);
            values[k] = live ? v[k] : 0;
            V = towards(V, q[k], unpack2(values[k], T()));
            lengthen(own, q[k]);
        }
        if (round + 1 < p.rounds) load(s0 + stride);
        run_of[par][warp][w.lane] = both(own.P, own.M);
        left_by[par][warp][w.lane] = V;
        __syncthreads();
        h = carried[par][last][w.lane];
        for (int r = first; r < warp; ++r) {
            const float4 run = run_of[par][r][w.lane];
            h = through(h, {low(run), high(run)}, left_by[par][r][w.lane]);
        }
        if (p.states && s0 % kRecKept == 0 && w.in && s0 < p.T) st_state(p.states, int64_t(s0 / kRecKept) * p.B * p.H + w.state, h);
#pragma unroll
        for (int k = 0; k < kRecSteps; ++k) {
            h = towards(h, q[k], unpack2(values[k], T()));
            if (w.in && s0 + k < p.T) st_pair(out[k], w.inside(s0 + k) ? pack2(h, T()) : 0);
        }
        out.at += stride * out.step;
        if (warp == last) carried[par ^ 1][warp][w.lane] = h;
    }
    __syncthreads();                  // the other runs' outputs come first
    if (w.in && warp == last) {
        const float2 h0 = ld_state(p.h0, w.state);
        if (broke(h0, h)) h = RecAgain<T>{p, w.b, w.channel, w.from, w.to}.forward(0, p.T, h0, true);
    }
    // by the threads that have read h0, which may be the same
    if (p.h_last && w.in && warp == last) st_state(p.h_last, w.state, h);
}

// Backwards: tiles, and the runs of a tile, are joined from the last to the first.
template <typename T>
__global__ void __launch_bounds__(kRecThreads, 2)
recurrence_direct_backward_kernel(const RecDev p) {
    __shared__ float4 run_of[2][kRecThreads / 32][32], left_by[2][kRecThreads / 32][32];     // P and M of every run; V and D
    // a thread's own values: held in registers they took 128 registers and more, and loads that are spilled are waited for (2400 : 3070 us at [65536, 1, 514])
    __shared__ uint32_t kept_grads[kRecSteps][kRecThreads], kept_values[kRecSteps][kRecThreads];
    __shared__ float2 carried[2][kRecThreads / 32][32];                    // what reaches the tile from behind, by the first run's warp
    const int warp = threadIdx.x >> 5, run = warp & (p.runs - 1), first = warp - run, last = first + p.runs - 1;
    RecPlace w(p, int(blockIdx.x) * (kRecThreads / 32 / p.runs) + warp / p.runs);
    const int stride = p.runs * kRecSteps;
    int tile0 = (p.rounds - 1) * stride, s0 = tile0 + run * kRecSteps;
    RecWalk gate(p, p.gate, w, s0), value(p, p.value, w, s0), grad(p, p.grad, w, s0), dgate(p, p.grad_gate, w, s0), dvalue(p, p.grad_value, w, s0);
    dependency_wait();
    w.measure(p);
    float2 x = ld_state(p.grad_last, w.state), kept = make_float2(0.f, 0.f);
    uint32_t g[kRecSteps], v[kRecSteps], dy[kRecSteps];
    auto load = [&](int s, int tile) {
#pragma unroll
        for (int k = 0; k < kRecSteps; ++k) {
            g[k] = s + k < p.T ? ld_pair(gate[k]) : 0;
            v[k] = s + k < p.T ? ld_pair(value[k]) : 0;
            dy[k] = s + k < p.T ? ld_pair(grad[k]) : 0;
        }
        kept = ld_state(p.states, int64_t(tile / kRecKept) * p.B * p.H + w.state);   // the state in front of the tile
        gate.at -= stride * gate.step;
        value.at -= stride * value.step;
        grad.at -= stride * grad.step;
    };
    bool regular = true;              // all states so far
    if (p.rounds > 0) load(s0, tile0);
    if (warp == first) carried[(p.rounds - 1) & 1][warp][w.lane] = x;
    for (int round = p.rounds - 1; round >= 0; --round, s0 -= stride, tile0 -= stride) {
        const int par = round & 1;
        float2 q[kRecSteps], V = make_float2(0.f, 0.f), D = V, h = kept;
        RecRun<float2> own = no_run<float2>();
#pragma unroll
        for (int k = 0; k < kRecSteps; ++k) {
            const bool live = w.inside(s0 + k);
            const uint32_t here = live ? v[k] : 0;
            kept_values[k][threadIdx.x] = here;
            kept_grads[k][threadIdx.x] = live ? dy[k] : 0;
            q[k] = live ? gate_step(unpack2(g[k], T())) : make_float2(-0.f, -0.f);
            V = towards(V, q[k], unpack2(here, T()));
            lengthen(own, q[k]);
        }
        if (round > 0) load(s0 - stride, tile0 - stride);
#pragma unroll
        for (int k = kRecSteps - 1; k >= 0; --k) D = let_through(add2(D, unpack2(kept_grads[k][threadIdx.x], T())), q[k]);
        run_of[par][warp][w.lane] = both(own.P, own.M);
        left_by[par][warp][w.lane] = both(V, D);
        regular = regular && !broke(zero_of<float2>(), V);
        __syncthreads();
        for (int r = first; r < warp; ++r) {
            const float4 run = run_of[par][r][w.lane];
            h = through(h, {low(run), high(run)}, low(left_by[par][r][w.lane]));
        }
        x = carried[par][first][w.lane];
        for (int r = last; r > warp; --r) {
            const float4 run = run_of[par][r][w.lane];
            x = through(x, {low(run), high(run)}, high(left_by[par][r][w.lane]));
        }
        const float2 start = h;
        float2 u[kRecSteps];                                    // (h - v) f c, with the state in front of each step
#pragma unroll
        for (int k = 0; k < kRecSteps; ++k) {
            const float2 now = unpack2(kept_values[k][threadIdx.x], T());
            u[k] = times(minus(h, now), gate_slope(q[k]));
            h = towards(h, q[k], now);
        }
#pragma unroll
        for (int k = kRecSteps - 1; k >= 0; --k) {
            const float2 e = add2(x, unpack2(kept_grads[k][threadIdx.x], T()));
            const uint32_t dg = pack2(mul2(e, u[k]), T()), dv = pack2(let_in(e, q[k]), T());
            x = let_through(e, q[k]);
            if (w.in && s0 + k < p.T) {
                const bool live = w.inside(s0 + k);
                st_pair(dgate[k], live ? dg : 0);
                st_pair(dvalue[k], live ? dv : 0);
            }
        }
        regular = regular && !broke(start, h);
        dgate.at -= stride * dgate.step;
        dvalue.at -= stride * dvalue.step;
        if (warp == first) carried[par ^ 1][warp][w.lane] = x;
    }
    __shared__ int irregular[kRecThreads / 32][32];
    irregular[warp][w.lane] = !regular;
    __syncthreads();                  // the other runs' outputs come first
    if (w.in && warp == first) {
        const float2 behind = ld_state(p.grad_last, w.state);
        for (int r = first; r <= last; ++r) regular = regular && !irregular[r][w.lane];
        if (!regular || broke(behind, x)) x = RecAgain<T>{p, w.b, w.channel, w.from, w.to}.backward(0, p.T, behind);
    }
    if (p.grad_h0 && w.in && warp == first) st_state(p.grad_h0, w.state, x);
}

// ---- a warp by itself -----------------------------------------------------------------------------
// A warp takes 64 channels of a chunk (CH = 2 per lane) or 32 (CH = 1) through all steps, in tiles of 16 that asynchronous copies of 16 bytes per lane
// bring into a ring of its own. No warp waits for another, and a step costs its two chained operations and the gate: 36 instructions for 64 values forwards and 55
// backwards with copies and stores, four of them of the special-function unit. (Tiles that eight warps share and join with a barrier each took 234 + 500 us, by an earlier form of the step, where
// this form takes 208 + 371; TMA boxes of 16 rows for the copies the same time at rows of 128 bytes and more at 64.)
//
// SEGMENTED: where chunks and channels are fewer than that needs, the warps of a CTA (and the CTAs of a cluster) take segments of the steps. Each
// first finds what its segment does as one run; the runs are joined once, and then the segment is walked from the state in front of it. Its tiles are read a second time,
// from L2 as a rule. [65536, 1, 512] 90 us in 16 clusters of 6 CTAs (with cold caches 99; clusters of 8, which run in two rounds, 142), where the 96 SMs that work issue 3.3 of 4 instructions a cycle and the 134 MB
// of inputs do not stay in L2 between the walks; [1000, 32, 512] 33: 256 CTAs on 148 SMs, of which 108 have two, and no unit is full (special-function unit 48 %, 2.1 of 4 instructions a cycle).
constexpr int kRecTile = 16;
static_assert(kRecKept == kRecTile, "a tile begins with a kept state");

template <int CH, int TENSORS, int WARPS, int STAGES, bool SEGMENTED>
struct RecLayout {
    static constexpr int kRow = 64 * CH, kTensor = kRecTile * kRow, kStage = TENSORS * kTensor, kRing = STAGES * kStage;
    static constexpr int kOffRuns = WARPS * kRing;                                         // (segmented) WARPS x 32 lanes: P, M and V or D
    static constexpr int kOffTotals = kOffRuns + (SEGMENTED ? WARPS * 32 * 12 * CH : 0);   // kRecMostCluster x 32
    static constexpr int kDynamic = kOffTotals + (SEGMENTED ? kRecMostCluster * 32 * 12 * CH : 0);
};

// Where such a warp works.
template <int CH>
struct RecWarp {
    int b, channel0, channel, lane, from, to;
    bool in;
    int64_t state;
    __device__ __forceinline__ RecWarp(const RecDev &p, int slab) {
        b = slab / p.slabs;
        lane = threadIdx.x & 31;
        channel0 = (slab - b * p.slabs) * (32 * CH);
        channel = channel0 + CH * lane;
        in = channel < p.H;
        state = int64_t(b) * p.H + min(channel, p.H - CH);
    }
    __device__ __forceinline__ void measure(const RecDev &p) {   // reads global memory
        const int length = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
        from = p.reverse ? p.T - length : 0;
        to = p.reverse ? p.T : length;
    }
    __device__ __forceinline__ bool inside(int s) const { return s >= from && s < to; }
    __device__ __forceinline__ bool tile_inside(int s) const { return s >= from && s + kRecTile <= to; }
};
__device__ __forceinline__ void copy16(uint32_t to, const void *from, uint32_t bytes) {   // zeros behind `bytes`
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// The copies of a tensor's tiles: which 16 bytes of which rows are this lane's. Rows lie in processing order.
template <int CH>
struct RecCopy {
    static constexpr int kPieces = 4 * CH, kRows = 32 / kPieces, kTurns = kRecTile / kRows;   // 16 bytes each, per row; rows at a time
    const char *at;                   // of this lane's row of the first tile
    int64_t step;                     // bytes from step to step, in processing order
    uint32_t to, bytes;               // shared address in a tile, bytes that the piece has (0: none)
    int row;
    template <typename X>
    __device__ __forceinline__ RecCopy(const RecDev &p, const X &x, const RecWarp<CH> &w, uint32_t tile0) {
        const int piece = w.lane % kPieces;
        row = w.lane / kPieces;
        step = (p.reverse ? -x.step : x.step) * 2;
        const int channel = w.channel0 + piece * 8, have = min(max(p.H - channel, 0), 8);
        bytes = have * 2;
        at = static_cast<const char *>(x.at) + (w.b * x.chunk + (have > 0 ? channel : 0) + (p.reverse ? p.T - 1 : 0) * x.step) * 2 + row * step;
        to = tile0 + row * (64 * CH) + piece * 16;
    }
    // Steps s .. s + 15, those that the tensor has
    __device__ __forceinline__ void tile(const RecDev &p, int s, uint32_t offset) const {
        const char *src = at + s * step;
        if (s + kRecTile <= p.T) {
#pragma unroll
            for (int i = 0; i < kTurns; ++i) copy16(to + offset + i * (kRows * 64 * CH), src + i * (kRows * step), bytes);
        } else {
#pragma unroll
            for (int i = 0; i < kTurns; ++i) {
                const bool has = s + row + i * kRows < p.T;
                copy16(to + offset + i * (kRows * 64 * CH), has ? src + i * (kRows * step) : at, has ? bytes : 0);
            }
        }
    }
};
// Where a lane's channels of step s go.
template <int CH>
struct RecPut {
    char *at;
    int64_t step;
    template <typename X>
    __device__ __forceinline__ RecPut(const RecDev &p, const X &x, const RecWarp<CH> &w) {
        step = (p.reverse ? -x.step : x.step) * 2;
        at = static_cast<char *>(x.at) + (w.b * x.chunk + w.channel + (p.reverse ? p.T - 1 : 0) * x.step) * 2;
    }
};

// What the runs of a CTA's warps, or of a cluster's CTAs, do to a lane's channels: [run, P M V, lane] in shared memory.
template <typename F>
struct RecRuns {
    F *at;
    __device__ __forceinline__ RecRuns(uint8_t *smem, int lane) : at(reinterpret_cast<F *>(smem) + lane) {}
    __device__ __forceinline__ void put(int r, const RecRun<F> &run, F left_of_zero) const {
        at[r * 96] = run.P;
        at[r * 96 + 32] = run.M;
        at[r * 96 + 64] = left_of_zero;
    }
    __device__ __forceinline__ RecRun<F> run(int r) const { return {at[r * 96], at[r * 96 + 32]}; }
    __device__ __forceinline__ F left(int r) const { return at[r * 96 + 64]; }
    // into the shared memory of CTA `rank` of the cluster
    __device__ __forceinline__ void tell_all(int r, int rank, const RecRun<F> &run, F left_of_zero) const {
        tell(at + r * 96, rank, run.P);
        tell(at + r * 96 + 32, rank, run.M);
        tell(at + r * 96 + 64, rank, left_of_zero);
    }
};

// (Registers: three CTAs of the plain form per SM, 168 each; with 172 there were two, [1000, 128, 768] 122 us : 116. Segments run one CTA per SM or two.)
template <typename T, int CH, int WARPS, int STAGES, bool SEGMENTED>
__global__ void __launch_bounds__(WARPS * 32, SEGMENTED ? 1 : 3)
recurrence_warp_kernel(const RecDev p) {
    using L = RecLayout<CH, 2, WARPS, STAGES, SEGMENTED>;
    using F = typename RecLane<CH>::F;
    using Raw = typename RecLane<CH>::Raw;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) >> 5, 0);
    const int rank = SEGMENTED ? int(blockIdx.x) % p.split : 0, slab = SEGMENTED ? int(blockIdx.x) / p.split : int(blockIdx.x) * WARPS + warp;
    if (SEGMENTED && p.split > 1) cluster_arrive_relaxed();   // this CTA runs: awaited before others are told anything
    dependency_wait();
    if (slab >= p.B * p.slabs) return;
    RecWarp<CH> w(p, slab);
    // the steps of this warp, in processing order, and their tiles; a segment's are walked twice
    const int segment = rank * WARPS + warp, first = SEGMENTED ? int(min(int64_t(segment) * p.segment, int64_t(p.T))) : 0, end = SEGMENTED ? min(first + p.segment, p.T) : p.T;
    const int n = (end - first + kRecTile - 1) / kRecTile, visits = SEGMENTED ? 2 * n : n;
    uint8_t *ring = smem + warp * L::kRing;
    const RecCopy<CH> gates(p, p.gate, w, smem_u32(ring)), values(p, p.value, w, smem_u32(ring) + L::kTensor);
    int put_stage = 0, put = 0, stage = 0;
    // Every turn asks for a tile, or for nothing behind the last: the copies of the turn STAGES - 1 before this one have then arrived.
    auto ask = [&] {
        if (put < visits) {
            const int s = first + (SEGMENTED && put >= n ? put - n : put) * kRecTile;
            gates.tile(p, s, put_stage * L::kStage);
            values.tile(p, s, put_stage * L::kStage);
        }
        copy_commit();
        ++put;
        if (++put_stage == STAGES) put_stage = 0;
    };
    for (int i = 0; i < STAGES - 1; ++i) ask();
    w.measure(p);
    F h = ld_state<CH>(p.h0, w.state);
    // The next tile's gates and values: fetched a tile ahead, so that its gates are computed beside the chain of the one before. (Alone on its scheduler a
    // warp is as fast as what it has to issue side by side.) Behind the last tile what the ring holds is fetched, and not used.
    F q[kRecTile], next_q[kRecTile];
    Raw v[kRecTile], next_v[kRecTile];
    auto fetch = [&](int s) {
        copy_wait<STAGES - 2>();
        __syncwarp();                 // all lanes' copies; and all lanes have read the tile whose place the next one takes
        ask();
        const uint8_t *tile = ring + stage * L::kStage + w.lane * sizeof(Raw);
        Raw g[kRecTile];
#pragma unroll
        for (int k = 0; k < kRecTile; ++k) {
            g[k] = *reinterpret_cast<const Raw *>(tile + k * L::kRow);
            next_v[k] = *reinterpret_cast<const Raw *>(tile + k * L::kRow + L::kTensor);
        }
        if (!w.tile_inside(s)) {
            // behind a chunk's end nothing changes, whatever stands there
#pragma unroll
            for (int k = 0; k < kRecTile; ++k)
                if (!w.inside(s + k)) {
                    g[k] = closed_gates<Raw>(T());
                    next_v[k] = 0;
                }
        }
        if (++stage == STAGES) stage = 0;
#pragma unroll
        for (int k = 0; k < kRecTile; ++k) next_q[k] = gate_step(widen<T>(g[k]));
    };
    auto advance = [&] {
#pragma unroll
        for (int k = 0; k < kRecTile; ++k) {
            q[k] = next_q[k];
            v[k] = next_v[k];
        }
    };
    fetch(first);
    advance();
    const RecAgain<T, CH> again{p, w.b, w.channel, w.from, w.to};
    if (SEGMENTED) {
        RecRun<F> own = no_run<F>();
        F V = zero_of<F>();
        for (int i = 0; i < n; ++i) {
            fetch(i + 1 < n ? first + (i + 1) * kRecTile : first);
#pragma unroll
            for (int k = 0; k < kRecTile; ++k) {
                V = towards(V, q[k], widen<T>(v[k]));
                lengthen(own, q[k]);
            }
            advance();
        }
        if (w.in && broke(zero_of<F>(), V)) V = again.forward(first, end, zero_of<F>(), false);
        RecRuns<F> runs(smem + L::kOffRuns, w.lane), totals(smem + L::kOffTotals, w.lane);
        runs.put(warp, own, V);
        __syncthreads();
        RecRun<F> before = no_run<F>();
        F before_v = zero_of<F>();
#pragma unroll 4
        for (int r = 0; r < warp; ++r) {
            before_v = through(before_v, runs.run(r), runs.left(r));
            before = joined(before, runs.run(r));
        }
        if (p.split > 1) {
            cluster_wait();
            if (warp == WARPS - 1) {
                const RecRun<F> all = joined(before, own);
                const F all_v = through(before_v, own, V);
                for (int r = 0; r < p.split; ++r) totals.tell_all(rank, r, all, all_v);
            }
            cluster_sync_threads();
            for (int r = 0; r < rank; ++r) h = through(h, totals.run(r), totals.left(r));
        }
        h = through(h, before, before_v);
    }
    const F start = h;
    const RecPut<CH> out(p, p.out, w);
    for (int i = 0; i < n; ++i) {
        const int s = first + i * kRecTile;
        if (p.states && w.in) st_state(p.states, int64_t(s / kRecKept) * p.B * p.H + w.state, h);
        fetch(s + kRecTile);
#pragma unroll
        for (int k = 0; k < kRecTile; ++k) {
            h = towards(h, q[k], widen<T>(v[k]));
            v[k] = narrow<T>(h);
        }
        char *to = out.at + s * out.step;
        if (w.tile_inside(s)) {
            if (w.in)
#pragma unroll
                for (int k = 0; k < kRecTile; ++k, to += out.step) *reinterpret_cast<Raw *>(to) = v[k];
        } else {
#pragma unroll
            for (int k = 0; k < kRecTile; ++k, to += out.step)
                if (w.in && s + k < p.T) *reinterpret_cast<Raw *>(to) = w.inside(s + k) ? v[k] : Raw(0);
        }
        advance();
    }
    if (w.in && broke(start, h)) h = again.forward(first, end, start, true);
    // By threads that have read h0 themselves, or are behind a barrier that all who do have passed: it may lie in the same place.
    if (p.h_last && w.in && (!SEGMENTED || segment == p.split * WARPS - 1)) st_state(p.h_last, w.state, h);
}

// Backwards: steps are walked from the last to the first. In a tile the states are computed again from the one that the forward pass kept.
// (Without a bound on the blocks per SM the compiler stays at 130 registers in the plain form and issues a tile's gates one after the other: [256, 64, 512] 28.5 us : 20.1 with 206.)
template <typename T, int CH, int WARPS, int STAGES, bool SEGMENTED>
__global__ void __launch_bounds__(WARPS * 32, 1)
recurrence_warp_backward_kernel(const RecDev p) {
    using L = RecLayout<CH, 3, WARPS, STAGES, SEGMENTED>;
    using F = typename RecLane<CH>::F;
    using Raw = typename RecLane<CH>::Raw;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) >> 5, 0);
    const int rank = SEGMENTED ? int(blockIdx.x) % p.split : 0, slab = SEGMENTED ? int(blockIdx.x) / p.split : int(blockIdx.x) * WARPS + warp;
    if (SEGMENTED && p.split > 1) cluster_arrive_relaxed();   // this CTA runs: awaited before others are told anything
    dependency_wait();
    if (slab >= p.B * p.slabs) return;
    RecWarp<CH> w(p, slab);
    const int segment = rank * WARPS + warp, first = SEGMENTED ? int(min(int64_t(segment) * p.segment, int64_t(p.T))) : 0, end = SEGMENTED ? min(first + p.segment, p.T) : p.T;
    const int n = (end - first + kRecTile - 1) / kRecTile, visits = SEGMENTED ? 2 * n : n;
    uint8_t *ring = smem + warp * L::kRing;
    const uint32_t ring0 = smem_u32(ring);
    const RecCopy<CH> gates(p, p.gate, w, ring0), values(p, p.value, w, ring0 + L::kTensor), grads(p, p.grad, w, ring0 + 2 * L::kTensor);
    int put_stage = 0, put = 0, stage = 0;
    auto ask = [&] {
        if (put < visits) {
            const bool run_only = SEGMENTED && put < n;   // the first walk takes no values
            const int s = first + (n - 1 - (SEGMENTED && !run_only ? put - n : put)) * kRecTile;
            gates.tile(p, s, put_stage * L::kStage);
            if (!run_only) values.tile(p, s, put_stage * L::kStage);
            grads.tile(p, s, put_stage * L::kStage);
        }
        copy_commit();
        ++put;
        if (++put_stage == STAGES) put_stage = 0;
    };
    for (int i = 0; i < STAGES - 1; ++i) ask();
    w.measure(p);
    F x = ld_state<CH>(p.grad_last, w.state);
    // the next tile, `values_too` or only gates and gradients
    Raw g[kRecTile], v[kRecTile], dy[kRecTile];
    auto take = [&](int s, auto values_too) {
        copy_wait<STAGES - 2>();
        __syncwarp();                 // all lanes' copies; and all lanes have read the tile whose place the next one takes
        ask();
        const uint8_t *tile = ring + stage * L::kStage + w.lane * sizeof(Raw);
#pragma unroll
        for (int k = 0; k < kRecTile; ++k) {
            g[k] = *reinterpret_cast<const Raw *>(tile + k * L::kRow);
            if constexpr (decltype(values_too)::value) v[k] = *reinterpret_cast<const Raw *>(tile + k * L::kRow + L::kTensor);
            dy[k] = *reinterpret_cast<const Raw *>(tile + k * L::kRow + 2 * L::kTensor);
        }
        if (!w.tile_inside(s)) {
#pragma unroll
            for (int k = 0; k < kRecTile; ++k)
                if (!w.inside(s + k)) {
                    g[k] = closed_gates<Raw>(T());
                    v[k] = dy[k] = 0;
                }
        }
        if (++stage == STAGES) stage = 0;
    };
    const RecAgain<T, CH> again{p, w.b, w.channel, w.from, w.to};
    if (SEGMENTED) {
        RecRun<F> own = no_run<F>();
        F D = zero_of<F>();
        for (int i = n - 1; i >= 0; --i) {
            take(first + i * kRecTile, std::false_type());
            F q[kRecTile];
#pragma unroll
            for (int k = 0; k < kRecTile; ++k) q[k] = gate_step(widen<T>(g[k]));
#pragma unroll
            for (int k = kRecTile - 1; k >= 0; --k) {
                D = let_through(plus(D, widen<T>(dy[k])), q[k]);
                lengthen(own, q[k]);
            }
        }
        if (w.in && broke(zero_of<F>(), D)) D = again.run_back(first, end, zero_of<F>());
        RecRuns<F> runs(smem + L::kOffRuns, w.lane), totals(smem + L::kOffTotals, w.lane);
        runs.put(warp, own, D);
        __syncthreads();
        RecRun<F> behind = no_run<F>();
        F behind_d = zero_of<F>();
#pragma unroll 4
        for (int r = WARPS - 1; r > warp; --r) {
            behind_d = through(behind_d, runs.run(r), runs.left(r));
            behind = joined(behind, runs.run(r));
        }
        if (p.split > 1) {
            cluster_wait();
            if (warp == 0) {
                const RecRun<F> all = joined(behind, own);
                const F all_d = through(behind_d, own, D);
                for (int r = 0; r < p.split; ++r) totals.tell_all(rank, r, all, all_d);
            }
            cluster_sync_threads();
            for (int r = p.split - 1; r > rank; --r) x = through(x, totals.run(r), totals.left(r));
        }
        x = through(x, behind, behind_d);
    }
    const RecPut<CH> dgate(p, p.grad_gate, w), dvalue(p, p.grad_value, w);
    // the state in front of a tile, asked for a tile ahead
    auto state_at = [&](int i) { return i >= 0 ? ld_state<CH>(p.states, int64_t((first + i * kRecTile) / kRecKept) * p.B * p.H + w.state) : zero_of<F>(); };
    F kept = state_at(n - 1);
    // What a tile needs of gates and states: q, and (h - v) f c with the state h in front of the step. With one channel per lane the registers hold two
    // tiles', and one's are computed beside the chain of the other, which goes back in time.
    constexpr bool kAhead = CH == 1;
    F q[kRecTile], u[kRecTile];
    Raw e_in[kRecTile];
    const F start = x;
    bool regular = true;              // all states so far
    auto prepare = [&](int i, F (&tq)[kRecTile], F (&tu)[kRecTile], Raw (&te)[kRecTile]) {
        const F before = kept;
        F h = before;
        kept = state_at(i - 1);
        take(first + i * kRecTile, std::true_type());
#pragma unroll
        for (int k = 0; k < kRecTile; ++k) {
            tq[k] = gate_step(widen<T>(g[k]));
            te[k] = dy[k];
        }
#pragma unroll
        for (int k = 0; k < kRecTile; ++k) {
            const F now = widen<T>(v[k]);
            tu[k] = times(minus(h, now), gate_slope(tq[k]));
            h = towards(h, tq[k], now);
        }
        regular = regular && (i < 0 || !broke(before, h));
    };
    auto finish = [&](int s) {
        Raw dg[kRecTile], dv[kRecTile];
#pragma unroll
        for (int k = kRecTile - 1; k >= 0; --k) {
            const F e = plus(x, widen<T>(e_in[k]));
            dg[k] = narrow<T>(times(e, u[k]));
            dv[k] = narrow<T>(let_in(e, q[k]));
            x = let_through(e, q[k]);
        }
        char *to_g = dgate.at + s * dgate.step, *to_v = dvalue.at + s * dvalue.step;
        if (w.tile_inside(s)) {
            if (w.in)
#pragma unroll
                for (int k = 0; k < kRecTile; ++k, to_g += dgate.step, to_v += dvalue.step) {
                    *reinterpret_cast<Raw *>(to_g) = dg[k];
                    *reinterpret_cast<Raw *>(to_v) = dv[k];
                }
        } else {
#pragma unroll
            for (int k = 0; k < kRecTile; ++k, to_g += dgate.step, to_v += dvalue.step)
                if (w.in && s + k < p.T) {
                    *reinterpret_cast<Raw *>(to_g) = w.inside(s + k) ? dg[k] : Raw(0);
                    *reinterpret_cast<Raw *>(to_v) = w.inside(s + k) ? dv[k] : Raw(0);
                }
        }
    };
    if constexpr (kAhead) {
        if (n > 0) prepare(n - 1, q, u, e_in);
        for (int i = n - 1; i >= 0; --i) {
            F next_q[kRecTile], next_u[kRecTile];
            Raw next_e[kRecTile];
            prepare(i - 1, next_q, next_u, next_e);   // in front of the first tile: what the ring holds, and not used
            finish(first + i * kRecTile);
#pragma unroll
            for (int k = 0; k < kRecTile; ++k) {
                q[k] = next_q[k];
                u[k] = next_u[k];
                e_in[k] = next_e[k];
            }
        }
    } else {
        for (int i = n - 1; i >= 0; --i) {
            prepare(i, q, u, e_in);
            finish(first + i * kRecTile);
        }
    }
    if (w.in && (!regular || broke(start, x))) x = again.backward(first, end, start);
    if (p.grad_h0 && w.in && (!SEGMENTED || segment == 0)) st_state(p.grad_h0, w.state, x);
}

template <typename T>
int recurrence_direct(RecDev p, bool backward, cudaStream_t stream) {
    // no more runs than the steps fill
    p.slabs = (p.H + 63) / 64;
    p.runs = kRecThreads / 32;
    while (p.runs > 1 && p.runs / 2 * kRecSteps >= p.T) p.runs /= 2;
    const int per_cta = kRecThreads / 32 / p.runs, tile = p.runs * kRecSteps;
    p.rounds = (p.T + tile - 1) / tile;
    const int64_t blocks = (int64_t(p.B) * p.slabs + per_cta - 1) / per_cta;
    if (blocks > INT32_MAX / 8) return (int)cudaErrorInvalidValue;   // slabs are counted in 32 bits
    return launch_dependent(backward ? recurrence_direct_backward_kernel<T> : recurrence_direct_kernel<T>, int(blocks), kRecThreads, 0, stream, p);
}

// Whether copies of 16 bytes can take a tensor's rows.
template <typename X>
bool rec_pieces_ok(const RecDev &p, const X &x) {
    return (reinterpret_cast<uintptr_t>(x.at) & 15u) == 0 && (p.T <= 1 || x.step % 8 == 0) && (p.B <= 1 || x.chunk % 8 == 0);
}

// The two directions of a form, for its number of CTAs per cluster and its capacity.
template <typename T, int CH, int WARPS, int STAGES, bool SEGMENTED, bool BACKWARD>
constexpr auto rec_warp_kernel() {
    if constexpr (BACKWARD) return recurrence_warp_backward_kernel<T, CH, WARPS, STAGES, SEGMENTED>;
    else return recurrence_warp_kernel<T, CH, WARPS, STAGES, SEGMENTED>;
}
template <typename T, int CH, int WARPS, int STAGES, bool SEGMENTED, bool BACKWARD>
int recurrence_warps(RecDev p, cudaStream_t stream) {
    constexpr auto kernel = rec_warp_kernel<T, CH, WARPS, STAGES, SEGMENTED, BACKWARD>();
    constexpr int kSmem = RecLayout<CH, BACKWARD ? 3 : 2, WARPS, STAGES, SEGMENTED>::kDynamic;
    static_assert(kSmem <= 232448, "shared memory");
    p.slabs = (p.H + 32 * CH - 1) / (32 * CH);
    const int64_t all = int64_t(p.B) * p.slabs;
    if (all > INT32_MAX / 16) return (int)cudaErrorInvalidValue;   // slabs are counted in 32 bits
    p.split = 1;
    if (SEGMENTED)
        // as many CTAs per cluster as run at once, with two tiles per warp at least
        for (int c = kRecMostCluster; c > 1 && p.split == 1; --c)
            if (all * c <= device_sm_count() && int64_t(p.T) >= int64_t(c) * WARPS * 2 * kRecTile && all <= cluster_capacity<kernel>(c, WARPS * 32, kSmem)) p.split = c;
    // whole tiles
    p.segment = int(((int64_t(p.T) + p.split * WARPS - 1) / (p.split * WARPS) + kRecTile - 1) / kRecTile * kRecTile);
    const int64_t blocks = SEGMENTED ? all * p.split : (all + WARPS - 1) / WARPS;
    const int rc = configure_smem<kernel>(kSmem);
    if (rc) return rc;
    return launch_dependent_clusters(kernel, p.split, dim3(int(blocks)), WARPS * 32, kSmem, stream, p);
}

template <typename T, bool BACKWARD>
int recurrence_launch(RecDev p, cudaStream_t stream) {
    const bool pieces = rec_pieces_ok(p, p.gate) && rec_pieces_ok(p, p.value) && (!BACKWARD || rec_pieces_ok(p, p.grad));
    const int64_t pairs = int64_t(p.B) * (p.H / 2);
    if (p.T <= 8 && pairs <= INT32_MAX - 256) {
        auto kernel = p.T <= 1 ? recurrence_steps_kernel<T, 1, BACKWARD> : p.T <= 4 ? recurrence_steps_kernel<T, 4, BACKWARD> : recurrence_steps_kernel<T, 8, BACKWARD>;
        return launch_dependent(kernel, int((pairs + 255) / 256), 256, 0, stream, p, uint32_t(pairs));
    }
    if (!pieces) return recurrence_direct<T>(p, BACKWARD, stream);
    const int64_t narrow = int64_t(p.B) * ((p.H + 31) / 32);
    // Us per call, forward and gradients, measured with cold caches, form by form (64 channels a warp : segments of 4 warps : segments of 16 warps of 32 channels): [256, 64, 512]
    // 21 + 27 : 29 + 33 : 43 + 53, [1000, 32, 512] 51 + 75 : 39 + 48 : 55 + 72, [333, 7, 520] 23 + 33 : 14 + 16 : 12 + 14, [16384, 4, 256] 684 + 1071 : 66 + 85 : 46 + 62. From 200 to 1023 runs of 32 channels the second
    // is taken whatever the number of steps, also where more warps per chunk would be faster: [65536, 13, 512] 1342 + 1745 there, 1052 + 1546 in segments of 16 warps, 1008 + 1336 in those of 8 warps of 64 channels.
    if (narrow >= 1024 || p.T <= 64) return recurrence_warps<T, 2, 4, BACKWARD ? 3 : 4, false, BACKWARD>(p, stream);
    if (narrow >= 200) return recurrence_warps<T, 2, 4, 4, true, BACKWARD>(p, stream);
    // Long segments of 64 channels, 8 warps : of 32 channels, 16 warps: [2000, 10, 512] 41 + 51 : 46 + 61, [4096, 8, 256] 27 + 32 : 29 + 38, [8000, 3, 512] 37 + 45 : 45 + 60,
    // [16384, 4, 256] 53 + 70 : 46 + 62.
    if (p.T >= 1024 && narrow >= 40) return recurrence_warps<T, 2, 8, 3, true, BACKWARD>(p, stream);
    return recurrence_warps<T, 1, 16, 4, true, BACKWARD>(p, stream);
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
    if (p.T == 0) return {};
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
    p.h0 = r->h0; p.h_last = r->h_last; p.grad_last = r->grad_last; p.grad_h0 = r->grad_h0;
    p.states = r->T > 0 ? r->states : nullptr;   // without steps there are none, whatever the address
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
            if (!in_place && !rec_apart(out[o], in[i])) return (int)cudaErrorInvalidValue;
        }
        for (int other = 0; other < o; ++other)
            if (!rec_apart(out[o], out[other])) return (int)cudaErrorInvalidValue;
        if (out[o].H && !rec_rows_apart(out[o])) return (int)cudaErrorInvalidValue;
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (backward) return r->bf16 ? recurrence_launch<__nv_bfloat16, true>(p, s) : recurrence_launch<__half, true>(p, s);
    return r->bf16 ? recurrence_launch<__nv_bfloat16, false>(p, s) : recurrence_launch<__half, false>(p, s);
}

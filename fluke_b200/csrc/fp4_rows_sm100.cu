// fp4_rows_sm100.cu -- the memory-bound kernels of microscaled 4-bit floating point: quantisation of
// rows in two formats, reading back, and the norms before and after a block (with its gate and
// residual scale) whose result may leave quantised.
//
// Elements are E2M1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and sign), two to a byte, the earlier one in the low half;
// rounding to nearest, ties to the even code, saturating at 6.
//   MX  blocks of 32 along the row (OCP Microscaling Formats v1.0): scale 2^e, e = floor(log2(amax)) - 2 limited to
//       -127 .. 127, stored as e + 127; an all-zero block has e = -127. Scaling is exact, so the
//       only rounding is that of the element.
//   NV  blocks of 16 under an e4m3 scale s, and a power of two g per row: the least with
//       amax(row) <= 2688 g = 6 * 448 g (at least 2^-100; 1 for a row of zeros). s = e4m3(bmax / (6 g)),
//       element = e2m1(x / (s g)), both quotients rounded to f32 first; s = 0 gives zeros.
//       A power of two keeps s g exact in four bits, so that ties are what they are in real numbers.
// A block (MX) or row (NV) with an infinity or a NaN has no value: its scale is the NaN code (MX 255; NV
// 0x7F, and g is NaN) and its elements are zero.
//
// Block scales are stored in the order in which a tensor-memory copy wants them: 512-byte tiles of 128 rows
// x 4 blocks, tile (r / 128, c / 4) with block c of row r at byte (r % 32) * 16 + (r / 32 % 4) * 4 + c % 4. Blocks behind
// the end of a row up to the next multiple of 4 are written as zero; rows behind the last are left as they were.
#include <cuda_bf16.h>

namespace fluke_sm100 {
namespace {

enum Fp4Out { kFp4Plain = 0, kFp4Mx = 1, kFp4Nv = 2, kFp4None = 3 };

__device__ __forceinline__ float2 unpack2(uint32_t v, __half) { return half2_bits_to_float2(v); }
__device__ __forceinline__ float2 unpack2(uint32_t v, __nv_bfloat16) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
}
__device__ __forceinline__ uint32_t pack2(float2 f, __half) { return float2_to_half2_bits(f); }
__device__ __forceinline__ uint32_t pack2(float2 f, __nv_bfloat16) {
    const __nv_bfloat162 h = __float22bfloat162_rn(f);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Eight values as codes, the first in the lowest four bits.
__device__ __forceinline__ uint32_t e2m1x8(float2 a, float2 b, float2 c, float2 d) {
    uint32_t w;
    asm("{\n.reg .b8 p, q, r, s;\n"
        "cvt.rn.satfinite.e2m1x2.f32 p, %2, %1;\n"
        "cvt.rn.satfinite.e2m1x2.f32 q, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 r, %6, %5;\n"
        "cvt.rn.satfinite.e2m1x2.f32 s, %8, %7;\n"
        "mov.b32 %0, {p, q, r, s};\n}"
        : "=r"(w) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y), "f"(d.x), "f"(d.y));
    return w;
}
// Eight codes as values.
__device__ __forceinline__ void e2m1x8_to_float(uint32_t w, float2 (&v)[4]) {
    uint32_t h[4];
    asm("{\n.reg .b8 p, q, r, s;\n"
        "mov.b32 {p, q, r, s}, %4;\n"
        "cvt.rn.f16x2.e2m1x2 %0, p;\n"
        "cvt.rn.f16x2.e2m1x2 %1, q;\n"
        "cvt.rn.f16x2.e2m1x2 %2, r;\n"
        "cvt.rn.f16x2.e2m1x2 %3, s;\n}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = half2_bits_to_float2(h[i]);
}

// max(|a|, |b|, |c|), NaN where one of them is.
__device__ __forceinline__ float max_abs3(float a, float b, float c) {
    float m;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
    return m;
}
// The bit pattern of the largest magnitude of 16 values: patterns order like the values, infinities above every
// number and NaNs above those.
__device__ __forceinline__ uint32_t max_bits16(const float2 (&v)[8]) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max_abs3(m, v[i].x, v[i].y);
    return __float_as_uint(m);
}
constexpr uint32_t kInfBits = 0x7F800000u;

// 2^(e - 127) for a stored exponent of 0 .. 254, the smallest of which is not a normal number; 255 gives NaN.
__device__ __forceinline__ float e8m0_value(uint32_t e) {
    return __uint_as_float(e == 0 ? 0x00400000u : e == 255 ? 0x7FFFFFFFu : e << 23);
}
__device__ __forceinline__ float e4m3_value(uint32_t s) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(s)));
    return half2_bits_to_float2(h).x;
}

// Byte of the scale of block c of row r; `tiles` of four blocks to a row.
__device__ __forceinline__ int64_t scale_byte(int64_t r, int c, int tiles) {
    return ((r >> 7) * tiles + (c >> 2)) * 512 + int((r & 31) * 16 + ((r >> 5) & 3) * 4) + (c & 3);
}
// Zeros behind the last block of a row, up to a multiple of four.
__device__ __forceinline__ void pad_scales(uint8_t *scale, int64_t row, int blocks, int tiles) {
    for (int c = blocks; c < tiles * 4; ++c) scale[scale_byte(row, c, tiles)] = 0;
}

// MX: the stored exponent of a block by the bits of its largest magnitude. 255: no value.
__device__ __forceinline__ uint32_t mx_exponent(uint32_t amax_bits) {
    if (amax_bits >= kInfBits) return 255;
    const uint32_t e = amax_bits >> 23;
    return e > 2 ? e - 2 : 0;
}
// MX: 16 codes of a block with that exponent.
__device__ __forceinline__ uint2 mx_codes(const float2 (&v)[8], uint32_t e) {
    if (e == 255) return make_uint2(0, 0);
    const float f = __uint_as_float((254 - e) << 23);  // 2^(127 - e), e <= 253
    const float2 f2 = make_float2(f, f);
    float2 q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = mul2(v[i], f2);
    return make_uint2(e2m1x8(q[0], q[1], q[2], q[3]), e2m1x8(q[4], q[5], q[6], q[7]));
}

// NV: the power of two of a row by the bits of its largest magnitude; NaN without one.
__device__ __forceinline__ float nv_row_scale(uint32_t amax_bits) {
    if (amax_bits == 0) return 1.0f;
    if (amax_bits >= kInfBits) return __uint_as_float(0x7FFFFFFFu);
    // amax = f 2^E with 1 <= f < 2 and 2688 = 1.3125 * 2^11
    const int E = int(amax_bits >> 23) - 127 - 11 + ((amax_bits & 0x7FFFFFu) > 0x280000u ? 1 : 0);
    return __uint_as_float(uint32_t(max(E, -100) + 127) << 23);
}
// NV: 16 codes of a block (its own largest magnitude given) in a row of scale g, and its e4m3 scale.
__device__ __forceinline__ uint2 nv_codes(const float2 (&v)[8], uint32_t bmax_bits, float g, uint32_t &s8) {
    if (!(g > 0.f)) {
        s8 = 0x7F;
        return make_uint2(0, 0);
    }
    // Two quotients, each correctly rounded: q = v r with the correctly rounded reciprocal r of the divisor, then q + (v - q s) r with an exact residual, one fused
    // operation each (P. Markstein, IBM J. Res. Dev. 34, 1990). In general that leaves the last quotient to be proved; for the divisors here, six and four
    // significant bits, every mantissa was tried (tests/test_fp4_range_cpu.py). No step leaves the normal numbers where a code depends on it: s g is at
    // least 2^-109 and a value below a quarter of it is zero. First bmax / (6 g), g a power of two.
    const float b = __uint_as_float(bmax_bits) * __uint_as_float((254u << 23) - __float_as_uint(g));
    constexpr float kSixth = 1.0f / 6.0f;
    float t = b * kSixth;
    t = fmaf(fmaf(-6.0f, t, b), kSixth, t);
    uint16_t pair;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(pair) : "f"(0.f), "f"(t));
    s8 = pair & 0xFFu;
    if (s8 == 0) return make_uint2(0, 0);
    // Then v / s, computed as its negative: like this a zero keeps its sign through the residual, and all signs are turned at once.
    const float s = e4m3_value(s8) * g, r = -__frcp_rn(s);
    const float2 r2 = make_float2(r, r), s2 = make_float2(s, s);
    float2 q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        q[i] = mul2(v[i], r2);
        q[i] = fma2(fma2(q[i], s2, v[i]), r2, q[i]);
    }
    return make_uint2(e2m1x8(q[0], q[1], q[2], q[3]) ^ 0x88888888u, e2m1x8(q[4], q[5], q[6], q[7]) ^ 0x88888888u);
}

// A unit: 16 consecutive values of a row, 32 bytes in 16 bits and 8 as codes.
template <typename T>
__device__ __forceinline__ void unpack16(const uint32_t (&r)[8], float2 (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = unpack2(r[i], T());
}

// ---- quantisation, MX -------------------------------------------------------------------------
// Blocks do not depend on their row: thread = unit, a block is two neighbouring lanes (rows are whole blocks, so
// a pair never straddles two; row0 is the row of the first unit). Bound by memory: 2 bytes in and 0.53 out per value; [32000, 512] 7.0 us, 0.91 of the measured copy rate.
template <typename T>
__global__ void __launch_bounds__(256)
quant_mxfp4_kernel(const T *in, uint8_t *codes, uint8_t *scale, uint32_t units, uint32_t units_per_row, int tiles, uint32_t row0) {
    dependency_wait();
    const uint32_t u = blockIdx.x * 256u + threadIdx.x;
    const bool live = u < units;
    uint32_t raw[8] = {};
    if (live) load32(in + int64_t(u) * 16, raw);
    float2 v[8];
    unpack16<T>(raw, v);
    uint32_t m = max_bits16(v);
    m = max(m, __shfl_xor_sync(kFull, m, 1));
    if (!live) return;
    const uint32_t e = mx_exponent(m);
    *reinterpret_cast<uint2 *>(codes + int64_t(u) * 8) = mx_codes(v, e);
    const uint32_t r = u / units_per_row, at = u - r * units_per_row, row = row0 + r;
    if ((at & 1u) == 0) scale[scale_byte(row, int(at >> 1), tiles)] = uint8_t(e);
    if (at == units_per_row - 1) pad_scales(scale, row, int(units_per_row >> 1), tiles);
}

// ---- reading back -----------------------------------------------------------------------------
// value = code * 2^e, or (code * s) * g, rounded once. Thread = unit. Bound by memory: [32000, 512] from mxfp4 6.2 us, [9331, 2048] from nvfp4 7.4.
template <typename T, bool MX>
__global__ void __launch_bounds__(256)
dequant_fp4_kernel(const uint8_t *codes, const uint8_t *scale, const float *row_scale, T *out, uint32_t units, uint32_t units_per_row,
                   int tiles, uint32_t row0) {
    dependency_wait();
    const uint32_t u = blockIdx.x * 256u + threadIdx.x;
    if (u >= units) return;
    const uint32_t row = u / units_per_row, at = u - row * units_per_row;
    const uint2 c = *reinterpret_cast<const uint2 *>(codes + int64_t(u) * 8);
    const uint32_t s8 = scale[scale_byte(int64_t(row0) + row, int(MX ? at >> 1 : at), tiles)];
    const float s = MX ? e8m0_value(s8) : e4m3_value(s8), g = MX ? 1.f : row_scale[row];
    const float2 s2 = make_float2(s, s), g2 = make_float2(g, g);
    float2 lo[4], hi[4];
    e2m1x8_to_float(c.x, lo);
    e2m1x8_to_float(c.y, hi);
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = mul2(lo[i], s2), b = mul2(hi[i], s2);
        r[i] = pack2(MX ? a : mul2(a, g2), T());
        r[i + 4] = pack2(MX ? b : mul2(b, g2), T());
    }
    store32(out + int64_t(u) * 16, r);
}

// ---- rows held in registers -------------------------------------------------------------------
// A row belongs to half a warp or a warp (blocks whose warps walk rows), or to a block of up to 16 warps; lane l of the row's `lanes`
// holds units l, l + lanes, ... (U of them). Maximum and sum of a block's row:
constexpr int kFp4RowWarps = 16, kFp4WalkWarps = 8, kFp4NormWarps = 4;   // of a block that holds a row, at most; of blocks that walk rows

__device__ __forceinline__ uint32_t row_max(uint32_t m, uint32_t *shared) {
    m = __reduce_max_sync(kFull, m);
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) shared[warp] = m;
    __syncthreads();
    m = 0;
    for (int w = 0; w < warps; ++w) m = max(m, shared[w]);
    return m;
}
__device__ __forceinline__ double row_sum(double s, double *shared) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(kFull, s, d);
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) shared[warp] = s;
    __syncthreads();
    s = 0;
    for (int w = 0; w < warps; ++w) s += shared[w];
    return s;
}

// The units of a row that this lane holds; zeros from unit `have` on.
template <int U>
__device__ __forceinline__ void load_row(const void *base, int64_t row, int have, int units, int lane, int lanes, uint32_t (&raw)[U][8]) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
        if (lane + j * lanes < have) load32(static_cast<const uint8_t *>(base) + (row * units + lane + j * lanes) * 32, raw[j]);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) raw[j][i] = 0;
    }
}
template <int U>
__device__ __forceinline__ void copy_row(uint32_t (&to)[U][8], const uint32_t (&from)[U][8]) {
#pragma unroll
    for (int j = 0; j < U; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) to[j][i] = from[j][i];
}

// Quantisation, NV. LANES lanes (half a warp or one) hold a row, and a warp works through rows with the next ones on their way while it computes
// ([9331, 2048] bf16 19.4 -> 12.2 us against a warp per row; 9.9 with the quotients of nv_codes and the three-operand maximum, 0.76 of the copy
// rate; with four units per lane two registers spill at 128). Two or four warps to such a row instead of one: 10.8, 11.8. Half a warp: [16384, 256] 4.7 -> 3.3, [32000, 512] 9.0 -> 8.5, [16384, 768] 7.8 -> 6.8.
template <typename T, int LANES, int U>
__global__ void __launch_bounds__(kFp4WalkWarps * 32, U == 1 ? 4 : U == 2 ? 3 : 2)
quant_nvfp4_rows_kernel(const T *in, uint8_t *codes, uint8_t *scale, float *row_scale, int rows, int units, int tiles) {
    constexpr int kGroups = 32 / LANES;   // rows of a warp at a time
    dependency_wait();
    const int lane = threadIdx.x & (LANES - 1), group = (threadIdx.x & 31) / LANES;
    const int step = int(gridDim.x) * kFp4WalkWarps * kGroups;
    // the loop is the same for all lanes of a warp; rows behind the last are zeros and not written
    int first = (int(blockIdx.x) * kFp4WalkWarps + (int(threadIdx.x) >> 5)) * kGroups;
    uint32_t raw[U][8], ahead[U][8];
    auto load = [&](int row, uint32_t (&r)[U][8]) { load_row<U>(in, row, row < rows ? units : 0, units, lane, LANES, r); };
    if (first < rows) load(first + group, raw);
    for (; first < rows; first += step) {
        const int row = first + group, mine = row < rows ? units : 0;
        if (first + step < rows) load(row + step, ahead);
        uint32_t bmax[U], amax = 0;
#pragma unroll
        for (int j = 0; j < U; ++j) {
            float2 v[8];
            unpack16<T>(raw[j], v);
            bmax[j] = max_bits16(v);
            amax = max(amax, bmax[j]);
        }
        const float g = nv_row_scale(__reduce_max_sync(LANES == 32 ? kFull : 0xFFFFu << (threadIdx.x & 16), amax));
        if (lane == 0 && mine) row_scale[row] = g;
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int at = lane + j * LANES;
            if (at >= mine) break;
            float2 v[8];
            unpack16<T>(raw[j], v);
            uint32_t s8;
            *reinterpret_cast<uint2 *>(codes + (int64_t(row) * units + at) * 8) = nv_codes(v, bmax[j], g, s8);
            scale[scale_byte(row, at, tiles)] = uint8_t(s8);
            if (at == units - 1) pad_scales(scale, row, units, tiles);
        }
        copy_row<U>(raw, ahead);
    }
}
// A row held by a block.
template <typename T, int U>
__global__ void __launch_bounds__(kFp4RowWarps * 32, 1)
quant_nvfp4_block_kernel(const T *in, uint8_t *codes, uint8_t *scale, float *row_scale, int units, int tiles) {
    __shared__ uint32_t shared[kFp4RowWarps];
    dependency_wait();
    const int lane = threadIdx.x, lanes = blockDim.x;
    const int64_t row = blockIdx.x;
    uint32_t raw[U][8], bmax[U], amax = 0;
    load_row<U>(in, row, units, units, lane, lanes, raw);
#pragma unroll
    for (int j = 0; j < U; ++j) {
        float2 v[8];
        unpack16<T>(raw[j], v);
        bmax[j] = max_bits16(v);
        amax = max(amax, bmax[j]);
    }
    const float g = nv_row_scale(row_max(amax, shared));
    if (lane == 0) row_scale[row] = g;
#pragma unroll
    for (int j = 0; j < U; ++j) {
        const int at = lane + j * lanes;
        if (at >= units) break;
        float2 v[8];
        unpack16<T>(raw[j], v);
        uint32_t s8;
        *reinterpret_cast<uint2 *>(codes + (row * units + at) * 8) = nv_codes(v, bmax[j], g, s8);
        scale[scale_byte(row, at, tiles)] = uint8_t(s8);
        if (at == units - 1) pad_scales(scale, row, units, tiles);
    }
}

// Norms around a block. Per row, with r(v) = 1 / sqrt(mean(v^2) + eps):
//     y = round16(alpha * residual + gate * ((x * r(x)) * w_post))          the new residual stream
//     h = (y * r(y)) * w_pre                                                 the next block's input
// every product and sum rounded to f32 on its own, in this order. The means are taken in 64 bits and r is
// rounded once to f32: what is quantised behind them lies next to borders, and like this the result depends on
// the values alone, not on how a row is spread over lanes. One Newton step from the hardware's reciprocal root r, with 1 - a r^2 in 64
// bits, leaves a relative error of 1e-13 before that rounding.
// Bound by instructions: [32000, 512] to mxfp4 21.3 us (16.4 at the copy rate). With a warp per row it was 23.2 us and some 450 instructions per row;
// without any access to memory 19.7, without the 64-bit sums as well 13.7. Rows brought ahead by bulk copies into shared memory instead of registers: 24.8.
// Squares exact in 32 bits and moved to 64 by a shift of their bits instead of conversions: 22.4 -> 26.2.
__device__ __forceinline__ float inv_rms(double sum, double inv_n, double eps) {
    const double a = fma(sum, inv_n, eps);
    const float f = float(a);
    if (!(f > 1e-37f && f < 1e38f)) return float(1.0 / sqrt(a));  // no f32 holds it: rows of very large or very small bf16 values, NaN
    float r;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(f));
    const double d = double(r);
    return fmaf(r, 0.5f * float(fma(-a * d, d, 1.0)), r);
}

struct RmsnormBlockDev {
    const void *x, *residual, *w_post, *gate, *w_pre;
    void *residual_out, *out;
    uint8_t *scale;
    float *row_scale;
    int rows, units, tiles, seqlen;
    float alpha, eps;
};

// A unit of a weight vector, which stays in L1.
template <typename T>
__device__ __forceinline__ void load_weight(const void *w, int64_t at, uint32_t (&r)[8]) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "l"(static_cast<const T *>(w) + at * 16) : "memory");
}
// Adds the squares of a unit to four sums (one chain of 64-bit additions after the other would take longer than the loads).
template <typename T>
__device__ __forceinline__ void add_squares(const uint32_t (&raw)[8], double (&s)[4]) {
    float2 v[8];
    unpack16<T>(raw, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        s[2 * (i & 1)] = fma(double(v[i].x), double(v[i].x), s[2 * (i & 1)]);
        s[2 * (i & 1) + 1] = fma(double(v[i].y), double(v[i].y), s[2 * (i & 1) + 1]);
    }
}

// What both forms of the norms do with a unit. y = round16(alpha res + gate ((x rx) post)); the stream's unit replaces x.
template <typename T>
__device__ __forceinline__ void stream_unit(uint32_t (&x)[8], const uint32_t (&res)[8], bool normed, float rx, const float2 (&post)[8], bool gated,
                                            const float2 (&gate)[8], float alpha) {
    float2 v[8], r[8];
    unpack16<T>(x, v);
    unpack16<T>(res, r);
    if (normed)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = mul2(mul2(v[i], make_float2(rx, rx)), post[i]);
    if (gated)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = mul2(gate[i], v[i]);
    const float2 one = make_float2(1.f, 1.f), a2 = make_float2(alpha, alpha);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = pack2(fma2(mul2(a2, r[i]), one, v[i]), T());
}
// h = (y ry) pre
template <typename T>
__device__ __forceinline__ void normed_unit(const uint32_t (&y)[8], float ry, const float2 (&pre)[8], float2 (&h)[8]) {
    unpack16<T>(y, h);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = mul2(mul2(h[i], make_float2(ry, ry)), pre[i]);
}
// Writes unit `at` of the next block's input; all lanes of a warp come here (MX: the pair of lanes that shares a block), `in` is whether
// the unit is one of the row.
template <typename T, int OUT>
__device__ __forceinline__ void write_unit(const RmsnormBlockDev &p, int64_t row, int at, int units, int tiles, bool in, const float2 (&h)[8],
                                           uint32_t bmax, float g) {
    if constexpr (OUT == kFp4Plain) {
        if (!in) return;
        uint32_t r[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = pack2(h[i], T());
        store32(static_cast<T *>(p.out) + (row * units + at) * 16, r);
    } else {
        uint8_t *codes = static_cast<uint8_t *>(p.out) + (row * units + at) * 8;
        if constexpr (OUT == kFp4Mx) {
            uint32_t m = in ? max_bits16(h) : 0;
            m = max(m, __shfl_xor_sync(kFull, m, 1));
            if (!in) return;
            const uint32_t e = mx_exponent(m);
            *reinterpret_cast<uint2 *>(codes) = mx_codes(h, e);
            if ((at & 1) == 0) p.scale[scale_byte(row, at >> 1, tiles)] = uint8_t(e);
            if (at == units - 1) pad_scales(p.scale, row, units >> 1, tiles);
        } else {
            if (!in) return;
            uint32_t s8;
            *reinterpret_cast<uint2 *>(codes) = nv_codes(h, bmax, g, s8);
            p.scale[scale_byte(row, at, tiles)] = uint8_t(s8);
            if (at == units - 1) pad_scales(p.scale, row, units, tiles);
        }
    }
}

// Rows of up to 2048 values: LANES lanes (half a warp or one) hold a row, lane l units l, l + LANES, ... (U of them), and a block's warps walk
// rows. The weights that all rows share lie in shared memory as f32, which saves a conversion per value and row. FULL: rows of exactly
// LANES * U units, where no lane has to ask for its end. The next rows are asked for while these are computed with two units per lane (us,
// with : without: [32000, 512] to mxfp4 21.3 : 23.8, [9331, 1024] 13.2 : 14.2; one unit [16384, 256] 7.1 : 6.6, whose registers carry six blocks without),
// and behind the other loads: a use of those waits for every load in front of it. At 128 registers (four blocks) forms of four units and some of two spill up to 14.
template <typename T, int OUT, int LANES, int U, bool FULL>
__global__ void __launch_bounds__(kFp4NormWarps * 32, U == 1 ? 6 : 4)
rmsnorm_rows_kernel(const RmsnormBlockDev p) {
    constexpr bool kAhead = U == 2;
    constexpr int kGroups = 32 / LANES;   // rows of a warp at a time
    // unit u's four pieces of four values are `units` pieces apart: lanes that read the same piece of neighbouring units meet no bank twice
    extern __shared__ float4 weights[];
    const int units = FULL ? LANES * U : p.units, tiles = !FULL ? p.tiles : OUT == kFp4Mx ? (units / 2 + 3) / 4 : (units + 3) / 4;
    const bool own_gate = p.gate && p.seqlen > 0;
    float4 *const post = weights, *const gate = weights + 4 * units, *const pre = weights + 8 * units;
    dependency_wait();
    for (int w = 0; w < 3; ++w) {
        const void *src = w == 0 ? p.w_post : w == 1 ? (own_gate ? nullptr : p.gate) : OUT != kFp4None ? p.w_pre : nullptr;
        if (src)
            for (int u = threadIdx.x; u < units; u += kFp4NormWarps * 32) {
                uint32_t raw[8];
                float2 v[8];
                load_weight<T>(src, u, raw);
                unpack16<T>(raw, v);
#pragma unroll
                for (int c = 0; c < 4; ++c) weights[(w * 4 + c) * units + u] = make_float4(v[2 * c].x, v[2 * c].y, v[2 * c + 1].x, v[2 * c + 1].y);
            }
    }
    __syncthreads();
    auto weight = [&](const float4 *w, int at, float2 (&v)[8]) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float4 q = w[c * units + at];
            v[2 * c] = make_float2(q.x, q.y);
            v[2 * c + 1] = make_float2(q.z, q.w);
        }
    };
    const int lane = threadIdx.x & (LANES - 1), group = (threadIdx.x & 31) / LANES;
    const double inv_n = 1.0 / (double(units) * 16.0), eps = double(p.eps);
    auto sum_of = [&](const double (&s)[4]) {
        double t = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
        for (int d = LANES / 2; d > 0; d >>= 1) t += __shfl_xor_sync(kFull, t, d);
        return t;
    };
    const int step = int(gridDim.x) * kFp4NormWarps * kGroups;
    uint32_t x[U][8], res[U][8], x_ahead[kAhead ? U : 1][8], res_ahead[kAhead ? U : 1][8];
    // `first` is the row of the warp's first group: the loop is the same for all lanes, rows behind the last are zeros and not written
    int first = (int(blockIdx.x) * kFp4NormWarps + (int(threadIdx.x) >> 5)) * kGroups;
    auto load = [&](int row, auto &a, auto &b) {
        const int have = row < p.rows ? units : 0;
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int at = lane + j * LANES;
            if (FULL ? row < p.rows : at < have) {
                load32(static_cast<const T *>(p.x) + (int64_t(row) * units + at) * 16, a[j]);
                load32(static_cast<const T *>(p.residual) + (int64_t(row) * units + at) * 16, b[j]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) a[j][i] = b[j][i] = 0;
            }
        }
    };
    if (kAhead && first < p.rows) load(first + group, x, res);
    for (; first < p.rows; first += step) {
        const int row = first + group;
        const bool live = row < p.rows;
        if constexpr (!kAhead) load(row, x, res);
        const int64_t gate_at = own_gate && live ? int64_t(row / p.seqlen) * units : 0;
        float rx = 1.f;
        if (p.w_post) {
            double s[4] = {};
#pragma unroll
            for (int j = 0; j < U; ++j) add_squares<T>(x[j], s);
            rx = inv_rms(sum_of(s), inv_n, eps);
        }
        double s[4] = {};
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int at = lane + j * LANES;
            const bool in = FULL ? live : live && at < units;
            const int safe = FULL || at < units ? at : 0;
            float2 wp[8], wg[8];
            if (p.w_post) weight(post, safe, wp);
            if (own_gate) {
                uint32_t raw[8];
                load_weight<T>(p.gate, gate_at + safe, raw);
                unpack16<T>(raw, wg);
            } else if (p.gate) {
                weight(gate, safe, wg);
            }
            stream_unit<T>(x[j], res[j], p.w_post != nullptr, rx, wp, p.gate != nullptr, wg, p.alpha);
            if (!FULL && at >= units)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[j][i] = 0;
            if (in) store32(static_cast<T *>(p.residual_out) + (int64_t(row) * units + at) * 16, x[j]);
            if constexpr (OUT != kFp4None) add_squares<T>(x[j], s);
        }
        if constexpr (kAhead)
            if (first + step < p.rows) load(row + step, x_ahead, res_ahead);
        if constexpr (OUT != kFp4None) {
            const float ry = inv_rms(sum_of(s), inv_n, eps);
            float2 h[8], wn[8];
            uint32_t bmax[U], amax = 0;
            float g = 1.f;
            auto unit = [&](int j) {
                const int at = lane + j * LANES;
                weight(pre, FULL || at < units ? at : 0, wn);
                normed_unit<T>(x[j], ry, wn, h);
            };
            if constexpr (OUT == kFp4Nv) {
#pragma unroll
                for (int j = 0; j < U; ++j) {
                    unit(j);
                    bmax[j] = FULL || lane + j * LANES < units ? max_bits16(h) : 0;
                    amax = max(amax, bmax[j]);
                }
                amax = __reduce_max_sync(LANES == 32 ? kFull : 0xFFFFu << (threadIdx.x & 16), amax);
                g = nv_row_scale(amax);
                if (lane == 0 && live) p.row_scale[row] = g;
            }
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int at = lane + j * LANES;
                if (OUT != kFp4Nv || U > 1) unit(j);
                write_unit<T, OUT>(p, row, at, units, tiles, FULL ? live : live && at < units, h, OUT == kFp4Nv ? bmax[j] : 0, g);
            }
        }
        if constexpr (kAhead) {
            copy_row<U>(x, x_ahead);
            copy_row<U>(res, res_ahead);
        }
    }
}

// A row held by a block: few rows, or more than 2048 values.
template <typename T, int OUT, int U>
__global__ void __launch_bounds__(kFp4RowWarps * 32, 1)
rmsnorm_block_kernel(const RmsnormBlockDev p) {
    __shared__ double sums[2][kFp4RowWarps];
    __shared__ uint32_t maxima[kFp4RowWarps];
    dependency_wait();
    const int lanes = blockDim.x, lane = threadIdx.x, units = p.units;
    const int64_t row = blockIdx.x;
    const double inv_n = 1.0 / (double(units) * 16.0), eps = double(p.eps);
    uint32_t x[U][8], res[U][8], post[U][8], gate[U][8], pre[U][8];
    load_row<U>(p.x, row, units, units, lane, lanes, x);
    load_row<U>(p.residual, row, units, units, lane, lanes, res);
    const int64_t gate_at = p.seqlen > 0 ? row / p.seqlen * units : 0;
    auto weights = [&](const void *w, int64_t base, uint32_t (&raw)[U][8]) {
#pragma unroll
        for (int j = 0; j < U; ++j) load_weight<T>(w, base + min(lane + j * lanes, units - 1), raw[j]);
    };
    if (p.w_post) weights(p.w_post, 0, post);
    if (p.gate) weights(p.gate, gate_at, gate);
    if constexpr (OUT != kFp4None) weights(p.w_pre, 0, pre);
    float rx = 1.f;
    if (p.w_post) {
        double s[4] = {};
#pragma unroll
        for (int j = 0; j < U; ++j) add_squares<T>(x[j], s);
        rx = inv_rms(row_sum((s[0] + s[1]) + (s[2] + s[3]), sums[0]), inv_n, eps);
    }
    double s[4] = {};
#pragma unroll
    for (int j = 0; j < U; ++j) {
        const int at = lane + j * lanes;
        if (at >= units) break;
        float2 wp[8], wg[8];
        if (p.w_post) unpack16<T>(post[j], wp);
        if (p.gate) unpack16<T>(gate[j], wg);
        stream_unit<T>(x[j], res[j], p.w_post != nullptr, rx, wp, p.gate != nullptr, wg, p.alpha);
        store32(static_cast<T *>(p.residual_out) + (row * units + at) * 16, x[j]);
        if constexpr (OUT != kFp4None) add_squares<T>(x[j], s);
    }
    if constexpr (OUT != kFp4None) {
        const float ry = inv_rms(row_sum((s[0] + s[1]) + (s[2] + s[3]), sums[1]), inv_n, eps);
        float2 h[U][8];
        uint32_t bmax[U], amax = 0;
        float g = 1.f;
#pragma unroll
        for (int j = 0; j < U; ++j) {
            float2 wn[8];
            unpack16<T>(pre[j], wn);
            normed_unit<T>(x[j], ry, wn, h[j]);
            bmax[j] = lane + j * lanes < units ? max_bits16(h[j]) : 0;
            amax = max(amax, bmax[j]);
        }
        if constexpr (OUT == kFp4Nv) {
            g = nv_row_scale(row_max(amax, maxima));
            if (lane == 0) p.row_scale[row] = g;
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int at = lane + j * lanes;
            write_unit<T, OUT>(p, row, at, units, p.tiles, at < units, h[j], bmax[j], g);
        }
    }
}

// Blocks of `kernel` that the device holds at once.
inline int resident_blocks(const void *kernel, int block, int smem = 0) {
    struct Seen { const void *kernel; int dev, smem, blocks; };
    static thread_local Seen seen[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    Seen &s = seen[(reinterpret_cast<uintptr_t>(kernel) >> 4) & 63];
    if (s.kernel != kernel || s.dev != dev || s.smem != smem) {
        int per_sm = 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, block, smem) != cudaSuccess || per_sm < 1) {
            cudaGetLastError();
            return device_sm_count();   // one per SM; the next call asks again
        }
        s = {kernel, dev, smem, per_sm * device_sm_count()};
    }
    return s.blocks;
}
template <typename T, int LANES, int U>
int launch_quant_nvfp4_rows(const T *in, uint8_t *codes, uint8_t *scale, float *row_scale, int rows, int units, cudaStream_t stream) {
    constexpr auto kernel = quant_nvfp4_rows_kernel<T, LANES, U>;
    constexpr int kBlock = kFp4WalkWarps * 32, kRows = kFp4WalkWarps * 32 / LANES;
    const int blocks = (rows + kRows - 1) / kRows, most = resident_blocks(reinterpret_cast<const void *>(kernel), kBlock);
    return launch_dependent(kernel, blocks < most ? blocks : most, kBlock, 0, stream, in, codes, scale, row_scale, rows, units, (units + 3) / 4);
}
template <typename T, int U>
int launch_quant_nvfp4_block(const T *in, uint8_t *codes, uint8_t *scale, float *row_scale, int rows, int units, cudaStream_t stream) {
    return launch_dependent(quant_nvfp4_block_kernel<T, U>, rows, (units + 32 * U - 1) / (32 * U) * 32, 0, stream, in, codes, scale, row_scale, units,
                            (units + 3) / 4);
}
// Few rows: a block each, as many warps as the row has units for. Else half a warp per row up to 768 values, a warp up to 2048, and a block of warps
// with two units per lane, from 4096 values on four ([4096, 4096] two : four 10.2 : 11.3 us, [1024, 16384] 15.7 : 12.1).
template <typename T>
int launch_quant_nvfp4(const T *in, uint8_t *codes, uint8_t *scale, float *row_scale, int rows, int units, cudaStream_t s) {
    const bool few = rows < 4 * device_sm_count();
    if (few && units > 16 && units <= 32 * kFp4RowWarps) return launch_quant_nvfp4_block<T, 1>(in, codes, scale, row_scale, rows, units, s);
    if (units > 256) return launch_quant_nvfp4_block<T, 4>(in, codes, scale, row_scale, rows, units, s);
    if (units > 128) return launch_quant_nvfp4_block<T, 2>(in, codes, scale, row_scale, rows, units, s);
    if (units <= 16) return launch_quant_nvfp4_rows<T, 16, 1>(in, codes, scale, row_scale, rows, units, s);
    if (units <= 32) return launch_quant_nvfp4_rows<T, 16, 2>(in, codes, scale, row_scale, rows, units, s);
    if (units <= 48) return launch_quant_nvfp4_rows<T, 16, 3>(in, codes, scale, row_scale, rows, units, s);
    if (units <= 64) return launch_quant_nvfp4_rows<T, 32, 2>(in, codes, scale, row_scale, rows, units, s);
    if (units <= 96) return launch_quant_nvfp4_rows<T, 32, 3>(in, codes, scale, row_scale, rows, units, s);
    return launch_quant_nvfp4_rows<T, 32, 4>(in, codes, scale, row_scale, rows, units, s);
}

template <typename T, int OUT, int LANES, int U, bool FULL>
int launch_rmsnorm_rows(const RmsnormBlockDev &p, cudaStream_t stream) {
    constexpr auto kernel = rmsnorm_rows_kernel<T, OUT, LANES, U, FULL>;
    const int smem = 12 * p.units * int(sizeof(float4)), block = kFp4NormWarps * 32;
    constexpr int kRows = kFp4NormWarps * 32 / LANES;
    const int blocks = (p.rows + kRows - 1) / kRows, most = resident_blocks(reinterpret_cast<const void *>(kernel), block, smem);
    return launch_dependent(kernel, blocks < most ? blocks : most, block, smem, stream, p);
}
template <typename T, int OUT, int LANES, int U>
int launch_rmsnorm_rows(const RmsnormBlockDev &p, cudaStream_t stream) {
    return p.units == LANES * U ? launch_rmsnorm_rows<T, OUT, LANES, U, true>(p, stream) : launch_rmsnorm_rows<T, OUT, LANES, U, false>(p, stream);
}
// Few rows: a block each, as many warps as the row has units for. Else half a warp per row up to 768 values (a sum over 16 lanes serves two rows at
// once), a warp up to 2048, and a block of warps with two units per lane beyond.
template <typename T, int OUT>
int launch_rmsnorm_block(const RmsnormBlockDev &p, cudaStream_t stream) {
    const int units = p.units;
    const bool few = p.rows < 4 * device_sm_count();
    if (units > 128 || (few && units > 16)) {
        const int each = !few || units > 32 * kFp4RowWarps ? 2 : 1, warps = (units + 32 * each - 1) / (32 * each);
        return launch_dependent(each == 1 ? rmsnorm_block_kernel<T, OUT, 1> : rmsnorm_block_kernel<T, OUT, 2>, p.rows, warps * 32, 0, stream, p);
    }
    if (units <= 16) return launch_rmsnorm_rows<T, OUT, 16, 1>(p, stream);
    if (units <= 32) return launch_rmsnorm_rows<T, OUT, 16, 2>(p, stream);
    if (units <= 48) return launch_rmsnorm_rows<T, OUT, 16, 3>(p, stream);
    if (units <= 64) return launch_rmsnorm_rows<T, OUT, 32, 2>(p, stream);
    if (units <= 96) return launch_rmsnorm_rows<T, OUT, 32, 3>(p, stream);
    return launch_rmsnorm_rows<T, OUT, 32, 4>(p, stream);
}
template <typename T>
int launch_rmsnorm_block(const RmsnormBlockDev &p, int out, cudaStream_t stream) {
    switch (out) {
        case kFp4Plain: return launch_rmsnorm_block<T, kFp4Plain>(p, stream);
        case kFp4Mx: return launch_rmsnorm_block<T, kFp4Mx>(p, stream);
        case kFp4Nv: return launch_rmsnorm_block<T, kFp4Nv>(p, stream);
        default: return launch_rmsnorm_block<T, kFp4None>(p, stream);
    }
}

// Sizes and addresses that every kernel here needs: rows of whole blocks (and of whole 16-byte pieces as codes, which the
// products ask for), 16-bit tensors on 32 bytes, codes and scales on 16.
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool aligned4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
// kFp4MaxSize: the next tile's end and a grid's step from the last row still fit 32 bits.
constexpr int kFp4MaxSize = INT32_MAX - (1 << 20);
inline bool fp4_shape_ok(int rows, int cols) { return rows >= 0 && rows <= kFp4MaxSize && cols >= 32 && cols <= kFp4MaxSize && cols % 32 == 0; }
// Kernels whose thread is a unit count units in 32 bits: launch(first row, rows) for runs of rows of at most INT32_MAX units (one run, as a rule).
template <typename F>
int in_row_runs(int rows, int units, F launch) {
    const int most = INT32_MAX / units;
    for (int row = 0; row < rows;) {
        const int n = rows - row < most ? rows - row : most, rc = launch(row, n);
        if (rc) return rc;
        row += n;
    }
    return 0;
}
inline int unit_blocks(int rows, int units) { return int((int64_t(rows) * units + 255) / 256); }
inline int fp4_tiles(int cols, int format) { return (cols / (format == FLUKE_SM100_FP4_MX ? 32 : 16) + 3) / 4; }

}  // namespace
}  // namespace fluke_sm100

using namespace fluke_sm100;

extern "C" int fluke_sm100_quant_fp4(const void *in, void *codes, void *scale, void *row_scale, int rows, int cols, int format, int bf16,
                                     void *stream) {
    if (!fp4_shape_ok(rows, cols) || (format == FLUKE_SM100_FP4_NV && cols > FLUKE_SM100_FP4_MAX_ROW)) return (int)cudaErrorInvalidValue;
    if (rows == 0) return 0;
    if (!in || !codes || !scale || (format == FLUKE_SM100_FP4_NV && !row_scale)) return (int)cudaErrorInvalidValue;
    if (!aligned32(in) || !aligned16(codes) || !aligned16(scale) || (format == FLUKE_SM100_FP4_NV && !aligned4(row_scale))) return (int)cudaErrorMisalignedAddress;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int units = cols / 16;
    if (format == FLUKE_SM100_FP4_NV) {
        uint8_t *c = static_cast<uint8_t *>(codes), *b = static_cast<uint8_t *>(scale);
        float *r = static_cast<float *>(row_scale);
        return bf16 ? launch_quant_nvfp4(static_cast<const __nv_bfloat16 *>(in), c, b, r, rows, units, s)
                    : launch_quant_nvfp4(static_cast<const __half *>(in), c, b, r, rows, units, s);
    }
    if (format != FLUKE_SM100_FP4_MX) return (int)cudaErrorInvalidValue;
    const int tiles = fp4_tiles(cols, format);
    return in_row_runs(rows, units, [&](int row0, int n) {
        auto run = [&](auto *x) {
            using T = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
            return launch_dependent(quant_mxfp4_kernel<T>, unit_blocks(n, units), 256, 0, s, x + int64_t(row0) * cols,
                                    static_cast<uint8_t *>(codes) + int64_t(row0) * (cols / 2), static_cast<uint8_t *>(scale), uint32_t(n) * uint32_t(units),
                                    uint32_t(units), tiles, uint32_t(row0));
        };
        return bf16 ? run(static_cast<const __nv_bfloat16 *>(in)) : run(static_cast<const __half *>(in));
    });
}

extern "C" int fluke_sm100_dequant_fp4(const void *codes, const void *scale, const void *row_scale, void *out, int rows, int cols, int format,
                                       int bf16, void *stream) {
    if (!fp4_shape_ok(rows, cols) || (format != FLUKE_SM100_FP4_MX && format != FLUKE_SM100_FP4_NV)) return (int)cudaErrorInvalidValue;
    if (rows == 0) return 0;
    if (!out || !codes || !scale || (format == FLUKE_SM100_FP4_NV && !row_scale)) return (int)cudaErrorInvalidValue;
    if (!aligned32(out) || !aligned16(codes) || !aligned16(scale) || (format == FLUKE_SM100_FP4_NV && !aligned4(row_scale))) return (int)cudaErrorMisalignedAddress;
    const bool mx = format == FLUKE_SM100_FP4_MX;
    const int units = cols / 16;
    return in_row_runs(rows, units, [&](int row0, int n) {
        auto run = [&](auto *o) {
            using T = std::remove_pointer_t<decltype(o)>;
            return launch_dependent(mx ? dequant_fp4_kernel<T, true> : dequant_fp4_kernel<T, false>, unit_blocks(n, units), 256, 0,
                                    static_cast<cudaStream_t>(stream), static_cast<const uint8_t *>(codes) + int64_t(row0) * (cols / 2),
                                    static_cast<const uint8_t *>(scale), mx ? nullptr : static_cast<const float *>(row_scale) + row0, o + int64_t(row0) * cols,
                                    uint32_t(n) * uint32_t(units), uint32_t(units), fp4_tiles(cols, format), uint32_t(row0));
        };
        return bf16 ? run(static_cast<__nv_bfloat16 *>(out)) : run(static_cast<__half *>(out));
    });
}

extern "C" int fluke_sm100_rmsnorm_block(const fluke_sm100_rmsnorm_block_t *b, void *stream) {
    if (!b || !fp4_shape_ok(b->rows, b->cols) || b->cols > FLUKE_SM100_FP4_MAX_ROW || b->seqlen < 0) return (int)cudaErrorInvalidValue;
    if (b->out_format < kFp4Plain || b->out_format > kFp4None) return (int)cudaErrorInvalidValue;
    if (b->rows == 0) return 0;
    const bool quant = b->out_format == kFp4Mx || b->out_format == kFp4Nv;
    if (!b->x || !b->residual || !b->residual_out) return (int)cudaErrorInvalidValue;
    if (b->out_format != kFp4None && (!b->w_pre || !b->out)) return (int)cudaErrorInvalidValue;
    if ((quant && !b->scale) || (b->out_format == kFp4Nv && !b->row_scale)) return (int)cudaErrorInvalidValue;
    if (!aligned32(b->x, b->residual, b->residual_out, quant ? nullptr : b->out) || (quant && !(aligned16(b->out) && aligned16(b->scale))) ||
        !aligned32(b->w_post, b->gate, b->w_pre) || (b->out_format == kFp4Nv && !aligned4(b->row_scale)))
        return (int)cudaErrorMisalignedAddress;
    // A row is read before it is written, but rows come in any order: the stream and a 16-bit result lie where x or the residual of the same rows does, or apart
    // from everything; what all rows read, and scales, lie apart from everything.
    const uint64_t row_bytes = uint64_t(b->cols) * 2, bytes = b->rows * row_bytes, out_bytes = b->out_format == kFp4None ? 0 : quant ? bytes / 4 : bytes;
    const uint64_t gates = b->seqlen > 0 ? (uint64_t(b->rows) + b->seqlen - 1) / b->seqlen : 1;
    const uint64_t scale_bytes = quant ? (uint64_t(b->rows) + 127) / 128 * fp4_tiles(b->cols, b->out_format) * 512 : 0;
    struct Range { const void *at; uint64_t n; };
    auto apart = [](Range a, Range c) {
        const uint64_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(c.at);
        return a.n == 0 || c.n == 0 || x + a.n <= y || y + c.n <= x;
    };
    const Range in[] = {{b->x, bytes}, {b->residual, bytes}, {b->w_post, b->w_post ? row_bytes : 0}, {b->gate, b->gate ? gates * row_bytes : 0},
                        {b->w_pre, b->out_format != kFp4None ? row_bytes : 0}};
    const Range out[] = {{b->residual_out, bytes}, {b->out, out_bytes}, {b->scale, scale_bytes}, {b->row_scale, b->out_format == kFp4Nv ? uint64_t(b->rows) * 4 : 0}};
    for (int o = 0; o < 4; ++o) {
        for (int i = 0; i < 5; ++i) {
            const bool in_place = i < 2 && out[o].at == in[i].at && (o == 0 || (o == 1 && !quant));
            if (!in_place && !apart(out[o], in[i])) return (int)cudaErrorInvalidValue;
        }
        for (int other = 0; other < o; ++other)
            if (!apart(out[o], out[other])) return (int)cudaErrorInvalidValue;
    }
    RmsnormBlockDev p;
    p.x = b->x; p.residual = b->residual; p.w_post = b->w_post; p.gate = b->gate; p.w_pre = b->w_pre;
    p.residual_out = b->residual_out; p.out = b->out;
    p.scale = static_cast<uint8_t *>(b->scale); p.row_scale = b->row_scale;
    p.rows = b->rows; p.units = b->cols / 16; p.seqlen = b->gate ? b->seqlen : 0;
    p.tiles = b->out_format == kFp4Mx ? fp4_tiles(b->cols, FLUKE_SM100_FP4_MX) : fp4_tiles(b->cols, FLUKE_SM100_FP4_NV);
    p.alpha = b->alpha; p.eps = b->eps;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return b->bf16 ? launch_rmsnorm_block<__nv_bfloat16>(p, b->out_format, s) : launch_rmsnorm_block<__half>(p, b->out_format, s);
}

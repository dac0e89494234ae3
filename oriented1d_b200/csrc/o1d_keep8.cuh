// Activation checkpoints in 8 bits, and the GELU and LayerNorm passes that write and read them.
//
// A row of C values is cut into groups of 128 columns (the last may be shorter).  With lo and hi the least and
// greatest value of a group, s = (hi - lo) * (1/255) and q = round((v - lo) * (1/s)), all in fp32 and each operation
// rounded on its own, so that a checkpoint's bits follow from its values alone; q stands for lo + q*s, which is at most
// s/2 (and a rounding) away from v.  A group of equal values, or one whose step is below the normal numbers, has s = 0
// and stands for lo.  A group that holds a NaN or an infinity, or whose range overflows, has s = NaN: everything
// read back from it is NaN.  Kept per row: C bytes of codes, two floats a group: 1.06 bytes a value.
//
// Why lo/hi and not the largest magnitude: an activation's argument is rarely centred, and this step is never the wider.
// Why 128: the two floats cost 6 % there (12 % at 64), and a group is what one warp holds with a vector a lane.
#pragma once

#include "o1d_common.cuh"
#include "o1d_keep8.h"
#include "o1d_pair.cuh"

namespace o1d {

constexpr int kKeepThreads = 256;
constexpr int kKeepWarps = kKeepThreads / 32;
constexpr int kKeepLane = 8;             // values of a vector: 16 bytes of bf16

__device__ __forceinline__ float min_nan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float min_nan(float a, float b, float c) { float r; asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }
__device__ __forceinline__ float max_nan(float a, float b, float c) { float r; asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }

// Sums over the L lanes that share something, for U of them at once.
template <int L, int U>
__device__ __forceinline__ void lane_sums(float (&v)[U]) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1)
#pragma unroll
        for (int u = 0; u < U; u++) v[u] += __shfl_xor_sync(0xffffffffu, v[u], o);
}

// Exact GELU and its slope without erff, of which the passes below would be nothing else (20 instructions a value each).
//   P(-|h|) = erfc(z)/2,  z = |h|/sqrt 2,  erfc(z) = t q(t) exp(-z^2),  t = 1/(1 + 0.33 z)
// the form of Abramowitz and Stegun 7.1.26, with a polynomial q fitted to exp(z^2) erfc(z) on 0 <= z <= 10 by iterated weighted
// least squares: of degree 7 for bf16 (relative error 1e-7, in the tail too), of degree 9 for fp32 (5e-9, its mean 1e-9; an error of
// the fit is alike for like values, and the bias gradient adds them up).  These are the errors of the numbers below: 0.33 / sqrt 2 was
// rounded to fp32 before the fit, and the coefficients one after the other, the others fitted anew each time (all at once: 3.5e-8,
// nearly all of one sign).  One reciprocal and one exponential, which the slope needs anyway.
// For a pair of values: m = |h| (at most 64), q = -P(-|h|), bell = exp(-h^2/2).  Then GELU(h) = max(h, 0) + m q and
// GELU'(h) = 1/2 + sign(h) (1/2 + q + m bell / sqrt(2 pi)).
struct Normal { F2 m, q, bell; };
template <bool FP32>
__device__ __forceinline__ Normal normal_of(F2 h) {
    constexpr int N = FP32 ? 10 : 8;
    constexpr float slope = 0.23334524035453796f;        // 0.33 / sqrt 2
    constexpr float fit[10] = {FP32 ? 0.1861456036567688f : 0.1863577961921692f,
                               FP32 ? 0.18700088560581207f : 0.18295611441135406f,
                               FP32 ? 0.16811716556549072f : 0.2012227475643158f,
                               FP32 ? 0.1999654918909073f : 0.047224510461091995f,
                               FP32 ? -0.02961677871644497f : 0.4084925055503845f,
                               FP32 ? 0.45998188853263855f : -0.3511412739753723f,
                               FP32 ? -0.5105260610580444f : 0.4602320194244385f,
                               FP32 ? 0.5900679230690002f : -0.13534443080425262f,
                               FP32 ? -0.30766230821609497f : 0.f,
                               FP32 ? 0.05652618780732155f : 0.f};
    const float2 a = apart(h);
    const F2 m = two(fminf(fabsf(a.x), 64.f), fminf(fabsf(a.y), 64.f));      // (q is 0 there: an infinity times it would be NaN)
    const float2 d = apart(fma2(m, both(slope), both(1.f))), z = apart(mul2(mul2(h, h), both(-0.72134752f)));
    float2 r, e;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(d.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(d.y));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(z.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(z.y));
    const F2 t = two(r.x, r.y), bell = two(e.x, e.y);
    F2 q = both(-0.5f * fit[N - 1]);
#pragma unroll
    for (int i = N - 2; i >= 0; i--) q = fma2(t, q, both(-0.5f * fit[i]));
    return {m, mul2(q, mul2(t, bell)), bell};
}
__device__ __forceinline__ F2 gelu_of(F2 h, const Normal &n) {
    const float2 a = apart(h);
    return fma2(n.m, n.q, two(fmaxf(a.x, 0.f), fmaxf(a.y, 0.f)));            // (NaN comes back through q)
}
__device__ __forceinline__ F2 gelu_slope(F2 h, const Normal &n) {
    const float2 a = apart(h), w = apart(add2(fma2(mul2(n.m, both(0.3989422804014327f)), n.bell, n.q), both(0.5f)));
    return add2(two(__uint_as_float(__float_as_uint(w.x) ^ (__float_as_uint(a.x) & 0x80000000u)),
                    __uint_as_float(__float_as_uint(w.y) ^ (__float_as_uint(a.y) & 0x80000000u))), both(0.5f));
}

// A lane's eight values of a group of L lanes.  VEC: columns c .. c+7 (C % 8 == 0 and all aligned, so that all exist or
// none); otherwise columns c, c+L, ..., c+7L, one element each.  `at`: the address of column c; `end`: the columns of the row, or
// of its part, that exist.
template <bool VEC, int L> __device__ __forceinline__ int col_of(int c, int i) { return VEC ? c + i : c + i * L; }
template <bool VEC> __device__ __forceinline__ int first_col(int lane) { return VEC ? lane * kKeepLane : lane; }
// A lane has NV vectors of a group, L * 8 columns apart.  Lanes with more of a row need fewer exchanges to find its range and its sums.

__device__ __forceinline__ float from_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float from_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// A lane's eight values as they come from memory (bf16 vectors stay packed until they are used: half the registers in flight).
template <typename T, bool VEC> struct Raw8 { float f[8]; };
template <> struct Raw8<__nv_bfloat16, true> { uint4 v; };
template <bool VEC, int L, typename T>
__device__ __forceinline__ void load8(const T *at, int c, int end, Raw8<T, VEC> &r) {
    if constexpr (VEC && sizeof(T) == 2) {
        r.v = c < end ? __ldg(reinterpret_cast<const uint4 *>(at)) : make_uint4(0u, 0u, 0u, 0u);
    } else if constexpr (VEC) {
        const bool on = c < end;
        const float4 a = on ? __ldg(reinterpret_cast<const float4 *>(at)) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float4 b = on ? __ldg(reinterpret_cast<const float4 *>(at) + 1) : make_float4(0.f, 0.f, 0.f, 0.f);
        r.f[0] = a.x; r.f[1] = a.y; r.f[2] = a.z; r.f[3] = a.w; r.f[4] = b.x; r.f[5] = b.y; r.f[6] = b.z; r.f[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) r.f[i] = c + i * L < end ? ld(at + i * L) : 0.f;
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void unpack8(const Raw8<T, VEC> &r, F2 (&f)[4]) {
    if constexpr (VEC && sizeof(T) == 2) {
        f[0] = two(from_lo(r.v.x), from_hi(r.v.x)); f[1] = two(from_lo(r.v.y), from_hi(r.v.y));
        f[2] = two(from_lo(r.v.z), from_hi(r.v.z)); f[3] = two(from_lo(r.v.w), from_hi(r.v.w));
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = two(r.f[2 * i], r.f[2 * i + 1]);
    }
}
template <bool VEC, int L, typename T>
__device__ __forceinline__ void store8(T *at, int c, int end, const F2 (&v)[4]) {
    const float2 a = apart(v[0]), b = apart(v[1]), d = apart(v[2]), e = apart(v[3]);
    if constexpr (VEC) {
        if (c >= end) return;
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4 *>(at)[0] = make_float4(a.x, a.y, b.x, b.y);
            reinterpret_cast<float4 *>(at)[1] = make_float4(d.x, d.y, e.x, e.y);
        } else {
            const __nv_bfloat162 h[4] = {__float22bfloat162_rn(a), __float22bfloat162_rn(b), __float22bfloat162_rn(d), __float22bfloat162_rn(e)};
            *reinterpret_cast<uint4 *>(at) = *reinterpret_cast<const uint4 *>(h);
        }
    } else {
        const float f[8] = {a.x, a.y, b.x, b.y, d.x, d.y, e.x, e.y};
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (c + i * L < end) st(at + i * L, f[i]);
    }
}
// Parameters of the lane's columns (0 where there is none).
template <bool VEC, int L>
__device__ __forceinline__ void load_params(const void *p, int bf16, int c, int end, F2 (&v)[4]) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = p && col_of<VEC, L>(c, i) < end ? ld_param(p, col_of<VEC, L>(c, i), bf16) : 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = two(f[2 * i], f[2 * i + 1]);
}
// Codes travel as bytes and become numbers in the mantissa of 2^23 + q: integer conversions run at an eighth of the rate.
template <bool VEC, int L>
__device__ __forceinline__ uint2 load_codes(const uint8_t *at, int c, int end) {
    if constexpr (VEC) return c < end ? __ldg(reinterpret_cast<const uint2 *>(at)) : make_uint2(0u, 0u);
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (c + i * L < end) w[i >> 2] |= (uint32_t)__ldg(at + i * L) << (8 * (i & 3));
    return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void restore_codes(uint2 q, float2 range, F2 (&f)[4]) {
    const F2 step = both(range.y), lo = both(range.x);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w = i < 2 ? q.x : q.y;
        const F2 v = two(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7650 | (2 * i & 3))), __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7650 | ((2 * i + 1) & 3))));
        f[i] = fma2(add2(v, both(-8388608.f)), step, lo);
    }
}

// Codes of the lane's eight values and their group's range, for U groups at once (each step of the butterflies waits for the
// one before it, and shuffles stay in the order they are written in: one group after the other, those waits were what the
// kernels did).  end: 0 for a row that does not exist.
template <bool VEC, int L, int NV, int U>
__device__ __forceinline__ void keep_groups(const F2 (&f)[U][NV][4], const int (&c)[NV], const int (&end)[U], uint2 (&codes)[U][NV], float2 (&range)[U]) {
    const float none = __int_as_float(0x7f800000);
    const bool upper = threadIdx.x & (L / 2);
    float m[U], send[U], lo[U], inv[U], step[U];
    uint32_t mask[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        float least, most;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const float2 a = apart(f[u][j][0]), b = apart(f[u][j][1]), d = apart(f[u][j][2]), e = apart(f[u][j][3]);
            float l, h;
            if (VEC) {
                l = min_nan(min_nan(a.x, a.y, b.x), min_nan(b.y, d.x, d.y), min_nan(e.x, e.y));
                h = max_nan(max_nan(a.x, a.y, b.x), max_nan(b.y, d.x, d.y), max_nan(e.x, e.y));
                if (c[j] >= end[u]) { l = none; h = -none; }
            } else {
                const float v[8] = {a.x, a.y, b.x, b.y, d.x, d.y, e.x, e.y};
                l = none; h = -none;
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (c[j] + i * L < end[u]) { l = min_nan(l, v[i]); h = max_nan(h, v[i]); }
            }
            least = j ? min_nan(least, l) : l;
            most = j ? max_nan(most, h) : h;
        }
        // One butterfly finds both ends: the lanes of the upper half take over the (negated) greatest values, those of the
        // lower half the least ones, and the last exchange hands each the other's result.
        m[u] = upper ? -most : least;
        send[u] = upper ? least : -most;
    }
#pragma unroll
    for (int u = 0; u < U; u++) m[u] = min_nan(m[u], __shfl_xor_sync(0xffffffffu, send[u], L / 2));
#pragma unroll
    for (int o = L / 4; o > 0; o >>= 1)
#pragma unroll
        for (int u = 0; u < U; u++) m[u] = min_nan(m[u], __shfl_xor_sync(0xffffffffu, m[u], o));
#pragma unroll
    for (int u = 0; u < U; u++) send[u] = __shfl_xor_sync(0xffffffffu, m[u], L / 2);
#pragma unroll
    for (int u = 0; u < U; u++) {
        lo[u] = upper ? send[u] : m[u];
        const float hi = -(upper ? m[u] : send[u]);
        step[u] = __fmul_rn(__fsub_rn(hi, lo[u]), 1.f / 255.f);
        const bool lost = !(step[u] <= 3.402823466e38f), some = step[u] >= 1.175494351e-38f;        // (neither, either, not both)
        inv[u] = __frcp_rn(fmaxf(step[u], 1.175494351e-38f));
        inv[u] = some && !lost ? inv[u] : 0.f;
        step[u] = lost ? __int_as_float(0x7fffffff) : some ? step[u] : 0.f;
        mask[u] = lost ? 0u : 0xffffffffu;                            // a NaN or an infinity: the group is lost
        range[u] = make_float2(lo[u], step[u]);
    }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int j = 0; j < NV; j++) {
            uint32_t q[8];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                // 2^23 + t has round(t) in its lowest bits.  (Not a packed sum: the assembler makes one operation of a packed
                // product and the packed sum behind it, with one rounding, which on ties is another code.)
                const float2 t = apart(mul2(add2(f[u][j][i], both(-lo[u])), both(inv[u])));
                q[2 * i] = __float_as_uint(__fadd_rn(t.x, 8388608.f));
                q[2 * i + 1] = __float_as_uint(__fadd_rn(t.y, 8388608.f));
            }
            codes[u][j] = make_uint2(__byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410) & mask[u],
                                     __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410) & mask[u]);
        }
}
template <bool VEC, int L>
__device__ __forceinline__ void store_codes(uint8_t *row, int c, int end, uint2 q) {
    if constexpr (VEC) {
        if (c < end) *reinterpret_cast<uint2 *>(row) = q;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (c + i * L < end) row[i * L] = (uint8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
    }
}

// The elementwise kinds.  CTA (bx, by): the columns of group bx, blocks of UN * ROWS rows in steps of all the grid's; L lanes
// hold a row's part of the group, NV vectors each, 32/L rows a warp, UN rows of a lane are in flight at once.  Column sums of the GELU
// backward (its bias gradient) stay in registers over all rows of a thread and leave as one partial per (by, column),
// added in a fixed order by sum_slices_kernel.  Addresses are a base that the whole CTA shares plus an offset that never
// changes: as 64-bit products of row and column for every access they were half of all instructions.
template <int KIND, typename T, bool VEC, int L, int NV, int UN>
__global__ void __launch_bounds__(kKeepThreads)
keep_kernel(const KeepArgs a) {
    constexpr int RW = 32 / L, ROWS = kKeepWarps * RW;           // rows of a warp, of the CTA
    const int lane = threadIdx.x % L, sub = (threadIdx.x & 31) / L, warp = threadIdx.x >> 5;
    const int g = blockIdx.x, G = gridDim.x, C = a.C;
    const int c0 = g * kKeepGroup + first_col<VEC>(lane);
    const int lim = min(C, (g + 1) * kKeepGroup);                // end of the group
    const int my_row = warp * RW + sub;
    const unsigned off = (unsigned)my_row * (unsigned)C + (unsigned)c0, range_off = (unsigned)my_row * (unsigned)G + (unsigned)g;
    constexpr int NEXT = L * kKeepLane;                          // columns from one of a lane's vectors to the next
    int c[NV];
    F2 b[NV][4], sum[NV][4];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        c[j] = c0 + j * NEXT;
        if (KIND == KEEP_GELU_FWD) load_params<VEC, L>(a.bias, a.pbf16, c[j], lim, b[j]);
#pragma unroll
        for (int i = 0; i < 4; i++) sum[j][i] = both(0.f);
    }
    struct Rows {
        Raw8<T, VEC> raw[UN][NV];
        uint2 q[UN][NV];
        float2 range[UN];
    };
    // end of the row part of round r0, row u: a row past the last one has no columns
    auto row_end = [&](long long r0, int u) { return my_row < a.rows - r0 - u * ROWS ? lim : 0; };
    auto load = [&](long long r0, Rows &w) {
        const T *x = static_cast<const T *>(a.x) + r0 * C;
        const uint8_t *codes = a.codes + r0 * C;
        const float2 *ranges = reinterpret_cast<const float2 *>(a.ranges) + r0 * G;
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const int end = row_end(r0, u);
#pragma unroll
            for (int j = 0; j < NV; j++) {
                if (KIND != KEEP_RESTORE) load8<VEC, L>(x + (long long)(u * ROWS) * C + off + j * NEXT, c[j], end, w.raw[u][j]);
                if (KIND == KEEP_RESTORE || KIND == KEEP_GELU_BWD) w.q[u][j] = load_codes<VEC, L>(codes + (long long)(u * ROWS) * C + off + j * NEXT, c[j], end);
            }
            if (KIND == KEEP_RESTORE || KIND == KEEP_GELU_BWD)
                w.range[u] = end ? __ldg(ranges + (long long)(u * ROWS) * G + range_off) : make_float2(0.f, 0.f);
        }
    };
    // Whole CTAs go round together (the groups' ranges are found with warp-wide instructions).  The next round's values are
    // on their way while this one's are worked on.
    Rows next;
    const long long round = (long long)gridDim.y * (UN * ROWS);
    load((long long)blockIdx.y * (UN * ROWS), next);
    for (long long r0 = (long long)blockIdx.y * (UN * ROWS); r0 < a.rows; r0 += round) {
        T *y = static_cast<T *>(a.y) + r0 * C, *dx = static_cast<T *>(a.dx) + r0 * C;
        uint8_t *codes = a.codes + r0 * C;
        float2 *ranges = reinterpret_cast<float2 *>(a.ranges) + r0 * G;
        const Rows now = next;
        load(r0 + round, next);
        const Raw8<T, VEC> (&raw)[UN][NV] = now.raw;
        int end[UN];
#pragma unroll
        for (int u = 0; u < UN; u++) end[u] = row_end(r0, u);
        if constexpr (KIND == KEEP_FWD || KIND == KEEP_GELU_FWD) {
            F2 f[UN][NV][4];
#pragma unroll
            for (int u = 0; u < UN; u++)
#pragma unroll
                for (int j = 0; j < NV; j++) {
                    unpack8<T, VEC>(raw[u][j], f[u][j]);
                    if constexpr (KIND == KEEP_GELU_FWD) {
                        F2 v[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            f[u][j][i] = add2(f[u][j][i], b[j][i]);
                            v[i] = gelu_of(f[u][j][i], normal_of<sizeof(T) == 4>(f[u][j][i]));
                        }
                        store8<VEC, L>(y + (long long)(u * ROWS) * C + off + j * NEXT, c[j], end[u], v);
                    }
                }
            if (KIND == KEEP_FWD || a.codes) {
                uint2 q[UN][NV];
                float2 range[UN];
                keep_groups<VEC, L, NV, UN>(f, c, end, q, range);
#pragma unroll
                for (int u = 0; u < UN; u++) {
#pragma unroll
                    for (int j = 0; j < NV; j++) store_codes<VEC, L>(codes + (long long)(u * ROWS) * C + off + j * NEXT, c[j], end[u], q[u][j]);
                    if (end[u] && lane == 0) ranges[(long long)(u * ROWS) * G + range_off] = range[u];
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < UN; u++)
#pragma unroll
                for (int j = 0; j < NV; j++) {
                    F2 v[4];
                    restore_codes(now.q[u][j], now.range[u], v);
                    if constexpr (KIND == KEEP_GELU_BWD) {
                        F2 d[4], f[4];
                        unpack8<T, VEC>(raw[u][j], f);
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const Normal n = normal_of<sizeof(T) == 4>(v[i]);
                            d[i] = mul2(f[i], gelu_slope(v[i], n));
                            sum[j][i] = add2(sum[j][i], d[i]);   // rows that do not exist add zeros; columns are never read
                            if (a.y) v[i] = gelu_of(v[i], n);
                        }
                        store8<VEC, L>(dx + (long long)(u * ROWS) * C + off + j * NEXT, c[j], end[u], d);
                    }
                    if (KIND == KEEP_RESTORE || a.y) store8<VEC, L>(y + (long long)(u * ROWS) * C + off + j * NEXT, c[j], end[u], v);
                }
        }
    }
    if constexpr (KIND == KEEP_GELU_BWD) {
        if (!a.dbias) return;
        __shared__ float red[kKeepWarps][kKeepGroup];
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float t = i & 1 ? apart(sum[j][i >> 1]).y : apart(sum[j][i >> 1]).x;
#pragma unroll
                for (int o = L; o < 32; o <<= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
                if (sub == 0) red[warp][col_of<VEC, L>(first_col<VEC>(lane) + j * NEXT, i)] = t;
            }
        __syncthreads();
        if (threadIdx.x < lim - g * kKeepGroup) {
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < kKeepWarps; w++) s += red[w][threadIdx.x];
            a.partial[(size_t)blockIdx.y * C + g * kKeepGroup + threadIdx.x] = s;
        }
    }
}

// Sums over the TEAM warps that share a row.  `slot`: a buffer that no warp of the team still reads (the callers
// alternate).  Each team has a hardware barrier of its own.
template <int TEAM, int NV>
__device__ __forceinline__ void team_sum(float (&v)[NV], float (*slot)[NV], int team, int wt) {
    if constexpr (TEAM > 1) {
        if ((threadIdx.x & 31) == 0) {
#pragma unroll
            for (int k = 0; k < NV; k++) slot[team * TEAM + wt][k] = v[k];
        }
        asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(TEAM * 32) : "memory");
#pragma unroll
        for (int k = 0; k < NV; k++) v[k] = 0.f;
#pragma unroll
        for (int w = 0; w < TEAM; w++)
#pragma unroll
            for (int k = 0; k < NV; k++) v[k] += slot[team * TEAM + w][k];
    }
}

// How a row is held: LR lanes (4 to 16 for one group, 32/LR rows a warp; 32 for two groups side by side), a team of TEAM
// warps, NG passes of a warp's lanes along the row.  L: lanes of a group.
// A lane has NV vectors of each of its groups.
template <int LR, int TEAM, int NG, int NV> struct LnRow {
    static constexpr int L = LR < 16 ? LR : 16, PER_PASS = LR == 32 ? 2 : 1, RW = 32 / LR, TEAMS = kKeepWarps / TEAM;
    static constexpr int NP = NG * NV;               // vectors of a lane
    static constexpr int ROWS = TEAMS * RW;          // rows of a CTA
    int lane, team, wt, half, row;                   // lane within its group; group of the pass; row of the CTA
    __device__ __forceinline__ LnRow() {
        const int warp = threadIdx.x >> 5, l = threadIdx.x & 31;
        lane = l % L; half = LR == 32 ? l / 16 : 0; team = warp / TEAM; wt = warp % TEAM; row = team * RW + l / LR;
    }
    __device__ __forceinline__ int group(int j) const { return (wt * NG + j) * PER_PASS + half; }
    template <bool VEC> __device__ __forceinline__ int column(int v) const {      // the first of vector v
        return group(v / NV) * kKeepGroup + first_col<VEC>(lane) + v % NV * (L * kKeepLane);
    }
};

// LayerNorm over rows of up to 8192 columns, y = (x - mean) * rstd * gamma + beta, the row held in registers.  Statistics are
// two-pass, fp32.  Kept for the backward pass: the codes of x, mean and rstd.  UN rows of a lane are in flight at once
// (short rows: what bounds the kernel is memory, and a lane's piece of a row is 16 bytes).
template <typename T, bool VEC, int LR, int TEAM, int NG, int NV, int UN>
__global__ void __launch_bounds__(kKeepThreads)
ln_keep_kernel(const LnKeepArgs a) {
    using R = LnRow<LR, TEAM, NG, NV>;
    constexpr int L = R::L, NP = R::NP;
    __shared__ float s1[kKeepWarps][UN], s2[kKeepWarps][UN];
    const R w;
    const int C = a.C, G = (C + kKeepGroup - 1) / kKeepGroup;
    const float inv_c = 1.f / (float)C;
    const unsigned off = (unsigned)(w.row * C), range_off = (unsigned)(w.row * G);
    F2 gm[NP][4], bt[NP][4];
    int c[NP], lim[NP];
#pragma unroll
    for (int j = 0; j < NP; j++) {
        c[j] = w.template column<VEC>(j);
        lim[j] = min(C, (w.group(j / NV) + 1) * kKeepGroup);
        load_params<VEC, L>(a.gamma, a.pbf16, c[j], lim[j], gm[j]);
        load_params<VEC, L>(a.beta, a.pbf16, c[j], lim[j], bt[j]);
    }
    struct Rows { Raw8<T, VEC> raw[UN][NP]; };
    auto exists = [&](long long r0, int u) { return w.row < a.rows - r0 - u * R::ROWS; };
    auto load = [&](long long r0, Rows &to) {
        const T *x = static_cast<const T *>(a.x) + r0 * C;
#pragma unroll
        for (int u = 0; u < UN; u++)
#pragma unroll
            for (int j = 0; j < NP; j++)
                load8<VEC, L>(x + (long long)(u * R::ROWS) * C + (off + c[j]), c[j], exists(r0, u) ? lim[j] : 0, to.raw[u][j]);
    };
    // the next round's rows are on their way while this one's are worked on
    Rows next;
    const long long round = (long long)gridDim.x * (UN * R::ROWS);
    load((long long)blockIdx.x * (UN * R::ROWS), next);
    for (long long r0 = (long long)blockIdx.x * (UN * R::ROWS); r0 < a.rows; r0 += round) {
        T *y = static_cast<T *>(a.y) + r0 * C;
        uint8_t *codes = a.codes + r0 * C;
        float2 *ranges = reinterpret_cast<float2 *>(a.ranges) + r0 * G, *stats = reinterpret_cast<float2 *>(a.stats) + r0;
        const Rows now = next;
        load(r0 + round, next);
        const Raw8<T, VEC> (&raw)[UN][NP] = now.raw;
        float s[UN], mean[UN];
        bool act[UN];
#pragma unroll
        for (int u = 0; u < UN; u++) act[u] = exists(r0, u);
#pragma unroll
        for (int u = 0; u < UN; u++) {
            s[u] = 0.f;
#pragma unroll
            for (int j = 0; j < NP; j++) {
                F2 f[4];
                unpack8<T, VEC>(raw[u][j], f);
                const float2 t = apart(add2(add2(f[0], f[1]), add2(f[2], f[3])));
                s[u] += t.x + t.y;
            }
        }
        lane_sums<LR, UN>(s);
        team_sum<TEAM, UN>(s, s1, w.team, w.wt);
#pragma unroll
        for (int u = 0; u < UN; u++) {
            mean[u] = s[u] * inv_c;
            s[u] = 0.f;
#pragma unroll
            for (int j = 0; j < NP; j++) {
                F2 f[4], sq = both(0.f);
                unpack8<T, VEC>(raw[u][j], f);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    F2 d = add2(f[i], both(-mean[u]));
                    if (!VEC) {
                        const float2 v = apart(d);
                        d = two(c[j] + 2 * i * L < lim[j] ? v.x : 0.f, c[j] + (2 * i + 1) * L < lim[j] ? v.y : 0.f);
                    }
                    sq = fma2(d, d, sq);
                }
                const float2 t = apart(sq);
                if (!VEC || c[j] < C) s[u] += t.x + t.y;
            }
        }
        lane_sums<LR, UN>(s);
        team_sum<TEAM, UN>(s, s2, w.team, w.wt);
#pragma unroll
        for (int u = 0; u < UN; u++) {
            s[u] = rsqrtf(s[u] * inv_c + a.eps);
            if (a.codes && act[u] && w.lane == 0 && w.half == 0 && w.wt == 0) stats[u * R::ROWS + w.row] = make_float2(mean[u], s[u]);
        }
#pragma unroll
        for (int k = 0; k < NG; k++) {
            if ((w.wt * NG + k) * R::PER_PASS >= G) break;                      // the same for the whole warp
            F2 f[UN][NV][4];
            int end[UN], col[NV];
            uint2 q[UN][NV];
            float2 range[UN];
#pragma unroll
            for (int u = 0; u < UN; u++) {
                end[u] = act[u] ? lim[k * NV] : 0;
#pragma unroll
                for (int v = 0; v < NV; v++) {
                    const int j = k * NV + v;
                    col[v] = c[j];
                    F2 o[4];
                    unpack8<T, VEC>(raw[u][j], f[u][v]);
#pragma unroll
                    for (int i = 0; i < 4; i++) o[i] = fma2(mul2(add2(f[u][v][i], both(-mean[u])), both(s[u])), gm[j][i], bt[j][i]);
                    store8<VEC, L>(y + (long long)(u * R::ROWS) * C + (off + c[j]), c[j], end[u], o);
                }
            }
            if (!a.codes) continue;
            keep_groups<VEC, L, NV, UN>(f, col, end, q, range);
#pragma unroll
            for (int u = 0; u < UN; u++) {
#pragma unroll
                for (int v = 0; v < NV; v++)
                    store_codes<VEC, L>(codes + (long long)(u * R::ROWS) * C + (off + col[v]), col[v], end[u], q[u][v]);
                if (act[u] && w.lane == 0 && w.group(k) < G) ranges[(long long)(u * R::ROWS) * G + (range_off + w.group(k))] = range[u];
            }
        }
    }
}

// Its backward pass from the checkpoint x' of x:  xhat = (x' - mean) * rstd,  g = dy * gamma,
//   dx = rstd * (g - mean_C(g) - xhat * mean_C(g * xhat)),  dgamma = sum_rows dy * xhat,  dbeta = sum_rows dy.
// Column sums as in layernorm_cl_bwd_kernel: registers, then the CTA's teams in order, then the CTAs in order
// (sum_slices_kernel).  Dynamic shared memory: teams x 2 x C floats where a CTA has more than one team.
template <typename T, bool VEC, int LR, int TEAM, int NG, int NV, int UN>
__global__ void __launch_bounds__(kKeepThreads)
ln_keep_bwd_kernel(const LnKeepArgs a) {
    using R = LnRow<LR, TEAM, NG, NV>;
    constexpr int L = R::L, NP = R::NP;
    extern __shared__ float ln_cols[];
    __shared__ float s1[2][kKeepWarps][2 * UN];
    const R w;
    const int C = a.C, G = (C + kKeepGroup - 1) / kKeepGroup;
    const float inv_c = 1.f / (float)C;
    const unsigned off = (unsigned)(w.row * C), range_off = (unsigned)(w.row * G);
    F2 gm[NP][4], sg[NP][4], sb[NP][4];
    int c[NP], lim[NP];
#pragma unroll
    for (int j = 0; j < NP; j++) {
        c[j] = w.template column<VEC>(j);
        lim[j] = min(C, (w.group(j / NV) + 1) * kKeepGroup);
        load_params<VEC, L>(a.gamma, a.pbf16, c[j], lim[j], gm[j]);
#pragma unroll
        for (int i = 0; i < 4; i++) sg[j][i] = sb[j][i] = both(0.f);
    }
    // xhat of the lane's values.  Of a group that is NaN, single columns may still not exist.
    auto normalised = [&](uint2 q, float2 range, float2 st, int j, F2 (&h)[4]) {
        restore_codes(q, range, h);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            h[i] = mul2(add2(h[i], both(-st.x)), both(st.y));
            if (!VEC) {
                const float2 v = apart(h[i]);
                h[i] = two(c[j] + 2 * i * L < lim[j] ? v.x : 0.f, c[j] + (2 * i + 1) * L < lim[j] ? v.y : 0.f);
            }
        }
    };
    struct Rows {
        Raw8<T, VEC> raw[UN][NP];
        float2 st[UN], range[UN][NG];
        uint2 q[UN][NP];
    };
    auto exists = [&](long long r0, int u) { return w.row < a.rows - r0 - u * R::ROWS; };
    auto load = [&](long long r0, Rows &to) {
        const T *dy = static_cast<const T *>(a.x) + r0 * C;
        const uint8_t *codes = a.codes + r0 * C;
        const float2 *ranges = reinterpret_cast<const float2 *>(a.ranges) + r0 * G, *stats = reinterpret_cast<const float2 *>(a.stats) + r0;
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const bool on = exists(r0, u);
            to.st[u] = on ? __ldg(stats + u * R::ROWS + w.row) : make_float2(0.f, 0.f);
#pragma unroll
            for (int j = 0; j < NP; j++) {
                const int end = on ? lim[j] : 0;
                load8<VEC, L>(dy + (long long)(u * R::ROWS) * C + (off + c[j]), c[j], end, to.raw[u][j]);
                to.q[u][j] = load_codes<VEC, L>(codes + (long long)(u * R::ROWS) * C + (off + c[j]), c[j], end);
                // (columns that do not exist: dy, gamma and this are zero, whatever their group holds; with more vectors than one the
                // row is that group)
                if (j % NV == 0) to.range[u][j / NV] = c[j] < end ? __ldg(ranges + (long long)(u * R::ROWS) * G + (range_off + w.group(j / NV))) : make_float2(0.f, 0.f);
            }
        }
    };
    // the next round's rows are on their way while this one's are worked on, where there are registers for both
    constexpr bool AHEAD = NG * UN <= 2;
    Rows next;
    const long long round = (long long)gridDim.x * (UN * R::ROWS);
    if (AHEAD) load((long long)blockIdx.x * (UN * R::ROWS), next);
    int turn = 0;
    for (long long r0 = (long long)blockIdx.x * (UN * R::ROWS); r0 < a.rows; r0 += round) {
        T *dx = static_cast<T *>(a.dx) + r0 * C, *y = static_cast<T *>(a.y) + r0 * C;
        if (!AHEAD) load(r0, next);
        const Rows now = next;
        if (AHEAD) load(r0 + round, next);
        const Raw8<T, VEC> (&raw)[UN][NP] = now.raw;
        const float2 (&st)[UN] = now.st, (&range)[UN][NG] = now.range;
        const uint2 (&q)[UN][NP] = now.q;
        float s[2 * UN];
        bool act[UN];
#pragma unroll
        for (int u = 0; u < UN; u++) act[u] = exists(r0, u);
#pragma unroll
        for (int u = 0; u < UN; u++) {
            F2 t1 = both(0.f), t2 = both(0.f);
#pragma unroll
            for (int j = 0; j < NP; j++) {
                F2 d[4], h[4];
                normalised(q[u][j], range[u][j / NV], st[u], j, h);
                unpack8<T, VEC>(raw[u][j], d);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const F2 gg = mul2(d[i], gm[j][i]);
                    t1 = add2(t1, gg);
                    t2 = fma2(gg, h[i], t2);
                    sg[j][i] = fma2(d[i], h[i], sg[j][i]);
                    sb[j][i] = add2(sb[j][i], d[i]);
                }
            }
            s[2 * u] = apart(t1).x + apart(t1).y;
            s[2 * u + 1] = apart(t2).x + apart(t2).y;
        }
        lane_sums<LR, 2 * UN>(s);
        team_sum<TEAM, 2 * UN>(s, s1[turn], w.team, w.wt);
        turn ^= 1;
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const float c1 = s[2 * u] * inv_c, c2 = s[2 * u + 1] * inv_c;
#pragma unroll
            for (int j = 0; j < NP; j++) {
                const int end = act[u] ? lim[j] : 0;
                F2 d[4], h[4], o[4];
                normalised(q[u][j], range[u][j / NV], st[u], j, h);
                unpack8<T, VEC>(raw[u][j], d);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    o[i] = mul2(fma2(h[i], both(-c2), fma2(d[i], gm[j][i], both(-c1))), both(st[u].y));
                store8<VEC, L>(dx + (long long)(u * R::ROWS) * C + (off + c[j]), c[j], end, o);
                if (a.y) {
                    F2 bt[4];
                    load_params<VEC, L>(a.beta, a.pbf16, c[j], end, bt);
#pragma unroll
                    for (int i = 0; i < 4; i++) o[i] = fma2(h[i], gm[j][i], bt[i]);
                    store8<VEC, L>(y + (long long)(u * R::ROWS) * C + (off + c[j]), c[j], end, o);
                }
            }
        }
    }
    float *out = a.partial + (size_t)blockIdx.x * 2 * C;
#pragma unroll
    for (int j = 0; j < NP; j++) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int k = col_of<VEC, L>(c[j], i);
            float tg = i & 1 ? apart(sg[j][i >> 1]).y : apart(sg[j][i >> 1]).x, tb = i & 1 ? apart(sb[j][i >> 1]).y : apart(sb[j][i >> 1]).x;
#pragma unroll
            for (int o = LR; o < 32; o <<= 1) {
                tg += __shfl_xor_sync(0xffffffffu, tg, o);
                tb += __shfl_xor_sync(0xffffffffu, tb, o);
            }
            if (w.row % R::RW == 0 && k < lim[j]) {
                float *to = R::TEAMS > 1 ? ln_cols + (size_t)w.team * 2 * C : out;
                to[k] = tg;
                to[C + k] = tb;
            }
        }
    }
    if constexpr (R::TEAMS > 1) {
        __syncthreads();
        for (int e = threadIdx.x; e < 2 * C; e += kKeepThreads) {
            float t = 0.f;
#pragma unroll
            for (int k = 0; k < R::TEAMS; k++) t += ln_cols[(size_t)k * 2 * C + e];
            out[e] = t;
        }
    }
}

}  // namespace o1d

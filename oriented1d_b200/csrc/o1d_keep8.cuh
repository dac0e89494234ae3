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

namespace o1d {

constexpr int kKeepThreads = 256;
constexpr int kKeepWarps = kKeepThreads / 32;

__device__ __forceinline__ float min_nan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

// Least and greatest value over the L lanes that share a group; a NaN anywhere gives NaN.
template <int L>
__device__ __forceinline__ void group_range(float &lo, float &hi) {
    if constexpr (L == 32) {
        asm volatile("redux.sync.min.NaN.f32 %0, %0, 0xffffffff;" : "+f"(lo));
        asm volatile("redux.sync.max.NaN.f32 %0, %0, 0xffffffff;" : "+f"(hi));
    } else {
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) {
            lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
    }
}
template <int L>
__device__ __forceinline__ float lane_sum(float v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Four values of a lane.  VEC: columns c .. c+3, one vector access (C % 4 == 0 and aligned, so all four exist or none);
// otherwise columns c, c+L, c+2L, c+3L, one element each.
template <bool VEC, int L> __device__ __forceinline__ int col_of(int c, int i) { return VEC ? c + i : c + i * L; }

template <bool VEC, int L, typename T>
__device__ __forceinline__ void load4(const T *row, int c, int C, float fill, float (&f)[4]) {
    if constexpr (VEC) {
        if (c < C) {
            if constexpr (sizeof(T) == 4) {
                const float4 v = __ldg(reinterpret_cast<const float4 *>(row + c));
                f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
            } else {
                const uint2 v = __ldg(reinterpret_cast<const uint2 *>(row + c));
                f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xffff0000u);
                f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xffff0000u);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = fill;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = c + i * L < C ? ld(row + c + i * L) : fill;
    }
}
template <bool VEC, int L, typename T>
__device__ __forceinline__ void store4(T *row, int c, int C, const float (&f)[4]) {
    if constexpr (VEC) {
        if (c >= C) return;
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4 *>(row + c) = make_float4(f[0], f[1], f[2], f[3]);
        } else {
            __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
            *reinterpret_cast<uint2 *>(row + c) = make_uint2(*reinterpret_cast<uint32_t *>(&a), *reinterpret_cast<uint32_t *>(&b));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (c + i * L < C) st(row + c + i * L, f[i]);
    }
}
template <bool VEC, int L>
__device__ __forceinline__ void load_codes(const uint8_t *row, int c, int C, uint32_t (&q)[4]) {
    if constexpr (VEC) {
        const uint32_t v = c < C ? __ldg(reinterpret_cast<const uint32_t *>(row + c)) : 0u;
#pragma unroll
        for (int i = 0; i < 4; i++) q[i] = (v >> (8 * i)) & 0xffu;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) q[i] = c + i * L < C ? __ldg(row + c + i * L) : 0u;
    }
}
template <bool VEC, int L>
__device__ __forceinline__ void store_codes(uint8_t *row, int c, int C, const uint32_t (&q)[4]) {
    if constexpr (VEC) {
        if (c < C) *reinterpret_cast<uint32_t *>(row + c) = q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (c + i * L < C) row[c + i * L] = (uint8_t)q[i];
    }
}

// Codes of the lane's four values, and the group's range (written by the group's first lane).
template <bool VEC, int L>
__device__ __forceinline__ void keep_group(const float (&f)[4], int c, int C, int lane, uint8_t *codes, float *range) {
    float lo = __int_as_float(0x7f800000), hi = -lo;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (col_of<VEC, L>(c, i) >= C) continue;
        lo = min_nan(lo, f[i]);
        hi = max_nan(hi, f[i]);
    }
    group_range<L>(lo, hi);
    float step = __fmul_rn(__fsub_rn(hi, lo), 1.f / 255.f);
    if (!(step <= 3.402823466e38f)) step = __int_as_float(0x7fffffff);        // NaN or infinite: the group is lost
    float inv = 0.f;
    if (step < 1.175494351e-38f) step = 0.f; else inv = __frcp_rn(step);
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; i++) q[i] = min(__float2uint_rn(__fmul_rn(__fsub_rn(f[i], lo), inv)), 255u);
    store_codes<VEC, L>(codes, c, C, q);
    if (lane == 0) *reinterpret_cast<float2 *>(range) = make_float2(lo, step);
}
__device__ __forceinline__ float restored(uint32_t q, float2 range) { return fmaf((float)q, range.y, range.x); }

// The elementwise kinds.  CTA (bx, by): the columns of group bx, rows by*8+warp, ... in steps of gridDim.y*8 (a warp
// holds 32/L rows at once where rows are short).  Column sums of the GELU backward (its bias gradient) stay in
// registers over all rows of a thread and leave as one partial per (by, column), added in a fixed order by
// sum_slices_kernel.  UN rows of a warp are in flight at once: the kernels are bound by memory, and a lane's piece of
// a row is only 8 or 16 bytes.
template <int KIND, typename T, bool VEC, int L, int UN>
__global__ void __launch_bounds__(kKeepThreads)
keep_kernel(const KeepArgs a) {
    constexpr int RW = 32 / L;                                   // rows of a warp
    const int lane = threadIdx.x % L, sub = (threadIdx.x & 31) / L, warp = threadIdx.x >> 5;
    const int g = blockIdx.x, G = gridDim.x, C = a.C;
    const int c = g * kKeepGroup + (VEC ? lane * 4 : lane);
    const int lim = min(C, (g + 1) * kKeepGroup);                // end of the group
    const long long stride = (long long)gridDim.y * kKeepWarps * RW;
    const T *x = static_cast<const T *>(a.x);
    T *y = static_cast<T *>(a.y), *dx = static_cast<T *>(a.dx);
    float b[4] = {0.f, 0.f, 0.f, 0.f}, sum[4] = {0.f, 0.f, 0.f, 0.f};
    if (KIND == KEEP_GELU_FWD && a.bias) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (col_of<VEC, L>(c, i) < lim) b[i] = ld_param(a.bias, col_of<VEC, L>(c, i), a.pbf16);
    }
    // whole warps leave the loop together (the groups' ranges are found with warp-wide instructions)
    for (long long r0 = ((long long)blockIdx.y * kKeepWarps + warp) * RW; r0 < a.rows; r0 += stride * UN) {
        float f[UN][4];
        uint32_t q[UN][4];
        float2 range[UN];
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const long long r = r0 + sub + u * stride;
            const bool act = r < a.rows;
            if (KIND != KEEP_RESTORE) load4<VEC, L>(x + (act ? r : 0) * C, c, act ? lim : 0, 0.f, f[u]);
            if (KIND == KEEP_RESTORE || KIND == KEEP_GELU_BWD) {
                load_codes<VEC, L>(a.codes + (act ? r : 0) * C, c, act ? lim : 0, q[u]);
                range[u] = __ldg(reinterpret_cast<const float2 *>(a.ranges) + (act ? r : 0) * G + g);
            }
        }
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const long long r = r0 + sub + u * stride;
            const bool act = r < a.rows;
            const int end = act ? lim : 0;                       // a row past the last one has no columns
            const long long ro = (act ? r : 0) * C;
            if constexpr (KIND == KEEP_FWD || KIND == KEEP_GELU_FWD) {
                if constexpr (KIND == KEEP_GELU_FWD) {
                    float v[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        f[u][i] = __fadd_rn(f[u][i], b[i]);
                        v[i] = gelu_exact(f[u][i]);
                    }
                    store4<VEC, L>(y + ro, c, end, v);
                }
                if (KIND == KEEP_FWD || a.codes)
                    keep_group<VEC, L>(f[u], c, end, act ? lane : 1, a.codes + ro, a.ranges + ((act ? r : 0) * G + g) * 2);
            } else {
                float v[4], d[4];
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = restored(q[u][i], range[u]);
                if constexpr (KIND == KEEP_GELU_BWD) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        d[i] = f[u][i] * gelu_exact_grad(v[i]);
                        if (col_of<VEC, L>(c, i) < end) sum[i] += d[i];
                        v[i] = gelu_exact(v[i]);
                    }
                    store4<VEC, L>(dx + ro, c, end, d);
                }
                if (KIND == KEEP_RESTORE || y) store4<VEC, L>(y + ro, c, end, v);
            }
        }
    }
    if constexpr (KIND == KEEP_GELU_BWD) {
        if (!a.dbias) return;
        __shared__ float red[kKeepWarps][kKeepGroup];
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma unroll
            for (int o = L; o < 32; o <<= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
            if (sub == 0) red[warp][col_of<VEC, L>(VEC ? lane * 4 : lane, i)] = sum[i];
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

// LayerNorm over rows of up to 8192 columns, y = (x - mean) * rstd * gamma + beta.  A row is held in registers by L lanes
// (short rows: 32/L rows a warp), by a warp (up to 512 columns) or by a team of TEAM warps, NG groups of 128 columns a
// warp.  Statistics are two-pass, fp32.  Kept for the backward pass: the codes of x, mean and rstd.
template <typename T, bool VEC, int L, int TEAM, int NG>
__global__ void __launch_bounds__(kKeepThreads)
ln_keep_kernel(const LnKeepArgs a) {
    constexpr int RW = 32 / L, TEAMS = kKeepWarps / TEAM;
    __shared__ float s1[kKeepWarps][1], s2[kKeepWarps][1];
    const int lane = threadIdx.x % L, sub = (threadIdx.x & 31) / L, warp = threadIdx.x >> 5;
    const int team = warp / TEAM, wt = warp % TEAM, C = a.C, G = (C + kKeepGroup - 1) / kKeepGroup;
    const T *x = static_cast<const T *>(a.x);
    T *y = static_cast<T *>(a.y);
    const float inv_c = 1.f / (float)C;
    for (long long r0 = ((long long)blockIdx.x * TEAMS + team) * RW; r0 < a.rows; r0 += (long long)gridDim.x * TEAMS * RW) {
        const long long r = r0 + sub;
        const bool act = r < a.rows;
        const long long ro = (act ? r : 0) * C;
        float f[NG][4], s[1] = {0.f};
#pragma unroll
        for (int j = 0; j < NG; j++) {
            const int c = (wt * NG + j) * kKeepGroup + (VEC ? lane * 4 : lane);
            load4<VEC, L>(x + ro, c, act ? min(C, (wt * NG + j + 1) * kKeepGroup) : 0, 0.f, f[j]);
        }
#pragma unroll
        for (int j = 0; j < NG; j++) s[0] += (f[j][0] + f[j][1]) + (f[j][2] + f[j][3]);
        s[0] = lane_sum<L>(s[0]);
        team_sum<TEAM, 1>(s, s1, team, wt);
        const float mean = s[0] * inv_c;
        s[0] = 0.f;
#pragma unroll
        for (int j = 0; j < NG; j++) {
            const int c = (wt * NG + j) * kKeepGroup + (VEC ? lane * 4 : lane);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float d = f[j][i] - mean;
                if (col_of<VEC, L>(c, i) < C) s[0] += d * d;
            }
        }
        s[0] = lane_sum<L>(s[0]);
        team_sum<TEAM, 1>(s, s2, team, wt);
        const float rstd = rsqrtf(s[0] * inv_c + a.eps);
        if (act && lane == 0 && wt == 0) *reinterpret_cast<float2 *>(a.stats + r * 2) = make_float2(mean, rstd);
#pragma unroll
        for (int j = 0; j < NG; j++) {
            const int g = wt * NG + j, c = g * kKeepGroup + (VEC ? lane * 4 : lane);
            if (g >= G) break;
            const int end = act ? min(C, (g + 1) * kKeepGroup) : 0;
            float o[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int k = col_of<VEC, L>(c, i);
                o[i] = k < end ? (f[j][i] - mean) * rstd * ld_param(a.gamma, k, a.pbf16) + ld_param(a.beta, k, a.pbf16) : 0.f;
            }
            store4<VEC, L>(y + ro, c, end, o);
            keep_group<VEC, L>(f[j], c, end, act ? lane : 1, a.codes + ro, a.ranges + ((act ? r : 0) * G + g) * 2);
        }
    }
}

// Its backward pass from the checkpoint x' of x:  xhat = (x' - mean) * rstd,  g = dy * gamma,
//   dx = rstd * (g - mean_C(g) - xhat * mean_C(g * xhat)),  dgamma = sum_rows dy * xhat,  dbeta = sum_rows dy.
// Column sums as in layernorm_cl_bwd_kernel: registers, then the CTA's teams in order, then the CTAs in order
// (sum_slices_kernel).  Dynamic shared memory: teams x 2 x C floats where a CTA has more than one team.
template <typename T, bool VEC, int L, int TEAM, int NG>
__global__ void __launch_bounds__(kKeepThreads)
ln_keep_bwd_kernel(const LnKeepArgs a) {
    constexpr int RW = 32 / L, TEAMS = kKeepWarps / TEAM;
    extern __shared__ float ln_cols[];
    __shared__ float s1[2][kKeepWarps][2];
    const int lane = threadIdx.x % L, sub = (threadIdx.x & 31) / L, warp = threadIdx.x >> 5;
    const int team = warp / TEAM, wt = warp % TEAM, C = a.C, G = (C + kKeepGroup - 1) / kKeepGroup;
    const T *dy = static_cast<const T *>(a.x);
    T *dx = static_cast<T *>(a.dx), *y = static_cast<T *>(a.y);
    const float inv_c = 1.f / (float)C;
    float gm[NG][4], sg[NG][4], sb[NG][4];
#pragma unroll
    for (int j = 0; j < NG; j++) {
        const int c = (wt * NG + j) * kKeepGroup + (VEC ? lane * 4 : lane);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int k = col_of<VEC, L>(c, i);
            gm[j][i] = k < min(C, (wt * NG + j + 1) * kKeepGroup) ? ld_param(a.gamma, k, a.pbf16) : 0.f;
            sg[j][i] = sb[j][i] = 0.f;
        }
    }
    int turn = 0;
    for (long long r0 = ((long long)blockIdx.x * TEAMS + team) * RW; r0 < a.rows; r0 += (long long)gridDim.x * TEAMS * RW) {
        const long long r = r0 + sub;
        const bool act = r < a.rows;
        const long long ro = (act ? r : 0) * C;
        const float2 st = __ldg(reinterpret_cast<const float2 *>(a.stats) + (act ? r : 0));
        float d[NG][4], h[NG][4], s[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NG; j++) {
            const int g = wt * NG + j, c = g * kKeepGroup + (VEC ? lane * 4 : lane);
            const int end = act ? min(C, (g + 1) * kKeepGroup) : 0;
            uint32_t q[4];
            load4<VEC, L>(dy + ro, c, end, 0.f, d[j]);
            load_codes<VEC, L>(a.codes + ro, c, end, q);
            const float2 range = g < G ? __ldg(reinterpret_cast<const float2 *>(a.ranges) + (act ? r : 0) * G + g) : make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 4; i++) h[j][i] = col_of<VEC, L>(c, i) < end ? (restored(q[i], range) - st.x) * st.y : 0.f;
        }
#pragma unroll
        for (int j = 0; j < NG; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float gg = d[j][i] * gm[j][i];
                s[0] += gg;
                s[1] += gg * h[j][i];
                sg[j][i] += d[j][i] * h[j][i];
                sb[j][i] += d[j][i];
            }
        s[0] = lane_sum<L>(s[0]);
        s[1] = lane_sum<L>(s[1]);
        team_sum<TEAM, 2>(s, s1[turn], team, wt);
        turn ^= 1;
        const float c1 = s[0] * inv_c, c2 = s[1] * inv_c;
#pragma unroll
        for (int j = 0; j < NG; j++) {
            const int g = wt * NG + j, c = g * kKeepGroup + (VEC ? lane * 4 : lane);
            if (g >= G) break;
            const int end = act ? min(C, (g + 1) * kKeepGroup) : 0;
            float o[4];
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = st.y * (d[j][i] * gm[j][i] - c1 - h[j][i] * c2);
            store4<VEC, L>(dx + ro, c, end, o);
            if (y) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int k = col_of<VEC, L>(c, i);
                    o[i] = k < end ? h[j][i] * gm[j][i] + ld_param(a.beta, k, a.pbf16) : 0.f;
                }
                store4<VEC, L>(y + ro, c, end, o);
            }
        }
    }
    float *out = a.partial + (size_t)blockIdx.x * 2 * C;
#pragma unroll
    for (int j = 0; j < NG; j++) {
        const int c = (wt * NG + j) * kKeepGroup + (VEC ? lane * 4 : lane);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int k = col_of<VEC, L>(c, i);
#pragma unroll
            for (int o = L; o < 32; o <<= 1) {
                sg[j][i] += __shfl_xor_sync(0xffffffffu, sg[j][i], o);
                sb[j][i] += __shfl_xor_sync(0xffffffffu, sb[j][i], o);
            }
            if (sub == 0 && k < min(C, (wt * NG + j + 1) * kKeepGroup)) {
                float *to = TEAMS > 1 ? ln_cols + (size_t)team * 2 * C : out;
                to[k] = sg[j][i];
                to[C + k] = sb[j][i];
            }
        }
    }
    if constexpr (TEAMS > 1) {
        __syncthreads();
        for (int e = threadIdx.x; e < 2 * C; e += kKeepThreads) {
            float t = 0.f;
#pragma unroll
            for (int w = 0; w < TEAMS; w++) t += ln_cols[(size_t)w * 2 * C + e];
            out[e] = t;
        }
    }
}

}  // namespace o1d

// Launches of the 8-bit checkpoint kernels.
#include "o1d_keep8.cuh"
#include "o1d_slices.cuh"

namespace o1d {

namespace {

inline int groups_of(int C) { return (C + kKeepGroup - 1) / kKeepGroup; }
inline bool aligned(const void *p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }
// Lanes that hold a group's part of a row, eight values each.
inline int lanes_of(int C) { return C <= 32 ? 4 : C <= 64 ? 8 : 16; }
// Whole vectors: rows of eight values, 16 bytes of the elements, 8 of the codes.
inline bool vectors(int C, const void *x, const void *y, const void *dx, const void *codes) {
    return C % 8 == 0 && aligned(x, 16) && aligned(y, 16) && aligned(dx, 16) && aligned(codes, 8);
}

// Vectors of a lane in flight: two where there are rows enough for four CTAs on every SM, else one, so that short tensors
// reach all SMs.  Of two rows, or (bf16, whole vectors) of one row that eight lanes hold: an exchange less and half as many ranges a
// value, but more registers.  100352 x 768 bf16, GELU forward / backward: one 92 / 87 us, two rows 82 / 85, three 90 / 99, eight
// lanes 84 / 81; 12544 x 2048 bf16, there / back: two rows 20.6 / 12.7, eight lanes 17.7 / 10.3, four lanes of four vectors
// 17.9 / 10.9; fp32: two rows 26.0 / 28.2, eight lanes 25.5 / 28.7.
constexpr int kKeepFlight = 2;
inline bool keep_many(long long rows, int C, int sms) { return rows * groups_of(C) >= (long long)kKeepWarps * (32 / lanes_of(C)) * kKeepFlight * sms * 4; }

// Slices of the rows that the grid has along y, for CTAs that take `per` rows a round.
int slices_of(long long rows, int C, int per, int sms) {
    const int G = groups_of(C);
    const long long most = (rows + per - 1) / per;
    long long s = ((long long)sms * 16 + G - 1) / G;
    s = s < most ? s : most;
    return (int)(s < 1 ? 1 : s > 65535 ? 65535 : s);
}

template <int KIND, typename T, bool VEC, int L, int NV, int UN>
cudaError_t keep_go(const KeepArgs &a, int sms, cudaStream_t st) {
    const dim3 grid(groups_of(a.C), slices_of(a.rows, a.C, kKeepWarps * (32 / L) * UN, sms));
    keep_kernel<KIND, T, VEC, L, NV, UN><<<grid, kKeepThreads, 0, st>>>(a);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess && KIND == KEEP_GELU_BWD && a.dbias ? sum_slices(a.partial, a.dbias, a.C, nullptr, 0, a.pbf16, (int)grid.y, st) : e;
}
template <int KIND, typename T, bool VEC>
cudaError_t keep_lanes(const KeepArgs &a, int sms, cudaStream_t st) {
    const bool many = keep_many(a.rows, a.C, sms);
    constexpr int N = kKeepFlight;
    if (a.C <= 32) return many ? keep_go<KIND, T, VEC, 4, 1, N>(a, sms, st) : keep_go<KIND, T, VEC, 4, 1, 1>(a, sms, st);
    if (a.C <= 64) return many ? keep_go<KIND, T, VEC, 8, 1, N>(a, sms, st) : keep_go<KIND, T, VEC, 8, 1, 1>(a, sms, st);
    if (!many) return keep_go<KIND, T, VEC, 16, 1, 1>(a, sms, st);
    if constexpr (VEC && sizeof(T) == 2 && KIND != KEEP_GELU_FWD) return keep_go<KIND, T, VEC, 8, 2, 1>(a, sms, st);
    else return keep_go<KIND, T, VEC, 16, 1, N>(a, sms, st);
}
template <int KIND, typename T>
cudaError_t keep_vec(const KeepArgs &a, int sms, cudaStream_t st) {
    return vectors(a.C, a.x, a.y, a.dx, a.codes) ? keep_lanes<KIND, T, true>(a, sms, st) : keep_lanes<KIND, T, false>(a, sms, st);
}
template <typename T>
cudaError_t keep_kind(int kind, const KeepArgs &a, int sms, cudaStream_t st) {
    switch (kind) {
        case KEEP_FWD: return keep_vec<KEEP_FWD, T>(a, sms, st);
        case KEEP_RESTORE: return keep_vec<KEEP_RESTORE, T>(a, sms, st);
        case KEEP_GELU_FWD: return keep_vec<KEEP_GELU_FWD, T>(a, sms, st);
        default: return keep_vec<KEEP_GELU_BWD, T>(a, sms, st);
    }
}

// Warps that share a row of the LayerNorm kernels, and rows that a CTA holds at once: two groups a warp up to 256
// columns, four beyond, eight for the longest rows.
inline int ln_team(int C) { return C <= 512 ? 1 : C <= 1024 ? 2 : C <= 2048 ? 4 : 8; }
inline int ln_cta_rows(int C) { return C <= 128 ? kKeepWarps * (32 / lanes_of(C)) : kKeepWarps / ln_team(C); }

// Short rows: several of a lane in flight where there are rows enough for four CTAs on every SM.  401408 x 96 bf16, forward /
// backward: two 58 / 57 us, three 52 / 61, four 54 / 81 (registers).  Forward, bf16, whole vectors, 65 to 96 columns: four lanes hold a
// row instead, three vectors each (two exchanges a sum instead of four, and at 96 no lane without values): 40.  Not elsewhere:
// 200000 x 128 (four vectors a lane) 41 instead of 28, fp32 200000 x 96 42 instead of 33, backward 61 instead of 57 (registers).
constexpr int kLnFlightFwd = 3, kLnFlightBwd = 2;
template <bool BWD> inline int ln_flight(long long rows, int C, int sms) {
    constexpr int n = BWD ? kLnFlightBwd : kLnFlightFwd;
    return C <= 256 && rows >= (long long)n * ln_cta_rows(C) * sms * 4 ? n : 1;
}
int ln_ctas(long long rows, int per, int sms) {
    const long long need = (rows + per - 1) / per, cap = (long long)sms * 4;
    return (int)(need < cap ? need : cap);
}

template <bool BWD, typename T, bool VEC, int LR, int TEAM, int NG, int NV, int UN>
cudaError_t ln_go(const LnKeepArgs &a, int sms, cudaStream_t st) {
    const int grid = ln_ctas(a.rows, LnRow<LR, TEAM, NG, NV>::ROWS * UN, sms);
    if constexpr (BWD) {
        constexpr int TEAMS = kKeepWarps / TEAM;
        const int smem = TEAMS > 1 ? TEAMS * 2 * a.C * (int)sizeof(float) : 0;        // at most 32 KB
        ln_keep_bwd_kernel<T, VEC, LR, TEAM, NG, NV, UN><<<grid, kKeepThreads, smem, st>>>(a);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
        return sum_slices(a.partial, a.dgamma, a.C, a.dbeta, a.C, a.pbf16, grid, st);
    } else {
        ln_keep_kernel<T, VEC, LR, TEAM, NG, NV, UN><<<grid, kKeepThreads, 0, st>>>(a);
        return cudaGetLastError();
    }
}
template <bool BWD, typename T, bool VEC, int LR>
cudaError_t ln_short(const LnKeepArgs &a, int sms, cudaStream_t st) {
    constexpr int n = BWD ? kLnFlightBwd : kLnFlightFwd;
    if (ln_flight<BWD>(a.rows, a.C, sms) == 1) return ln_go<BWD, T, VEC, LR, 1, 1, 1, 1>(a, sms, st);
    if constexpr (!BWD && VEC && LR == 16 && sizeof(T) == 2)
        if (a.C <= 96) return ln_go<false, T, true, 4, 1, 1, 3, 1>(a, sms, st);
    return ln_go<BWD, T, VEC, LR, 1, 1, 1, n>(a, sms, st);
}
template <bool BWD, typename T, bool VEC>
cudaError_t ln_width(const LnKeepArgs &a, int sms, cudaStream_t st) {
    const int C = a.C;
    if (C <= 32) return ln_short<BWD, T, VEC, 4>(a, sms, st);
    if (C <= 64) return ln_short<BWD, T, VEC, 8>(a, sms, st);
    if (C <= 128) return ln_short<BWD, T, VEC, 16>(a, sms, st);
    if (C <= 256) return ln_short<BWD, T, VEC, 32>(a, sms, st);
    if (C <= 512) return ln_go<BWD, T, VEC, 32, 1, 2, 1, 1>(a, sms, st);
    if (C <= 1024) return ln_go<BWD, T, VEC, 32, 2, 2, 1, 1>(a, sms, st);
    if (C <= 2048) return ln_go<BWD, T, VEC, 32, 4, 2, 1, 1>(a, sms, st);
    if (C <= 4096) return ln_go<BWD, T, VEC, 32, 8, 2, 1, 1>(a, sms, st);
    return ln_go<BWD, T, VEC, 32, 8, 4, 1, 1>(a, sms, st);
}
template <bool BWD, typename T>
cudaError_t ln_vec(const LnKeepArgs &a, int sms, cudaStream_t st) {
    return vectors(a.C, a.x, a.y, a.dx, a.codes) ? ln_width<BWD, T, true>(a, sms, st) : ln_width<BWD, T, false>(a, sms, st);
}

}  // namespace

// (of the kernels that take fewest rows a round)
int keep_slices(long long rows, int C, int sms) { return slices_of(rows, C, kKeepWarps * (32 / lanes_of(C)), sms); }

cudaError_t keep_launch(int kind, bool bf16, const KeepArgs &a, int sms, cudaStream_t st) {
    return bf16 ? keep_kind<__nv_bfloat16>(kind, a, sms, st) : keep_kind<float>(kind, a, sms, st);
}

// (of the kernels that take fewest rows a round)
int ln_keep_ctas(long long rows, int C, int sms) { return ln_ctas(rows, ln_cta_rows(C), sms); }

cudaError_t ln_keep_launch(bool backward, bool bf16, const LnKeepArgs &a, int sms, cudaStream_t st) {
    if (backward) return bf16 ? ln_vec<true, __nv_bfloat16>(a, sms, st) : ln_vec<true, float>(a, sms, st);
    return bf16 ? ln_vec<false, __nv_bfloat16>(a, sms, st) : ln_vec<false, float>(a, sms, st);
}

}  // namespace o1d

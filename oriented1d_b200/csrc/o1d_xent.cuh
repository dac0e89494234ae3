// Softmax cross entropy of a linear classifier, without the logits.
//   l[n, v] = sum_d x[n, d] w[v, d] + b[v],  lse[n] = log sum_v exp l[n, v],  e = label smoothing,
//   loss[n] = lse[n] - (1-e) l[n, t_n] - (e/V) sum_v l[n, v],
//   G[n, v] = u_n (exp(l[n, v] - lse[n]) - (1-e) [v = t_n] - e/V),   dx = G w,  dw = G^T x,  db = G^T 1.
// Three matrix products on the tensor cores with one kernel body (xent_kernel):
//   LOGITS   tiles of x w^T stay in tensor memory; the epilogue keeps a running maximum and sum a row and writes two
//            floats a row and CTA run: the logits exist nowhere else.
//   GRAD     the same tiles once more; the epilogue turns a piece of them into G (bf16) in the workspace.
//   OUT      G w and G^T x over that piece, to the output or to fp32 sums that later pieces (and the other parts of a
//            split K axis) add to in a fixed order.
// Logits are formed twice (8NDV operations where 6NDV would do): kept between the passes they are the memory that this operator
// is there to save (4096 x 1024 x 21841 in fp32: 358 MB, and 109 us to write and read, about what the product takes), and in bf16
// they cost the softmax its accuracy.
//
// fp32 inputs are cut into three bf16 planes each (x = x0 + x1 + x2 exactly, 8 bits a plane); of the nine products of
// planes the six above 2^-24 are taken.  x0 w0 has an accumulator of its own, the five small ones share another, and
// both are added to fp32 registers every 256 of K: a tensor core adds with truncation, which over thousands of steps
// would show.
//
// Rounding: G is rounded to bf16 for bf16 inputs (2^-8 of an element at most, as dx and dw are themselves), or to two planes of it
// where that costs nothing (XENT_FINE).  Where rows differ so do these roundings, and they cancel in the sums; where rows have an
// element of G in common they do not.  The coefficient 1-e of the target is kept out: G is divided by it, so that the target's -1
// is exact, and the factor applied to the fp32 sums.  What stays is e/V of the classes that a row gives no weight, and all of G
// where logits are alike: dx and dw are then off by up to 2^-8 before their own rounding (8192 x 512 x 1000, rows sure of their
// class: e = 0.1 2.2e-3 norm-wise, e = 0.3 2.0e-3; rounding the results alone is 1.7e-3).  All sums, statistics and the loss are
// fp32 or wider.  A bf16 logit is one accumulator's sum over D, which truncates as it adds: D/16 additions, each off by up to
// 2^-23 of the sum so far (the loss of 256 x D x 200: within 9.5e-6 at D = 1024, 2.3e-5 at 2048; in fp32 1.3e-6).
#pragma once

#include "o1d_common.cuh"
#include "o1d_pair.cuh"
#include "o1d_tc.cuh"

namespace o1d {

enum : int { XENT_LOGITS = 0, XENT_GRAD, XENT_DX, XENT_DW };
// What the operands are.  XENT_FINE: bf16, but G in two planes (16 bits), so that dx and dw are as exact as their own rounding
// lets them be; taken where the products are small (see fine_of in o1d_xent.cu).
enum : int { XENT_BF16 = 0, XENT_F32, XENT_FINE };

constexpr int kXM = 128, kXK = 64;               // tile rows; K elements of a stage (one 128-byte swizzled row)
constexpr int kXFinish = 16;                     // warps that finish tiles: four a scheduler (with two, half the issue slots stayed
                                                 // empty behind the chain load, exponential, pack, store of a piece)
constexpr int kXThreads = 128 + 32 * kXFinish;   // warp 0 loads, 1 multiplies, 2 owns tensor memory, 4-19 finish tiles
constexpr int kXStaging = 2048;                  // bytes of a warp's store buffer: 32 rows of 64 bytes
constexpr int kXChunk = 4;                       // fp32: stages of one accumulation
// Tiles of 128 x 128 (fp32, whose two accumulators of 256 columns would not fit twice, and products with too few tiles to go
// round), 128 x 256, or 256 x 256 on a pair of CTAs (each loads half of either operand: a third less than 128 x 256 reads
// for the same products).  See shape_of in o1d_xent.cu.
template <int KIND, int MODE, int BN_, bool PAIR> struct XentShape {
    static constexpr int TM = PAIR ? 2 * kXM : kXM, BN = BN_;
    static constexpr int PLA = MODE == XENT_F32 ? 3 : MODE == XENT_FINE && KIND >= XENT_DX ? 2 : 1, PLB = MODE == XENT_F32 ? 3 : 1;
    static constexpr int B_COLS = PAIR ? BN / 2 : BN;               // columns that one CTA loads
    static constexpr int A_BYTES = kXM * kXK * 2, B_BYTES = B_COLS * kXK * 2, STAGE = PLA * A_BYTES + PLB * B_BYTES;
    static constexpr int STAGES = MODE == XENT_F32 ? 2 : STAGE > 32768 ? 4 : 6;
    static constexpr int SMEM = STAGES * STAGE + kXFinish * kXStaging + 256 + 1024;
};

struct XentParams {
    int M, N;                    // extents of the product
    int m_tiles, n_tiles, k_steps;
    int splits;                  // OUT: parts of the K axis
    int tiles;                   // m_tiles * n_tiles * splits
    int along_n;                 // neighbouring tiles share rows of A (the larger operand: B then stays in the L2 cache), not of B
    // LOGITS, GRAD
    const void *bias;
    int bias_bf16;
    int col0, V;                 // vocabulary index of the product's first column; size of the vocabulary
    const long long *target;     // of the product's first row
    long long ignore;
    // LOGITS: [slots][rows] of (maximum, sum) and, when smoothing, of the sum of logits; the target's logit a row
    float2 *part;
    float *part_sum, *target_logit;
    long long part_rows;
    int smooth;
    // GRAD
    const float *lse, *lse_lo, *log2p, *up;      // lse + lse_lo; of the target's probability; per-row gradient of the loss, or null
    float factor_log2, one, eps_v;   // log2(1-e), coefficient of the target, e/V; both divided by 1-e
    __nv_bfloat16 *g;
    long long g_plane;           // elements of a plane of G
    int g_ld;
    float *cols;                 // [rows / 32][cols_ld] column sums of G, or null
    long long cols_ld;
    // OUT
    void *out;                   // dx or dw (rows of N elements), or the fp32 sums of split 0
    long long split_elems;       // elements of one split's sums
    int out_kind;                // 0: bf16 result, 1: fp32 result, 2: fp32 sums, written, 3: fp32 sums, added to; 4, 5: bf16 / fp32 result from
                                 // `before`, the sums of earlier pieces, and this product
    const float *before;
    int vec;                     // rows of the output start on 16 bytes
    const float *alpha_up, *alpha_count;
    float alpha;
    int *err_flag;
};

// Gradient of the loss with respect to a row's loss where all rows share it, times the factor kept out of G.
__device__ __forceinline__ float xent_alpha(const float *up, const float *count, float f) {
    if (up) f *= __ldg(up);
    if (count) { const float c = __ldg(count); f = c > 0.f ? f / c : 0.f; }      // no row counts: nothing has a gradient
    return f;
}

__device__ __forceinline__ float exp2_fast(float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }

// The tiles of a CTA (or pair), one after the other.  Found by division once and by steps from there: a tile of a narrow product
// takes 2 us, of which the divisions of sixteen warps were a quarter.
struct XentTile {
    int m, n, split, k0, k1;
    int left;                                        // tiles still to come, this one included
    int dm, dn, dsplit;                              // a step, in tiles
};
template <int KIND>
__device__ __forceinline__ void xent_span(const XentParams &p, XentTile &t) {
    t.k0 = 0; t.k1 = p.k_steps;
    if (KIND >= XENT_DX && p.splits > 1) {
        t.k0 = (int)((long long)p.k_steps * t.split / p.splits);
        t.k1 = (int)((long long)p.k_steps * (t.split + 1) / p.splits);
    }
}
template <int KIND>
__device__ __forceinline__ XentTile xent_first(const XentParams &p, int me, int all) {
    XentTile r;
    if (KIND == XENT_LOGITS) {                       // along the vocabulary: a CTA keeps its rows' statistics in registers
        const int t = (int)((long long)me * p.tiles / all);
        r.left = (int)((long long)(me + 1) * p.tiles / all) - t;
        r.m = t / p.n_tiles; r.n = t - r.m * p.n_tiles;
        r.split = r.dm = r.dn = r.dsplit = 0;
    } else {
        const int inner = p.along_n ? p.n_tiles : p.m_tiles, mn = p.m_tiles * p.n_tiles;
        r.left = me < p.tiles ? (p.tiles - 1 - me) / all + 1 : 0;
        auto cut = [&](int t, int &m, int &n, int &split) {
            split = t / mn; t -= split * mn;
            const int o = t / inner, i = t - o * inner;
            m = p.along_n ? o : i; n = p.along_n ? i : o;
        };
        cut(me, r.m, r.n, r.split);
        cut(all, r.dm, r.dn, r.dsplit);
    }
    xent_span<KIND>(p, r);
    return r;
}
template <int KIND>
__device__ __forceinline__ void xent_next(const XentParams &p, XentTile &t) {
    t.left--;
    if (KIND == XENT_LOGITS) {
        if (++t.n == p.n_tiles) { t.n = 0; t.m++; }
        return;
    }
    t.m += t.dm; t.n += t.dn; t.split += t.dsplit;
    if (p.along_n) {                                 // n is the inner axis
        if (t.n >= p.n_tiles) { t.n -= p.n_tiles; t.m++; }
        if (t.m >= p.m_tiles) { t.m -= p.m_tiles; t.split++; }
    } else {
        if (t.m >= p.m_tiles) { t.m -= p.m_tiles; t.n++; }
        if (t.n >= p.n_tiles) { t.n -= p.n_tiles; t.split++; }
    }
    xent_span<KIND>(p, t);
}
// LOGITS: the runs of CTAs differ by one tile at most (CTA i begins at i * tiles / ctas).
// CTA whose run holds tile t.
__host__ __device__ inline int xent_owner(int t, int tiles, int ctas) { return (int)((((long long)t + 1) * ctas - 1) / tiles); }

// Moves 32 rows x 64 bytes from the lanes that own the rows to memory: `vals` are the lane's four 16-byte pieces.
// Rows go out as whole 64-byte segments.  F(row, piece, value) stores one piece.
__device__ __forceinline__ char *xent_staged(char *stage, int lane, int j) { return stage + lane * 64 + ((j ^ (lane >> 1)) & 3) * 16; }
template <typename F, typename P>
__device__ __forceinline__ void xent_transpose(char *stage, int lane, const uint4 (&vals)[4], F &&store, P &&patch) {
#pragma unroll
    for (int j = 0; j < 4; j++) *reinterpret_cast<uint4 *>(xent_staged(stage, lane, j)) = vals[j];
    patch();                                             // what the lane puts over its row
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int row = i * 8 + (lane >> 2), piece = lane & 3;
        store(row, piece, *reinterpret_cast<const uint4 *>(xent_staged(stage, row, piece)));
    }
    __syncwarp();
}
template <typename F>
__device__ __forceinline__ void xent_transpose(char *stage, int lane, const uint4 (&vals)[4], F &&store) { xent_transpose(stage, lane, vals, store, [] {}); }

// The same where rows start anywhere: lanes go along a row, an element each, so that its stores meet in as few sectors as they can
// (eight elements of four lanes a row each: dx of 84547 x 785 bf16 362 us, so 89).  F(row, column, value).
template <typename T, typename F>
__device__ __forceinline__ void xent_transpose_any(char *stage, int lane, const uint4 (&vals)[4], F &&store) {
    constexpr int W = 64 / (int)sizeof(T), V = 16 / (int)sizeof(T);      // columns; of a piece
#pragma unroll
    for (int j = 0; j < 4; j++) *reinterpret_cast<uint4 *>(xent_staged(stage, lane, j)) = vals[j];
    __syncwarp();
#pragma unroll 8
    for (int i = 0; i < W; i++) {
        const int row = i * (32 / W) + lane / W, col = lane % W;
        store(row, col, reinterpret_cast<const T *>(xent_staged(stage, row, col / V))[col % V]);
    }
    __syncwarp();
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// The next 8 bits of v, and what is left of it.  Zero is left of what is not finite.
__device__ __forceinline__ float take_bf16(float &v) {
    const float top = __uint_as_float(__float_as_uint(v) & 0xffff0000u);
    if (fabsf(v) <= 3.402823466e38f) { v -= top; return top; }
    const float r = isnan(v) ? __uint_as_float(0x7fc00000u) : top;
    v = 0.f;
    return r;
}

// Sums over the warp's lanes of 32 values each, of which a lane may have one (`at`, or -1) that is `hot` instead; in a fixed order.
// The lane gets the sum of value column_of(lane).  Through the store buffer, half of the values at a time, the target's put over
// what is there: a lane adds four rows of four columns, and three exchanges join the eight lanes of a column.  76 instructions;
// by exchanges alone 124, and 64 to put the target among the registers (xent_dense_kernel, 133200 x 96 x 150: 33.5 us and 37.5).
__device__ __forceinline__ int column_of(int lane) { return (lane & 4) * 4 + (lane & 3) * 4 + (lane >> 3 & 2) + (lane >> 3 & 1); }
__device__ __forceinline__ float column_sums(const float (&a)[32], int lane, char *stage, int at, float hot) {
    float s[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
#pragma unroll
        for (int j = 0; j < 4; j++)
            *reinterpret_cast<float4 *>(xent_staged(stage, lane, j)) = make_float4(a[h * 16 + j * 4], a[h * 16 + j * 4 + 1], a[h * 16 + j * 4 + 2], a[h * 16 + j * 4 + 3]);
        if (at >> 4 == h) reinterpret_cast<float *>(xent_staged(stage, lane, at >> 2 & 3))[at & 3] = hot;
        __syncwarp();
        float4 v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = *reinterpret_cast<const float4 *>(xent_staged(stage, i * 8 + (lane >> 2), lane & 3));
        __syncwarp();
        const float2 x = apart(add2(add2(two(v[0].x, v[0].y), two(v[1].x, v[1].y)), add2(two(v[2].x, v[2].y), two(v[3].x, v[3].y))));
        const float2 y = apart(add2(add2(two(v[0].z, v[0].w), two(v[1].z, v[1].w)), add2(two(v[2].z, v[2].w), two(v[3].z, v[3].w))));
        const bool p = lane & 16, q = lane & 8;
        const float t0 = (p ? y.x : x.x) + __shfl_xor_sync(0xffffffffu, p ? x.x : y.x, 16);
        const float t1 = (p ? y.y : x.y) + __shfl_xor_sync(0xffffffffu, p ? x.y : y.y, 16);
        s[h] = (q ? t1 : t0) + __shfl_xor_sync(0xffffffffu, q ? t0 : t1, 8);
    }
    const bool u = lane & 4;
    return (u ? s[1] : s[0]) + __shfl_xor_sync(0xffffffffu, u ? s[0] : s[1], 4);
}

__device__ __forceinline__ float max3(float a, float b, float c) { float r; asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }
// a[at], 0 <= at < 32, by halves.
__device__ __forceinline__ float pick(const float (&a)[32], int at) {
    float t[16];
#pragma unroll
    for (int i = 0; i < 16; i++) t[i] = at & 16 ? a[i + 16] : a[i];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < o; i++) t[i] = at & o ? t[i + o] : t[i];
    return t[0];
}

// What a row's gradient G needs besides its logits.  G = u (p - (1-e) [target] - e/V), all over 1-e.  The target's value is formed
// once a row, as expm1 of its own exponent (p - 1 without cancellation), and put over what the other columns' formula gives
// where the row is in shared memory on its way out: in registers it would cost an instruction or two for every column.
struct XentRow {
    long long tgt;               // -1: none of these columns
    float lse, lse_lo;           // what the exponents are taken from; +inf for a row without a loss, whose G then is zero
    float eps, scale, hot;
    bool bad;                    // a row without a loss whose logits are not finite: nothing comes of it either
};
struct XentAhead { long long tgt; float lse, lse_lo, log2p, scale; };      // as they are stored
__device__ __forceinline__ XentAhead xent_fetch(long long row, const XentParams &p) {
    XentAhead f{p.ignore, __int_as_float(0x7f800000), 0.f, 0.f, 1.f};
    if (row < p.M) {
        f.tgt = __ldg(p.target + row);
        f.lse = __ldg(p.lse + row);
        f.lse_lo = __ldg(p.lse_lo + row);
        f.log2p = __ldg(p.log2p + row);
        if (p.up) f.scale = __ldg(p.up + row);
    }
    return f;
}
__device__ __forceinline__ XentRow xent_row(const XentAhead &f, const XentParams &p) {
    const bool ignored = f.tgt == p.ignore, none = f.tgt < 0 || f.tgt >= p.V;
    XentRow r;
    r.tgt = ignored || none || p.one == 0.f ? -1 : f.tgt - p.col0;
    r.lse = ignored ? __int_as_float(0x7f800000) : none ? __int_as_float(0x7fffffff) : f.lse;      // no such class: NaN, not silence
    r.lse_lo = f.lse_lo + p.factor_log2;
    r.bad = ignored && !(fabsf(f.lse) <= 3.402823466e38f);
    r.eps = ignored || !p.smooth ? 0.f : p.eps_v;
    r.scale = ignored ? 0.f : f.scale;
    r.hot = (expm1f(0.6931471805599453f * (f.log2p - p.factor_log2)) - r.eps) * r.scale;
    return r;
}
// G of 32 columns, from c0 on, but for the target: from exponents log2 p.
__device__ __forceinline__ void xent_gradient(float (&a)[32], int c0, const XentRow &r, const XentParams &p) {
#pragma unroll
    for (int i = 0; i < 32; i++) a[i] = exp2_fast(a[i]);
    if (p.smooth) {
#pragma unroll
        for (int i = 0; i < 32; i++) a[i] -= c0 + i < p.N ? r.eps : 0.f;
    }
    if (p.up) {
#pragma unroll
        for (int i = 0; i < 32; i++) a[i] *= r.scale;
    }
    if (__any_sync(0xffffffffu, r.bad)) {
#pragma unroll
        for (int i = 0; i < 32; i++) a[i] = r.bad ? 0.f : a[i];
    }
}
// Of 32 columns from c0 on, which one is the target; or -1.
__device__ __forceinline__ int xent_at(const XentRow &r, int c0) { const long long off = r.tgt - c0; return off >= 0 && off < 32 ? (int)off : -1; }
// 32 columns of a bf16 result of rows of `n` from a lane's row of values, for the warp's 32 rows from r0 on.  vec: rows start on vectors.
__device__ __forceinline__ void xent_store(__nv_bfloat16 *to, char *stage, int lane, const float (&a)[32], float alpha, int r0, int rows, int c0, int n, int vec) {
    uint4 out[4];
    uint32_t *o = reinterpret_cast<uint32_t *>(out);
#pragma unroll
    for (int i = 0; i < 16; i++) o[i] = pack_bf16(alpha * a[2 * i], alpha * a[2 * i + 1]);
    if (vec)
        xent_transpose(stage, lane, out, [&](int r, int piece, uint4 val) {
            const int c = c0 + piece * 8;
            if (r0 + r < rows && c < n) *reinterpret_cast<uint4 *>(to + (long long)(r0 + r) * n + c) = val;
        });
    else
        xent_transpose_any<__nv_bfloat16>(stage, lane, out, [&](int r, int c, __nv_bfloat16 val) {
            if (r0 + r < rows && c0 + c < n) to[(long long)(r0 + r) * n + c0 + c] = val;
        });
}

template <int KIND, int MODE, int BN, bool PAIR>
__global__ void __launch_bounds__(kXThreads, 1)
xent_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const XentParams p) {
    using S = XentShape<KIND, MODE, BN, PAIR>;
    constexpr bool SPLIT = MODE == XENT_F32;
    constexpr int GPL = SPLIT ? 3 : MODE == XENT_FINE ? 2 : 1;      // planes of G
    constexpr bool A_MN = KIND == XENT_DW, B_MN = KIND == XENT_DX || KIND == XENT_DW;
    constexpr int PIECES = BN / 128;                 // of 32 columns, for each of the four warps that share 32 rows
    constexpr uint32_t INSTR = tc::instruction(S::TM, BN, A_MN, B_MN);
    extern __shared__ __align__(1024) unsigned char raw[];
    unsigned char *smem = raw + ((1024u - (tc::smem_addr(raw) & 1023u)) & 1023u);
    char *staging = reinterpret_cast<char *>(smem + S::STAGES * S::STAGE);
    uint64_t *full = reinterpret_cast<uint64_t *>(staging + kXFinish * kXStaging), *empty = full + S::STAGES;
    uint64_t *done = empty + S::STAGES, *taken = done + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(taken + 2);
    volatile int *dead = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // PAIR: `me` and `all` count pairs; rank 0 of a pair issues the products
    const int rank = PAIR ? (int)tc::cluster_rank() : 0, me = PAIR ? blockIdx.x >> 1 : blockIdx.x, all = PAIR ? gridDim.x >> 1 : gridDim.x;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::STAGES; i++) { tc::bar_init(full + i, 1); tc::bar_init(empty + i, 1); }
        for (int i = 0; i < 2; i++) { tc::bar_init(done + i, 1); tc::bar_init(taken + i, PAIR ? 2 * kXFinish : kXFinish); }
        *dead = 0;
        tc::bar_init_fence();
        tc::tma_prefetch(&map_a);
        tc::tma_prefetch(&map_b);
    }
    if (warp == 2) tc::tmem_alloc<PAIR>(tmem_slot, 512);
    tc::fence_before();
    if (PAIR) tc::cluster_sync(); else __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0 && lane == 0) {                                   // ---- loads
        int stage = 0, issued = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (XentTile w = xent_first<KIND>(p, me, all); ok && w.left > 0; xent_next<KIND>(p, w)) {
            for (int k = w.k0; k < w.k1; k++) {
                if (!(ok = tc::bar_wait(empty + stage, phase ^ 1, dead, p.err_flag))) break;
                unsigned char *a = smem + stage * S::STAGE, *b = a + S::PLA * S::A_BYTES;
                if (rank == 0) tc::bar_expect(full + stage, PAIR ? 2 * S::STAGE : S::STAGE);
                const uint32_t bar = PAIR ? tc::in_cta(full + stage, 0) : 0;
                auto load = [&](void *dst, const CUtensorMap *map, int x, int y, int z) {
                    if constexpr (PAIR) tc::tma_load3_pair(dst, map, bar, x, y, z);
                    else tc::tma_load3(dst, map, full + stage, x, y, z);
                };
                const int row = w.m * S::TM + rank * kXM, col = w.n * BN + rank * S::B_COLS;
#pragma unroll
                for (int pl = 0; pl < S::PLA; pl++) {
                    if (A_MN) {
#pragma unroll
                        for (int j = 0; j < kXM / 64; j++) load(a + pl * S::A_BYTES + j * 8192, &map_a, row + j * 64, k * kXK, pl);
                    } else {
                        load(a + pl * S::A_BYTES, &map_a, k * kXK, row, pl);
                    }
                }
#pragma unroll
                for (int pl = 0; pl < S::PLB; pl++) {
                    if (B_MN) {
#pragma unroll
                        for (int j = 0; j < S::B_COLS / 64; j++) load(b + pl * S::B_BYTES + j * 8192, &map_b, col + j * 64, k * kXK, pl);
                    } else {
                        load(b + pl * S::B_BYTES, &map_b, k * kXK, col, pl);
                    }
                }
                issued++;
                if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
            }
        }
        if (!ok && rank == 0) {                                     // copies in flight (a pair's all count here) end before the CTA does
            for (int i = 0; i < S::STAGES && i < issued; i++) {
                stage = stage == 0 ? S::STAGES - 1 : stage - 1;
                if (stage == S::STAGES - 1) phase ^= 1;
                tc::bar_drain(full + stage, phase);
            }
        }
    } else if (warp == 1 && lane == 0 && rank == 0) {               // ---- products
        int stage = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true;
        for (XentTile w = xent_first<KIND>(p, me, all); ok && w.left > 0; xent_next<KIND>(p, w)) {
            for (int c = w.k0; ok && c < w.k1; c += SPLIT ? kXChunk : w.k1 - w.k0) {
                const int c_end = SPLIT ? min(c + kXChunk, w.k1) : w.k1;
                if (!(ok = tc::bar_wait(taken + acc, acc_phase ^ 1, dead, p.err_flag))) break;
                tc::fence_after();
                const uint32_t d = tmem + acc * 256;
                for (int k = c; k < c_end; k++) {
                    if (!(ok = tc::bar_wait(full + stage, phase, dead, p.err_flag))) break;
                    tc::fence_after();
                    unsigned char *a = smem + stage * S::STAGE, *b = a + S::PLA * S::A_BYTES;
                    uint64_t da[S::PLA], db[S::PLB];
#pragma unroll
                    for (int pl = 0; pl < S::PLA; pl++) da[pl] = tc::operand(a + pl * S::A_BYTES, A_MN ? 8192 : 16, 1024);
#pragma unroll
                    for (int pl = 0; pl < S::PLB; pl++) db[pl] = tc::operand(b + pl * S::B_BYTES, B_MN ? 8192 : 16, 1024);
#pragma unroll
                    for (int kk = 0; kk < kXK / 16; kk++) {         // 16 of K: 32 bytes of a K-major row, or 16 rows
                        const uint64_t oa = kk * (A_MN ? 128 : 2), ob = kk * (B_MN ? 128 : 2);
                        const bool add = k > c || kk > 0;
                        if constexpr (S::PLA == 2) tc::mma<PAIR>(d, da[1] + oa, db[0] + ob, INSTR, add);
                        tc::mma<PAIR>(d, da[0] + oa, db[0] + ob, INSTR, add || S::PLA == 2);
                        if constexpr (SPLIT) {
                            tc::mma<PAIR>(d + 128, da[0] + oa, db[2] + ob, INSTR, add);
                            tc::mma<PAIR>(d + 128, da[1] + oa, db[1] + ob, INSTR, true);
                            tc::mma<PAIR>(d + 128, da[2] + oa, db[0] + ob, INSTR, true);
                            tc::mma<PAIR>(d + 128, da[0] + oa, db[1] + ob, INSTR, true);
                            tc::mma<PAIR>(d + 128, da[1] + oa, db[0] + ob, INSTR, true);
                        }
                    }
                    tc::commit<PAIR>(empty + stage);
                    if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
                }
                if (!ok) break;
                tc::commit<PAIR>(done + acc);
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1;
            }
        }
        if (!ok) {                                                  // products in flight read shared memory: wait for them
            tc::commit<PAIR>(done + acc);
            tc::bar_drain(done + acc, acc_phase);
        }
    } else if (warp >= 4) {                                         // ---- epilogue: a thread owns a quarter of a row
        const int quarter = warp & 3, part = (warp - 4) >> 2;
        char *stage = staging + (warp - 4) * kXStaging;
        const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
        // The four warps of 32 rows take every fourth piece of 32 columns, each starting one further with every tile: where the
        // columns end inside a tile, no warp has more to do than another (133200 x 150 classes have 5 pieces a tile).
        auto piece_of = [&](int pc, int tile) { return 4 * pc + ((part + tile) & 3); };
        int acc = 0, m_now = -1, tile = 0;                          // tile: of this CTA
        uint32_t acc_phase = 0;
        bool ok = true;
        // LOGITS: running maximum and sum of the row's columns that this warp sees, in units of log2
        float mx = 0.f, sum = 0.f, total = 0.f;
        long long tgt = -1;
        XentRow mine{};                                              // GRAD
        float alpha = 1.f;
        if (KIND >= XENT_DX && (p.out_kind < 2 || p.out_kind > 3)) alpha = xent_alpha(p.alpha_up, p.alpha_count, p.alpha);

        auto release = [&](int i) {                                 // the accumulator may be written again
            if (rank == 0) tc::bar_arrive(taken + i); else tc::bar_arrive_in(tc::in_cta(taken + i, 0));
        };
        int run = 0;                                                // LOGITS: of the runs that share the row tile, which this one is
        auto flush = [&]() {
            const long long row = (long long)m_now * S::TM + rank * kXM + quarter * 32 + lane;
            if (row >= p.M) return;
            const int slot = run * 4 + part;
            p.part[(long long)slot * p.part_rows + row] = make_float2(mx, sum);
            if (p.smooth) p.part_sum[(long long)slot * p.part_rows + row] = total;
        };

        // What a tile needs from memory, fetched while the one before it is worked on: bits as they are stored, since any arithmetic
        // on them here would wait for them.
        struct Ahead { XentAhead row; uint32_t bias[PIECES]; };
        auto fetch = [&](const XentTile &w, int tile) {
            Ahead f{};
            if (KIND > XENT_GRAD || w.left <= 0) return f;
            const long long row = (long long)w.m * S::TM + rank * kXM + quarter * 32 + lane;
            if (KIND == XENT_GRAD) f.row = xent_fetch(row, p);
            else f.row.tgt = row < p.M ? __ldg(p.target + row) : p.ignore;
#pragma unroll
            for (int i = 0; i < PIECES; i++) {
                const int c = w.n * BN + piece_of(i, tile) * 32 + lane;
                f.bias[i] = 0u;
                if (p.bias && c < p.N) {
                    if (p.bias_bf16) f.bias[i] = __ldg(static_cast<const unsigned short *>(p.bias) + p.col0 + c);
                    else f.bias[i] = __ldg(static_cast<const uint32_t *>(p.bias) + p.col0 + c);
                }
            }
            return f;
        };
        XentTile coming = xent_first<KIND>(p, me, all);
        if (KIND == XENT_LOGITS) run = me - xent_owner(coming.m * p.n_tiles, p.tiles, all);
        Ahead next = fetch(coming, 0);
        for (; ok && coming.left > 0; tile++) {
            const XentTile w = coming;
            xent_next<KIND>(p, coming);
            const int r0 = w.m * S::TM + rank * kXM + quarter * 32, row = r0 + lane, n0 = w.n * BN;
            float bias[PIECES];
            if constexpr (KIND <= XENT_GRAD) {
                if (w.m != m_now) {
                    if (KIND == XENT_LOGITS && m_now >= 0) { flush(); run = 0; }      // the next row tile begins here
                    m_now = w.m;
                    mx = __int_as_float(0xff800000); sum = 0.f; total = 0.f;
                }
                tgt = next.row.tgt;
                if (KIND == XENT_GRAD) mine = xent_row(next.row, p);
                // in units of log2; -inf where the vocabulary ends, so that those columns weigh nothing
#pragma unroll
                for (int i = 0; i < PIECES; i++)
                    bias[i] = n0 + piece_of(i, tile) * 32 + lane < p.N ? 1.4426950408889634f * __uint_as_float(p.bias_bf16 ? next.bias[i] << 16 : next.bias[i])
                                                                      : __int_as_float(0xff800000);
                next = fetch(coming, tile + 1);
            }
            float v[SPLIT ? PIECES : 1][32];
            if constexpr (SPLIT) {
#pragma unroll
                for (int pc = 0; pc < PIECES; pc++)
#pragma unroll
                    for (int i = 0; i < 32; i++) v[pc][i] = 0.f;
                for (int c = w.k0; c < w.k1; c += kXChunk) {
                    ok = __all_sync(0xffffffffu, tc::bar_wait(done + acc, acc_phase, dead, p.err_flag));
                    if (!ok) break;
                    tc::fence_after();
#pragma unroll
                    for (int pc = 0; pc < PIECES; pc++)
#pragma unroll
                        for (int part_sum = 1; part_sum >= 0; part_sum--) {          // the five small products, then x0 w0
                            uint32_t r[32];
                            tc::tmem_load32(lane_base + acc * 256 + part_sum * 128 + piece_of(pc, tile) * 32, r);
                            tc::tmem_wait32(r);
#pragma unroll
                            for (int i = 0; i < 32; i++) v[pc][i] += __uint_as_float(r[i]);
                        }
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) release(acc);
                    acc ^= 1;
                    if (acc == 0) acc_phase ^= 1;
                }
            } else {
                ok = __all_sync(0xffffffffu, tc::bar_wait(done + acc, acc_phase, dead, p.err_flag));
                if (ok) tc::fence_after();
            }
            if (!ok) break;
#pragma unroll
            for (int pc = 0; pc < PIECES; pc++) {
                float (&a)[32] = v[SPLIT ? pc : 0];
                const int c0 = n0 + piece_of(pc, tile) * 32;        // first column of the piece
                const bool some = c0 < (KIND == XENT_GRAD ? p.g_ld : p.N);      // the same for the whole warp
                if constexpr (!SPLIT) {
                    if (some) {
                        uint32_t r[32];
                        tc::tmem_load32(lane_base + acc * 256 + piece_of(pc, tile) * 32, r);
                        tc::tmem_wait32(r);
#pragma unroll
                        for (int i = 0; i < 32; i++) a[i] = __uint_as_float(r[i]);
                    }
                    if (pc == PIECES - 1) {
                        tc::fence_before();
                        __syncwarp();
                        if (lane == 0) release(acc);
                        acc ^= 1;
                        if (acc == 0) acc_phase ^= 1;
                    }
                }
                if (!some) continue;
                if constexpr (KIND <= XENT_GRAD) {
                    // logits in units of log2; the piece's bias through the store buffer, from lane i to every lane's value i
                    const F2 log2e = both(1.4426950408889634f);
                    float *bs = reinterpret_cast<float *>(stage);
                    bs[lane] = bias[pc];
                    __syncwarp();
                    // fp32: the piece's exponents relative to `ref` (the row's greatest so far, or lse in two parts).  The product is
                    // taken from ref in one operation, so that what is rounded is small where it counts.
                    auto exponents = [&](float ref, float lo) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 b = *reinterpret_cast<const float4 *>(bs + i);
                            const F2 u = add2(fma2(two(a[i], a[i + 1]), log2e, both(-ref)), add2(two(b.x, b.y), both(-lo)));
                            const F2 v = add2(fma2(two(a[i + 2], a[i + 3]), log2e, both(-ref)), add2(two(b.z, b.w), both(-lo)));
                            a[i] = apart(u).x; a[i + 1] = apart(u).y; a[i + 2] = apart(v).x; a[i + 3] = apart(v).y;
                        }
                        __syncwarp();
                    };
                    float top = mx;                                  // LOGITS
                    if constexpr (SPLIT && KIND == XENT_GRAD) {
                        exponents(mine.lse, mine.lse_lo);
                    } else {
                        float top2 = __int_as_float(0xff800000);
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 b = *reinterpret_cast<const float4 *>(bs + i);
                            const float2 u = apart(fma2(two(a[i], a[i + 1]), log2e, two(b.x, b.y))), v = apart(fma2(two(a[i + 2], a[i + 3]), log2e, two(b.z, b.w)));
                            if constexpr (KIND == XENT_LOGITS) {
                                top = max3(top, u.x, u.y);
                                top2 = max3(top2, v.x, v.y);
                                if (p.smooth) {
                                    const int left = p.N - (c0 + i);
                                    total += ((left > 0 ? u.x : 0.f) + (left > 1 ? u.y : 0.f)) + ((left > 2 ? v.x : 0.f) + (left > 3 ? v.y : 0.f));
                                }
                            }
                            if constexpr (!SPLIT) { a[i] = u.x; a[i + 1] = u.y; a[i + 2] = v.x; a[i + 3] = v.y; }
                        }
                        top = fmaxf(top, top2);
                        if (!SPLIT) __syncwarp();
                    }
                    if constexpr (KIND == XENT_LOGITS) {
                        const long long off = tgt - p.col0 - c0;     // where the target lies in this piece
                        const int at = off >= 0 && off < 32 ? (int)off : -1;
                        if (__any_sync(0xffffffffu, at >= 0)) {
                            float l = pick(a, at);
                            if (SPLIT) l = fmaf(l, 1.4426950408889634f, bs[at & 31]);
                            if (at >= 0 && row < p.M) p.target_logit[row] = l;
                        }
                        const float ref = top == __int_as_float(0xff800000) ? 0.f : top;
                        F2 s0 = both(0.f), s1 = both(0.f);
                        if constexpr (SPLIT) exponents(ref, 0.f);
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            float2 u = make_float2(a[i], a[i + 1]), v = make_float2(a[i + 2], a[i + 3]);
                            if constexpr (!SPLIT) { u = apart(add2(two(u.x, u.y), both(-ref))); v = apart(add2(two(v.x, v.y), both(-ref))); }
                            s0 = add2(s0, two(exp2_fast(u.x), exp2_fast(u.y)));
                            s1 = add2(s1, two(exp2_fast(v.x), exp2_fast(v.y)));
                        }
                        const float2 s2 = apart(add2(s0, s1));
                        sum = sum * exp2_fast(mx - ref) + (s2.x + s2.y);
                        mx = top;
                    } else {
                        if constexpr (!SPLIT) {
                            const F2 l = both(-(mine.lse + mine.lse_lo));
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                const float2 u = apart(add2(two(a[i], a[i + 1]), l));
                                a[i] = u.x;
                                a[i + 1] = u.y;
                            }
                        }
                        xent_gradient(a, c0, mine, p);
                        const int at = xent_at(mine, c0);
                        if (p.cols && r0 < p.M) p.cols[(long long)(r0 >> 5) * p.cols_ld + c0 + column_of(lane)] = column_sums(a, lane, stage, at, mine.hot);
                        float hot = mine.hot;
#pragma unroll
                        for (int pl = 0; pl < GPL; pl++) {
                            uint4 out[4];
                            uint32_t *o = reinterpret_cast<uint32_t *>(out);
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                if constexpr (SPLIT) {
                                    const float lo = take_bf16(a[2 * i]), hi = take_bf16(a[2 * i + 1]);
                                    o[i] = __float_as_uint(lo) >> 16 | (__float_as_uint(hi) & 0xffff0000u);
                                } else {
                                    o[i] = pack_bf16(a[2 * i], a[2 * i + 1]);
                                    if (GPL > 1) {
                                        a[2 * i] -= __uint_as_float(o[i] << 16);
                                        a[2 * i + 1] -= __uint_as_float(o[i] & 0xffff0000u);
                                    }
                                }
                            }
                            const __nv_bfloat16 hot_now = __float2bfloat16_rn(SPLIT ? take_bf16(hot) : hot);
                            if (!SPLIT) hot -= __bfloat162float(hot_now);
                            __nv_bfloat16 *to = p.g + pl * p.g_plane + c0;
                            xent_transpose(stage, lane, out, [&](int r, int piece, uint4 val) {
                                if (r0 + r < p.M) *reinterpret_cast<uint4 *>(to + (long long)(r0 + r) * p.g_ld + piece * 8) = val;
                            }, [&] { if (at >= 0) reinterpret_cast<__nv_bfloat16 *>(xent_staged(stage, lane, at >> 3))[at & 7] = hot_now; });
                        }
                    }
                } else {
                    if (p.out_kind == 0) {
                        xent_store(static_cast<__nv_bfloat16 *>(p.out), stage, lane, a, alpha, r0, p.M, c0, p.N, p.vec);
                    } else {
                        float *to = static_cast<float *>(p.out) + (p.out_kind == 2 || p.out_kind == 3 ? w.split * p.split_elems : 0);
                        const float *before = p.out_kind >= 4 ? p.before : to;
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            uint4 out[4];
                            float *o = reinterpret_cast<float *>(out);
#pragma unroll
                            for (int i = 0; i < 16; i++) o[i] = p.out_kind == 1 ? alpha * a[h * 16 + i] : a[h * 16 + i];
                            const float f = p.out_kind >= 4 ? alpha : 1.f;      // (of what is the result of a sum; kind 1 has it already)
                            if (!p.vec) {
                                xent_transpose_any<float>(stage, lane, out, [&](int r, int col, float x) {
                                    const int c = c0 + h * 16 + col;
                                    if (r0 + r >= p.M || c >= p.N) return;
                                    const long long at = (long long)(r0 + r) * p.N + c;
                                    if (p.out_kind >= 3) x += before[at];
                                    if (p.out_kind == 4) static_cast<__nv_bfloat16 *>(p.out)[at] = __float2bfloat16_rn(f * x);
                                    else to[at] = f * x;
                                });
                                continue;
                            }
                            xent_transpose(stage, lane, out, [&](int r, int piece, uint4 val) {
                                const int c = c0 + h * 16 + piece * 4;
                                if (r0 + r >= p.M || c >= p.N) return;
                                const long long at = (long long)(r0 + r) * p.N + c;
                                float x[4] = {__uint_as_float(val.x), __uint_as_float(val.y), __uint_as_float(val.z), __uint_as_float(val.w)};
                                if (p.out_kind >= 3) {
                                    const float4 old = *reinterpret_cast<const float4 *>(before + at);
                                    x[0] += old.x; x[1] += old.y; x[2] += old.z; x[3] += old.w;
                                }
                                if (p.out_kind == 4)
                                    *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(p.out) + at) =
                                        make_uint2(pack_bf16(f * x[0], f * x[1]), pack_bf16(f * x[2], f * x[3]));
                                else *reinterpret_cast<float4 *>(to + at) = make_float4(f * x[0], f * x[1], f * x[2], f * x[3]);
                            });
                        }
                    }
                }
            }
        }
        if (KIND == XENT_LOGITS && ok && m_now >= 0) flush();
    }
    tc::fence_before();
    if (PAIR) tc::cluster_sync(); else __syncthreads();             // a pair ends together: either reads and signals in the other
    tc::fence_after();
    if (warp == 2) tc::tmem_free<PAIR>(tmem, 512);
}

// One matrix as the bf16 planes that tensor copies read: fp32 cut into three, bf16 whose rows do not start on 16 bytes
// copied.  planes: [3 or 1][rows][ld], ld a multiple of 8 (what lies past D is never read).  A warp a row; a lane writes a vector of a
// plane, from one load where the rows of x start on vectors (`vec`), else from an element each.
template <typename T>
__global__ void __launch_bounds__(256)
xent_planes_kernel(const T *__restrict__ x, __nv_bfloat16 *__restrict__ planes, long long rows, int D, int ld, int vec) {
    const long long plane = rows * ld;
    const int lane = threadIdx.x & 31;
    for (long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += (long long)gridDim.x * 8) {
        const T *from = x + r * D;
        __nv_bfloat16 *to = planes + r * ld;
        if constexpr (sizeof(T) == 4) {
#pragma unroll 2
            for (int c = lane * 4; c < D; c += 128) {
                float v[4];
                if (vec) {
                    const float4 q = __ldg(reinterpret_cast<const float4 *>(from + c));
                    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) v[i] = c + i < D ? __ldg(from + c + i) : 0.f;
                }
#pragma unroll
                for (int pl = 0; pl < 3; pl++) {
                    uint32_t b[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) b[i] = __float_as_uint(take_bf16(v[i]));                  // exact: eight bits each
                    *reinterpret_cast<uint2 *>(to + pl * plane + c) = make_uint2(b[0] >> 16 | (b[1] & 0xffff0000u), b[2] >> 16 | (b[3] & 0xffff0000u));
                }
            }
        } else {
            for (int c = lane * 8; c < D; c += 256) {
                uint32_t v[8];
                const unsigned short *p = reinterpret_cast<const unsigned short *>(from) + c;
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = c + i < D ? __ldg(p + i) : 0;
                *reinterpret_cast<uint4 *>(to + c) = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
            }
        }
    }
}

// LOGITS for up to eight rows (an evaluation of single images): a tile of 128 rows would be nearly all padding, and fp32 would
// be cut into planes first.  What counts is to read w once, over all SMs: a warp takes CU classes at a time, its lanes 16 bytes
// each, with the rows of x in shared memory, fp32 sums.  Lane n keeps the statistics of row n; a slot for each CTA.
// Measured, one row, 768 x 1000 fp32: 5.3 us; tiles and planes 22 us.
constexpr int kFewRows = 8, kFewBytes = 32768;         // rows; bytes of x in shared memory
template <typename T, int NR, bool VEC>
__global__ void __launch_bounds__(256)
xent_few_kernel(const T *__restrict__ x, const T *__restrict__ w, const XentParams p, int D) {
    constexpr int CU = NR == 8 ? 2 : 4, VE = 16 / (int)sizeof(T);
    extern __shared__ __align__(16) float few_x[];         // [NR][D4], D4 = D to a multiple of 8
    __shared__ float stats[3][8][kFewRows];
    const int D4 = (D + 7) & ~7, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = threadIdx.x; i < NR * D4; i += 256) {
        const int n = i / D4, c = i - n * D4;
        few_x[i] = n < p.M && c < D ? ld(x + (long long)n * D + c) : 0.f;
    }
    __syncthreads();
    const int row = lane < NR && lane < p.M ? lane : -1;
    const long long tgt = row >= 0 ? __ldg(p.target + row) : -1;
    float mx = __int_as_float(0xff800000), sum = 0.f, total = 0.f;
    for (int v0 = (blockIdx.x * 8 + warp) * CU; v0 < p.V; v0 += gridDim.x * 8 * CU) {
        float acc[CU][NR];
#pragma unroll
        for (int c = 0; c < CU; c++)
#pragma unroll
            for (int n = 0; n < NR; n++) acc[c][n] = 0.f;
        if constexpr (VEC) {
#pragma unroll 2
            for (int d = lane * VE; d < D; d += 32 * VE) {
                float f[CU][VE];
#pragma unroll
                for (int c = 0; c < CU; c++) {
                    const uint4 q = v0 + c < p.V ? __ldg(reinterpret_cast<const uint4 *>(w + (long long)(v0 + c) * D + d)) : make_uint4(0u, 0u, 0u, 0u);
                    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if constexpr (sizeof(T) == 4) f[c][i] = __uint_as_float(u[i]);
                        else { f[c][2 * i] = __uint_as_float(u[i] << 16); f[c][2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
                    }
                }
#pragma unroll
                for (int n = 0; n < NR; n++)
#pragma unroll
                    for (int i = 0; i < VE; i += 4) {
                        const float4 a = *reinterpret_cast<const float4 *>(few_x + n * D4 + d + i);
#pragma unroll
                        for (int c = 0; c < CU; c++)
                            acc[c][n] = fmaf(f[c][i], a.x, fmaf(f[c][i + 1], a.y, fmaf(f[c][i + 2], a.z, fmaf(f[c][i + 3], a.w, acc[c][n]))));
                    }
            }
        } else {
            for (int d = lane; d < D; d += 32)
#pragma unroll
                for (int c = 0; c < CU; c++) {
                    const float f = v0 + c < p.V ? ld(w + (long long)(v0 + c) * D + d) : 0.f;
#pragma unroll
                    for (int n = 0; n < NR; n++) acc[c][n] = fmaf(f, few_x[n * D4 + d], acc[c][n]);
                }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int c = 0; c < CU; c++)
#pragma unroll
                for (int n = 0; n < NR; n++) acc[c][n] += __shfl_xor_sync(0xffffffffu, acc[c][n], o);
#pragma unroll
        for (int c = 0; c < CU; c++) {
            if (v0 + c >= p.V) break;
            float l = acc[c][0];
#pragma unroll
            for (int n = 1; n < NR; n++) l = lane == n ? acc[c][n] : l;
            l *= 1.4426950408889634f;
            if (p.bias) l += 1.4426950408889634f * ld_param(p.bias, v0 + c, p.bias_bf16);
            if (tgt == v0 + c) p.target_logit[row] = l;
            total += l;
            const float top = fmaxf(mx, l), ref = top == __int_as_float(0xff800000) ? 0.f : top;
            sum = sum * exp2_fast(mx - ref) + exp2_fast(l - ref);
            mx = top;
        }
    }
    if (lane < NR) { stats[0][warp][lane] = mx; stats[1][warp][lane] = sum; stats[2][warp][lane] = total; }
    __syncthreads();
    if (threadIdx.x < NR && threadIdx.x < p.M) {
        const int n = threadIdx.x;
        float top = stats[0][0][n], s = 0.f, t = 0.f;
#pragma unroll
        for (int k = 1; k < 8; k++) top = fmaxf(top, stats[0][k][n]);
        const float ref = top == __int_as_float(0xff800000) ? 0.f : top;
#pragma unroll
        for (int k = 0; k < 8; k++) { s += stats[1][k][n] * exp2_fast(stats[0][k][n] - ref); t += stats[2][k][n]; }
        p.part[(long long)blockIdx.x * p.part_rows + n] = make_float2(top, s);
        if (p.smooth) p.part_sum[(long long)blockIdx.x * p.part_rows + n] = t;
    }
}

// Loss of every row from the statistics of its tiles' runs, and lse (in units of log2) for the backward pass; L lanes a row.  Each
// block also sums its rows' losses and counts the rows that have one; a block alone finishes the reduction.
struct XentRows {
    const float2 *part;
    const float *part_sum, *target_logit;
    const long long *target;
    long long ignore, rows;
    float smoothing;
    int V, tile_rows, n_tiles, tiles, units;     // as the runs were cut; tile_rows 0: `slots` for every row
    int slots, mean;
    float *lse, *loss_rows, *loss, *count;       // loss_rows, or loss and count
    double2 *sums;
};
template <int L>
__global__ void __launch_bounds__(1024)
xent_rows_kernel(const XentRows a) {
    const long long row = ((long long)blockIdx.x * blockDim.x + threadIdx.x) / L;
    const int lane = threadIdx.x % L;
    const bool real = row < a.rows;
    int slots = real ? a.slots : 0;
    if (real && a.tile_rows) {
        const int m = (int)(row / a.tile_rows);
        slots = 4 * (xent_owner((m + 1) * a.n_tiles - 1, a.tiles, a.units) - xent_owner(m * a.n_tiles, a.tiles, a.units) + 1);
    }
    float top = __int_as_float(0xff800000), total = 0.f, sum = 0.f;
    for (int s = lane; s < slots; s += L) top = fmaxf(top, a.part[s * a.rows + row].x);
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float ref = top == __int_as_float(0xff800000) ? 0.f : top;
    for (int s = lane; s < slots; s += L) {
        const float2 v = a.part[s * a.rows + row];
        sum += v.y * exp2f(v.x - ref);
        if (a.smoothing > 0.f) total += a.part_sum[s * a.rows + row];
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    double loss = 0., counted = 0.;
    if (real && lane == 0) {
        // lse = ref + log2(sum), as two floats; the loss, and log2 of the target's probability, from its parts (where the target is the greatest, ref is its logit)
        const float ls = log2f(sum), hi = ref + ls;
        if (a.lse) {
            const float r1 = hi - ls;
            a.lse[row] = hi;
            a.lse[a.rows + row] = fabsf(hi) <= 3.402823466e38f ? (ref - r1) + (ls - (hi - r1)) : 0.f;
        }
        const long long t = a.target[row];
        float out = 0.f, log2p = 0.f;
        if (t != a.ignore) {
            if (t < 0 || t >= a.V) out = __int_as_float(0x7fffffff);
            else {
                out = (ref - a.target_logit[row]) + ls;
                log2p = -out;
                if (a.smoothing != 0.f) {
                    out = a.smoothing < 1.f ? (1.f - a.smoothing) * out : 0.f;
                    out += a.smoothing * ((ref - total / (float)a.V) + ls);
                }
                out *= 0.6931471805599453f;
            }
            loss = out;
            counted = 1.;
        }
        if (a.lse) a.lse[2 * a.rows + row] = log2p;
        if (a.loss_rows) a.loss_rows[row] = out;
    }
    if (a.loss_rows) return;
    __shared__ double red[2][32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        loss += __shfl_xor_sync(0xffffffffu, loss, o);
        counted += __shfl_xor_sync(0xffffffffu, counted, o);
    }
    if ((threadIdx.x & 31) == 0) { red[0][threadIdx.x >> 5] = loss; red[1][threadIdx.x >> 5] = counted; }
    __syncthreads();
    if (threadIdx.x == 0) {
        double s = 0., n = 0.;
        for (int w = 0; w < blockDim.x / 32; w++) { s += red[0][w]; n += red[1][w]; }
        if (gridDim.x > 1) { a.sums[blockIdx.x] = make_double2(s, n); return; }
        *a.count = (float)n;
        *a.loss = (float)(a.mean ? s / n : s);                               // no row counts: 0 / 0, as the mean of nothing
    }
}
__global__ void __launch_bounds__(256)
xent_total_kernel(const double2 *__restrict__ sums, int blocks, int mean, float *__restrict__ loss, float *__restrict__ count) {
    __shared__ double red[2][256];
    double a = 0., b = 0.;
    for (int i = threadIdx.x; i < blocks; i += 256) { a += sums[i].x; b += sums[i].y; }
    red[0][threadIdx.x] = a; red[1][threadIdx.x] = b;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if (threadIdx.x < o) { red[0][threadIdx.x] += red[0][threadIdx.x + o]; red[1][threadIdx.x] += red[1][threadIdx.x + o]; }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        *count = (float)red[1][0];
        *loss = (float)(mean ? red[0][0] / red[1][0] : red[0][0]);
    }
}

// out = alpha * sum over slots of sums[slot], in a fixed order.  Block (32, Y): 32 elements, the slots congruent to y modulo Y.  The
// blocks behind the first n elements add another matrix of sums (of n2 elements, rows of ld2) to out2.
template <typename T, int Y>
__global__ void __launch_bounds__(32 * Y)
xent_finish_kernel(const float *__restrict__ sums, T *__restrict__ out, long long n, int slots, const float *__restrict__ sums2, void *__restrict__ out2, int n2,
                   int ld2, int slots2, int bf16_2, const float *up, const float *count, float f) {
    __shared__ double part[Y][33];
    const long long first = (n + 31) / 32;
    const bool more = blockIdx.x >= first;
    const long long i = ((long long)blockIdx.x - (more ? first : 0)) * 32 + threadIdx.x, all = more ? n2 : n, step = more ? ld2 : n;
    const float *from = (more ? sums2 : sums) + i;
    const int rows = more ? slots2 : slots;
    double s = 0.;
    if (i < all)
#pragma unroll 8
        for (int k = threadIdx.y; k < rows; k += Y) s += from[k * step];
    part[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && i < all) {
        double t = 0.;
#pragma unroll
        for (int y = 0; y < Y; y++) t += part[y][threadIdx.x];
        const float r = xent_alpha(up, count, f) * (float)t;
        if (more) st_param(out2, i, bf16_2, r); else st(out + i, r);
    }
}
// The same where there are few slots and many elements: four elements a thread.
template <typename T>
__global__ void __launch_bounds__(256)
xent_finish_few_kernel(const float *__restrict__ sums, T *__restrict__ out, long long n, int slots, const float *up, const float *count, float f) {
    const float alpha = xent_alpha(up, count, f);
    const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    const bool whole = n % 4 == 0;                       // every slot then starts on a vector
    for (int k = 0; k < slots; k++) {
        if (whole) {
            const float4 v = *reinterpret_cast<const float4 *>(sums + k * n + i);
            s[0] += v.x; s[1] += v.y; s[2] += v.z; s[3] += v.w;
        } else {
            for (int j = 0; j < 4; j++)
                if (i + j < n) s[j] += sums[k * n + i + j];
        }
    }
    for (int j = 0; j < 4; j++)
        if (i + j < n) st(out + i + j, alpha * s[j]);
}

// Column sums over slices of 32 rows, in a fixed order.  Block (32, 32); CTA (bx, by): columns 32 bx .., slices by * per ..
// With one CTA along y the result is db (times alpha), else sums of `per` slices, written or (`add`: of a later piece of the rows) added to.
template <typename P>
__global__ void __launch_bounds__(1024)
xent_bias_kernel(const P *__restrict__ partial, long long part_ld, int slices, int per, void *__restrict__ db, int bf16, double *__restrict__ more,
                 long long more_ld, bool add, int V, const float *up, const float *count, float f) {
    __shared__ double part[32][33];
    const int c = blockIdx.x * 32 + threadIdx.x, end = min(slices, (int)(blockIdx.y + 1) * per);
    double s = 0.;
    if (c < V)
#pragma unroll 4
        for (int k = blockIdx.y * per + threadIdx.y; k < end; k += 32) s += partial[k * part_ld + c];
    part[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && c < V) {
        double t = 0.;
#pragma unroll
        for (int y = 0; y < 32; y++) t += part[y][threadIdx.x];
        if (more) {
            double &to = more[blockIdx.y * more_ld + c];
            to = add ? to + t : t;
        } else {
            st_param(db, c, bf16, xent_alpha(up, count, f) * (float)t);
        }
    }
}

}  // namespace o1d

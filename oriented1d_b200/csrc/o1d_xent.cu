// Linear cross entropy: cutting the work into pieces, tensor maps, launches.
#include <atomic>

#include "o1d_xent.cuh"
#include "o1d_xent_dense.cuh"
#include "o1d_tma_host.cuh"
#include "o1d_xent.h"

namespace o1d {

namespace {

// Bytes of G that are held at once.  Larger pieces have fewer waves that end half empty and fewer rounds of adding to fp32
// sums, which is worth more than finding a piece in the L2 cache; 4096 x 1024 x 21841 bf16, gradient alone: 40 MB 557 us,
// 80 MB 512, 128 MB 489, all 179 MB in one piece 452 (the step 694 -> 673; 2500 x 384 x 10007 fp32, 150 MB, 507 -> 497).  Where
// more pieces than one it is, bf16, with pieces of 128 / 192 / 448 MB: 8192 x 1024 x 21841 957 / 901 / 842 us, 6000 x 512 x 30000
// 755 / 686 / 646, 16384 x 384 x 10000 640 / 583 / 547, 65536 x 256 x 4000 704 / 737 / 681; fp32 4096 x 384 x 10007 588 / 609 / 589.
// A thousandth of the device's memory.  (At least 256 rows or columns: the products' tiles.)
constexpr long long kPieceBytes = 192ll << 20;
constexpr int kMinSplitSteps = 16;               // K steps that a part of a split axis has at least (joining parts costs a launch)
constexpr int kSlicesAtOnce = 512;               // column sums of more slices are added in two steps

inline long long up_to(long long v, long long m) { return (v + m - 1) / m * m; }
inline int cdiv(long long a, long long b) { return (int)((a + b - 1) / b); }

// A bf16 matrix as the tensor copies see it.
struct Mat {
    const __nv_bfloat16 *p;
    long long rows;
    int cols;                // that exist
    long long ld, plane;     // elements between rows / planes
    int planes;
};
Mat sub_rows(const Mat &m, long long row0, long long rows) {
    Mat r = m;
    r.p += row0 * m.ld;
    r.rows = rows;
    return r;
}

int encode(CUtensorMap *map, const Mat &m, int box_rows) {
    thread_local bool bound = false;
    if (!bound) { bind_primary_context(); bound = true; }
    PFN_encodeTiled enc = encode_tiled_fn();
    if (!enc) return -1;
    const cuuint64_t dims[3] = {(cuuint64_t)m.cols, (cuuint64_t)m.rows, (cuuint64_t)m.planes};
    const cuuint64_t strides[2] = {(cuuint64_t)m.ld * 2, (cuuint64_t)m.plane * 2};
    const cuuint32_t box[3] = {(cuuint32_t)kXK, (cuuint32_t)box_rows, 1}, es[3] = {1, 1, 1};
    CUresult r = CUDA_SUCCESS;
    for (int attempt = 0; attempt < 2; attempt++) {
        r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<__nv_bfloat16 *>(m.p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r == CUDA_SUCCESS) return 0;
        bind_primary_context();
    }
    return (int)r;
}

// How a product is tiled.  Waves of tiles times their steps; a step of 128 x 128 takes 0.6 of one of 128 x 256, a pair's
// (256 x 256 on two SMs) 0.9 (measured: 0.25, 0.42 and 0.38 us).
struct Shape { int tile_rows, bn, units; };      // units: CTAs, or pairs of them, that the device runs at once
// `narrow_only`: operands of more than one plane.
Shape shape_of(long long m, long long n, long long k, bool narrow_only, int sms) {
    const Shape narrow{kXM, 128, sms}, wide{kXM, 256, sms}, pair{2 * kXM, 256, sms / 2};
    if (narrow_only) return narrow;
    const long long steps = cdiv(k, kXK) + 6;
    auto cost = [&](const Shape &s, int weight) { return cdiv((long long)cdiv(m, s.tile_rows) * cdiv(n, s.bn), s.units) * steps * weight; };
    const long long cn = cost(narrow, 6), cw = cost(wide, 10), cp = cost(pair, 9);
    // (a pair's two epilogues wait for each other; with few steps a tile they are what counts: 133200 x 150 x 96 logits 30.6 us,
    // one CTA a tile 25.9)
    return k >= 512 && cp <= cw && cp <= cn ? pair : cn < cw ? narrow : wide;
}

// Sets a kernel's limit of shared memory once a device (a microsecond a call otherwise).
cudaError_t size_once(std::atomic<uint64_t> &sized, const void *kern, int bytes) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && (sized.load(std::memory_order_acquire) >> dev & 1))) return e;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) sized.fetch_or(1ull << dev, std::memory_order_release);
    return e;
}

struct Run {                 // of one call
    const XentArgs &a;
    int sms, *err_flag;
    cudaStream_t st;
    cudaError_t *cuda;
    int *enc;
    int fail(cudaError_t e) { *cuda = e; return O1D_ERR_CUDA; }

    template <int KIND, int MODE>
    int product(const Mat &ma, const Mat &mb, const XentParams &p) {
        constexpr bool A_MN = KIND == XENT_DW, B_MN = KIND == XENT_DX || KIND == XENT_DW;
        if constexpr (MODE == XENT_BF16) {
            const Shape s = shape_of(A_MN ? ma.cols : ma.rows, B_MN ? mb.cols : mb.rows, A_MN ? ma.rows : ma.cols, false, sms);
            if (s.tile_rows != kXM) return run<KIND, MODE, 256, true>(ma, mb, p);
            if (s.bn == 256) return run<KIND, MODE, 256, false>(ma, mb, p);
        }
        return run<KIND, MODE, 128, false>(ma, mb, p);
    }
    template <int KIND, int MODE, int BN, bool PAIR>
    int run(const Mat &ma, const Mat &mb, XentParams p) {
        using S = XentShape<KIND, MODE, BN, PAIR>;
        constexpr bool A_MN = KIND == XENT_DW, B_MN = KIND == XENT_DX || KIND == XENT_DW;
        CUtensorMap a_map, b_map;
        if ((*enc = encode(&a_map, ma, A_MN ? kXK : kXM)) || (*enc = encode(&b_map, mb, B_MN ? kXK : S::B_COLS))) return O1D_ERR_CUDA;
        p.M = (int)(A_MN ? ma.cols : ma.rows);
        p.N = (int)(B_MN ? mb.cols : mb.rows);
        const long long m_tiles = cdiv(p.M, S::TM), n_tiles = cdiv(p.N, BN);
        p.k_steps = cdiv(A_MN ? ma.rows : ma.cols, kXK);
        if (p.splits < 1) p.splits = 1;
        if (m_tiles * n_tiles * p.splits > 0x7fffffff) return O1D_ERR_UNSUPPORTED;
        p.m_tiles = (int)m_tiles;
        p.n_tiles = (int)n_tiles;
        p.tiles = p.m_tiles * p.n_tiles * p.splits;
        p.along_n = p.M > p.N;
        p.err_flag = err_flag;
        auto kern = xent_kernel<KIND, MODE, BN, PAIR>;
        static std::atomic<uint64_t> sized{0};       // devices that know how much shared memory the kernel takes
        cudaError_t e = size_once(sized, (const void *)kern, S::SMEM);
        if (e != cudaSuccess) return fail(e);
        const int units = PAIR ? sms / 2 : sms;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((p.tiles < units ? p.tiles : units) * (PAIR ? 2 : 1));
        cfg.blockDim = dim3(kXThreads);
        cfg.dynamicSmemBytes = S::SMEM;
        cfg.stream = st;
        cudaLaunchAttribute pair_attr;
        pair_attr.id = cudaLaunchAttributeClusterDimension;
        pair_attr.val.clusterDim.x = 2;
        pair_attr.val.clusterDim.y = pair_attr.val.clusterDim.z = 1;
        cfg.attrs = &pair_attr;
        cfg.numAttrs = PAIR ? 1 : 0;
        e = cudaLaunchKernelEx(&cfg, kern, a_map, b_map, p);
        return e == cudaSuccess ? O1D_OK : fail(e);
    }
};

// x or w as planes: in place where it can be, else in the workspace.
struct Operand { bool copy; long long rows; int D, ld, planes; size_t bytes; };
Operand operand_of(long long rows, int D, bool bf16) {
    Operand o;
    o.copy = !bf16 || D % 8 != 0;
    o.rows = rows; o.D = D;
    o.planes = bf16 ? 1 : 3;
    o.ld = o.copy ? (int)up_to(D, 8) : D;
    o.bytes = o.copy ? (size_t)up_to((long long)o.planes * rows * o.ld * 2, 256) : 0;
    return o;
}
int make_operand(Run &r, const void *src, const Operand &o, unsigned char **ws, Mat *m) {
    m->rows = o.rows; m->cols = o.D; m->ld = o.ld; m->plane = o.rows * o.ld; m->planes = o.planes;
    if (!o.copy) { m->p = (const __nv_bfloat16 *)src; return O1D_OK; }
    __nv_bfloat16 *to = (__nv_bfloat16 *)*ws;
    *ws += o.bytes;
    m->p = to;
    const long long blocks = (o.rows + 7) / 8;
    const int grid = (int)(blocks < (long long)r.sms * 16 ? blocks : (long long)r.sms * 16), vec = o.D % 4 == 0;
    if (o.planes == 3) xent_planes_kernel<float><<<grid, 256, 0, r.st>>>((const float *)src, to, o.rows, o.D, o.ld, vec);
    else xent_planes_kernel<__nv_bfloat16><<<grid, 256, 0, r.st>>>((const __nv_bfloat16 *)src, to, o.rows, o.D, o.ld, vec);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? O1D_OK : r.fail(e);
}

// G in two planes?  Up to 2^30 products, 2 us of a whole GPU, the second plane costs latency at most; and there are then few rows
// or classes over which the rounding of G to one plane could average out (without: errors of dx up to 1.8 times those of the
// same sums in fp32, rounded to bf16 once).
bool fine_of(const XentArgs &a) { return a.bf16 && (double)a.N * a.V * a.D <= (double)(1ll << 30); }
int planes_of(const XentArgs &a) { return !a.bf16 ? 3 : fine_of(a) ? 2 : 1; }

// Few classes and narrow features: one kernel for all of the backward pass (o1d_xent_dense.cuh), with one plane of G.
bool dense_of(const XentArgs &a) { return a.bf16 && !fine_of(a) && a.V <= kDenseV && a.D <= kDenseD; }
// Rows of one launch of it.  dw of a CTA's tiles is one sum in tensor memory, eight additions a tile, and a tensor core truncates as it
// adds: measured, sums of one sign lose 1.6e-8 of themselves with every addition.  256 tiles are 2048 additions, 3e-5 (19.4 M rows in one
// launch had 8192, 60 M 25000: 4e-4, a fifth of what a bf16 result is rounded by).  Each launch leaves sums of its own.
constexpr int kDenseTiles = 256;
long long dense_rows(int sms) { return (long long)kDenseTiles * sms * kXM; }
int dense_ctas(long long rows, int sms) { return cdiv(rows, kXM) < sms ? cdiv(rows, kXM) : sms; }
// Sums that all launches of a call leave: CTAs of each.
int dense_sums(const XentArgs &a, int sms) {
    const long long most = dense_rows(sms), rest = a.N % most;
    return (int)(a.N / most) * sms + (rest ? dense_ctas(rest, sms) : 0);
}

bool few_rows(long long N, int D) { return N <= kFewRows && (N <= 1 ? 1 : N <= 2 ? 2 : N <= 4 ? 4 : 8) * up_to(D, 8) * 4 <= kFewBytes; }
int few_ctas(long long N, int V, int sms) {
    const int need = cdiv(V, 8 * (N > 4 ? 2 : 4));
    return need < 2 * sms ? need : 2 * sms;
}

// Forward: statistics that a row has, at most.
int forward_slots(const XentArgs &a, int sms) {
    if (few_rows(a.N, a.D) && !a.lse) return few_ctas(a.N, a.V, sms);
    const Shape s = shape_of(a.N, a.V, a.D, !a.bf16, sms);
    const long long n_tiles = cdiv(a.V, s.bn), tiles = cdiv(a.N, s.tile_rows) * n_tiles;
    const long long ctas = tiles < s.units ? tiles : s.units, least = tiles / ctas;
    return 4 * (int)(cdiv(n_tiles, least) + 1);
}

// Backward: how G is cut, and into how many parts the K axes of the two products are.
struct Cut {
    bool by_rows;
    long long piece;         // rows, or columns of the vocabulary
    int pieces, ld;          // ld: columns of G in memory
    long long rows;          // rows of a piece
    int dx_parts, dw_parts;  // fp32 sums; 0: the product writes its result
    int col_blocks() const { return cdiv(cdiv(rows, 32), kSlicesAtOnce); }
    bool col_once() const { return (pieces == 1 || !by_rows) && col_blocks() == 1; }      // a class's sum is complete with its piece
};
int parts_of(long long m, long long n, long long k, bool narrow_only, int sms, bool adds) {
    const Shape shape = shape_of(m, n, k, narrow_only, sms);
    const long long tiles = (long long)cdiv(m, shape.tile_rows) * cdiv(n, shape.bn), steps = cdiv(k, kXK);
    long long s = shape.units / tiles;
    if (s > steps / kMinSplitSteps) s = steps / kMinSplitSteps;
    if (s < 1) s = 1;
    return s == 1 && !adds ? 0 : (int)s;
}
// Time of a cut in units of one K step of one tile (0.4 us): waves of tiles times their steps, which an epilogue of
// about six steps bounds from below, and six steps for each launch to begin and end.
long long cost_of(const XentArgs &a, bool by_rows, long long piece, int sms, int bn) {
    const long long axis = by_rows ? a.N : a.V;
    long long total = 0;
    auto waves = [&](long long tiles, long long steps) { return (tiles + sms - 1) / sms * (steps < 6 ? 6 : steps) + 6; };
    auto one = [&](long long n) {
        const long long rows = by_rows ? n : a.N, cols = by_rows ? a.V : n, m = cdiv(rows, kXM), d = cdiv(a.D, bn);
        return waves(m * cdiv(cols, bn), cdiv(a.D, kXK)) + waves(m * d, cdiv(cols, kXK)) + waves(cdiv(cols, kXM) * d, cdiv(rows, kXK));
    };
    total = axis / piece * one(piece);
    if (axis % piece) total += one(axis % piece);
    return total;
}
Cut cut_of(const XentArgs &a, int sms) {
    const int planes = planes_of(a), bn = planes == 1 ? 256 : 128;
    Cut c;
    c.by_rows = a.N > a.V;
    const long long all_ld = up_to(a.V, 64), axis = c.by_rows ? a.N : a.V;
    long long most = kPieceBytes / (2 * planes * (c.by_rows ? all_ld : a.N)) / 256 * 256;
    if (most < 256) most = 256;
    c.piece = axis;
    if (axis > most) {
        // equal pieces, or such as make whole waves of the tiles along the cut axis: whichever costs least
        long long best = 0;
        auto consider = [&](long long p) {
            if (p < 256 || p > most) return;
            const long long t = cost_of(a, c.by_rows, p, sms, bn);
            if (!best || t < best) { best = t; c.piece = p; }
        };
        const long long least = (axis + most - 1) / most;
        for (long long k = least; k < least + 3; k++) consider(up_to((axis + k - 1) / k, 256));
        const long long d = cdiv(a.D, bn);
        for (int w = 1; w <= 4; w++) {
            consider(w * sms / d * kXM / 256 * 256);
            if (!c.by_rows) consider(w * sms / cdiv(a.N, kXM) * bn / 256 * 256);
        }
        if (!best) c.piece = most;
    }
    c.pieces = cdiv(axis, c.piece);
    c.ld = (int)(c.by_rows ? all_ld : up_to(c.piece, 64));
    c.rows = c.by_rows ? c.piece : a.N;
    c.dx_parts = parts_of(c.rows, a.D, c.by_rows ? a.V : c.piece, planes > 1, sms, !c.by_rows && c.pieces > 1);
    c.dw_parts = parts_of(c.by_rows ? a.V : c.piece, a.D, c.rows, planes > 1, sms, c.by_rows && c.pieces > 1);
    return c;
}
struct BackwardBytes { size_t x, w, g, dx, dw, col, more; };
BackwardBytes backward_bytes(const XentArgs &a, const Cut &c) {
    const int planes = planes_of(a);
    BackwardBytes b;
    b.x = operand_of(a.N, a.D, a.bf16).bytes;
    b.w = operand_of(a.V, a.D, a.bf16).bytes;
    b.g = (size_t)up_to(2ll * planes * c.rows * c.ld, 256);
    // by rows, dx is complete with its piece; by vocabulary, dw is
    b.dx = (size_t)up_to(4ll * c.dx_parts * c.rows * a.D, 256);
    b.dw = (size_t)up_to(4ll * c.dw_parts * (c.by_rows ? a.V : c.piece) * a.D, 256);
    // column sums of a piece, in slices of 32 rows; and (by rows: of all pieces) of kSlicesAtOnce of those
    b.col = (size_t)up_to(4ll * cdiv(c.rows, 32) * c.ld, 256);
    b.more = c.col_once() ? 0 : (size_t)up_to(8ll * c.col_blocks() * c.ld, 256);
    return b;
}

XentRows rows_of(const XentArgs &a, const XentParams &p, double2 *sums) {
    XentRows q{};
    q.part = p.part; q.part_sum = p.part_sum; q.target_logit = p.target_logit; q.target = a.target; q.ignore = a.ignore; q.rows = a.N;
    q.smoothing = a.smoothing; q.V = a.V; q.mean = a.reduction == O1D_XENT_MEAN; q.lse = a.lse; q.sums = sums;
    if (a.reduction == O1D_XENT_NONE) q.loss_rows = a.loss;
    else { q.loss = a.loss; q.count = a.count; }
    return q;
}
// The rows' statistics to the loss.  More lanes a row where it has many slots and there are few rows (their vocabulary spread over
// all SMs); a lane's slots are far apart, so that with many rows one lane a row reads less (133200 rows, 8 slots: 5.5 us, 17 with
// eight lanes).
int reduce(Run &r, const XentRows &q) {
    const int lanes = q.slots <= 4 || q.rows > 16384 ? 1 : q.slots <= 64 ? 8 : 32;
    const int threads = q.rows * lanes <= 1024 ? 1024 : 256, blocks = cdiv(q.rows * lanes, threads);      // one block where it can be
    if (lanes == 1) xent_rows_kernel<1><<<blocks, threads, 0, r.st>>>(q);
    else if (lanes == 8) xent_rows_kernel<8><<<blocks, threads, 0, r.st>>>(q);
    else xent_rows_kernel<32><<<blocks, threads, 0, r.st>>>(q);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess && !q.loss_rows && blocks > 1) {
        xent_total_kernel<<<1, 256, 0, r.st>>>(q.sums, blocks, q.mean, q.loss, q.count);
        e = cudaGetLastError();
    }
    return e == cudaSuccess ? O1D_OK : r.fail(e);
}

template <typename T, int NR>
void few(const XentArgs &a, const XentParams &p, int ctas, bool vec, cudaStream_t st) {
    const int smem = NR * (int)up_to(a.D, 8) * 4;
    if (vec) xent_few_kernel<T, NR, true><<<ctas, 256, smem, st>>>((const T *)a.x, (const T *)a.w, p, a.D);
    else xent_few_kernel<T, NR, false><<<ctas, 256, smem, st>>>((const T *)a.x, (const T *)a.w, p, a.D);
}
template <typename T>
void few(const XentArgs &a, const XentParams &p, int ctas, cudaStream_t st) {
    const bool vec = a.D % (16 / (int)sizeof(T)) == 0;
    if (a.N <= 1) few<T, 1>(a, p, ctas, vec, st);
    else if (a.N <= 2) few<T, 2>(a, p, ctas, vec, st);
    else if (a.N <= 4) few<T, 4>(a, p, ctas, vec, st);
    else few<T, 8>(a, p, ctas, vec, st);
}

template <int MODE>
int forward(Run &r) {
    constexpr bool SPLIT = MODE == XENT_F32;
    const XentArgs &a = r.a;
    unsigned char *ws = (unsigned char *)a.workspace;
    const int slots = forward_slots(a, r.sms);
    XentParams p{};
    p.bias = a.bias; p.bias_bf16 = a.bias_bf16; p.V = a.V; p.target = a.target; p.ignore = a.ignore;
    p.part = (float2 *)ws; ws += up_to(8ll * slots * a.N, 256);
    p.target_logit = (float *)ws; ws += up_to(4 * a.N, 256);
    p.smooth = a.smoothing > 0.f;
    p.part_sum = (float *)ws; ws += up_to(4ll * slots * a.N, 256);
    double2 *sums = (double2 *)ws; ws += up_to(16ll * cdiv(a.N, 8), 256);
    p.part_rows = a.N;
    XentRows q = rows_of(a, p, sums);
    q.slots = slots;
    if (few_rows(a.N, a.D) && !a.lse) {              // (a backward pass wants the logits that its own tiles will form)
        p.M = (int)a.N;
        if (SPLIT) few<float>(a, p, slots, r.st); else few<__nv_bfloat16>(a, p, slots, r.st);
        const cudaError_t e = cudaGetLastError();
        return e == cudaSuccess ? reduce(r, q) : r.fail(e);
    }
    Mat x, w;
    int rc = make_operand(r, a.x, operand_of(a.N, a.D, a.bf16), &ws, &x);
    if (!rc) rc = make_operand(r, a.w, operand_of(a.V, a.D, a.bf16), &ws, &w);
    if (!rc) rc = r.product<XENT_LOGITS, MODE>(x, w, p);
    if (rc) return rc;
    const Shape s = shape_of(a.N, a.V, a.D, SPLIT, r.sms);
    q.tile_rows = s.tile_rows;
    q.n_tiles = cdiv(a.V, s.bn);
    q.tiles = cdiv(a.N, s.tile_rows) * q.n_tiles;
    q.units = q.tiles < s.units ? q.tiles : s.units;
    return reduce(r, q);
}

template <typename T>
cudaError_t finish(const float *sums, void *out, long long n, int slots, const float *up, const float *count, float f, cudaStream_t st) {
    if (slots > 4) xent_finish_kernel<T, 8><<<cdiv(n, 32), dim3(32, 8), 0, st>>>(sums, (T *)out, n, slots, nullptr, nullptr, 0, 0, 0, 0, up, count, f);
    else xent_finish_few_kernel<T><<<cdiv(n, 1024), 256, 0, st>>>(sums, (T *)out, n, slots, up, count, f);
    return cudaGetLastError();
}
int backward_dense(Run &r) {
    const XentArgs &a = r.a;
    const int sums = dense_sums(a, r.sms);
    unsigned char *ws = (unsigned char *)a.workspace;
    float *dws = (float *)ws; ws += up_to(4ll * sums * a.V * a.D, 256);
    float *cols = (float *)ws; ws += up_to(4ll * sums * kDenseV, 256);
    Mat x, w;
    int rc = make_operand(r, a.x, operand_of(a.N, a.D, true), &ws, &x);
    if (!rc) rc = make_operand(r, a.w, operand_of(a.V, a.D, true), &ws, &w);
    if (rc) return rc;
    CUtensorMap x_map, w_map;
    if ((*r.enc = encode(&w_map, w, (int)up_to(a.V, 32)))) return O1D_ERR_CUDA;
    const bool each = a.reduction == O1D_XENT_NONE;
    const float f = a.smoothing < 1.f ? 1.f - a.smoothing : 1.f;
    const float *up = each ? nullptr : a.dloss, *count = a.reduction == O1D_XENT_MEAN ? a.count : nullptr;
    XentParams p{};
    p.N = a.V;
    p.bias = a.bias; p.bias_bf16 = a.bias_bf16; p.V = a.V; p.ignore = a.ignore;
    p.smooth = a.smoothing > 0.f;
    p.factor_log2 = log2f(f); p.one = a.smoothing < 1.f ? 1.f : 0.f; p.eps_v = a.smoothing / (float)a.V / f;
    p.cols_ld = kDenseV;
    p.vec = ((uintptr_t)a.dx & 15) == 0 && a.D % 8 == 0;             // (a launch's rows start on a multiple of 128)
    p.alpha_up = up; p.alpha_count = count; p.alpha = f;
    p.err_flag = r.err_flag;
    static std::atomic<uint64_t> sized{0};
    cudaError_t e = size_once(sized, (const void *)xent_dense_kernel, kDenseSmem);
    if (e != cudaSuccess) return r.fail(e);
    int at = 0;                                                       // sums that the launches so far leave
    for (long long row0 = 0; e == cudaSuccess && row0 < a.N; row0 += dense_rows(r.sms)) {
        const long long rows = a.N - row0 < dense_rows(r.sms) ? a.N - row0 : dense_rows(r.sms);
        const int ctas = dense_ctas(rows, r.sms);
        if ((*r.enc = encode(&x_map, sub_rows(x, row0, rows), kXM))) return O1D_ERR_CUDA;
        p.M = (int)rows; p.tiles = cdiv(rows, kXM);
        p.target = a.target + row0;
        p.lse = a.lse + row0; p.lse_lo = a.lse + a.N + row0; p.log2p = a.lse + 2 * a.N + row0; p.up = each ? a.dloss + row0 : nullptr;
        p.cols = a.db ? cols + (long long)at * kDenseV : nullptr;
        xent_dense_kernel<<<ctas, kXThreads, kDenseSmem, r.st>>>(x_map, w_map, p, a.D, a.dx ? (__nv_bfloat16 *)a.dx + row0 * a.D : nullptr,
                                                                 a.dw ? dws + (long long)at * a.V * a.D : nullptr);
        e = cudaGetLastError();
        at += ctas;
    }
    const long long dw_n = a.dw ? (long long)a.V * a.D : 0;
    const int db_n = a.db ? a.V : 0;
    if (e == cudaSuccess && dw_n + db_n > 0) {
        xent_finish_kernel<__nv_bfloat16, 16><<<cdiv(dw_n, 32) + cdiv(db_n, 32), dim3(32, 16), 0, r.st>>>(
            dws, (__nv_bfloat16 *)a.dw, dw_n, sums, cols, a.db, db_n, kDenseV, sums, a.bias_bf16, up, count, f);
        e = cudaGetLastError();
    }
    return e == cudaSuccess ? O1D_OK : r.fail(e);
}
template <int MODE>
int backward(Run &r) {
    const XentArgs &a = r.a;
    const Cut c = cut_of(a, r.sms);
    const BackwardBytes b = backward_bytes(a, c);
    unsigned char *ws = (unsigned char *)a.workspace;
    const int es = a.bf16 ? 2 : 4;
    __nv_bfloat16 *g = (__nv_bfloat16 *)ws; ws += b.g;
    float *dxs = (float *)ws; ws += b.dx;
    float *dws = (float *)ws; ws += b.dw;
    float *cols = (float *)ws; ws += b.col;
    double *more = (double *)ws; ws += b.more;
    Mat x, w;
    int rc = make_operand(r, a.x, operand_of(a.N, a.D, a.bf16), &ws, &x);
    if (!rc) rc = make_operand(r, a.w, operand_of(a.V, a.D, a.bf16), &ws, &w);
    if (rc) return rc;

    const bool each = a.reduction == O1D_XENT_NONE;
    const float f = a.smoothing < 1.f ? 1.f - a.smoothing : 1.f;
    const float *up = each ? nullptr : a.dloss, *count = a.reduction == O1D_XENT_MEAN ? a.count : nullptr;
    // One product's way out: its result at once, or sums that `finish` turns into it.
    // (the last piece of a product whose pieces have one part adds the others to what it writes)
    auto out_of = [&](XentParams &p, int parts, bool first, bool last, void *result, float *sums, long long elems, long long k) {
        p.splits = parts < 1 ? 1 : parts;
        const long long steps = cdiv(k, kXK);
        if (p.splits > steps) p.splits = (int)steps;                  // a short last piece
        const bool joins = parts == 1 && last && !first;
        p.out = parts && !joins ? (void *)sums : result;
        p.before = sums;
        p.split_elems = elems;
        p.out_kind = joins ? (a.bf16 ? 4 : 5) : parts ? (first ? 2 : 3) : a.bf16 ? 0 : 1;
        // (rows of fp32 sums and of the result start on their vectors alike: four elements of the one, four or eight of the other)
        p.vec = p.out_kind == 0 ? ((uintptr_t)p.out & 15) == 0 && a.D % 8 == 0
                                : ((uintptr_t)p.out & 15) == 0 && a.D % 4 == 0;
        p.alpha_up = up; p.alpha_count = count; p.alpha = f;
    };
    auto end = [&](int parts, bool joined, float *sums, void *result, long long elems) {
        if (!parts || (parts == 1 && joined)) return cudaSuccess;
        return a.bf16 ? finish<__nv_bfloat16>(sums, result, elems, parts, up, count, f, r.st)
                      : finish<float>(sums, result, elems, parts, up, count, f, r.st);
    };
    for (int i = 0; i < c.pieces; i++) {
        const long long at = i * c.piece, axis = c.by_rows ? a.N : a.V, n = axis - at < c.piece ? axis - at : c.piece;
        const long long row0 = c.by_rows ? at : 0, rows = c.by_rows ? n : a.N;
        const int col0 = c.by_rows ? 0 : (int)at, colsn = c.by_rows ? a.V : (int)n, ld = (int)up_to(colsn, 64);
        const Mat xs = sub_rows(x, row0, rows), wp = sub_rows(w, col0, colsn);
        const Mat gm{g, rows, ld, ld, rows * ld, planes_of(a)};
        XentParams p{};
        p.bias = a.bias; p.bias_bf16 = a.bias_bf16; p.col0 = col0; p.V = a.V; p.target = a.target + row0; p.ignore = a.ignore;
        p.smooth = a.smoothing > 0.f;
        p.lse = a.lse + row0; p.lse_lo = a.lse + a.N + row0; p.log2p = a.lse + 2 * a.N + row0; p.up = each ? a.dloss + row0 : nullptr;
        p.factor_log2 = log2f(f); p.one = a.smoothing < 1.f ? 1.f : 0.f; p.eps_v = a.smoothing / (float)a.V / f;
        p.g = g; p.g_plane = gm.plane; p.g_ld = ld;
        p.cols = a.db ? cols : nullptr; p.cols_ld = ld;
        // exp(l - lse) / f = exp2(l2 - (lse2 + log2 f))
        if ((rc = r.product<XENT_GRAD, MODE>(xs, wp, p))) return rc;
        cudaError_t e = cudaSuccess;
        if (a.dx) {
            XentParams q{};
            void *to = (char *)a.dx + row0 * a.D * es;
            out_of(q, c.dx_parts, c.by_rows || i == 0, i == c.pieces - 1, to, dxs, rows * a.D, ld);
            if ((rc = r.product<XENT_DX, MODE>(gm, wp, q))) return rc;
            if (c.by_rows || i == c.pieces - 1) e = end(c.dx_parts, !c.by_rows && i > 0, dxs, to, rows * a.D);
        }
        if (e == cudaSuccess && a.dw) {
            XentParams q{};
            void *to = (char *)a.dw + (long long)col0 * a.D * es;
            Mat gv = gm;
            gv.cols = colsn;                                          // rows of dw that exist
            out_of(q, c.dw_parts, !c.by_rows || i == 0, i == c.pieces - 1, to, dws, (long long)colsn * a.D, rows);
            if ((rc = r.product<XENT_DW, MODE>(gv, xs, q))) return rc;
            if (!c.by_rows || i == c.pieces - 1) e = end(c.dw_parts, c.by_rows && i > 0, dws, to, (long long)colsn * a.D);
        }
        if (e == cudaSuccess && a.db) {
            const int slices = cdiv(rows, 32);
            void *to = (char *)a.db + (long long)col0 * (a.bias_bf16 ? 2 : 4);
            if (c.col_once()) {
                xent_bias_kernel<<<cdiv(colsn, 32), dim3(32, 32), 0, r.st>>>(cols, ld, slices, slices, to, a.bias_bf16, nullptr, 0, false, colsn, up, count, f);
            } else {
                xent_bias_kernel<<<dim3(cdiv(colsn, 32), cdiv(slices, kSlicesAtOnce)), dim3(32, 32), 0, r.st>>>(
                    cols, ld, slices, kSlicesAtOnce, nullptr, 0, more, c.ld, c.by_rows && i > 0, colsn, nullptr, nullptr, 1.f);
                if (!c.by_rows || i == c.pieces - 1)
                    xent_bias_kernel<<<cdiv(colsn, 32), dim3(32, 32), 0, r.st>>>(more, c.ld, c.col_blocks(), c.col_blocks(), to, a.bias_bf16, nullptr, 0, false, colsn,
                                                                                 up, count, f);
            }
            e = cudaGetLastError();
        }
        if (e != cudaSuccess) return r.fail(e);
    }
    return O1D_OK;
}

}  // namespace

size_t xent_workspace(const XentArgs &a, bool back, int sms) {
    if (back && dense_of(a)) {
        const int sums = dense_sums(a, sms);
        return operand_of(a.N, a.D, true).bytes + operand_of(a.V, a.D, true).bytes + (size_t)(up_to(4ll * sums * a.V * a.D, 256) + up_to(4ll * sums * kDenseV, 256));
    }
    if (back) {
        const BackwardBytes b = backward_bytes(a, cut_of(a, sms));
        return b.x + b.w + b.g + b.dx + b.dw + b.col + b.more;
    }
    const int slots = forward_slots(a, sms);
    if (few_rows(a.N, a.D) && !a.lse) return (size_t)(up_to(8ll * slots * a.N, 256) + up_to(4 * a.N, 256) + up_to(4ll * slots * a.N, 256) + up_to(16ll * cdiv(a.N, 8), 256));
    return operand_of(a.N, a.D, a.bf16).bytes + operand_of(a.V, a.D, a.bf16).bytes + (size_t)(up_to(8ll * slots * a.N, 256) + up_to(4 * a.N, 256) +
           up_to(4ll * slots * a.N, 256) + up_to(16ll * cdiv(a.N, 8), 256));
}
int xent_forward(const XentArgs &a, int sms, int *err_flag, cudaStream_t st, cudaError_t *cuda, int *enc) {
    Run r{a, sms, err_flag, st, cuda, enc};
    return a.bf16 ? forward<XENT_BF16>(r) : forward<XENT_F32>(r);
}
int xent_backward(const XentArgs &a, int sms, int *err_flag, cudaStream_t st, cudaError_t *cuda, int *enc) {
    Run r{a, sms, err_flag, st, cuda, enc};
    if (dense_of(a)) return backward_dense(r);
    return !a.bf16 ? backward<XENT_F32>(r) : fine_of(a) ? backward<XENT_FINE>(r) : backward<XENT_BF16>(r);
}

}  // namespace o1d

// Backward pass of the linear cross entropy for few classes and narrow features (a dense prediction head): everything of a row tile
// in one kernel.  With V <= 192 and D <= 128 the tensor memory of an SM holds the logits of 128 rows (192 columns), the
// gradient of their features (128) and the CTA's sum of the weight's gradient (192) side by side, so that
//     L = x w^T,   G = softmax gradient of L,   dx = G w,   dw^T += x^T G
// run one behind the other: x is read once, G never leaves shared memory, and dw leaves the CTA once, as one of the sums that
// xent_finish_kernel adds in a fixed order.  One copy of each operand serves two products, since a tile of rows of 64 elements is
// K-major along its rows and MN-major across them: x in L and dw, w in L and dx, G in dx and dw.
//
// What bounds it: the finishing warps.  The products of a tile take 0.5 us, its softmax and stores two pieces of 32 x 32 a warp.
// They run beside each other: the logits of the next tile are formed while this one's are worked on (their registers are loaded
// first), dx and dw of a tile while its successor's softmax is taken.
#pragma once

#include "o1d_xent.cuh"

namespace o1d {

constexpr int kDenseV = 192, kDenseD = 128;      // the widest that fits; multiples of 64, which an MN-major operand comes in
constexpr int kDenseStages = 3, kDenseX = kXM * kDenseD * 2, kDenseW = kDenseV * kDenseD * 2, kDenseG = kXM * kDenseV * 2;
constexpr int kDenseSmem = kDenseStages * kDenseX + kDenseW + kDenseG + kXFinish * kXStaging + kDenseV * 4 + 256 + 1024;
// tensor memory: columns of dw^T, of the logits and of dx
constexpr uint32_t kDenseTW = 0, kDenseTL = kDenseV, kDenseTX = 2 * kDenseV;

__global__ void __launch_bounds__(kXThreads, 1)
xent_dense_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const XentParams p, int D, __nv_bfloat16 *dx,
                  float *dw) {
    extern __shared__ __align__(1024) unsigned char raw[];
    unsigned char *smem = raw + ((1024u - (tc::smem_addr(raw) & 1023u)) & 1023u);
    unsigned char *sx = smem, *sw = sx + kDenseStages * kDenseX, *sg = sw + kDenseW;
    char *staging = reinterpret_cast<char *>(sg + kDenseG);
    float *bias = reinterpret_cast<float *>(staging + kXFinish * kXStaging);
    uint64_t *full = reinterpret_cast<uint64_t *>(bias + kDenseV), *empty = full + kDenseStages;       // of x
    uint64_t *w_full = empty + kDenseStages;
    uint64_t *logits = w_full + 1, *read = logits + 1;               // logits are there; are in registers
    uint64_t *ready = read + 1, *done = ready + 1, *taken = done + 1;      // G is written; its products are done; dx is in registers
    uint64_t *last = taken + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(last + 1);
    volatile int *dead = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int v32 = (p.V + 31) & ~31, d_blocks = D > 64 ? 2 : 1;      // rows of w in shared memory; blocks of 64 features
    const int mine = (p.tiles - 1 - (int)blockIdx.x) / (int)gridDim.x + 1;      // tiles blockIdx.x, + gridDim.x, ..

    if (threadIdx.x == 0) {
        for (int i = 0; i < kDenseStages; i++) { tc::bar_init(full + i, 1); tc::bar_init(empty + i, 1); }
        tc::bar_init(w_full, 1);
        tc::bar_init(logits, 1); tc::bar_init(read, kXFinish);
        tc::bar_init(ready, kXFinish); tc::bar_init(done, 1); tc::bar_init(taken, kXFinish);
        tc::bar_init(last, 1);
        *dead = 0;
        tc::bar_init_fence();
        tc::tma_prefetch(&map_x);
        tc::tma_prefetch(&map_w);
    }
    if (warp == 2) tc::tmem_alloc<false>(tmem_slot, 512);
    // the bias in units of log2; -inf where the vocabulary ends, so that those columns weigh nothing
    if (warp >= 4)
        for (int c = threadIdx.x - 128; c < kDenseV; c += 32 * kXFinish)
            bias[c] = c >= p.V ? __int_as_float(0xff800000) : p.bias ? 1.4426950408889634f * ld_param(p.bias, c, p.bias_bf16) : 0.f;
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0 && lane == 0) {                                   // ---- loads
        tc::bar_expect(w_full, d_blocks * v32 * 128);
        for (int j = 0; j < d_blocks; j++) tc::tma_load3(sw + j * v32 * 128, &map_w, w_full, j * 64, 0, 0);
        int stage = 0, issued = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int i = 0; i < mine; i++) {
            if (!(ok = tc::bar_wait(empty + stage, phase ^ 1, dead, p.err_flag))) break;
            tc::bar_expect(full + stage, kDenseX);
            // (both blocks whatever D: dw^T has 128 rows)
            for (int j = 0; j < 2; j++) tc::tma_load3(sx + stage * kDenseX + j * 16384, &map_x, full + stage, j * 64, (blockIdx.x + i * gridDim.x) * kXM, 0);
            issued++;
            if (++stage == kDenseStages) { stage = 0; phase ^= 1; }
        }
        if (!ok) {                                                  // copies in flight end before the CTA does
            tc::bar_drain(w_full, 0);
            for (int i = 0; i < kDenseStages && i < issued; i++) {
                stage = stage == 0 ? kDenseStages - 1 : stage - 1;
                if (stage == kDenseStages - 1) phase ^= 1;
                tc::bar_drain(full + stage, phase);
            }
        }
    } else if (warp == 1 && lane == 0) {                            // ---- products
        const int v64 = (p.V + 63) & ~63, d64 = d_blocks * 64;
        const uint32_t as_l = tc::instruction(kXM, v32, false, false), as_x = tc::instruction(kXM, d64, false, true),
                       as_w = tc::instruction(kXM, v64, true, true);
        const uint64_t wk = tc::operand(sw, 16, 1024), wn = tc::operand(sw, v32 * 128, 1024);
        const uint64_t gk = tc::operand(sg, 16, 1024), gn = tc::operand(sg, 16384, 1024);
        const int k_l = (D + 15) / 16, k_x = v32 / 16;
        int stage = 0, ahead = 0;                                    // of the tile whose dx and dw are next; of the one whose logits are
        uint32_t ahead_phase = 0;
        auto form = [&](int i) {                                     // logits of tile i
            if (!tc::bar_wait(full + ahead, ahead_phase, dead, p.err_flag)) return false;
            if (i > 0 && !tc::bar_wait(read, (i - 1) & 1, dead, p.err_flag)) return false;
            tc::fence_after();
            const uint64_t xk = tc::operand(sx + ahead * kDenseX, 16, 1024);
            for (int kk = 0; kk < k_l; kk++)
                tc::mma<false>(tmem + kDenseTL, xk + (kk >> 2) * 1024 + (kk & 3) * 2, wk + (kk >> 2) * (v32 * 8) + (kk & 3) * 2, as_l, kk > 0);
            tc::commit<false>(logits);
            if (++ahead == kDenseStages) { ahead = 0; ahead_phase ^= 1; }
            return true;
        };
        bool ok = tc::bar_wait(w_full, 0, dead, p.err_flag) && form(0);
        for (int i = 0; ok && i < mine; i++) {
            if (i + 1 < mine && !(ok = form(i + 1))) break;
            if (!(ok = tc::bar_wait(ready, i & 1, dead, p.err_flag))) break;
            tc::fence_after();
            if (dw) {
                const uint64_t xm = tc::operand(sx + stage * kDenseX, 16384, 1024);
                for (int kk = 0; kk < kXM / 16; kk++) tc::mma<false>(tmem + kDenseTW, xm + kk * 128, gn + kk * 128, as_w, i > 0 || kk > 0);
            }
            tc::commit<false>(empty + stage);
            if (++stage == kDenseStages) stage = 0;
            if (i > 0 && !(ok = tc::bar_wait(taken, (i - 1) & 1, dead, p.err_flag))) break;
            tc::fence_after();
            if (dx)
                for (int kk = 0; kk < k_x; kk++)
                    tc::mma<false>(tmem + kDenseTX, gk + (kk >> 2) * 1024 + (kk & 3) * 2, wn + kk * 128, as_x, kk > 0);
            tc::commit<false>(done);
        }
        if (!ok) {                                                  // products in flight read shared memory: wait for them
            tc::commit<false>(last);
            tc::bar_drain(last, 0);
        }
    } else if (warp >= 4) {                                         // ---- softmax and stores: a thread owns pieces of a row
        const int quarter = warp & 3, part = (warp - 4) >> 2;
        char *stage = staging + (warp - 4) * kXStaging;
        const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
        // The pieces of 32 columns of G, and behind them those of dx of the tile before, go round among the four warps of 32 rows
        // (150 classes, 96 features: 5 and 3, two for each).
        const int g_pieces = v32 / 32, x_pieces = dx ? (D + 31) / 32 : 0, first_x = (part - g_pieces) & 3;
        const float alpha = xent_alpha(p.alpha_up, p.alpha_count, p.alpha);
        double cols[2] = {0., 0.};                                   // column sums of G, of this warp's pieces and rows
        auto row_of = [&](int i) { return ((int)blockIdx.x + i * (int)gridDim.x) * kXM + quarter * 32; };
        auto await = [&](uint64_t *bar, int i) {
            const bool ok = __all_sync(0xffffffffu, tc::bar_wait(bar, i & 1, dead, p.err_flag));
            if (ok) tc::fence_after();
            return ok;
        };
        auto load = [&](uint32_t col, float (&a)[32]) {
            uint32_t r[32];
            tc::tmem_load32(lane_base + col, r);
            tc::tmem_wait32(r);
#pragma unroll
            for (int k = 0; k < 32; k++) a[k] = __uint_as_float(r[k]);
        };
        auto release = [&](uint64_t *bar) {
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tc::bar_arrive(bar);
        };
        auto store_dx = [&](int i) {
            const int r0 = row_of(i);
            if (first_x >= x_pieces) release(taken);
            for (int pc = first_x; pc < x_pieces; pc += 4) {
                float a[32];
                load(kDenseTX + pc * 32, a);
                if (pc + 4 >= x_pieces) release(taken);
                xent_store(dx, stage, lane, a, alpha, r0, p.M, pc * 32, D, p.vec);
            }
        };
        // (fetched while the tile before is worked on)
        auto fetch = [&](int i) { return xent_fetch(i < mine ? (long long)row_of(i) + lane : p.M, p); };
        if ((g_pieces & 1) && part == 0) {                          // the rest of the last block of G, which nothing writes
            const int row = quarter * 32 + lane;
#pragma unroll
            for (int j = 4; j < 8; j++) *reinterpret_cast<uint4 *>(sg + (g_pieces >> 1) * 16384 + row * 128 + ((j ^ (row & 7)) * 16)) = make_uint4(0u, 0u, 0u, 0u);
        }
        bool ok = true;
        XentAhead next = fetch(0);
        for (int i = 0; i < mine; i++) {
            const XentRow me = xent_row(next, p);
            const F2 lse = both(-(me.lse + me.lse_lo));
            next = fetch(i + 1);
            if (!(ok = await(logits, i))) break;
            if (part >= g_pieces) release(read);
            for (int j = 0, pc = part; pc < g_pieces; j++, pc += 4) {
                const int c0 = pc * 32;
                float a[32];
                load(kDenseTL + c0, a);
                if (pc + 4 >= g_pieces) release(read);
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                    const float4 b = *reinterpret_cast<const float4 *>(bias + c0 + k);
                    const float2 u = apart(add2(fma2(two(a[k], a[k + 1]), both(1.4426950408889634f), two(b.x, b.y)), lse));
                    const float2 v = apart(add2(fma2(two(a[k + 2], a[k + 3]), both(1.4426950408889634f), two(b.z, b.w)), lse));
                    a[k] = u.x; a[k + 1] = u.y; a[k + 2] = v.x; a[k + 3] = v.y;
                }
                xent_gradient(a, c0, me, p);
                const int at = xent_at(me, c0);
                if (p.cols) {
                    const float s = column_sums(a, lane, stage, at, me.hot);
                    if (j == 0) cols[0] += s; else cols[1] += s;
                }
                uint4 out[4];
                uint32_t *o = reinterpret_cast<uint32_t *>(out);
#pragma unroll
                for (int k = 0; k < 16; k++) o[k] = pack_bf16(a[2 * k], a[2 * k + 1]);
                if (j == 0 && i > 0 && !(ok = await(done, i - 1))) break;      // G of the tile before is read
                const int row = quarter * 32 + lane;
                unsigned char *to = sg + (pc >> 1) * 16384 + row * 128;
                auto chunk = [&](int k) { return to + (((pc & 1) * 4 + k) ^ (row & 7)) * 16; };
#pragma unroll
                for (int k = 0; k < 4; k++) *reinterpret_cast<uint4 *>(chunk(k)) = out[k];
                if (at >= 0) reinterpret_cast<__nv_bfloat16 *>(chunk(at >> 3))[at & 7] = __float2bfloat16_rn(me.hot);
            }
            if (ok && part >= g_pieces && i > 0) ok = await(done, i - 1);
            if (!ok) break;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // the products read what was written
            __syncwarp();
            if (lane == 0) tc::bar_arrive(ready);
            if (i > 0) store_dx(i - 1);
        }
        if (ok && (ok = await(done, mine - 1))) {
            store_dx(mine - 1);
            if (dw && quarter * 32 < D) {                            // dw^T: a lane owns a feature, so that lanes store side by side
                const int d = quarter * 32 + lane;
                float *to = dw + (long long)blockIdx.x * p.V * D + d;
                for (int pc = part; pc < g_pieces; pc += 4) {
                    float a[32];
                    load(kDenseTW + pc * 32, a);
#pragma unroll
                    for (int k = 0; k < 32; k++)
                        if (d < D && pc * 32 + k < p.V) to[(long long)(pc * 32 + k) * D] = a[k];
                }
            }
        }
        if (p.cols) {                                               // the four quarters' sums of a column in one
            double *mine_of = reinterpret_cast<double *>(stage);
            mine_of[lane] = cols[0];
            mine_of[lane + 32] = cols[1];
            asm volatile("bar.sync 1, %0;" ::"n"(32 * kXFinish) : "memory");      // (those that gave up come here, too)
            for (int h = quarter; h < 2; h += 4) {
                double t = 0.;
#pragma unroll
                for (int q = 0; q < 4; q++) t += reinterpret_cast<const double *>(staging + (part * 4 + q) * kXStaging)[h * 32 + lane];
                if (ok && part + 4 * h < g_pieces) p.cols[(long long)blockIdx.x * p.cols_ld + (part + 4 * h) * 32 + column_of(lane)] = (float)t;
            }
        }
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (warp == 2) tc::tmem_free<false>(tmem, 512);
}

}  // namespace o1d

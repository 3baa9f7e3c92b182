// How the linear operators' products are cut (linear.cu): host code without CUDA, so that it can be
// compiled and walked where there is no GPU.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <algorithm>

namespace brk {

constexpr int kLF = 128;                // MMA rows (TMEM lanes) per CTA
constexpr int kLK = 64;                 // k per step: one 128-byte swizzled row
constexpr int kDrainK = 16;             // k steps per accumulator set when draining
constexpr uint32_t kRing = 208 * 1024;  // bytes of the load ring
constexpr int kMaxStages = 16;

// Columns that an epilogue warp handles at a time in the kernel of token tile nt_kernel.  f32 outputs (which
// drain) come with a residual's loads to hide: 32 (2048 x 2560 -> 10240 112 us, 124 with 16); fp16 outputs
// are bound by the epilogue's instructions, whose registers spill at 32 (3000 x 1024 -> 4096 31.5 us, 26.7
// with 16).
constexpr int linear_chunk(int nt_kernel, bool drain) { return drain && nt_kernel >= 64 ? 32 : 16; }

// Whether brk_linear's accumulators are drained on the way, every 1024 of k: the tensor cores' f32
// accumulation truncates, and loses up to 5.9e-9 of the sum for each of k (operands of one sign; 6e-5 at
// 10240, 3.9e-4 at 65536; drained 5.5e-6 at any k).  An f32 output always, an fp16 one (half a step is
// 4.9e-4) where it would lose more than a fifth of that.
constexpr bool linear_drains(bool f32_out, int k) { return f32_out || k > 16384; }

constexpr int linear_round_up(int v, int m) { return (v + m - 1) / m * m; }

// How a linear product is cut: the kernel's token tile, tokens per tile, rows of the TMA boxes of x
// and w, tiles, k, CTAs, workspace floats and counters.
struct LinearPlan {
    bool pair, ranged, flat, drain;
    int cs, nt_kernel, nt, x_rows, w_rows, f_rows, half_cols, tiles_m, nk, kb, stages, drain_steps, ctas;
    long long tiles, tiles_whole;
    int range_units, range_extra;
    size_t ws_floats, counters;
};

// The cheapest cut by a model in SM cycles.  A k step of a tile costs the larger of its products
// (nt / 2 cycles, at least 32 for reading 128 rows, for each 16 of k and accumulator) and its bytes
// through L2 (48 per cycle and SM with every SM loading); the whole product at least its weights from
// HBM (3390 bytes a cycle).  On top: launch, ramp and the last tile's epilogue, and what joins split
// tiles.  drain: the accumulators are drained on the way (mats 1).  max_clusters(size): how many clusters
// of that many CTAs fit at once.
template <typename Clusters>
LinearPlan linear_plan_for(int rows, int k, int n, int mats, bool drain, int sms, Clusters max_clusters) {
    const int nkb = (k + kLK - 1) / kLK;
    const double hbm = 2.0 * mats * n * (double)k / 3390.0;
    LinearPlan best;
    double best_cost = 1e300;
    auto consider = [&](bool pair, int tiles_m, int f, int cs, bool ranged) {
        LinearPlan p;
        const int unit = pair ? 32 : 16, ctas = pair ? 2 : 1;
        p.pair = pair;
        p.cs = cs;
        p.tiles_m = tiles_m;
        p.nt = linear_round_up((rows + tiles_m - 1) / tiles_m, unit);
        if (p.nt > 256) return;
        p.nt_kernel = p.nt <= 16 ? 16 : p.nt <= 32 ? 32 : p.nt <= 64 ? 64 : p.nt <= 128 ? 128 : 256;
        if (pair && p.nt_kernel < 128) p.nt_kernel = 128;
        p.f_rows = f;
        const int accs = pair ? 1 : mats;
        if (cs > 1 && (uint32_t)(accs * p.nt * kLF * 4) > kRing) return;
        const long long ftiles = (n + (long long)f * ctas - 1) / (f * ctas);
        p.tiles = ftiles * tiles_m;
        const long long slots = std::max(1, cs > 1 ? max_clusters(ctas * cs) : sms / ctas);
        if (cs > 1 && p.tiles > slots) return;
        const int lanes = pair ? kLF : f * mats;  // weight rows of a k step and CTA
        const double step = std::max(accs * 4.0 * std::max(p.nt / 2, 32), (lanes + p.nt / ctas) * 128 / 48.0);
        const double epilogue = 800.0 + p.nt * (accs == 2 ? 60.0 : 24.0);
        double cost;
        if (ranged) {
            const double join = 4000.0 + p.nt * 60.0;
            cost = (double)p.tiles * nkb / slots * step + join + epilogue;
        } else if (cs > 1) {
            cost = (double)((nkb + cs - 1) / cs) * step + 3000.0 + accs * p.nt * 12.0 + epilogue / cs;
        } else {
            cost = (double)((p.tiles + slots - 1) / slots) * nkb * step + epilogue;
        }
        cost = std::max(cost, hbm) + (pair ? 5000.0 : 4000.0);
        if (cost < best_cost) {
            best_cost = cost;
            p.ranged = ranged;
            best = p;
        }
    };
    const int tm0 = (rows + 255) / 256, pair_f = mats == 2 ? kLF / 2 : kLF;
    for (int tm = tm0; tm <= tm0 + 2; ++tm) {
        if (tm > tm0 && tm > rows) break;
        // One CTA (cluster) per tile: the feature count that makes the tiles fill one, two, ... waves.
        for (int cs = 1; cs <= 8; ++cs) {
            if (cs > nkb) break;
            const int slots = cs > 1 ? max_clusters(cs) : sms;
            for (int w = 1; w <= (cs > 1 ? 1 : 4); ++w) {
                const long long ft = (long long)slots * w / tm;
                if (ft < 1) continue;
                const int f = linear_round_up((int)((n + ft - 1) / ft), 8);
                if (f <= kLF) {
                    consider(false, tm, f, cs, false);
                    break;
                }
            }
        }
        consider(false, tm, kLF, 1, true);
        if (rows > 32) {
            for (int cs = 1; cs <= 4 && cs <= nkb; ++cs) consider(true, tm, pair_f, cs, false);
            consider(true, tm, pair_f, 1, true);
        }
    }
    LinearPlan &p = best;
    const int ctas = p.pair ? 2 : 1;
    p.x_rows = p.nt / ctas;
    // Whole chunks: the drain stores its sums back in chunks, and a column that both epilogue warps of a lane
    // quarter stored would count the earlier sets of one of them twice.
    p.drain = drain;
    p.half_cols = p.nt_kernel >= 64 ? linear_round_up((p.nt + 1) / 2, linear_chunk(p.nt_kernel, drain)) : p.nt;
    p.w_rows = p.f_rows;
    // k steps per stage: one TMA fetches up to eight (k a multiple of 64), a stage about 32 KB.
    const bool by_step = k % kLK == 0 && !p.pair;
    const int step_rows = (p.pair ? kLF : p.f_rows * mats) + p.x_rows;
    p.kb = 1;
    while (by_step && p.kb < 8 && 2 * p.kb * step_rows * 128 <= 40 * 1024 && nkb >= 4 * p.kb * p.cs) p.kb *= 2;
    p.flat = p.kb == 1;
    p.stages = std::min<int>(kMaxStages, kRing / (p.kb * step_rows * 128));
    p.nk = (nkb + p.kb - 1) / p.kb;
    p.drain_steps = kDrainK / p.kb;
    // Workers: a CTA (pair, cluster) per SM (two, ...), no more than there is work for.
    long long workers = p.cs > 1 ? p.tiles : std::max(1, sms / ctas);
    workers = std::min<long long>(workers, p.ranged ? p.tiles * p.nk : p.tiles);
    // Ranged: whole waves of tiles, but for the last one to two waves' (unless they divide).
    p.tiles_whole = p.tiles;
    if (p.ranged && p.tiles % workers) {
        const long long waves = p.tiles / workers;
        p.tiles_whole = waves > 0 ? (waves - 1) * workers : 0;
    }
    p.ctas = (int)workers * ctas * p.cs;
    const long long units = (p.tiles - p.tiles_whole) * p.nk;
    p.range_units = (int)(units / workers), p.range_extra = (int)(units % workers);
    p.counters = (size_t)(p.tiles - p.tiles_whole) * ctas;
    p.ws_floats = p.tiles > p.tiles_whole ? (size_t)p.ctas * 2 * ((p.pair ? 1 : mats) * p.nt + 16) * kLF : 0;
    return p;
}

}  // namespace brk

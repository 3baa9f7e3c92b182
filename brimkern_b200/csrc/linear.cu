// Matrix products of the layer around the attention operator on fp16 activations: the linear
// operator y = act(x W^T + b) + r and the gated feed-forward's first half
// h = act(x Wg^T + bg) * (x Wu^T + bu) (the FFN of recordLayerKV, kernels.ts:1737-1744).
//
// linear_kernel<NT, MATS, PAIR, DRAIN> computes D^T = W X^T on tcgen05: weight rows (output features) on the
// MMA's M, up to NT tokens on its N, so a single token pads 15 MMA columns and not 127 rows, and the
// token tile follows the row count in steps of 16 (32).  PAIR: two SMs of a cluster work on one tile
// (cta_group::2, M 256): each holds its 128 features' weights and half of the tokens, so a k step
// costs an SM half the activation bytes.  With MATS = 2 a CTA holds the gate and the up tile of the
// same features in two accumulators, and the product leaves through one epilogue.
//
// Work is dealt so that every SM has the same amount: first whole waves of tiles (neighbouring CTAs
// on neighbouring token tiles, so they share weights in L2), the last one to two waves' tiles as
// (tile, k step) units in equal contiguous ranges.  A range's first and last piece may cover part
// of a tile's k; such pieces leave f32 partials in the workspace, and the last CTA of a tile to
// finish adds them in k order (the same order whoever is last: results do not change from run to
// run).  The ranges come first, so that the joins run under the whole tiles.  Few tokens, bound by
// streaming the weights once, have nothing but ranges.
//
// The tensor core's f32 accumulation truncates: its error is a bias that grows with k (measured on
// N(0,1) operands against 64 bits: 3.1e-6 of the result at k 2560, 1.2e-5 at 10240).  For f32
// outputs (DRAIN) the accumulators are drained every kDrainSteps k steps and the parts added in
// registers; fp16 outputs (half a step 4.9e-4) do not need it.
#include <algorithm>

#include "common.cuh"
#include "internal.h"
#include "tcgen05.cuh"

namespace brk {

namespace {

constexpr int kLF = 128;         // output features per CTA and tile (TMEM lanes)
constexpr int kLK = 64;          // k per step: one 128-byte swizzled row
constexpr int kDrainSteps = 16;  // 1024 of k per accumulator

template <int NT, int MATS, bool PAIR>
struct LinearLayout {
    static constexpr int kCtas = PAIR ? 2 : 1;
    static constexpr uint32_t kWBox = kLF * 128;
    static constexpr uint32_t kXBox = NT / kCtas * 128;
    static constexpr uint32_t kStageBytes = MATS * kWBox + kXBox;
    static constexpr int kFit = (204 * 1024) / kStageBytes;
    static constexpr int kStages = kFit < 12 ? kFit : 12;
    static constexpr uint32_t kCols = MATS * NT;                  // one accumulator set
    static constexpr int kBufs = 2 * kCols <= 512 ? 2 : 1;
    static constexpr uint32_t kTmemCols = kBufs * kCols < 32 ? 32 : kBufs * kCols;
    static constexpr int kHalves = NT >= 64 ? 2 : 1;              // epilogue warps per TMEM lane quarter
    static constexpr int kEpiWarps = 4 * kHalves;
    static constexpr int kEpiCols = NT / kHalves;                 // most columns of an epilogue thread
    static constexpr int kChunk = 16;                             // columns handled at a time
    static constexpr int kProducer = kEpiWarps, kMma = kEpiWarps + 1;
    static constexpr int kThreads = (kEpiWarps + 2) * 32;
    static constexpr uint32_t kBarOff = kStages * kStageBytes;
    static constexpr uint32_t kSmemBytes = 1024 + kBarOff + (2 * kStages + 4) * 8 + 16;
    static_assert(kTmemCols <= 512 && (kTmemCols & (kTmemCols - 1)) == 0, "TMEM columns");
    static_assert(kSmemBytes <= 232448 - 64, "more than 227 KB of shared memory per CTA");
};

// The ranged tiles' units are dealt to the workers in contiguous ranges: the first a.range_extra
// workers have a.range_units + 1, the others a.range_units.
__device__ __forceinline__ int range_begin(const LinearArgs &a, int c) { return c * a.range_units + min(c, a.range_extra); }
__device__ __forceinline__ int worker_of(const LinearArgs &a, int u) {
    const int longer = a.range_extra * (a.range_units + 1);
    return u < longer ? u / (a.range_units + 1) : a.range_extra + (u - longer) / a.range_units;
}

// The pieces (tile, k steps [k0, k1)) of worker c, in the order every role walks them, with the
// tile's feature and token tile.
struct Pieces {
    int u, u_hi, whole_next, whole_end, step, nk, tiles_m;
    int tile, ftile, mtile, k0, k1;
    __device__ Pieces(const LinearArgs &a, int c, int workers) {
        u = range_begin(a, c), u_hi = range_begin(a, c + 1);
        whole_next = c, whole_end = a.tiles_whole, step = workers;
        nk = a.nk, tiles_m = a.tiles_m;
    }
    __device__ bool next() {
        if (u < u_hi) {
            const int t = u / nk;
            tile = whole_end + t;
            k0 = u - t * nk;
            k1 = min(nk, k0 + u_hi - u);
            u += k1 - k0;
        } else if (whole_next < whole_end) {
            tile = whole_next;
            whole_next += step;
            k0 = 0, k1 = nk;
        } else {
            return false;
        }
        ftile = tile / tiles_m;
        mtile = tile - ftile * tiles_m;
        return true;
    }
};

// The k steps of all pieces, one after the other.
struct Steps {
    Pieces p;
    int k = -1;
    __device__ Steps(const Pieces &pieces) : p(pieces) { p.k1 = 0; }
    __device__ bool next() {
        if (++k < p.k1) return true;
        if (!p.next()) return false;
        k = p.k0;
        return true;
    }
};

// v * 1 / (1 + e^-z): with the hardware's 2^x and reciprocal, a few 2^-23 of the result.
__device__ __forceinline__ float times_sigmoid(float v, float z) {
    return v * rcp_fast(1.f + ex2_fast(-1.4426950408889634f * z));
}

// act(v) in f32; tanh y = 2 sigmoid(2 y) - 1 turns gelu_tanh into a sigmoid too.
template <int ACT>
__device__ __forceinline__ float apply_act(float v) {
    if constexpr (ACT == BRK_ACT_SILU) return times_sigmoid(v, v);
    if constexpr (ACT == BRK_ACT_GELU) return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
    if constexpr (ACT == BRK_ACT_GELU_TANH) return times_sigmoid(v, 1.5957691216057308f * fmaf(0.044715f * v * v, v, v));
    if constexpr (ACT == BRK_ACT_QUICK_GELU) return times_sigmoid(v, 1.702f * v);
    return v;
}

// The finished values of one feature for CH tokens, at out[o + e * n] (e < count): act(v + b0)
// (* (w + b1)), + residual.
template <int ACT, int MATS, int CH>
__device__ __forceinline__ void finish_act(const LinearArgs &a, size_t o, int count, float b0, float b1,
                                           const float (&v)[CH], const float (&w)[CH]) {
    const size_t n = (size_t)a.n;
    float y[CH];
    if (MATS == 1 && a.residual) {
        const float *res = a.residual + o;
#pragma unroll
        for (int e = 0; e < CH; ++e) y[e] = e < count ? res[e * n] : 0.f;
    } else {
#pragma unroll
        for (int e = 0; e < CH; ++e) y[e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < CH; ++e) {
        const float x = apply_act<ACT>(v[e] + b0);
        y[e] = MATS == 2 ? x * (w[e] + b1) : x + y[e];
    }
    if (a.out_half) {
        __half *out = static_cast<__half *>(a.out) + o;
#pragma unroll
        for (int e = 0; e < CH; ++e)
            if (e < count) out[e * n] = __float2half_rn(y[e]);
    } else {
        float *out = static_cast<float *>(a.out) + o;
#pragma unroll
        for (int e = 0; e < CH; ++e)
            if (e < count) out[e * n] = y[e];
    }
}
template <int MATS, int CH>
__device__ __forceinline__ void finish(const LinearArgs &a, size_t o, int count, float b0, float b1, const float (&v)[CH],
                                       const float (&w)[CH]) {
    switch (a.act) {
        case BRK_ACT_SILU: return finish_act<BRK_ACT_SILU, MATS, CH>(a, o, count, b0, b1, v, w);
        case BRK_ACT_GELU: return finish_act<BRK_ACT_GELU, MATS, CH>(a, o, count, b0, b1, v, w);
        case BRK_ACT_GELU_TANH: return finish_act<BRK_ACT_GELU_TANH, MATS, CH>(a, o, count, b0, b1, v, w);
        case BRK_ACT_QUICK_GELU: return finish_act<BRK_ACT_QUICK_GELU, MATS, CH>(a, o, count, b0, b1, v, w);
        default: return finish_act<BRK_ACT_NONE, MATS, CH>(a, o, count, b0, b1, v, w);
    }
}

// 16 consecutive 32-bit TMEM columns of this thread's lane (no wait).
__device__ __forceinline__ void tc_ld16_nowait(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// The address, in the cluster's shared memory, of `p`'s counterpart in CTA `rank`.
__device__ __forceinline__ uint32_t cluster_addr(const void *p, uint32_t rank) {
    uint32_t d;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(smem_addr(p)), "r"(rank));
    return d;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// 2-D tiled TMA load into this CTA's shared memory whose bytes count on a barrier of the CTA pair.
__device__ __forceinline__ void tma_load_2d_pair(void *dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tc_mma_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                            bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}
// Arrives on `bar` (and its counterpart in the other CTA of the pair) when the MMAs so far are done.
__device__ __forceinline__ void tc_commit_pair(uint64_t *bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_addr(bar)),
        "h"((uint16_t)3)
        : "memory");
}

template <int NT, int MATS, bool PAIR, bool DRAIN>
__global__ void __launch_bounds__(LinearLayout<NT, MATS, PAIR>::kThreads, 1)
    linear_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw0,
                  const __grid_constant__ CUtensorMap tw1, const __grid_constant__ LinearArgs a) {
    using L = LinearLayout<NT, MATS, PAIR>;
    constexpr int S = L::kStages, CH = L::kChunk, CTAS = L::kCtas, BUFS = L::kBufs;
    constexpr int EPI = L::kEpiWarps * 32;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::kBarOff);  // PAIR: the even CTA's count
    uint64_t *empty = full + S;
    uint64_t *accfull = empty + S;
    uint64_t *accfree = accfull + 2;                                   // PAIR: the even CTA's count
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(accfree + 2);
    __shared__ int s_last;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = PAIR ? (int)(blockIdx.x & 1) : 0;
    const int worker = blockIdx.x / CTAS, workers = gridDim.x / CTAS;
    const int nt = a.nt;  // tokens per tile: the MMA's N
    const Pieces pieces(a, worker, workers);

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&accfull[i], 1);
            mbar_init(&accfree[i], L::kEpiWarps * CTAS);  // a warp's arrival each
        }
        fence_barrier_init();
    }
    if (warp == L::kMma) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                         "r"(L::kTmemCols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                         "r"(L::kTmemCols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_sync_all();  // both CTAs' barriers and TMEM are there
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == L::kProducer) {
        if (lane == 0) {
            tma_prefetch_desc(&tx);
            tma_prefetch_desc(&tw0);
            if constexpr (MATS == 2) tma_prefetch_desc(&tw1);
            const uint32_t x_rows = (uint32_t)nt / CTAS;
            const uint32_t stage_tx = (MATS * L::kWBox + x_rows * 128) * CTAS;  // both CTAs' bytes
            auto arm = [&](int s) {
                if (rank == 0) mbar_arrive_expect_tx(&full[s], stage_tx);
            };
            auto load = [&](void *dst, const CUtensorMap *map, int x, int y, int s) {
                if constexpr (PAIR)
                    tma_load_2d_pair(dst, map, x, y, cluster_addr(&full[s], 0));
                else
                    tma_load_2d(dst, map, x, y, &full[s]);
            };
            auto load_w = [&](const Steps &t, int s) {
                uint8_t *st = smem + s * L::kStageBytes;
                const int f0 = (t.p.ftile * CTAS + rank) * kLF;
                load(st, &tw0, t.k * kLK, f0, s);
                if constexpr (MATS == 2) load(st + L::kWBox, &tw1, t.k * kLK, f0, s);
            };
            auto load_x = [&](const Steps &t, int s) {
                const int m0 = t.p.mtile * nt + rank * (int)x_rows;
                load(smem + s * L::kStageBytes + MATS * L::kWBox, &tx, t.k * kLK, m0, s);
            };
            // The weights of the first ring do not depend on the kernel before (which, in the same
            // call, writes the activations): they are in flight before the wait for it.
            Steps w(pieces), x(pieces);
            int j = 0;  // k steps loaded
            bool more = true;
            while (j < S && (more = w.next())) {
                arm(j);
                load_w(w, j);
                ++j;
            }
            griddep_wait();
            for (int i = 0; i < j; ++i) {
                x.next();
                load_x(x, i);
            }
            uint32_t phase = 0;
            for (int s = 0; more && w.next(); ++j) {
                if (!mbar_wait(&empty[s], phase, a.err, kErrSlotTimeout)) break;
                arm(s);
                load_w(w, s);
                load_x(w, s);
                if (++s == S) s = 0, phase ^= 1;
            }
            // The next kernel of the call may start streaming its weights (what ran before this one is
            // complete: the wait above).
            griddep_launch_dependents();
            // No copy may still be in flight when a CTA exits (the even CTA's barriers count both's).
            for (int i = j > S ? j - S : 0; rank == 0 && i < j; ++i)
                mbar_wait(&full[i % S], (uint32_t)(i / S) & 1, a.err, kErrTmaTimeout);
        }
        __syncwarp();
    } else if (warp == L::kMma) {
        if (lane == 0 && rank == 0) {
            const uint32_t idesc = f16_idesc(kLF * CTAS, nt, 0, 0);
            auto commit = [&](uint64_t *bar) {
                if constexpr (PAIR)
                    tc_commit_pair(bar);
                else
                    tc_commit(bar);
            };
            Pieces p = pieces;
            int s = 0;              // ring stage, with its phase
            uint32_t phase = 0;
            int seg = 0;            // accumulator sets used
            constexpr int seg_steps = DRAIN ? kDrainSteps : 1 << 30;
            bool ok = true;
            while (ok && p.next()) {
                for (int ks = p.k0; ok && ks < p.k1; ks += seg_steps) {
                    const int ke = p.k1 - ks < seg_steps ? p.k1 : ks + seg_steps;
                    const int buf = seg % BUFS;
                    if (seg >= BUFS && !mbar_wait(&accfree[buf], ((seg / BUFS) - 1) & 1, a.err, kErrMmaTimeout)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t d = tmem + buf * L::kCols;
                    for (int kk = ks; kk < ke; ++kk) {
                        if (!mbar_wait(&full[s], phase, a.err, kErrTmaTimeout)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t w = smem_addr(smem + s * L::kStageBytes), x = w + MATS * L::kWBox;
#pragma unroll
                        for (int e = 0; e < kLK / 16; ++e)
#pragma unroll
                            for (int m = 0; m < MATS; ++m) {
                                const uint64_t wd = sw128_desc(w + m * L::kWBox + e * 32, 16, 1024);
                                const uint64_t xd = sw128_desc(x + e * 32, 16, 1024);
                                if constexpr (PAIR)
                                    tc_mma_pair(d + m * NT, wd, xd, idesc, kk > ks || e > 0);
                                else
                                    tc_mma(d + m * NT, wd, xd, idesc, kk > ks || e > 0);
                            }
                        commit(&empty[s]);
                        if (++s == S) s = 0, phase ^= 1;
                    }
                    if (ok) {
                        commit(&accfull[buf]);
                        ++seg;
                    }
                }
            }
            // Every MMA issued completes before TMEM is released: the last sets' commits.
            for (int b = 0; b < BUFS; ++b) {
                const int used = (seg + BUFS - 1 - b) / BUFS;  // sets committed on accumulator b
                if (used > 0) mbar_wait(&accfull[b], (used - 1) & 1, a.err, kErrMmaTimeout);
            }
        }
        __syncwarp();
    } else {
        // ---- epilogue warps: TMEM lane r <-> feature, columns <-> tokens; two warps per lane quarter
        // (NT >= 64) take half of the columns each.
        const int r = (warp & 3) * 32 + lane;
        const int col0 = (warp >> 2) * (L::kHalves == 1 ? 0 : a.half_cols);
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        griddep_wait();  // the residual may come from, and the output may be read by, what ran before
        auto ld_cols = [&](uint32_t col, uint32_t (&v)[CH]) { tc_ld16_nowait(tmem + lane_base + col, v); };
        auto st_cols = [&](uint32_t col, const uint32_t (&v)[CH]) { tc_st16(tmem + lane_base + col, v); };
        auto release = [&](int buf) {  // the accumulator may be overwritten
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR)
                    mbar_arrive_cluster(cluster_addr(&accfree[buf], 0));
                else
                    mbar_arrive(&accfree[buf]);
            }
        };
        Pieces p = pieces;
        int seg = 0;
        bool ok = true;
        bool first_piece = true;
        while (p.next()) {
            const int k0 = p.k0, k1 = p.k1;
            const bool at_lo = first_piece;  // a ranged piece that begins at the range's begin
            first_piece = false;
            const int feat = (p.ftile * CTAS + rank) * kLF + r;
            const int m0 = p.mtile * nt + col0;                   // token of this thread's first column
            const int ntok = min(min(a.half_cols, nt - col0), a.M - m0);  // columns that count (may be <= 0)
            const bool whole = k0 == 0 && k1 == a.nk;
            const size_t slot_floats = (size_t)MATS * nt * kLF;
            const bool in = feat < a.n;
            const float b0 = in && a.bias[0] ? a.bias[0][feat] : 0.f;
            const float b1 = MATS == 2 && in && a.bias[1] ? a.bias[1][feat] : 0.f;
            const size_t o0 = (size_t)m0 * a.n + feat;
            float *part = a.ws + ((size_t)blockIdx.x * 2 + (at_lo ? 0 : 1)) * slot_floats + (size_t)col0 * kLF + r;
            if constexpr (DRAIN) {
                // All accumulator sets of the piece but the last into registers; their sum goes back
                // into the last one's columns.
                if (k1 - k0 > kDrainSteps) {
                    float acc[L::kEpiCols];
#pragma unroll
                    for (int e = 0; e < L::kEpiCols; ++e) acc[e] = 0.f;
                    for (int ks = k0; ks < k1; ks += kDrainSteps) {
                        const int buf = seg % BUFS;
                        const bool last = ks + kDrainSteps >= k1;
                        const bool got = ok && mbar_wait(&accfull[buf], (seg / BUFS) & 1, a.err, kErrMmaTimeout);
                        ok = __all_sync(0xffffffffu, got);
                        tc_fence_after();
#pragma unroll
                        for (int c0 = 0; c0 < L::kEpiCols; c0 += CH) {
                            if (c0 < ntok) {
                                uint32_t v[CH];
                                ld_cols(buf * L::kCols + col0 + c0, v);
                                tc_wait_ld();
#pragma unroll
                                for (int e = 0; e < CH; ++e) acc[c0 + e] += __uint_as_float(v[e]);
                                if (last) {
#pragma unroll
                                    for (int e = 0; e < CH; ++e) v[e] = __float_as_uint(acc[c0 + e]);
                                    st_cols(buf * L::kCols + col0 + c0, v);
                                }
                            }
                        }
                        if (!last) {
                            release(buf);
                            ++seg;
                        }
                    }
                    tc_wait_st();
                }
            }
            const int buf = seg % BUFS;
            // After one timeout no further set is waited for (the error word is set).
            const bool got = ok && mbar_wait(&accfull[buf], (seg / BUFS) & 1, a.err, kErrMmaTimeout);
            ok = __all_sync(0xffffffffu, got);
            ++seg;
            tc_fence_after();
#pragma unroll 1
            for (int c0 = 0; c0 < ntok; c0 += CH) {
                uint32_t vr[CH], wr[CH];
                ld_cols(buf * L::kCols + col0 + c0, vr);
                if constexpr (MATS == 2) ld_cols(buf * L::kCols + NT + col0 + c0, wr);
                tc_wait_ld();
                float v[CH], w[CH];
#pragma unroll
                for (int e = 0; e < CH; ++e) v[e] = __uint_as_float(vr[e]), w[e] = MATS == 2 ? __uint_as_float(wr[e]) : 0.f;
                if (whole) {
                    if (in) finish<MATS, CH>(a, o0 + (size_t)c0 * a.n, ntok - c0, b0, b1, v, w);
                } else {
                    float *dst = part + (size_t)c0 * kLF;
#pragma unroll
                    for (int e = 0; e < CH; ++e)
                        if (c0 + e < ntok) {
                            __stcg(dst + e * kLF, v[e]);
                            if constexpr (MATS == 2) __stcg(dst + (size_t)(nt + e) * kLF, w[e]);
                        }
                }
            }
            release(buf);
            if (!whole) {
                // The last CTA of the tile (and rank) to finish adds the pieces in k order.
                __threadfence();
                named_barrier_sync(2, EPI);
                const int t0 = (p.tile - a.tiles_whole) * a.nk;
                const int c_first = worker_of(a, t0), c_last = worker_of(a, t0 + a.nk - 1);
                if (threadIdx.x == 0) {
                    int *counter = a.counters + (p.tile - a.tiles_whole) * CTAS + rank;
                    const int prev = atomicAdd(counter, 1);
                    s_last = prev == c_last - c_first;
                    if (s_last) *counter = 0;  // ready for the next launch
                }
                named_barrier_sync(2, EPI);
                if (s_last) {
                    __threadfence();
#pragma unroll 1
                    for (int c0 = 0; c0 < ntok; c0 += CH) {
                        float v[CH], w[CH];
#pragma unroll
                        for (int e = 0; e < CH; ++e) v[e] = w[e] = 0.f;
                        // Two pieces' loads in flight at a time.
#pragma unroll 1
                        for (int q = c_first; q <= c_last; q += 2) {
                            float x[2][MATS][CH];
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const bool there = q + h <= c_last;
                                const int slot = range_begin(a, q + h) >= t0 ? 0 : 1;
                                const float *src = a.ws + ((size_t)((q + h) * CTAS + rank) * 2 + slot) * slot_floats +
                                                   (size_t)(col0 + c0) * kLF + r;
#pragma unroll
                                for (int m = 0; m < MATS; ++m)
#pragma unroll
                                    for (int e = 0; e < CH; ++e)
                                        x[h][m][e] = there && c0 + e < ntok ? __ldcg(src + (size_t)(m * nt + e) * kLF) : 0.f;
                            }
#pragma unroll
                            for (int h = 0; h < 2; ++h)
#pragma unroll
                                for (int e = 0; e < CH; ++e) {
                                    v[e] += x[h][0][e];
                                    if constexpr (MATS == 2) w[e] += x[h][MATS - 1][e];
                                }
                        }
                        if (in) finish<MATS, CH>(a, o0 + (size_t)c0 * a.n, ntok - c0, b0, b1, v, w);
                    }
                }
                named_barrier_sync(2, EPI);  // s_last is read before the next piece writes it
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_sync_all();  // no CTA leaves while the other's copies or commits reach it
    tc_fence_after();
    if (warp == L::kMma) {
        if constexpr (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::kTmemCols) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::kTmemCols) : "memory");
    }
}

template <int NT, int MATS, bool PAIR, bool DRAIN>
cudaError_t launch_linear_k(const CUtensorMap &tx, const CUtensorMap *tw, const LinearArgs &a, int ctas, cudaStream_t s,
                            bool pdl) {
    using L = LinearLayout<NT, MATS, PAIR>;
    static unsigned long long configured = 0;  // one bit per device: the opt-in is per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 64 || !(configured & (1ull << dev))) {
        cudaError_t e = cudaFuncSetAttribute(linear_kernel<NT, MATS, PAIR, DRAIN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             L::kSmemBytes);
        if (e != cudaSuccess) return e;
        if (dev < 64) configured |= 1ull << dev;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(L::kThreads);
    cfg.dynamicSmemBytes = L::kSmemBytes;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (PAIR) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = 2;
        attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, linear_kernel<NT, MATS, PAIR, DRAIN>, tx, tw[0], tw[MATS - 1], a);
}

// f32 outputs (linear only) drain their accumulators.
template <int NT, int MATS, bool PAIR>
cudaError_t launch_linear_t(const CUtensorMap &tx, const CUtensorMap *tw, const LinearArgs &a, int ctas, cudaStream_t s,
                            bool pdl) {
    if constexpr (MATS == 1)
        if (!a.out_half) return launch_linear_k<NT, 1, PAIR, true>(tx, tw, a, ctas, s, pdl);
    return launch_linear_k<NT, MATS, PAIR, false>(tx, tw, a, ctas, s, pdl);
}

template <int MATS>
cudaError_t launch_linear_m(const LinearPlan &p, const CUtensorMap &tx, const CUtensorMap *tw, const LinearArgs &a,
                            cudaStream_t s, bool pdl) {
    switch (p.nt_kernel) {
        case 16: return launch_linear_t<16, MATS, false>(tx, tw, a, p.ctas, s, pdl);
        case 32: return launch_linear_t<32, MATS, false>(tx, tw, a, p.ctas, s, pdl);
        case 64: return launch_linear_t<64, MATS, false>(tx, tw, a, p.ctas, s, pdl);
        case 128: return launch_linear_t<128, MATS, true>(tx, tw, a, p.ctas, s, pdl);
        case 256: return launch_linear_t<256, MATS, true>(tx, tw, a, p.ctas, s, pdl);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace

LinearPlan linear_plan(int rows, int k, int n, int mats, int sms) {
    LinearPlan p;
    const bool pair = rows > 64;
    // Token tiles: as few as 256 rows each allow, of equal size.
    p.tiles_m = (rows + 255) / 256;
    const int per = (rows + p.tiles_m - 1) / p.tiles_m, unit = pair ? 32 : 16;
    p.nt = (per + unit - 1) / unit * unit;
    p.nt_kernel = p.nt <= 16 ? 16 : p.nt <= 32 ? 32 : p.nt <= 64 ? 64 : p.nt <= 128 ? 128 : 256;
    if (!pair) p.nt = p.nt_kernel;
    const int ctas = pair ? 2 : 1;
    p.x_rows = p.nt / ctas;
    p.half_cols = p.nt_kernel >= 64 ? (p.nt / 2 + 15) / 16 * 16 : p.nt;
    const int feats = kLF * ctas;
    p.tiles = (long long)((n + feats - 1) / feats) * p.tiles_m;
    p.nk = (k + kLK - 1) / kLK;
    // Workers: a CTA (pair) per SM (two), no more than there are units.
    long long workers = sms / ctas;
    if (workers < 1) workers = 1;
    workers = std::min<long long>(workers, p.tiles * p.nk);
    // Whole waves of tiles, leaving one to two waves' tiles to the ranges (or none when they divide).
    long long waves = p.tiles / workers;
    if (p.tiles % workers && waves > 0) --waves;
    p.tiles_whole = waves * workers;
    p.ctas = (int)workers * ctas;
    const long long units = (p.tiles - p.tiles_whole) * p.nk;
    p.range_units = (int)(units / workers), p.range_extra = (int)(units % workers);
    p.counters = (size_t)(p.tiles - p.tiles_whole) * ctas;
    p.ws_floats = p.tiles > p.tiles_whole ? (size_t)p.ctas * 2 * mats * p.nt * kLF : 0;
    return p;
}

cudaError_t launch_linear(int mats, const LinearPlan &p, const CUtensorMap &tx, const CUtensorMap *tw,
                          const LinearArgs &a, cudaStream_t s, bool pdl) {
    return mats == 2 ? launch_linear_m<2>(p, tx, tw, a, s, pdl) : launch_linear_m<1>(p, tx, tw, a, s, pdl);
}

}  // namespace brk

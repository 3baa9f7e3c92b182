// Matrix products of the layer around the attention operator on fp16 activations: the linear
// operator y = act(x W^T + b) + r and the gated feed-forward's first half
// h = act(x Wg^T + bg) * (x Wu^T + bu) (the FFN of recordLayerKV, kernels.ts:1737-1744).
//
// linear_kernel computes D^T = W X^T on tcgen05: weight rows (output features) on the MMA's M, up to
// NT tokens on its N, so a single token pads 15 MMA columns and not 127 rows, and the token tile
// follows the row count in steps of 16 (32).  Three forms:
//   - one CTA per tile, for few tokens, which are bound by streaming the weights once: the tile's
//     feature count F (a multiple of 8, at most 128 of the MMA's rows) is chosen so that the tiles
//     just fill the SMs and none has to be split along k; a stage of the ring holds several k steps
//     when F is small (one TMA fetches them, [k step][row][64]);
//   - PAIR: two SMs of a cluster work on one tile (cta_group::2, M 256), each with its 128 features'
//     weights and half of the tokens, so that a k step costs an SM half the activation bytes: for
//     many tokens, bound by the tensor cores;
//   - few tiles over a long k: a cluster of `cs` CTAs (pairs) splits the k of one tile and joins the
//     parts through distributed shared memory, each CTA finishing a share of the tokens, so that the
//     SMs stream without a way through global memory;
//   - products whose tiles do not fill whole waves: the last one to two waves' tiles are dealt as
//     (tile, k step) units in equal contiguous ranges.  A range's first and last piece may cover part
//     of a tile's k; such pieces leave f32 partials in the workspace (the last to finish keeps its own
//     in TMEM), and the last CTA of a tile to finish adds them in k order, as the cluster's join does
//     (the same order whoever is last: results do not change from run to run).  The ranges come first,
//     so that the joins run under the whole tiles.
// Gate-up (MODE): a CTA holds the gate and the up tile of the same F features in two accumulators
// (kTwoAcc); with PAIR they are interleaved, 64 gate rows and 64 up rows in one accumulator
// (kInterleaved), which leaves TMEM for a second set: the epilogue of a tile runs under the next
// tile's products, and its warps swap halves of a chunk through shared memory.
//
// The tensor core's f32 accumulation truncates: its error is a bias that grows with k (measured on
// N(0,1) operands against 64 bits: 3.1e-6 of the result at k 2560, 1.2e-5 at 10240; on operands of one sign
// 6e-5).  For f32 outputs, and wide fp16 ones (linear_drains), the accumulators are drained every 1024 of k
// and the parts added in registers (DRAIN).
//
// Measured, replayed from a graph (eager, caches cold): gate-up 2560 -> 10240 of one token 18.6 us (18.9), 5.6
// TB/s of weights; of 64 tokens 25.5 us (26.7), bound by the stream and the exposed ramp and epilogue of one
// tile a CTA; of 2048 tokens 158 us (186, at the power cap), 1358 TFLOP/s, tensor pipe 76% active.  Linear 2048
// x 10240 -> 2560 with a residual 109 us (129) in f32, 93 in fp16 without: tensor pipe 53% active, then a join
// and an epilogue (9 to 12 thousand cycles) that no next tile hides.
#include <algorithm>

#include "common.cuh"
#include "internal.h"
#include "linear_plan.h"
#include "tcgen05.cuh"

namespace brk {

namespace {

constexpr uint32_t kSlack = 16 * 1024;   // behind the ring: the MMA's rows past F, or the gate / up swap

enum : int { kLinear = 0, kTwoAcc = 1, kInterleaved = 2 };

template <int NT, int MODE, bool PAIR>
struct LinearLayout {
    static constexpr int kCtas = PAIR ? 2 : 1;
    static constexpr int kMats = MODE == kTwoAcc ? 2 : 1;         // accumulators of a set
    static constexpr uint32_t kCols = kMats * NT;                 // TMEM columns of a set
    static constexpr int kBufs = 2 * kCols <= 512 ? 2 : 1;
    static constexpr uint32_t kTmemCols = kBufs * kCols < 32 ? 32 : kBufs * kCols;
    static constexpr int kHalves = NT >= 64 ? 2 : 1;              // epilogue warps per TMEM lane quarter
    static constexpr int kEpiWarps = 4 * kHalves;
    static constexpr int kEpiCols = NT / kHalves;                 // most columns of an epilogue thread
    template <bool DRAIN>
    static constexpr int chunk = linear_chunk(NT, DRAIN);         // columns that it handles at a time
    static constexpr int kProducer = kEpiWarps, kMma = kEpiWarps + 1;
    static constexpr int kThreads = (kEpiWarps + 2) * 32;
    static constexpr uint32_t kBarOff = kRing + kSlack;
    static constexpr uint32_t kSmemBytes = 1024 + kBarOff + (2 * kMaxStages + 4) * 8 + 16;
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
    int u, u_hi, whole_next, whole_end, step, nk, tiles_m, kw0, kw1;
    int tile, ftile, mtile, k0, k1;
    // split: the CTA's (pair's) part of a tile's k, of a.cs.
    __device__ Pieces(const LinearArgs &a, int c, int workers, int split) {
        u = range_begin(a, c), u_hi = range_begin(a, c + 1);
        whole_next = c, whole_end = a.tiles_whole, step = workers;
        nk = a.nk, tiles_m = a.tiles_m;
        kw0 = nk * split / a.cs, kw1 = nk * (split + 1) / a.cs;
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
            k0 = kw0, k1 = kw1;
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

// v[e] at out[e * n], e < count.  (A test per element is a branch each: 75 cycles a value and warp, 25
// without.)
__device__ __forceinline__ void store_as(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_as(float *p, float v) { *p = v; }
template <int CH, typename T>
__device__ __forceinline__ void store_column(T *out, size_t n, int count, const float (&v)[CH]) {
    if (count >= CH) {
#pragma unroll
        for (int e = 0; e < CH; ++e, out += n) store_as(out, v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < CH; ++e)
            if (e < count) store_as(out + e * n, v[e]);
    }
}

// The finished values of one feature for CH tokens, at out[o + e * n] (e < count): act(v + b0)
// * (w + b1) when GATED, else act(v + b0) + res.
template <int ACT, bool GATED, int CH>
__device__ __forceinline__ void finish_act(const LinearArgs &a, size_t o, int count, float b0, float b1,
                                           const float (&v)[CH], const float (&w)[CH]) {
    const size_t n = (size_t)a.n;
    float y[CH];
#pragma unroll
    for (int e = 0; e < CH; ++e) {
        const float x = apply_act<ACT>(v[e] + b0);
        y[e] = GATED ? x * (w[e] + b1) : x + w[e];
    }
    if (a.out_half)
        store_column<CH>(static_cast<__half *>(a.out) + o, n, count, y);
    else
        store_column<CH>(static_cast<float *>(a.out) + o, n, count, y);
}
template <bool GATED, int CH>
__device__ __forceinline__ void finish(const LinearArgs &a, size_t o, int count, float b0, float b1, const float (&v)[CH],
                                       const float (&w)[CH]) {
    switch (a.act) {
        case BRK_ACT_SILU: return finish_act<BRK_ACT_SILU, GATED, CH>(a, o, count, b0, b1, v, w);
        case BRK_ACT_GELU: return finish_act<BRK_ACT_GELU, GATED, CH>(a, o, count, b0, b1, v, w);
        case BRK_ACT_GELU_TANH: return finish_act<BRK_ACT_GELU_TANH, GATED, CH>(a, o, count, b0, b1, v, w);
        case BRK_ACT_QUICK_GELU: return finish_act<BRK_ACT_QUICK_GELU, GATED, CH>(a, o, count, b0, b1, v, w);
        default: return finish_act<BRK_ACT_NONE, GATED, CH>(a, o, count, b0, b1, v, w);
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
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}
__device__ __forceinline__ int ld_acquire_gpu(const int *p) {
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// 3-D tiled TMA load into this CTA's shared memory; PAIR: its bytes count on a barrier of the CTA pair.
template <bool PAIR>
__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
    if constexpr (PAIR)
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
            "%3, %4}], [%5];" ::"r"(smem_addr(dst)),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
            "[%5];" ::"r"(smem_addr(dst)),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
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
// Arrives on `bar` in both CTAs of the pair (their bits of the cluster in `pair_mask`) when the MMAs so
// far are done.
__device__ __forceinline__ void tc_commit_pair(uint64_t *bar, uint16_t pair_mask) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_addr(bar)),
        "h"(pair_mask)
        : "memory");
}

template <int NT, int MODE, bool PAIR, bool DRAIN>
__global__ void __launch_bounds__(LinearLayout<NT, MODE, PAIR>::kThreads, 1)
    linear_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw0,
                  const __grid_constant__ CUtensorMap tw1, const __grid_constant__ LinearArgs a) {
    using L = LinearLayout<NT, MODE, PAIR>;
    constexpr int CTAS = L::kCtas, BUFS = L::kBufs, MATS = L::kMats;
    constexpr int CH = L::template chunk<DRAIN>;  // columns handled at a time
    constexpr int EPI = L::kEpiWarps * 32;
    constexpr bool GATED = MODE != kLinear;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::kBarOff);  // PAIR: the even CTA's count
    uint64_t *empty = full + kMaxStages;
    uint64_t *accfull = empty + kMaxStages;
    uint64_t *accfree = accfull + 2;                                   // PAIR: the even CTA's count
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(accfree + 2);
    __shared__ int s_last;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cs = a.cs;                                        // parts of a tile's k across the cluster
    const int crank = PAIR || cs > 1 ? (int)blockIdx.x % (CTAS * cs) : 0;
    const int rank = PAIR ? crank & 1 : 0, split = crank / CTAS;
    const uint32_t lead = crank - rank;                         // the pair's even CTA in the cluster
    const int worker = blockIdx.x / (CTAS * cs), workers = gridDim.x / (CTAS * cs);
    const int nt = a.nt;          // tokens per tile: the MMA's N
    const int F = a.f_rows;       // features of this CTA's tile (per matrix)
    const int S = a.stages, KB = PAIR ? 1 : a.kb;
    const Pieces pieces(a, worker, workers, split);
    // A stage: W [matrix][k step][F rows][128 B] (interleaved: 64 gate rows, 64 up rows), then
    // X [k step][token rows][128 B].
    const uint32_t w_step = MODE == kInterleaved ? kLF * 128 : F * 128;  // bytes of one k step of an A operand
    const uint32_t x_step = (uint32_t)(nt / CTAS) * 128;
    const uint32_t x_off = MATS * KB * w_step, stage_bytes = x_off + KB * x_step;

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
    } else if (warp == L::kProducer && lane == 0) {
        tma_prefetch_desc(&tx);
        tma_prefetch_desc(&tw0);
        if constexpr (GATED) tma_prefetch_desc(&tw1);
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_sync_all();  // both CTAs' barriers and TMEM are there
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == L::kProducer) {
        if (lane == 0) {
            const uint32_t stage_tx =
                (GATED ? 2 : 1) * KB * (MODE == kInterleaved ? kLF / 2 : F) * 128u * CTAS + KB * x_step * CTAS;
            auto arm = [&](int s) {
                if (rank == 0) mbar_arrive_expect_tx(&full[s], stage_tx);  // both CTAs' bytes
            };
            auto bar_of = [&](int s) { return PAIR ? cluster_addr(&full[s], lead) : smem_addr(&full[s]); };
            // k step t.k covers KB steps of 64; a flat map has k along x, the other along z.
            auto load_w = [&](const Steps &t, int s) {
                uint8_t *st = smem + s * stage_bytes;
                const int f0 = (t.p.ftile * CTAS + rank) * F;
                const int x = a.flat ? t.k * kLK : 0, z = a.flat ? 0 : t.k * KB;
                tma_load_3d<PAIR>(st, &tw0, x, f0, z, bar_of(s));
                if constexpr (GATED)
                    tma_load_3d<PAIR>(st + (MODE == kInterleaved ? kLF / 2 * 128 : KB * w_step), &tw1, x, f0, z, bar_of(s));
            };
            auto load_x = [&](const Steps &t, int s) {
                const int m0 = t.p.mtile * nt + rank * (nt / CTAS);
                tma_load_3d<PAIR>(smem + s * stage_bytes + x_off, &tx, a.flat ? t.k * kLK : 0, m0, a.flat ? 0 : t.k * KB,
                                  bar_of(s));
            };
            Steps w(pieces);
            int j = 0;  // stages loaded
            bool more = true;
            if (a.early_w) {
                // The weights of the first ring do not depend on the kernel before, which, in the same
                // call, writes the activations: they are in flight before the wait for it.
                Steps x(pieces);
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
            } else {
                griddep_wait();
                while (j < S && (more = w.next())) {
                    arm(j);
                    load_w(w, j);
                    load_x(w, j);
                    ++j;
                }
            }
            uint32_t phase = 0;
            for (int s = 0; more && w.next(); ++j) {
                if (!mbar_wait(&empty[s], phase, a.err, kErrSlotTimeout)) break;
                arm(s);
                load_w(w, s);
                load_x(w, s);
                if (++s == S) s = 0, phase ^= 1;
            }
            // The next kernel may be scheduled (what ran before this one is complete: the wait above).
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
                    tc_commit_pair(bar, (uint16_t)(3u << lead));
                else
                    tc_commit(bar);
            };
            Pieces p = pieces;
            int s = 0;              // ring stage, with its phase
            uint32_t phase = 0;
            int seg = 0;            // accumulator sets used
            const int seg_steps = DRAIN ? a.drain_steps : 1 << 30;
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
                        uint32_t w = smem_addr(smem) + s * stage_bytes, x = w + x_off;
#pragma unroll 1
                        for (int b = 0; b < KB; ++b, w += w_step, x += x_step) {
#pragma unroll
                            for (int e = 0; e < kLK / 16; ++e)
#pragma unroll
                                for (int m = 0; m < MATS; ++m) {
                                    const uint64_t wd = sw128_desc(w + m * KB * w_step + e * 32, 16, 1024);
                                    const uint64_t xd = sw128_desc(x + e * 32, 16, 1024);
                                    const bool acc = kk > ks || b > 0 || e > 0;
                                    if constexpr (PAIR)
                                        tc_mma_pair(d + m * NT, wd, xd, idesc, acc);
                                    else
                                        tc_mma(d + m * NT, wd, xd, idesc, acc);
                                }
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
        // ---- epilogue warps: TMEM lane <-> feature, columns <-> tokens; two warps per lane quarter
        // (NT >= 64) take half of the columns each.  Interleaved: lanes 0-63 gate, 64-127 up.
        const int quarter = warp & 3;
        const int lrow = quarter * 32 + lane;
        const int r = MODE == kInterleaved ? lrow & 63 : lrow;  // feature of the CTA's tile
        const int col0 = (warp >> 2) * (L::kHalves == 1 ? 0 : a.half_cols);
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        const bool idle = MODE != kInterleaved && quarter * 32 >= F;  // a warp without features
        griddep_wait();  // the residual may come from, and the output may be read by, what ran before
        auto ld_cols = [&](uint32_t col, uint32_t (&v)[CH]) {
            if constexpr (CH == 32)
                tc_ld32_nowait(tmem + lane_base + col, v);
            else
                tc_ld16_nowait(tmem + lane_base + col, v);
        };
        auto st_cols = [&](uint32_t col, const uint32_t (&v)[CH]) {
            if constexpr (CH == 32)
                tc_st32(tmem + lane_base + col, v);
            else
                tc_st16(tmem + lane_base + col, v);
        };
        auto release = [&](int buf) {  // the accumulator may be overwritten
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR)
                    mbar_arrive_cluster(cluster_addr(&accfree[buf], lead));
                else
                    mbar_arrive(&accfree[buf]);
            }
        };
        // Interleaved: a gate warp and the up warp of the same features swap halves of a chunk, in
        // two buffers in turn, so that each finishes 8 of its 16 tokens.
        float *swap = reinterpret_cast<float *>(smem + kRing) + (size_t)((warp >> 2) * 2 + (quarter & 1)) * 2 * 512;
        int swaps = 0;
        Pieces p = pieces;
        int seg = 0;
        bool ok = true;
        bool first_piece = true;
        while (p.next()) {
            const int k0 = p.k0, k1 = p.k1;
            const bool at_lo = first_piece;  // a ranged piece that begins at the range's begin
            first_piece = false;
            const int feat = (p.ftile * CTAS + rank) * F + r;
            const int m0 = p.mtile * nt + col0;                    // token of this thread's first column
            const int ntok = idle ? 0 : min(min(a.half_cols, nt - col0), a.M - m0);  // columns that count (may be <= 0)
            const bool whole = cs > 1 || (k0 == 0 && k1 == a.nk);
            // A partial tile: [matrix][token / 4][128 lanes][4], in whole chunks (nt is a multiple of 16;
            // what a last chunk of 32 has past it is never used).
            const size_t slot_floats = (size_t)(MATS * nt + (CH == 32 ? 16 : 0)) * kLF;
            const bool in = r < F && feat < a.n;
            const float b0 = in && a.bias[0] ? a.bias[0][feat] : 0.f;
            const float b1 = GATED && in && a.bias[1] ? a.bias[1][feat] : 0.f;
            const size_t o0 = (size_t)m0 * a.n + feat;
            auto load_res = [&](int c0, float (&res)[CH]) {
                const float *src = a.residual + o0 + (size_t)c0 * a.n;
                if (in && c0 + CH <= ntok) {
#pragma unroll
                    for (int e = 0; e < CH; ++e, src += a.n) res[e] = *src;
                } else {
#pragma unroll
                    for (int e = 0; e < CH; ++e) res[e] = in && c0 + e < ntok ? src[(size_t)e * a.n] : 0.f;
                }
            };
            const bool has_res = !GATED && a.residual;
            float res[CH];
#pragma unroll
            for (int e = 0; e < CH; ++e) res[e] = 0.f;
            if (has_res) {
                // The residual on its way to L2 while the products run: a thread per 128-byte line of
                // the CTA's tile.
                const int f0 = (p.ftile * CTAS + rank) * F, fn = min(F, a.n - f0);
                const int lines = (fn * 4 + 127) / 128, t0 = p.mtile * nt, tn = min(nt, a.M - t0);
                for (int i = threadIdx.x; i < lines * tn; i += EPI) {
                    const float *src = a.residual + (size_t)(t0 + i / lines) * a.n + f0 + i % lines * 32;
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(src));
                }
            }
            if (!DRAIN && has_res && whole && cs == 1) load_res(0, res);
            float *part = a.ws + ((size_t)blockIdx.x * 2 + (at_lo ? 0 : 1)) * slot_floats + (size_t)col0 * kLF + lrow * 4;
            if constexpr (DRAIN) {
                // All accumulator sets of the piece but the last into registers; their sum goes back
                // into the last one's columns.
                if (k1 - k0 > a.drain_steps) {
                    float acc[L::kEpiCols];
#pragma unroll
                    for (int e = 0; e < L::kEpiCols; ++e) acc[e] = 0.f;
                    for (int ks = k0; ks < k1; ks += a.drain_steps) {
                        const int buf = seg % BUFS;
                        const bool last = ks + a.drain_steps >= k1;
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
            // A part of a tile: when all the others have arrived this one need not go through memory.
            const int t0 = (p.tile - a.tiles_whole) * a.nk;
            const int c_first = whole ? 0 : worker_of(a, t0), c_last = whole ? 0 : worker_of(a, t0 + a.nk - 1);
            int *counter = a.counters + (p.tile - a.tiles_whole) * CTAS + rank;
            bool joining = false;
            if (!whole) {
                if (threadIdx.x == 0) {
                    s_last = ld_acquire_gpu(counter) == c_last - c_first;
                    if (s_last) *counter = 0;  // ready for the next launch
                }
                named_barrier_sync(2, EPI);
                joining = s_last;
            }
            if (has_res && cs == 1 && (joining || (DRAIN && whole))) load_res(0, res);
#pragma unroll 1
            for (int c0 = 0; c0 < ntok; c0 += CH) {
                uint32_t vr[CH], wr[CH];
                ld_cols(buf * L::kCols + col0 + c0, vr);
                if constexpr (MATS == 2) ld_cols(buf * L::kCols + NT + col0 + c0, wr);
                tc_wait_ld();
                if (cs > 1) {
                    // This CTA's part [matrix][token / 4][128 lanes][4], in whole chunks, in the ring (its
                    // copies and the products that read them are complete).
                    float *dst = reinterpret_cast<float *>(smem) + (size_t)(col0 + c0) * kLF + lrow * 4;
#pragma unroll
                    for (int e = 0; e < CH; e += 4) {
                        *reinterpret_cast<uint4 *>(dst + e * kLF) = make_uint4(vr[e], vr[e + 1], vr[e + 2], vr[e + 3]);
                        if constexpr (MATS == 2)
                            *reinterpret_cast<uint4 *>(dst + (size_t)nt * kLF + e * kLF) =
                                make_uint4(wr[e], wr[e + 1], wr[e + 2], wr[e + 3]);
                    }
                } else if (whole || joining) {
                    float v[CH], w[CH];
                    if (joining) {
                        // The parts added in k order, this one from TMEM in its place.
                        float sum[MATS][CH];
#pragma unroll
                        for (int m = 0; m < MATS; ++m)
#pragma unroll
                            for (int e = 0; e < CH; ++e) sum[m][e] = 0.f;
#pragma unroll 1
                        for (int q = c_first; q <= c_last; ++q) {
                            if (q == worker) {
#pragma unroll
                                for (int e = 0; e < CH; ++e) {
                                    sum[0][e] += __uint_as_float(vr[e]);
                                    if constexpr (MATS == 2) sum[MATS - 1][e] += __uint_as_float(wr[e]);
                                }
                                continue;
                            }
                            const int slot = range_begin(a, q) >= t0 ? 0 : 1;
                            const float *src = a.ws + ((size_t)(q * CTAS + rank) * 2 + slot) * slot_floats +
                                               (size_t)(col0 + c0) * kLF + lrow * 4;
                            constexpr int XC = CH == 32 ? 16 : CH;  // at 32 the registers would spill
#pragma unroll
                            for (int h = 0; h < CH; h += XC) {
                                float4 x[MATS][XC / 4];
#pragma unroll
                                for (int m = 0; m < MATS; ++m)
#pragma unroll
                                    for (int e = 0; e < XC / 4; ++e)
                                        x[m][e] =
                                            __ldcg(reinterpret_cast<const float4 *>(src + (size_t)(m * nt + h + 4 * e) * kLF));
#pragma unroll
                                for (int m = 0; m < MATS; ++m)
#pragma unroll
                                    for (int e = 0; e < XC / 4; ++e) {
                                        float *to = &sum[m][h + 4 * e];
                                        to[0] += x[m][e].x, to[1] += x[m][e].y, to[2] += x[m][e].z, to[3] += x[m][e].w;
                                    }
                            }
                        }
#pragma unroll
                        for (int e = 0; e < CH; ++e) {
                            vr[e] = __float_as_uint(sum[0][e]);
                            if constexpr (MATS == 2) wr[e] = __float_as_uint(sum[MATS - 1][e]);
                        }
                    }
                    if constexpr (MODE == kInterleaved) {
                        const bool up = quarter >= 2;
                        float *buf_g = swap + (swaps & 1) * 512, *buf_u = buf_g + 256;
                        ++swaps;
                        // Gate warps give tokens 8-15 and take the up values of 0-7; up warps the reverse.
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            if (up)
                                buf_u[e * 32 + lane] = __uint_as_float(vr[e]);
                            else
                                buf_g[e * 32 + lane] = __uint_as_float(vr[8 + e]);
                        }
                        named_barrier_sync(3 + (warp >> 2) * 2 + (quarter & 1), 64);
                        float g8[8], u8[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            g8[e] = up ? buf_g[e * 32 + lane] : __uint_as_float(vr[e]);
                            u8[e] = up ? __uint_as_float(vr[8 + e]) : buf_u[e * 32 + lane];
                        }
                        const int c8 = c0 + (up ? 8 : 0);
                        if (in) finish<true, 8>(a, o0 + (size_t)c8 * a.n, ntok - c8, b0, b1, g8, u8);
                    } else {
#pragma unroll
                        for (int e = 0; e < CH; ++e) {
                            v[e] = __uint_as_float(vr[e]);
                            w[e] = MATS == 2 ? __uint_as_float(wr[e]) : res[e];
                        }
                        if (has_res && c0 + CH < ntok) load_res(c0 + CH, res);  // the next chunk's
                        if (in) finish<GATED, CH>(a, o0 + (size_t)c0 * a.n, ntok - c0, b0, b1, v, w);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < CH; e += 4) {
                        float *dst = part + (size_t)(c0 + e) * kLF;
                        __stcg(reinterpret_cast<uint4 *>(dst), make_uint4(vr[e], vr[e + 1], vr[e + 2], vr[e + 3]));
                        if constexpr (MATS == 2)
                            __stcg(reinterpret_cast<uint4 *>(dst + (size_t)nt * kLF),
                                   make_uint4(wr[e], wr[e + 1], wr[e + 2], wr[e + 3]));
                    }
                }
            }
            release(buf);
            if (joining) named_barrier_sync(2, EPI);  // s_last is read before the next piece writes it
            if (!whole && !joining) {
                // Others are still at it: the last of them to finish -- this one after all, maybe -- adds
                // the pieces in k order.
                named_barrier_sync(2, EPI);
                if (threadIdx.x == 0) {
                    __threadfence();  // the CTA's partial (ordered before by the barrier) before the count
                    const int prev = atomicAdd(counter, 1);
                    s_last = prev == c_last - c_first;
                    if (s_last) *counter = 0;
                    __threadfence();
                }
                named_barrier_sync(2, EPI);
                if (s_last) {
                    // Interleaved: the gate warps join the even chunks, the up warps the odd ones.
                    constexpr int STEP = MODE == kInterleaved ? 2 * CH : CH;
                    const int c_begin = MODE == kInterleaved && quarter >= 2 ? CH : 0;
#pragma unroll 1
                    for (int c0 = c_begin; c0 < ntok; c0 += STEP) {
                        float v[CH], w[CH];
                        if (has_res) {
                            load_res(c0, w);
                        } else {
#pragma unroll
                            for (int e = 0; e < CH; ++e) w[e] = 0.f;
                        }
#pragma unroll
                        for (int e = 0; e < CH; ++e) v[e] = 0.f;
                        // Two pieces' loads in flight at a time.
#pragma unroll 1
                        for (int q = c_first; q <= c_last; q += 2) {
                            float4 x[2][GATED ? 2 : 1][CH / 4];
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                if (q + h > c_last) break;
                                const int slot = range_begin(a, q + h) >= t0 ? 0 : 1;
                                const float *src = a.ws + ((size_t)((q + h) * CTAS + rank) * 2 + slot) * slot_floats +
                                                   (size_t)(col0 + c0) * kLF + r * 4;
                                const size_t other = MODE == kInterleaved ? 64 * 4 : (size_t)nt * kLF;
#pragma unroll
                                for (int e = 0; e < CH / 4; ++e) {
                                    x[h][0][e] = __ldcg(reinterpret_cast<const float4 *>(src + e * 4 * kLF));
                                    if constexpr (GATED)
                                        x[h][1][e] = __ldcg(reinterpret_cast<const float4 *>(src + other + e * 4 * kLF));
                                }
                            }
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                if (q + h > c_last) break;
#pragma unroll
                                for (int e = 0; e < CH / 4; ++e) {
                                    v[4 * e] += x[h][0][e].x, v[4 * e + 1] += x[h][0][e].y;
                                    v[4 * e + 2] += x[h][0][e].z, v[4 * e + 3] += x[h][0][e].w;
                                    if constexpr (GATED) {
                                        w[4 * e] += x[h][1][e].x, w[4 * e + 1] += x[h][1][e].y;
                                        w[4 * e + 2] += x[h][1][e].z, w[4 * e + 3] += x[h][1][e].w;
                                    }
                                }
                            }
                        }
                        if (in) finish<GATED, CH>(a, o0 + (size_t)c0 * a.n, ntok - c0, b0, b1, v, w);
                    }
                }
                named_barrier_sync(2, EPI);  // s_last is read before the next piece writes it
            }
        }
    }
    if (cs > 1) {
        __syncwarp();
        cluster_sync_all();  // every part is in its CTA's shared memory
        if (warp < L::kEpiWarps) {
            // Groups of four tokens dealt over the cluster's CTAs and their warps; the parts added in k
            // order.  Interleaved: the gate warps and the up warps take different groups.
            Pieces p = pieces;
            p.next();
            const int quarter = warp & 3, lrow = quarter * 32 + lane;
            const int r = MODE == kInterleaved ? lrow & 63 : lrow;
            const int feat = (p.ftile * CTAS + rank) * F + r, m0 = p.mtile * nt, ntok = min(nt, a.M - m0);
            constexpr int SHARES = L::kHalves * (MODE == kInterleaved ? 2 : 1);
            const int share = (warp >> 2) * (MODE == kInterleaved ? 2 : 1) + (MODE == kInterleaved ? quarter >> 1 : 0);
            const bool in = r < F && feat < a.n;
            const float b0 = in && a.bias[0] ? a.bias[0][feat] : 0.f;
            const float b1 = GATED && in && a.bias[1] ? a.bias[1][feat] : 0.f;
            const uint32_t other = MODE == kInterleaved ? 64 * 16 : (uint32_t)nt * kLF * 4;
#pragma unroll 1
            for (int g = split * SHARES + share; 4 * g < ntok && in; g += cs * SHARES) {
                const size_t o = (size_t)(m0 + 4 * g) * a.n + feat;
                float v[4] = {0.f, 0.f, 0.f, 0.f}, w[4] = {0.f, 0.f, 0.f, 0.f};
                if (!GATED && a.residual) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = 4 * g + e < ntok ? a.residual[o + (size_t)e * a.n] : 0.f;
                }
                const float *src = reinterpret_cast<const float *>(smem) + (size_t)g * 4 * kLF + r * 4;
                float4 x[8][GATED ? 2 : 1];
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (q < cs) {
                        const uint32_t at = cluster_addr(src, q * CTAS + rank);
                        x[q][0] = ld_cluster_f32x4(at);
                        if constexpr (GATED) x[q][1] = ld_cluster_f32x4(at + other);
                    }
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (q < cs) {
                        v[0] += x[q][0].x, v[1] += x[q][0].y, v[2] += x[q][0].z, v[3] += x[q][0].w;
                        if constexpr (GATED) w[0] += x[q][1].x, w[1] += x[q][1].y, w[2] += x[q][1].z, w[3] += x[q][1].w;
                    }
                finish<GATED, 4>(a, o, ntok - 4 * g, b0, b1, v, w);
            }
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR || cs > 1) cluster_sync_all();  // no CTA leaves while another's copies, commits or reads reach it
    tc_fence_after();
    if (warp == L::kMma) {
        if constexpr (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::kTmemCols) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::kTmemCols) : "memory");
    }
}

template <int NT, int MODE, bool PAIR, bool DRAIN>
cudaError_t launch_linear_k(const CUtensorMap &tx, const CUtensorMap *tw, const LinearArgs &a, int ctas, cudaStream_t s) {
    using L = LinearLayout<NT, MODE, PAIR>;
    static unsigned long long configured = 0;  // one bit per device: the opt-in is per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 64 || !(configured & (1ull << dev))) {
        cudaError_t e = cudaFuncSetAttribute(linear_kernel<NT, MODE, PAIR, DRAIN>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmemBytes);
        if (e != cudaSuccess) return e;
        if (dev < 64) configured |= 1ull << dev;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(L::kThreads);
    cfg.dynamicSmemBytes = L::kSmemBytes;
    cfg.stream = s;
    // A programmatic dependent of whatever ran before: the CTAs' set-up overlaps its tail, and every
    // access to memory (but the weights, when an earlier launch of the same call comes before) waits
    // for it.
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = L::kCtas * a.cs;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = L::kCtas * a.cs > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, linear_kernel<NT, MODE, PAIR, DRAIN>, tx, tw[0], tw[MODE == kLinear ? 0 : 1], a);
}

// Up to four tokens (linear_rows_max): no tile at all.  A warp takes WROWS weight rows (two neighbouring features, or
// the gate and the up row of one), each lane 16 bytes of a 512-byte chunk, with the loads of U chunks
// in flight; products and sums in f32 pairs, then a tree over the lanes.  The MMA form would read 128
// rows of shared memory for every 16 of k whatever it needs of them, and its ring, TMEM and barriers
// cost more than these products.
template <int R, int WROWS, bool GATED>
__global__ void __launch_bounds__(128) rows_kernel(const __grid_constant__ LinearArgs a) {
    constexpr int U = R == 1 ? 8 : 4;
    const int lane = threadIdx.x & 31;
    const int unit = blockIdx.x * 4 + (threadIdx.x >> 5);
    const int f = GATED ? unit : unit * WROWS;
    if (!a.early_w) griddep_wait();
    if (f >= a.n) {
        if (a.early_w) griddep_wait();
        griddep_launch_dependents();
        return;
    }
    const uint4 *w[WROWS];
#pragma unroll
    for (int i = 0; i < WROWS; ++i) {
        const int row = GATED ? f : min(f + i, a.n - 1);
        w[i] = reinterpret_cast<const uint4 *>(a.w[GATED ? i : 0] + (size_t)row * a.K) + lane;
    }
    const uint4 *x[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
        x[r] = reinterpret_cast<const uint4 *>(a.x + (size_t)min(r, a.M - 1) * a.K) + lane;
    const int chunks = (a.K + 255) / 256, k8 = a.K / 8 - lane;  // this lane's pieces: chunk * 32 < k8
    float2 acc[WROWS][R];
#pragma unroll
    for (int i = 0; i < WROWS; ++i)
#pragma unroll
        for (int r = 0; r < R; ++r) acc[i][r] = make_float2(0.f, 0.f);
    bool waited = !a.early_w;
    for (int c = 0; c < chunks; c += U) {
        uint4 wv[U][WROWS], xv[U][R];
        const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < WROWS; ++i) wv[u][i] = (c + u) * 32 < k8 ? __ldcs(w[i] + (c + u) * 32) : zero;
        if (!waited) {
            griddep_wait();
            waited = true;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < R; ++r) xv[u][r] = (c + u) * 32 < k8 ? x[r][(c + u) * 32] : zero;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float2 wf[WROWS][4];
#pragma unroll
            for (int i = 0; i < WROWS; ++i) {
                const __half2 *h = reinterpret_cast<const __half2 *>(&wv[u][i]);
#pragma unroll
                for (int e = 0; e < 4; ++e) wf[i][e] = __half22float2(h[e]);
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const __half2 *h = reinterpret_cast<const __half2 *>(&xv[u][r]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 xf = __half22float2(h[e]);
#pragma unroll
                    for (int i = 0; i < WROWS; ++i) acc[i][r] = ffma2(wf[i][e], xf, acc[i][r]);
                }
            }
        }
    }
    griddep_launch_dependents();
    // Lane r + R i ends up with the sum of (row i, token r).
    float mine = 0.f, other = 0.f;  // GATED: every lane r gets both rows of its token
#pragma unroll
    for (int i = 0; i < WROWS; ++i)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float v = acc[i][r].x + acc[i][r].y;
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
            if (GATED) {
                if (lane == r) (i ? other : mine) = v;
            } else if (lane == r + R * i) {
                mine = v;
            }
        }
    const int r = GATED ? lane : lane % R, feat = GATED ? f : f + lane / R;
    if (lane < (GATED ? R : R * WROWS) && r < a.M && feat < a.n) {
        const size_t o = (size_t)r * a.n + feat;
        const float v[1] = {mine};
        const float w1[1] = {GATED ? other : a.residual ? a.residual[o] : 0.f};
        finish<GATED, 1>(a, o, 1, a.bias[0] ? a.bias[0][feat] : 0.f, GATED && a.bias[1] ? a.bias[1][feat] : 0.f, v, w1);
    }
}

template <int R, int WROWS, bool GATED>
cudaError_t launch_rows_t(const LinearArgs &a, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    const int units = GATED ? a.n : (a.n + WROWS - 1) / WROWS;
    cfg.gridDim = dim3((units + 3) / 4);
    cfg.blockDim = dim3(128);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, rows_kernel<R, WROWS, GATED>, a);
}

template <int NT, bool PAIR>
cudaError_t launch_linear_t(int mats, const LinearPlan &p, const CUtensorMap &tx, const CUtensorMap *tw,
                            const LinearArgs &a, cudaStream_t s) {
    if (mats == 2) return launch_linear_k<NT, PAIR ? kInterleaved : kTwoAcc, PAIR, false>(tx, tw, a, p.ctas, s);
    return p.drain ? launch_linear_k<NT, kLinear, PAIR, true>(tx, tw, a, p.ctas, s)
                   : launch_linear_k<NT, kLinear, PAIR, false>(tx, tw, a, p.ctas, s);
}

}  // namespace

// How many clusters of `size` CTAs of these kernels (one CTA per SM) fit on the device at once.
static int max_clusters(int size, int sms) {
    static int cache[64][9] = {};  // per device and size; the GPU's partition into GPCs is fixed
    if (size <= 1) return sms;
    int dev = 0;
    cudaGetDevice(&dev);
    int n = dev < 64 ? cache[dev][size] : 0;
    if (n == 0) {
        using L = LinearLayout<16, kLinear, false>;
        cudaFuncSetAttribute(linear_kernel<16, kLinear, false, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             L::kSmemBytes);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(size * 64);
        cfg.blockDim = dim3(L::kThreads);
        cfg.dynamicSmemBytes = L::kSmemBytes;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = size;
        attr.val.clusterDim.y = 1;
        attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&n, linear_kernel<16, kLinear, false, false>, &cfg) != cudaSuccess) {
            cudaGetLastError();
            n = 0;
        }
        if (n <= 0) n = -1;
        if (dev < 64) cache[dev][size] = n;
    }
    return n > 0 ? n : 0;
}

LinearPlan linear_plan(int rows, int k, int n, int mats, bool drain, int sms) {
    return linear_plan_for(rows, k, n, mats, drain, sms, [sms](int size) { return max_clusters(size, sms); });
}

int linear_rows_max() { return 4; }

cudaError_t launch_linear_rows(int mats, const LinearArgs &a, cudaStream_t s) {
    if (mats == 2)
        return a.M == 1 ? launch_rows_t<1, 2, true>(a, s)
                        : a.M == 2 ? launch_rows_t<2, 2, true>(a, s) : launch_rows_t<4, 2, true>(a, s);
    return a.M == 1 ? launch_rows_t<1, 1, false>(a, s)
                    : a.M == 2 ? launch_rows_t<2, 2, false>(a, s) : launch_rows_t<4, 2, false>(a, s);
}

cudaError_t launch_linear(int mats, const LinearPlan &p, const CUtensorMap &tx, const CUtensorMap *tw,
                          const LinearArgs &a, cudaStream_t s) {
    if (p.pair)
        return p.nt_kernel == 128 ? launch_linear_t<128, true>(mats, p, tx, tw, a, s)
                                  : launch_linear_t<256, true>(mats, p, tx, tw, a, s);
    switch (p.nt_kernel) {
        case 16: return launch_linear_t<16, false>(mats, p, tx, tw, a, s);
        case 32: return launch_linear_t<32, false>(mats, p, tx, tw, a, s);
        case 64: return launch_linear_t<64, false>(mats, p, tx, tw, a, s);
        case 128: return launch_linear_t<128, false>(mats, p, tx, tw, a, s);
        default: return launch_linear_t<256, false>(mats, p, tx, tw, a, s);
    }
}

}  // namespace brk

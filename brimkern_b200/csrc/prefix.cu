// Attention of a whole batch over one shared prefix, on the 5th-generation tensor cores (tcgen05 +
// TMEM): the partials (m, l, o) of every sequence's query rows over the prefix's cache rows, which
// brk_attn_decode_prefix joins with each sequence's own rows (decode_kernel's H form).
//
// The query rows of one kv head -- (sequence, token, q head of the group), B * T * G of them -- are
// the MMA's M, so the prefix is read from HBM once for the batch and a decode step becomes a dense
// product: 4 D flops per (row, key) for 4 D bytes per key, which passes the ridge near 250 rows.
// A CTA takes one kv head, one block of rows and one split of the keys, in 64-key tiles:
//   S = Q K^T (M 128, N 64) in TMEM, each row's softmax by one thread (running maximum and sum in
//   f32), P as two fp16 terms (its rounding and what that leaves off) in TMEM, O += P V in TMEM.
// With one term the rounding of P, 2^-11 of each, is as large as an fp16 output's own (relative error
// against 64 bits 2.9e-4, with two 2.1e-4); the second costs MMAs and conversions: 8 sequences behind 131001
// rows 67 -> 75-78 us (eager), 16 x 2 tokens over int8 rows 32.8 -> 34.3, 64 behind 4096 34.3 -> 35.4, the
// window no time.
// Two streams of 128 rows run a tile apart so that one's exponentials overlap the other's products:
// with more rows than one stream holds the streams are two row tiles that share every K/V tile; with
// fewer they take alternate key tiles of the same rows.  head_dim 256 leaves TMEM for one stream.
// Few rows (COPIES 2 or 4): the MMA's 128 rows hold the same query rows 2 or 4 times, and each copy
// takes its own 32 or 16 keys of a tile and leaves P = 0 for the others, so that all threads share the
// exponentials instead of one warp doing them: what bounds the loop is then the K/V stream.
//
// The end: streams and copies are joined in shared memory and the split's partial leaves in coalesced
// rows; the own rows' kernel or prefix_merge_kernel joins the splits with the own rows.  (Joining the splits of a
// cluster through distributed shared memory first, for an eighth of the partials: 131 KB a CTA took
// 5 us there.)
//
// Whole calls, own rows and joins included, replayed from a graph (eager, caches cold): 8 sequences (32 /
// 8 heads of 64) behind 131001 rows 65 us (75-78), DRAM at 4.0 TB/s and the tensor pipe 42% active: bound by a
// tile's chain of scores, softmax and product, and 10 us of ramp and joins; 64 sequences (32 / 8 of 128) behind
// 4096 rows 34 us (35), this kernel alone 24.7 on 64 SMs, the own rows alone 19.6 on all; 32 (8 / 4 of 256) with
// a window of 4096 21 us (23), bound by the one stream's softmax between its products.
//
// int8 prefix: the codes, as exact fp16 integers, are the operands; the K scale multiplies the
// scores and the V scale the probabilities, so nothing is rounded that the fp16 form does not round.  The
// maximum that the probabilities are relative to counts the V scales in (v_scale_log2), so that their
// products stay in fp16's normal range whatever the size of V (without: 1% off at |V| 0.001).
#include <math_constants.h>

#include <algorithm>

#include "common.cuh"
#include "internal.h"
#include "tcgen05.cuh"

namespace brk {

namespace {

constexpr int kXQ = 128;                  // rows per stream (MMA M)
constexpr int kXK = 64;                   // keys per tile
constexpr uint32_t kXTmemCols = 512;
constexpr float kXLn2 = 0.6931471805599453f;

template <int D>
struct PrefixLayout {
    static constexpr int kStreams = D == 256 ? 1 : 2;
    static constexpr int kSoftWarps = 4 * kStreams;
    static constexpr int kProducer = kSoftWarps, kMma = kSoftWarps + 1;
    static constexpr int kThreads = (kSoftWarps + 1 + kStreams) * 32;
    static constexpr int kStages = D == 64 ? 6 : D == 128 ? 4 : 2;
    static constexpr int kBlocks = D / 64;
    static constexpr uint32_t kQBlock = kXQ * 128;
    static constexpr uint32_t kKVBlock = kXK * 128;
    static constexpr uint32_t kQBytes = kBlocks * kQBlock;
    static constexpr uint32_t kTileBytes = kBlocks * kKVBlock;
    static constexpr uint32_t kOffKV = kStreams * kQBytes;
    static constexpr uint32_t kOffScale = kOffKV + kStages * 2 * kTileBytes;  // int8: [stage][K, V][64] f32
    static constexpr uint32_t kOffState = kOffScale + kStages * 2 * kXK * 4;  // [m, l][stream][128] f32
    static constexpr uint32_t kOffBar = kOffState + 2 * kStreams * kXQ * 4;
    static constexpr uint32_t kSmemBytes = 1024 + kOffBar + 36 * 8 + 16;
    // TMEM columns: S, then P's two terms (fp16 pairs), then O from column 256.
    static constexpr uint32_t kColS = 0, kColP = kStreams * kXK, kColR = kColP + kStreams * kXK / 2, kColO = 256;
    static_assert(kColR + kStreams * kXK / 2 <= kColO && kColO + kStreams * D <= kXTmemCols, "TMEM columns");
    static_assert(kSmemBytes <= 232448, "more than 227 KB of shared memory per CTA");
    // The join: every stream's O [128][kJoin] f32 over q and the ring; the padding spreads the banks.
    static constexpr uint32_t kJoin = D + 4;
    static_assert(kStreams * kXQ * kJoin * 4 <= kOffScale, "join buffer");
};

enum : int {
    kXKFull = 0,     // [6] TMA (K) -> MMA
    kXVFull = 6,     // [6] TMA (V, int8: and the scales) -> MMA, softmax
    kXKEmpty = 12,   // [6] MMA commit (S done) -> producer
    kXVEmpty = 18,   // [6] MMA commit (PV done) -> producer
    kXSFull = 24,    // [2] MMA commit (S ready) -> softmax
    kXSFree = 26,    // [2] softmax (S read) -> MMA
    kXPFull = 28,    // [2] softmax (P written, O rescaled) -> MMA
    kXODone = 30,    // [2] MMA commit (PV done) -> softmax
    kXQFull = 32,    // TMA (q) -> MMA
    kXMmaDone = 33,  // [2] everything an issuer issued has completed -> teardown
    kXStagger = 35,  // stream 0's first P written -> stream 1's issuer starts
    kXBars = 36,
};

// 3-D tiled TMA load (CTA-local).
__device__ __forceinline__ void tma_load_q(void *dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
            "r"(smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
        : "memory");
}
// KC consecutive S columns of this thread's lane (no wait), and KC / 2 P columns.
template <int KC>
__device__ __forceinline__ void ld_scores(uint32_t taddr, uint32_t (&v)[KC]) {
    if constexpr (KC == 16) {
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
            "%15}, [%16];"
            : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
              "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
            : "r"(taddr));
    } else {
        uint32_t(&lo)[32] = reinterpret_cast<uint32_t(&)[32]>(v[0]);
        tc_ld32_nowait(taddr, lo);
        if constexpr (KC == 64) {
            uint32_t(&hi)[32] = reinterpret_cast<uint32_t(&)[32]>(v[32]);
            tc_ld32_nowait(taddr + 32, hi);
        }
    }
}
template <int N>
__device__ __forceinline__ void st_probs(uint32_t taddr, const uint32_t (&r)[N]) {
    if constexpr (N == 32) {
        tc_st32(taddr, r);
    } else if constexpr (N == 16) {
        asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
            "%14, %15, %16};" ::"r"(taddr),
            "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
            "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
            : "memory");
    } else {
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
                     "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                     : "memory");
    }
}

template <int D, int COPIES, bool Q8>
__global__ void __launch_bounds__(PrefixLayout<D>::kThreads, 1)
    prefix_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                  const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tms,
                  const __grid_constant__ PrefixArgs a) {
    using L = PrefixLayout<D>;
    constexpr int NS = L::kStreams;
    constexpr int RC = kXQ / COPIES;  // MMA rows of a copy
    constexpr int KC = kXK / COPIES;  // keys of a tile that a copy takes
    // Raise the running max (and rescale O) only when a tile's max exceeds it by more than this many powers
    // of two.  P is relative to 2^-6 of the maximum, and so stays below 2^14 (int8: times the row's V scale,
    // below 2^15, v_scale_log2): fp16's normal range then reaches further down.
    constexpr float kRaise = Q8 ? 2.f : 8.f;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kOffBar);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + kXBars);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.x, kvh = blockIdx.y;
    // Tokens (of any sequence) in the block: G query rows each, nbt to a stream's copy.
    const int nbt = RC / a.G, bt_total = a.B * a.T;
    const int bt0 = blockIdx.z * (NS == 2 && COPIES == 1 ? 2 : 1) * nbt;
    const int n_bt = min((NS == 2 && COPIES == 1 ? 2 : 1) * nbt, bt_total - bt0);
    const bool pair = NS == 2 && COPIES == 1 && n_bt > nbt;  // streams: two row tiles, or alternate key tiles
    const int kb = a.k_begin + split * a.tiles_per_split * kXK;
    const int ke = min(a.k_end, kb + a.tiles_per_split * kXK);
    const int nk = kb < ke ? (ke - kb + kXK - 1) / kXK : 0;
    const int seg_row = a.row0 + kvh * a.head_rows;
    // Stream s takes tiles first_s, first_s + step, ...: count_s of them.
    const int step = pair || NS == 1 ? 1 : 2;
    auto first_tile = [&](int s) { return step == 2 ? s : 0; };
    auto tile_count = [&](int s) { return step == 2 ? (nk - s + 1) / 2 : nk; };

    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; ++i) {
            mbar_init(&bars[kXKFull + i], 1);
            mbar_init(&bars[kXVFull + i], 1);
            mbar_init(&bars[kXKEmpty + i], pair ? 2 : 1);  // one commit per stream that reads the tile
            mbar_init(&bars[kXVEmpty + i], pair ? 2 : 1);
        }
        for (int s = 0; s < NS; ++s) {
            mbar_init(&bars[kXSFull + s], 1);
            mbar_init(&bars[kXSFree + s], 128);
            mbar_init(&bars[kXPFull + s], 128);
            mbar_init(&bars[kXODone + s], 1);
            mbar_init(&bars[kXMmaDone + s], 1);
        }
        mbar_init(&bars[kXQFull], 1);
        mbar_init(&bars[kXStagger], 128);
        fence_barrier_init();
    }
    if (warp == L::kMma) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                     "r"(kXTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else if (warp == L::kProducer && lane == 0) {
        tma_prefetch_desc(&tmk);
        tma_prefetch_desc(&tmv);
        tma_prefetch_desc(&tmq);
        if constexpr (Q8) tma_prefetch_desc(&tms);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    auto sQ = [&](int s) { return smem + (pair ? s : 0) * L::kQBytes; };
    auto sK = [&](int st) { return smem + L::kOffKV + st * 2 * L::kTileBytes; };
    auto sV = [&](int st) { return smem + L::kOffKV + st * 2 * L::kTileBytes + L::kTileBytes; };
    float *sScale = reinterpret_cast<float *>(smem + L::kOffScale);

    if (warp == L::kProducer) {
        if (lane == 0) {
            griddep_wait();  // q, the cache rows, or the staged codes may come from the kernel before
            // Everything before this grid is complete: the own rows' kernel may start streaming.
            griddep_launch_dependents();
            // q: boxes [nbt tokens][G heads][64] -- rows of 128 bytes in the MMA's K-major layout.  Rows
            // of a copy past nbt * G, and past the last token, hold anything: no output takes them.
            const int tiles = pair ? 2 : COPIES;
            mbar_arrive_expect_tx(&bars[kXQFull], (uint32_t)(tiles * L::kBlocks * nbt * a.G * 128));
            for (int t = 0; t < tiles; ++t)
#pragma unroll
                for (int blk = 0; blk < L::kBlocks; ++blk)
                    tma_load_q(smem + (pair ? t * L::kQBytes : t * RC * 128) + blk * L::kQBlock, &tmq, blk * 64, kvh * a.G,
                               bt0 + (pair ? t * nbt : 0), &bars[kXQFull]);
            // A K slot is free again after the tile's scores, a V slot after its product: K runs ahead.
            int issued = 0;
            bool ok = true;
            for (int j = 0; ok && j < nk; ++j) {
                const int st = j % L::kStages;
                const int key = kb + j * kXK, y = seg_row + key;
                const uint32_t phase = ((j / L::kStages) - 1) & 1;
                if (j >= L::kStages && !mbar_wait(&bars[kXKEmpty + st], phase, a.err, kErrSlotTimeout)) break;
                mbar_arrive_expect_tx(&bars[kXKFull + st], L::kTileBytes);
#pragma unroll
                for (int blk = 0; blk < L::kBlocks; ++blk)
                    tma_load_2d(sK(st) + blk * L::kKVBlock, &tmk, blk * 64, y, &bars[kXKFull + st]);
                if (j >= L::kStages && !mbar_wait(&bars[kXVEmpty + st], phase, a.err, kErrSlotTimeout)) ok = false;
                mbar_arrive_expect_tx(&bars[kXVFull + st], L::kTileBytes + (Q8 ? 2 * kXK * 4 : 0));
#pragma unroll
                for (int blk = 0; blk < L::kBlocks; ++blk)
                    tma_load_2d(sV(st) + blk * L::kKVBlock, &tmv, blk * 64, y, &bars[kXVFull + st]);
                if constexpr (Q8) tma_load_2d(sScale + st * 2 * kXK, &tms, key, a.scale_row + kvh * 2, &bars[kXVFull + st]);
                issued = j + 1;
            }
            mbar_wait(&bars[kXQFull], 0, a.err, kErrTmaTimeout);
            for (int j = issued > L::kStages ? issued - L::kStages : 0; j < issued; ++j) {
                mbar_wait(&bars[kXKFull + j % L::kStages], (j / L::kStages) & 1, a.err, kErrTmaTimeout);
                mbar_wait(&bars[kXVFull + j % L::kStages], (j / L::kStages) & 1, a.err, kErrTmaTimeout);
            }
        }
        __syncwarp();
    } else if (warp >= L::kMma) {
        const int s = warp - L::kMma;
        const int cnt = tile_count(s), j0 = first_tile(s);
        if (lane == 0 && cnt > 0) {
            constexpr uint32_t idesc_qk = f16_idesc(kXQ, kXK, 0, 0);
            constexpr uint32_t idesc_pv = f16_idesc(kXQ, D, 0, 1);
            // The V rows past the range end are zeroed in the last tile, by stream 0's softmax when
            // both streams read that tile; stream 1's product of it then waits for that too.
            const bool tail = kb + nk * kXK > ke;
            bool ok = mbar_wait(&bars[kXQFull], 0, a.err, kErrMmaTimeout);
            auto issue_s = [&](int i) -> bool {
                const int j = j0 + i * step, st = j % L::kStages;
                if (!mbar_wait(&bars[kXKFull + st], (j / L::kStages) & 1, a.err, kErrTmaTimeout)) return false;
                if (i >= 1 && !mbar_wait(&bars[kXSFree + s], (i - 1) & 1, a.err, kErrMmaTimeout)) return false;
                tc_fence_after();
                const uint32_t q_base = smem_addr(sQ(s)), k_base = smem_addr(sK(st));
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                    tc_mma(tmem + L::kColS + s * kXK,
                           sw128_desc(q_base + (ks >> 2) * L::kQBlock + (ks & 3) * 32, 16, 1024),
                           sw128_desc(k_base + (ks >> 2) * L::kKVBlock + (ks & 3) * 32, 16, 1024), idesc_qk, ks > 0);
                tc_commit(&bars[kXSFull + s]);
                tc_commit(&bars[kXKEmpty + st]);
                return true;
            };
            auto issue_pv = [&](int i) -> bool {
                const int j = j0 + i * step, st = j % L::kStages;
                if (!mbar_wait(&bars[kXPFull + s], i & 1, a.err, kErrMmaTimeout)) return false;
                if (!mbar_wait(&bars[kXVFull + st], (j / L::kStages) & 1, a.err, kErrTmaTimeout)) return false;
                if (pair && s == 1 && tail && j == nk - 1 && !mbar_wait(&bars[kXPFull], i & 1, a.err, kErrMmaTimeout))
                    return false;
                tc_fence_after();
                const uint32_t v_base = smem_addr(sV(st));
#pragma unroll
                for (int kk = 0; kk < kXK / 16; ++kk) {
                    const uint64_t vd = sw128_desc(v_base + kk * 16 * 128, L::kKVBlock, 1024);
                    tc_mma_ts(tmem + L::kColO + s * D, tmem + L::kColP + s * (kXK / 2) + kk * 8, vd, idesc_pv, i > 0 || kk > 0);
                    tc_mma_ts(tmem + L::kColO + s * D, tmem + L::kColR + s * (kXK / 2) + kk * 8, vd, idesc_pv, true);
                }
                tc_commit(&bars[kXODone + s]);
                tc_commit(&bars[kXVEmpty + st]);
                return true;
            };
            if (ok && s == 1) ok = mbar_wait(&bars[kXStagger], 0, a.err, kErrMmaTimeout);
            if (ok) ok = issue_s(0);
            for (int i = 0; ok && i < cnt; ++i) {
                // S of the next tile needs only that this one's was read: it runs under the softmax.
                if (i + 1 < cnt && !issue_s(i + 1)) break;
                if (!issue_pv(i)) break;
            }
            tc_commit(&bars[kXMmaDone + s]);
            mbar_wait(&bars[kXMmaDone + s], 0, a.err, kErrMmaTimeout);
        }
        __syncwarp();
    } else {
        // ---- softmax warps: stream s = warp / 4, thread r <-> MMA row r of the stream (TMEM lane r).
        const int s = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const int copy = r / RC, rc = r % RC;      // the copy is the same for the whole warp
        const int bt_of = rc / a.G;                // token within the stream's tile
        const int bt = bt0 + (pair ? s * nbt : 0) + bt_of;
        const bool row_ok = bt_of < nbt && bt < bt_total;
        const int cnt = tile_count(s), j0 = first_tile(s);
        const int lo = a.window > 0 && row_ok ? a.past_len[bt / a.T] + bt % a.T - a.window + 1 : INT_MIN;
        // The first key that a row of this warp attends: what lies before it may hold anything.
        const int warp_lo = __reduce_min_sync(0xffffffffu, row_ok ? lo : INT_MAX);
        const uint32_t tS = tmem + L::kColS + s * kXK + lane_base + copy * KC;
        const uint32_t tO = tmem + L::kColO + s * D + lane_base;
        const uint32_t tP = tmem + L::kColP + s * (kXK / 2) + lane_base;
        const uint32_t tR = tmem + L::kColR + s * (kXK / 2) + lane_base;
        // A warp without rows only keeps the barriers going.
        const bool idle = !__any_sync(0xffffffffu, row_ok);
        if (COPIES > 1 || idle) {
            // The keys of the other copies: P = 0 for good.
            uint32_t zero[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) zero[e] = 0u;
            tc_st32(tP, zero);
            tc_st32(tR, zero);
            tc_wait_st();
        }
        float m_used = -CUDART_INF_F;  // the maximum that the probabilities are relative to (log2 units)
        float l_run = 0.f;
        bool ok = true;
        const bool cap = a.softcap > 0.f;
        for (int i = 0; i < cnt; ++i) {
            const int j = j0 + i * step, st = j % L::kStages;
            const int kbase = kb + j * kXK + copy * KC;  // this thread's first key
            const bool tail = kb + (j + 1) * kXK > ke;
            if (!__all_sync(0xffffffffu, mbar_wait(&bars[kXSFull + s], i & 1, a.err, kErrMmaTimeout))) {
                ok = false;
                break;
            }
            tc_fence_after();
            bool waited = false;
            uint32_t pk[KC / 2], rk[KC / 2];  // P's terms: its fp16 rounding, and what that left off
            float rsum = 0.f;
            if (idle) {
                mbar_arrive(&bars[kXSFree + s]);
            } else {
                float v[KC];
                {
                    uint32_t raw[KC];
                    ld_scores<KC>(tS, raw);
                    tc_wait_ld();
                    tc_fence_before();
                    mbar_arrive(&bars[kXSFree + s]);
#pragma unroll
                    for (int e = 0; e < KC; ++e) v[e] = __uint_as_float(raw[e]);
                }
                const float *ksc = sScale + st * 2 * kXK + copy * KC, *vsc = ksc + kXK;
                if constexpr (Q8) {
                    const bool there = mbar_wait(&bars[kXVFull + st], (j / L::kStages) & 1, a.err, kErrTmaTimeout);
                    if (!__all_sync(0xffffffffu, there)) {
                        ok = false;
                        break;
                    }
#pragma unroll
                    for (int e = 0; e < KC; e += 4) {
                        const float4 k4 = *reinterpret_cast<const float4 *>(ksc + e);
                        v[e] *= k4.x, v[e + 1] *= k4.y, v[e + 2] *= k4.z, v[e + 3] *= k4.w;
                    }
                }
                const bool edge = __any_sync(0xffffffffu, tail || kbase < lo);
                if (edge) {
#pragma unroll
                    for (int e = 0; e < KC; ++e) v[e] = kbase + e >= lo && kbase + e < ke ? v[e] : -CUDART_INF_F;
                }
                const float mraw = max_tree(v);
                float mt = mraw == -CUDART_INF_F ? -CUDART_INF_F
                           : cap                 ? softcap_log2(mraw, a.cap_k1, a.cap_k2)
                                                 : mraw * a.scale_log2;
                if constexpr (Q8) {
                    // At least the maximum of probability times V scale, which is what is rounded to fp16:
                    // with the largest scale of the keys in range (positive floats compare as their bits).
                    unsigned top = 0u;
#pragma unroll
                    for (int e = 0; e < KC; e += 32) {
                        const int x = KC < 32 ? lane % KC : e + lane;
                        if (kbase + x >= warp_lo && kbase + x < ke) top = max(top, __float_as_uint(vsc[x]));
                    }
                    mt += v_scale_log2(__uint_as_float(__reduce_max_sync(0xffffffffu, top)));
                } else {
                    mt -= 6.f;
                }
                // Rows raise their maximum separately; the rescale pass is warp-collective.
                const bool raise = mt > m_used + kRaise || (m_used == -CUDART_INF_F && mt != -CUDART_INF_F);
                const bool rescale = raise && m_used != -CUDART_INF_F && i >= 1;
                if (__any_sync(0xffffffffu, rescale)) {
                    const bool got = mbar_wait(&bars[kXODone + s], (i - 1) & 1, a.err, kErrMmaTimeout);
                    if (!__all_sync(0xffffffffu, got)) {
                        ok = false;
                        break;
                    }
                    waited = true;
                    tc_fence_after();
                    const float alpha = rescale ? ex2_fast(m_used - mt) : 1.f;
#pragma unroll 1
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t o[32];
                        tc_ld32_nowait(tO + c * 32, o);
                        tc_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        tc_st32(tO + c * 32, o);
                    }
                    tc_wait_st();
                    l_run *= alpha;
                }
                if (raise) m_used = mt;
                const float m_eff = m_used == -CUDART_INF_F ? 0.f : m_used;
                if (cap) {
#pragma unroll
                    for (int e = 0; e < KC; ++e) {
                        const float p = ex2_fast(softcap_log2(v[e], a.cap_k1, a.cap_k2) - m_eff);
                        v[e] = v[e] == -CUDART_INF_F ? 0.f : p;
                    }
                } else {
                    const float2 sc2 = make_float2(a.scale_log2, a.scale_log2), nm2 = make_float2(-m_eff, -m_eff);
#pragma unroll
                    for (int u = 0; u < KC / 2; ++u) {
                        const float2 x = ffma2(make_float2(v[2 * u], v[2 * u + 1]), sc2, nm2);
                        v[2 * u] = ex2_fast(x.x);
                        v[2 * u + 1] = ex2_fast(x.y);
                    }
                }
                float2 acc[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[k] = make_float2(0.f, 0.f);
#pragma unroll
                for (int u = 0; u < KC / 2; ++u) acc[u & 3] = fadd2(acc[u & 3], make_float2(v[2 * u], v[2 * u + 1]));
                const float2 acc01 = fadd2(acc[0], acc[1]), acc23 = fadd2(acc[2], acc[3]);
                rsum = (acc01.x + acc01.y) + (acc23.x + acc23.y);
                if constexpr (Q8) {
                    // The V scale goes into the probability; a masked key's (P 0) is not taken, as it
                    // may be anything.
#pragma unroll
                    for (int e = 0; e < KC; e += 4) {
                        const float4 s4 = *reinterpret_cast<const float4 *>(vsc + e);
                        v[e] *= s4.x, v[e + 1] *= s4.y, v[e + 2] *= s4.z, v[e + 3] *= s4.w;
                    }
                    if (edge) {
#pragma unroll
                        for (int e = 0; e < KC; ++e) v[e] = kbase + e >= lo && kbase + e < ke ? v[e] : 0.f;
                    }
                }
#pragma unroll
                for (int u = 0; u < KC / 2; ++u) {
                    pk[u] = pack_half2(v[2 * u], v[2 * u + 1]);
                    rk[u] = half2_rest(v[2 * u], v[2 * u + 1], pk[u]);
                }
            }
            if (i >= 1 && !waited) {
                const bool got = mbar_wait(&bars[kXODone + s], (i - 1) & 1, a.err, kErrMmaTimeout);
                if (!__all_sync(0xffffffffu, got)) {
                    ok = false;
                    break;
                }
            }
            if (!idle) {
                st_probs<KC / 2>(tP + copy * (KC / 2), pk);
                st_probs<KC / 2>(tR + copy * (KC / 2), rk);
            }
            // Keys past the range end: zero V rows, so that 0 * (whatever the tile holds) stays 0.
            if ((s == 0 || !pair) && tail) {
                const int key = kb + j * kXK + r;
                if (!__all_sync(0xffffffffu, mbar_wait(&bars[kXVFull + st], (j / L::kStages) & 1, a.err, kErrTmaTimeout))) {
                    ok = false;
                    break;
                }
                if (r < kXK && key >= ke) {
#pragma unroll
                    for (int blk = 0; blk < L::kBlocks; ++blk)
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            *reinterpret_cast<uint4 *>(sV(st) + blk * L::kKVBlock + sw128(r, c)) = make_uint4(0u, 0u, 0u, 0u);
                }
                __syncwarp();
                fence_proxy_async_smem();
            }
            tc_wait_st();
            // The scales of this stage were read with ordinary loads; the stage's next copies are
            // asynchronous and ordered behind this fence through the product's commit.
            if constexpr (Q8) fence_proxy_async_smem();
            tc_fence_before();
            mbar_arrive(&bars[kXPFull + s]);
            if (s == 0 && i == 0) mbar_arrive(&bars[kXStagger]);
            l_run += rsum;
        }
        // Every product of this stream has landed.
        if (ok && cnt > 0) ok = __all_sync(0xffffffffu, mbar_wait(&bars[kXODone + s], (cnt - 1) & 1, a.err, kErrMmaTimeout));
        tc_fence_after();
        // ---- join.  Every stream's (m, l, O) to shared memory, over q and the ring: all products that
        // read them are complete behind the barrier.
        constexpr int NT = L::kSoftWarps * 32;
        float *jo = reinterpret_cast<float *>(smem);                 // [stream][128][kJoin]
        float *jm = reinterpret_cast<float *>(smem + L::kOffState);  // [stream][128] m, then l
        float *jl = jm + NS * kXQ;
        named_barrier_sync(1, NT);
        jm[s * kXQ + r] = m_used;
        jl[s * kXQ + r] = l_run;
        if (!idle && cnt > 0) {
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                tc_ld32_nowait(tO + c * 32, o);
                tc_wait_ld();
                uint4 *dst = reinterpret_cast<uint4 *>(jo + (size_t)(s * kXQ + r) * L::kJoin + c * 32);
#pragma unroll
                for (int e = 0; e < 8; ++e) dst[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            }
        }
        named_barrier_sync(1, NT);
        // Rows by (half-)warps, lanes over the row's float4s, UR rows at a time.  The sources of a row:
        // the copies of every stream that took tiles, or (pair) its own stream.
        constexpr int D4 = D / 4, LPR = D4 < 32 ? D4 : 32, RPW = 32 / LPR, VPL = D4 / LPR;
        constexpr int UR = COPIES == 1 ? 4 : COPIES == 2 ? 2 : 1, MOST = NS * COPIES;
        const int n_rows = n_bt * a.G, rt = nbt * a.G;
        const int sub = lane / LPR, l4 = lane % LPR;
        const size_t rows_total = (size_t)bt_total * a.Hq;
        float *out_o = a.part_o + (size_t)split * rows_total * D, *out_ml = a.part_ml + (size_t)split * rows_total * 2;
        for (int x0 = (warp * RPW + sub) * UR; x0 < n_rows; x0 += L::kSoftWarps * RPW * UR) {
#pragma unroll
            for (int u = 0; u < UR; ++u) {
                const int x = min(x0 + u, n_rows - 1);
                // The row's first MMA row in shared memory, and how many sources it has.
                const int at = pair && x >= rt ? kXQ + x - rt : x;
                float m[MOST], M = -CUDART_INF_F, l = 0.f;
#pragma unroll
                for (int q = 0; q < MOST; ++q) {
                    const bool there = pair ? q == 0 : tile_count(q / COPIES) > 0;
                    m[q] = there ? jm[at + (q / COPIES) * kXQ + (q % COPIES) * RC] : -CUDART_INF_F;
                    M = fmaxf(M, m[q]);
                }
                float4 O[VPL];
#pragma unroll
                for (int v = 0; v < VPL; ++v) O[v] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int q = 0; q < MOST; ++q)
                    if (m[q] != -CUDART_INF_F) {
                        const int src = at + (q / COPIES) * kXQ + (q % COPIES) * RC;
                        const float f = ex2_fast(m[q] - M);
                        l = fmaf(f, jl[src], l);
#pragma unroll
                        for (int v = 0; v < VPL; ++v) {
                            const float4 y = *reinterpret_cast<const float4 *>(jo + (size_t)src * L::kJoin + 4 * (l4 + v * LPR));
                            O[v].x = fmaf(f, y.x, O[v].x), O[v].y = fmaf(f, y.y, O[v].y);
                            O[v].z = fmaf(f, y.z, O[v].z), O[v].w = fmaf(f, y.w, O[v].w);
                        }
                    }
                if (x0 + u < n_rows) {
                    const int xt = x * a.g_magic >> 16;  // x / G
                    const size_t R = (size_t)(bt0 + xt) * a.Hq + kvh * a.G + (x - xt * a.G);
#pragma unroll
                    for (int v = 0; v < VPL; ++v)
                        *reinterpret_cast<float4 *>(out_o + R * D + 4 * (l4 + v * LPR)) = O[v];
                    if (l4 == 0)
                        *reinterpret_cast<float2 *>(out_ml + R * 2) = make_float2(M == -CUDART_INF_F ? M : M * kXLn2, l);
                }
            }
        }
    }
    // Teardown: every TMEM access and MMA is complete; the allocating warp releases TMEM.
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == L::kMma)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kXTmemCols) : "memory");
}

template <int D, int COPIES, bool Q8>
cudaError_t launch_prefix_t(const CUtensorMap &tmk, const CUtensorMap &tmv, const CUtensorMap &tmq, const CUtensorMap &tms,
                            const PrefixArgs &a, int splits, int blocks, cudaStream_t s, bool pdl) {
    using L = PrefixLayout<D>;
    static unsigned long long configured = 0;  // one bit per device: the opt-in is per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 64 || !(configured & (1ull << dev))) {
        cudaError_t e = cudaFuncSetAttribute(prefix_kernel<D, COPIES, Q8>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             L::kSmemBytes);
        if (e != cudaSuccess) return e;
        if (dev < 64) configured |= 1ull << dev;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(splits, a.Hkv, blocks);
    cfg.blockDim = dim3(L::kThreads);
    cfg.dynamicSmemBytes = L::kSmemBytes;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, prefix_kernel<D, COPIES, Q8>, tmk, tmv, tmq, tms, a);
}

template <int D>
cudaError_t launch_prefix_d(const CUtensorMap &tmk, const CUtensorMap &tmv, const CUtensorMap &tmq, const CUtensorMap &tms,
                            const PrefixArgs &a, const PrefixPlan &p, cudaStream_t s, bool pdl) {
    const bool q8 = a.scale_row >= 0;
    switch (p.copies) {
        case 1:
            return q8 ? launch_prefix_t<D, 1, true>(tmk, tmv, tmq, tms, a, p.splits, p.blocks, s, pdl)
                      : launch_prefix_t<D, 1, false>(tmk, tmv, tmq, tms, a, p.splits, p.blocks, s, pdl);
        case 2:
            return q8 ? launch_prefix_t<D, 2, true>(tmk, tmv, tmq, tms, a, p.splits, p.blocks, s, pdl)
                      : launch_prefix_t<D, 2, false>(tmk, tmv, tmq, tms, a, p.splits, p.blocks, s, pdl);
        default:
            return q8 ? launch_prefix_t<D, 4, true>(tmk, tmv, tmq, tms, a, p.splits, p.blocks, s, pdl)
                      : launch_prefix_t<D, 4, false>(tmk, tmv, tmq, tms, a, p.splits, p.blocks, s, pdl);
    }
}

static_assert(kPrefixMostParts == 64, "the merge's two weights per lane");

// A warp per row: the partials' weights by lanes, then the row's float4s by lanes with eight partials'
// loads in flight.  M = max m, o = sum e^{m - M} o / sum e^{m - M} l.
__global__ void __launch_bounds__(128) prefix_merge_kernel(const __grid_constant__ PrefixMergeArgs a) {
    griddep_wait();
    const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= a.rows) return;
    const size_t R = row, n = a.rows;
    const int n0 = a.parts[0], parts = n0 + a.parts[1];
    constexpr int NU = kPrefixMostParts / 32;
    float2 ml[NU];
    float M = -CUDART_INF_F;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        const int p = lane + 32 * u;
        ml[u] = make_float2(-CUDART_INF_F, 0.f);
        if (p < parts)
            ml[u] = *reinterpret_cast<const float2 *>(p < n0 ? a.ml[0] + ((size_t)p * n + R) * 2
                                                             : a.ml[1] + ((size_t)(p - n0) * n + R) * 2);
        M = fmaxf(M, ml[u].x);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
    float w[NU], l = 0.f;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        w[u] = ml[u].x == -CUDART_INF_F ? 0.f : expf(ml[u].x - M);
        l = fmaf(w[u], ml[u].y, l);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    const float inv = 1.f / l;
    for (int d0 = 0; d0 < a.D / 4; d0 += 32) {
        const int d4 = d0 + lane;
        const bool in = d4 < a.D / 4;  // (head_dim 64: half of the warp has none, but has weights)
        float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int p0 = 0; p0 < parts; p0 += 8) {
            float4 v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int p = p0 + u;
                const float *src = p < n0 ? a.o[0] + ((size_t)p * n + R) * a.D : a.o[1] + ((size_t)(p - n0) * n + R) * a.D;
                v[u] = in && p < parts ? __ldcs(reinterpret_cast<const float4 *>(src) + d4) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                // Partials that hold nothing (weight 0) are not multiplied: an idle split's row may be anything.
                const int p = p0 + u;
                const float f = __shfl_sync(0xffffffffu, p < 32 ? w[0] : w[1], p & 31);
                if (p < parts && f != 0.f)
                    O.x = fmaf(f, v[u].x, O.x), O.y = fmaf(f, v[u].y, O.y), O.z = fmaf(f, v[u].z, O.z),
                    O.w = fmaf(f, v[u].w, O.w);
            }
        }
        O.x *= inv, O.y *= inv, O.z *= inv, O.w *= inv;
        if (!in) continue;
        if (a.out16)
            reinterpret_cast<uint2 *>(a.out16 + R * a.D)[d4] = make_uint2(pack_half2(O.x, O.y), pack_half2(O.z, O.w));
        else
            reinterpret_cast<float4 *>(a.out + R * a.D)[d4] = O;
    }
}

// fp16 rows from f32 ones (q), eight elements per thread.
__global__ void half_rows_kernel(const float *src, __half *dst, long long n8) {
    griddep_wait();
    griddep_launch_dependents();
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n8) return;
    const float4 x = reinterpret_cast<const float4 *>(src)[2 * i], y = reinterpret_cast<const float4 *>(src)[2 * i + 1];
    reinterpret_cast<uint4 *>(dst)[i] =
        make_uint4(pack_half2(x.x, x.y), pack_half2(x.z, x.w), pack_half2(y.x, y.y), pack_half2(y.z, y.w));
}

// Codes (biased by +128) of rows [row0, row0 + rows) of every kv head as exact fp16 integers
// [Hkv][rows][D], 16 codes per thread and matrix.
__global__ void codes_to_half_kernel(const uint8_t *kc, const uint8_t *vc, __half *k, __half *v, int Hkv, int D, int cap,
                                     int row0, int rows) {
    griddep_wait();  // the codes may come from the kernel before
    griddep_launch_dependents();
    const int cs = D / 16;
    const long long n = (long long)Hkv * rows * cs;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        const int c = (int)(i % cs);
        const long long hr = i / cs;
        const int r = (int)(hr % rows), h = (int)(hr / rows);
        const size_t src = ((size_t)h * cap + row0 + r) * D + 16 * c, dst = (size_t)hr * D + 16 * c;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const uint4 w = *reinterpret_cast<const uint4 *>((which ? vc : kc) + src);
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
            uint32_t o[8];
            const __half2 bias = __floats2half2_rn(kCodeBias, kCodeBias);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t u = codes_biased_half2(ws[e >> 1], e & 1 ? 0x4342u : 0x4140u);
                const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&u), bias);  // exact
                o[e] = *reinterpret_cast<const uint32_t *>(&x);
            }
            uint4 *d = reinterpret_cast<uint4 *>((which ? v : k) + dst);
            d[0] = make_uint4(o[0], o[1], o[2], o[3]);
            d[1] = make_uint4(o[4], o[5], o[6], o[7]);
        }
    }
}

}  // namespace

int prefix_tile_keys() { return kXK; }

// Rows: as many copies of them as fit the MMA's 128 rows, or blocks of two row tiles.  Splits of the
// key tiles over one CTA per SM: a split's fixed cost (ramp, join) is worth about six tiles, and every
// partial costs the merge a quarter of one.  The own rows' kernel runs beside this one on the SMs that
// it leaves (an SM has room for one or the other), so the SMs are shared out by the work of both, at
// most half of them to the own rows: 64 sequences of 256 own rows behind 4096 take 39.6 us with 16
// splits for 8 kv heads (one after the other), 30.5 with 8, 45.6 with 3.
PrefixPlan prefix_plan(int head_dim, int tokens, int group, int kv_heads, int ntiles, double own_tiles, int sms) {
    PrefixPlan p;
    const int streams = head_dim == 256 ? 1 : 2;
    p.copies = tokens * group <= (kXQ / 4 / group) * group ? 4 : tokens * group <= (kXQ / 2 / group) * group ? 2 : 1;
    p.tokens_box = kXQ / p.copies / group;
    const int per_block = p.tokens_box * (p.copies == 1 ? streams : 1);
    p.blocks = (tokens + per_block - 1) / per_block;
    const long long units = (long long)kv_heads * p.blocks;
    // Thousands of cycles of an SM: a tile here, a tile of own rows there (half: two of its CTAs run).
    const double tile = streams == 1 || (p.copies == 1 && tokens > p.tokens_box) ? 2.0 : p.copies == 1 ? 1.0 : 0.75;
    const double mine = (double)units * ntiles * tile, theirs = 0.5 * own_tiles;
    const int share = std::max(1, (int)(sms * (1.0 - std::min(0.5, theirs / (mine + theirs)))));
    double best = 1e300;
    // No split longer than 256 tiles, while 32 splits do: a sum in the tensor cores loses up to 2^-24 of itself
    // with each product of 16 keys and term of P (16384 keys, V of one sign: 1.2e-4 at most; 131072 keys in one
    // split, twice an fp16 output's half step).
    for (int n = std::min(32, (ntiles + 255) / 256); n <= 32 && (n == 1 || 2 * n <= ntiles); ++n) {
        const int tps = (ntiles + n - 1) / n;
        if ((ntiles + tps - 1) / tps != n) continue;  // no empty split
        const double cost = (double)((units * n + share - 1) / share) * (tps + 6) + 0.25 * n;
        if (cost < best - 1e-9) {
            best = cost;
            p.splits = n, p.tiles_per_split = tps;
        }
    }
    return p;
}

cudaError_t launch_prefix(int head_dim, const CUtensorMap &tmk, const CUtensorMap &tmv, const CUtensorMap &tmq,
                          const CUtensorMap &tms, const PrefixArgs &a, const PrefixPlan &p, cudaStream_t s, bool pdl) {
    switch (head_dim) {
        case 64: return launch_prefix_d<64>(tmk, tmv, tmq, tms, a, p, s, pdl);
        case 128: return launch_prefix_d<128>(tmk, tmv, tmq, tms, a, p, s, pdl);
        case 256: return launch_prefix_d<256>(tmk, tmv, tmq, tms, a, p, s, pdl);
        default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_prefix_merge(const PrefixMergeArgs &a, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((a.rows + 3) / 4));
    cfg.blockDim = dim3(128);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, prefix_merge_kernel, a);
}

cudaError_t launch_half_rows(const float *src, __half *dst, size_t n, cudaStream_t s, bool pdl) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((n / 8 + 127) / 128));
    cfg.blockDim = dim3(128);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, half_rows_kernel, src, dst, (long long)(n / 8));
}

cudaError_t launch_codes_to_half(const uint8_t *kc, const uint8_t *vc, __half *k, __half *v, int n_kv_heads,
                                 int head_dim, int cap, int row0, int rows, cudaStream_t s, bool pdl) {
    const long long n = (long long)n_kv_heads * rows * (head_dim / 16);
    if (n == 0) return cudaSuccess;
    const long long g = (n + 255) / 256;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(g < 8192 ? g : 8192));
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, codes_to_half_kernel, kc, vc, k, v, n_kv_heads, head_dim, cap, row0, rows);
}

}  // namespace brk

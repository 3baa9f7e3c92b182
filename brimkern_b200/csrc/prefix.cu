// Attention of a whole batch over one shared prefix, on the 5th-generation tensor cores (tcgen05 +
// TMEM): the partials (m, l, o) of every sequence's query rows over the prefix's cache rows, which
// brk_attn_decode_prefix joins with each sequence's own rows (decode_kernel's H form).
//
// The query rows of one kv head -- (sequence, token, q head of the group), B * T * G of them -- are
// the MMA's M, so the prefix is read from HBM once for the batch and a decode step becomes a dense
// product: 4 D flops per (row, key) for 4 D bytes per key, which passes the ridge near 250 rows.
// A CTA takes one kv head, one block of rows and one split of the keys, in 64-key tiles:
//   S = Q K^T (M 128, N 64) in TMEM, each row's softmax by one thread (running maximum and sum in
//   f32), P as fp16 pairs in TMEM, O += P V in TMEM.
// Two streams of 128 rows run a tile apart so that one's exponentials overlap the other's products:
// with more than 128 rows in the block the streams are two row tiles that share every K/V tile; with
// fewer they take alternate key tiles of the same rows, and their (m, l, O) are joined in shared
// memory at the end.  head_dim 256 leaves TMEM for one stream.
//
// int8 prefix: the codes, as exact fp16 integers, are the operands; the K scale multiplies the
// scores and the V scale the probabilities, so nothing is rounded that the fp16 form does not round.
#include <math_constants.h>

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
    static constexpr uint32_t kOffBar = kOffKV + kStages * 2 * kTileBytes;
    static constexpr uint32_t kSmemBytes = 1024 + kOffBar + 28 * 8 + 16;
    // TMEM columns: S, then P (fp16 pairs), then O from column 256 (one stream of D 256) or 192.
    static constexpr uint32_t kColS = 0, kColP = kStreams * kXK, kColO = kStreams == 1 ? 256 : 192;
    static_assert(kColP + kStreams * kXK / 2 <= kColO && kColO + kStreams * D <= kXTmemCols, "TMEM columns");
    static_assert(kSmemBytes <= 232448, "more than 227 KB of shared memory per CTA");
    // The streams' join: stream 1's O [D][128] f32, then m and l, in the K/V ring.
    static_assert(kStreams == 1 || (D * 128 + 256) * 4 <= kStages * 2 * kTileBytes, "join buffer");
};

enum : int {
    kXKvFull = 0,    // [6] TMA -> MMA
    kXKvEmpty = 6,   // [6] MMA commit -> producer
    kXSFull = 12,    // [2] MMA commit (S ready) -> softmax
    kXSFree = 14,    // [2] softmax (S read) -> MMA
    kXPFull = 16,    // [2] softmax (P written, O rescaled) -> MMA
    kXODone = 18,    // [2] MMA commit (PV done) -> softmax
    kXQFull = 20,    // q staged -> MMA
    kXMmaDone = 21,  // [2] everything an issuer issued has completed -> teardown
    kXStagger = 23,  // stream 0's first P written -> stream 1's issuer starts
};

template <int D, bool CAP, bool Q8>
__global__ void __launch_bounds__(PrefixLayout<D>::kThreads, 1)
    prefix_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                  const __grid_constant__ PrefixArgs a) {
    using L = PrefixLayout<D>;
    constexpr int NS = L::kStreams;
    // Raise the running max (and rescale O) only when a tile's max exceeds it by more than this
    // many powers of two: P stays below 2^8, or, times an int8 row's V scale, below 4 scales.
    constexpr float kRaise = Q8 ? 2.f : 8.f;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kOffBar);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 28);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.x, kvh = blockIdx.y;
    constexpr int RB = NS * kXQ;
    const int blk0 = blockIdx.z * RB;                 // first row of the block
    const int nblk = min(RB, a.rows - blk0);          // rows of the block
    const bool pair = nblk > kXQ;                     // streams: two row tiles, or alternate key tiles
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
            mbar_init(&bars[kXKvFull + i], 1);
            mbar_init(&bars[kXKvEmpty + i], pair ? 2 : 1);  // one commit per stream that reads the tile
        }
        for (int s = 0; s < NS; ++s) {
            mbar_init(&bars[kXSFull + s], 1);
            mbar_init(&bars[kXSFree + s], 128);
            mbar_init(&bars[kXPFull + s], 128);
            mbar_init(&bars[kXODone + s], 1);
            mbar_init(&bars[kXMmaDone + s], 1);
        }
        mbar_init(&bars[kXQFull], NS * 128);
        mbar_init(&bars[kXStagger], 128);
        fence_barrier_init();
    }
    if (warp == L::kMma) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                     "r"(kXTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    auto sQ = [&](int s) { return smem + (pair ? s : 0) * L::kQBytes; };
    auto sK = [&](int st) { return smem + L::kOffKV + st * 2 * L::kTileBytes; };
    auto sV = [&](int st) { return smem + L::kOffKV + st * 2 * L::kTileBytes + L::kTileBytes; };

    if (warp == L::kProducer) {
        if (lane == 0) {
            tma_prefetch_desc(&tmk);
            tma_prefetch_desc(&tmv);
            griddep_wait();  // the rows, or the staged codes, may come from the kernel before
            // Everything before this grid is complete: the own rows' kernel may start streaming.
            griddep_launch_dependents();
            int issued = 0;
            for (int j = 0; j < nk; ++j) {
                const int st = j % L::kStages;
                if (j >= L::kStages && !mbar_wait(&bars[kXKvEmpty + st], ((j / L::kStages) - 1) & 1, a.err, kErrSlotTimeout))
                    break;
                const int y = seg_row + kb + j * kXK;
                mbar_arrive_expect_tx(&bars[kXKvFull + st], 2 * L::kTileBytes);
#pragma unroll
                for (int blk = 0; blk < L::kBlocks; ++blk)
                    tma_load_2d(sK(st) + blk * L::kKVBlock, &tmk, blk * 64, y, &bars[kXKvFull + st]);
#pragma unroll
                for (int blk = 0; blk < L::kBlocks; ++blk)
                    tma_load_2d(sV(st) + blk * L::kKVBlock, &tmv, blk * 64, y, &bars[kXKvFull + st]);
                issued = j + 1;
            }
            for (int j = issued > L::kStages ? issued - L::kStages : 0; j < issued; ++j)
                mbar_wait(&bars[kXKvFull + j % L::kStages], (j / L::kStages) & 1, a.err, kErrTmaTimeout);
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
                if (!mbar_wait(&bars[kXKvFull + st], (j / L::kStages) & 1, a.err, kErrTmaTimeout)) return false;
                if (i >= 1 && !mbar_wait(&bars[kXSFree + s], (i - 1) & 1, a.err, kErrMmaTimeout)) return false;
                tc_fence_after();
                const uint32_t q_base = smem_addr(sQ(s)), k_base = smem_addr(sK(st));
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                    tc_mma(tmem + L::kColS + s * kXK,
                           sw128_desc(q_base + (ks >> 2) * L::kQBlock + (ks & 3) * 32, 16, 1024),
                           sw128_desc(k_base + (ks >> 2) * L::kKVBlock + (ks & 3) * 32, 16, 1024), idesc_qk, ks > 0);
                tc_commit(&bars[kXSFull + s]);
                return true;
            };
            auto issue_pv = [&](int i) -> bool {
                const int j = j0 + i * step, st = j % L::kStages;
                if (!mbar_wait(&bars[kXPFull + s], i & 1, a.err, kErrMmaTimeout)) return false;
                if (pair && s == 1 && tail && j == nk - 1 && !mbar_wait(&bars[kXPFull], i & 1, a.err, kErrMmaTimeout))
                    return false;
                tc_fence_after();
                const uint32_t v_base = smem_addr(sV(st));
#pragma unroll
                for (int kk = 0; kk < kXK / 16; ++kk)
                    tc_mma_ts(tmem + L::kColO + s * D, tmem + L::kColP + s * (kXK / 2) + kk * 8,
                              sw128_desc(v_base + kk * 16 * 128, L::kKVBlock, 1024), idesc_pv, i > 0 || kk > 0);
                tc_commit(&bars[kXODone + s]);
                return true;
            };
            if (ok && s == 1) ok = mbar_wait(&bars[kXStagger], 0, a.err, kErrMmaTimeout);
            if (ok) ok = issue_s(0);
            for (int i = 0; ok && i < cnt; ++i) {
                // S of the next tile needs only that this one's was read: it runs under the softmax.
                if (i + 1 < cnt && !issue_s(i + 1)) break;
                if (!issue_pv(i)) break;
                tc_commit(&bars[kXKvEmpty + (j0 + i * step) % L::kStages]);
            }
            tc_commit(&bars[kXMmaDone + s]);
            mbar_wait(&bars[kXMmaDone + s], 0, a.err, kErrMmaTimeout);
        }
        __syncwarp();
    } else {
        // ---- softmax warps: stream s = warp / 4, thread r <-> row r of the stream (TMEM lane r).
        const int s = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const int TG = a.T * a.G;
        griddep_wait();  // q may come from the kernel before
        // Stage q as fp16 rows in the MMA's swizzled K-major layout: a warp per row, lane l holding
        // PE consecutive elements, eight rows' loads in flight.
        {
            constexpr int PE = D / 32, kB = 8;
            const int tiles = pair ? 2 : 1;
#pragma unroll 1
            for (int base = 0; base < tiles * kXQ; base += L::kSoftWarps * kB) {
                uint32_t h[kB][PE / 2];
#pragma unroll
                for (int u = 0; u < kB; ++u) {
                    const int rr = base + u * L::kSoftWarps + warp;
                    const bool okr = rr < nblk;
                    const int row = blk0 + (okr ? rr : 0);
                    const int b = row / TG, tg = row % TG;
                    const size_t R = ((size_t)b * a.T + tg / a.G) * a.Hq + kvh * a.G + tg % a.G;
                    if (a.q16) {
                        const uint32_t *src = reinterpret_cast<const uint32_t *>(a.q16 + R * D) + lane * (PE / 2);
#pragma unroll
                        for (int e = 0; e < PE / 2; ++e) h[u][e] = okr ? src[e] : 0u;
                    } else {
                        const float2 *src = reinterpret_cast<const float2 *>(a.q + R * D) + lane * (PE / 2);
#pragma unroll
                        for (int e = 0; e < PE / 2; ++e) {
                            const float2 x = okr ? src[e] : make_float2(0.f, 0.f);
                            h[u][e] = pack_half2(x.x, x.y);
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < kB; ++u) {
                    const int rr = base + u * L::kSoftWarps + warp;
                    const int i = PE * lane;
                    uint8_t *d = smem + (rr >> 7) * L::kQBytes + (i >> 6) * L::kQBlock + sw128(rr & 127, (i & 63) >> 3) +
                                 (i & 7) * 2;
#pragma unroll
                    for (int e = 0; e < PE / 2; ++e) reinterpret_cast<uint32_t *>(d)[e] = h[u][e];
                }
            }
            fence_proxy_async_smem();
            mbar_arrive(&bars[kXQFull]);
        }
        const int cnt = tile_count(s), j0 = first_tile(s);
        const int rr = (pair ? s * kXQ : 0) + r;
        const bool row_ok = rr < nblk;
        const int row = blk0 + (row_ok ? rr : 0);
        const int b = row / TG, tg = row % TG;
        const size_t R = ((size_t)b * a.T + tg / a.G) * a.Hq + kvh * a.G + tg % a.G;
        const int lo = a.window > 0 && row_ok ? a.past_len[b] + tg / a.G - a.window + 1 : INT_MIN;
        const uint32_t tS = tmem + L::kColS + s * kXK + lane_base;
        const uint32_t tO = tmem + L::kColO + s * D + lane_base;
        const uint32_t tP = tmem + L::kColP + s * (kXK / 2) + lane_base;
        const float *ksc = Q8 ? a.scales + (size_t)kvh * 2 * a.scale_pitch : nullptr;
        const float *vsc = Q8 ? ksc + a.scale_pitch : nullptr;
        float m_used = -CUDART_INF_F;  // the maximum that the probabilities are relative to (log2 units)
        float l_run = 0.f;
        bool ok = true;
        for (int i = 0; i < cnt; ++i) {
            const int j = j0 + i * step, kbase = kb + j * kXK;
            const bool inside = kbase + kXK <= ke;
            if (!__all_sync(0xffffffffu, mbar_wait(&bars[kXSFull + s], i & 1, a.err, kErrMmaTimeout))) {
                ok = false;
                break;
            }
            tc_fence_after();
            uint32_t raw[2][32];
            tc_ld32_nowait(tS, raw[0]);
            tc_ld32_nowait(tS + 32, raw[1]);
            tc_wait_ld();
            tc_fence_before();
            mbar_arrive(&bars[kXSFree + s]);
            float v[64];
#pragma unroll
            for (int e = 0; e < 64; ++e) v[e] = __uint_as_float(raw[e >> 5][e & 31]);
            if constexpr (Q8) {
                if (inside) {
#pragma unroll
                    for (int e = 0; e < 64; e += 4) {
                        const float4 k4 = *reinterpret_cast<const float4 *>(ksc + kbase + e);
                        v[e] *= k4.x, v[e + 1] *= k4.y, v[e + 2] *= k4.z, v[e + 3] *= k4.w;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 64; ++e) v[e] *= kbase + e < ke ? ksc[kbase + e] : 0.f;
                }
            }
            const bool edge = !inside || kbase < lo;
            if (__any_sync(0xffffffffu, edge)) {
#pragma unroll
                for (int e = 0; e < 64; ++e) v[e] = kbase + e >= lo && kbase + e < ke ? v[e] : -CUDART_INF_F;
            }
            auto score = [&](float dot) {
                if constexpr (CAP)
                    return softcap_log2(dot, a.cap_k1, a.cap_k2);
                else
                    return dot * a.scale_log2;
            };
            const float mraw = max_tree(v);
            const float mt = mraw == -CUDART_INF_F ? -CUDART_INF_F : score(mraw);
            // Rows raise their maximum separately; the rescale pass is warp-collective.
            const bool raise = mt > m_used + kRaise || (m_used == -CUDART_INF_F && mt != -CUDART_INF_F);
            const bool rescale = raise && m_used != -CUDART_INF_F && i >= 1;
            bool waited = false;
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
            float2 acc[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[k] = make_float2(0.f, 0.f);
            uint32_t pk[32];
#pragma unroll
            for (int u = 0; u < 32; ++u) {
                float p0, p1;
                if constexpr (CAP) {
                    p0 = v[2 * u] == -CUDART_INF_F ? 0.f : ex2_fast(score(v[2 * u]) - m_eff);
                    p1 = v[2 * u + 1] == -CUDART_INF_F ? 0.f : ex2_fast(score(v[2 * u + 1]) - m_eff);
                } else {
                    const float2 x = ffma2(make_float2(v[2 * u], v[2 * u + 1]), make_float2(a.scale_log2, a.scale_log2),
                                           make_float2(-m_eff, -m_eff));
                    p0 = ex2_fast(x.x);
                    p1 = ex2_fast(x.y);
                }
                acc[u & 3] = fadd2(acc[u & 3], make_float2(p0, p1));
                if constexpr (Q8) {
                    // The V scale goes into the probability (a masked key's is not looked at).
                    const int key = kbase + 2 * u;
                    if (inside) {
                        const float2 s2 = *reinterpret_cast<const float2 *>(vsc + key);
                        p0 = v[2 * u] == -CUDART_INF_F ? 0.f : p0 * s2.x;
                        p1 = v[2 * u + 1] == -CUDART_INF_F ? 0.f : p1 * s2.y;
                    } else {
                        p0 = v[2 * u] == -CUDART_INF_F ? 0.f : p0 * vsc[key];
                        p1 = v[2 * u + 1] == -CUDART_INF_F ? 0.f : p1 * vsc[key + 1];
                    }
                }
                pk[u] = pack_half2(p0, p1);
            }
            const float2 acc01 = fadd2(acc[0], acc[1]), acc23 = fadd2(acc[2], acc[3]);
            const float rsum = (acc01.x + acc01.y) + (acc23.x + acc23.y);
            if (i >= 1 && !waited) {
                const bool got = mbar_wait(&bars[kXODone + s], (i - 1) & 1, a.err, kErrMmaTimeout);
                if (!__all_sync(0xffffffffu, got)) {
                    ok = false;
                    break;
                }
            }
            tc_st32(tP, pk);
            // Keys past the range end: zero V rows, so that 0 * (whatever the tile holds) stays 0.
            if ((s == 0 || !pair) && !inside) {
                bool zok = true;
                if (r < kXK && kbase + r >= ke) {
                    zok = mbar_wait(&bars[kXKvFull + j % L::kStages], (j / L::kStages) & 1, a.err, kErrTmaTimeout);
                    if (zok) {
#pragma unroll
                        for (int blk = 0; blk < L::kBlocks; ++blk)
#pragma unroll
                            for (int c = 0; c < 8; ++c)
                                *reinterpret_cast<uint4 *>(sV(j % L::kStages) + blk * L::kKVBlock + sw128(r, c)) =
                                    make_uint4(0u, 0u, 0u, 0u);
                    }
                }
                if (!__all_sync(0xffffffffu, zok)) {
                    ok = false;
                    break;
                }
                fence_proxy_async_smem();
            }
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(&bars[kXPFull + s]);
            if (s == 0 && i == 0) mbar_arrive(&bars[kXStagger]);
            l_run += rsum;
        }
        // Every product of this stream has landed.
        if (ok && cnt > 0) ok = __all_sync(0xffffffffu, mbar_wait(&bars[kXODone + s], (cnt - 1) & 1, a.err, kErrMmaTimeout));
        tc_fence_after();
        const int rows_total = a.B * a.T * a.Hq;
        float *dst = a.part_o + ((size_t)split * rows_total + R) * D;
        float f0 = 1.f, f1 = 0.f, m_fin = m_used, l_fin = l_run;
        float *jo = reinterpret_cast<float *>(smem + L::kOffKV);  // [D][128]
        float *jm = jo + D * 128, *jl = jm + 128;
        if (NS == 2 && !pair) {
            // Join the streams: stream 1 leaves its rows in the K/V ring (free: both streams'
            // products, which read it, are complete at the barrier), stream 0 adds them to its own.
            named_barrier_sync(1, 256);
            if (s == 1) {
                jm[r] = m_used;
                jl[r] = l_run;
#pragma unroll 1
                for (int c = 0; cnt > 0 && c < D / 32; ++c) {
                    uint32_t o[32];
                    tc_ld32_nowait(tO + c * 32, o);
                    tc_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; ++e) jo[(c * 32 + e) * 128 + r] = __uint_as_float(o[e]);
                }
            }
            named_barrier_sync(1, 256);
            if (s == 0) {
                const float m1 = jm[r];
                m_fin = fmaxf(m_used, m1);
                const float m_eff = m_fin == -CUDART_INF_F ? 0.f : m_fin;
                f0 = ex2_fast(m_used - m_eff);
                f1 = ex2_fast(m1 - m_eff);
                l_fin = l_run * f0 + jl[r] * f1;
            }
        }
        if (s == 0 || pair) {
            const bool other = NS == 2 && !pair && tile_count(1) > 0;
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = 0u;
                if (cnt > 0) {
                    tc_ld32_nowait(tO + c * 32, o);
                    tc_wait_ld();
                }
                float y[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    y[e] = __uint_as_float(o[e]) * f0;
                    if (other) y[e] = fmaf(jo[(c * 32 + e) * 128 + r], f1, y[e]);
                }
                if (row_ok) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<float4 *>(dst + c * 32 + e) = make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
                }
            }
            if (row_ok) {
                float *ml = a.part_ml + ((size_t)split * rows_total + R) * 2;
                *reinterpret_cast<float2 *>(ml) =
                    make_float2(m_fin == -CUDART_INF_F ? -CUDART_INF_F : m_fin * kXLn2, l_fin);
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

template <int D, bool CAP, bool Q8>
cudaError_t launch_prefix_t(const CUtensorMap &tmk, const CUtensorMap &tmv, const PrefixArgs &a, int splits,
                            cudaStream_t s, bool pdl) {
    using L = PrefixLayout<D>;
    static unsigned long long configured = 0;  // one bit per device: the opt-in is per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 64 || !(configured & (1ull << dev))) {
        cudaError_t e = cudaFuncSetAttribute(prefix_kernel<D, CAP, Q8>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             L::kSmemBytes);
        if (e != cudaSuccess) return e;
        if (dev < 64) configured |= 1ull << dev;
    }
    const int rb = prefix_block_rows(D, a.rows);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(splits, a.Hkv, (a.rows + rb - 1) / rb);
    cfg.blockDim = dim3(L::kThreads);
    cfg.dynamicSmemBytes = L::kSmemBytes;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, prefix_kernel<D, CAP, Q8>, tmk, tmv, a);
}

template <int D>
cudaError_t launch_prefix_d(const CUtensorMap &tmk, const CUtensorMap &tmv, const PrefixArgs &a, int splits,
                            cudaStream_t s, bool pdl) {
    if (a.softcap > 0.f)
        return a.scales ? launch_prefix_t<D, true, true>(tmk, tmv, a, splits, s, pdl)
                        : launch_prefix_t<D, true, false>(tmk, tmv, a, splits, s, pdl);
    return a.scales ? launch_prefix_t<D, false, true>(tmk, tmv, a, splits, s, pdl)
                    : launch_prefix_t<D, false, false>(tmk, tmv, a, splits, s, pdl);
}

// Codes (biased by +128) of rows [row0, row0 + rows) of every kv head as exact fp16 integers
// [Hkv][rows][D], 16 codes per thread and matrix.
__global__ void codes_to_half_kernel(const uint8_t *kc, const uint8_t *vc, __half *k, __half *v, int Hkv, int D, int cap,
                                     int row0, int rows) {
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

int prefix_block_rows(int head_dim, int rows) {
    (void)rows;
    return head_dim == 256 ? kXQ : 2 * kXQ;
}

cudaError_t launch_prefix(int head_dim, const CUtensorMap &tmk, const CUtensorMap &tmv, const PrefixArgs &a, int splits,
                          cudaStream_t s, bool pdl) {
    switch (head_dim) {
        case 64: return launch_prefix_d<64>(tmk, tmv, a, splits, s, pdl);
        case 128: return launch_prefix_d<128>(tmk, tmv, a, splits, s, pdl);
        case 256: return launch_prefix_d<256>(tmk, tmv, a, splits, s, pdl);
        default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_codes_to_half(const uint8_t *kc, const uint8_t *vc, __half *k, __half *v, int n_kv_heads,
                                 int head_dim, int cap, int row0, int rows, cudaStream_t s) {
    const long long n = (long long)n_kv_heads * rows * (head_dim / 16);
    if (n == 0) return cudaSuccess;
    const long long g = (n + 255) / 256;
    codes_to_half_kernel<<<(unsigned)(g < 8192 ? g : 8192), 256, 0, s>>>(kc, vc, k, v, n_kv_heads, head_dim, cap, row0,
                                                                         rows);
    return cudaGetLastError();
}

}  // namespace brk

// Matrix products of the layer around the attention operator on fp16 activations: the linear
// operator y = act(x W^T + b) + r and the gated feed-forward's first half
// h = act(x Wg^T + bg) * (x Wu^T + bu) (the FFN of recordLayerKV, kernels.ts:1737-1744).
//
// linear_kernel<NT, MATS> computes D^T = W X^T on tcgen05: 128 weight rows (output features) on
// the MMA's M, up to NT = 16 .. 128 tokens on its N, so a single token pads 15 MMA columns and
// not 127 rows.  With MATS = 2 a CTA holds the gate and the up tile of the same 128 features in two
// accumulators, and the product leaves through one epilogue.
//
// Few tokens are bound by streaming the weights once (2 n k bytes a matrix), so what counts is
// that every SM streams all the time: the (tile, k step) units of the whole product are dealt to
// one CTA per SM in equal contiguous ranges.  A range's first and last piece may cover part of a
// tile's k range; such pieces leave f32 partials in the workspace, and the last CTA of a tile to
// finish adds them in k order (the same order whoever is last: results do not change from run to
// run).
//
// The tensor core's f32 accumulation truncates: its error is a bias that grows with k (measured on
// N(0,1) operands against 64 bits: 3.1e-6 of the result at k 2560, 1.2e-5 at 10240).  Linear
// outputs may be f32, so its accumulators are drained every kDrainSteps k steps and the parts added
// in registers; gate-up outputs are fp16 (half a step 4.9e-4), which does not need it.
#include "common.cuh"
#include "internal.h"
#include "tcgen05.cuh"

namespace brk {

namespace {

constexpr int kLF = 128;      // output features per tile (MMA M, TMEM lanes)
constexpr int kLK = 64;       // k per step: one 128-byte swizzled row
constexpr int kLThreads = 192;
constexpr int kLProducer = 4, kLMma = 5;
constexpr int kDrainSteps = 16;  // 1024 of k per accumulator

template <int NT, int MATS>
struct LinearLayout {
    static constexpr uint32_t kWBox = kLF * 128;
    static constexpr uint32_t kXBox = NT * 128;
    static constexpr uint32_t kStageBytes = MATS * kWBox + kXBox;
    static constexpr int kFit = (200 * 1024) / kStageBytes;
    static constexpr int kStages = kFit < 12 ? kFit : 12;
    static constexpr uint32_t kCols = MATS * NT;                       // one accumulator set
    static constexpr uint32_t kTmemCols = 2 * kCols < 32 ? 32 : 2 * kCols;  // double-buffered
    static constexpr uint32_t kBarOff = kStages * kStageBytes;
    static constexpr uint32_t kSmemBytes = 1024 + kBarOff + (2 * kStages + 4) * 8 + 16;
    static constexpr int kSegSteps = MATS == 1 ? kDrainSteps : 1 << 30;
    static_assert(kTmemCols <= 512 && (kTmemCols & (kTmemCols - 1)) == 0, "TMEM columns");
    static_assert(kSmemBytes <= 232448, "more than 227 KB of shared memory per CTA");
};

// The unit ranges of the grid's CTAs: CTA c of G takes units [c U / G, (c + 1) U / G).
__device__ __forceinline__ long long range_begin(long long units, int c, int g) { return units * c / g; }
// The CTA whose range holds unit u (the largest c with range_begin(c) <= u).
__device__ __forceinline__ int cta_of(long long units, long long u, int g) { return (int)(((u + 1) * g - 1) / units); }

}  // namespace

// act(v) in f32 (BRK_ACT_*).
__device__ __forceinline__ float apply_act(float v, int act) {
    switch (act) {
        case BRK_ACT_SILU: return v / (1.f + expf(-v));
        case BRK_ACT_GELU: return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
        case BRK_ACT_GELU_TANH: return 0.5f * v * (1.f + tanhf(0.79788456080286536f * (v + 0.044715f * v * v * v)));
        case BRK_ACT_QUICK_GELU: return v / (1.f + expf(-1.702f * v));
        default: return v;
    }
}

namespace {

// 16 consecutive 32-bit TMEM columns of this thread's lane (no wait).
__device__ __forceinline__ void tc_ld16_nowait(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

template <int NT, int MATS>
__global__ void __launch_bounds__(kLThreads, 1)
    linear_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw0,
                  const __grid_constant__ CUtensorMap tw1, const __grid_constant__ LinearArgs a) {
    using L = LinearLayout<NT, MATS>;
    constexpr int S = L::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::kBarOff);
    uint64_t *empty = full + S;
    uint64_t *accfull = empty + S;
    uint64_t *accfree = accfull + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(accfree + 2);
    __shared__ int s_last;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nk = a.nk, g = gridDim.x, c = blockIdx.x;
    const long long units = (long long)a.tiles * nk;
    const long long u_lo = range_begin(units, c, g), u_hi = range_begin(units, c + 1, g);

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&accfull[i], 1);
            mbar_init(&accfree[i], 128);
        }
        fence_barrier_init();
    }
    if (warp == kLMma) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                     "r"(L::kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == kLProducer) {
        if (lane == 0) {
            tma_prefetch_desc(&tx);
            tma_prefetch_desc(&tw0);
            if constexpr (MATS == 2) tma_prefetch_desc(&tw1);
            // The weights of the first ring do not depend on the kernel before (which, in the same
            // call, writes the activations): they are in flight before the wait for it.
            const long long n_all = u_hi - u_lo;
            const int pre = (int)(n_all < S ? n_all : S);
            auto load_w = [&](long long u, uint8_t *st, uint64_t *bar) {
                const int tile = (int)(u / nk), kk = (int)(u % nk), f0 = tile / a.tiles_m * kLF;
                tma_load_2d(st, &tw0, kk * kLK, f0, bar);
                if constexpr (MATS == 2) tma_load_2d(st + L::kWBox, &tw1, kk * kLK, f0, bar);
            };
            auto load_x = [&](long long u, uint8_t *st, uint64_t *bar) {
                const int tile = (int)(u / nk), kk = (int)(u % nk), m0 = tile % a.tiles_m * NT;
                tma_load_2d(st + MATS * L::kWBox, &tx, kk * kLK, m0, bar);
            };
            for (int j = 0; j < pre; ++j) {
                mbar_arrive_expect_tx(&full[j], L::kStageBytes);
                load_w(u_lo + j, smem + j * L::kStageBytes, &full[j]);
            }
            griddep_wait();
            for (int j = 0; j < pre; ++j) load_x(u_lo + j, smem + j * L::kStageBytes, &full[j]);
            long long issued = pre;
            for (long long j = pre; j < n_all; ++j) {
                const int s = (int)(j % S);
                if (!mbar_wait(&empty[s], (uint32_t)((j / S) - 1) & 1, a.err, kErrSlotTimeout)) break;
                uint8_t *st = smem + s * L::kStageBytes;
                mbar_arrive_expect_tx(&full[s], L::kStageBytes);
                load_w(u_lo + j, st, &full[s]);
                load_x(u_lo + j, st, &full[s]);
                issued = j + 1;
            }
            // The next kernel of the call may start streaming its weights (what ran before this one is
            // complete: the wait above).
            griddep_launch_dependents();
            // No copy may still be in flight when the CTA exits.
            for (long long j = issued > S ? issued - S : 0; j < issued; ++j)
                mbar_wait(&full[j % S], (uint32_t)(j / S) & 1, a.err, kErrTmaTimeout);
        }
        __syncwarp();
    } else if (warp == kLMma) {
        if (lane == 0) {
            constexpr uint32_t idesc = f16_idesc(kLF, NT, 0, 0);
            long long j = 0;   // k steps consumed
            int seg = 0;       // accumulator sets used
            bool ok = true;
            for (long long u = u_lo; ok && u < u_hi;) {
                const int k0 = (int)(u % nk);
                const int k1 = (int)(u_hi - u < nk - k0 ? k0 + (u_hi - u) : nk);
                for (int ks = k0; ok && ks < k1; ks += L::kSegSteps) {
                    const int ke = k1 - ks < L::kSegSteps ? k1 : ks + L::kSegSteps;
                    const int buf = seg & 1;
                    if (seg >= 2 && !mbar_wait(&accfree[buf], ((seg >> 1) - 1) & 1, a.err, kErrMmaTimeout)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t d = tmem + buf * L::kCols;
                    for (int kk = ks; kk < ke; ++kk, ++j) {
                        const int s = (int)(j % S);
                        if (!mbar_wait(&full[s], (uint32_t)(j / S) & 1, a.err, kErrTmaTimeout)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t w = smem_addr(smem + s * L::kStageBytes), x = w + MATS * L::kWBox;
#pragma unroll
                        for (int e = 0; e < kLK / 16; ++e)
#pragma unroll
                            for (int m = 0; m < MATS; ++m)
                                tc_mma(d + m * NT, sw128_desc(w + m * L::kWBox + e * 32, 16, 1024),
                                       sw128_desc(x + e * 32, 16, 1024), idesc, kk > ks || e > 0);
                        tc_commit(&empty[s]);
                    }
                    if (ok) {
                        tc_commit(&accfull[buf]);
                        ++seg;
                    }
                }
                u += k1 - k0;
            }
            // Every MMA this thread issued completes before TMEM is released (the epilogue waits
            // for every set's commit; after a timeout the last sets are waited for here).
            for (int b = 0; b < 2; ++b) {
                const int used = (seg + 1 - b) / 2;  // sets committed on accumulator b
                if (used > 0) mbar_wait(&accfull[b], (used - 1) & 1, a.err, kErrMmaTimeout);
            }
        }
        __syncwarp();
    } else {
        // ---- epilogue warps: thread r <-> feature f0 + r (TMEM lane r), columns = tokens.
        const int r = threadIdx.x;
        const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
        griddep_wait();  // the residual may come from, and the output may be read by, what ran before
        int seg = 0;
        constexpr int CH = NT < 32 ? 16 : 32;  // columns handled at a time
        auto ld_cols = [&](uint32_t col, uint32_t (&v)[CH]) {
            if constexpr (CH == 16)
                tc_ld16_nowait(tmem + lane_base + col, v);
            else
                tc_ld32_nowait(tmem + lane_base + col, v);
        };
        bool ok = true;
        for (long long u = u_lo; u < u_hi;) {
            const int tile = (int)(u / nk), k0 = (int)(u % nk);
            const int k1 = (int)(u_hi - u < nk - k0 ? k0 + (u_hi - u) : nk);
            const int feat = tile / a.tiles_m * kLF + r, m0 = tile % a.tiles_m * NT;
            const int ntok = min(NT, a.M - m0);
            const bool whole = k0 == 0 && k1 == nk;
            float *part = nullptr;  // this piece's partial: [MATS][NT][128]
            if (!whole) part = a.ws + ((size_t)c * 2 + (u == u_lo ? 0 : 1)) * (MATS * NT * kLF) + r;
            const bool in = feat < a.n;
            const float b0 = in && a.bias[0] ? a.bias[0][feat] : 0.f;
            const float b1 = MATS == 2 && in && a.bias[1] ? a.bias[1][feat] : 0.f;
            // The finished values of CH tokens from column c0 on: act(v + b0) (* (w + b1)) (+ residual).
            auto finish = [&](int c0, const float (&v)[CH], const float (&w)[CH]) {
                float res[CH];
#pragma unroll
                for (int e = 0; e < CH; ++e)
                    res[e] = MATS == 1 && a.residual && in && c0 + e < ntok
                                 ? a.residual[(size_t)(m0 + c0 + e) * a.n + feat]
                                 : 0.f;
#pragma unroll
                for (int e = 0; e < CH; ++e) {
                    if (c0 + e < ntok && in) {
                        float y = apply_act(v[e] + b0, a.act);
                        if constexpr (MATS == 2)
                            y *= w[e] + b1;
                        else
                            y += res[e];
                        const size_t o = (size_t)(m0 + c0 + e) * a.n + feat;
                        if (a.out_half)
                            static_cast<__half *>(a.out)[o] = __float2half_rn(y);
                        else
                            static_cast<float *>(a.out)[o] = y;
                    }
                }
            };
            if constexpr (MATS == 1) {
                float acc[NT];
#pragma unroll
                for (int e = 0; e < NT; ++e) acc[e] = 0.f;
                for (int ks = k0; ks < k1; ks += L::kSegSteps, ++seg) {
                    const int buf = seg & 1;
                    // After one timeout no further set is waited for (the error word is set).
                    const bool got = ok && mbar_wait(&accfull[buf], (seg >> 1) & 1, a.err, kErrMmaTimeout);
                    ok = __all_sync(0xffffffffu, got);
                    tc_fence_after();
#pragma unroll
                    for (int c0 = 0; c0 < NT; c0 += CH) {
                        if (c0 < ntok) {
                            uint32_t v[CH];
                            ld_cols(buf * L::kCols + c0, v);
                            tc_wait_ld();
#pragma unroll
                            for (int e = 0; e < CH; ++e) acc[c0 + e] += __uint_as_float(v[e]);
                        }
                    }
                    tc_fence_before();
                    mbar_arrive(&accfree[buf]);
                }
#pragma unroll
                for (int c0 = 0; c0 < NT; c0 += CH) {
                    if (c0 < ntok) {
                        if (whole) {
                            float v[CH];
#pragma unroll
                            for (int e = 0; e < CH; ++e) v[e] = acc[c0 + e];
                            finish(c0, v, v);
                        } else {
#pragma unroll
                            for (int e = 0; e < CH; ++e)
                                if (c0 + e < ntok) __stcg(part + (c0 + e) * kLF, acc[c0 + e]);
                        }
                    }
                }
            } else {
                const int buf = seg & 1;
                const bool got = ok && mbar_wait(&accfull[buf], (seg >> 1) & 1, a.err, kErrMmaTimeout);
                ok = __all_sync(0xffffffffu, got);
                ++seg;
                tc_fence_after();
#pragma unroll 1
                for (int c0 = 0; c0 < ntok; c0 += CH) {
                    uint32_t vr[CH], wr[CH];
                    ld_cols(buf * L::kCols + c0, vr);
                    ld_cols(buf * L::kCols + NT + c0, wr);
                    tc_wait_ld();
                    float v[CH], w[CH];
#pragma unroll
                    for (int e = 0; e < CH; ++e) v[e] = __uint_as_float(vr[e]), w[e] = __uint_as_float(wr[e]);
                    if (whole) {
                        finish(c0, v, w);
                    } else {
#pragma unroll
                        for (int e = 0; e < CH; ++e)
                            if (c0 + e < ntok) {
                                __stcg(part + (c0 + e) * kLF, v[e]);
                                __stcg(part + (NT + c0 + e) * kLF, w[e]);
                            }
                    }
                }
                tc_fence_before();
                mbar_arrive(&accfree[buf]);
            }
            if (!whole) {
                // The last CTA of the tile to finish adds the pieces in k order.
                __threadfence();
                named_barrier_sync(2, 128);
                const long long t0 = (long long)tile * nk;
                const int c_first = cta_of(units, t0, g), c_last = cta_of(units, t0 + nk - 1, g);
                if (threadIdx.x == 0) {
                    const int prev = atomicAdd(&a.counters[tile], 1);
                    s_last = prev == c_last - c_first;
                    if (s_last) a.counters[tile] = 0;  // ready for the next launch
                }
                named_barrier_sync(2, 128);
                if (s_last) {
                    __threadfence();
#pragma unroll 1
                    for (int c0 = 0; c0 < ntok; c0 += CH) {
                        float v[CH], w[CH];
#pragma unroll
                        for (int e = 0; e < CH; ++e) v[e] = w[e] = 0.f;
                        for (int p = c_first; p <= c_last; ++p) {
                            const int slot = range_begin(units, p, g) >= t0 ? 0 : 1;
                            const float *src = a.ws + ((size_t)p * 2 + slot) * (MATS * NT * kLF) + r;
#pragma unroll
                            for (int e = 0; e < CH; ++e)
                                if (c0 + e < ntok) {
                                    v[e] += __ldcg(src + (c0 + e) * kLF);
                                    if constexpr (MATS == 2) w[e] += __ldcg(src + (NT + c0 + e) * kLF);
                                }
                        }
                        finish(c0, v, w);
                    }
                }
                named_barrier_sync(2, 128);  // s_last is read before the next piece writes it
            }
            u += k1 - k0;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kLMma)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::kTmemCols) : "memory");
}

template <int NT, int MATS>
cudaError_t launch_linear_t(const CUtensorMap &tx, const CUtensorMap *tw, const LinearArgs &a, int grid, cudaStream_t s,
                            bool pdl) {
    using L = LinearLayout<NT, MATS>;
    static unsigned long long configured = 0;  // one bit per device: the opt-in is per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 64 || !(configured & (1ull << dev))) {
        cudaError_t e = cudaFuncSetAttribute(linear_kernel<NT, MATS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             L::kSmemBytes);
        if (e != cudaSuccess) return e;
        if (dev < 64) configured |= 1ull << dev;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kLThreads);
    cfg.dynamicSmemBytes = L::kSmemBytes;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, linear_kernel<NT, MATS>, tx, tw[0], tw[MATS - 1], a);
}

template <int MATS>
cudaError_t launch_linear_m(int nt, const CUtensorMap &tx, const CUtensorMap *tw, const LinearArgs &a, int grid,
                            cudaStream_t s, bool pdl) {
    switch (nt) {
        case 16: return launch_linear_t<16, MATS>(tx, tw, a, grid, s, pdl);
        case 32: return launch_linear_t<32, MATS>(tx, tw, a, grid, s, pdl);
        case 64: return launch_linear_t<64, MATS>(tx, tw, a, grid, s, pdl);
        case 128: return launch_linear_t<128, MATS>(tx, tw, a, grid, s, pdl);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace

LinearPlan linear_plan(int rows, int k, int n, int mats, int sms) {
    LinearPlan p;
    p.nt = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
    p.tiles_m = (rows + p.nt - 1) / p.nt;
    p.tiles = (long long)((n + kLF - 1) / kLF) * p.tiles_m;
    p.nk = (k + kLK - 1) / kLK;
    const long long units = p.tiles * p.nk;
    p.grid = (int)(units < sms ? units : sms);
    p.ws_floats = (size_t)p.grid * 2 * mats * p.nt * kLF;
    return p;
}

cudaError_t launch_linear(int mats, const LinearPlan &p, const CUtensorMap &tx, const CUtensorMap *tw,
                          const LinearArgs &a, cudaStream_t s, bool pdl) {
    return mats == 2 ? launch_linear_m<2>(p.nt, tx, tw, a, p.grid, s, pdl)
                     : launch_linear_m<1>(p.nt, tx, tw, a, p.grid, s, pdl);
}

}  // namespace brk

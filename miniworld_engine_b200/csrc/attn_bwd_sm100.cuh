// Cross attention, backward, on the tensor cores (bf16, head dimension a multiple of 8 up to 128).
//
//   p_ij = exp(x_ij - m_i) / l_i       dp_ij = dout_i . v_j       ds_ij = p_ij (dp_ij - delta_i)
//   dv_j = sum_i p_ij dout_i           dk_j = scale sum_i ds_ij q_i           dq_i = scale sum_j ds_ij k_j
//
// Two kinds of blocks in one launch, each of which recomputes the scores and owns its results, so the same call gives the same
// bits: one per key tile walks over the queries (dk, dv), one per query tile over the keys (dq, and ds where the bias wants it).
// Together seven products of the scores' size instead of the five that a single kind would need, which would have to add up dq
// through memory.  Where the blocks of a kind are few and their loops long, several share a loop and write fp32 parts.
//
// What bounds it (2048 x 4096, 16 query heads on 4 key heads of 128: 243 us, 990 TFLOP/s of the seven products): a step of dq takes
// 2700 cycles, of which its products, whose operands come from shared memory at 94 cycles per 128 x 128 x 16, take 2000 to 2200;
// one of dk, dv 3180 with 2050 of products, since exponentials, probabilities' product and ds's product of a tile follow each other.
// In short loops (4 x 512 x 768, 16 heads of 64: 81 us) the start and the end of a block weigh as much as its steps.
//
// Both: 384 threads (TMA producer, UMMA issuer, a helper warp, bias producer, two groups of four softmax warps that share
// a 128 x 128 tile by halves of its columns).  p and ds go back to tensor memory as A operands of the second products,
// each group's half into the first 32 columns of the half of the scores (of dp) that the group itself has read.  Those
// columns are written again by products issued later by the same thread, which run in the order of issue.
// The second products of a tile and the first ones of the next are interleaved so that the tensor cores have work while
// the softmax warps wait for neither.
#pragma once

#include "attn_fwd_sm100.cuh"

namespace trimul {

constexpr int kAbThreads = 384;
constexpr int kStageIdAttnDkv = 12;
constexpr int kStageIdAttnDq = 13;

struct AttnBwdParams {
    AttnParams a;
    int n_tiles;                 // key tiles
    const uint32_t* words;       // as in the forward kernel
    const int* list;
    int bias_b1, bias_h1;
    AttnBwdSplit w;
};

template <int kD, bool kBias>
struct AbKvLayout {              // key-tile kernel: K, V, a ring of (Q, dout) pairs, bias tiles, row statistics
    static constexpr int kTile = kD / 64 * kAfSub;
    static constexpr int kStages = kD == 64 ? (kBias ? 3 : 4) : 2;
    static constexpr int kBiasBufs = kBias ? (kD == 64 ? 2 : 1) : 0;
    static constexpr int kOffRing = 2 * kTile;
    static constexpr int kOffBias = kOffRing + kStages * 2 * kTile;
    static constexpr int kOffStat = kOffBias + kBiasBufs * 2 * kAfSub;
    static constexpr int kStats = kBias && kD == 128 ? 1 : 2;    // buffers of 3 x 128 floats
    static constexpr int kOffBars = kOffStat + kStats * 3 * 128 * 4;
    static constexpr int kSmem = kOffBars + 256;
    static_assert((15 + 2 * kStages) * 8 + 8 <= 256, "barriers");
    static_assert(kSmem <= 227 * 1024, "shared memory");
};
template <int kD, bool kBias>
struct AbQLayout {               // query-tile kernel: Q, dout, rings of key and value tiles, bias tiles
    static constexpr int kTile = kD / 64 * kAfSub;
    static constexpr int kKSt = kD == 64 ? 4 : (kBias ? 2 : 3);
    static constexpr int kVSt = kD == 64 ? 4 : 2;
    static constexpr int kBiasBufs = kBias ? (kD == 64 ? 2 : 1) : 0;
    static constexpr int kOffK = 2 * kTile;
    static constexpr int kOffV = kOffK + kKSt * kTile;
    static constexpr int kOffBias = kOffV + kVSt * kTile;
    static constexpr int kOffBars = kOffBias + kBiasBufs * 2 * kAfSub;
    static constexpr int kSmem = kOffBars + 256;
    static_assert((11 + 3 * kKSt + 2 * kVSt) * 8 + 8 <= 256, "barriers");
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

// D = A[smem, K-major] B[smem, K-major]^T over kD, both tiles as kD / 64 swizzled sub-tiles of 64 columns
template <int kD>
__device__ __forceinline__ void ab_scores(uint32_t d, uint32_t a, uint32_t b) {
    constexpr uint32_t idesc = umma_idesc_bf16(128, 128);
    const uint64_t da = umma_smem_desc_sw128(a), db = umma_smem_desc_sw128(b);
#pragma unroll
    for (int kk = 0; kk < kD / 16; ++kk) {
        const uint64_t off = ((kk >> 2) * kAfSub + (kk & 3) * 32) >> 4;
        umma_ss_warp(d, da + off, db + off, idesc, kk > 0);
    }
}
// D += A[tensor memory, 128 columns of 16 bits: 64 in columns [0, 32), 64 in [64, 96)] B[smem, 128 rows of kD]
template <int kD>
__device__ __forceinline__ void ab_mix(uint32_t d, uint32_t a, uint32_t b, bool add) {
    constexpr uint32_t idesc = umma_idesc_bf16(128, kD, 0, 1);
    const uint64_t db = umma_smem_desc_mn_sw128(b, kAfSub, 1024);
#pragma unroll
    for (int kk = 0; kk < 8; ++kk)
        umma_ts_warp(d, a + (kk >> 2) * 64 + (kk & 3) * 8, db + ((kk * 2048) >> 4), idesc, add || kk > 0);
}
// 64 fp32 values as bf16 into columns [0, 32) of a tile half
__device__ __forceinline__ void ab_put(uint32_t t, const float (&f)[64]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) pk[e] = pack_bf16x2(f[32 * k + 2 * e], f[32 * k + 2 * e + 1]);
        tmem_st_32x16(t + 16 * k, pk);
    }
    tmem_st_wait();
}
__device__ __forceinline__ void ab_get(uint32_t t, float (&f)[64]) {
    uint32_t r[2][32];
    tmem_ld_32x32(t, r[0]);
    tmem_ld_32x32(t + 32, r[1]);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 64; ++e) f[e] = __uint_as_float(r[e >> 5][e & 31]);
}
// A row of a result: kD columns of tensor memory, times `f`, to global memory (`write`: the row exists; zero: all zeros)
template <int kD>
__device__ __forceinline__ void ab_row_out(uint32_t t, __nv_bfloat16* dst, int D, float f, bool write, bool zero) {
#pragma unroll 1
    for (int cc = 0; cc < kD; cc += 16) {
        if (cc >= D) break;
        uint32_t o[16];
        tmem_ld_32x16(t + cc, o);
        tmem_ld_wait();
        if (!write) continue;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            if (cc + 8 * g >= D) break;
            uint32_t y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                y[e] = zero ? 0u : pack_bf16x2(__uint_as_float(o[8 * g + 2 * e]) * f, __uint_as_float(o[8 * g + 2 * e + 1]) * f);
            *reinterpret_cast<uint4*>(dst + cc + 8 * g) = make_uint4(y[0], y[1], y[2], y[3]);
        }
    }
}

// The same of a part: fp32
template <int kD>
__device__ __forceinline__ void ab_part_out(uint32_t t, float* dst, int D, float f, bool write, bool zero) {
#pragma unroll 1
    for (int cc = 0; cc < kD; cc += 16) {
        if (cc >= D) break;
        uint32_t o[16];
        tmem_ld_32x16(t + cc, o);
        tmem_ld_wait();
        if (!write) continue;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            if (cc + 4 * g >= D) break;
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = zero ? 0.f : __uint_as_float(o[4 * g + e]) * f;
            *reinterpret_cast<float4*>(dst + cc + 4 * g) = make_float4(y[0], y[1], y[2], y[3]);
        }
    }
}

// ---------------------------------------------------------------------------------------
// dk, dv: a block per (key tile, key head, batch element).  Scores transposed: a lane of tensor memory is a key, a column a query.  Masked keys
// only ever meet their own lanes, so whatever their rows hold stays there, and their results are written as zeros.
// ---------------------------------------------------------------------------------------
template <int kD, bool kBias>
__device__ __forceinline__ void attn_dkv_block(const CUtensorMap& tmQ, const CUtensorMap& tmK, const CUtensorMap& tmV,
                                               const CUtensorMap& tmG, const CUtensorMap& tmBias, const AttnBwdParams& bp, int block) {
    using L = AbKvLayout<kD, kBias>;
    const AttnParams& p = bp.a;
    constexpr int kSt = L::kStages, kBb = L::kBiasBufs > 0 ? L::kBiasBufs : 1;
    extern __shared__ __align__(1024) uint8_t smem[];
    if ((smem_u32(smem) & 1023u) != 0u) {
        if (threadIdx.x == 0) report_timeout(p.status, kStageIdAttnDkv, 900);
        return;
    }
    uint8_t* ring = smem + L::kOffRing;
    float* stat = reinterpret_cast<float*>(smem + L::kOffStat);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBars);
    uint64_t* kv_full = bars;                     // [2] K, V
    uint64_t* s_full = bars + 2;                  // scores
    uint64_t* dp_full = bars + 3;
    uint64_t* p_full = bars + 4;                  // probabilities in tensor memory
    uint64_t* ds_full = bars + 5;
    uint64_t* done = bars + 6;
    uint64_t* st_full = bars + 7;                 // [2] statistics of a query tile
    uint64_t* st_empty = bars + 9;                // [2]
    uint64_t* b_full = bars + 11;                 // [2]
    uint64_t* b_empty = bars + 13;                // [2]
    uint64_t* full = bars + 15;                   // [kSt]
    uint64_t* empty = full + kSt;                 // [kSt]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(empty + kSt);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = warp_uniform((int)threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int tile = block % bp.n_tiles, j0 = tile * kAfRows, hk = block / bp.n_tiles % p.Hk;
    const int b = block / bp.n_tiles / p.Hk % p.B, split = block / bp.n_tiles / p.Hk / p.B;
    const int group = p.H / p.Hk, nq = (p.Lq + kAfRows - 1) / kAfRows;

    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(&kv_full[s], 1);
            mbar_init(&st_full[s], 1);
            mbar_init(&st_empty[s], 8);
            mbar_init(&b_full[s], 1);
            mbar_init(&b_empty[s], 8);
        }
        mbar_init(s_full, 1);
        mbar_init(dp_full, 1);
        mbar_init(p_full, 8);
        mbar_init(ds_full, 8);
        mbar_init(done, 1);
        for (int s = 0; s < kSt; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        *abort_flag = 0;
        fence_mbarrier_init();
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
        tma_prefetch_desc(&tmG);
        if (kBias) tma_prefetch_desc(&tmBias);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = warp_uniform(*tmem_slot);
    const uint32_t tS = tmem, tP = tmem + 128, tV = tmem + 256, tK = tmem + 256 + kD;
    griddep_wait();
    griddep_launch_dependents();

    const uint4 w4 = bp.words != nullptr ? at_load(reinterpret_cast<const uint4*>(bp.words) + (long long)b * bp.n_tiles + tile)
                                         : make_uint4(~0u, ~0u, ~0u, ~0u);
    const int first = split * bp.w.kv_share;             // of the query tiles, head after head
    const int n = warp_uniform((w4.x | w4.y | w4.z | w4.w) != 0u ? max(0, min(bp.w.kv_share, group * nq - first)) : 0);
    auto head_of = [&](int it) { return hk * group + (first + it) / nq; };
    auto row_of = [&](int it) { return ((first + it) % nq) * kAfRows; };

    if (warp == 0) {
        if (lane == 0 && n > 0) {
            for (int u = 0; u < 2; ++u) {
                mbar_arrive_expect_tx(&kv_full[u], L::kTile);
#pragma unroll
                for (int s = 0; s < kD / 64; ++s)
                    tma_load_4d(smem + u * L::kTile + s * kAfSub, u ? &tmV : &tmK, &kv_full[u], s * 64, j0, hk, b);
            }
            for (int it = 0; it < n; ++it) {
                const int s = it % kSt;
                if (!mbar_wait<true>(&empty[s], ((it / kSt) & 1) ^ 1, abort_flag, p.status, kStageIdAttnDkv, 100 + s)) break;
                mbar_arrive_expect_tx(&full[s], 2 * L::kTile);
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int c = 0; c < kD / 64; ++c)
                        tma_load_4d(ring + (2 * s + u) * L::kTile + c * kAfSub, u ? &tmG : &tmQ, &full[s], c * 64, row_of(it), head_of(it), b);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (n > 0) {
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t ph, int detail) {
                ok = ok && warp_wait(bar, ph, lane, abort_flag, p.status, kStageIdAttnDkv, detail);
                tcgen05_fence_after();
                return ok;
            };
            const uint32_t k = smem_u32(smem), v = k + L::kTile, r0 = smem_u32(ring);
            auto q_at = [&](int it) { return r0 + (it % kSt) * 2 * L::kTile; };
            if (wait(&kv_full[0], 0, 300) && wait(&full[0], 0, 301)) {
                ab_scores<kD>(tS, k, q_at(0));
                umma_commit_warp(s_full);
                if (wait(&kv_full[1], 0, 302)) {
                    ab_scores<kD>(tP, v, q_at(0) + L::kTile);
                    umma_commit_warp(dp_full);
                }
            }
            for (int it = 0; ok && it < n; ++it) {
                const bool more = it + 1 < n;
                if (!wait(p_full, it & 1, 310)) break;
                ab_mix<kD>(tV, tS, q_at(it) + L::kTile, it > 0);
                if (more) {
                    if (!wait(&full[(it + 1) % kSt], ((it + 1) / kSt) & 1, 320)) break;
                    ab_scores<kD>(tS, k, q_at(it + 1));
                    umma_commit_warp(s_full);
                }
                if (!wait(ds_full, it & 1, 330)) break;
                ab_mix<kD>(tK, tP, q_at(it), it > 0);
                umma_commit_warp(&empty[it % kSt]);
                if (more) {
                    ab_scores<kD>(tP, v, q_at(it + 1) + L::kTile);
                    umma_commit_warp(dp_full);
                } else {
                    umma_commit_warp(done);
                }
            }
        }
    } else if (warp == 2) {
        // row statistics of a query tile.  Without a bias the maximum and the sum are one number; rows behind the last
        // one get probability zero
        for (int it = 0; it < n; ++it) {
            const int s = it % L::kStats, i0 = row_of(it);
            const long long base = ((long long)b * p.H + head_of(it)) * p.Lq;
            float2 ml[4];
            float dl[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = i0 + 32 * e + lane;
                ml[e] = i < p.Lq ? at_load(p.stats + base + i) : make_float2(0.f, INFINITY);
                dl[e] = i < p.Lq ? at_load(p.delta + base + i) : 0.f;
            }
            if (!warp_wait(&st_empty[s], ((it / L::kStats) & 1) ^ 1, lane, abort_flag, p.status, kStageIdAttnDkv, 500 + s)) break;
            float* d = stat + s * 384 + lane;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                d[32 * e] = kBias ? -ml[e].x : -fmaf(ml[e].x, kLog2e, ml[e].y);
                d[128 + 32 * e] = -dl[e];
                if (kBias) d[256 + 32 * e] = -ml[e].y;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&st_full[s]);
        }
    } else if (warp == 3) {
        if (kBias && lane == 0) {
            for (int it = 0; it < n; ++it) {
                const int s = it % kBb;
                if (!mbar_wait<true>(&b_empty[s], ((it / kBb) & 1) ^ 1, abort_flag, p.status, kStageIdAttnDkv, 600 + s)) break;
                mbar_arrive_expect_tx(&b_full[s], 2 * kAfSub);
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    tma_load_4d(smem + L::kOffBias + (s * 2 + u) * kAfSub, &tmBias, &b_full[s], j0 + u * 64, row_of(it),
                                bp.bias_h1 ? 0 : head_of(it), bp.bias_b1 ? 0 : b);
            }
        }
        __syncwarp();
    } else {
        const int g = (warp - 4) >> 2, q = warp & 3, row = q * 32 + lane, j = j0 + row;
        const uint32_t lane_off = (uint32_t)(q * 32) << 16;
        const float c2 = p.scale * kLog2e;
        bool ok = true;
        for (int it = 0; it < n; ++it) {
            const int s = it % L::kStats;
            const float* sa = stat + s * 384 + g * 64;
            if (!(ok = warp_wait(&st_full[s], (it / L::kStats) & 1, lane, abort_flag, p.status, kStageIdAttnDkv, 400))) break;
            if (!(ok = warp_wait(s_full, it & 1, lane, abort_flag, p.status, kStageIdAttnDkv, 401))) break;
            tcgen05_fence_after();
            float x[64];
            ab_get(tS + g * 64 + lane_off, x);
            if constexpr (kBias) {
                const int bs = it % kBb;
                if (!(ok = warp_wait(&b_full[bs], (it / kBb) & 1, lane, abort_flag, p.status, kStageIdAttnDkv, 402))) break;
                // column `row` of the bias tile: lanes are neighbouring keys, two bytes each
                const uint8_t* bb = smem + L::kOffBias + (bs * 2 + (row >> 6)) * kAfSub + g * 64 * 128 + (row & 7) * 2;
                const uint32_t chunk = (row & 63) >> 3;
#pragma unroll
                for (int e = 0; e < 64; ++e) {
                    const float bias = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(bb + e * 128 + ((chunk ^ (e & 7)) << 4)) << 16);
                    x[e] = fmaf(x[e], p.scale, bias);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&b_empty[bs]);
            }
#pragma unroll
            for (int e = 0; e < 64; e += 4) {
                const float4 a = *reinterpret_cast<const float4*>(sa + e);
                const float na[4] = {a.x, a.y, a.z, a.w};
                if constexpr (kBias) {
                    const float4 l4 = *reinterpret_cast<const float4*>(sa + 256 + e);
                    const float nl[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
                    for (int u = 0; u < 4; ++u) x[e + u] = ex2f(fmaf(x[e + u] + na[u], kLog2e, nl[u]));
                } else {
#pragma unroll
                    for (int u = 0; u < 4; ++u) x[e + u] = ex2f(fmaf(x[e + u], c2, na[u]));
                }
            }
            ab_put(tS + g * 64 + lane_off, x);
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full);
            if (!(ok = warp_wait(dp_full, it & 1, lane, abort_flag, p.status, kStageIdAttnDkv, 403))) break;
            tcgen05_fence_after();
            float dp[64];
            ab_get(tP + g * 64 + lane_off, dp);
#pragma unroll
            for (int e = 0; e < 64; e += 4) {
                const float4 a = *reinterpret_cast<const float4*>(sa + 128 + e);
                const float nd[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                for (int u = 0; u < 4; ++u) x[e + u] *= dp[e + u] + nd[u];
            }
            ab_put(tP + g * 64 + lane_off, x);
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(ds_full);
                mbar_arrive(&st_empty[s]);
            }
        }
        if (n > 0 && ok) ok = warp_wait(done, 0, lane, abort_flag, p.status, kStageIdAttnDkv, 404);
        tcgen05_fence_after();
        if (ok) {
            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
            const bool zero = n == 0 || ((w[q] >> lane) & 1u) == 0u;
            const uint32_t acc = (g == 0 ? tV : tK) + lane_off;
            const float f = g == 0 ? 1.f : p.scale;
            if (bp.w.dk != nullptr) {
                const long long prow = (((long long)split * p.B + b) * p.Hk + hk) * p.Lk + j;
                ab_part_out<kD>(acc, (g == 0 ? bp.w.dv : bp.w.dk) + prow * p.D, p.D, f, j < p.Lk, zero);
            } else {
                const AttnTensor& t = g == 0 ? p.dv : p.dk;
                __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(t.p) + b * t.b + (long long)j * t.l + hk * t.h;
                ab_row_out<kD>(acc, dst, p.D, f, j < p.Lk, zero);
            }
        }
    }

    if (*abort_flag != 0) {
        for (int t = 0; t < 256; ++t) __nanosleep(1000);
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 1) {
        tcgen05_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---------------------------------------------------------------------------------------
// dq and ds: a block per (query tile, head, batch element).  A lane of tensor memory is a query, a column a key.  Key rows of masked keys are
// zeroed in shared memory, where ds K would read them.
// ---------------------------------------------------------------------------------------
template <int kD, bool kBias, typename Ds>
__device__ __forceinline__ void attn_dq_block(const CUtensorMap& tmQ, const CUtensorMap& tmK, const CUtensorMap& tmV,
                                              const CUtensorMap& tmG, const CUtensorMap& tmBias, const AttnBwdParams& bp, int block) {
    using L = AbQLayout<kD, kBias>;
    const AttnParams& p = bp.a;
    constexpr int kKSt = L::kKSt, kVSt = L::kVSt, kBb = L::kBiasBufs > 0 ? L::kBiasBufs : 1;
    extern __shared__ __align__(1024) uint8_t smem[];
    if ((smem_u32(smem) & 1023u) != 0u) {
        if (threadIdx.x == 0) report_timeout(p.status, kStageIdAttnDq, 900);
        return;
    }
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBars);
    uint64_t* q_full = bars;                      // [2] Q, dout
    uint64_t* s_full = bars + 2;
    uint64_t* s_read = bars + 3;                  // scores are in registers
    uint64_t* dp_full = bars + 4;
    uint64_t* ds_full = bars + 5;
    uint64_t* done = bars + 6;
    uint64_t* b_full = bars + 7;                  // [2]
    uint64_t* b_empty = bars + 9;                 // [2]
    uint64_t* k_full = bars + 11;                 // [kKSt]
    uint64_t* k_ok = k_full + kKSt;               // [kKSt] rows of masked keys zeroed
    uint64_t* k_empty = k_ok + kKSt;              // [kKSt]
    uint64_t* v_full = k_empty + kKSt;            // [kVSt]
    uint64_t* v_empty = v_full + kVSt;            // [kVSt]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_empty + kVSt);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = warp_uniform((int)threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int nq = (p.Lq + kAfRows - 1) / kAfRows;
    const int i0 = block % nq * kAfRows, h = block / nq % p.H, hk = h / (p.H / p.Hk);
    const int b = block / nq / p.H % p.B, split = block / nq / p.H / p.B;

    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(&q_full[s], 1);
            mbar_init(&b_full[s], 1);
            mbar_init(&b_empty[s], 8);
        }
        mbar_init(s_full, 1);
        mbar_init(s_read, 8);
        mbar_init(dp_full, 1);
        mbar_init(ds_full, 8);
        mbar_init(done, 1);
        for (int s = 0; s < kKSt; ++s) {
            mbar_init(&k_full[s], 1);
            mbar_init(&k_ok[s], 1);
            mbar_init(&k_empty[s], 1);
        }
        for (int s = 0; s < kVSt; ++s) {
            mbar_init(&v_full[s], 1);
            mbar_init(&v_empty[s], 1);
        }
        *abort_flag = 0;
        fence_mbarrier_init();
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
        tma_prefetch_desc(&tmG);
        if (kBias) tma_prefetch_desc(&tmBias);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = warp_uniform(*tmem_slot);
    const uint32_t tS = tmem, tP = tmem + 128, tQ = tmem + 256;
    griddep_wait();
    griddep_launch_dependents();

    const int* list = bp.list != nullptr ? bp.list + (long long)b * (bp.n_tiles + 1) : nullptr;
    // of the listed key tiles a block takes its share
    const int listed = warp_uniform(list != nullptr ? list[0] : bp.n_tiles), share = (listed + bp.w.q_splits - 1) / bp.w.q_splits;
    const int first = min(split * share, listed), n = min(share, listed - first);
    auto tile_at = [&](int it) { return list != nullptr ? at_load(list + 1 + first + it) : first + it; };

    if (warp == 0) {
        if (lane == 0 && n > 0) {
            auto load = [&](uint8_t* dst, const CUtensorMap* m, uint64_t* bar, int r, int head) {
                mbar_arrive_expect_tx(bar, L::kTile);
#pragma unroll
                for (int c = 0; c < kD / 64; ++c) tma_load_4d(dst + c * kAfSub, m, bar, c * 64, r, head, b);
            };
            for (int it = 0; it < n; ++it) {
                const int ks = it % kKSt, vs = it % kVSt, j0 = tile_at(it) * kAfRows;
                if (it == 0) load(smem, &tmQ, &q_full[0], i0, h);
                if (!mbar_wait<true>(&k_empty[ks], ((it / kKSt) & 1) ^ 1, abort_flag, p.status, kStageIdAttnDq, 100 + ks)) break;
                load(smem + L::kOffK + ks * L::kTile, &tmK, &k_full[ks], j0, hk);
                if (it == 0) load(smem + L::kTile, &tmG, &q_full[1], i0, h);
                if (!mbar_wait<true>(&v_empty[vs], ((it / kVSt) & 1) ^ 1, abort_flag, p.status, kStageIdAttnDq, 110 + vs)) break;
                load(smem + L::kOffV + vs * L::kTile, &tmV, &v_full[vs], j0, hk);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (n > 0) {
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t ph, int detail) {
                ok = ok && warp_wait(bar, ph, lane, abort_flag, p.status, kStageIdAttnDq, detail);
                tcgen05_fence_after();
                return ok;
            };
            const uint32_t q = smem_u32(smem), gq = q + L::kTile, k0 = q + L::kOffK, v0 = q + L::kOffV;
            uint64_t* k_ready = bp.words != nullptr ? k_ok : k_full;
            auto scores = [&](int it) {
                if (!wait(&k_ready[it % kKSt], (it / kKSt) & 1, 300)) return;
                ab_scores<kD>(tS, q, k0 + (it % kKSt) * L::kTile);
                umma_commit_warp(s_full);
            };
            auto products = [&](int it) {                // dp = dout v^T
                if (!wait(&v_full[it % kVSt], (it / kVSt) & 1, 310)) return;
                ab_scores<kD>(tP, gq, v0 + (it % kVSt) * L::kTile);
                umma_commit_warp(dp_full);
                umma_commit_warp(&v_empty[it % kVSt]);
            };
            if (wait(&q_full[0], 0, 320)) scores(0);
            if (wait(&q_full[1], 0, 321)) products(0);
            for (int it = 0; ok && it < n; ++it) {
                if (it + 1 < n && wait(s_read, it & 1, 330)) scores(it + 1);
                if (!wait(ds_full, it & 1, 340)) break;
                ab_mix<kD>(tQ, tP, k0 + (it % kKSt) * L::kTile, it > 0);
                umma_commit_warp(&k_empty[it % kKSt]);
                if (it + 1 < n) products(it + 1);
                else umma_commit_warp(done);
            }
        }
    } else if (warp == 2) {
        if (bp.words != nullptr) {
            for (int it = 0; it < n; ++it) {
                const int s = it % kKSt, t = tile_at(it);
                const uint4 w4 = at_load(reinterpret_cast<const uint4*>(bp.words) + (long long)b * bp.n_tiles + t);
                if (!warp_wait(&k_full[s], (it / kKSt) & 1, lane, abort_flag, p.status, kStageIdAttnDq, 500 + s)) break;
                if ((w4.x & w4.y & w4.z & w4.w) != 0xffffffffu) {
                    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
                    uint8_t* k = smem + L::kOffK + s * L::kTile;
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        for (int r = lane >> 3; r < 32; r += 4)
                            if (((w[c] >> r) & 1u) == 0u)
#pragma unroll
                                for (int u = 0; u < kD / 64; ++u)
                                    *reinterpret_cast<uint4*>(k + u * kAfSub + (c * 32 + r) * 128 + (lane & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&k_ok[s]);
            }
        }
    } else if (warp == 3) {
        if (kBias && lane == 0) {
            for (int it = 0; it < n; ++it) {
                const int s = it % kBb, j0 = tile_at(it) * kAfRows;
                if (!mbar_wait<true>(&b_empty[s], ((it / kBb) & 1) ^ 1, abort_flag, p.status, kStageIdAttnDq, 600 + s)) break;
                mbar_arrive_expect_tx(&b_full[s], 2 * kAfSub);
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    tma_load_4d(smem + L::kOffBias + (s * 2 + u) * kAfSub, &tmBias, &b_full[s], j0 + u * 64, i0,
                                bp.bias_h1 ? 0 : h, bp.bias_b1 ? 0 : b);
            }
        }
        __syncwarp();
    } else {
        const int g = (warp - 4) >> 2, q = warp & 3, row = q * 32 + lane, i = i0 + row;
        const uint32_t lane_off = (uint32_t)(q * 32) << 16;
        const float c2 = p.scale * kLog2e;
        const long long srow = ((long long)b * p.H + h) * p.Lq + i;
        const float2 ml = i < p.Lq ? at_load(p.stats + srow) : make_float2(0.f, INFINITY);
        const float delta = i < p.Lq ? at_load(p.delta + srow) : 0.f;
        const float both = -fmaf(ml.x, kLog2e, ml.y);
        constexpr int kVec = 16 / (int)sizeof(Ds);
        constexpr bool kParts = sizeof(Ds) == 4;           // ds_parts: 16 bytes are four columns of a row, the next row's after them
        Ds* ds = p.ds != nullptr ? static_cast<Ds*>(p.ds) + b * p.ds_b + h * p.ds_h + (kParts ? 4ll * i : i * p.ds_i) : nullptr;
        auto ds_at = [&](int col) { return reinterpret_cast<uint4*>(kParts ? ds + (long long)col * p.Lq : ds + col); };
        bool ok = true;
        int t_next = first > 0 ? tile_at(-1) + 1 : 0;      // first key tile whose ds is not written yet
        auto clear_ds = [&](int t_end) {
            if (ds != nullptr && i < p.Lq)
                for (int t = t_next; t < t_end; ++t)
                    for (int e = 0; e < 64; e += kVec)
                        if (t * kAfRows + g * 64 + e < p.Lk)
                            *ds_at(t * kAfRows + g * 64 + e) = make_uint4(0u, 0u, 0u, 0u);
            t_next = t_end + 1;
        };
        for (int it = 0; it < n; ++it) {
            const int t = tile_at(it);
            uint4 w4 = make_uint4(~0u, ~0u, ~0u, ~0u);
            if (bp.words != nullptr) w4 = at_load(reinterpret_cast<const uint4*>(bp.words) + (long long)b * bp.n_tiles + t);
            else if ((t + 1) * kAfRows > p.Lk) w4 = tail_words(p.Lk - t * kAfRows);
            const uint32_t w[2] = {g == 0 ? w4.x : w4.z, g == 0 ? w4.y : w4.w};
            if (!(ok = warp_wait(s_full, it & 1, lane, abort_flag, p.status, kStageIdAttnDq, 400))) break;
            tcgen05_fence_after();
            float x[64];
            ab_get(tS + g * 64 + lane_off, x);
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_read);
            if constexpr (kBias) {
                const int bs = it % kBb;
                if (!(ok = warp_wait(&b_full[bs], (it / kBb) & 1, lane, abort_flag, p.status, kStageIdAttnDq, 401))) break;
                const uint8_t* br = smem + L::kOffBias + (bs * 2 + g) * kAfSub + row * 128;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint4 v = *reinterpret_cast<const uint4*>(br + ((e ^ (row & 7)) << 4));
                    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        x[8 * e + 2 * c] = fmaf(x[8 * e + 2 * c], p.scale, bf16_lo(u[c]));
                        x[8 * e + 2 * c + 1] = fmaf(x[8 * e + 2 * c + 1], p.scale, bf16_hi(u[c]));
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&b_empty[bs]);
#pragma unroll
                for (int e = 0; e < 64; ++e) x[e] = ex2f(fmaf(x[e] - ml.x, kLog2e, -ml.y));
            } else {
#pragma unroll
                for (int e = 0; e < 64; ++e) x[e] = ex2f(fmaf(x[e], c2, both));
            }
            const bool holes = (w[0] & w[1]) != 0xffffffffu;
            if (!(ok = warp_wait(dp_full, it & 1, lane, abort_flag, p.status, kStageIdAttnDq, 402))) break;
            tcgen05_fence_after();
            float dp[64];
            ab_get(tP + g * 64 + lane_off, dp);
#pragma unroll
            for (int e = 0; e < 64; ++e) x[e] *= dp[e] - delta;
            if (holes) {
#pragma unroll
                for (int e = 0; e < 64; ++e)
                    if (((w[e >> 5] >> (e & 31)) & 1u) == 0u) x[e] = 0.f;
            }
            ab_put(tP + g * 64 + lane_off, x);
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(ds_full);
            if (ds != nullptr) {
                clear_ds(t);
                if (i < p.Lq) {
#pragma unroll
                    for (int e = 0; e < 64; e += kVec)
                        if (t * kAfRows + g * 64 + e < p.Lk) {
                            if constexpr (sizeof(Ds) == 2)
                                *ds_at(t * kAfRows + g * 64 + e) =
                                    make_uint4(pack_bf16x2(x[e], x[e + 1]), pack_bf16x2(x[e + 2], x[e + 3]),
                                               pack_bf16x2(x[e + 4], x[e + 5]), pack_bf16x2(x[e + 6], x[e + 7]));
                            else
                                *ds_at(t * kAfRows + g * 64 + e) = make_uint4(__float_as_uint(x[e]), __float_as_uint(x[e + 1]),
                                                                              __float_as_uint(x[e + 2]), __float_as_uint(x[e + 3]));
                        }
                }
            }
        }
        if (ok && split == bp.w.q_splits - 1) clear_ds(bp.n_tiles);
        if (n > 0 && ok) ok = warp_wait(done, 0, lane, abort_flag, p.status, kStageIdAttnDq, 403);
        tcgen05_fence_after();
        if (ok && g == 0) {
            if (bp.w.dq != nullptr) {
                const long long prow = (((long long)split * p.B + b) * p.H + h) * p.Lq + i;
                ab_part_out<kD>(tQ + lane_off, bp.w.dq + prow * p.D, p.D, p.scale, i < p.Lq, n == 0);
            } else {
                __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.dq.p) + b * p.dq.b + (long long)i * p.dq.l + h * p.dq.h;
                ab_row_out<kD>(tQ + lane_off, dst, p.D, p.scale, i < p.Lq, n == 0);
            }
        }
    }

    if (*abort_flag != 0) {
        for (int t = 0; t < 256; ++t) __nanosleep(1000);
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 1) {
        tcgen05_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Both kinds of blocks in one launch, the kind whose blocks take longer first: its last wave is filled with the other kind's.
// Ds: how the scores' gradients are written, where they are.
template <int kD, bool kBias, typename Ds>
__global__ void __launch_bounds__(kAbThreads, 1)
attn_bwd_sm100_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmG,
                      const __grid_constant__ CUtensorMap tmBias, const __grid_constant__ AttnBwdParams bp) {
    const int first = bp.w.q_first ? bp.w.q_blocks : bp.w.kv_blocks;
    const bool second = (int)blockIdx.x >= first;
    const int block = second ? (int)blockIdx.x - first : (int)blockIdx.x;
    if (second != (bp.w.q_first != 0)) attn_dq_block<kD, kBias, Ds>(tmQ, tmK, tmV, tmG, tmBias, bp, block);
    else attn_dkv_block<kD, kBias>(tmQ, tmK, tmV, tmG, tmBias, bp, block);
}

}  // namespace trimul

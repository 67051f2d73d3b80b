// Cross attention, forward, on the tensor cores (bf16) for head dimensions of 72 to 128, and what the tensor-core kernels
// share.  Narrower heads: attn_fwd64_sm100.cuh.
//
// One pass over the keys with a running maximum and sum: S = Q K^T and O += P V are tcgen05.mma with accumulators in
// tensor memory, P goes back to tensor memory as the A operand of the second product and never touches shared memory.
// A block owns two tiles of 128 queries of one head.  While the softmax warps of one tile exponentiate, the tensor cores
// work for the other.  384 threads:
//   warp 0      TMA producer: queries once, then key and value tiles of 128 rows through one ring of slots.  What tells that a
//               tile has come belongs to the tile, not to its slot: the ring is odd, so a slot holds keys and values in turn,
//               and a warp that waits for the values alone would miss a phase of a slot's barrier.  Where the key tile before
//               them came late, it would take the open phase's predecessor for the one that it waits for
//   warp 1      UMMA issuer (a second one, a warp per query tile, made it 15 % slower)
//   warp 2      with a key mask: zeroes the value rows of masked keys in shared memory, whose probabilities are zero but
//               which may hold infinities or NaN
//   warp 3      TMA producer of the bias tiles [128 queries][128 keys], one buffer per query tile
//   warps 4-7, 8-11   softmax of one query tile each: a thread owns a row
// The running maximum a row is scaled by lags behind the true one by up to 2^8: O is rescaled only when a row's maximum
// has grown by more (accumulators and sums are fp32, where a common factor of 2^8 costs nothing).
// Tensor memory is full: S of both tiles [0, 256), O of both from 256.  P overlays the first half of its own S, and the next
// scores follow the product that reads P (tcgen05.mma of one thread run in the order of issue, so they cannot overtake it).
// P is handed over in halves of 64 keys, so that its product starts while the rest is exponentiated.
// What bounds it: softmax, product and next scores of a query tile wait for each other (3500 cycles a round for both tiles, of
// which the tensor cores work 2100 and the exponentials 2048), and blocks of 256 queries: 4096 x 8192 with 16 heads of 128 is
// 256 blocks for 148 SMs.  268 us there in a call by itself, 1026 TFLOP/s (0.62 of the measured GEMM rate); 281 in a row of calls.
// Softmax by two warps per row (each half the keys) measured the same.
// Head dimensions below 128 are filled with zeros by the TMA loads.
#pragma once

#include "attn_common.cuh"

namespace trimul {

constexpr int kAfThreads = 384;
constexpr int kAfRows = 128;                     // rows of a query or key tile
constexpr int kAfSub = 128 * 128;                // 128 rows x 64 bf16, swizzled
constexpr int kAfClean = 4;                      // at least the key (the value) tiles that the ring holds at once
constexpr int kStageIdAttnFwd = 11;
constexpr int kAfD = 128;                        // columns of head dimension
constexpr float kAfSlack = 8.f;                  // log2 of what a row's maximum may grow without a rescale

template <bool kBias>
struct AfLayout {
    static constexpr int kTile = 2 * kAfSub;                              // one query, key or value tile
    static constexpr int kStages = kBias ? 3 : 5;
    static_assert((kStages + 1) / 2 <= kAfClean, "a value tile must be consumed before its barrier is used again");
    static constexpr int kOffBias = 2 * kTile;
    static constexpr int kOffRing = kOffBias + (kBias ? 2 * 2 * kAfSub : 0);
    static constexpr int kOffBars = kOffRing + kStages * kTile;
    static constexpr int kSmem = kOffBars + 256;
    static_assert((14 + kStages + 3 * kAfClean) * 8 + 8 <= 256, "barriers");
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

struct AttnFwdParams {
    AttnParams a;
    int n_tiles;                 // key tiles without a mask
    int splits, tiles_per_split; // over the (kept) key tiles
    const uint32_t* words;       // key mask as bits, 4 words a tile, [B][n_tiles][4], or null
    const int* list;             // [B][n_tiles + 1]: number of tiles with a kept key, then those tiles
    float* part_o;               // splits > 1: [splits][B][H][Lq][D] sums, not yet divided
    float2* part_ml;             //             [splits][B][H][Lq]: maximum and sum
    int bias_b1, bias_h1;        // bias shared along the batch / the heads
};

__device__ __forceinline__ uint4 tail_words(int left) {      // bits of the first `left` of 128 keys
    auto w = [](int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; };
    return make_uint4(w(left), w(left - 32), w(left - 64), w(left - 96));
}

template <bool kBias>
__global__ void __launch_bounds__(kAfThreads, 1)
attn_fwd_sm100_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmBias,
                      const __grid_constant__ AttnFwdParams fp) {
    using L = AfLayout<kBias>;
    constexpr int kD = kAfD;
    const AttnParams& p = fp.a;
    constexpr int kSt = L::kStages;
    extern __shared__ __align__(1024) uint8_t smem[];
    if ((smem_u32(smem) & 1023u) != 0u) {
        if (threadIdx.x == 0) report_timeout(p.status, kStageIdAttnFwd, 900);
        return;
    }
    uint8_t* sQ = smem;
    uint8_t* sBias = smem + L::kOffBias;
    uint8_t* ring = smem + L::kOffRing;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBars);
    uint64_t* q_full = bars;                   // [2]
    uint64_t* s_full = q_full + 2;             // [2] scores of a key tile complete
    uint64_t* p_full = s_full + 2;             // [2][2] half of the probabilities in tensor memory, O rescaled where it had to be
    uint64_t* o_full = p_full + 4;             // [2] last product complete
    uint64_t* b_full = o_full + 2;             // [2]
    uint64_t* b_empty = b_full + 2;            // [2]
    uint64_t* empty = b_empty + 2;             // [kSt]
    uint64_t* k_full = empty + kSt;            // [kAfClean] key tile j at j % kAfClean, and so
    uint64_t* v_full = k_full + kAfClean;      // [kAfClean] value tile j
    uint64_t* v_ok = v_full + kAfClean;        // [kAfClean] its masked rows zeroed
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_ok + kAfClean);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = warp_uniform((int)threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int i0 = blockIdx.x * 2 * kAfRows, h = blockIdx.y, b = blockIdx.z / fp.splits, split = blockIdx.z % fp.splits;
    const int hk = h / (p.H / p.Hk);
    const bool two = i0 + kAfRows < p.Lq;

    if (threadIdx.x == 0) {
        for (int w = 0; w < 2; ++w) {
            mbar_init(&q_full[w], 1);
            mbar_init(&s_full[w], 1);
            mbar_init(&p_full[2 * w], 4);
            mbar_init(&p_full[2 * w + 1], 4);
            mbar_init(&o_full[w], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&b_full[s], 1);
            mbar_init(&b_empty[s], 4);
        }
        for (int s = 0; s < kSt; ++s) mbar_init(&empty[s], 1);
        for (int s = 0; s < kAfClean; ++s) {
            mbar_init(&k_full[s], 1);
            mbar_init(&v_full[s], 1);
            mbar_init(&v_ok[s], 1);
        }
        *abort_flag = 0;
        fence_mbarrier_init();
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
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
    griddep_wait();
    griddep_launch_dependents();

    // the key tiles of this block
    const int* list = fp.list != nullptr ? fp.list + (long long)b * (fp.n_tiles + 1) : nullptr;
    const int kept = warp_uniform(list != nullptr ? list[0] : fp.n_tiles);
    const int t_first = split * fp.tiles_per_split;
    const int n = max(0, min(fp.tiles_per_split, kept - t_first));
    auto tile_at = [&](int j) { return list != nullptr ? at_load(list + 1 + t_first + j) : t_first + j; };

    if (warp == 0) {
        if (lane == 0 && n > 0) {
            auto load_q = [&](int w) {
                mbar_arrive_expect_tx(&q_full[w], L::kTile);
#pragma unroll
                for (int s = 0; s < kD / 64; ++s)
                    tma_load_4d(sQ + w * L::kTile + s * kAfSub, &tmQ, &q_full[w], s * 64, i0 + w * kAfRows, h, b);
            };
            load_q(0);
            for (int it = 0; it < 2 * n; ++it) {
                const int s = it % kSt;
                if (!mbar_wait<true>(&empty[s], ((it / kSt) & 1) ^ 1, abort_flag, p.status, kStageIdAttnFwd, 100 + s)) break;
                uint64_t* full = ((it & 1) ? v_full : k_full) + (it >> 1) % kAfClean;
                mbar_arrive_expect_tx(full, L::kTile);
                const int j0 = tile_at(it >> 1) * kAfRows;
#pragma unroll
                for (int u = 0; u < kD / 64; ++u)
                    tma_load_4d(ring + s * L::kTile + u * kAfSub, (it & 1) ? &tmV : &tmK, full, u * 64, j0, hk, b);
                if (it == 0 && two) load_q(1);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (n > 0) {
            const int tiles = two ? 2 : 1;
            constexpr uint32_t idesc_s = umma_idesc_bf16(128, 128);
            constexpr uint32_t idesc_o = umma_idesc_bf16(128, kD, 0, 1);
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t ph, int detail) {
                ok = ok && warp_wait(bar, ph, lane, abort_flag, p.status, kStageIdAttnFwd, detail);
                tcgen05_fence_after();
                return ok;
            };
            const uint64_t dq = umma_smem_desc_sw128(smem_u32(sQ)), dk = umma_smem_desc_sw128(smem_u32(ring));
            const uint64_t dv = umma_smem_desc_mn_sw128(smem_u32(ring), kAfSub, 1024);
            auto scores = [&](int w, int slot) {         // S_w = Q_w K^T, K in ring slot `slot`
                const uint64_t a = dq + (uint64_t)(w * (L::kTile >> 4)), k = dk + (uint64_t)(slot * (L::kTile >> 4));
#pragma unroll
                for (int kk = 0; kk < kD / 16; ++kk) {
                    const uint64_t off = ((kk >> 2) * kAfSub + (kk & 3) * 32) >> 4;
                    umma_ss_warp(tmem + w * 128, a + off, k + off, idesc_s, kk > 0);
                }
                umma_commit_warp(&s_full[w]);
            };
            auto mix = [&](int w, int slot, int half, bool add) {     // O_w += P_w V over 64 keys
                const uint64_t v = dv + (uint64_t)(slot * (L::kTile >> 4));
                const uint32_t pt = tmem + w * 128;
#pragma unroll
                for (int kk = 4 * half; kk < 4 * half + 4; ++kk)
                    umma_ts_warp(tmem + 256 + w * kD, pt + kk * 8, v + ((kk * 2048) >> 4), idesc_o, add || kk > 0);
            };
            // ring position of the key tile that is next, and of the value tile
            int sk = 0, sv = 1 % kSt;
            auto step = [&](int& slot) {
                slot += 2;
                if (slot >= kSt) slot -= kSt;
            };
            if (wait(&k_full[0], 0, 300)) {
                for (int w = 0; ok && w < tiles; ++w)
                    if (wait(&q_full[w], 0, 310 + w)) scores(w, 0);
                umma_commit_warp(&empty[0]);
            }
            step(sk);
            uint64_t* v_ready = fp.words != nullptr ? v_ok : v_full;
            for (int j = 0; ok && j < n; ++j) {
                const bool more = j + 1 < n;
                wait(&v_ready[j % kAfClean], (j / kAfClean) & 1, 320);
                for (int w = 0; ok && w < tiles; ++w) {
                    for (int half = 0; half < 2; ++half)
                        if (wait(&p_full[2 * w + half], j & 1, 330 + w)) mix(w, sv, half, j > 0);
                    if (!ok) break;
                    if (!more) umma_commit_warp(&o_full[w]);
                    if (w == tiles - 1) umma_commit_warp(&empty[sv]);
                    if (more) {
                        if (w == 0 && !wait(&k_full[(j + 1) % kAfClean], ((j + 1) / kAfClean) & 1, 340)) break;
                        scores(w, sk);
                        if (w == tiles - 1) umma_commit_warp(&empty[sk]);
                    }
                }
                step(sk);
                step(sv);
            }
        }
    } else if (warp == 2) {
        if (fp.words != nullptr) {
            for (int j = 0; j < n; ++j) {
                const int s = (2 * j + 1) % kSt, t = tile_at(j);
                const uint4 w4 = at_load(reinterpret_cast<const uint4*>(fp.words) + (long long)b * fp.n_tiles + t);
                if (!warp_wait(&v_full[j % kAfClean], (j / kAfClean) & 1, lane, abort_flag, p.status, kStageIdAttnFwd, 500 + s)) break;
                if ((w4.x & w4.y & w4.z & w4.w) != 0xffffffffu) {
                    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
                    uint8_t* v = ring + s * L::kTile;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        // eight lanes clear a row's 128 bytes, four rows at a time
                        for (int r = lane >> 3; r < 32; r += 4)
                            if (((w[k] >> r) & 1u) == 0u)
#pragma unroll
                                for (int u = 0; u < kD / 64; ++u)
                                    *reinterpret_cast<uint4*>(v + u * kAfSub + (k * 32 + r) * 128 + (lane & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_ok[j % kAfClean]);
            }
        }
    } else if (warp == 3) {
        if (kBias && lane == 0) {
            bool ok = true;
            for (int j = 0; ok && j < n; ++j) {
                const int j0 = tile_at(j) * kAfRows;
                for (int w = 0; ok && w < (two ? 2 : 1); ++w) {
                    ok = mbar_wait<true>(&b_empty[w], (j & 1) ^ 1, abort_flag, p.status, kStageIdAttnFwd, 600 + w);
                    if (!ok) break;
                    mbar_arrive_expect_tx(&b_full[w], 2 * kAfSub);
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        tma_load_4d(sBias + (w * 2 + u) * kAfSub, &tmBias, &b_full[w], j0 + u * 64, i0 + w * kAfRows,
                                    fp.bias_h1 ? 0 : h, fp.bias_b1 ? 0 : b);
                }
            }
        }
        __syncwarp();
    } else {
        const int w = (warp - 4) >> 2, q = warp & 3, row = q * 32 + lane, i = i0 + w * kAfRows + row;
        if (w == 0 || two) {
            const uint32_t lane_off = (uint32_t)(q * 32) << 16;
            const uint32_t tS = tmem + w * 128 + lane_off;
            const uint32_t tP = tS, tO = tmem + 256 + w * kD + lane_off;
            // scores are kept in units of which `mul` makes base-2 exponents: raw products, or with a bias (or a scale that is
            // not positive) what they come to
            const float c2 = p.scale * kLog2e;
            const bool raw = !kBias && c2 > 0.f;
            const float mul = kBias ? kLog2e : raw ? c2 : 1.f;
            const float unit = kBias ? 1.f : raw ? p.scale : 0.6931471805599453f;
            const float slack = kAfSlack / mul;
            float m = -INFINITY, l = 0.f;
            bool ok = true;
            for (int j = 0; j < n; ++j) {
                const int t = tile_at(j);
                uint4 w4 = make_uint4(~0u, ~0u, ~0u, ~0u);
                if (fp.words != nullptr) w4 = at_load(reinterpret_cast<const uint4*>(fp.words) + (long long)b * fp.n_tiles + t);
                else if ((t + 1) * kAfRows > p.Lk) w4 = tail_words(p.Lk - t * kAfRows);
                if (!(ok = warp_wait(&s_full[w], j & 1, lane, abort_flag, p.status, kStageIdAttnFwd, 400 + w))) break;
                tcgen05_fence_after();
                uint32_t s[4][32];
#pragma unroll
                for (int k = 0; k < 4; ++k) tmem_ld_32x32(tS + 32 * k, s[k]);
                tmem_ld_wait();
                if constexpr (kBias) {
                    if (!(ok = warp_wait(&b_full[w], j & 1, lane, abort_flag, p.status, kStageIdAttnFwd, 410 + w))) break;
                    const f32x2 sc = f2_pack(p.scale, p.scale);
                    const uint8_t* br = sBias + w * 2 * kAfSub + row * 128;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint4 v = *reinterpret_cast<const uint4*>(br + (k >> 1) * kAfSub + ((((k & 1) * 4 + e) ^ (row & 7)) << 4));
                            const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int g = 0; g < 4; ++g) {
                                float lo, hi;
                                f2_unpack(f2_fma(f2_pack(__uint_as_float(s[k][e * 8 + 2 * g]), __uint_as_float(s[k][e * 8 + 2 * g + 1])), sc,
                                                 f2_from_bf16x2(u[g])), lo, hi);
                                s[k][e * 8 + 2 * g] = __float_as_uint(lo);
                                s[k][e * 8 + 2 * g + 1] = __float_as_uint(hi);
                            }
                        }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&b_empty[w]);
                } else if (!raw) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int e = 0; e < 32; ++e) s[k][e] = __float_as_uint(__uint_as_float(s[k][e]) * c2);
                }
                if ((w4.x & w4.y & w4.z & w4.w) != 0xffffffffu) {
                    const uint32_t wk[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (((wk[k] >> e) & 1u) == 0u) s[k][e] = 0xff800000u;
                }
                float mx[4] = {m, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 32; e += 2)
#pragma unroll
                    for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], __uint_as_float(s[k][e]), __uint_as_float(s[k][e + 1]));
                const float mn = max3(mx[0], mx[1], fmaxf(mx[2], mx[3]));
                const bool grow = mn > m + slack;
                const float f = j > 0 && grow ? ex2f((m - mn) * mul) : 1.f;
                if (j == 0 || grow) m = mn;
                const bool rescale = j > 0 && __any_sync(0xffffffffu, grow);
                l *= f;
                const float base = m == -INFINITY ? 0.f : m;
                f32x2 sum[2] = {0ull, 0ull};
                const f32x2 mul2 = f2_pack(mul, mul), off2 = f2_pack(-base * mul, -base * mul), nb2 = f2_pack(-base, -base);
                // these scores were issued after the product of the tile before: O and P may change
                if (rescale) {
#pragma unroll 1
                    for (int cc = 0; cc < kD; cc += 16) {
                        uint32_t o[16];
                        tmem_ld_32x16(tO + cc, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st_32x16(tO + cc, o);
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const f32x2 x = f2_pack(__uint_as_float(s[k][2 * e]), __uint_as_float(s[k][2 * e + 1]));
                        float a, d;
                        f2_unpack(kBias ? f2_mul(f2_add(x, nb2), mul2) : f2_fma(x, mul2, off2), a, d);
                        a = ex2f(a);
                        d = ex2f(d);
                        sum[e & 1] = f2_add(sum[e & 1], f2_pack(a, d));
                        pk[e] = pack_bf16x2(a, d);
                    }
                    tmem_st_32x16(tP + 16 * k, pk);
                    if (k & 1) {             // half of the keys: the product with their values can start
                        tmem_st_wait();
                        tcgen05_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&p_full[2 * w + (k >> 1)]);
                    }
                }
                l += f2_hsum(f2_add(sum[0], sum[1]));
            }
            if (n > 0 && ok) ok = warp_wait(&o_full[w], 0, lane, abort_flag, p.status, kStageIdAttnFwd, 420 + w);
            tcgen05_fence_after();
            if (ok) {
                const bool nothing = l == 0.f;                // no kept key; NaN is none of these
                const float inv = nothing ? 0.f : 1.f / l;
                const bool live = i < p.Lq;
                const long long srow = ((long long)b * p.H + h) * p.Lq + i;
                if (fp.splits > 1) {
                    const long long prow = ((long long)split * p.B * p.H) * p.Lq + srow;
                    if (live) fp.part_ml[prow] = make_float2(nothing ? -INFINITY : m * unit, l);
#pragma unroll 1
                    for (int cc = 0; cc < kD; cc += 16) {
                        if (cc >= p.D) break;
                        uint32_t o[16];
                        if (n > 0) {
                            tmem_ld_32x16(tO + cc, o);
                            tmem_ld_wait();
                        }
                        if (live) {
                            float4* dst = reinterpret_cast<float4*>(fp.part_o + prow * p.D + cc);
#pragma unroll
                            for (int g = 0; g < 4; ++g)
                                if (cc + 4 * g < p.D)
                                    dst[g] = nothing ? make_float4(0.f, 0.f, 0.f, 0.f)
                                                     : make_float4(__uint_as_float(o[4 * g]), __uint_as_float(o[4 * g + 1]),
                                                                   __uint_as_float(o[4 * g + 2]), __uint_as_float(o[4 * g + 3]));
                        }
                    }
                } else {
                    if (live && p.stats != nullptr) p.stats[srow] = nothing ? make_float2(0.f, INFINITY) : make_float2(m * unit, log2f(l));
                    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.o.p) + b * p.o.b + (long long)i * p.o.l + h * p.o.h;
                    __nv_bfloat16* lo = p.o_lo != nullptr ? static_cast<__nv_bfloat16*>(p.o_lo) + (((long long)b * p.Lq + i) * p.H + h) * p.D : nullptr;
#pragma unroll 1
                    for (int cc = 0; cc < kD; cc += 16) {
                        if (cc >= p.D) break;
                        uint32_t o[16];
                        if (n > 0) {
                            tmem_ld_32x16(tO + cc, o);
                            tmem_ld_wait();
                        }
                        if (live) {
#pragma unroll
                            for (int g = 0; g < 2; ++g) {
                                if (cc + 8 * g >= p.D) break;
                                uint32_t y[4], z[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const float a = nothing ? 0.f : __uint_as_float(o[8 * g + 2 * e]) * inv;
                                    const float d = nothing ? 0.f : __uint_as_float(o[8 * g + 2 * e + 1]) * inv;
                                    y[e] = pack_bf16x2(a, d);
                                    z[e] = pack_bf16x2(a - bf16_lo(y[e]), d - bf16_hi(y[e]));
                                }
                                *reinterpret_cast<uint4*>(dst + cc + 8 * g) = make_uint4(y[0], y[1], y[2], y[3]);
                                if (lo != nullptr) *reinterpret_cast<uint4*>(lo + cc + 8 * g) = make_uint4(z[0], z[1], z[2], z[3]);
                            }
                        }
                    }
                }
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

// Joins the parts of a row, a warp per row.  Lane s holds the weight of part s (and of s + 32, ...: all blocks of a row fit
// into a wave, so there are a few hundred parts at most).
template <typename T>
__global__ void __launch_bounds__(256)
attn_combine_kernel(const __grid_constant__ AttnParams p, const float* part_o, const float2* part_ml, int splits) {
    griddep_wait();
    griddep_launch_dependents();
    const long long rows = (long long)p.B * p.H * p.Lq;
    const long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (r >= rows) return;
    const int lane = threadIdx.x & 31;
    float m = -INFINITY;
    for (int s = lane; s < splits; s += 32) m = fmaxf(m, at_load(part_ml + s * rows + r).x);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f, y[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = 0.f;
    for (int s0 = 0; s0 < splits; s0 += 32) {
        const float2 ml = s0 + lane < splits ? at_load(part_ml + (s0 + lane) * rows + r) : make_float2(-INFINITY, 0.f);
        const float w = ex2f((ml.x - base) * kLog2e);
        l = fmaf(ml.y, w, l);
        const int n = min(32, splits - s0);
#pragma unroll
        for (int k = 0; k < 8; ++k) {           // columns lane + 32 k
            const int d = lane + 32 * k;
            if (32 * k >= p.D) break;
            const float* o = part_o + (s0 * rows + r) * p.D + min(d, p.D - 1);
#pragma unroll 8
            for (int s = 0; s < n; ++s) y[k] = fmaf(at_load(o + s * rows * p.D), __shfl_sync(0xffffffffu, w, s), y[k]);
        }
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    const bool nothing = l == 0.f;
    const float inv = nothing ? 0.f : 1.f / l;
    const int i = (int)(r % p.Lq), h = (int)((r / p.Lq) % p.H), b = (int)(r / p.Lq / p.H);
    if (lane == 0 && p.stats != nullptr) p.stats[r] = nothing ? make_float2(0.f, INFINITY) : make_float2(m, log2f(l));
    T* dst = static_cast<T*>(p.o.p) + b * p.o.b + (long long)i * p.o.l + h * p.o.h;
    const long long lo = (((long long)b * p.Lq + i) * p.H + h) * p.D;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int d = lane + 32 * k;
        if (d >= p.D) break;
        const float v = nothing ? 0.f : y[k] * inv;
        at_store(dst + d, v);
        if constexpr (sizeof(T) == 2) {
            if (p.o_lo != nullptr)
                static_cast<__nv_bfloat16*>(p.o_lo)[lo + d] = __float2bfloat16_rn(v - __bfloat162float(__float2bfloat16_rn(v)));
        }
    }
}

}  // namespace trimul

// Cross attention, forward, on the tensor cores for head dimensions up to 64.
//
// With 64 columns of head dimension the exponentials (16 per cycle and SM) take longer than the products, so what counts is
// that they never pause.  A block owns two tiles of 128 queries and runs FOUR chains of scores -> softmax -> P V: (query
// tile w, half p of every tile of 128 keys), each with its own softmax warps (a thread owns a row), its own running maximum
// and sum and its own O in tensor memory; while one chain loads scores or waits for its products, the other three
// exponentiate.  At the end the two chains of a query tile are joined through shared memory.  Two chains over whole key
// tiles (as for wider heads) left the exponentials idle for two fifths of the time: 71 us instead of 62 for 2048 x 4096,
// 18 heads of 64.
// 640 threads: warp 0 TMA producer, warps 1 and 3 UMMA issuers of query tiles 0 and 1 (one warp for all four chains was busy
// for longer than the exponentials take), warp 2 cleans value rows of masked keys, warps 4 + 4 c ... the softmax warps of
// chain c = 2 p + w.
// Tensor memory of chain c: S (64 columns, P overlays the first 32) at 128 c, O (64 columns) after it.  The next scores of a
// chain are issued after the product that reads its P, and tcgen05.mma of one thread run in the order of issue.
#pragma once

#include "attn_fwd_sm100.cuh"

namespace trimul {

constexpr int kA6Threads = 640;
constexpr int kStageIdAttnFwd64 = 14;

template <bool kBias>
struct A6Layout {
    static constexpr int kTile = kAfSub;                                  // [128 rows][64] bf16
    static constexpr int kBiasBufs = kBias ? 2 : 0;                       // per chain, [128 queries][64 keys] each
    static constexpr int kStages = kBias ? 4 : 6;
    static constexpr int kOffBias = 2 * kTile;
    // the second half's chains leave their O here: 32 KB each, with a bias in their own bias buffers
    static constexpr int kOffRing = kOffBias + (kBias ? 4 * kBiasBufs * kTile : 4 * kTile);
    static constexpr int kOffBars = kOffRing + kStages * kTile;
    static constexpr int kBars = 2 + 3 * 4 + 2 + 4 * 4 + 2 * kStages + kAfClean;
    static constexpr int kOffJoin = kOffBars + (8 * kBars + 8 + 127) / 128 * 128;      // (m, l) of those chains' rows
    static constexpr int kSmem = kOffJoin + 2 * kAfRows * 8;
    static_assert((kStages + 1) / 2 <= kAfClean, "a value tile must be consumed before its barrier is used again");
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

template <bool kBias>
__global__ void __launch_bounds__(kA6Threads, 1)
attn_fwd64_sm100_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                        const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmBias,
                        const __grid_constant__ AttnFwdParams fp) {
    using L = A6Layout<kBias>;
    const AttnParams& p = fp.a;
    constexpr int kSt = L::kStages, kBb = kBias ? L::kBiasBufs : 1;
    extern __shared__ __align__(1024) uint8_t smem[];
    if ((smem_u32(smem) & 1023u) != 0u) {
        if (threadIdx.x == 0) report_timeout(p.status, kStageIdAttnFwd64, 900);
        return;
    }
    uint8_t* sQ = smem;
    uint8_t* sBias = smem + L::kOffBias;
    uint8_t* ring = smem + L::kOffRing;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBars);
    uint64_t* q_full = bars;                   // [2]
    uint64_t* s_full = q_full + 2;             // [4] scores of a chain's next half tile complete
    uint64_t* p_full = s_full + 4;             // [4] its probabilities in tensor memory, O rescaled where it had to be
    uint64_t* o_full = p_full + 4;             // [4] its last product complete
    uint64_t* join = o_full + 4;               // [2] the second half's O, maxima and sums are in shared memory
    uint64_t* b_full = join + 2;               // [4][2]
    uint64_t* b_empty = b_full + 8;            // [4][2]
    uint64_t* full = b_empty + 8;              // [kSt]
    uint64_t* empty = full + kSt;              // [kSt]
    uint64_t* v_ok = empty + kSt;              // [kAfClean] masked value rows zeroed, value tile j at j % kAfClean
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_ok + kAfClean);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float2* join_ml = reinterpret_cast<float2*>(smem + L::kOffJoin);       // [2][128]

    const int warp = warp_uniform((int)threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int i0 = blockIdx.x * 2 * kAfRows, h = blockIdx.y, b = blockIdx.z / fp.splits, split = blockIdx.z % fp.splits;
    const int hk = h / (p.H / p.Hk);
    const bool two = i0 + kAfRows < p.Lq;

    if (threadIdx.x == 0) {
        for (int w = 0; w < 2; ++w) {
            mbar_init(&q_full[w], 1);
            mbar_init(&join[w], 4);
        }
        for (int c = 0; c < 4; ++c) {
            mbar_init(&s_full[c], 1);
            mbar_init(&p_full[c], 4);
            mbar_init(&o_full[c], 1);
        }
        for (int s = 0; s < 8; ++s) {
            mbar_init(&b_full[s], 1);
            mbar_init(&b_empty[s], 4);
        }
        for (int s = 0; s < kSt; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], two ? 2 : 1);       // one commit per issuer
        }
        for (int s = 0; s < kAfClean; ++s) mbar_init(&v_ok[s], 1);
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

    const int* list = fp.list != nullptr ? fp.list + (long long)b * (fp.n_tiles + 1) : nullptr;
    const int kept = warp_uniform(list != nullptr ? list[0] : fp.n_tiles);
    const int t_first = split * fp.tiles_per_split;
    const int n = max(0, min(fp.tiles_per_split, kept - t_first));
    auto tile_at = [&](int j) { return list != nullptr ? at_load(list + 1 + t_first + j) : t_first + j; };

    if (warp == 0) {
        if (lane == 0 && n > 0) {
            auto load_q = [&](int w) {
                mbar_arrive_expect_tx(&q_full[w], L::kTile);
                tma_load_4d(sQ + w * L::kTile, &tmQ, &q_full[w], 0, i0 + w * kAfRows, h, b);
            };
            load_q(0);
            for (int it = 0; it < 2 * n; ++it) {
                const int s = it % kSt;
                if (!mbar_wait<true>(&empty[s], ((it / kSt) & 1) ^ 1, abort_flag, p.status, kStageIdAttnFwd64, 100 + s)) break;
                mbar_arrive_expect_tx(&full[s], L::kTile);
                tma_load_4d(ring + s * L::kTile, (it & 1) ? &tmV : &tmK, &full[s], 0, tile_at(it >> 1) * kAfRows, hk, b);
                if (it == 0 && two) load_q(1);
                if (kBias && (it & 1) == 0) {            // the chains' bias tiles between keys and values
                    const int j = it >> 1, buf = j % kBb;
                    bool ok = true;
                    for (int c = 0; ok && c < 4; ++c) {
                        if ((c & 1) != 0 && !two) continue;
                        ok = mbar_wait<true>(&b_empty[c * 2 + buf], ((j / kBb) & 1) ^ 1, abort_flag, p.status, kStageIdAttnFwd64, 600 + c);
                        if (!ok) break;
                        mbar_arrive_expect_tx(&b_full[c * 2 + buf], L::kTile);
                        tma_load_4d(sBias + (c * kBb + buf) * L::kTile, &tmBias, &b_full[c * 2 + buf], tile_at(j) * kAfRows + (c >> 1) * 64,
                                    i0 + (c & 1) * kAfRows, fp.bias_h1 ? 0 : h, fp.bias_b1 ? 0 : b);
                    }
                    if (!ok) break;
                }
            }
        }
        __syncwarp();
    } else if (warp == 1 || warp == 3) {
        const int w = warp == 3;
        if (n > 0 && (w == 0 || two)) {
            constexpr uint32_t idesc_s = umma_idesc_bf16(128, 64);
            constexpr uint32_t idesc_o = umma_idesc_bf16(128, 64, 0, 1);
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t ph, int detail) {
                ok = ok && warp_wait(bar, ph, lane, abort_flag, p.status, kStageIdAttnFwd64, detail);
                tcgen05_fence_after();
                return ok;
            };
            const uint64_t dq = umma_smem_desc_sw128(smem_u32(sQ + w * L::kTile)), dk = umma_smem_desc_sw128(smem_u32(ring));
            const uint64_t dv = umma_smem_desc_mn_sw128(smem_u32(ring), kAfSub, 1024);
            constexpr uint64_t kHalf = (64 * 128) >> 4;          // 64 rows of a tile
            auto scores = [&](int half, int slot) {
                const uint64_t k = dk + (uint64_t)(slot * (L::kTile >> 4)) + half * kHalf;
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    umma_ss_warp(tmem + (2 * half + w) * 128, dq + kk * kDescKStep, k + kk * kDescKStep, idesc_s, kk > 0);
                umma_commit_warp(&s_full[2 * half + w]);
            };
            auto mix = [&](int half, int slot, bool add) {
                const uint64_t v = dv + (uint64_t)(slot * (L::kTile >> 4)) + half * kHalf;
                const uint32_t t = tmem + (2 * half + w) * 128;
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) umma_ts_warp(t + 64, t + kk * 8, v + ((kk * 2048) >> 4), idesc_o, add || kk > 0);
            };
            int sk = 0, sv = 1;                 // ring position of the next key tile, and of the value tile
            uint32_t phk = 0, phv = 0;
            auto step = [&](int& slot, uint32_t& ph) {
                slot += 2;
                if (slot >= kSt) { slot -= kSt; ph ^= 1u; }
            };
            if (wait(&full[0], 0, 300) && wait(&q_full[w], 0, 310 + w)) {
                scores(0, 0);
                scores(1, 0);
                umma_commit_warp(&empty[0]);
            }
            step(sk, phk);
            for (int j = 0; ok && j < n; ++j) {
                const bool more = j + 1 < n;
                if (fp.words != nullptr) wait(&v_ok[j % kAfClean], (j / kAfClean) & 1, 320);
                else wait(&full[sv], phv, 321);
                if (more) wait(&full[sk], phk, 340);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (!wait(&p_full[2 * half + w], j & 1, 330 + 2 * half + w)) break;
                    mix(half, sv, j > 0);
                    if (more) scores(half, sk);
                    else umma_commit_warp(&o_full[2 * half + w]);
                }
                if (!ok) break;
                umma_commit_warp(&empty[sv]);
                if (more) umma_commit_warp(&empty[sk]);
                step(sk, phk);
                step(sv, phv);
            }
        }
    } else if (warp == 2) {
        if (fp.words != nullptr) {
            for (int j = 0; j < n; ++j) {
                const int s = (2 * j + 1) % kSt, t = tile_at(j);
                const uint4 w4 = at_load(reinterpret_cast<const uint4*>(fp.words) + (long long)b * fp.n_tiles + t);
                if (!warp_wait(&full[s], ((2 * j + 1) / kSt) & 1, lane, abort_flag, p.status, kStageIdAttnFwd64, 500 + s)) break;
                if ((w4.x & w4.y & w4.z & w4.w) != 0xffffffffu) {
                    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
                    uint8_t* v = ring + s * L::kTile;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        for (int r = lane >> 3; r < 32; r += 4)
                            if (((w[k] >> r) & 1u) == 0u)
                                *reinterpret_cast<uint4*>(v + (k * 32 + r) * 128 + (lane & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_ok[j % kAfClean]);
            }
        }
    } else {
        const int c = (warp - 4) >> 2, w = c & 1, half = c >> 1, q = warp & 3, row = q * 32 + lane, i = i0 + w * kAfRows + row;
        if (w == 0 || two) {
            const uint32_t tS = tmem + c * 128 + ((uint32_t)(q * 32) << 16), tO = tS + 64;
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
                uint32_t keep[2] = {~0u, ~0u};
                if (fp.words != nullptr) {
                    const uint2 w2 = at_load(reinterpret_cast<const uint2*>(fp.words) + ((long long)b * fp.n_tiles + t) * 2 + half);
                    keep[0] = w2.x;
                    keep[1] = w2.y;
                } else if ((t + 1) * kAfRows > p.Lk) {
                    const uint4 w4 = tail_words(p.Lk - t * kAfRows);
                    keep[0] = half ? w4.z : w4.x;
                    keep[1] = half ? w4.w : w4.y;
                }
                if (!(ok = warp_wait(&s_full[c], j & 1, lane, abort_flag, p.status, kStageIdAttnFwd64, 400 + c))) break;
                tcgen05_fence_after();
                uint32_t s[2][32];
                tmem_ld_32x32(tS, s[0]);
                tmem_ld_32x32(tS + 32, s[1]);
                tmem_ld_wait();
                if constexpr (kBias) {
                    const int buf = j % kBb;
                    if (!(ok = warp_wait(&b_full[c * 2 + buf], (j / kBb) & 1, lane, abort_flag, p.status, kStageIdAttnFwd64, 410 + c))) break;
                    const f32x2 sc = f2_pack(p.scale, p.scale);
                    const uint8_t* br = sBias + (c * kBb + buf) * L::kTile + row * 128;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint4 v = *reinterpret_cast<const uint4*>(br + ((e ^ (row & 7)) << 4));
                        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            uint32_t* x = &s[e >> 2][(e & 3) * 8 + 2 * g];
                            float lo, hi;
                            f2_unpack(f2_fma(f2_pack(__uint_as_float(x[0]), __uint_as_float(x[1])), sc, f2_from_bf16x2(u[g])), lo, hi);
                            x[0] = __float_as_uint(lo);
                            x[1] = __float_as_uint(hi);
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&b_empty[c * 2 + buf]);
                } else if (!raw) {
#pragma unroll
                    for (int e = 0; e < 64; ++e) s[e >> 5][e & 31] = __float_as_uint(__uint_as_float(s[e >> 5][e & 31]) * c2);
                }
                if ((keep[0] & keep[1]) != 0xffffffffu) {
#pragma unroll
                    for (int e = 0; e < 64; ++e)
                        if (((keep[e >> 5] >> (e & 31)) & 1u) == 0u) s[e >> 5][e & 31] = 0xff800000u;
                }
                float mx[4] = {m, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 64; e += 2)
                    mx[(e >> 1) & 3] = max3(mx[(e >> 1) & 3], __uint_as_float(s[e >> 5][e & 31]), __uint_as_float(s[e >> 5][(e & 31) + 1]));
                const float mn = max3(mx[0], mx[1], fmaxf(mx[2], mx[3]));
                const bool grow = mn > m + slack;
                if (j == 0) {
                    m = mn;
                } else if (__any_sync(0xffffffffu, grow)) {
                    // the product of the half tile before is complete: these scores were issued after it
                    const float f = grow ? ex2f((m - mn) * mul) : 1.f;
                    if (grow) m = mn;
                    l *= f;
#pragma unroll 1
                    for (int cc = 0; cc < 64; cc += 16) {
                        uint32_t o[16];
                        tmem_ld_32x16(tO + cc, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st_32x16(tO + cc, o);
                    }
                }
                const float base = m == -INFINITY ? 0.f : m;
                f32x2 sum[2] = {0ull, 0ull};
                const f32x2 mul2 = f2_pack(mul, mul), off2 = f2_pack(-base * mul, -base * mul), nb2 = f2_pack(-base, -base);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
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
                    tmem_st_32x16(tS + 16 * k, pk);
                }
                l += f2_hsum(f2_add(sum[0], sum[1]));
                tmem_st_wait();
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[c]);
            }
            if (n > 0 && ok) ok = warp_wait(&o_full[c], 0, lane, abort_flag, p.status, kStageIdAttnFwd64, 420 + c);
            tcgen05_fence_after();
            if (ok) {
                float* left = reinterpret_cast<float*>(sBias + (kBias ? (2 + w) * kBb : 2 * w) * L::kTile) + row;     // [64][128]
                if (half == 1) {
                    // column after column, a row per lane: no bank conflicts either way
                    if (n > 0) {
#pragma unroll 1
                        for (int cc = 0; cc < 64; cc += 16) {
                            if (cc >= p.D) break;
                            uint32_t o[16];
                            tmem_ld_32x16(tO + cc, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 16; ++e) left[(cc + e) * kAfRows] = __uint_as_float(o[e]);
                        }
                    }
                    join_ml[w * kAfRows + row] = make_float2(m, l);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&join[w]);
                } else if ((ok = warp_wait(&join[w], 0, lane, abort_flag, p.status, kStageIdAttnFwd64, 440 + w))) {
                    const float2 ml = join_ml[w * kAfRows + row];
                    const float mm = fmaxf(m, ml.x), base = mm == -INFINITY ? 0.f : mm;
                    const float f0 = ex2f((m - base) * mul), f1 = ex2f((ml.x - base) * mul);
                    l = l * f0 + ml.y * f1;
                    const bool nothing = l == 0.f;
                    const float inv = nothing ? 0.f : fp.splits > 1 ? 1.f : 1.f / l;
                    const float g0 = f0 * inv, g1 = f1 * inv;
                    const bool live = i < p.Lq;
                    const long long srow = ((long long)b * p.H + h) * p.Lq + i, prow = (long long)split * p.B * p.H * p.Lq + srow;
                    if (live) {
                        if (fp.splits > 1) fp.part_ml[prow] = make_float2(nothing ? -INFINITY : mm * unit, l);
                        else if (p.stats != nullptr) p.stats[srow] = nothing ? make_float2(0.f, INFINITY) : make_float2(mm * unit, log2f(l));
                    }
                    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.o.p) + b * p.o.b + (long long)i * p.o.l + h * p.o.h;
                    __nv_bfloat16* lo = p.o_lo != nullptr ? static_cast<__nv_bfloat16*>(p.o_lo) + (((long long)b * p.Lq + i) * p.H + h) * p.D : nullptr;
#pragma unroll 1
                    for (int cc = 0; cc < 64; cc += 16) {
                        if (cc >= p.D) break;
                        uint32_t o[16];
                        if (n > 0) {
                            tmem_ld_32x16(tO + cc, o);
                            tmem_ld_wait();
                        }
                        if (!live) continue;
                        float y[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            y[e] = nothing ? 0.f : fmaf(__uint_as_float(o[e]), g0, left[(cc + e) * kAfRows] * g1);
                        if (fp.splits > 1) {
                            float4* part = reinterpret_cast<float4*>(fp.part_o + prow * p.D + cc);
#pragma unroll
                            for (int g = 0; g < 4; ++g)
                                if (cc + 4 * g < p.D) part[g] = make_float4(y[4 * g], y[4 * g + 1], y[4 * g + 2], y[4 * g + 3]);
                        } else {
#pragma unroll
                            for (int g = 0; g < 2; ++g) {
                                if (cc + 8 * g >= p.D) break;
                                uint32_t a[4], z[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    a[e] = pack_bf16x2(y[8 * g + 2 * e], y[8 * g + 2 * e + 1]);
                                    z[e] = pack_bf16x2(y[8 * g + 2 * e] - bf16_lo(a[e]), y[8 * g + 2 * e + 1] - bf16_hi(a[e]));
                                }
                                *reinterpret_cast<uint4*>(dst + cc + 8 * g) = make_uint4(a[0], a[1], a[2], a[3]);
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

}  // namespace trimul

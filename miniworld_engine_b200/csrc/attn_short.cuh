// Cross attention, forward, for few query rows per key head (single tokens): the query rows of all heads that share a
// key head go through its keys and values together, which are read once.
//
// Bound by memory: a key and its value are 4 D bytes for 4 D R operations.  A key row is covered by D / 8 lanes (bf16, 16
// bytes each), so a warp's load takes 32 / (D / 8) keys; a warp takes as_loads of those loads of keys and of values at
// once (all in flight before the first is used), and keeps a running maximum, sum and R rows of output of its own; nothing is
// shared until the end, when the warps of a block, and then the blocks that split the keys, join their parts.
// Masked keys are neither multiplied nor added: their rows may hold anything.
#pragma once

#include "attn_common.cuh"

namespace trimul {

constexpr int kAsThreads = 128;
constexpr int kAsWarps = kAsThreads / 32;
template <int kR> __host__ __device__ constexpr int as_loads() { return kR == 1 ? 8 : 4; }      // what the rows' sums leave registers for
// blocks on an SM at once, by the registers of the rows' sums
__host__ __device__ constexpr int as_blocks(int rows) { return rows <= 1 ? 4 : rows <= 2 ? 5 : rows <= 4 ? 4 : 2; }

struct AttnShortParams {
    AttnParams a;
    int splits, keys_per_split;
    float* part_o;               // splits > 1, as in the tensor-core kernel
    float2* part_ml;
};

template <typename T> struct AsVec;
template <> struct AsVec<__nv_bfloat16> {
    static constexpr int kN = 8;
    static __device__ __forceinline__ void unpack(const uint4& v, f32x2 (&f)[4]) {
        f[0] = f2_from_bf16x2(v.x); f[1] = f2_from_bf16x2(v.y); f[2] = f2_from_bf16x2(v.z); f[3] = f2_from_bf16x2(v.w);
    }
};
template <> struct AsVec<float> {
    static constexpr int kN = 4;
    static __device__ __forceinline__ void unpack(const uint4& v, f32x2 (&f)[2]) {
        f[0] = f2_pack(__uint_as_float(v.x), __uint_as_float(v.y));
        f[1] = f2_pack(__uint_as_float(v.z), __uint_as_float(v.w));
    }
};

// kLanes lanes per key row; kR query rows; grid (splits, Hk, B)
template <typename T, int kLanes, int kR>
__global__ void __launch_bounds__(kAsThreads, as_blocks(kR))
attn_short_kernel(const __grid_constant__ AttnShortParams sp) {
    constexpr int kN = AsVec<T>::kN, kP = kN / 2;
    constexpr int kKeys = 32 / kLanes;                 // keys of one load
    constexpr int kAsLoads = as_loads<kR>();
    constexpr int kChunk = kKeys * kAsLoads;           // keys of one step of a warp
    const AttnParams& p = sp.a;
    __shared__ float2 s_ml[kAsWarps][kR];
    __shared__ float s_o[kAsWarps][kR][kLanes * kN];
    griddep_wait();
    griddep_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / kLanes, dl = lane % kLanes, d0 = dl * kN;
    const int hk = blockIdx.y, b = blockIdx.z, split = blockIdx.x, group = p.H / p.Hk, nr = group * p.Lq;
    const bool in = d0 < p.D;
    auto row = [&](int r, int& h, int& i) {
        const int x = min(r, nr - 1);
        h = hk * group + x / p.Lq;
        i = x % p.Lq;
    };
    const float c2 = p.scale * kLog2e;
    const bool biased = p.bias != nullptr;
    // queries times what makes their products base-2 exponents; with a bias plain scores (a mask of the type's lowest
    // value must not overflow), scaled once the maximum is off
    f32x2 q[kR][kP], o[kR][kP];
    float m[kR], l[kR];
    const T* bias[kR];
#pragma unroll
    for (int r = 0; r < kR; ++r) {
        int h, i;
        row(r, h, i);
        const T* src = static_cast<const T*>(p.q.p) + b * p.q.b + (long long)i * p.q.l + h * p.q.h + d0;
        const float f = biased ? p.scale : c2;
#pragma unroll
        for (int e = 0; e < kP; ++e) {
            q[r][e] = in ? f2_pack(at_float(src[2 * e]) * f, at_float(src[2 * e + 1]) * f) : 0ull;
            o[r][e] = 0ull;
        }
        m[r] = -INFINITY;
        l[r] = 0.f;
        bias[r] = biased ? static_cast<const T*>(p.bias) + b * p.bias_b + h * p.bias_h + (long long)i * p.bias_i : nullptr;
    }
    const float mul = biased ? kLog2e : 1.f, unit = biased ? 1.f : 0.6931471805599453f;
    const T* k = static_cast<const T*>(p.k.p) + b * p.k.b + hk * p.k.h + d0;
    const T* v = static_cast<const T*>(p.v.p) + b * p.v.b + hk * p.v.h + d0;
    const uint8_t* mask = p.mask != nullptr ? p.mask + b * p.mask_b : nullptr;
    const int k_end = min(p.Lk, (split + 1) * sp.keys_per_split);
    // bit u: this lane's key of load u counts
    auto kept = [&](int j0) {
        uint32_t bits = 0;
#pragma unroll
        for (int u = 0; u < kAsLoads; ++u) {
            const int j = j0 + u * kKeys + sub;
            bits |= (uint32_t)(j < k_end && (mask == nullptr || at_load(mask + j) != 0)) << u;
        }
        return bits;
    };
    const int j_first = split * sp.keys_per_split + warp * kChunk;
    uint32_t next = kept(j_first);
    for (int j0 = j_first; j0 < k_end; j0 += kAsWarps * kChunk) {
        const uint32_t keep = next;
        next = kept(j0 + kAsWarps * kChunk);         // a step ahead: the loads below do not wait for the mask
        if (mask != nullptr && __all_sync(0xffffffffu, keep == 0u)) continue;
        uint4 kv[kAsLoads], vv[kAsLoads];
#pragma unroll
        for (int u = 0; u < kAsLoads; ++u) {
            const int j = j0 + u * kKeys + sub;
            kv[u] = vv[u] = make_uint4(0u, 0u, 0u, 0u);
            if (in && ((keep >> u) & 1u)) kv[u] = at_load(reinterpret_cast<const uint4*>(k + (long long)j * p.k.l));
        }
#pragma unroll
        for (int u = 0; u < kAsLoads; ++u) {
            const int j = j0 + u * kKeys + sub;
            if (in && ((keep >> u) & 1u)) vv[u] = at_load(reinterpret_cast<const uint4*>(v + (long long)j * p.v.l));
        }
        float s[kAsLoads][kR];
#pragma unroll
        for (int u = 0; u < kAsLoads; ++u) {
            f32x2 kf[kP];
            AsVec<T>::unpack(kv[u], kf);
#pragma unroll
            for (int r = 0; r < kR; ++r) {
                f32x2 t = f2_mul(q[r][0], kf[0]);
#pragma unroll
                for (int e = 1; e < kP; ++e) t = f2_fma(q[r][e], kf[e], t);
                float x = f2_hsum(t);
#pragma unroll
                for (int w = kLanes / 2; w >= 1; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
                s[u][r] = x;
            }
        }
#pragma unroll
        for (int u = 0; u < kAsLoads; ++u) {
            const bool counts = (keep >> u) & 1u;
#pragma unroll
            for (int r = 0; r < kR; ++r) {
                if (biased && counts) s[u][r] += at_float(bias[r][j0 + u * kKeys + sub]);
                if (!counts) s[u][r] = -INFINITY;
            }
        }
#pragma unroll
        for (int r = 0; r < kR; ++r) {
            float mx = s[0][r];
#pragma unroll
            for (int u = 1; u < kAsLoads; ++u) mx = fmaxf(mx, s[u][r]);
#pragma unroll
            for (int w = 16; w >= kLanes; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
            const float mn = fmaxf(m[r], mx);
            const float base = mn == -INFINITY ? 0.f : mn;
            const float f = ex2f((m[r] - base) * mul);
            m[r] = mn;
            l[r] *= f;
#pragma unroll
            for (int e = 0; e < kP; ++e) o[r][e] = f2_mul(o[r][e], f2_pack(f, f));
#pragma unroll
            for (int u = 0; u < kAsLoads; ++u) {
                s[u][r] = ex2f((s[u][r] - base) * mul);
                l[r] += s[u][r];
            }
        }
#pragma unroll
        for (int u = 0; u < kAsLoads; ++u) {
            f32x2 vf[kP];
            AsVec<T>::unpack(vv[u], vf);
#pragma unroll
            for (int r = 0; r < kR; ++r) {
                const f32x2 w2 = f2_pack(s[u][r], s[u][r]);
#pragma unroll
                for (int e = 0; e < kP; ++e) o[r][e] = f2_fma(w2, vf[e], o[r][e]);
            }
        }
    }
    // the keys of a load lie kLanes lanes apart: every key group has its own sums
#pragma unroll
    for (int r = 0; r < kR; ++r) {
#pragma unroll
        for (int w = 16; w >= kLanes; w >>= 1) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], w);
#pragma unroll
            for (int e = 0; e < kP; ++e) o[r][e] = f2_add(o[r][e], __shfl_xor_sync(0xffffffffu, o[r][e], w));
        }
        if (lane == 0) s_ml[warp][r] = make_float2(m[r], l[r]);
        if (lane < kLanes) {
#pragma unroll
            for (int e = 0; e < kP; ++e) {
                float a, c;
                f2_unpack(o[r][e], a, c);
                s_o[warp][r][d0 + 2 * e] = a;
                s_o[warp][r][d0 + 2 * e + 1] = c;
            }
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < nr * p.D; e += kAsThreads) {
        const int r = e / p.D, d = e % p.D;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < kAsWarps; ++w) mx = fmaxf(mx, s_ml[w][r].x);
        const float base = mx == -INFINITY ? 0.f : mx;
        float sum = 0.f, y = 0.f;
#pragma unroll
        for (int w = 0; w < kAsWarps; ++w) {
            const float f = ex2f((s_ml[w][r].x - base) * mul);
            sum = fmaf(s_ml[w][r].y, f, sum);
            y = fmaf(s_o[w][r][d], f, y);
        }
        int h, i;
        row(r, h, i);
        const bool nothing = sum == 0.f;
        const long long srow = ((long long)b * p.H + h) * p.Lq + i;
        if (sp.splits > 1) {
            const long long prow = (long long)split * p.B * p.H * p.Lq + srow;
            sp.part_o[prow * p.D + d] = nothing ? 0.f : y;
            if (d == 0) sp.part_ml[prow] = make_float2(nothing ? -INFINITY : mx * unit, sum);
        } else {
            y = nothing ? 0.f : y / sum;
            at_store(static_cast<T*>(p.o.p) + b * p.o.b + (long long)i * p.o.l + h * p.o.h + d, y);
            if constexpr (sizeof(T) == 2) {
                if (p.o_lo != nullptr)
                    static_cast<__nv_bfloat16*>(p.o_lo)[(((long long)b * p.Lq + i) * p.H + h) * p.D + d] =
                        __float2bfloat16_rn(y - __bfloat162float(__float2bfloat16_rn(y)));
            }
            if (d == 0 && p.stats != nullptr) p.stats[srow] = nothing ? make_float2(0.f, INFINITY) : make_float2(mx * unit, log2f(sum));
        }
    }
}

}  // namespace trimul

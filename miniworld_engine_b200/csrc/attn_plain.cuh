// Cross attention on the CUDA cores: fp32 inputs, head dimensions that the tensor-core kernels do not take, and the
// cross-check of those kernels.  All arithmetic in fp32.
//
// A block owns kT rows of queries (forward, gradient of q and of the bias) or of keys (gradients of k and v) and walks
// over tiles of kT rows of the other side.  256 threads as 16 x 16; thread (ty, tx) owns rows ty * kR + r and columns
// tx + 16 c of a kT x kT tile of scores, r, c < kR = kT / 16, both operands read from shared memory in four-element
// pieces along the head dimension (pitch D rounded up to 4, plus 4: the sixteen rows that a half warp reads at once then
// lie in different banks).  What bounds it is the shared-memory pipe: 2 kR reads of 16 bytes for 4 kR^2 multiply-adds, and where
// there are few blocks their latency (fp32, 2 x 256 x 320, 8 heads of 32: forward 21 us in 192 blocks of two or fewer steps, backward
// 39 in 144 of four or five).  Backward above 64 columns on 32-row tiles: the accumulators of dk and dv of 64 rows would not fit
// into the registers.
#pragma once

#include "attn_common.cuh"

namespace trimul {

constexpr int kApThreads = 256;

__host__ __device__ inline int ap_pitch(int D) { return (D + 3) / 4 * 4 + 4; }
template <int kT> __host__ __device__ inline int ap_ppitch() { return kT + 4; }
// `tiles` operand tiles and `scores` score tiles of shared memory
template <int kT> inline int ap_smem(int D, int tiles, int scores) {
    return (tiles * kT * ap_pitch(D) + scores * kT * ap_ppitch<kT>() + 3 * kT) * 4;
}

// kT rows of a tensor on their way into shared memory as fp32, with zeros behind the last row, in masked rows and behind
// column D.  `fetch` issues the loads (four consecutive columns a piece where rows allow it), `put` stores what came: between
// the two a tile's loads run behind the arithmetic of the tile before.
template <typename T> struct ApRaw;
template <> struct ApRaw<float> { using V = float4; };
template <> struct ApRaw<__nv_bfloat16> { using V = uint2; };
__device__ __forceinline__ float4 ap_wide(const float4& v) { return v; }
__device__ __forceinline__ float4 ap_wide(const uint2& v) { return make_float4(bf16_lo(v.x), bf16_hi(v.x), bf16_lo(v.y), bf16_hi(v.y)); }

template <typename T, int kT, int kC>
struct ApTile {
    static constexpr int kPieces = kT * kC * 4 / kApThreads;      // of four columns, per thread, D = 16 kC
    float4 v[kPieces];
    __device__ __forceinline__ void fetch(const T* src, long long stride, int row0, int rows, int D, const uint8_t* keep, bool vec) {
        const int cols = (ap_pitch(D) - 4) >> 2, total = kT * cols;
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
            const int e = threadIdx.x + k * kApThreads;
            v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (e >= total) continue;
            const int r = e / cols, d = (e - r * cols) * 4;
            if (row0 + r >= rows || (keep != nullptr && keep[row0 + r] == 0)) continue;
            const T* p = src + (long long)(row0 + r) * stride + d;
            if (vec) {
                v[k] = ap_wide(*reinterpret_cast<const typename ApRaw<T>::V*>(p));
            } else {
                v[k].x = at_float(p[0]);
                if (d + 1 < D) v[k].y = at_float(p[1]);
                if (d + 2 < D) v[k].z = at_float(p[2]);
                if (d + 3 < D) v[k].w = at_float(p[3]);
            }
        }
    }
    __device__ __forceinline__ void put(float* dst, int D) const {
        const int pitch = ap_pitch(D), cols = (pitch - 4) >> 2, total = kT * cols;
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
            const int e = threadIdx.x + k * kApThreads;
            if (e >= total) continue;
            const int r = e / cols;
            *reinterpret_cast<float4*>(dst + r * pitch + (e - r * cols) * 4) = v[k];
        }
    }
};
// Rows of four-column pieces at the alignment their loads need
template <typename T> __device__ __forceinline__ bool ap_vec(const AttnTensor& t, int D) {
    return (D & 3) == 0 && ((t.b | t.l | t.h) & 3) == 0 && (reinterpret_cast<uintptr_t>(t.p) & (4 * sizeof(T) - 1)) == 0;
}

// acc[r][c] = A[ty kR + r] . B[tx + 16 c]
template <int kR>
__device__ __forceinline__ void ap_dot(float (&acc)[kR][kR], const float* A, const float* B, int D, int ty, int tx) {
    const int pitch = ap_pitch(D);
#pragma unroll
    for (int r = 0; r < kR; ++r)
#pragma unroll
        for (int c = 0; c < kR; ++c) acc[r][c] = 0.f;
    for (int d = 0; d < D; d += 4) {
        float4 a[kR], b[kR];
#pragma unroll
        for (int r = 0; r < kR; ++r) a[r] = *reinterpret_cast<const float4*>(A + (ty * kR + r) * pitch + d);
#pragma unroll
        for (int c = 0; c < kR; ++c) b[c] = *reinterpret_cast<const float4*>(B + (tx + 16 * c) * pitch + d);
#pragma unroll
        for (int r = 0; r < kR; ++r)
#pragma unroll
            for (int c = 0; c < kR; ++c) {
                acc[r][c] = fmaf(a[r].x, b[c].x, acc[r][c]);
                acc[r][c] = fmaf(a[r].y, b[c].y, acc[r][c]);
                acc[r][c] = fmaf(a[r].z, b[c].z, acc[r][c]);
                acc[r][c] = fmaf(a[r].w, b[c].w, acc[r][c]);
            }
    }
}
// out[r][c] += sum_j P[ty kR + r][j] X[j][tx + 16 c], c < kC
template <int kT, int kR, int kC>
__device__ __forceinline__ void ap_mix(float (&out)[kR][kC], const float* P, const float* X, int D, int ty, int tx) {
    const int pitch = ap_pitch(D), pp = ap_ppitch<kT>();
    for (int j = 0; j < kT; j += 4) {
        float4 a[kR];
#pragma unroll
        for (int r = 0; r < kR; ++r) a[r] = *reinterpret_cast<const float4*>(P + (ty * kR + r) * pp + j);
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            const int d = tx + 16 * c;
            if (d >= D) break;
            const float x0 = X[j * pitch + d], x1 = X[(j + 1) * pitch + d], x2 = X[(j + 2) * pitch + d],
                        x3 = X[(j + 3) * pitch + d];
#pragma unroll
            for (int r = 0; r < kR; ++r) {
                out[r][c] = fmaf(a[r].x, x0, out[r][c]);
                out[r][c] = fmaf(a[r].y, x1, out[r][c]);
                out[r][c] = fmaf(a[r].z, x2, out[r][c]);
                out[r][c] = fmaf(a[r].w, x3, out[r][c]);
            }
        }
    }
}
// Largest and sum over the sixteen threads of a row (a half warp).
__device__ __forceinline__ float ap_row_max(float v) {
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float ap_row_sum(float v) {
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Bias values and kept keys of a tile, fetched ahead of the products; then scores: scale and bias, -inf at masked keys and
// behind the last one.
template <typename T, int kR>
struct ApBias {
    float v[kR][kR];
    bool kept[kR];
    __device__ __forceinline__ void fetch(const AttnParams& p, int b, int h, int i0, int j0, int ty, int tx) {
        const uint8_t* keep = p.mask != nullptr ? p.mask + b * p.mask_b : nullptr;
        const T* bias = p.bias != nullptr ? static_cast<const T*>(p.bias) + b * p.bias_b + h * p.bias_h : nullptr;
#pragma unroll
        for (int c = 0; c < kR; ++c) {
            const int j = j0 + tx + 16 * c;
            kept[c] = j < p.Lk && (keep == nullptr || keep[j] != 0);
#pragma unroll
            for (int r = 0; r < kR; ++r) {
                const int i = i0 + ty * kR + r;
                v[r][c] = bias != nullptr && i < p.Lq && j < p.Lk ? at_float(bias[i * p.bias_i + j]) : 0.f;
            }
        }
    }
    __device__ __forceinline__ void apply(float (&s)[kR][kR], float scale) const {
#pragma unroll
        for (int c = 0; c < kR; ++c)
#pragma unroll
            for (int r = 0; r < kR; ++r) s[r][c] = kept[c] ? fmaf(s[r][c], scale, v[r][c]) : -INFINITY;
    }
};

// ---------------------------------------------------------------------------------------
// forward: grid (query tiles, H, B)
// ---------------------------------------------------------------------------------------
template <typename T, int kT, int kC>
__global__ void __launch_bounds__(kApThreads) attn_plain_fwd_kernel(const __grid_constant__ AttnParams p, int splits, int share, float* part_o, float2* part_ml) {
    constexpr int kR = kT / 16;
    extern __shared__ __align__(16) float sm[];
    const int pitch = ap_pitch(p.D), pp = ap_ppitch<kT>();
    float *Q = sm, *K = Q + kT * pitch, *V = K + kT * pitch, *P = V + kT * pitch;
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    const int i0 = blockIdx.x * kT, h = blockIdx.y, b = blockIdx.z / splits, split = blockIdx.z % splits, hk = h / (p.H / p.Hk);
    const int first = split * share * kT, end = min(p.Lk, first + share * kT);      // keys of this block
    griddep_wait();
    griddep_launch_dependents();
    const uint8_t* keep = p.mask != nullptr ? p.mask + b * p.mask_b : nullptr;
    const T* k = static_cast<const T*>(p.k.p) + b * p.k.b + hk * p.k.h;
    const T* v = static_cast<const T*>(p.v.p) + b * p.v.b + hk * p.v.h;
    const bool vk = ap_vec<T>(p.k, p.D), vv = ap_vec<T>(p.v, p.D);
    ApTile<T, kT, kC> tk, tv;
    tk.fetch(static_cast<const T*>(p.q.p) + b * p.q.b + h * p.q.h, p.q.l, i0, p.Lq, p.D, nullptr, ap_vec<T>(p.q, p.D));
    tk.put(Q, p.D);
    tk.fetch(k, p.k.l, first, p.Lk, p.D, keep, vk);
    tv.fetch(v, p.v.l, first, p.Lk, p.D, keep, vv);
    float o[kR][kC], m[kR], l[kR];
#pragma unroll
    for (int r = 0; r < kR; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int c = 0; c < kC; ++c) o[r][c] = 0.f;
    }
    for (int j0 = first; j0 < end; j0 += kT) {
        __syncthreads();
        tk.put(K, p.D);
        tv.put(V, p.D);
        __syncthreads();
        ApBias<T, kR> bias;
        bias.fetch(p, b, h, i0, j0, ty, tx);
        if (j0 + kT < end) {
            tk.fetch(k, p.k.l, j0 + kT, p.Lk, p.D, keep, vk);
            tv.fetch(v, p.v.l, j0 + kT, p.Lk, p.D, keep, vv);
        }
        float s[kR][kR];
        ap_dot<kR>(s, Q, K, p.D, ty, tx);
        bias.apply(s, p.scale);
#pragma unroll
        for (int r = 0; r < kR; ++r) {
            float mx = s[r][0];
#pragma unroll
            for (int c = 1; c < kR; ++c) mx = fmaxf(mx, s[r][c]);
            const float mn = fmaxf(m[r], ap_row_max(mx));
            const float base = mn == -INFINITY ? 0.f : mn;
            const float corr = exp2f((m[r] - base) * kLog2e);
            m[r] = mn;
            float t = 0.f;
#pragma unroll
            for (int c = 0; c < kR; ++c) {
                const float e = exp2f((s[r][c] - base) * kLog2e);
                t += e;
                P[(ty * kR + r) * pp + tx + 16 * c] = e;
            }
            l[r] = l[r] * corr + ap_row_sum(t);
#pragma unroll
            for (int c = 0; c < kC; ++c) o[r][c] *= corr;
        }
        __syncwarp();            // a row's probabilities are written and read by the same half warp
        ap_mix<kT, kR, kC>(o, P, V, p.D, ty, tx);
    }
#pragma unroll
    for (int r = 0; r < kR; ++r) {
        const int i = i0 + ty * kR + r;
        if (i >= p.Lq) continue;
        if (part_o != nullptr) {             // not yet divided: attn_combine_kernel joins the parts
            const long long row = (((long long)split * p.B + b) * p.H + h) * p.Lq + i;
#pragma unroll
            for (int c = 0; c < kC; ++c)
                if (tx + 16 * c < p.D) part_o[row * p.D + tx + 16 * c] = o[r][c];
            if (tx == 0) part_ml[row] = make_float2(m[r], l[r]);
            continue;
        }
        const bool empty = l[r] == 0.f;
        const float inv = empty ? 0.f : 1.f / l[r];
        T* dst = static_cast<T*>(p.o.p) + b * p.o.b + (long long)i * p.o.l + h * p.o.h;
        const long long lo = (((long long)b * p.Lq + i) * p.H + h) * p.D;
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            const int d = tx + 16 * c;
            if (d >= p.D) break;
            const float y = empty ? 0.f : o[r][c] * inv;
            at_store(dst + d, y);
            if constexpr (sizeof(T) == 2) {
                if (p.o_lo != nullptr) {
                    const float rest = y - __bfloat162float(__float2bfloat16_rn(y));
                    static_cast<__nv_bfloat16*>(p.o_lo)[lo + d] = __float2bfloat16_rn(rest);
                }
            }
        }
        if (tx == 0 && p.stats != nullptr)
            p.stats[((long long)b * p.H + h) * p.Lq + i] = empty ? make_float2(0.f, INFINITY) : make_float2(m[r], log2f(l[r]));
    }
}

// Statistics of a thread's rows; then probabilities and score gradients from scores s and products g = dout . v.
template <int kR>
struct ApStats {
    float2 st[kR];
    float delta[kR];
    __device__ __forceinline__ void fetch(const AttnParams& p, int b, int h, int i0, int ty) {
#pragma unroll
        for (int r = 0; r < kR; ++r) {
            const int i = i0 + ty * kR + r;
            st[r] = make_float2(0.f, INFINITY);
            delta[r] = 0.f;
            if (i < p.Lq) {
                st[r] = p.stats[((long long)b * p.H + h) * p.Lq + i];
                delta[r] = p.delta[((long long)b * p.H + h) * p.Lq + i];
            }
        }
    }
    __device__ __forceinline__ void apply(float (&s)[kR][kR], float (&g)[kR][kR]) const {
#pragma unroll
        for (int r = 0; r < kR; ++r)
#pragma unroll
            for (int c = 0; c < kR; ++c) {
                const float e = exp2f(fmaf(s[r][c] - st[r].x, kLog2e, -st[r].y));
                s[r][c] = e;
                g[r][c] = e == 0.f ? 0.f : e * (g[r][c] - delta[r]);
            }
    }
};

// ---------------------------------------------------------------------------------------
// gradient of q, and of the scores where the bias wants one: a block per query tile, head and batch element
// ---------------------------------------------------------------------------------------
template <typename T, int kT, int kC>
__device__ __forceinline__ void ap_dq_block(const AttnParams& p, const AttnBwdSplit& w, int tile, int h, int b, int split) {
    constexpr int kR = kT / 16;
    extern __shared__ __align__(16) float sm[];
    const int pitch = ap_pitch(p.D), pp = ap_ppitch<kT>();
    float *Q = sm, *G = Q + kT * pitch, *K = G + kT * pitch, *V = K + kT * pitch, *P = V + kT * pitch;
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    const int i0 = tile * kT, hk = h / (p.H / p.Hk);
    const int first = split * w.q_share * kT, end = min(p.Lk, first + w.q_share * kT);      // keys of this block
    const uint8_t* keep = p.mask != nullptr ? p.mask + b * p.mask_b : nullptr;
    const T* k = static_cast<const T*>(p.k.p) + b * p.k.b + hk * p.k.h;
    const T* v = static_cast<const T*>(p.v.p) + b * p.v.b + hk * p.v.h;
    const bool vk = ap_vec<T>(p.k, p.D), vv = ap_vec<T>(p.v, p.D);
    ApTile<T, kT, kC> tk, tv;
    tk.fetch(static_cast<const T*>(p.q.p) + b * p.q.b + h * p.q.h, p.q.l, i0, p.Lq, p.D, nullptr, ap_vec<T>(p.q, p.D));
    tv.fetch(static_cast<const T*>(p.dout.p) + b * p.dout.b + h * p.dout.h, p.dout.l, i0, p.Lq, p.D, nullptr, ap_vec<T>(p.dout, p.D));
    tk.put(Q, p.D);
    tv.put(G, p.D);
    tk.fetch(k, p.k.l, first, p.Lk, p.D, keep, vk);
    tv.fetch(v, p.v.l, first, p.Lk, p.D, keep, vv);
    ApStats<kR> st;
    st.fetch(p, b, h, i0, ty);
    float o[kR][kC];
#pragma unroll
    for (int r = 0; r < kR; ++r)
#pragma unroll
        for (int c = 0; c < kC; ++c) o[r][c] = 0.f;
    for (int j0 = first; j0 < end; j0 += kT) {
        __syncthreads();
        tk.put(K, p.D);
        tv.put(V, p.D);
        __syncthreads();
        ApBias<T, kR> bias;
        bias.fetch(p, b, h, i0, j0, ty, tx);
        if (j0 + kT < end) {
            tk.fetch(k, p.k.l, j0 + kT, p.Lk, p.D, keep, vk);
            tv.fetch(v, p.v.l, j0 + kT, p.Lk, p.D, keep, vv);
        }
        float s[kR][kR], g[kR][kR];
        ap_dot<kR>(s, Q, K, p.D, ty, tx);
        ap_dot<kR>(g, G, V, p.D, ty, tx);
        bias.apply(s, p.scale);
        st.apply(s, g);
#pragma unroll
        for (int r = 0; r < kR; ++r) {
            const int i = i0 + ty * kR + r;
#pragma unroll
            for (int c = 0; c < kR; ++c) {
                const int j = j0 + tx + 16 * c;
                P[(ty * kR + r) * pp + tx + 16 * c] = g[r][c];
                if (p.ds != nullptr && i < p.Lq && j < p.Lk) {
                    const long long head = b * p.ds_b + h * p.ds_h;
                    const float ds = bias.kept[c] ? g[r][c] : 0.f;         // zero also in a row whose statistics are NaN
                    if (p.ds_parts) static_cast<float*>(p.ds)[head + ((long long)(j >> 2) * p.Lq + i) * 4 + (j & 3)] = ds;
                    else at_store(static_cast<T*>(p.ds) + head + i * p.ds_i + j, ds);
                }
            }
        }
        __syncwarp();
        ap_mix<kT, kR, kC>(o, P, K, p.D, ty, tx);
    }
#pragma unroll
    for (int r = 0; r < kR; ++r) {
        const int i = i0 + ty * kR + r;
        if (i >= p.Lq) continue;
        if (w.dq != nullptr) {
            float* part = w.dq + ((((long long)split * p.B + b) * p.H + h) * p.Lq + i) * p.D;
#pragma unroll
            for (int c = 0; c < kC; ++c)
                if (tx + 16 * c < p.D) part[tx + 16 * c] = o[r][c] * p.scale;
            continue;
        }
        T* dst = static_cast<T*>(p.dq.p) + b * p.dq.b + (long long)i * p.dq.l + h * p.dq.h;
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            const int d = tx + 16 * c;
            if (d >= p.D) break;
            at_store(dst + d, o[r][c] * p.scale);
        }
    }
}

// ---------------------------------------------------------------------------------------
// gradients of k and v: a block per key tile, key head and batch element; the query heads that share the key head are
// summed here
// ---------------------------------------------------------------------------------------
template <typename T, int kT, int kC>
__device__ __forceinline__ void ap_dkv_block(const AttnParams& p, const AttnBwdSplit& w, int tile, int hk, int b, int split) {
    constexpr int kR = kT / 16;
    extern __shared__ __align__(16) float sm[];
    const int pitch = ap_pitch(p.D), pp = ap_ppitch<kT>();
    float *Q = sm, *G = Q + kT * pitch, *K = G + kT * pitch, *V = K + kT * pitch, *P = V + kT * pitch, *S = P + kT * pp;
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    const int j0 = tile * kT, group = p.H / p.Hk;
    const uint8_t* keep = p.mask != nullptr ? p.mask + b * p.mask_b : nullptr;
    const bool vq = ap_vec<T>(p.q, p.D), vg = ap_vec<T>(p.dout, p.D);
    const int nq = (p.Lq + kT - 1) / kT;
    const int first = split * w.kv_share, end = min(group * nq, first + w.kv_share);        // query tiles, head after head
    ApTile<T, kT, kC> tq, tg;
    tq.fetch(static_cast<const T*>(p.k.p) + b * p.k.b + hk * p.k.h, p.k.l, j0, p.Lk, p.D, keep, ap_vec<T>(p.k, p.D));
    tg.fetch(static_cast<const T*>(p.v.p) + b * p.v.b + hk * p.v.h, p.v.l, j0, p.Lk, p.D, keep, ap_vec<T>(p.v, p.D));
    tq.put(K, p.D);
    tg.put(V, p.D);
    auto fetch = [&](int it) {
        const int h = hk * group + it / nq, i0 = it % nq * kT;
        tq.fetch(static_cast<const T*>(p.q.p) + b * p.q.b + h * p.q.h, p.q.l, i0, p.Lq, p.D, nullptr, vq);
        tg.fetch(static_cast<const T*>(p.dout.p) + b * p.dout.b + h * p.dout.h, p.dout.l, i0, p.Lq, p.D, nullptr, vg);
    };
    fetch(first);
    float dk[kR][kC], dv[kR][kC];
#pragma unroll
    for (int r = 0; r < kR; ++r)
#pragma unroll
        for (int c = 0; c < kC; ++c) dk[r][c] = dv[r][c] = 0.f;
    for (int it = first; it < end; ++it) {
        const int h = hk * group + it / nq, i0 = it % nq * kT;
        __syncthreads();
        tq.put(Q, p.D);
        tg.put(G, p.D);
        __syncthreads();
        ApBias<T, kR> bias;
        bias.fetch(p, b, h, i0, j0, ty, tx);
        ApStats<kR> st;
        st.fetch(p, b, h, i0, ty);
        if (it + 1 < end) fetch(it + 1);
        float s[kR][kR], g[kR][kR];
        ap_dot<kR>(s, Q, K, p.D, ty, tx);
        ap_dot<kR>(g, G, V, p.D, ty, tx);
        bias.apply(s, p.scale);
        st.apply(s, g);
#pragma unroll
        for (int r = 0; r < kR; ++r)
#pragma unroll
            for (int c = 0; c < kR; ++c) {              // transposed: rows of keys
                P[(tx + 16 * c) * pp + ty * kR + r] = s[r][c];
                S[(tx + 16 * c) * pp + ty * kR + r] = g[r][c];
            }
        __syncthreads();
        ap_mix<kT, kR, kC>(dv, P, G, p.D, ty, tx);
        ap_mix<kT, kR, kC>(dk, S, Q, p.D, ty, tx);
    }
#pragma unroll
    for (int r = 0; r < kR; ++r) {
        const int j = j0 + ty * kR + r;
        if (j >= p.Lk) continue;
        const bool kept = keep == nullptr || keep[j] != 0;     // zero whatever the upstream gradient holds
        if (w.dk != nullptr) {
            const long long row = ((((long long)split * p.B + b) * p.Hk + hk) * p.Lk + j) * p.D;
#pragma unroll
            for (int c = 0; c < kC; ++c) {
                const int d = tx + 16 * c;
                if (d >= p.D) break;
                w.dk[row + d] = kept ? dk[r][c] * p.scale : 0.f;
                w.dv[row + d] = kept ? dv[r][c] : 0.f;
            }
            continue;
        }
        T* dkp = static_cast<T*>(p.dk.p) + b * p.dk.b + (long long)j * p.dk.l + hk * p.dk.h;
        T* dvp = static_cast<T*>(p.dv.p) + b * p.dv.b + (long long)j * p.dv.l + hk * p.dv.h;
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            const int d = tx + 16 * c;
            if (d >= p.D) break;
            at_store(dkp + d, kept ? dk[r][c] * p.scale : 0.f);
            at_store(dvp + d, kept ? dv[r][c] : 0.f);
        }
    }
}

// Both kinds of blocks in one grid, the longer kind first: where neither fills the device, they run side by side.
template <typename T, int kT, int kC>
__global__ void __launch_bounds__(kApThreads)
attn_plain_bwd_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ AttnBwdSplit w) {
    const int first = w.q_first ? w.q_blocks : w.kv_blocks;
    const bool second = (int)blockIdx.x >= first, over_keys = second != (w.q_first != 0);
    const int n = second ? (int)blockIdx.x - first : (int)blockIdx.x;
    const int tiles = ((over_keys ? p.Lq : p.Lk) + kT - 1) / kT, heads = over_keys ? p.H : p.Hk;
    const int tile = n % tiles, h = n / tiles % heads, b = n / tiles / heads % p.B, split = n / tiles / heads / p.B;
    griddep_wait();
    griddep_launch_dependents();
    if (over_keys) ap_dq_block<T, kT, kC>(p, w, tile, h, b, split);
    else ap_dkv_block<T, kT, kC>(p, w, tile, h, b, split);
}

// The parts of a gradient added up, in order: a thread per element; blockIdx.y: which of two tensors of one shape
template <typename T>
__global__ void __launch_bounds__(kApThreads)
attn_join_kernel(const float* part0, const float* part1, AttnTensor t0, AttnTensor t1, int splits, int L, int heads, int D, long long n) {
    griddep_wait();
    griddep_launch_dependents();
    const float* part = blockIdx.y ? part1 : part0;
    const AttnTensor& t = blockIdx.y ? t1 : t0;
    for (long long e = (long long)blockIdx.x * kApThreads + threadIdx.x; e < n; e += (long long)gridDim.x * kApThreads) {
        float y = 0.f;
#pragma unroll 8
        for (int s = 0; s < splits; ++s) y += part[s * n + e];
        const long long row = e / D, bh = row / L;
        at_store(static_cast<T*>(t.p) + bh / heads * t.b + (row - bh * L) * t.l + bh % heads * t.h + (e - row * D), y);
    }
}

// Gradient of a bias that serves several batch elements or heads: the scores' gradients (AttnParams::ds_parts) summed over the
// broadcast axes in fp32, in a fixed order, and rounded once.  bf16 summands would halve the way through memory (4 x 512 x 768,
// 16 heads of 64, a training pass: 137 us instead of 143), but where they cancel, their roundings are all that is left.  A block
// takes 32 rows of eight 16-byte pieces: reads run along the rows, as the parts lie, writes along the columns.  Bound by the
// parts' way from memory: 18 us for the 113 MB of that call, 6.1 TB/s.  (Parts of whole rows, a lane of the backward kernel
// writing 16 bytes of each: 105 us for that kernel instead of 81.)
constexpr int kApSumRows = 32, kApSumChunks = kApThreads / kApSumRows;
template <typename T>
__global__ void __launch_bounds__(kApThreads)
attn_bias_sum_kernel(const float* ds, long long ds_b, long long ds_h, T* out, long long out_b, long long out_h, long long out_i,
                     int B, int H, int Lq, int Lk, int sum_b, int sum_h) {
    constexpr int kN = 16 / (int)sizeof(T), kLoads = kN / 4;
    __shared__ uint4 tile[kApSumRows][kApSumChunks + 1];
    griddep_wait();
    griddep_launch_dependents();
    const int nch = (Lk + kN - 1) / kN, row_tiles = (Lq + kApSumRows - 1) / kApSumRows, col_tiles = (nch + kApSumChunks - 1) / kApSumChunks;
    const int ob = sum_b ? 1 : B, oh = sum_h ? 1 : H;
    const int nb = sum_b ? B : 1, nh = sum_h ? H : 1;
    const long long tiles = (long long)ob * oh * row_tiles * col_tiles;
    for (long long t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int c0 = (int)(t % col_tiles) * kApSumChunks;
        const long long r = t / col_tiles;
        const int i0 = (int)(r % row_tiles) * kApSumRows, x = (int)(r / row_tiles);
        const int h0 = x % oh, b0 = x / oh;
        const int row = threadIdx.x % kApSumRows, chunk = threadIdx.x / kApSumRows, i = i0 + row, c = c0 + chunk;
        float acc[kN];
#pragma unroll
        for (int e = 0; e < kN; ++e) acc[e] = 0.f;
        if (i < Lq && c < nch) {
#pragma unroll 4
            for (int s = 0; s < nb * nh; ++s) {
                const int b = b0 + s / nh, h = h0 + s % nh;
                const float4* src = reinterpret_cast<const float4*>(ds + b * ds_b + h * ds_h) + (long long)c * kLoads * Lq + i;
#pragma unroll
                for (int l = 0; l < kLoads; ++l) {
                    const float4 v = at_load(src + (long long)l * Lq);
                    acc[4 * l] += v.x;
                    acc[4 * l + 1] += v.y;
                    acc[4 * l + 2] += v.z;
                    acc[4 * l + 3] += v.w;
                }
            }
        }
        if constexpr (sizeof(T) == 2)
            tile[row][chunk] = make_uint4(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]), pack_bf16x2(acc[4], acc[5]), pack_bf16x2(acc[6], acc[7]));
        else
            tile[row][chunk] = make_uint4(__float_as_uint(acc[0]), __float_as_uint(acc[1]), __float_as_uint(acc[2]), __float_as_uint(acc[3]));
        __syncthreads();
        const int row2 = threadIdx.x / kApSumChunks, chunk2 = threadIdx.x % kApSumChunks;
        if (i0 + row2 < Lq && c0 + chunk2 < nch)
            *(reinterpret_cast<uint4*>(out + b0 * out_b + h0 * out_h + (i0 + row2) * out_i) + c0 + chunk2) = tile[row2][chunk2];
        __syncthreads();
    }
}

}  // namespace trimul

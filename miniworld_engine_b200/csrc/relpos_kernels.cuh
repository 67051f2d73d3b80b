// Learned relative position bias by buckets, and the gradient of its table.
//
//   u(b,i,j) = bucket(q_pos[b,i] - k_pos[b,j])      (a bucket of its own for positions of different segments)
//   heads:  out[b,h,i,j]  = table[u, h]             an attention's additive bias, j contiguous
//   pair:   out[b,i,j,c]  = add[b,i,j,c] + table[u, c]     the pair tensor's input embedding, c contiguous
//   d table[u, c] = sum of the upstream gradient over all positions of bucket u
//
// Every kernel is bound by device memory: the large tensor is read or written once.  The bucket of a distance is looked
// up in a table over [-M, M] in shared memory that each block builds from the rule (distances beyond M share the
// outermost buckets), so no rule costs more per element than another and nothing has to be kept between calls.
#pragma once

#include "../../include/trimul_b200.h"
#include "ptx_sm100.cuh"

namespace trimul {

constexpr int kRpPosLimit = (1 << 30) - 1;   // positions are clamped here: no difference overflows 32 bits

struct RelposParams {
    int B, Lq, Lk, C;
    int rows;                              // buckets, the segments' one included
    int M;                                 // largest distance of the look-up table
    const void *q_pos, *k_pos, *q_seg, *k_seg;      // seg: null when segments are not told apart
    long long q_pos_b, k_pos_b, q_seg_b, k_seg_b;   // batch strides in elements (0: shared)
    int q_pos64, k_pos64, q_seg64, k_seg64;         // 64-bit integers instead of 32-bit ones
    const void* table;
    int table_bf16;
    long long sB, sH, sI;                  // strides of out / grad in elements (heads); sB only (pair)
};

__device__ __forceinline__ int rp_load(const void* p, long long i, int is64) {
    if (is64) {
        const long long v = __ldg(static_cast<const long long*>(p) + i);
        return (int)(v > kRpPosLimit ? kRpPosLimit : v < -kRpPosLimit ? -kRpPosLimit : v);
    }
    return min(max(__ldg(static_cast<const int*>(p) + i), -kRpPosLimit), kRpPosLimit);
}
// Segments are only compared for equality, so they are taken as they are, in full width
__device__ __forceinline__ long long rp_segment(const void* p, long long i, int is64) {
    return is64 ? __ldg(static_cast<const long long*>(p) + i) : (long long)__ldg(static_cast<const int*>(p) + i);
}
__device__ __forceinline__ float rp_table(const RelposParams& p, int u, int c) {
    const long long i = (long long)u * p.C + c;
    return p.table_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.table)[i])
                        : static_cast<const float*>(p.table)[i];
}

// Bucket of distance d, |d| <= M, straight from the rule.  Logarithmic rules: exact up to `near`, then one bucket per
// threshold reached.
__device__ __forceinline__ int rp_rule(const trimul_buckets& b, int d) {
    if (b.kind == TRIMUL_BUCKETS_CLIPPED) return d + b.max_distance;
    const int half = b.kind == TRIMUL_BUCKETS_LOG ? b.count / 2 : b.count;
    const int n = b.kind == TRIMUL_BUCKETS_LOG ? abs(d) : max(d, 0);
    int lo = 0, hi = b.n_thresholds;
    if (hi <= 32) {          // all threads read the same threshold at a time: no divergent reads of the parameter space
        for (int t = 0; t < b.n_thresholds; ++t) lo += b.thresholds[t] <= n;
        hi = lo;
    }
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (b.thresholds[mid] <= n) lo = mid + 1; else hi = mid;
    }
    return min(n, half / 2) + lo + (b.kind == TRIMUL_BUCKETS_LOG && d < 0 ? half : 0);
}
__device__ __forceinline__ void rp_build_lut(uint16_t* lut, const trimul_buckets& b, int M) {
    for (int i = threadIdx.x; i <= 2 * M; i += blockDim.x) lut[i] = (uint16_t)rp_rule(b, i - M);
}
__device__ __forceinline__ int rp_bucket(const uint16_t* lut, int M, int d) { return lut[min(max(d, -M), M) + M]; }

template <typename T> struct RpVec;       // 16 bytes of T
template <> struct RpVec<__nv_bfloat16> {
    static constexpr int kN = 8;
    static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
        f[0] = bf16_lo(v.x); f[1] = bf16_hi(v.x); f[2] = bf16_lo(v.y); f[3] = bf16_hi(v.y);
        f[4] = bf16_lo(v.z); f[5] = bf16_hi(v.z); f[6] = bf16_lo(v.w); f[7] = bf16_hi(v.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
        return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
    }
};
template <> struct RpVec<float> {
    static constexpr int kN = 4;
    static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[4]) {
        f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};
__device__ __forceinline__ float rp_float(float v) { return v; }
__device__ __forceinline__ float rp_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void rp_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void rp_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// ---------------------------------------------------------------------------------------
// heads, forward.  One block column (blockIdx.y) per group of kN heads; an item is kN consecutive j of one row: kN
// table rows of the group (16 bytes each) are turned into kN 16-byte stores, one per head.  Rows of `out` are padded to
// whole 16-byte pieces by the caller, so the last piece of a row is stored whole.
// Table rows are kept with their low three bits xor-ed by the next three: neighbouring lanes of a warp are kN rows apart
// where buckets follow the distance, and would otherwise meet in one bank.
// ---------------------------------------------------------------------------------------
constexpr int kRpThreads = 128;

__device__ __forceinline__ void rp_transpose(uint4 (&r)[8]) {        // 8 x 8 bf16, rows of 16 bytes
    uint4 o[8];
    const uint32_t* in = &r[0].x;
    uint32_t* out = &o[0].x;
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t a = in[(2 * j) * 4 + m], b = in[(2 * j + 1) * 4 + m];
            out[(2 * m) * 4 + j] = __byte_perm(a, b, 0x5410);
            out[(2 * m + 1) * 4 + j] = __byte_perm(a, b, 0x7632);
        }
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = o[i];
}
__device__ __forceinline__ void rp_transpose(uint4 (&r)[4]) {        // 4 x 4 fp32
    const uint4 a = r[0], b = r[1], c = r[2], d = r[3];
    r[0] = make_uint4(a.x, b.x, c.x, d.x);
    r[1] = make_uint4(a.y, b.y, c.y, d.y);
    r[2] = make_uint4(a.z, b.z, c.z, d.z);
    r[3] = make_uint4(a.w, b.w, c.w, d.w);
}

template <typename T>
__global__ void __launch_bounds__(kRpThreads)
relpos_heads_kernel(const __grid_constant__ RelposParams p, const __grid_constant__ trimul_buckets rule, T* out) {
    constexpr int kN = RpVec<T>::kN;
    extern __shared__ __align__(16) uint8_t rp_smem[];
    T* tab = reinterpret_cast<T*>(rp_smem);                                      // [rows rounded up to 64][kN]
    uint16_t* lut = reinterpret_cast<uint16_t*>(rp_smem + ((p.rows + 63) & ~63) * 16);
    rp_build_lut(lut, rule, p.M);
    griddep_wait();
    griddep_launch_dependents();
    const int h0 = blockIdx.y * kN;
    for (int e = threadIdx.x; e < p.rows * kN; e += kRpThreads) {
        const int u = e / kN, h = e % kN;
        rp_store(tab + (u ^ ((u >> 3) & 7)) * kN + h, h0 + h < p.C ? rp_table(p, u, h0 + h) : 0.f);
    }
    __syncthreads();
    const int nch = (p.Lk + kN - 1) / kN;
    const long long items = (long long)p.B * p.Lq * nch;
    const int nh = min(kN, p.C - h0);
    for (long long it = (long long)blockIdx.x * kRpThreads + threadIdx.x; it < items; it += (long long)gridDim.x * kRpThreads) {
        const long long row = it / nch;
        const int j0 = (int)(it - row * nch) * kN;
        const int b = (int)(row / p.Lq), i = (int)(row - (long long)b * p.Lq);
        const int q = rp_load(p.q_pos, b * p.q_pos_b + i, p.q_pos64);
        const long long qs = p.q_seg != nullptr ? rp_segment(p.q_seg, b * p.q_seg_b + i, p.q_seg64) : 0;
        uint4 r[kN];
#pragma unroll
        for (int e = 0; e < kN; ++e) {
            const int j = min(j0 + e, p.Lk - 1);
            int u = rp_bucket(lut, p.M, q - rp_load(p.k_pos, b * p.k_pos_b + j, p.k_pos64));
            if (p.q_seg != nullptr && rp_segment(p.k_seg, b * p.k_seg_b + j, p.k_seg64) != qs) u = p.rows - 1;
            r[e] = *reinterpret_cast<const uint4*>(tab + (u ^ ((u >> 3) & 7)) * kN);
        }
        rp_transpose(r);
        T* o = out + b * p.sB + h0 * p.sH + i * p.sI + j0;
#pragma unroll
        for (int h = 0; h < kN; ++h)
            if (h < nh) *reinterpret_cast<uint4*>(o + h * p.sH) = r[h];
    }
}

// ---------------------------------------------------------------------------------------
// pair, forward.  A block takes runs of kRpPairThreads consecutive positions: first each thread finds the bucket of one
// position, then all stream the run's channels, 16 bytes a piece (kVec; else single channels), eight pieces in flight each;
// the table's rows come through L1 (a few buckets are live at a time).
// ---------------------------------------------------------------------------------------
constexpr int kRpPairThreads = 256;

struct RpCursor {          // position -> (batch element, row, column), stepped without divisions
    int b, i, j;
    __device__ __forceinline__ void init(const RelposParams& p, long long pos) {
        const long long row = pos / p.Lk;
        j = (int)(pos - row * p.Lk);
        b = (int)(row / p.Lq);
        i = (int)(row - (long long)b * p.Lq);
    }
    __device__ __forceinline__ void step(const RelposParams& p, int n) {
        j += n;
        while (j >= p.Lk) {
            j -= p.Lk;
            if (++i == p.Lq) { i = 0; ++b; }
        }
    }
    __device__ __forceinline__ int bucket(const RelposParams& p, const uint16_t* lut) const {
        const int d = rp_load(p.q_pos, b * p.q_pos_b + i, p.q_pos64) - rp_load(p.k_pos, b * p.k_pos_b + j, p.k_pos64);
        int u = rp_bucket(lut, p.M, d);
        if (p.q_seg != nullptr && rp_segment(p.q_seg, b * p.q_seg_b + i, p.q_seg64) != rp_segment(p.k_seg, b * p.k_seg_b + j, p.k_seg64))
            u = p.rows - 1;
        return u;
    }
};

template <typename T, bool kVec>
__global__ void __launch_bounds__(kRpPairThreads)
relpos_pair_kernel(const __grid_constant__ RelposParams p, const __grid_constant__ trimul_buckets rule, const T* add, T* out,
                   int per_block) {
    constexpr int kN = kVec ? RpVec<T>::kN : 1;
    constexpr int kU = 8;
    extern __shared__ __align__(16) uint8_t rp_smem[];
    int* su = reinterpret_cast<int*>(rp_smem);                                 // buckets of kRpPairThreads positions
    uint16_t* lut = reinterpret_cast<uint16_t*>(su + kRpPairThreads);
    rp_build_lut(lut, rule, p.M);
    griddep_wait();
    griddep_launch_dependents();
    const long long total = (long long)p.B * p.Lq * p.Lk;
    const long long first = (long long)blockIdx.x * per_block, last = min(first + per_block, total);
    const int per_pos = p.C / kN;
    RpCursor cur;
    if (first + threadIdx.x < last) cur.init(p, first + threadIdx.x);
    // vector v of a run is channel piece v % per_pos of position v / per_pos: stepped, not divided
    const int step_pos = kRpPairThreads / per_pos, step_c = kRpPairThreads % per_pos;
    for (long long pos = first; pos < last; pos += kRpPairThreads) {
        const int n = (int)min((long long)kRpPairThreads, last - pos);
        __syncthreads();
        if ((int)threadIdx.x < n) {
            su[threadIdx.x] = cur.bucket(p, lut);
            cur.step(p, kRpPairThreads);
        }
        __syncthreads();
        const long long base = pos * per_pos;
        const int vectors = n * per_pos;
        int x = threadIdx.x / per_pos, c = threadIdx.x % per_pos;
        for (int v0 = threadIdx.x; v0 < vectors; v0 += kU * kRpPairThreads) {
            if constexpr (kVec) {
                uint4 a[kU];
#pragma unroll
                for (int s = 0; s < kU; ++s) {
                    const int v = v0 + s * kRpPairThreads;
                    a[s] = add != nullptr && v < vectors ? __ldcs(reinterpret_cast<const uint4*>(add) + base + v)
                                                         : make_uint4(0u, 0u, 0u, 0u);
                }
#pragma unroll
                for (int s = 0; s < kU; ++s) {
                    const int v = v0 + s * kRpPairThreads;
                    if (v < vectors) {
                        const long long t0 = (long long)su[x] * p.C + c * kN;
                        float f[kN];
                        RpVec<T>::unpack(a[s], f);
                        if (p.table_bf16) {
#pragma unroll
                            for (int e = 0; e < kN; ++e) f[e] += __bfloat162float(static_cast<const __nv_bfloat16*>(p.table)[t0 + e]);
                        } else {
                            const float4* t = reinterpret_cast<const float4*>(static_cast<const float*>(p.table) + t0);
#pragma unroll
                            for (int e = 0; e < kN / 4; ++e) {
                                const float4 w = __ldg(t + e);
                                f[4 * e] += w.x; f[4 * e + 1] += w.y; f[4 * e + 2] += w.z; f[4 * e + 3] += w.w;
                            }
                        }
                        __stcs(reinterpret_cast<uint4*>(out) + base + v, RpVec<T>::pack(f));
                    }
                    x += step_pos;
                    c += step_c;
                    if (c >= per_pos) { c -= per_pos; ++x; }
                }
            } else {
#pragma unroll
                for (int s = 0; s < kU; ++s) {
                    const int v = v0 + s * kRpPairThreads;
                    if (v < vectors)
                        rp_store(out + base + v, (add != nullptr ? rp_float(add[base + v]) : 0.f) + rp_table(p, su[x], c));
                    x += step_pos;
                    c += step_c;
                    if (c >= per_pos) { c -= per_pos; ++x; }
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------------------
// heads, gradient of the table.  Block (part, group of kH heads) sums the rows of its part.  Sums live in shared memory,
// [rows][kH][threads]: a column per thread, no atomics, so the result does not depend on the order of anything.  A thread
// keeps kN consecutive j and walks down the rows, all kH heads at once: the bucket of a position is found once for them.
// Where the outermost distances of a piece share a bucket (buckets are monotone on either side of zero, so everything
// between shares it too), the piece is summed in registers; the running bucket's sums go to shared memory when it changes.
// Seg: what holds a segment, 64 bits where either side's numbers have them: they cost registers, by which the resident
// blocks are counted (16 x 2048^2 with three chains, forward and gradient: 129 us with 32-bit segments, 139 with 64-bit ones).
// ---------------------------------------------------------------------------------------
template <typename T, bool kVec, int kH, typename Seg>
__global__ void __launch_bounds__(kRpThreads)
relpos_heads_grad_kernel(const __grid_constant__ RelposParams p, const __grid_constant__ trimul_buckets rule, const T* grad,
                         float* partial, int parts_per_b, int rows_per_part) {
    constexpr int kN = RpVec<T>::kN;
    constexpr int kU = 4 / kH;
    extern __shared__ __align__(16) uint8_t rp_smem[];
    float* acc = reinterpret_cast<float*>(rp_smem);                               // [rows][kH][threads]
    const int nt = blockDim.x, tid = threadIdx.x;
    Seg* sg = reinterpret_cast<Seg*>(acc + (size_t)p.rows * kH * nt);             // the part's query segments, then positions
    int* sq = reinterpret_cast<int*>(sg + rows_per_part);
    uint16_t* lut = reinterpret_cast<uint16_t*>(sq + rows_per_part);
    rp_build_lut(lut, rule, p.M);
    for (int u = 0; u < p.rows * kH; ++u) acc[u * nt + tid] = 0.f;
    griddep_wait();
    griddep_launch_dependents();
    const int h0 = blockIdx.y * kH;
    const int nch = (p.Lk + kN - 1) / kN;
    const int tpr = min(nch, nt);                             // threads of one row
    const int side = nt / tpr;                                // rows at once
    const int ty = tid / tpr, tx = tid % tpr;
    const int b = blockIdx.x / parts_per_b;
    // row r of the part is query first + r parts_per_b: near pairs, whose pieces have several buckets and cost most, then come
    // to all threads alike as r goes on (with consecutive rows a few warps had them all: 95 us instead of 82 for forward and
    // gradient of 16 x 2048^2 with logarithmic buckets, 111 instead of 88 with 65 clipped ones)
    const int first = blockIdx.x - b * parts_per_b, r1 = (p.Lq - first + parts_per_b - 1) / parts_per_b;
    const long long row_stride = p.sI * parts_per_b;
    const T* gb = grad + b * p.sB + h0 * p.sH + first * p.sI;
    for (int r = tid; r < r1; r += nt) {
        const int i = first + r * parts_per_b;
        sq[r] = rp_load(p.q_pos, b * p.q_pos_b + i, p.q_pos64);
        sg[r] = p.q_seg != nullptr ? (Seg)rp_segment(p.q_seg, b * p.q_seg_b + i, p.q_seg64) : 0;
    }
    __syncthreads();
    int run = 0;
    float sum[kH];
#pragma unroll
    for (int h = 0; h < kH; ++h) sum[h] = 0.f;
    auto move_to = [&](int u) {
        if (u == run) return;
#pragma unroll
        for (int h = 0; h < kH; ++h) {
            acc[(run * kH + h) * nt + tid] += sum[h];
            sum[h] = 0.f;
        }
        run = u;
    };
    if (ty < side) {
        for (int c = tx; c < nch; c += tpr) {
            const int j0 = c * kN, nj = min(kN, p.Lk - j0);
            int kp[kN];
            Seg ks[kN];
#pragma unroll
            for (int e = 0; e < kN; ++e) {
                const int j = min(j0 + e, p.Lk - 1);
                kp[e] = rp_load(p.k_pos, b * p.k_pos_b + j, p.k_pos64);
                ks[e] = p.k_seg != nullptr ? (Seg)rp_segment(p.k_seg, b * p.k_seg_b + j, p.k_seg64) : 0;
            }
            int kmin = kp[0], kmax = kp[0];
            bool one_seg = true;
#pragma unroll
            for (int e = 1; e < kN; ++e) {
                kmin = min(kmin, kp[e]);
                kmax = max(kmax, kp[e]);
                one_seg = one_seg && ks[e] == ks[0];
            }
            const T* src = gb + j0;
            // kU rows of this thread's piece; the next kU are in flight while these are added up
            auto load = [&](uint4 (&raw)[kU][kH], int r) {
#pragma unroll
                for (int s = 0; s < kU; ++s)
#pragma unroll
                    for (int h = 0; h < kH; ++h) {
                        const bool in = r + s * side < r1 && h0 + h < p.C;
                        const T* row = src + (r + s * side) * row_stride + h * p.sH;
                        raw[s][h] = make_uint4(0u, 0u, 0u, 0u);
                        if (kVec && nj == kN) {
                            if (in) raw[s][h] = __ldcs(reinterpret_cast<const uint4*>(row));
                        } else if (in) {
                            float g[kN];
#pragma unroll
                            for (int e = 0; e < kN; ++e) g[e] = e < nj ? rp_float(row[e]) : 0.f;
                            raw[s][h] = RpVec<T>::pack(g);
                        }
                    }
            };
            auto add = [&](const uint4 (&raw)[kU][kH], int r) {
#pragma unroll
                for (int s = 0; s < kU; ++s) {
                    const int rr = r + s * side;
                    if (rr >= r1) break;
                    const int q = sq[rr];
                    const Seg qs = sg[rr];
                    const bool apart = one_seg && ks[0] != qs;
                    const int ulo = rp_bucket(lut, p.M, q - kmax), uhi = rp_bucket(lut, p.M, q - kmin);
                    float g[kH][kN];
#pragma unroll
                    for (int h = 0; h < kH; ++h) RpVec<T>::unpack(raw[s][h], g[h]);
                    if (apart || (one_seg && ulo == uhi)) {
                        move_to(apart ? p.rows - 1 : ulo);
#pragma unroll
                        for (int h = 0; h < kH; ++h) {
#pragma unroll
                            for (int w = kN / 2; w >= 1; w >>= 1)
#pragma unroll
                                for (int e = 0; e < w; ++e) g[h][e] += g[h][e + w];
                            sum[h] += g[h][0];
                        }
                    } else {
                        int u[kN];
#pragma unroll
                        for (int e = 0; e < kN; ++e) {
                            u[e] = rp_bucket(lut, p.M, q - kp[e]);
                            if (ks[e] != qs) u[e] = p.rows - 1;
                        }
#pragma unroll
                        for (int e = 0; e < kN; ++e) {
                            if (e < nj) {
                                move_to(u[e]);
#pragma unroll
                                for (int h = 0; h < kH; ++h) sum[h] += g[h][e];
                            }
                        }
                    }
                }
            };
            uint4 x[kU][kH], y[kU][kH];
            const int step = kU * side;
            load(x, ty);
            for (int r = ty; r < r1; r += 2 * step) {
                load(y, r + step);
                add(x, r);
                load(x, r + 2 * step);
                add(y, r + step);
            }
        }
    }
#pragma unroll
    for (int h = 0; h < kH; ++h) acc[(run * kH + h) * nt + tid] += sum[h];
    __syncthreads();
    // a warp per sum: lanes over the threads' columns
    const int warp = tid >> 5, lane = tid & 31, warps = nt >> 5;
    constexpr int kX = 4;                   // sums of a warp at a time
    for (int x0 = warp * kX; x0 < p.rows * kH; x0 += warps * kX) {
        float t[kX];
#pragma unroll
        for (int k = 0; k < kX; ++k) {
            t[k] = 0.f;
            if (x0 + k < p.rows * kH)
                for (int e = lane; e < nt; e += 32) t[k] += acc[(x0 + k) * nt + e];
        }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1)
#pragma unroll
            for (int k = 0; k < kX; ++k) t[k] += __shfl_xor_sync(0xffffffffu, t[k], o);
#pragma unroll
        for (int k = 0; k < kX; ++k) {
            const int u = (x0 + k) / kH, h = h0 + (x0 + k) % kH;
            if (lane == 0 && u < p.rows && h < p.C) partial[((long long)blockIdx.x * p.rows + u) * p.C + h] = t[k];
        }
    }
}

// ---------------------------------------------------------------------------------------
// pair, gradient of the table.  A warp owns a run of consecutive positions and 32 kL channels (blockIdx.y), kL per lane,
// and a private set of sums [rows][32 kL] in shared memory; the running bucket's sum stays in registers until the bucket
// changes (the test is uniform over the warp).
// ---------------------------------------------------------------------------------------
template <typename T, int kL> struct RpLane { using V = T; };             // kL channels of a lane
template <> struct RpLane<__nv_bfloat16, 4> { using V = uint2; };
template <> struct RpLane<float, 4> { using V = float4; };
template <int kL> struct RpSum { f32x2 v[(kL + 1) / 2]; };                // kL sums as packed pairs
__device__ __forceinline__ void rp_add(RpSum<1>& s, const __nv_bfloat16& v) { s.v[0] = f2_add(s.v[0], f2_pack(__bfloat162float(v), 0.f)); }
__device__ __forceinline__ void rp_add(RpSum<1>& s, const float& v) { s.v[0] = f2_add(s.v[0], f2_pack(v, 0.f)); }
__device__ __forceinline__ void rp_add(RpSum<4>& s, const uint2& v) {
    s.v[0] = f2_add(s.v[0], f2_from_bf16x2(v.x));
    s.v[1] = f2_add(s.v[1], f2_from_bf16x2(v.y));
}
__device__ __forceinline__ void rp_add(RpSum<4>& s, const float4& v) {
    s.v[0] = f2_add(s.v[0], f2_pack(v.x, v.y));
    s.v[1] = f2_add(s.v[1], f2_pack(v.z, v.w));
}
// the sums to their bucket's row in shared memory, and back to zero
template <int kL> __device__ __forceinline__ void rp_flush(float* acc, int row, RpSum<kL>& s) {
    float f[(kL + 1) / 2 * 2];
#pragma unroll
    for (int e = 0; e < (kL + 1) / 2; ++e) {
        f2_unpack(s.v[e], f[2 * e], f[2 * e + 1]);
        s.v[e] = 0ull;
    }
    float* a = acc + row * 32 * kL;
    if constexpr (kL == 4) {
        float4 x = *reinterpret_cast<float4*>(a);
        x.x += f[0]; x.y += f[1]; x.z += f[2]; x.w += f[3];
        *reinterpret_cast<float4*>(a) = x;
    } else {
        a[0] += f[0];
    }
}

// `kRun` positions of one warp (their channels of this lane, and a bucket per lane).  Two of them live in registers: one is
// added up while the other is in flight.
template <typename T, int kL, int kRun>
struct RpRun {
    typename RpLane<T, kL>::V g[kRun];
    int u, n;
    __device__ __forceinline__ void load(const RelposParams& p, const uint16_t* lut, const T* grad, long long pos, long long last, int c0,
                                         int lane, RpCursor& cur) {
        using V = typename RpLane<T, kL>::V;
        n = (int)max(0ll, min((long long)kRun, last - pos));
        const char* src = reinterpret_cast<const char*>(grad + pos * p.C + c0);
        const uint32_t step = (uint32_t)p.C * (uint32_t)sizeof(T);
        if (n == kRun && c0 < p.C) {
#pragma unroll
            for (int s = 0; s < kRun; ++s) g[s] = __ldcs(reinterpret_cast<const V*>(src + s * step));
        } else {
#pragma unroll
            for (int s = 0; s < kRun; ++s) {
                g[s] = V();
                if (s < n && c0 < p.C) g[s] = __ldcs(reinterpret_cast<const V*>(src + s * step));
            }
        }
        u = -1;
        if (lane < n) {
            u = cur.bucket(p, lut);
            cur.step(p, kRun);
        }
    }
    __device__ __forceinline__ void add(float* acc, int& run, RpSum<kL>& sum, int lane) const {
        // bit s: position s starts another bucket than the one before it
        const int before = __shfl_up_sync(0xffffffffu, u, 1);
        const uint32_t starts = __ballot_sync(0xffffffffu, lane < n && u != (lane == 0 ? run : before));
        if (n == kRun && starts == 0u) {               // most runs: no test per position
#pragma unroll
            for (int s = 0; s < kRun; ++s) rp_add(sum, g[s]);
            return;
        }
#pragma unroll
        for (int s = 0; s < kRun; ++s) {
            if ((starts >> s) & 1u) {
                rp_flush(acc, run, sum);
                run = __shfl_sync(0xffffffffu, u, s);
            }
            rp_add(sum, g[s]);                         // zero behind the last position
        }
    }
};

template <typename T, int kL>
__global__ void __launch_bounds__(256, 1)
relpos_pair_grad_kernel(const __grid_constant__ RelposParams p, const __grid_constant__ trimul_buckets rule,
                                        const T* grad, float* partial, long long pos_per_warp) {
    constexpr int kRun = sizeof(T) * kL == 16 ? 16 : 32;      // 64 registers a run
    extern __shared__ __align__(16) uint8_t rp_smem[];
    const int nt = blockDim.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = nt >> 5;
    float* sums = reinterpret_cast<float*>(rp_smem);                              // [warps][rows][32 kL]
    uint16_t* lut = reinterpret_cast<uint16_t*>(rp_smem + (size_t)warps * p.rows * 32 * kL * 4);
    rp_build_lut(lut, rule, p.M);
    for (int e = tid; e < warps * p.rows * 32 * kL; e += nt) sums[e] = 0.f;
    griddep_wait();
    griddep_launch_dependents();
    __syncthreads();
    const int c0 = blockIdx.y * 32 * kL + lane * kL;
    float* acc = sums + (size_t)warp * p.rows * 32 * kL + lane * kL;
    const long long total = (long long)p.B * p.Lq * p.Lk;
    const long long first = ((long long)blockIdx.x * warps + warp) * pos_per_warp, last = min(first + pos_per_warp, total);
    int run = 0;
    RpSum<kL> sum = {};
    RpCursor cur;
    if (first < last) cur.init(p, min(first + lane, total - 1));
    RpRun<T, kL, kRun> a, b;
    a.load(p, lut, grad, first, last, c0, lane, cur);
    for (long long pos = first; pos < last; pos += 2 * kRun) {
        b.load(p, lut, grad, pos + kRun, last, c0, lane, cur);
        a.add(acc, run, sum, lane);
        a.load(p, lut, grad, pos + 2 * kRun, last, c0, lane, cur);
        b.add(acc, run, sum, lane);
    }
    rp_flush(acc, run, sum);
    __syncthreads();
    const int width = min(32 * kL, p.C - (int)blockIdx.y * 32 * kL);
    for (int e = tid; e < p.rows * 32 * kL; e += nt) {
        const int c = e % (32 * kL), u = e / (32 * kL);
        if (c >= width) continue;
        float t = 0.f;
        for (int w = 0; w < warps; ++w) t += sums[(size_t)w * p.rows * 32 * kL + e];
        partial[((long long)blockIdx.x * p.rows + u) * p.C + blockIdx.y * 32 * kL + c] = t;
    }
}

// partial [parts][n] -> out [n], in a fixed order: eight threads share an output's parts.
constexpr int kRpReduceThreads = 256;
__global__ void __launch_bounds__(kRpReduceThreads)
relpos_reduce_kernel(const float* partial, void* out, int out_bf16, int parts, int n) {
    __shared__ float s[8][33];
    griddep_wait();
    griddep_launch_dependents();
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const int o = blockIdx.x * 32 + x;
    float t = 0.f;
    if (o < n) {
#pragma unroll 8
        for (int k = y; k < parts; k += 8) t += partial[(long long)k * n + o];
    }
    s[y][x] = t;
    __syncthreads();
    if (y == 0 && o < n) {
        for (int k = 1; k < 8; ++k) t += s[k][x];
        if (out_bf16) static_cast<__nv_bfloat16*>(out)[o] = __float2bfloat16_rn(t);
        else static_cast<float*>(out)[o] = t;
    }
}

}  // namespace trimul

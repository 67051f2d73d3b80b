// What a call prepares before its main kernel, in one launch of as many kinds of blocks as the call needs: the key mask as bits
// with a list of the tiles that keep something, a bias as rows that TMA can fetch, and the backward pass's delta.  They need nothing
// of each other, and a small call's time is its launches (2 x 61 x 77, 8 heads of 32, odd bias and mask, against a launch each:
// forward 9.7 -> 7.7 us, forward and backward 22.7 -> 17.3).  512 threads a block: with 1024 only one fits on an SM, 2 us more for
// the delta of 2048 x 16 heads of 128.
#pragma once

#include "attn_plain.cuh"

namespace trimul {

constexpr int kPrepThreads = 512;
constexpr int kPrepWarps = kPrepThreads / 32;

struct AttnPrep {
    int mask_blocks, bias_blocks;          // in this order; the rest of the grid is delta's
    int n_tiles;                           // key tiles of the mask
    uint32_t* words;                       // [B][n_tiles][4] bits of a tile's keys
    int* list;                             // [B][1 + n_tiles]: how many tiles keep something, and which
    uint32_t* bias;                        // [bias_batch][bias_heads][Lq][bias_pitch]
    int bias_heads, bias_pitch;
    long long bias_rows;
};

// A bias whose rows do not start on 16 bytes, as rows that do: two neighbouring values a thread, so that a warp reads and
// writes 128 bytes in a row.
__device__ __forceinline__ void attn_bias_rows_block(const AttnParams& p, const AttnPrep& w, int block) {
    constexpr int kU = 4;
    const int words = w.bias_pitch / 2;
    for (long long r = (long long)block * kPrepWarps + (threadIdx.x >> 5); r < w.bias_rows; r += (long long)w.bias_blocks * kPrepWarps) {
        const int i = (int)(r % p.Lq);
        const long long bh = r / p.Lq;
        const __nv_bfloat16* s = static_cast<const __nv_bfloat16*>(p.bias) + bh / w.bias_heads * p.bias_b + bh % w.bias_heads * p.bias_h + i * p.bias_i;
        for (int w0 = threadIdx.x & 31; w0 < words; w0 += 32 * kU) {
            __nv_bfloat162 v[kU];
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int j = 2 * (w0 + 32 * u);
                v[u].x = j < p.Lk ? s[j] : __nv_bfloat16();
                v[u].y = j + 1 < p.Lk ? s[j + 1] : __nv_bfloat16();
            }
#pragma unroll
            for (int u = 0; u < kU; ++u)
                if (w0 + 32 * u < words) w.bias[r * words + w0 + 32 * u] = *reinterpret_cast<const uint32_t*>(&v[u]);
        }
    }
}

// Key mask as bits, and the list of tiles that keep something.  A block per batch element.
__device__ __forceinline__ void attn_mask_block(const AttnParams& p, const AttnPrep& w, int b) {
    __shared__ int any[kPrepWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint8_t* m = p.mask + b * p.mask_b;
    int* out = w.list + (long long)b * (w.n_tiles + 1);
    int count = 0;
    for (int t0 = 0; t0 < w.n_tiles; t0 += kPrepWarps) {
        const int t = t0 + warp;
        uint32_t all = 0;
        if (t < w.n_tiles) {
            uint32_t bits[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int j = t * 128 + k * 32 + lane;
                bits[k] = __ballot_sync(0xffffffffu, j < p.Lk && m[min(j, p.Lk - 1)] != 0);
                all |= bits[k];
            }
            if (lane == 0)
                *reinterpret_cast<uint4*>(w.words + ((long long)b * w.n_tiles + t) * 4) = make_uint4(bits[0], bits[1], bits[2], bits[3]);
        }
        if (lane == 0) any[warp] = all != 0;
        __syncthreads();
        int before = 0, total = 0;
        for (int k = 0; k < kPrepWarps; ++k) {
            if (k < warp) before += any[k];
            total += any[k];
        }
        if (lane == 0 && all != 0) out[1 + count + before] = t;
        count += total;
        __syncthreads();
    }
    if (threadIdx.x == 0) out[0] = count;
}

// delta_i = sum_d dout_id o_id, kLanes lanes per row (four columns a piece where rows allow it).  With 16-bit outputs the part
// that rounding took off o is added back: where the probabilities' gradients nearly cancel against delta, half a step of o
// would be all that is left.
template <typename T, int kLanes>
__device__ __forceinline__ void attn_delta_block(const AttnParams& p, int block) {
    const long long row = ((long long)block * kPrepThreads + threadIdx.x) / kLanes;
    const int lane = threadIdx.x % kLanes;
    const bool in = row < (long long)p.B * p.Lq * p.H;
    float t = 0.f;
    int h = 0, i = 0, b = 0;
    if (in) {
        h = (int)(row % p.H);
        const long long bi = row / p.H;
        i = (int)(bi % p.Lq);
        b = (int)(bi / p.Lq);
        const T* o = static_cast<const T*>(p.o.p) + b * p.o.b + (long long)i * p.o.l + h * p.o.h;
        const T* g = static_cast<const T*>(p.dout.p) + b * p.dout.b + (long long)i * p.dout.l + h * p.dout.h;
        const T* lo = sizeof(T) == 2 && p.o_lo != nullptr ? static_cast<const T*>(p.o_lo) + row * p.D : nullptr;
        if (ap_vec<T>(p.o, p.D) && ap_vec<T>(p.dout, p.D) && (lo == nullptr || (reinterpret_cast<uintptr_t>(lo) & 7) == 0)) {
            using V = typename ApRaw<T>::V;
            for (int d = lane * 4; d < p.D; d += kLanes * 4) {
                float4 y = ap_wide(*reinterpret_cast<const V*>(o + d));
                const float4 x = ap_wide(*reinterpret_cast<const V*>(g + d));
                if (lo != nullptr) {
                    const float4 z = ap_wide(*reinterpret_cast<const V*>(lo + d));
                    y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
                }
                t = fmaf(y.x, x.x, fmaf(y.y, x.y, fmaf(y.z, x.z, fmaf(y.w, x.w, t))));
            }
        } else {
            for (int d = lane; d < p.D; d += kLanes) t = fmaf(at_float(o[d]) + (lo != nullptr ? at_float(lo[d]) : 0.f), at_float(g[d]), t);
        }
    }
#pragma unroll
    for (int s = kLanes / 2; s >= 1; s >>= 1) t += __shfl_xor_sync(0xffffffffu, t, s);
    if (in && lane == 0) p.delta[((long long)b * p.H + h) * p.Lq + i] = t;
}

template <typename T, int kLanes>
__global__ void __launch_bounds__(kPrepThreads)
attn_prep_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ AttnPrep w) {
    griddep_wait();
    griddep_launch_dependents();
    const int block = blockIdx.x;
    if (block < w.mask_blocks) attn_mask_block(p, w, block);
    else if (block < w.mask_blocks + w.bias_blocks) attn_bias_rows_block(p, w, block - w.mask_blocks);
    else attn_delta_block<T, kLanes>(p, block - w.mask_blocks - w.bias_blocks);
}

}  // namespace trimul

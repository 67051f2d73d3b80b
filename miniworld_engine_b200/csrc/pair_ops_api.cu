// C-ABI of the operators beside the block: the relative position bias by buckets and cross attention.  Argument
// checks, choice of kernel and launches; declarations in include/trimul_b200.h.  Nothing here allocates device
// memory, synchronises or throws.

#include "../../include/trimul_b200.h"

#include <algorithm>
#include <cstddef>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "host_common.cuh"
#include "attn_bwd_sm100.cuh"
#include "attn_fwd64_sm100.cuh"
#include "attn_fwd_sm100.cuh"
#include "attn_plain.cuh"
#include "attn_prep.cuh"
#include "attn_short.cuh"
#include "relpos_kernels.cuh"

using namespace trimul;

namespace {

constexpr int kMaxSmem = 227 * 1024;
inline bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t align_up(int64_t v, int64_t m) { return ceil_div(v, m) * m; }
inline int elem_size(int dtype) { return dtype == TRIMUL_DTYPE_BF16 ? 2 : 4; }
inline bool known_dtype(int d) { return d == TRIMUL_DTYPE_BF16 || d == TRIMUL_DTYPE_FP32; }

// ---------------------------------------------------------------------------------------
// relative position bias
// ---------------------------------------------------------------------------------------
int lut_reach(const trimul_buckets* b) {       // distances beyond it share the outermost buckets
    if (b->kind == TRIMUL_BUCKETS_CLIPPED) return b->max_distance;
    const int near = b->kind == TRIMUL_BUCKETS_LOG ? b->count / 4 : b->count / 2;
    return b->n_thresholds > 0 ? b->thresholds[b->n_thresholds - 1] : near;
}

int check_buckets(const trimul_buckets* b) {
    if (b == nullptr || b->count <= 0) return TRIMUL_E_INVALID;
    if (b->kind == TRIMUL_BUCKETS_CLIPPED) {
        if (b->max_distance < 0 || (int64_t)b->count != 2 * (int64_t)b->max_distance + 1) return TRIMUL_E_INVALID;
    } else if (b->kind == TRIMUL_BUCKETS_LOG || b->kind == TRIMUL_BUCKETS_CAUSAL) {
        if (b->kind == TRIMUL_BUCKETS_LOG && (b->count % 2) != 0) return TRIMUL_E_INVALID;
        const int half = b->kind == TRIMUL_BUCKETS_LOG ? b->count / 2 : b->count, near = half / 2;
        if (near < 1 || b->n_thresholds < 0 || b->n_thresholds > TRIMUL_MAX_THRESHOLDS) return TRIMUL_E_INVALID;
        if (near + b->n_thresholds > half - 1) return TRIMUL_E_INVALID;
        for (int i = 0; i < b->n_thresholds; ++i)
            if (b->thresholds[i] < (i == 0 ? near : b->thresholds[i - 1])) return TRIMUL_E_INVALID;
    } else {
        return TRIMUL_E_INVALID;
    }
    if ((int64_t)b->count + (b->segments != 0) > TRIMUL_MAX_BUCKETS) return TRIMUL_E_UNSUPPORTED;
    if (lut_reach(b) > TRIMUL_MAX_LUT) return TRIMUL_E_UNSUPPORTED;
    return TRIMUL_OK;
}

int check_relpos(const trimul_relpos_desc* d, const trimul_buckets* b) {
    if (d == nullptr || d->struct_bytes != sizeof(trimul_relpos_desc)) return TRIMUL_E_INVALID;
    const int rc = check_buckets(b);
    if (rc != TRIMUL_OK) return rc;
    if (d->layout != TRIMUL_RELPOS_HEADS && d->layout != TRIMUL_RELPOS_PAIR) return TRIMUL_E_INVALID;
    if (!known_dtype(d->dtype) || !known_dtype(d->table_dtype)) return TRIMUL_E_INVALID;
    if (d->B <= 0 || d->Lq <= 0 || d->Lk <= 0 || d->channels <= 0) return TRIMUL_E_INVALID;
    if (d->wide_index < 0 || d->wide_index > 15) return TRIMUL_E_INVALID;
    if (d->channels > 8192 || d->Lk > (1 << 24)) return TRIMUL_E_UNSUPPORTED;
    if ((int64_t)d->B * d->Lq > (1 << 30)) return TRIMUL_E_UNSUPPORTED;
    if (d->layout == TRIMUL_RELPOS_HEADS &&
        (d->stride_b < 0 || d->stride_h < 0 || d->stride_i < 0)) return TRIMUL_E_INVALID;
    return TRIMUL_OK;
}

RelposParams relpos_params(const trimul_relpos_desc* d, const trimul_buckets* b, const void* table, const void* q_pos,
                           const void* k_pos, const void* q_seg, const void* k_seg) {
    RelposParams p = {};
    p.B = d->B; p.Lq = d->Lq; p.Lk = d->Lk; p.C = d->channels;
    p.rows = b->count + (b->segments != 0);
    p.M = lut_reach(b);
    p.q_pos = q_pos; p.k_pos = k_pos;
    if (b->segments != 0) { p.q_seg = q_seg; p.k_seg = k_seg; }
    p.q_pos_b = d->q_pos_b; p.k_pos_b = d->k_pos_b; p.q_seg_b = d->q_seg_b; p.k_seg_b = d->k_seg_b;
    p.q_pos64 = d->wide_index & 1; p.k_pos64 = (d->wide_index >> 1) & 1;
    p.q_seg64 = (d->wide_index >> 2) & 1; p.k_seg64 = (d->wide_index >> 3) & 1;
    p.table = table;
    p.table_bf16 = d->table_dtype == TRIMUL_DTYPE_BF16;
    p.sB = d->stride_b; p.sH = d->stride_h; p.sI = d->stride_i;
    return p;
}

inline int lut_bytes(int M) { return (2 * M + 1) * 2; }

template <typename T>
int run_relpos_forward(const trimul_relpos_desc* d, const trimul_buckets* b, const RelposParams& p, const void* add,
                       void* out, cudaStream_t st) {
    constexpr int kN = RpVec<T>::kN;
    if (d->layout == TRIMUL_RELPOS_HEADS) {
        const int64_t items = (int64_t)d->B * d->Lq * ceil_div(d->Lk, kN);
        const int groups = (int)ceil_div(d->channels, kN);
        const int64_t blocks = std::min<int64_t>(ceil_div(items, kRpThreads), ceil_div(16 * (int64_t)sm_count(), groups));
        const int smem = ((p.rows + 63) & ~63) * 16 + lut_bytes(p.M);
        if (!ensure_smem(relpos_heads_kernel<T>, TRIMUL_MAX_BUCKETS * 16 + lut_bytes(TRIMUL_MAX_LUT))) return TRIMUL_E_CUDA;
        return launch_stage(relpos_heads_kernel<T>, dim3((unsigned)blocks, (unsigned)groups), kRpThreads, smem, st, true, p, *b,
                            static_cast<T*>(out));
    }
    // 16-byte pieces of channels where the tensors allow them
    const bool vec = (d->channels % kN) == 0 && aligned(add, 16) && aligned(out, 16) && aligned(p.table, 16);
    const int per_pos = vec ? d->channels / kN : d->channels;
    const int64_t total = (int64_t)d->B * d->Lq * d->Lk;
    // eight pieces a thread at least, then as many positions as make all blocks resident at once
    const int64_t per_block = std::max<int64_t>(ceil_div(total, 8 * (int64_t)sm_count()), ceil_div(8 * kRpPairThreads, per_pos));
    if (per_block > (1 << 30)) return TRIMUL_E_UNSUPPORTED;
    const dim3 grid((unsigned)ceil_div(total, per_block));
    auto kernel = vec ? relpos_pair_kernel<T, true> : relpos_pair_kernel<T, false>;
    if (!ensure_smem(kernel, lut_bytes(TRIMUL_MAX_LUT) + 4 * kRpPairThreads)) return TRIMUL_E_CUDA;
    return launch_stage(kernel, grid, kRpPairThreads, lut_bytes(p.M) + 4 * kRpPairThreads, st, true, p, *b, static_cast<const T*>(add),
                        static_cast<T*>(out), (int)per_block);
}

inline bool wide_segments(const trimul_relpos_desc* d, const trimul_buckets* b) { return b->segments != 0 && (d->wide_index & 12) != 0; }

// Launch shape of the gradient: `parts` partial tables of rows * channels sums each.
struct RelposGradPlan {
    int threads, smem, parts, lane_channels, column_blocks, parts_per_b, heads;
    int64_t per_part;          // rows (heads) or positions of a warp (pair)
};
RelposGradPlan plan_relpos_grad(const trimul_relpos_desc* d, const trimul_buckets* b, bool wide_lanes) {
    RelposGradPlan g = {};
    const int rows = b->count + (b->segments != 0), lut = lut_bytes(lut_reach(b));
    const int kN = d->dtype == TRIMUL_DTYPE_BF16 ? 8 : 4;
    if (d->layout == TRIMUL_RELPOS_HEADS) {
        // four heads a block where three blocks' sums fit into an SM's shared memory, two where that holds for them; one head
        // (and more rows at once) where there is little to do
        g.threads = 128;
        const int64_t all = (int64_t)d->B * d->Lq * d->Lk * d->channels;
        g.heads = all < (8 << 20) ? 1 : d->channels >= 4 && rows * 4 * 128 * 4 <= 72 * 1024 ? 4 : d->channels >= 2 && rows * 2 * 128 * 4 <= 72 * 1024 ? 2 : 1;
        while (g.threads > 32 && rows * g.threads * 4 > 96 * 1024) g.threads /= 2;
        // as many blocks as are resident at once, parts of at least four steps and at most 1024 rows (whose positions a
        // block keeps)
        const int sums = rows * g.heads * g.threads * 4, nch = (int)ceil_div(d->Lk, kN);
        const int side = std::max(1, g.threads / std::min(nch, g.threads));
        const int64_t resident = std::max(1, std::min(5, kMaxSmem / (sums + 4096)));
        const int64_t parts = std::max<int64_t>(1, resident * sm_count() / ceil_div(d->channels, g.heads) / d->B);
        g.per_part = std::min<int64_t>(1024, std::max<int64_t>(ceil_div(d->Lq, parts), std::min<int64_t>(16 / g.heads * side, d->Lq)));
        g.parts_per_b = (int)ceil_div(d->Lq, g.per_part);
        g.parts = d->B * g.parts_per_b;
        g.column_blocks = (int)ceil_div(d->channels, g.heads);
        g.smem = sums + (int)g.per_part * (wide_segments(d, b) ? 12 : 8) + lut;
        return g;
    }
    const int64_t total = (int64_t)d->B * d->Lq * d->Lk;
    g.lane_channels = wide_lanes && rows * 128 * 4 + lut <= kMaxSmem ? 4 : 1;
    const int copy = rows * 32 * g.lane_channels * 4;
    const int warps = std::min(8, (kMaxSmem - lut) / copy);
    g.threads = 32 * warps;
    g.smem = warps * copy + lut;
    g.column_blocks = (int)ceil_div(d->channels, 32 * g.lane_channels);
    const int64_t blocks = std::max<int64_t>(1, sm_count() / g.column_blocks);
    g.per_part = align_up(std::max<int64_t>(ceil_div(total, blocks * warps), 32), 32);
    g.parts = (int)ceil_div(total, g.per_part * warps);
    return g;
}

// whether a lane of the pair gradient may take four channels at a time
bool wide_lanes(const trimul_relpos_desc* d, const void* grad) {
    return (d->channels % 4) == 0 && aligned(grad, 4 * elem_size(d->dtype));
}

template <typename T, typename Seg>
auto heads_grad_kernel(bool vec, int heads) {
    return heads == 4 ? (vec ? relpos_heads_grad_kernel<T, true, 4, Seg> : relpos_heads_grad_kernel<T, false, 4, Seg>)
         : heads == 2 ? (vec ? relpos_heads_grad_kernel<T, true, 2, Seg> : relpos_heads_grad_kernel<T, false, 2, Seg>)
                      : (vec ? relpos_heads_grad_kernel<T, true, 1, Seg> : relpos_heads_grad_kernel<T, false, 1, Seg>);
}

template <typename T>
int run_relpos_grad(const trimul_relpos_desc* d, const trimul_buckets* b, const RelposParams& p, const void* grad,
                    void* dtable, float* partial, cudaStream_t st) {
    constexpr int kN = RpVec<T>::kN;
    int rc;
    const RelposGradPlan g = plan_relpos_grad(d, b, wide_lanes(d, grad));
    if (d->layout == TRIMUL_RELPOS_HEADS) {
        const bool vec = aligned(grad, 16) && (p.sB % kN) == 0 && (p.sH % kN) == 0 && (p.sI % kN) == 0;
        auto kernel = wide_segments(d, b) ? heads_grad_kernel<T, long long>(vec, g.heads) : heads_grad_kernel<T, int>(vec, g.heads);
        if (!ensure_smem(kernel, kMaxSmem)) return TRIMUL_E_CUDA;
        rc = launch_stage(kernel, dim3((unsigned)g.parts, (unsigned)g.column_blocks), g.threads, g.smem, st, true, p, *b,
                          static_cast<const T*>(grad), partial, g.parts_per_b, (int)g.per_part);
    } else {
        auto kernel = g.lane_channels == 4 ? relpos_pair_grad_kernel<T, 4> : relpos_pair_grad_kernel<T, 1>;
        if (!ensure_smem(kernel, kMaxSmem)) return TRIMUL_E_CUDA;
        rc = launch_stage(kernel, dim3((unsigned)g.parts, (unsigned)g.column_blocks), g.threads, g.smem, st, true, p, *b,
                          static_cast<const T*>(grad), partial, (long long)g.per_part);
    }
    if (rc != TRIMUL_OK || partial == dtable) return rc;
    const int n = p.rows * p.C;
    return launch_stage(relpos_reduce_kernel, dim3((unsigned)ceil_div(n, 32)), kRpReduceThreads, 0, st, true,
                        static_cast<const float*>(partial), dtable, p.table_bf16, g.parts, n);
}

// ---------------------------------------------------------------------------------------
// cross attention
// ---------------------------------------------------------------------------------------
int check_attn(const trimul_attn_desc* d) {
    if (d == nullptr || d->struct_bytes != sizeof(trimul_attn_desc)) return TRIMUL_E_INVALID;
    if (!known_dtype(d->dtype)) return TRIMUL_E_INVALID;
    if (d->B <= 0 || d->Lq <= 0 || d->Lk <= 0 || d->H <= 0 || d->Hk <= 0 || d->D <= 0) return TRIMUL_E_INVALID;
    if ((d->H % d->Hk) != 0) return TRIMUL_E_INVALID;
    if (d->D > 256 || d->B > 65535 || d->H > 65535) return TRIMUL_E_UNSUPPORTED;
    if (!aligned(d->stats, 8)) return TRIMUL_E_INVALID;         // read and written as pairs
    if (d->Lq > (1 << 24) || d->Lk > (1 << 24)) return TRIMUL_E_UNSUPPORTED;
    if ((d->bias != nullptr || d->dbias != nullptr) &&
        ((d->bias_batch != 1 && d->bias_batch != d->B) || (d->bias_heads != 1 && d->bias_heads != d->H)))
        return TRIMUL_E_INVALID;
    if (d->dbias != nullptr) {
        const int n = 16 / elem_size(d->dtype);
        if (d->bias == nullptr || !aligned(d->dbias, 16)) return TRIMUL_E_INVALID;
        if ((d->dbias_b % n) || (d->dbias_h % n) || (d->dbias_i % n) || d->dbias_i < align_up(d->Lk, n)) return TRIMUL_E_INVALID;
    }
    return TRIMUL_OK;
}
inline bool sums_bias(const trimul_attn_desc* d) {
    return d->dbias != nullptr && ((d->bias_batch == 1 && d->B > 1) || (d->bias_heads == 1 && d->H > 1));
}
inline AttnTensor tensor_of(const trimul_attn_tensor& t) { return AttnTensor{t.p, t.b, t.l, t.h}; }

AttnParams attn_params(const trimul_attn_desc* d, int32_t* status) {
    AttnParams p = {};
    p.B = d->B; p.Lq = d->Lq; p.Lk = d->Lk; p.H = d->H; p.Hk = d->Hk; p.D = d->D;
    p.scale = d->scale;
    p.q = tensor_of(d->q); p.k = tensor_of(d->k); p.v = tensor_of(d->v); p.o = tensor_of(d->o);
    p.dout = tensor_of(d->dout); p.dq = tensor_of(d->dq); p.dk = tensor_of(d->dk); p.dv = tensor_of(d->dv);
    p.bias = d->bias;
    p.bias_b = d->bias_batch == 1 ? 0 : d->bias_b;
    p.bias_h = d->bias_heads == 1 ? 0 : d->bias_h;
    p.bias_i = d->bias_i;
    p.mask = d->mask; p.mask_b = d->mask_b;
    p.stats = reinterpret_cast<float2*>(d->stats);
    p.o_lo = d->dtype == TRIMUL_DTYPE_BF16 ? d->o_lo : nullptr;
    p.status = status;
    return p;
}

// ---------------------------------------------------------------------------------------
// choice of kernels.  Tensor cores: bf16 whose rows TMA can fetch (16-byte aligned, no axis repeated in place)
// ---------------------------------------------------------------------------------------
bool tma_rows(const trimul_attn_tensor& t, int L, int H, int B) {
    auto ok = [](int n, int64_t s) { return n == 1 || (s > 0 && (s % 8) == 0); };
    return aligned(t.p, 16) && ok(L, t.l) && ok(H, t.h) && ok(B, t.b);
}
bool tensor_cores(const trimul_attn_desc* d) {
    if (d->dtype != TRIMUL_DTYPE_BF16 || (d->flags & TRIMUL_ATTN_FLAG_PLAIN) != 0) return false;
    return (d->D % 8) == 0 && d->D <= 128;
}
bool copies_bias(const trimul_attn_desc* d) {
    return tensor_cores(d) && d->bias != nullptr && (d->flags & TRIMUL_ATTN_FLAG_COPY_BIAS) != 0;
}
bool tensor_core_forward(const trimul_attn_desc* d) {
    if (!tensor_cores(d) || !tma_rows(d->q, d->Lq, d->H, d->B) || !tma_rows(d->k, d->Lk, d->Hk, d->B) ||
        !tma_rows(d->v, d->Lk, d->Hk, d->B) || !tma_rows(d->o, d->Lq, d->H, d->B) || !aligned(d->o_lo, 16))
        return false;
    if (d->bias == nullptr || copies_bias(d)) return true;
    return tma_rows(trimul_attn_tensor{const_cast<void*>(d->bias), d->bias_b, d->bias_i, d->bias_h}, d->Lq, d->bias_heads, d->bias_batch);
}

bool tensor_core_backward(const trimul_attn_desc* d) {
    return tensor_core_forward(d) && tma_rows(d->dout, d->Lq, d->H, d->B) && tma_rows(d->dq, d->Lq, d->H, d->B) &&
           tma_rows(d->dk, d->Lk, d->Hk, d->B) && tma_rows(d->dv, d->Lk, d->Hk, d->B);
}

bool encode_rows(CUtensorMap* map, const AttnTensor& t, int D, int L, int H, int B) {
    const uint64_t dims[4] = {(uint64_t)D, (uint64_t)L, (uint64_t)H, (uint64_t)B};
    const uint64_t any = (uint64_t)align_up(D, 8);       // of an axis with one entry
    const uint64_t strides[3] = {L > 1 ? (uint64_t)t.l : any, H > 1 ? (uint64_t)t.h : any, B > 1 ? (uint64_t)t.b : any};
    const uint32_t box[4] = {64, kAfRows, 1, 1};
    return encode_bf16(map, t.p, 4, dims, strides, box, 128);
}
bool encode_bias(CUtensorMap* map, const trimul_attn_desc* d) {
    return encode_rows(map, AttnTensor{const_cast<void*>(d->bias), d->bias_b, d->bias_i, d->bias_h}, d->Lk, d->Lq, d->bias_heads,
                       d->bias_batch);
}

// Few query rows per key head: the kernel that reads keys and values once for all of them.  Its rows are 16-byte pieces.  Where
// the tensor-core kernel is the alternative, it has to serve at least as many heads as queries with each key: 8 x 4096 keys, 16
// key heads of 64 take it 31 / 38 / 57 / 94 us for 1 / 2 / 4 / 8 rows, the tensor-core kernel (which works on 128 rows anyway,
// and again for every query head) 39 us for any number of queries and one query head per key head; with two query heads per
// key head 21 against 39.  Heads of 128: 53 / 68 against 60 us for one and two queries, 39 against 60 for two heads.
constexpr int kShortRows = 8;
bool short_sizes(const trimul_attn_desc* d) {
    const int n = 16 / elem_size(d->dtype), group = d->H / d->Hk;
    if ((d->flags & TRIMUL_ATTN_FLAG_PLAIN) != 0 || (d->D % n) != 0 || d->D > 32 * n) return false;
    return (int64_t)d->Lq * group <= kShortRows && (!tensor_cores(d) || d->Lq <= group);
}
bool short_rows(const trimul_attn_desc* d) {
    const int n = 16 / elem_size(d->dtype);
    auto ok = [&](const trimul_attn_tensor& t) {
        return aligned(t.p, 16) && (t.l % n) == 0 && (t.h % n) == 0 && (t.b % n) == 0;
    };
    return short_sizes(d) && ok(d->k) && ok(d->v);
}
// As many blocks as are resident at once, and keys for two steps of every warp.
int short_splits(const trimul_attn_desc* d) {
    const int64_t blocks = (int64_t)d->B * d->Hk;
    return (int)std::max<int64_t>(1, std::min<int64_t>(as_blocks(d->Lq * (d->H / d->Hk)) * sm_count() / blocks, d->Lk / 256));
}

// Key splits of the forward pass: where the blocks leave SMs idle, each block takes a share of the key tiles and a second kernel
// joins the parts.  Four tiles at least, since the parts cost a launch and their way through memory: 8 heads, 64 queries of 64, us
// with one / two / four tiles at least: 512 keys 10.4 / 10.1 / 8.5, 1024 9.8 / 11.1 / 12.2, 4096 14.7 / 13.4 / 12.9; 4 heads, 256
// queries of 128, 8192 keys 35 / 29 / 25.
int forward_splits(const trimul_attn_desc* d) {
    const int64_t blocks = ceil_div(d->Lq, 2 * kAfRows) * d->H * d->B, tiles = ceil_div(d->Lk, kAfRows);
    const int64_t room = sm_count() / blocks;
    return (int)std::max<int64_t>(1, std::min<int64_t>(room, tiles / 4));
}

// The CUDA-core kernels: rows of a tile, and key splits of the forward pass as above, up to three blocks for two SMs (a step takes
// long enough that one less pays for joining: 2 x 60 queries of 96, 1000 keys 188 -> 23 us, 2 x 256 of 32, 320 keys 27 -> 21).
int plain_rows(const trimul_attn_desc* d, bool backward) { return d->D <= (backward ? 64 : 128) ? 64 : 32; }
int plain_splits(const trimul_attn_desc* d) {
    const int rows = plain_rows(d, false);
    const int64_t blocks = ceil_div(d->Lq, rows) * d->H * d->B, tiles = ceil_div(d->Lk, rows);
    const int64_t splits = std::max<int64_t>(1, std::min<int64_t>(sm_count() * 3 / 2 / blocks, tiles));
    return (int)ceil_div(tiles, ceil_div(tiles, splits));
}

// Backward pass: a block's loop is split among several, whose parts a second kernel adds up, where it is twice as long as a
// block slot's share of all steps: few queries against many keys leave dq to a few long loops, many queries against few keys dk and dv.
// Tensor cores, 8 heads, us whole / split: 61 x 4096 of 64 41 / 20, of 128 46 / 29, 100 x 1024 of 64 13.8 / 10.8, 2048 x 100 of
// 128 37 / 22; a loop just over twice the share (700 x 1400, 4 heads of 128) 21.6 / 24.2, hence `margin`; shares of four steps at
// least instead of two 100 x 1024 12.2, 2048 x 100 25.1.  CUDA cores: 2 x 60 x 1000, 4 heads of 96 208 / 75, 500 x 60, 4 heads of
// 64 128 / 25, 188 x 169, 8 heads of 128 69 / 59.  There, too, one block fits on an SM (156 to 255 registers of 256 threads), but a
// step takes longer, so the shares are half an SM's and the last blocks end closer together.  A training pass in fp32 by half / whole
// shares: 1030 x 1700, a head of 40 152 / 182, 300 x 300, 8 heads of 64 109 / 131, 188 x 169, 8 heads of 128 115 / 125; the other way
// round 4 x 100 x 100, 8 heads of 64 86 / 80, 3 x 333 x 77, 4 heads of 24 51 / 49; no difference at 2 x 512 x 1024, 8 heads of 64.
AttnBwdSplit backward_split(const trimul_attn_desc* d, int rows, int least, int margin, int slots) {
    const int64_t nq = ceil_div(d->Lq, rows), nk = ceil_div(d->Lk, rows), q = nq * d->H * d->B, kv = nk * d->Hk * d->B;
    const int64_t kv_loop = nq * (d->H / d->Hk), share = std::max<int64_t>(least, ceil_div(q * nk + kv * kv_loop, slots));
    auto split = [&](int64_t loop) { return loop >= 2 * share + margin ? ceil_div(loop, ceil_div(loop, loop / share)) : 1; };
    AttnBwdSplit w = {};
    w.q_splits = (int)split(nk);
    w.kv_splits = (int)split(kv_loop);
    w.q_share = (int)ceil_div(nk, w.q_splits);
    w.kv_share = (int)ceil_div(kv_loop, w.kv_splits);
    const int64_t q_blocks = q * w.q_splits, kv_blocks = kv * w.kv_splits;
    const bool fits = q_blocks + kv_blocks <= INT32_MAX;          // one grid; 0 blocks: too many
    w.q_blocks = fits ? (int)q_blocks : 0;
    w.kv_blocks = fits ? (int)kv_blocks : 0;
    w.q_first = w.q_share * 3LL > w.kv_share * 4LL;                // three products a key tile, four a query tile
    return w;
}
AttnBwdSplit backward_split(const trimul_attn_desc* d, bool tensor) {
    return tensor ? backward_split(d, kAfRows, 2, 4, sm_count()) : backward_split(d, plain_rows(d, true), 1, 0, 2 * sm_count());
}
int64_t part_bytes(const trimul_attn_desc* d, const AttnBwdSplit& w, bool q) {
    if ((q ? w.q_splits : w.kv_splits) == 1) return 0;
    return align_up((q ? (int64_t)w.q_splits * d->H * d->Lq : (int64_t)w.kv_splits * d->Hk * d->Lk) * d->B * d->D * 4, 256);
}

// Workspace.  Both directions: the key mask as bits and its list of tiles.  Forward: the parts of split rows.  Backward:
// delta, then the scores' gradients where the bias's gradient sums them.  Depends on sizes, type, flags, the shape of the bias and
// on whether there are a mask and a gradient of the bias, not on addresses or strides.
struct AttnWorkspace {
    int64_t words, list, bias, part_o, part_ml, delta, dq, dk, dv, ds, ds_pitch, total;
};
AttnWorkspace attn_workspace(const trimul_attn_desc* d, bool backward) {
    AttnWorkspace w = {};
    int64_t at = 0;
    const bool tc = tensor_cores(d);
    const int64_t tiles = ceil_div(d->Lk, kAfRows);
    if (tc && d->mask != nullptr) {
        w.words = at;
        at += align_up(d->B * tiles * 16, 256);
        w.list = at;
        at += align_up(d->B * (tiles + 1) * 4, 256);
    }
    if (copies_bias(d)) {
        w.bias = at;
        at += align_up((int64_t)d->bias_batch * d->bias_heads * d->Lq * align_up(d->Lk, 8) * 2, 256);
    }
    // by sizes alone, so that a caller may keep the answer: room for either kernel's parts
    const int splits = backward ? 1 : std::max({short_sizes(d) ? short_splits(d) : 1, tc ? forward_splits(d) : 1, plain_splits(d)});
    if (splits > 1) {
        const int64_t rows = (int64_t)splits * d->B * d->H * d->Lq;
        w.part_o = at;
        at += align_up(rows * d->D * 4, 256);
        w.part_ml = at;
        at += align_up(rows * 8, 256);
    }
    if (backward) {
        w.delta = at;
        at += align_up((int64_t)d->B * d->H * d->Lq * 4, 256);
        int64_t q = 0, kv = 0;
        for (bool tensor : {false, true})
            if (!tensor || tc) {
                const AttnBwdSplit split = backward_split(d, tensor);
                q = std::max(q, part_bytes(d, split, true));
                kv = std::max(kv, part_bytes(d, split, false));
            }
        w.dq = at;
        w.dk = w.dq + q;
        w.dv = w.dk + kv;
        at = w.dv + kv;
        w.ds = at;
        w.ds_pitch = align_up(d->Lk, 8);
        if (sums_bias(d)) at += align_up((int64_t)d->B * d->H * d->Lq * w.ds_pitch * 4, 256);
    }
    w.total = at;
    return w;
}

template <typename T>
int run_combine(const AttnParams& p, const float* part_o, const float2* part_ml, int splits, cudaStream_t st) {
    const int64_t rows = (int64_t)p.B * p.H * p.Lq;
    return launch_stage(attn_combine_kernel<T>, dim3((unsigned)ceil_div(rows, 8)), 256, 0, st, true, p, part_o, part_ml, splits);
}

template <typename T, int kT, int kC>
int launch_plain_fwd(const AttnParams& p, int splits, float* part_o, float2* part_ml, cudaStream_t st) {
    auto kernel = attn_plain_fwd_kernel<T, kT, kC>;
    if (!ensure_smem(kernel, ap_smem<kT>(16 * kC, 3, 1))) return TRIMUL_E_CUDA;
    const int rc = launch_stage(kernel, dim3((unsigned)ceil_div(p.Lq, kT), p.H, p.B * splits), kApThreads, ap_smem<kT>(p.D, 3, 1), st, true,
                                p, splits, (int)ceil_div(ceil_div(p.Lk, kT), splits), part_o, part_ml);
    return rc != TRIMUL_OK || splits == 1 ? rc : run_combine<T>(p, part_o, part_ml, splits, st);
}
template <typename T, int kT, int kC> int launch_plain_bwd(const AttnParams& p, const AttnBwdSplit& w, cudaStream_t st) {
    auto kernel = attn_plain_bwd_kernel<T, kT, kC>;
    if (!ensure_smem(kernel, ap_smem<kT>(16 * kC, 4, 2))) return TRIMUL_E_CUDA;
    return launch_stage(kernel, dim3((unsigned)(w.kv_blocks + w.q_blocks)), kApThreads, ap_smem<kT>(p.D, 4, 2), st, true, p, w);
}
template <typename T> int run_plain_fwd(const trimul_attn_desc* d, const AttnParams& p, const AttnWorkspace& w, uint8_t* ws, cudaStream_t st) {
    const int splits = plain_splits(d);
    float* o = splits > 1 ? reinterpret_cast<float*>(ws + w.part_o) : nullptr;
    float2* ml = reinterpret_cast<float2*>(ws + w.part_ml);
    if (p.D <= 32) return launch_plain_fwd<T, 64, 2>(p, splits, o, ml, st);
    if (p.D <= 64) return launch_plain_fwd<T, 64, 4>(p, splits, o, ml, st);
    if (p.D <= 128) return launch_plain_fwd<T, 64, 8>(p, splits, o, ml, st);
    return launch_plain_fwd<T, 32, 16>(p, splits, o, ml, st);
}
template <typename T> int run_plain_bwd(const AttnParams& p, const AttnBwdSplit& w, cudaStream_t st) {
    if (p.D <= 32) return launch_plain_bwd<T, 64, 2>(p, w, st);
    if (p.D <= 64) return launch_plain_bwd<T, 64, 4>(p, w, st);
    if (p.D <= 128) return launch_plain_bwd<T, 32, 8>(p, w, st);
    return launch_plain_bwd<T, 32, 16>(p, w, st);
}
// The split loops' parts to their results
template <typename T> int run_join(const AttnParams& p, const AttnBwdSplit& w, cudaStream_t st) {
    auto join = [&](const float* a, const float* b, const AttnTensor& ta, const AttnTensor& tb, int splits, int L, int heads) {
        const int64_t n = (int64_t)p.B * heads * L * p.D;
        const dim3 grid((unsigned)std::min<int64_t>(ceil_div(n, kApThreads), 16 * (int64_t)sm_count()), b != nullptr ? 2 : 1);
        return launch_stage(attn_join_kernel<T>, grid, kApThreads, 0, st, true, a, b, ta, tb, splits, L, heads, p.D, (long long)n);
    };
    int rc = TRIMUL_OK;
    if (w.dq != nullptr) rc = join(w.dq, nullptr, p.dq, p.dq, w.q_splits, p.Lq, p.H);
    if (rc == TRIMUL_OK && w.dk != nullptr) rc = join(w.dk, w.dv, p.dk, p.dv, w.kv_splits, p.Lk, p.Hk);
    return rc;
}

// What the main kernel needs prepared; `d` gets the bias where the tensor-core kernels can fetch it
AttnPrep prepare(trimul_attn_desc* d, const AttnWorkspace& w, uint8_t* ws) {
    AttnPrep r = {};
    if (copies_bias(d)) {
        r.bias = reinterpret_cast<uint32_t*>(ws + w.bias);
        r.bias_heads = d->bias_heads;
        r.bias_pitch = (int)align_up(d->Lk, 8);
        r.bias_rows = (int64_t)d->bias_batch * d->bias_heads * d->Lq;
        r.bias_blocks = (int)std::min<int64_t>(ceil_div(r.bias_rows, kPrepWarps), 4 * (int64_t)sm_count());
        d->bias = r.bias;
        d->bias_i = r.bias_pitch;
        d->bias_h = d->bias_i * d->Lq;
        d->bias_b = d->bias_h * d->bias_heads;
    }
    if (d->mask != nullptr) {
        r.mask_blocks = d->B;
        r.n_tiles = (int)ceil_div(d->Lk, kAfRows);
        r.words = reinterpret_cast<uint32_t*>(ws + w.words);
        r.list = reinterpret_cast<int*>(ws + w.list);
    }
    return r;
}
int run_prep(const AttnParams& p, const AttnPrep& w, bool bf16, bool backward, cudaStream_t st) {
    const int lanes = p.D <= 64 ? 16 : 32;
    const int64_t delta = backward ? ceil_div((int64_t)p.B * p.Lq * p.H, kPrepThreads / lanes) : 0, blocks = w.mask_blocks + w.bias_blocks + delta;
    if (blocks == 0) return TRIMUL_OK;
    if (blocks > INT32_MAX) return TRIMUL_E_UNSUPPORTED;
    auto kernel = bf16 ? (lanes == 16 ? attn_prep_kernel<__nv_bfloat16, 16> : attn_prep_kernel<__nv_bfloat16, 32>)
                       : (lanes == 16 ? attn_prep_kernel<float, 16> : attn_prep_kernel<float, 32>);
    return launch_stage(kernel, dim3((unsigned)blocks), kPrepThreads, 0, st, true, p, w);
}

template <typename T, int kLanes>
int launch_short(const AttnShortParams& sp, int rows, cudaStream_t st) {
    auto kernel = rows <= 1 ? attn_short_kernel<T, kLanes, 1> : rows <= 2 ? attn_short_kernel<T, kLanes, 2>
                : rows <= 4 ? attn_short_kernel<T, kLanes, 4> : attn_short_kernel<T, kLanes, 8>;
    return launch_stage(kernel, dim3((unsigned)sp.splits, (unsigned)sp.a.Hk, (unsigned)sp.a.B), kAsThreads, 0, st,
                        true, sp);
}
template <typename T>
int run_short(const trimul_attn_desc* d, const AttnParams& p, const AttnWorkspace& w, uint8_t* ws, cudaStream_t st) {
    AttnShortParams sp = {};
    sp.a = p;
    sp.splits = short_splits(d);
    sp.keys_per_split = (int)ceil_div(d->Lk, sp.splits);
    if (sp.splits > 1) {
        sp.part_o = reinterpret_cast<float*>(ws + w.part_o);
        sp.part_ml = reinterpret_cast<float2*>(ws + w.part_ml);
    }
    const int rows = d->Lq * (d->H / d->Hk), pieces = d->D / (16 / (int)sizeof(T));
    int rc;
    if (pieces <= 4) rc = launch_short<T, 4>(sp, rows, st);
    else if (pieces <= 8) rc = launch_short<T, 8>(sp, rows, st);
    else if (pieces <= 16) rc = launch_short<T, 16>(sp, rows, st);
    else rc = launch_short<T, 32>(sp, rows, st);
    if (rc != TRIMUL_OK || sp.splits == 1) return rc;
    return run_combine<T>(p, sp.part_o, sp.part_ml, sp.splits, st);
}

template <bool kBias>
int launch_fwd(const AttnFwdParams& fp, const CUtensorMap (&m)[4], cudaStream_t st) {
    using L = AfLayout<kBias>;
    auto kernel = attn_fwd_sm100_kernel<kBias>;
    if (!ensure_smem(kernel, L::kSmem)) return TRIMUL_E_CUDA;
    const dim3 grid((unsigned)ceil_div(fp.a.Lq, 2 * kAfRows), (unsigned)fp.a.H, (unsigned)(fp.a.B * fp.splits));
    return launch_stage(kernel, grid, kAfThreads, L::kSmem, st, true, m[0], m[1], m[2], m[3], fp);
}
template <bool kBias>
int launch_fwd64(const AttnFwdParams& fp, const CUtensorMap (&m)[4], cudaStream_t st) {
    auto kernel = attn_fwd64_sm100_kernel<kBias>;
    if (!ensure_smem(kernel, A6Layout<kBias>::kSmem)) return TRIMUL_E_CUDA;
    const dim3 grid((unsigned)ceil_div(fp.a.Lq, 2 * kAfRows), (unsigned)fp.a.H, (unsigned)(fp.a.B * fp.splits));
    return launch_stage(kernel, grid, kA6Threads, A6Layout<kBias>::kSmem, st, true, m[0], m[1], m[2], m[3], fp);
}
int run_fwd(const trimul_attn_desc* given, const AttnParams& p, const AttnWorkspace& w, uint8_t* ws, cudaStream_t st) {
    trimul_attn_desc copy = *given;
    const trimul_attn_desc* d = &copy;
    const AttnPrep prep = prepare(&copy, w, ws);
    int rc = run_prep(p, prep, true, false, st);
    if (rc != TRIMUL_OK) return rc;
    AttnFwdParams fp = {};
    fp.a = p;
    fp.n_tiles = (int)ceil_div(d->Lk, kAfRows);
    fp.splits = forward_splits(d);
    fp.tiles_per_split = (int)ceil_div(fp.n_tiles, fp.splits);
    fp.words = prep.words;
    fp.list = prep.list;
    fp.bias_b1 = d->bias_batch == 1;
    fp.bias_h1 = d->bias_heads == 1;
    if (fp.splits > 1) {
        fp.part_o = reinterpret_cast<float*>(ws + w.part_o);
        fp.part_ml = reinterpret_cast<float2*>(ws + w.part_ml);
    }
    CUtensorMap m[4];
    if (!encode_rows(&m[0], p.q, d->D, d->Lq, d->H, d->B) || !encode_rows(&m[1], p.k, d->D, d->Lk, d->Hk, d->B) ||
        !encode_rows(&m[2], p.v, d->D, d->Lk, d->Hk, d->B))
        return TRIMUL_E_CUDA;
    m[3] = m[0];
    if (d->bias != nullptr && !encode_bias(&m[3], d)) return TRIMUL_E_CUDA;
    if (d->D <= 64) rc = d->bias != nullptr ? launch_fwd64<true>(fp, m, st) : launch_fwd64<false>(fp, m, st);
    else rc = d->bias != nullptr ? launch_fwd<true>(fp, m, st) : launch_fwd<false>(fp, m, st);
    if (rc != TRIMUL_OK || fp.splits == 1) return rc;
    return run_combine<__nv_bfloat16>(p, fp.part_o, fp.part_ml, fp.splits, st);
}

template <int kD, bool kBias, typename Ds = __nv_bfloat16>
int launch_bwd(const AttnBwdParams& bp, const CUtensorMap (&m)[5], cudaStream_t st) {
    constexpr int kSmem = std::max(AbKvLayout<kD, kBias>::kSmem, AbQLayout<kD, kBias>::kSmem);
    auto kernel = attn_bwd_sm100_kernel<kD, kBias, Ds>;
    if (!ensure_smem(kernel, kSmem)) return TRIMUL_E_CUDA;
    const dim3 grid((unsigned)(bp.w.kv_blocks + bp.w.q_blocks));
    return launch_stage(kernel, grid, kAbThreads, kSmem, st, true, m[0], m[1], m[2], m[3], m[4], bp);
}
int run_bwd(const trimul_attn_desc* given, const AttnParams& p, const AttnWorkspace& w, const AttnBwdSplit& split, uint8_t* ws,
            cudaStream_t st) {
    trimul_attn_desc copy = *given;
    const trimul_attn_desc* d = &copy;
    const AttnPrep prep = prepare(&copy, w, ws);
    const int rc = run_prep(p, prep, true, true, st);
    if (rc != TRIMUL_OK) return rc;
    AttnBwdParams bp = {};
    bp.a = p;
    bp.w = split;
    bp.n_tiles = (int)ceil_div(d->Lk, kAfRows);
    bp.words = prep.words;
    bp.list = prep.list;
    bp.bias_b1 = d->bias_batch == 1;
    bp.bias_h1 = d->bias_heads == 1;
    CUtensorMap m[5];
    if (!encode_rows(&m[0], p.q, d->D, d->Lq, d->H, d->B) || !encode_rows(&m[1], p.k, d->D, d->Lk, d->Hk, d->B) ||
        !encode_rows(&m[2], p.v, d->D, d->Lk, d->Hk, d->B) || !encode_rows(&m[3], p.dout, d->D, d->Lq, d->H, d->B))
        return TRIMUL_E_CUDA;
    m[4] = m[0];
    if (d->bias != nullptr && !encode_bias(&m[4], d)) return TRIMUL_E_CUDA;
    if (p.ds_parts) return d->D <= 64 ? launch_bwd<64, true, float>(bp, m, st) : launch_bwd<128, true, float>(bp, m, st);
    if (d->D <= 64) return d->bias != nullptr ? launch_bwd<64, true>(bp, m, st) : launch_bwd<64, false>(bp, m, st);
    return d->bias != nullptr ? launch_bwd<128, true>(bp, m, st) : launch_bwd<128, false>(bp, m, st);
}

}  // namespace

extern "C" {

int trimul_b200_relpos_bias(const trimul_relpos_desc* d, const trimul_buckets* b, const void* table, const void* q_pos,
                            const void* k_pos, const void* q_seg, const void* k_seg, const void* add, void* out,
                            void* stream) {
    const int rc = check_relpos(d, b);
    if (rc != TRIMUL_OK) return rc;
    if (table == nullptr || q_pos == nullptr || k_pos == nullptr || out == nullptr) return TRIMUL_E_INVALID;
    if (b->segments != 0 && (q_seg == nullptr || k_seg == nullptr)) return TRIMUL_E_INVALID;
    if (d->layout == TRIMUL_RELPOS_HEADS) {
        const int n = 16 / elem_size(d->dtype);
        if (add != nullptr || !aligned(out, 16)) return TRIMUL_E_INVALID;
        if ((d->stride_b % n) || (d->stride_h % n) || (d->stride_i % n) || d->stride_i < align_up(d->Lk, n))
            return TRIMUL_E_INVALID;
    }
    const RelposParams p = relpos_params(d, b, table, q_pos, k_pos, q_seg, k_seg);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return d->dtype == TRIMUL_DTYPE_BF16 ? run_relpos_forward<__nv_bfloat16>(d, b, p, add, out, st)
                                         : run_relpos_forward<float>(d, b, p, add, out, st);
}

int trimul_b200_relpos_bias_grad_workspace_bytes(const trimul_relpos_desc* d, const trimul_buckets* b, size_t* bytes) {
    const int rc = check_relpos(d, b);
    if (rc != TRIMUL_OK) return rc;
    if (bytes == nullptr) return TRIMUL_E_INVALID;
    int64_t parts = 0;
    for (bool wide : {false, true}) parts = std::max<int64_t>(parts, plan_relpos_grad(d, b, wide).parts);
    *bytes = (size_t)(parts * (b->count + (b->segments != 0)) * d->channels * 4);
    return TRIMUL_OK;
}

int trimul_b200_relpos_bias_grad(const trimul_relpos_desc* d, const trimul_buckets* b, const void* q_pos, const void* k_pos,
                                 const void* q_seg, const void* k_seg, const void* grad, void* dtable, void* workspace,
                                 size_t workspace_bytes, void* stream) {
    size_t need = 0;
    const int rc = trimul_b200_relpos_bias_grad_workspace_bytes(d, b, &need);
    if (rc != TRIMUL_OK) return rc;
    if (q_pos == nullptr || k_pos == nullptr || grad == nullptr || dtable == nullptr || workspace == nullptr)
        return TRIMUL_E_INVALID;
    if (b->segments != 0 && (q_seg == nullptr || k_seg == nullptr)) return TRIMUL_E_INVALID;
    if (workspace_bytes < need) return TRIMUL_E_WORKSPACE;
    if (!aligned(workspace, 16)) return TRIMUL_E_INVALID;
    const RelposParams p = relpos_params(d, b, nullptr, q_pos, k_pos, q_seg, k_seg);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // a single part is the result
    const int parts = plan_relpos_grad(d, b, wide_lanes(d, grad)).parts;
    float* partial = static_cast<float*>(parts == 1 && !p.table_bf16 ? dtable : workspace);
    return d->dtype == TRIMUL_DTYPE_BF16 ? run_relpos_grad<__nv_bfloat16>(d, b, p, grad, dtable, partial, st)
                                         : run_relpos_grad<float>(d, b, p, grad, dtable, partial, st);
}

int trimul_b200_attn_workspace_bytes(const trimul_attn_desc* d, int32_t backward, size_t* bytes) {
    const int rc = check_attn(d);
    if (rc != TRIMUL_OK) return rc;
    if (bytes == nullptr) return TRIMUL_E_INVALID;
    *bytes = (size_t)attn_workspace(d, backward != 0).total;
    return TRIMUL_OK;
}

int trimul_b200_attn_forward(const trimul_attn_desc* d, void* workspace, size_t workspace_bytes, void* stream,
                             int32_t* status) {
    const int rc = check_attn(d);
    if (rc != TRIMUL_OK) return rc;
    if (!d->q.p || !d->k.p || !d->v.p || !d->o.p) return TRIMUL_E_INVALID;
    const AttnWorkspace w = attn_workspace(d, false);
    if (w.total > 0 && (workspace == nullptr || !aligned(workspace, 256))) return TRIMUL_E_INVALID;
    if (workspace_bytes < (size_t)w.total) return TRIMUL_E_WORKSPACE;
    const AttnParams p = attn_params(d, status);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (short_rows(d))
        return d->dtype == TRIMUL_DTYPE_BF16 ? run_short<__nv_bfloat16>(d, p, w, static_cast<uint8_t*>(workspace), st)
                                             : run_short<float>(d, p, w, static_cast<uint8_t*>(workspace), st);
    if (tensor_core_forward(d)) return run_fwd(d, p, w, static_cast<uint8_t*>(workspace), st);
    return d->dtype == TRIMUL_DTYPE_BF16 ? run_plain_fwd<__nv_bfloat16>(d, p, w, static_cast<uint8_t*>(workspace), st)
                                         : run_plain_fwd<float>(d, p, w, static_cast<uint8_t*>(workspace), st);
}

int trimul_b200_attn_backward(const trimul_attn_desc* d, void* workspace, size_t workspace_bytes, void* stream,
                              int32_t* status) {
    int rc = check_attn(d);
    if (rc != TRIMUL_OK) return rc;
    if (!d->q.p || !d->k.p || !d->v.p || !d->o.p || !d->dout.p || !d->dq.p || !d->dk.p || !d->dv.p || !d->stats)
        return TRIMUL_E_INVALID;
    const AttnWorkspace w = attn_workspace(d, true);
    if (workspace == nullptr || !aligned(workspace, 256)) return TRIMUL_E_INVALID;
    if (workspace_bytes < (size_t)w.total) return TRIMUL_E_WORKSPACE;
    AttnParams p = attn_params(d, status);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    p.delta = reinterpret_cast<float*>(ws + w.delta);
    if (d->dbias != nullptr) {
        if (sums_bias(d)) {
            p.ds = ws + w.ds;
            p.ds_parts = 1;
            p.ds_h = w.ds_pitch * d->Lq; p.ds_b = p.ds_h * d->H;
        } else {
            p.ds = d->dbias;
            p.ds_i = d->dbias_i; p.ds_h = d->bias_heads == 1 ? 0 : d->dbias_h; p.ds_b = d->bias_batch == 1 ? 0 : d->dbias_b;
        }
    }
    const bool bf16 = d->dtype == TRIMUL_DTYPE_BF16;
    const bool tensor = tensor_core_backward(d);
    AttnBwdSplit split = backward_split(d, tensor);
    if (split.q_blocks == 0) return TRIMUL_E_UNSUPPORTED;
    if (split.q_splits > 1) split.dq = reinterpret_cast<float*>(ws + w.dq);
    if (split.kv_splits > 1) {
        split.dk = reinterpret_cast<float*>(ws + w.dk);
        split.dv = reinterpret_cast<float*>(ws + w.dv);
    }
    if (!tensor) rc = run_prep(p, AttnPrep{}, bf16, true, st);
    if (rc != TRIMUL_OK) return rc;
    if (tensor) rc = run_bwd(d, p, w, split, ws, st);
    else rc = bf16 ? run_plain_bwd<__nv_bfloat16>(p, split, st) : run_plain_bwd<float>(p, split, st);
    if (rc == TRIMUL_OK) rc = bf16 ? run_join<__nv_bfloat16>(p, split, st) : run_join<float>(p, split, st);
    if (rc != TRIMUL_OK || !sums_bias(d)) return rc;
    const int n = 16 / elem_size(d->dtype);
    const int64_t tiles = (int64_t)d->bias_batch * d->bias_heads * ceil_div(d->Lq, kApSumRows) * ceil_div(d->Lk, kApSumChunks * n);
    const dim3 sgrid((unsigned)std::min<int64_t>(tiles, 16 * (int64_t)sm_count()));
    const int sum_b = d->bias_batch == 1, sum_h = d->bias_heads == 1;
    auto sum = [&](auto kernel, auto* out) {
        return launch_stage(kernel, sgrid, kApThreads, 0, st, true, static_cast<const float*>(p.ds), p.ds_b, p.ds_h, out, (long long)d->dbias_b,
                            (long long)d->dbias_h, (long long)d->dbias_i, d->B, d->H, d->Lq, d->Lk, sum_b, sum_h);
    };
    return bf16 ? sum(attn_bias_sum_kernel<__nv_bfloat16>, static_cast<__nv_bfloat16*>(d->dbias))
                : sum(attn_bias_sum_kernel<float>, static_cast<float*>(d->dbias));
}

}  // extern "C"

// Cross attention: what its kernels share.
//
//   x_ij = scale q_i . k_j + bias_ij   over the kept keys j,   p_ij = exp(x_ij - m_i) / l_i,   o_i = sum_j p_ij v_j
//
// with m_i the row's maximum and l_i the sum of exp(x_ij - m_i).  A row without a kept key gives o_i = 0 and zero
// gradients; it is known by l_i = 0.  The maximum does not tell: it passes over NaN, so a row of nothing but NaN also leaves
// it at -inf, and that row's sum and result are NaN.  Statistics of a row are kept as the pair (m_i, log2 l_i) rather than their sum: a mask of the type's lowest
// value (-3.4e38) on a whole row would swallow log l_i, and every probability would come back as 1.  For the same reason
// x - m is formed before it is scaled to base 2 wherever a bias takes part.
#pragma once

#include "../../include/trimul_b200.h"
#include "ptx_sm100.cuh"

namespace trimul {

constexpr float kLog2e = 1.4426950408889634f;

// Strides in elements; the head dimension is contiguous.
struct AttnTensor {
    void* p;
    long long b, l, h;
};
struct AttnParams {
    int B, Lq, Lk, H, Hk, D;
    float scale;
    AttnTensor q, k, v, o, dout, dq, dk, dv;
    const void* bias;                      // null, or strides below (0 where one bias serves several)
    long long bias_b, bias_h, bias_i;
    const uint8_t* mask;                   // null, or [B] rows of Lk bytes, mask_b apart; 0 = masked key
    long long mask_b;
    float2* stats;                         // [B][H][Lq]: (m, log2 l); (0, +inf) for a row without keys
    void* o_lo;                            // [B][Lq][H][D]: what rounding o to 16 bits left over, or null
    float* delta;                          // [B][H][Lq]: sum_d dout o
    void* ds;                              // gradient of x, or null: written with the strides below
    long long ds_b, ds_h, ds_i;
    int ds_parts;                          // it is going to be summed: fp32 whatever the inputs are, for each head in groups of
                                           // four columns, [column / 4][Lq][4], so that a warp's rows lie side by side
    int32_t* status;
};

// Backward pass: how many blocks share the loop of a tile, and where their parts go ([split][row][D] in fp32, rows as
// [B][heads][length]; null: the loop is whole and the block writes the result)
struct AttnBwdSplit {
    int q_splits, kv_splits;
    int q_share, kv_share;                 // steps of a block, without masks
    int q_blocks, kv_blocks;               // with the splits
    int q_first;                           // the blocks over the keys come first
    float *dq, *dk, *dv;
};

// Loads of what an earlier kernel may have written (the key mask's bits and list, delta, parts of split rows and of a bias's
// gradient, inputs that a call before returned): plain ones.  A kernel of these calls is launched while the one before it still
// runs, and the non-coherent path (__ldg) is only defined for memory that nobody writes in a kernel's whole life, the time before
// griddep_wait() included.  No stale value was ever measured, and no difference in time.
template <typename V> __device__ __forceinline__ V at_load(const V* p) { return *p; }
__device__ __forceinline__ float at_float(float v) { return v; }
__device__ __forceinline__ float at_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void at_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void at_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ float ex2f(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// ---------------------------------------------------------------------------------------
// UMMAs issued by a whole warp.  Every lane runs the same code and one elected lane (the same each time) issues: descriptors
// and addresses are then warp-uniform values, which the instruction takes from uniform registers as it wants them.  Under an
// `if (lane == 0)` each operand is moved there first: 75 to 90 cycles per UMMA were measured in the attention kernels, whose
// tensor cores then waited for the issuing thread.
// ---------------------------------------------------------------------------------------
__device__ __forceinline__ int warp_uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }      // known to be, from here on
__device__ __forceinline__ uint32_t warp_uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ void umma_ss_warp(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add)
        : "memory");
}
__device__ __forceinline__ void umma_ts_warp(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "}\n"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add)
        : "memory");
}
__device__ __forceinline__ void umma_commit_warp(uint64_t* bar) {
    asm volatile(
        "{\n\t"
        ".reg .pred q;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t"
        "}\n"
        ::"r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "}\n"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return done != 0;
}
// Wait of a whole warp.  All lanes look once (where the phase is complete that is all there is to it), then wait suspended for
// up to the hint's 20 us, from which the warp wakes at once (with a sleeping poller instead, a wait took up to 3000 cycles
// longer); after that one lane polls, with the limit of every wait.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int lane, volatile int* abort_flag, int32_t* status,
                                          int stage, int detail) {
    if (__all_sync(0xffffffffu, mbar_test(bar, parity))) return true;
#pragma unroll 1
    for (int t = 0; t < 256; ++t)
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity) != 0)) return true;
    uint32_t ok = 1;
    if (lane == 0) ok = mbar_wait<true>(bar, parity, abort_flag, status, stage, detail);
    return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

}  // namespace trimul

// Host-side helpers shared by the library's translation units: tensor-map encoding, device properties,
// shared-memory opt-in and launches.
#pragma once

#include "../../include/trimul_b200.h"

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <mutex>
#include <utility>

namespace trimul {

// ---------------------------------------------------------------------------------------
// driver entry point for tensor-map encoding (resolved at run time: no link against libcuda)
// ---------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn get_encode_fn() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult qres;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qres) == cudaSuccess &&
            qres == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    });
    return fn;
}

// bf16 tensor of up to 4 dimensions, innermost first; strides in ELEMENTS for dims 1..3.
inline bool encode_bf16(CUtensorMap* map, const void* base, int rank, const uint64_t* dims, const uint64_t* strides_elems,
                 const uint32_t* box, int swizzle_bytes) {
    EncodeTiledFn fn = get_encode_fn();
    if (fn == nullptr) return false;
    cuuint64_t gdim[4];
    cuuint64_t gstride[3];
    cuuint32_t bdim[4];
    cuuint32_t estr[4];
    for (int i = 0; i < rank; ++i) {
        gdim[i] = dims[i];
        bdim[i] = box[i];
        estr[i] = 1;
    }
    for (int i = 0; i + 1 < rank; ++i) gstride[i] = strides_elems[i] * 2;
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<void*>(base), gdim, gstride,
                    bdim, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    swizzle_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B
                    : swizzle_bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                          : CU_TENSOR_MAP_SWIZZLE_NONE,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS;
}

inline int sm_count() {
    static int n = 0;
    if (n == 0) {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess) return 148;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    }
    return n;
}

// Opt the kernel in to `bytes` of dynamic shared memory — once per kernel and device: the
// attribute call is not free and these entry points sit on latency-sensitive host paths.
inline bool ensure_smem_once(const void* fn, int bytes) {
    struct Entry { const void* fn; uint64_t devices; };
    static Entry table[256];
    static int used = 0;
    static std::mutex mu;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    std::lock_guard<std::mutex> lock(mu);
    Entry* e = nullptr;
    for (int i = 0; i < used; ++i)
        if (table[i].fn == fn) e = &table[i];
    if (e != nullptr && dev < 64 && ((e->devices >> dev) & 1u)) return true;
    if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
    if (e == nullptr && used < 256) { e = &table[used++]; e->fn = fn; e->devices = 0; }
    if (e != nullptr && dev < 64) e->devices |= 1ull << dev;
    return true;
}
template <typename K>
bool ensure_smem(K kernel, int bytes) {
    return ensure_smem_once(reinterpret_cast<const void*>(kernel), bytes);
}

inline int launch_status() { return cudaGetLastError() == cudaSuccess ? TRIMUL_OK : TRIMUL_E_CUDA; }

// Launch of a kernel.  `overlap` asks for programmatic dependent launch: the
// kernel may be scheduled while its predecessor in the stream is still draining, runs its set-up
// (barriers, tensor memory, descriptor prefetch) and then blocks in griddepcontrol.wait until the
// predecessor has completed, so launch latency and set-up disappear from the critical path.  Every
// kernel launched this way executes that wait before it touches global memory.
template <typename... KArgs, typename... Args>
int launch_stage(void (*kernel)(KArgs...), dim3 grid, int block, int smem, cudaStream_t st, bool overlap,
                 Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)block, 1, 1);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap ? 1u : 0u;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...) == cudaSuccess ? TRIMUL_OK : TRIMUL_E_CUDA;
}

}  // namespace trimul

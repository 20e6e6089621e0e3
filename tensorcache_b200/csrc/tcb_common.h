// Shared host-side helpers of the tcb200 library: status codes, the per-thread
// error message, and CUDA error mapping.
#pragma once
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cuda_runtime.h>

#include "../../include/tcb200.h"

namespace tcb {

// Stores a printf-style message for tcb_last_error() and returns `code`.
int fail(int code, const char* fmt, ...);
void clear_error();

inline int cuda_fail(cudaError_t e, const char* what) {
    return fail(TCB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

#define TCB_CUDA_TRY(expr)                                       \
    do {                                                         \
        cudaError_t _e = (expr);                                 \
        if (_e != cudaSuccess) return ::tcb::cuda_fail(_e, #expr); \
    } while (0)

// Group sizes of the codec kernels (encode and decode); the fused GEMM and the no-allocation decode accept 16 / 32 / 64 only.
inline bool group_size_ok(int g) { return g == 8 || g == 16 || g == 24 || g == 32 || g == 48 || g == 64 || g == 128; }
inline bool core_group_size_ok(int g) { return g == 16 || g == 32 || g == 64; }

// Number of SMs of the current device (cached per device).
int sm_count();

#ifdef __CUDACC__
// Programmatic dependent launch: the kernel may start while its predecessor on the stream is finishing.  It calls
// await_predecessor() before it touches global memory, and afterwards lets its own successor start.  (In that order: a
// successor's L1 is then empty of anything that was read before this kernel's predecessor had finished.  What a predecessor
// both reads and changes must be read past L1.)
template <typename... Args>
cudaError_t launch_overlapped(void (*kernel)(Args...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}
// Streamed once: 32-byte accesses that leave L2 first.
__device__ __forceinline__ void ldg_stream_v8(const void* p, uint32_t* w) {
    asm volatile("ld.global.nc.L1::no_allocate.L2::evict_first.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
}
__device__ __forceinline__ void stg_stream_v8(void* p, const uint32_t* w) {
    asm volatile("st.global.L2::evict_first.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                 "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

__device__ __forceinline__ void await_predecessor() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
#endif

}  // namespace tcb

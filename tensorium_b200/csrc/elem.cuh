// elem.cuh -- the element types of the token operators (TB_F32, TB_BF16, TB_F16): conversions, dispatch on them, and the
// operators' launches.
#pragma once
#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <initializer_list>

namespace tbi {

template <typename T> struct Elem;
template <> struct Elem<float> {
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Elem<__half> {
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};

// elements in 16 bytes
template <typename T> struct Vec {
    static constexpr int N = 16 / sizeof(T);
};

inline bool elem_type_ok(int64_t t) { return t == TB_F32 || t == TB_BF16 || t == TB_F16; }
inline size_t elem_size(int64_t t) { return t == TB_F32 ? 4 : 2; }
// whether each address (null too) is a multiple of n bytes
inline bool aligned_to(size_t n, std::initializer_list<const void*> addresses) {
    for (const void* p : addresses)
        if ((uintptr_t)p % n) return false;
    return true;
}

// launch() that lets the kernel be scheduled while the one before it on the stream still runs: its set-up hides the
// launch's latency, and it waits for that kernel's end itself (TB_GRID_DEP_ENTRY) before it reads or writes
// global memory.
template <typename... KArgs, typename... Args>
int launch_early(tb_ctx* ctx, const char* what, void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, Args&&... args) {
    const int pdl = ctx->pdl;
    ctx->pdl = 1;
    const int r = launch(ctx, what, kernel, grid, block, smem, std::forward<Args>(args)...);
    ctx->pdl = pdl;
    return r;
}

// f(T()) for the element type t
template <typename F> int elem_dispatch(int64_t t, F&& f) {
    if (t == TB_F32) return f(float());
    if (t == TB_BF16) return f(__nv_bfloat16());
    return f(__half());
}

}  // namespace tbi

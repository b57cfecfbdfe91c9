// elem.cuh -- the element types of the token operators (TB_F32, TB_BF16, TB_F16): conversions and
// 16-byte accesses that never touch memory outside a row.
#pragma once
#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

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

// 16 bytes of elements
template <typename T> struct __align__(16) Vec {
    static constexpr int N = 16 / sizeof(T);
    T e[N];
};

inline bool elem_type_ok(int64_t t) { return t == TB_F32 || t == TB_BF16 || t == TB_F16; }
inline size_t elem_size(int64_t t) { return t == TB_F32 ? 4 : 2; }

// f(T()) for the element type t
template <typename F> int elem_dispatch(int64_t t, F&& f) {
    if (t == TB_F32) return f(float());
    if (t == TB_BF16) return f(__nv_bfloat16());
    return f(__half());
}

}  // namespace tbi

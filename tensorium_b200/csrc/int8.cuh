// int8.cuh -- what the int8 product's kernels share.
#pragma once
#include "elem.cuh"

namespace tbi {

// y[i][j] = act((a . w^T)[i][j] * (a_scales[i] * w_scales[j]) + bias[j]), i < m tokens, j < n channels
struct Int8Args {
    int64_t m, n, k;
    const int8_t* a;
    int64_t a_stride;
    const float* a_scales;
    const int8_t* w;
    int64_t w_stride;
    const float* w_scales;
    const float* bias;
    int act;
    void* y;
    int64_t y_stride;
};

__device__ __forceinline__ float int8_epilogue(int acc, float scale, float bias, bool has_bias, int act) {
    float v = __fmul_rn(__int2float_rn(acc), scale);
    if (has_bias) v = __fadd_rn(v, bias);
    return tb_activate_dev(v, act);
}

// tensor-core product (int8_tc.cu); after_quantize: the kernel before it on the stream is the one
// that writes a and a_scales, and lets this one start early
int int8_gemm_tc(tb_ctx* ctx, const Int8Args& p, int64_t y_type, bool after_quantize);

}  // namespace tbi

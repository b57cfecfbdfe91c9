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

// Tensor-core product (int8_tc.cu). after_quantize: the kernel before it on the stream is the one that
// writes a and a_scales, and lets this one start early. scratch: the workspace is free from there on; where that is not its
// start, int8_gemm_scratch more bytes have to be reserved.
int int8_gemm_tc(tb_ctx* ctx, const Int8Args& p, int64_t y_type, bool after_quantize, size_t scratch);
size_t int8_gemm_scratch(const tb_ctx* ctx, int64_t m);

}  // namespace tbi

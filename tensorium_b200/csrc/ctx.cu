// ctx.cu -- host code of the context (no kernels, no device code).
#include "ctx.cuh"

namespace tbi {

int take_status(tb_ctx* ctx, int* status) {
    *status = 0;
    TB_CHECK_CUDA(cudaStreamSynchronize(ctx->stream));
    TB_CHECK_CUDA(cudaMemcpy(status, ctx->d_status, sizeof(int), cudaMemcpyDeviceToHost));
    if (*status == 0) return TB_OK;
    // on the stream that the next launch is ordered behind (the legacy stream orders nothing before a non-blocking
    // one); the status word last, so that it stays where a counter could not be cleared
    TB_CHECK_CUDA(cudaMemsetAsync(ctx->tile_cnt, 0, sizeof(int) * ctx->tile_cnt_len, ctx->stream));
    for (auto& c : ctx->side_cnts) TB_CHECK_CUDA(cudaMemsetAsync(c.first, 0, sizeof(int) * c.second, ctx->stream));
    TB_CHECK_CUDA(cudaMemsetAsync(ctx->d_status, 0, sizeof(int), ctx->stream));
    TB_CHECK_CUDA(cudaStreamSynchronize(ctx->stream));
    return TB_OK;
}

}  // namespace tbi

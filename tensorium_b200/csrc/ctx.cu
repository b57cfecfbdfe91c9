// ctx.cu -- host code of the context (no kernels, no device code).
#include "ctx.cuh"

namespace tbi {

static bool capturing(cudaStream_t s) {
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    if (!s) return false;  // the legacy stream cannot be captured
    if (cudaStreamIsCapturing(s, &cs) != cudaSuccess) cudaGetLastError();
    return cs != cudaStreamCaptureStatusNone;
}

int ensure_workspace(tb_ctx* ctx, size_t bytes) {
    if (bytes <= ctx->ws_bytes) {
        if (!ctx->ws_in_graph) ctx->ws_in_graph = capturing(ctx->stream);
        return TB_OK;
    }
    if (capturing(ctx->stream))
        return fail(TB_ERR_STATE, "workspace of %zu bytes needed during stream capture (have %zu); "
                    "call tb_workspace_reserve first", bytes, ctx->ws_bytes);
    const size_t want = (bytes + ((1 << 20) - 1)) >> 20 << 20;
    void* p = nullptr;
    cudaError_t e = cudaMalloc(&p, want);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return cuda_fail(e, "cudaMalloc(workspace)");
    }
    if (ctx->ws && ctx->ws_in_graph) {
        ctx->ws_kept.push_back(ctx->ws);
    } else if (ctx->ws) {
        // the old buffer may still be read by queued work on this stream
        e = cudaStreamSynchronize(ctx->stream);
        if (e != cudaSuccess) {
            cudaFree(p);
            return cuda_fail(e, "cudaStreamSynchronize");
        }
        cudaFree(ctx->ws);
    }
    ctx->ws = p;
    ctx->ws_bytes = want;
    ctx->ws_in_graph = false;
    return TB_OK;
}

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

// ctx.cuh -- the context: what a tb_ctx holds and the host code that keeps it in order (ctx.cu). No device code.
#pragma once

#include <cuda_runtime_api.h>
#include <stddef.h>
#include <stdint.h>
#include <utility>
#include <vector>

#include "../../include/tensorium_b200.h"

struct tb_ctx {
    int device = 0;
    cudaStream_t stream = nullptr;      // current launch stream
    cudaStream_t own_stream = nullptr;  // stream created by tb_init
    void* ws = nullptr;                 // split-K / scratch workspace
    size_t ws_bytes = 0;
    bool ws_in_graph = false;           // a captured graph may hold ws's address
    std::vector<void*> ws_kept;         // outgrown workspaces that graphs may hold
    int* d_status = nullptr;            // device status word (kernels report errors here)
    int64_t math_mode = TB_MATH_FP32;
    int sm_count = 148;
    int max_smem_optin = 0;
    cudaEvent_t fork = nullptr, join = nullptr;  // order own_stream work with `stream`
    int* tile_cnt = nullptr;                      // split-K arrival counters (zeroed, self-resetting)
    int64_t tile_cnt_len = 0;
    std::vector<std::pair<int*, int64_t>> side_cnts;  // the same of its networks' branch streams
    int pdl = 0;  // launches through tbi::launch may overlap the previous kernel's tail (set while
                  // a network forward is captured)
};

namespace tbi {

int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t e, const char* what);
// The workspace holds at least `bytes` from here on (may allocate, except during capture). A workspace that a captured graph
// may use is kept until the context ends, so that the graph can be replayed after a growth.
int ensure_workspace(tb_ctx* ctx, size_t bytes);
// The device status word, once the work on ctx's stream has ended. A kernel that gave up leaves its arrival counters as they
// were: where there is a status, it and every counter are 0 again before this returns.
int take_status(tb_ctx* ctx, int* status);

}  // namespace tbi

#define TB_CHECK_CUDA(call)                                              \
    do {                                                                  \
        cudaError_t _e = (call);                                          \
        if (_e != cudaSuccess) return tbi::cuda_fail(_e, #call);          \
    } while (0)

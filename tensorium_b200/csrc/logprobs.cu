// logprobs.cu -- what a program reads off vocabulary-sized logits: the log probability of a given
// token, the entropy, the most probable tokens (tb_token_logprobs_fwd), and the gradient of the
// first two (tb_token_logprobs_bwd).
#include "elem.cuh"

namespace tbi {
namespace {

constexpr int TOP_MAX = 32;

struct LogprobArgs {
    int64_t rows, vocab;
    const void* logits;
    int64_t stride;
    const int64_t* tokens;
    float inv_t;
    int top;
    float* logprob;
    float* entropy;
    float* lse;
    float* row_max;
    float* log_sum;
    float* top_logprob;
    int64_t* top_token;
};

__device__ __forceinline__ float nan_f() { return __uint_as_float(0x7fffffffu); }

// Order of alternatives as one unsigned key: the value's order in the high half (-0 counts as 0), then
// the lower column first. 0 is below every key.
__device__ __forceinline__ unsigned long long top_key(float v, uint32_t col) {
    uint32_t u = __float_as_uint(v + 0.f);
    u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((unsigned long long)u << 32) | (uint32_t)~col;
}
__device__ __forceinline__ uint32_t key_col(unsigned long long k) { return ~(uint32_t)k; }
__device__ __forceinline__ float key_val(unsigned long long k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

template <typename V, typename F> __device__ V block_reduce(V v, V* part, F f) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[0];
    for (int i = 1; i < (int)blockDim.x / 32; ++i) v = f(v, part[i]);
    return v;
}

// One CTA per row, a pass for the maximum, one for the sums and one for each alternative.
template <typename T> __global__ void __launch_bounds__(256) k_token_logprobs(const LogprobArgs p) {
    TB_GRID_DEP_ENTRY();
    __shared__ float part[8];
    __shared__ unsigned long long kpart[8];
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.logits) + row * p.stride;
    float m = -INFINITY;
    bool bad = false;
    for (int64_t i = threadIdx.x; i < p.vocab; i += blockDim.x) {
        const float v = Elem<T>::get(x[i]);
        bad |= !(v < INFINITY);
        m = fmaxf(m, v);
    }
    m = block_reduce(m, part, [](float a, float b) { return fmaxf(a, b); });
    bad = __syncthreads_or(bad);
    const bool empty = m == -INFINITY;
    float z = 0.f, s = 0.f;
    if (!bad && !empty)
        for (int64_t i = threadIdx.x; i < p.vocab; i += blockDim.x) {
            const float t = fmaxf(__fmul_rn(__fsub_rn(Elem<T>::get(x[i]), m), p.inv_t), -200.f);
            const float e = expf(t);
            z += e;
            s = fmaf(e, t, s);
        }
    z = block_reduce(z, part, [](float a, float b) { return a + b; });
    s = block_reduce(s, part, [](float a, float b) { return a + b; });
    const float logz = logf(z);
    auto logprob = [&](float v) {
        return bad ? nan_f() : empty ? -INFINITY : __fsub_rn(__fmul_rn(__fsub_rn(v, m), p.inv_t), logz);
    };
    if (threadIdx.x == 0) {
        if (p.logprob) {
            const int64_t t = p.tokens[row];
            p.logprob[row] = t < 0 ? (bad ? nan_f() : 0.f) : t >= p.vocab ? nan_f() : logprob(Elem<T>::get(x[t]));
        }
        if (p.entropy) p.entropy[row] = bad ? nan_f() : empty ? 0.f : fmaxf(__fsub_rn(logz, __fdiv_rn(s, z)), 0.f);
        if (p.row_max) p.row_max[row] = bad ? nan_f() : m;
        if (p.log_sum) p.log_sum[row] = bad ? nan_f() : empty ? 0.f : logz;
        if (p.lse) p.lse[row] = bad ? nan_f() : empty ? -INFINITY : __fadd_rn(__fmul_rn(m, p.inv_t), logz);
    }
    unsigned long long last = ~0ull;
    for (int r = 0; r < p.top; ++r) {
        unsigned long long best = 0;
        for (int64_t i = threadIdx.x; i < p.vocab; i += blockDim.x) {
            const unsigned long long k = top_key(Elem<T>::get(x[i]), (uint32_t)i);
            if (k < last && k > best) best = k;
        }
        last = block_reduce(best, kpart, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; });
        if (threadIdx.x == 0) {
            p.top_token[row * p.top + r] = bad ? -1 : (int64_t)key_col(last);
            p.top_logprob[row * p.top + r] = logprob(key_val(last));
        }
    }
}

struct LogprobBwdArgs {
    int64_t rows, vocab;
    const void* logits;
    int64_t stride;
    const int64_t* tokens;
    float inv_t;
    const float* row_max;
    const float* log_sum;
    const float* entropy;
    const float* g_logprob;
    const float* g_entropy;
    void* dlogits;
    int64_t d_stride;
};

template <typename T> __global__ void __launch_bounds__(256) k_token_logprobs_bwd(const LogprobBwdArgs p) {
    TB_GRID_DEP_ENTRY();
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.logits) + row * p.stride;
    T* d = static_cast<T*>(p.dlogits) + row * p.d_stride;
    const float m = p.row_max[row], logz = p.log_sum[row];
    int64_t tok = p.g_logprob && p.tokens ? p.tokens[row] : -1;
    const float a = tok >= 0 ? p.g_logprob[row] : 0.f, b = p.g_entropy ? p.g_entropy[row] : 0.f;
    const float h = p.g_entropy ? p.entropy[row] : 0.f;
    const bool empty = m == -INFINITY, bad = logz != logz || tok >= p.vocab;
    for (int64_t i = threadIdx.x; i < p.vocab; i += blockDim.x) {
        float g = nan_f();
        if (empty) g = 0.f;
        else if (!bad) {
            const float lp = fmaxf(__fsub_rn(__fmul_rn(__fsub_rn(Elem<T>::get(x[i]), m), p.inv_t), logz), -200.f);
            const float q = expf(lp);
            g = __fmul_rn(__fsub_rn(i == tok ? a : 0.f, __fmul_rn(q, fmaf(b, __fadd_rn(lp, h), a))), p.inv_t);
        }
        d[i] = Elem<T>::put(g);
    }
}

int check_logits(int64_t rows, int64_t vocab, const void* logits, int64_t type, int64_t stride, float temperature) {
    if (rows < 0 || vocab <= 0 || rows > 2147483647 || vocab > 2147483647) return fail(TB_ERR_INVALID, "token logprobs: bad shape");
    if (!elem_type_ok(type)) return fail(TB_ERR_UNSUPPORTED, "token logprobs: element type %lld", (long long)type);
    if (!(temperature >= 0x1p-100f && temperature <= 0x1p100f)) return fail(TB_ERR_INVALID, "token logprobs: temperature has to be positive and finite");
    if (rows > 1 && stride < vocab) return fail(TB_ERR_INVALID, "token logprobs: row stride below the row's length");
    if (rows > 0 && !logits) return fail(TB_ERR_INVALID, "token logprobs: null pointer");
    if ((uintptr_t)logits % elem_size(type)) return fail(TB_ERR_INVALID, "token logprobs: misaligned pointer");
    return TB_OK;
}

}  // namespace
}  // namespace tbi

using namespace tbi;

extern "C" {

int tb_token_logprobs_fwd(tb_ctx* ctx, int64_t rows, int64_t vocab, const void* logits, int64_t type,
                          int64_t stride, const int64_t* tokens, float temperature, int64_t top,
                          float* logprob, float* entropy, float* lse, float* row_max, float* log_sum,
                          float* top_logprob, int64_t* top_token) {
    TB_ENTER(ctx);
    int r = check_logits(rows, vocab, logits, type, stride, temperature);
    if (r != TB_OK) return r;
    if (top < 0 || top > vocab) return fail(TB_ERR_INVALID, "token logprobs: top has to be between 0 and the vocabulary's size");
    if (top > TOP_MAX) return fail(TB_ERR_UNSUPPORTED, "token logprobs: top over %d", TOP_MAX);
    if (rows == 0) return TB_OK;
    if ((tokens && !logprob) || (top && (!top_logprob || !top_token))) return fail(TB_ERR_INVALID, "token logprobs: null pointer");
    const LogprobArgs p{rows, vocab, logits, stride, tokens, 1.f / temperature, (int)top, tokens ? logprob : nullptr, entropy, lse, row_max, log_sum, top_logprob, top_token};
    return elem_dispatch(type, [&](auto t) {
        return launch(ctx, "k_token_logprobs", k_token_logprobs<decltype(t)>, dim3((unsigned)rows), dim3(256), 0, p);
    });
}

int tb_token_logprobs_bwd(tb_ctx* ctx, int64_t rows, int64_t vocab, const void* logits, int64_t type,
                          int64_t stride, const int64_t* tokens, float temperature, const float* row_max,
                          const float* log_sum, const float* entropy, const float* g_logprob, const float* g_entropy,
                          void* dlogits, int64_t d_stride) {
    TB_ENTER(ctx);
    int r = check_logits(rows, vocab, logits, type, stride, temperature);
    if (r != TB_OK) return r;
    if (rows > 1 && d_stride < vocab) return fail(TB_ERR_INVALID, "token logprobs: row stride below the row's length");
    if (rows == 0) return TB_OK;
    if (!row_max || !log_sum || !dlogits || (g_logprob && !tokens) || (g_entropy && !entropy)) return fail(TB_ERR_INVALID, "token logprobs: null pointer");
    if ((uintptr_t)dlogits % elem_size(type)) return fail(TB_ERR_INVALID, "token logprobs: misaligned pointer");
    if (dlogits == logits && rows > 1 && d_stride != stride) return fail(TB_ERR_INVALID, "token logprobs: in place with another row stride");
    const LogprobBwdArgs p{rows, vocab, logits, stride, tokens, 1.f / temperature, row_max, log_sum, entropy, g_logprob, g_entropy, dlogits, d_stride};
    return elem_dispatch(type, [&](auto t) {
        return launch(ctx, "k_token_logprobs_bwd", k_token_logprobs_bwd<decltype(t)>, dim3((unsigned)rows), dim3(256), 0, p);
    });
}

}  // extern "C"

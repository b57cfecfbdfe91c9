// int8.cu -- the connected layer on int8 operands: rows quantized with a scale each
// (tb_quantize_rows), the product with scales for each token and output channel (tb_int8_gemm),
// and both in one call (tb_int8_connected_fwd).
#include "int8.cuh"

#include <algorithm>
#include <atomic>

namespace tbi {
namespace {

constexpr float QUANT_FLOOR = 0x1p-100f;   // smallest row maximum: 127 / amax stays finite
constexpr int64_t INT8_MAX_K = 131071;     // 128 * 128 * k < 2^31

// ---- quantization ---------------------------------------------------------------------------
// amax of a row as the largest |x| bit pattern: unsigned order is the order of magnitudes, and NaN
// and infinities come out on top (>= 0x7f800000).
struct RowScale {
    float factor, scale;
};
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return {0.f, __uint_as_float(0x7fffffffu)};
    const float amax = fmaxf(__uint_as_float(amax_bits), QUANT_FLOOR);
    return {__fdiv_rn(127.f, amax), __fdiv_rn(amax, 127.f)};
}
// 0 for a row of factor 0: x * 0 is 0 or NaN, and NaN converts to 0
__device__ __forceinline__ int quant_code(float v, float factor) { return __float2int_rn(__fmul_rn(v, factor)); }

// 16 bytes of a row from element i, as floats; past the row's end (or unaligned) element by element
template <typename T, bool VEC>
__device__ __forceinline__ void load_row(const T* __restrict__ x, int64_t i, int64_t cols, float* f) {
    constexpr int E = Vec<T>::N;
    if (VEC && i + E <= cols) {
        const Vec<T> v = *reinterpret_cast<const Vec<T>*>(x + i);
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = Elem<T>::get(v.e[e]);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = i + e < cols ? Elem<T>::get(x[i + e]) : 0.f;
    }
}

template <int E> __device__ __forceinline__ uint32_t max_bits(uint32_t m, const float* f) {
#pragma unroll
    for (int e = 0; e < E; ++e) m = max(m, __float_as_uint(f[e]) & 0x7fffffffu);
    return m;
}

// codes of E values at element i of a row; vec: the row's codes may be written E bytes at a time
template <int E>
__device__ __forceinline__ void put_codes(int8_t* codes, int64_t i, int64_t cols, const float* f, float factor, bool vec) {
    uint32_t w[E / 4];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const uint32_t q = (uint32_t)quant_code(f[e], factor) & 0xffu;
        w[e / 4] = e % 4 ? w[e / 4] | q << 8 * (e % 4) : q;
    }
    if (vec && i + E <= cols) {
        if constexpr (E == 8) *reinterpret_cast<uint2*>(codes + i) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t*>(codes + i) = w[0];
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (i + e < cols) codes[i + e] = (int8_t)(w[e / 4] >> 8 * (e % 4));
    }
}

// A warp (WARP) or a CTA per row. The first 4 x 16 bytes of each thread stay in registers between the
// maximum and the codes, so a row is read once unless it is longer than 64 bytes a thread.
// Memory bound: @@Q@@
template <typename T, bool VEC, bool WARP>
__global__ void k_quantize_rows(int64_t rows, int64_t cols, const T* __restrict__ x, int64_t x_stride, int8_t* codes,
                                int64_t code_stride, float* scales, bool code_vec) {
    TB_GRID_DEP_ENTRY();
    constexpr int E = Vec<T>::N, KEEP = 4;
    const int64_t row = WARP ? (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32 : (int64_t)blockIdx.x;
    if (row >= rows) return;  // whole warps; only where WARP
    const int g = WARP ? 32 : blockDim.x;
    x += row * x_stride;
    codes += row * code_stride;
    const int64_t first = (int64_t)(WARP ? threadIdx.x % 32 : threadIdx.x) * E, step = (int64_t)g * E;
    float f[KEEP][E];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < KEEP; ++j) load_row<T, VEC>(x, first + j * step, cols, f[j]);
#pragma unroll
    for (int j = 0; j < KEEP; ++j) m = max_bits<E>(m, f[j]);
    for (int64_t i = first + KEEP * step; i < cols; i += step) {
        float t[E];
        load_row<T, VEC>(x, i, cols, t);
        m = max_bits<E>(m, t);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if constexpr (!WARP) {
        __shared__ uint32_t part[32];
        if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = m;
        __syncthreads();
        m = threadIdx.x % 32 < blockDim.x / 32 ? part[threadIdx.x % 32] : 0;
        m = __reduce_max_sync(0xffffffffu, m);
    }
    const RowScale s = row_scale(m);
#pragma unroll
    for (int j = 0; j < KEEP; ++j) put_codes<E>(codes, first + j * step, cols, f[j], s.factor, code_vec);
    for (int64_t i = first + KEEP * step; i < cols; i += step) {
        float t[E];
        load_row<T, VEC>(x, i, cols, t);
        put_codes<E>(codes, i, cols, t, s.factor, code_vec);
    }
    if (first == 0) scales[row] = s.scale;
}

int quantize_rows(tb_ctx* ctx, int64_t rows, int64_t cols, const void* x, int64_t x_type, int64_t x_stride,
                  int8_t* codes, int64_t code_stride, float* scales) {
    return elem_dispatch(x_type, [&](auto t) {
        using T = decltype(t);
        constexpr int E = Vec<T>::N;
        const bool vec = aligned16(x) && (rows == 1 || x_stride % E == 0);
        const bool code_vec = (uintptr_t)codes % E == 0 && (rows == 1 || code_stride % E == 0);
        const int64_t vecs = ceil_div(cols, E);
        const T* xt = static_cast<const T*>(x);
        if (vecs <= 128) {
            const unsigned grid = (unsigned)ceil_div(rows, 4);
            return vec ? launch(ctx, "k_quantize_rows", k_quantize_rows<T, true, true>, dim3(grid), dim3(128), 0, rows, cols, xt, x_stride, codes, code_stride, scales, code_vec)
                       : launch(ctx, "k_quantize_rows", k_quantize_rows<T, false, true>, dim3(grid), dim3(128), 0, rows, cols, xt, x_stride, codes, code_stride, scales, code_vec);
        }
        // 64 bytes a thread where there are rows enough to fill the GPU, 16 where a row's latency counts
        const int64_t per = rows >= 4 * ctx->sm_count ? 4 : 1;
        const unsigned threads = (unsigned)std::min<int64_t>(1024, round_up(ceil_div(vecs, per), 32));
        return vec ? launch(ctx, "k_quantize_rows", k_quantize_rows<T, true, false>, dim3((unsigned)rows), dim3(threads), 0, rows, cols, xt, x_stride, codes, code_stride, scales, code_vec)
                   : launch(ctx, "k_quantize_rows", k_quantize_rows<T, false, false>, dim3((unsigned)rows), dim3(threads), 0, rows, cols, xt, x_stride, codes, code_stride, scales, code_vec);
    });
}

// ---- product for a few tokens --------------------------------------------------------------------
// M tokens (1, 2 or 4). The weights are read once and that bounds it, so they stream straight into
// registers: a warp takes two channels, each lane 16 bytes of k at a time, and multiplies them with
// the tokens' codes in shared memory (dp4a). Every CTA quantizes the tokens for itself while
// its first weights are on their way, which saves the launch, and the round trip, of a quantizer.
// @@V@@
constexpr int GEMV_WARPS = 8, GEMV_CH = 2, GEMV_U = 4;
constexpr int GEMV_SMEM = 64 * 1024;  // most bytes of codes

struct GemvArgs {
    Int8Args p;        // p.a, p.a_scales: null where x is given
    const void* x;
    int64_t x_stride;
    int y_type;
};

__device__ __forceinline__ int4 load_codes(const int8_t* __restrict__ row, int64_t v, int64_t k) {
    if ((v + 1) * 16 <= k) return __ldg(reinterpret_cast<const int4*>(row) + v);
    int4 r = make_int4(0, 0, 0, 0);  // the row's last, partial 16 bytes
    int8_t* b = reinterpret_cast<int8_t*>(&r);
    for (int i = 0; i < 16; ++i)
        if (v * 16 + i < k) b[i] = row[v * 16 + i];
    return r;
}

__device__ __forceinline__ void put_any(void* y, int type, int64_t i, float v) {
    if (type == TB_F32) static_cast<float*>(y)[i] = v;
    else if (type == TB_BF16) static_cast<__nv_bfloat16*>(y)[i] = Elem<__nv_bfloat16>::put(v);
    else static_cast<__half*>(y)[i] = Elem<__half>::put(v);
}

// T: x's type, or int8_t where the codes are given
template <typename T, bool VEC, int M>
__global__ void __launch_bounds__(GEMV_WARPS * 32) k_int8_gemv(const GemvArgs g) {
    TB_GRID_DEP_ENTRY();
    const Int8Args& p = g.p;
    extern __shared__ __align__(16) int8_t xs[];  // [M][kp]
    __shared__ float scales[M];
    __shared__ uint32_t part[GEMV_WARPS][M];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t k = p.k;
    const int kp = (int)((k + 15) / 16 * 16), nv = kp / 16;
    const int64_t c0 = ((int64_t)blockIdx.x * GEMV_WARPS + warp) * GEMV_CH;
    const int8_t* row[GEMV_CH];
#pragma unroll
    for (int c = 0; c < GEMV_CH; ++c) row[c] = p.w + min(c0 + c, p.n - 1) * p.w_stride;

    int4 w[GEMV_U][GEMV_CH];
    auto fetch = [&](int s) {
#pragma unroll
        for (int u = 0; u < GEMV_U; ++u) {
            const int v = (s + u) * 32 + lane;
#pragma unroll
            for (int c = 0; c < GEMV_CH; ++c) w[u][c] = v < nv ? load_codes(row[c], v, k) : make_int4(0, 0, 0, 0);
        }
    };
    fetch(0);

    if constexpr (sizeof(T) == 1) {
        for (int i = tid; i < M * nv; i += GEMV_WARPS * 32) {
            const int r = i / nv, v = i - r * nv;
            reinterpret_cast<int4*>(xs + r * kp)[v] = load_codes(p.a + r * p.a_stride, v, k);
        }
        if (tid < M) scales[tid] = p.a_scales[tid];
        __syncthreads();
    } else {
        constexpr int E = Vec<T>::N;
        const T* x = static_cast<const T*>(g.x);
        uint32_t m[M];
#pragma unroll
        for (int r = 0; r < M; ++r) {
            m[r] = 0;
            for (int64_t i = (int64_t)tid * E; i < k; i += GEMV_WARPS * 32 * E) {
                float f[E];
                load_row<T, VEC>(x + r * g.x_stride, i, k, f);
                m[r] = max_bits<E>(m[r], f);
            }
        }
#pragma unroll
        for (int r = 0; r < M; ++r) {
            m[r] = __reduce_max_sync(0xffffffffu, m[r]);
            if (lane == 0) part[warp][r] = m[r];
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < M; ++r) {
            m[r] = 0;
            for (int i = 0; i < GEMV_WARPS; ++i) m[r] = max(m[r], part[i][r]);
            const RowScale s = row_scale(m[r]);
            if (tid == 0) scales[r] = s.scale;
            for (int64_t i = (int64_t)tid * E; i < kp; i += GEMV_WARPS * 32 * E) {  // zeros between k and kp
                float f[E];
                load_row<T, VEC>(x + r * g.x_stride, i, k, f);
                put_codes<E>(xs + r * kp, i, kp, f, s.factor, true);
            }
        }
        __syncthreads();
    }

    int acc[GEMV_CH][M] = {};
    const int steps = (nv + 31) / 32;
    for (int s = 0; s < steps; s += GEMV_U) {
        int4 now[GEMV_U][GEMV_CH];
#pragma unroll
        for (int u = 0; u < GEMV_U; ++u)
#pragma unroll
            for (int c = 0; c < GEMV_CH; ++c) now[u][c] = w[u][c];
        if (s + GEMV_U < steps) fetch(s + GEMV_U);
#pragma unroll
        for (int u = 0; u < GEMV_U; ++u) {
            const int v = (s + u) * 32 + lane;
            if (v < nv) {
#pragma unroll
                for (int r = 0; r < M; ++r) {
                    const int4 q = reinterpret_cast<const int4*>(xs + r * kp)[v];
#pragma unroll
                    for (int c = 0; c < GEMV_CH; ++c) {
                        acc[c][r] = __dp4a(now[u][c].x, q.x, acc[c][r]);
                        acc[c][r] = __dp4a(now[u][c].y, q.y, acc[c][r]);
                        acc[c][r] = __dp4a(now[u][c].z, q.z, acc[c][r]);
                        acc[c][r] = __dp4a(now[u][c].w, q.w, acc[c][r]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int c = 0; c < GEMV_CH; ++c)
#pragma unroll
        for (int r = 0; r < M; ++r) {
            const int a = __reduce_add_sync(0xffffffffu, acc[c][r]);
            const int64_t ch = c0 + c;
            if (lane == 0 && ch < p.n)
                put_any(p.y, g.y_type, r * p.y_stride + ch,
                        int8_epilogue(a, __fmul_rn(scales[r], __ldg(p.w_scales + ch)), p.bias ? __ldg(p.bias + ch) : 0.f, p.bias != nullptr, p.act));
        }
}

// Up to 4 tokens whose codes fit, else the tensor cores: @@G@@
bool use_gemv(int64_t m, int64_t k) { return (m == 1 || m == 2 || m == 4) && m * round_up(k, 16) <= GEMV_SMEM; }

template <typename T, bool VEC, int M> int launch_gemv_m(tb_ctx* ctx, const GemvArgs& g) {
    const int smem = (int)(M * round_up(g.p.k, 16));
    static std::atomic<bool> done[64];  // the attribute is set once per kernel and device
    if (ctx->device >= 64 || !done[ctx->device].load(std::memory_order_acquire)) {
        cudaError_t e = cudaFuncSetAttribute(k_int8_gemv<T, VEC, M>, cudaFuncAttributeMaxDynamicSharedMemorySize, GEMV_SMEM);
        if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(int8 gemv)");
        if (ctx->device < 64) done[ctx->device].store(true, std::memory_order_release);
    }
    const int64_t grid = ceil_div(g.p.n, GEMV_WARPS * GEMV_CH);
    return launch(ctx, "k_int8_gemv", k_int8_gemv<T, VEC, M>, dim3((unsigned)grid), dim3(GEMV_WARPS * 32), (size_t)smem, g);
}

template <typename T, bool VEC> int launch_gemv(tb_ctx* ctx, const GemvArgs& g) {
    switch (g.p.m) {
    case 1: return launch_gemv_m<T, VEC, 1>(ctx, g);
    case 2: return launch_gemv_m<T, VEC, 2>(ctx, g);
    default: return launch_gemv_m<T, VEC, 4>(ctx, g);
    }
}

constexpr int64_t MAX_DIM = 2147483647;

int check_quantize(int64_t rows, int64_t cols, const void* x, int64_t x_type, int64_t x_stride) {
    if (rows < 0 || cols <= 0 || rows > MAX_DIM || cols > MAX_DIM) return fail(TB_ERR_INVALID, "quantize: bad shape");
    if (!elem_type_ok(x_type)) return fail(TB_ERR_UNSUPPORTED, "quantize: element type %lld", (long long)x_type);
    if (rows > 1 && x_stride != 0 && x_stride < cols) return fail(TB_ERR_INVALID, "quantize: row stride below the row's length");
    if (rows > 0 && !x) return fail(TB_ERR_INVALID, "quantize: null pointer");
    if ((uintptr_t)x % elem_size(x_type)) return fail(TB_ERR_INVALID, "quantize: misaligned pointer");
    return TB_OK;
}

// what the product asks of everything but its a operand
int check_product(int64_t m, int64_t n, int64_t k, const int8_t* w, int64_t w_stride, const float* w_scales,
                  int64_t act, void* y, int64_t y_type, int64_t y_stride) {
    if (m < 0 || n < 0 || k <= 0 || m > MAX_DIM || n > MAX_DIM) return fail(TB_ERR_INVALID, "int8 product: bad shape");
    if (k > INT8_MAX_K) return fail(TB_ERR_UNSUPPORTED, "int8 product: k over %lld can overflow the int32 sum", (long long)INT8_MAX_K);
    if (!act_supported(act)) return fail(TB_ERR_UNSUPPORTED, "int8 product: activation %lld not supported", (long long)act);
    if (!elem_type_ok(y_type)) return fail(TB_ERR_UNSUPPORTED, "int8 product: element type %lld", (long long)y_type);
    if (m == 0 || n == 0) return TB_OK;
    if (!w || !w_scales || !y) return fail(TB_ERR_INVALID, "int8 product: null pointer");
    if ((uintptr_t)y % elem_size(y_type)) return fail(TB_ERR_INVALID, "int8 product: misaligned output");
    if (!aligned16(w) || w_stride % 16) return fail(TB_ERR_INVALID, "int8 product: w and its stride have to be multiples of 16 bytes");
    if ((n > 1 && w_stride < k) || (m > 1 && y_stride < n)) return fail(TB_ERR_INVALID, "int8 product: row stride below the row's length");
    return TB_OK;
}

}  // namespace
}  // namespace tbi

using namespace tbi;

extern "C" {

int tb_quantize_rows(tb_ctx* ctx, int64_t rows, int64_t cols, const void* x, int64_t x_type, int64_t x_stride,
                     int8_t* codes, int64_t code_stride, float* scales) {
    TB_ENTER(ctx);
    int r = check_quantize(rows, cols, x, x_type, x_stride);
    if (r != TB_OK) return r;
    if (rows == 0) return TB_OK;
    if (!codes || !scales) return fail(TB_ERR_INVALID, "quantize: null pointer");
    if (rows > 1 && code_stride < cols) return fail(TB_ERR_INVALID, "quantize: row stride below the row's length");
    return quantize_rows(ctx, rows, cols, x, x_type, x_stride, codes, code_stride, scales);
}

int tb_int8_gemm(tb_ctx* ctx, int64_t m, int64_t n, int64_t k, const int8_t* a, int64_t a_stride,
                 const float* a_scales, const int8_t* w, int64_t w_stride, const float* w_scales,
                 const float* bias, int64_t activation, void* y, int64_t y_type, int64_t y_stride) {
    TB_ENTER(ctx);
    int r = check_product(m, n, k, w, w_stride, w_scales, activation, y, y_type, y_stride);
    if (r != TB_OK) return r;
    if (m == 0 || n == 0) return TB_OK;
    if (!a || !a_scales) return fail(TB_ERR_INVALID, "int8 product: null pointer");
    if (!aligned16(a) || a_stride % 16) return fail(TB_ERR_INVALID, "int8 product: a and its stride have to be multiples of 16 bytes");
    if (m > 1 && a_stride < k) return fail(TB_ERR_INVALID, "int8 product: row stride below the row's length");
    const Int8Args p{m, n, k, a, a_stride, a_scales, w, w_stride, w_scales, bias, (int)activation, y, y_stride};
    if (use_gemv(m, k)) return launch_gemv<int8_t, true>(ctx, GemvArgs{p, nullptr, 0, (int)y_type});
    return int8_gemm_tc(ctx, p, y_type, false);
}

int tb_int8_connected_fwd(tb_ctx* ctx, int64_t m, int64_t n, int64_t k, const void* x, int64_t x_type,
                          int64_t x_stride, const int8_t* w, int64_t w_stride, const float* w_scales,
                          const float* bias, int64_t activation, void* y, int64_t y_type, int64_t y_stride) {
    TB_ENTER(ctx);
    int r = check_product(m, n, k, w, w_stride, w_scales, activation, y, y_type, y_stride);
    if (r != TB_OK) return r;
    if ((r = check_quantize(m, k, x, x_type, x_stride)) != TB_OK) return r;
    if (m == 0 || n == 0) return TB_OK;
    Int8Args p{m, n, k, nullptr, 0, nullptr, w, w_stride, w_scales, bias, (int)activation, y, y_stride};
    if (use_gemv(m, k)) {
        const GemvArgs g{p, x, x_stride, (int)y_type};
        return elem_dispatch(x_type, [&](auto t) {
            using T = decltype(t);
            return aligned16(x) && (m == 1 || x_stride % Vec<T>::N == 0) ? launch_gemv<T, true>(ctx, g) : launch_gemv<T, false>(ctx, g);
        });
    }
    const int64_t stride = round_up(k, 16), scale_bytes = round_up(m * 4, 256);
    if ((r = ensure_workspace(ctx, (size_t)(scale_bytes + m * stride))) != TB_OK) return r;
    float* scales = static_cast<float*>(ctx->ws);
    int8_t* codes = reinterpret_cast<int8_t*>(scales) + scale_bytes;
    if ((r = quantize_rows(ctx, m, k, x, x_type, x_stride, codes, stride, scales)) != TB_OK) return r;
    p.a = codes;
    p.a_stride = stride;
    p.a_scales = scales;
    return int8_gemm_tc(ctx, p, y_type, true);
}

}  // extern "C"

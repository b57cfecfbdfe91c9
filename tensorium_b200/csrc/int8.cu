// int8.cu -- the connected layer on int8 operands: rows quantized with a scale each
// (tb_quantize_rows), the product with scales for each token and output channel (tb_int8_gemm),
// and both in one call (tb_int8_connected_fwd).
#include "elem.cuh"

#include <algorithm>

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

// One CTA per row, any length, any alignment: the row is read twice.
template <typename T>
__global__ void k_quantize_rows(int64_t cols, const T* __restrict__ x, int64_t x_stride, int8_t* __restrict__ codes,
                                int64_t code_stride, float* __restrict__ scales) {
    TB_GRID_DEP_ENTRY();
    const int64_t row = blockIdx.x;
    x += row * x_stride;
    codes += row * code_stride;
    uint32_t m = 0;
    for (int64_t i = threadIdx.x; i < cols; i += blockDim.x)
        m = max(m, __float_as_uint(Elem<T>::get(x[i])) & 0x7fffffffu);
    __shared__ uint32_t part[32];
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
    m = threadIdx.x % 32 < blockDim.x / 32 ? part[threadIdx.x % 32] : 0;
    m = __reduce_max_sync(0xffffffffu, m);
    const RowScale s = row_scale(m);
    for (int64_t i = threadIdx.x; i < cols; i += blockDim.x) codes[i] = (int8_t)quant_code(Elem<T>::get(x[i]), s.factor);
    if (threadIdx.x == 0) scales[row] = s.scale;
}

int quantize_rows(tb_ctx* ctx, int64_t rows, int64_t cols, const void* x, int64_t x_type, int64_t x_stride,
                  int8_t* codes, int64_t code_stride, float* scales) {
    return elem_dispatch(x_type, [&](auto t) {
        using T = decltype(t);
        return launch(ctx, "k_quantize_rows", k_quantize_rows<T>, dim3((unsigned)rows), dim3(256), 0, cols,
                      static_cast<const T*>(x), x_stride, codes, code_stride, scales);
    });
}

// ---- product ----------------------------------------------------------------------------------
struct GemmArgs {
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

// 64 tokens x 64 channels per CTA, 4 x 4 per thread, k in steps of 64 bytes.
template <typename T>
__global__ void __launch_bounds__(256) k_int8_gemm(const GemmArgs p) {
    TB_GRID_DEP_ENTRY();
    __shared__ int as[64][17], ws[64][17];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int64_t m0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
    int acc[4][4] = {};
    for (int64_t k0 = 0; k0 < p.k; k0 += 64) {
        for (int e = tid; e < 64 * 64; e += 256) {
            const int r = e >> 6, c = e & 63;
            const bool in = k0 + c < p.k;
            reinterpret_cast<int8_t*>(as[r])[c] = in && m0 + r < p.m ? p.a[(m0 + r) * p.a_stride + k0 + c] : (int8_t)0;
            reinterpret_cast<int8_t*>(ws[r])[c] = in && n0 + r < p.n ? p.w[(n0 + r) * p.w_stride + k0 + c] : (int8_t)0;
        }
        __syncthreads();
        for (int kk = 0; kk < 16; ++kk) {
            int av[4], wv[4];
            for (int i = 0; i < 4; ++i) av[i] = as[ty + 16 * i][kk], wv[i] = ws[tx + 16 * i][kk];
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(av[i], wv[j], acc[i][j]);
        }
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i) {
        const int64_t m = m0 + ty + 16 * i;
        if (m >= p.m) continue;
        const float s = p.a_scales[m];
        for (int j = 0; j < 4; ++j) {
            const int64_t n = n0 + tx + 16 * j;
            if (n >= p.n) continue;
            const float v = int8_epilogue(acc[i][j], __fmul_rn(s, p.w_scales[n]), p.bias ? p.bias[n] : 0.f, p.bias != nullptr, p.act);
            static_cast<T*>(p.y)[m * p.y_stride + n] = Elem<T>::put(v);
        }
    }
}

int int8_gemm(tb_ctx* ctx, const GemmArgs& p, int64_t y_type) {
    const int64_t gx = ceil_div(p.n, 64), gy = ceil_div(p.m, 64);
    if (gy > 65535) return fail(TB_ERR_UNSUPPORTED, "int8 product: more than 4194240 tokens");
    return elem_dispatch(y_type, [&](auto t) {
        return launch(ctx, "k_int8_gemm", k_int8_gemm<decltype(t)>, dim3((unsigned)gx, (unsigned)gy), dim3(256), 0, p);
    });
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
    return int8_gemm(ctx, GemmArgs{m, n, k, a, a_stride, a_scales, w, w_stride, w_scales, bias, (int)activation, y, y_stride}, y_type);
}

int tb_int8_connected_fwd(tb_ctx* ctx, int64_t m, int64_t n, int64_t k, const void* x, int64_t x_type,
                          int64_t x_stride, const int8_t* w, int64_t w_stride, const float* w_scales,
                          const float* bias, int64_t activation, void* y, int64_t y_type, int64_t y_stride) {
    TB_ENTER(ctx);
    int r = check_product(m, n, k, w, w_stride, w_scales, activation, y, y_type, y_stride);
    if (r != TB_OK) return r;
    if ((r = check_quantize(m, k, x, x_type, x_stride)) != TB_OK) return r;
    if (m == 0 || n == 0) return TB_OK;
    const int64_t stride = round_up(k, 16), scale_bytes = round_up(m * 4, 256);
    if ((r = ensure_workspace(ctx, (size_t)(scale_bytes + m * stride))) != TB_OK) return r;
    float* scales = static_cast<float*>(ctx->ws);
    int8_t* codes = reinterpret_cast<int8_t*>(scales) + scale_bytes;
    if ((r = quantize_rows(ctx, m, k, x, x_type, x_stride, codes, stride, scales)) != TB_OK) return r;
    return int8_gemm(ctx, GemmArgs{m, n, k, codes, stride, scales, w, w_stride, w_scales, bias, (int)activation, y, y_stride}, y_type);
}

}  // extern "C"

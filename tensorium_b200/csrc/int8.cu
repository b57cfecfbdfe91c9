// int8.cu -- the connected layer on int8 operands: rows quantized with a scale each
// (tb_quantize_rows), the product with scales for each token and output channel (tb_int8_gemm),
// and both in one call (tb_int8_connected_fwd).
#include "int8.cuh"

#include <algorithm>
#include <atomic>
#include <cstring>

namespace tbi {
namespace {

constexpr float QUANT_FLOOR = 0x1p-100f;   // smallest row maximum: 127 / amax stays finite
constexpr int64_t INT8_MAX_K = 131071;     // 128 * 128 * k < 2^31

// ---- quantization ---------------------------------------------------------------------------
// amax of a row as the largest |x| bit pattern: unsigned order is the order of magnitudes, and NaN
// and infinities come out on top (>= 0x7f800000).
struct RowScale {
    float factor, scale;
    uint32_t keep;  // 0 for a row with a NaN or an infinity, whose codes are 0
};
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return {0.f, __uint_as_float(0x7fffffffu), 0u};
    const float amax = fmaxf(__uint_as_float(amax_bits), QUANT_FLOOR);
    return {__fdiv_rn(127.f, amax), __fdiv_rn(amax, 127.f), ~0u};
}

// 16 bytes of a row of x: magnitudes and codes.
template <typename T> struct Raw {
    static constexpr int E = 16 / sizeof(T);
    // elements i .. i + E - 1, zeros past the row's end; not VEC: element by element
    template <bool VEC> static __device__ __forceinline__ uint4 load(const T* __restrict__ x, int64_t i, int64_t cols) {
        if (VEC && i + E <= cols) return *reinterpret_cast<const uint4*>(x + i);
        uint4 r = make_uint4(0, 0, 0, 0);
        if (i < cols) {
            T t[E];
            memcpy(t, &r, 16);
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (i + e < cols) t[e] = x[i + e];
            memcpy(&r, t, 16);
        }
        return r;
    }
    // running maximum of the magnitudes' bits: of floats, or of both halves of a word on their own
    static __device__ __forceinline__ uint32_t amax(uint32_t m, const uint4& r) {
        if constexpr (sizeof(T) == 4) {
            m = max(m, max(r.x & 0x7fffffffu, r.y & 0x7fffffffu));
            return max(m, max(r.z & 0x7fffffffu, r.w & 0x7fffffffu));
        } else {
            m = __vmaxu2(m, __vmaxu2(r.x & 0x7fff7fffu, r.y & 0x7fff7fffu));
            return __vmaxu2(m, __vmaxu2(r.z & 0x7fff7fffu, r.w & 0x7fff7fffu));
        }
    }
    // that maximum as the bits of a float
    static __device__ __forceinline__ uint32_t amax_bits(uint32_t m) {
        if constexpr (sizeof(T) == 4) return m;
        const unsigned short h = (unsigned short)max(m & 0xffffu, m >> 16);
        T v;
        memcpy(&v, &h, sizeof(T) == 4 ? 2 : sizeof(T));
        return __float_as_uint(Elem<T>::get(v));
    }
    // rint(v * factor) of the E elements as bytes: adding 1.5 * 2^23 rounds to a whole number (to even, as rint does) whose
    // low byte is the code's
    static __device__ __forceinline__ void codes(const uint4& r, const RowScale& s, uint32_t* out) {
        T t[E];
        memcpy(t, &r, 16);
        uint32_t q[E];
#pragma unroll
        for (int e = 0; e < E; ++e) q[e] = __float_as_uint(__fadd_rn(__fmul_rn(Elem<T>::get(t[e]), s.factor), 12582912.f));
#pragma unroll
        for (int e = 0; e < E; e += 4)
            out[e / 4] = __byte_perm(__byte_perm(q[e], q[e + 1], 0x0040), __byte_perm(q[e + 2], q[e + 3], 0x0040), 0x5410) & s.keep;
    }
};

// the codes of 16 bytes of x to element i of a row; vec: the row's codes may be written E bytes at a time
template <typename T>
__device__ __forceinline__ void put_codes(int8_t* codes, int64_t i, int64_t cols, const uint4& r, const RowScale& s, bool vec) {
    constexpr int E = Raw<T>::E;
    uint32_t w[E / 4];
    Raw<T>::codes(r, s, w);
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
// Memory bound: 8192 x 8192 bf16 in 34 us, 5.9 TB/s (0.91 of a copy's rate); one row of 4096 in 2.6 us, a launch's latency.
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
    uint4 f[KEEP];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < KEEP; ++j) f[j] = Raw<T>::template load<VEC>(x, first + j * step, cols);
#pragma unroll
    for (int j = 0; j < KEEP; ++j) m = Raw<T>::amax(m, f[j]);
#pragma unroll 4
    for (int64_t i = first + KEEP * step; i < cols; i += step) m = Raw<T>::amax(m, Raw<T>::template load<VEC>(x, i, cols));
    m = __reduce_max_sync(0xffffffffu, Raw<T>::amax_bits(m));
    if constexpr (!WARP) {
        __shared__ uint32_t part[32];
        if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = m;
        __syncthreads();
        m = threadIdx.x % 32 < blockDim.x / 32 ? part[threadIdx.x % 32] : 0;
        m = __reduce_max_sync(0xffffffffu, m);
    }
    const RowScale s = row_scale(m);
#pragma unroll
    for (int j = 0; j < KEEP; ++j) put_codes<T>(codes, first + j * step, cols, f[j], s, code_vec);
#pragma unroll 4
    for (int64_t i = first + KEEP * step; i < cols; i += step)
        put_codes<T>(codes, i, cols, Raw<T>::template load<VEC>(x, i, cols), s, code_vec);
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
            return vec ? launch_early(ctx, "k_quantize_rows", k_quantize_rows<T, true, true>, dim3(grid), dim3(128), 0, rows, cols, xt, x_stride, codes, code_stride, scales, code_vec)
                       : launch_early(ctx, "k_quantize_rows", k_quantize_rows<T, false, true>, dim3(grid), dim3(128), 0, rows, cols, xt, x_stride, codes, code_stride, scales, code_vec);
        }
        // 64 bytes a thread where there are rows enough to fill the GPU, 16 where a row's latency counts
        const int64_t per = rows >= 4 * ctx->sm_count ? 4 : 1;
        const unsigned threads = (unsigned)std::min<int64_t>(1024, round_up(ceil_div(vecs, per), 32));
        return vec ? launch_early(ctx, "k_quantize_rows", k_quantize_rows<T, true, false>, dim3((unsigned)rows), dim3(threads), 0, rows, cols, xt, x_stride, codes, code_stride, scales, code_vec)
                   : launch_early(ctx, "k_quantize_rows", k_quantize_rows<T, false, false>, dim3((unsigned)rows), dim3(threads), 0, rows, cols, xt, x_stride, codes, code_stride, scales, code_vec);
    });
}

// ---- product for a few tokens --------------------------------------------------------------------
// Up to 8 or 16 tokens (B8 tiles of 8). The weights are read once and that bounds it. A lane's 16 bytes of two
// weight rows are fragments of mma.m16n8k32 (16 channels x 32 k x 8 tokens) as they come: the sum over k may take
// k in any order, so they serve two products, with the tokens' codes taken from shared memory in the same
// order. One CTA per SM walks groups of 16 channels: KW of its warps share a group, each taking interleaved
// 64-byte steps of k through a ring of its own (cp.async, read back by the lane that copied it: no barrier), FEW_RING
// steps ahead and on into the next groups; the int32 partial sums meet in shared memory. A CTA quantizes the
// tokens for itself while its first weights are on their way, which saves the launch, and the round trip, of
// a quantizer. 1 to 4 tokens x 4096 x 4096: 7.0 to 7.3 us where the bytes take 2.6, the rest being the launch, the first loads' and the
// last sums' latency; 4 x 16384 x 4096: 16.1 us (4.2 TB/s). (Times in this file: in a graph of calls on
// several weights in turn, larger than L2 together.)
constexpr int FEW_WARPS = 16, FEW_RING = 6, FEW_THREADS = FEW_WARPS * 32;
constexpr int FEW_RING_BYTES = FEW_WARPS * FEW_RING * 1024;
constexpr int FEW_CODES = 96 * 1024;  // most bytes of codes

struct FewArgs {
    Int8Args p;        // p.a, p.a_scales: null where x is given
    const void* x;
    int64_t x_stride;
    int y_type;
    int kw;            // warps to a group of channels: 1, 2, 4, 8 or 16
};

__host__ __device__ constexpr int64_t few_pitch(int64_t k) {  // 64 more than a multiple of 128: conflict-free
    const int64_t kp = (k + 63) / 64 * 64;
    return kp % 128 ? kp : kp + 64;
}

// bytes of a row of k from byte i on, up to 16 (0 past its end)
__device__ __forceinline__ int left16(int64_t i, int64_t k) { return (int)max((int64_t)0, min((int64_t)16, k - i)); }

// 16 bytes of a row from byte i on into shared memory, zeros past the row's end
__device__ __forceinline__ void copy16(void* to, const int8_t* row, int64_t i, int64_t k) {
    const int n = left16(i, k);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(row + (n ? i : 0)), "r"(n)
                 : "memory");
}

__device__ __forceinline__ void put_any(void* y, int type, int64_t i, float v) {
    if (type == TB_F32) static_cast<float*>(y)[i] = v;
    else if (type == TB_BF16) static_cast<__nv_bfloat16*>(y)[i] = Elem<__nv_bfloat16>::put(v);
    else static_cast<__half*>(y)[i] = Elem<__half>::put(v);
}

__device__ __forceinline__ void mma_s8(int (&d)[4], int a0, int a1, int a2, int a3, int b0, int b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// T: x's type, or int8_t where the codes are given
template <typename T, bool VEC, int B8>
__global__ void __launch_bounds__(FEW_THREADS, 1) k_int8_few(const FewArgs g) {
    TB_GRID_DEP_ENTRY();
    constexpr int TOKENS = B8 * 8;
    const Int8Args& p = g.p;
    extern __shared__ __align__(16) int8_t dyn[];  // rings, then codes [m][pitch]
    __shared__ float scales[TOKENS];
    __shared__ uint32_t part[FEW_WARPS];
    __shared__ int sums[2][FEW_WARPS][TOKENS][17];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int m = (int)p.m, kw = g.kw, gw = FEW_WARPS / kw;  // gw groups at a time
    const int64_t k = p.k;
    const int pitch = (int)few_pitch(k), steps = (int)((k + 63) / 64);
    const int groups = (int)((p.n + 15) / 16), stride = gridDim.x * gw, s0 = warp % kw;
    int4* const ring = reinterpret_cast<int4*>(dyn) + warp * FEW_RING * 64 + lane;
    int8_t* const xs = dyn + FEW_RING_BYTES;

    // x first, then the weights' first steps: loads come back in order
    constexpr int E = 16 / sizeof(T);
    int wr = FEW_WARPS;  // the warps share out the rows: 16, 8, 4, 2 or 1 to a row
    while (wr > 1 && FEW_WARPS / wr < m) wr /= 2;
    const int r = warp / wr, t = (warp % wr) * 32 + lane, step = wr * 32 * E;
    [[maybe_unused]] uint4 f[4];
    [[maybe_unused]] const T* row = sizeof(T) == 1 ? nullptr : static_cast<const T*>(g.x) + (r < m ? r : 0) * g.x_stride;
    if constexpr (sizeof(T) > 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = Raw<T>::template load<VEC>(row, (int64_t)t * E + j * step, r < m ? k : 0);
    }

    int fgroup = blockIdx.x * gw + warp / kw, fs = s0, fslot = 0;  // the next step to fetch
    auto fetch = [&] {
        if (fgroup < groups) {
            const int64_t c = (int64_t)fgroup * 16 + lane / 4;
            const int64_t i = (int64_t)fs * 64 + lane % 4 * 16;
            if (fs < steps) {
                copy16(ring + fslot * 64, p.w + min(c, p.n - 1) * p.w_stride, i, k);
                copy16(ring + fslot * 64 + 32, p.w + min(c + 8, p.n - 1) * p.w_stride, i, k);
            }
            fs += kw;
            if (fs >= steps) fs = s0, fgroup += stride;
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
        fslot = fslot + 1 == FEW_RING ? 0 : fslot + 1;
    };
#pragma unroll 1
    for (int i = 0; i < FEW_RING; ++i) fetch();

    if constexpr (sizeof(T) == 1) {
        const int nv = steps * 4;
        for (int i = tid; i < m * nv; i += FEW_THREADS) {
            const int rr = i / nv, v = i - rr * nv, n = left16((int64_t)v * 16, k);
            const int8_t* from = p.a + rr * p.a_stride + (int64_t)v * 16;
            int4 q = make_int4(0, 0, 0, 0);
            if (n == 16) {
                q = __ldg(reinterpret_cast<const int4*>(from));
            } else {
                int8_t b[16];
                for (int e = 0; e < 16; ++e) b[e] = e < n ? from[e] : (int8_t)0;
                memcpy(&q, b, 16);
            }
            reinterpret_cast<int4*>(xs + rr * pitch)[v] = q;
        }
        if (tid < m) scales[tid] = p.a_scales[tid];
    } else {
        uint32_t a = 0;
        if (r < m) {
#pragma unroll
            for (int j = 0; j < 4; ++j) a = Raw<T>::amax(a, f[j]);
#pragma unroll 4
            for (int64_t i = (int64_t)t * E + 4 * step; i < k; i += step) a = Raw<T>::amax(a, Raw<T>::template load<VEC>(row, i, k));
        }
        a = __reduce_max_sync(0xffffffffu, Raw<T>::amax_bits(a));
        if (lane == 0) part[warp] = a;
        __syncthreads();
        if (r < m) {
            a = 0;
            for (int i = 0; i < wr; ++i) a = max(a, part[r * wr + i]);
            const RowScale s = row_scale(a);
            if (t == 0) scales[r] = s.scale;
            int8_t* to = xs + r * pitch;
            const int end = steps * 64;  // zeros from k on
#pragma unroll
            for (int j = 0; j < 4; ++j) put_codes<T>(to, (int64_t)t * E + j * step, end, f[j], s, true);
#pragma unroll 4
            for (int64_t i = (int64_t)t * E + 4 * step; i < end; i += step)
                put_codes<T>(to, i, end, Raw<T>::template load<VEC>(row, i, k), s, true);
        }
    }
    __syncthreads();

    int buf = 0, slot = 0;
    for (int base = blockIdx.x * gw; base < groups; base += stride, buf ^= 1) {  // the same rounds for all warps
        int acc[B8][4] = {};
        // a warp with no step of its own in a group (fewer steps than warps) has an empty one in its ring
        if (base + warp / kw < groups)
#pragma unroll 1
            for (int s = s0; s == s0 || s < steps; s += kw) {
                asm volatile("cp.async.wait_group %0;\n" ::"n"(FEW_RING - 1) : "memory");
                const int4 lo = ring[slot * 64], hi = ring[slot * 64 + 32];
                slot = slot + 1 == FEW_RING ? 0 : slot + 1;
                if (s < steps) {
#pragma unroll
                    for (int b = 0; b < B8; ++b) {
                        int4 q = make_int4(0, 0, 0, 0);
                        if (b * 8 + lane / 4 < m) q = *reinterpret_cast<const int4*>(xs + (b * 8 + lane / 4) * pitch + s * 64 + lane % 4 * 16);
                        mma_s8(acc[b], lo.x, hi.x, lo.y, hi.y, q.x, q.y);
                        mma_s8(acc[b], lo.z, hi.z, lo.w, hi.w, q.z, q.w);
                    }
                }
                fetch();
            }
#pragma unroll
        for (int b = 0; b < B8; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[buf][warp][b * 8 + lane % 4 * 2 + i % 2][lane / 4 + i / 2 * 8] = acc[b][i];
        __syncthreads();  // the buffer of two rounds ago has been read by every thread that is past this
        for (int i = tid; i < gw * m * 16; i += FEW_THREADS) {
            const int c = i % 16, j = i / 16 % gw, tok = i / 16 / gw;  // a token's groups side by side
            const int64_t ch = (int64_t)(base + j) * 16 + c;
            if (ch >= p.n) continue;
            int a = 0;
            for (int w = 0; w < kw; ++w) a += sums[buf][j * kw + w][tok][c];
            float v = __fmul_rn(__int2float_rn(a), __fmul_rn(scales[tok], __ldg(p.w_scales + ch)));
            if (p.bias) v = __fadd_rn(v, __ldg(p.bias + ch));
            put_any(p.y, g.y_type, tok * p.y_stride + ch, tb_activate_dev(v, p.act));
        }
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
}

// Up to 16 tokens whose codes fit, where that is the faster of the two. Measured, us: this one 4.6 + 0.178 a MB of
// weights + 0.1 a thousand values of x (each CTA quantizes them); the tensor cores 7.5 + 0.155 a MB, 4 more where
// their tiles are too few to fill the SMs whole. 4096 x 4096: 7.0 and 12.9 for 4 tokens, 13.8 and 13.4 for 16; 16384 x 4096: 16.1
// and 16.9 for 4 tokens, 18.6 and 17.0 for 8; 131072 x 4096: 103 and 92 for 1.
bool use_few(const tb_ctx* ctx, int64_t m, int64_t n, int64_t k) {
    if (m > 16 || m * few_pitch(k) > FEW_CODES) return false;
    const double more = 1e-4 * (double)(m * k) + 2.3e-8 * (double)(n * k);
    return more < (ceil_div(n, 128) * 5 >= (int64_t)ctx->sm_count * 4 ? 3.2 : 6.5);
}

template <typename T, bool VEC, int B8> int launch_few_b(tb_ctx* ctx, const FewArgs& g) {
    static std::atomic<bool> done[64];  // the attribute is set once per kernel and device
    if (ctx->device >= 64 || !done[ctx->device].load(std::memory_order_acquire)) {
        cudaError_t e = cudaFuncSetAttribute(k_int8_few<T, VEC, B8>, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW_RING_BYTES + FEW_CODES);
        if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(k_int8_few)");
        if (ctx->device < 64) done[ctx->device].store(true, std::memory_order_release);
    }
    // every warp four steps of a group or more, unless there are few groups: then all warps to each
    FewArgs a = g;
    const int64_t groups = ceil_div(g.p.n, 16), steps = ceil_div(g.p.k, 64);
    a.kw = FEW_WARPS;
    while (a.kw > 1 && steps < a.kw * 4 && groups >= (int64_t)ctx->sm_count * (FEW_WARPS / a.kw) * 2) a.kw /= 2;
    const int64_t grid = std::min<int64_t>(ceil_div(groups, FEW_WARPS / a.kw), ctx->sm_count);
    return launch_early(ctx, "k_int8_few", k_int8_few<T, VEC, B8>, dim3((unsigned)grid), dim3(FEW_THREADS),
                  (size_t)(FEW_RING_BYTES + g.p.m * few_pitch(g.p.k)), a);
}

template <typename T, bool VEC> int launch_few(tb_ctx* ctx, const FewArgs& g) {
    return g.p.m <= 8 ? launch_few_b<T, VEC, 1>(ctx, g) : launch_few_b<T, VEC, 2>(ctx, g);
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
                  const float* bias, int64_t act, void* y, int64_t y_type, int64_t y_stride) {
    if (m < 0 || n < 0 || k <= 0 || m > MAX_DIM || n > MAX_DIM) return fail(TB_ERR_INVALID, "int8 product: bad shape");
    if (k > INT8_MAX_K) return fail(TB_ERR_UNSUPPORTED, "int8 product: k over %lld can overflow the int32 sum", (long long)INT8_MAX_K);
    if (!act_supported(act)) return fail(TB_ERR_UNSUPPORTED, "int8 product: activation %lld not supported", (long long)act);
    if (!elem_type_ok(y_type)) return fail(TB_ERR_UNSUPPORTED, "int8 product: element type %lld", (long long)y_type);
    if (m == 0 || n == 0) return TB_OK;
    if (!w || !w_scales || !y) return fail(TB_ERR_INVALID, "int8 product: null pointer");
    if ((uintptr_t)y % elem_size(y_type)) return fail(TB_ERR_INVALID, "int8 product: misaligned output");
    if (!aligned_to(4, {w_scales, bias})) return fail(TB_ERR_INVALID, "int8 product: misaligned scales or bias");
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
    if (!aligned_to(4, {scales})) return fail(TB_ERR_INVALID, "quantize: misaligned scales");
    if (rows > 1 && code_stride < cols) return fail(TB_ERR_INVALID, "quantize: row stride below the row's length");
    return quantize_rows(ctx, rows, cols, x, x_type, x_stride, codes, code_stride, scales);
}

int tb_int8_gemm(tb_ctx* ctx, int64_t m, int64_t n, int64_t k, const int8_t* a, int64_t a_stride,
                 const float* a_scales, const int8_t* w, int64_t w_stride, const float* w_scales,
                 const float* bias, int64_t activation, void* y, int64_t y_type, int64_t y_stride) {
    TB_ENTER(ctx);
    int r = check_product(m, n, k, w, w_stride, w_scales, bias, activation, y, y_type, y_stride);
    if (r != TB_OK) return r;
    if (m == 0 || n == 0) return TB_OK;
    if (!a || !a_scales) return fail(TB_ERR_INVALID, "int8 product: null pointer");
    if (!aligned_to(4, {a_scales})) return fail(TB_ERR_INVALID, "int8 product: misaligned scales or bias");
    if (!aligned16(a) || a_stride % 16) return fail(TB_ERR_INVALID, "int8 product: a and its stride have to be multiples of 16 bytes");
    if (m > 1 && a_stride < k) return fail(TB_ERR_INVALID, "int8 product: row stride below the row's length");
    const Int8Args p{m, n, k, a, a_stride, a_scales, w, w_stride, w_scales, bias, (int)activation, y, y_stride};
    if (use_few(ctx, m, n, k)) return launch_few<int8_t, true>(ctx, FewArgs{p, nullptr, 0, (int)y_type, 0});
    return int8_gemm_tc(ctx, p, y_type, false, 0);
}

int tb_int8_connected_fwd(tb_ctx* ctx, int64_t m, int64_t n, int64_t k, const void* x, int64_t x_type,
                          int64_t x_stride, const int8_t* w, int64_t w_stride, const float* w_scales,
                          const float* bias, int64_t activation, void* y, int64_t y_type, int64_t y_stride) {
    TB_ENTER(ctx);
    int r = check_product(m, n, k, w, w_stride, w_scales, bias, activation, y, y_type, y_stride);
    if (r != TB_OK) return r;
    if ((r = check_quantize(m, k, x, x_type, x_stride)) != TB_OK) return r;
    if (m == 0 || n == 0) return TB_OK;
    Int8Args p{m, n, k, nullptr, 0, nullptr, w, w_stride, w_scales, bias, (int)activation, y, y_stride};
    if (use_few(ctx, m, n, k)) {
        const FewArgs g{p, x, x_stride, (int)y_type, 0};
        return elem_dispatch(x_type, [&](auto t) {
            using T = decltype(t);
            return aligned16(x) && (m == 1 || x_stride % Vec<T>::N == 0) ? launch_few<T, true>(ctx, g) : launch_few<T, false>(ctx, g);
        });
    }
    const int64_t stride = round_up(k, 16), scale_bytes = round_up(m * 4, 256), code_bytes = round_up(m * stride, 256);
    const size_t scratch = (size_t)(scale_bytes + code_bytes);
    if ((r = ensure_workspace(ctx, scratch + int8_gemm_scratch(ctx, m))) != TB_OK) return r;
    float* scales = static_cast<float*>(ctx->ws);
    int8_t* codes = reinterpret_cast<int8_t*>(scales) + scale_bytes;
    if ((r = quantize_rows(ctx, m, k, x, x_type, x_stride, codes, stride, scales)) != TB_OK) return r;
    p.a = codes;
    p.a_stride = stride;
    p.a_scales = scales;
    return int8_gemm_tc(ctx, p, y_type, true, scratch);
}

}  // extern "C"

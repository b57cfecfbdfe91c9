// logprobs.cu -- what a program reads off vocabulary-sized logits: the log probability of a given
// token, the entropy, the most probable tokens (tb_token_logprobs_fwd), and the gradient of the
// first two (tb_token_logprobs_bwd).
#include "elem.cuh"

#include <algorithm>
#include <cstring>
#include <type_traits>

namespace tbi {
namespace {

constexpr int TOP_MAX = 32;

struct Part;

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
    int steps;             // most steps of a part
    int splits;            // parts of a row, joined by the last of their CTAs to finish
    Part* parts;
    int* counters;         // finished parts of each row, left at 0
};

__device__ __forceinline__ float nan_f() { return __uint_as_float(0x7fffffffu); }

__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t u = __float_as_uint(v + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u); }

// Order of alternatives as one unsigned key: the value's order in the high half (-0 counts as 0), then
// the lower column first. 0 is below every key.
__device__ __forceinline__ unsigned long long top_key(float v, uint32_t col) {
    return ((unsigned long long)ordered(v) << 32) | (uint32_t)~col;
}
__device__ __forceinline__ uint32_t key_col(unsigned long long k) { return ~(uint32_t)k; }
__device__ __forceinline__ float key_val(unsigned long long k) { return unordered((uint32_t)(k >> 32)); }

// ---- arithmetic on two floats at a time ---------------------------------------------------------
struct F2 {
    float x, y;
};
__device__ __forceinline__ unsigned long long f2_bits(F2 a) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
    return r;
}
__device__ __forceinline__ F2 f2_of(unsigned long long b) {
    F2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(b));
    return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
    return f2_of(r);
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
    return f2_of(r);
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)), "l"(f2_bits(c)));
    return f2_of(r);
}
// 2^x to about 2^-22; 0 below 2^-126
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// Exponents are clamped here: 2^-200 is 0 in single precision, and -infinity (a mask) and the NaN of
// (-infinity) - (-infinity) become a finite number whose product with 0 is 0.
constexpr float EXP_FLOOR = -200.f;

// ---- 16 bytes of logits -----------------------------------------------------------------------
template <typename T> struct Chunk;
template <> struct Chunk<float> {
    static constexpr uint32_t MASKED = 0xff800000u;  // -infinity
    static constexpr float LOWEST = -0x1.fffffep127f;  // the type's lowest finite value
    // the largest logit of n chunks, NaN if one is
    template <int N> static __device__ __forceinline__ float vmax(const uint4 (&r)[N]) {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < N; ++i)
            m = max_nan(m, max_nan(max_nan(__uint_as_float(r[i].x), __uint_as_float(r[i].y)), max_nan(__uint_as_float(r[i].z), __uint_as_float(r[i].w))));
        return m;
    }
    // bit e: logit e is at least v
    static __device__ __forceinline__ uint32_t at_least(const uint4& r, float v) {
        return (__uint_as_float(r.x) >= v ? 1u : 0u) | (__uint_as_float(r.y) >= v ? 2u : 0u) | (__uint_as_float(r.z) >= v ? 4u : 0u) |
               (__uint_as_float(r.w) >= v ? 8u : 0u);
    }
    static __device__ __forceinline__ void get(const uint4& r, F2* f) {
        f[0] = {__uint_as_float(r.x), __uint_as_float(r.y)};
        f[1] = {__uint_as_float(r.z), __uint_as_float(r.w)};
    }
    static __device__ __forceinline__ uint4 put(const F2* f) {
        return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
    }
};
template <> struct Chunk<__nv_bfloat16> {
    static constexpr uint32_t MASKED = 0xff80ff80u;
    static constexpr float LOWEST = -0x1.fep127f;
    template <int N> static __device__ __forceinline__ float vmax(const uint4 (&r)[N]) {
        auto h = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
        __nv_bfloat162 m[N];
#pragma unroll
        for (int i = 0; i < N; ++i) m[i] = __hmax2_nan(__hmax2_nan(h(r[i].x), h(r[i].y)), __hmax2_nan(h(r[i].z), h(r[i].w)));
#pragma unroll
        for (int i = 1; i < N; ++i) m[0] = __hmax2_nan(m[0], m[i]);
        return max_nan(__low2float(m[0]), __high2float(m[0]));
    }
    static __device__ __forceinline__ uint32_t at_least(const uint4& r, float v) {
        const __nv_bfloat162 l = __float2bfloat162_rn(v);  // exact: v is a logit of this type
        auto ge = [&](uint32_t w) { return __hge2_mask(*reinterpret_cast<const __nv_bfloat162*>(&w), l); };
        const uint32_t m = (ge(r.x) & 0x00020001u) | (ge(r.y) & 0x00080004u) | (ge(r.z) & 0x00200010u) | (ge(r.w) & 0x00800040u);
        return (m | m >> 16) & 0xffu;
    }
    static __device__ __forceinline__ F2 two(uint32_t w) { return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)}; }
    static __device__ __forceinline__ void get(const uint4& r, F2* f) { f[0] = two(r.x), f[1] = two(r.y), f[2] = two(r.z), f[3] = two(r.w); }
    static __device__ __forceinline__ uint32_t one(F2 a) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a.x, a.y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ uint4 put(const F2* f) { return make_uint4(one(f[0]), one(f[1]), one(f[2]), one(f[3])); }
};
template <> struct Chunk<__half> {
    static constexpr uint32_t MASKED = 0xfc00fc00u;
    static constexpr float LOWEST = -65504.f;
    template <int N> static __device__ __forceinline__ float vmax(const uint4 (&r)[N]) {
        auto h = [](uint32_t w) { return *reinterpret_cast<const __half2*>(&w); };
        __half2 m[N];
#pragma unroll
        for (int i = 0; i < N; ++i) m[i] = __hmax2_nan(__hmax2_nan(h(r[i].x), h(r[i].y)), __hmax2_nan(h(r[i].z), h(r[i].w)));
#pragma unroll
        for (int i = 1; i < N; ++i) m[0] = __hmax2_nan(m[0], m[i]);
        return max_nan(__low2float(m[0]), __high2float(m[0]));
    }
    static __device__ __forceinline__ uint32_t at_least(const uint4& r, float v) {
        const __half2 l = __float2half2_rn(v);  // exact: v is a logit of this type
        auto ge = [&](uint32_t w) { return __hge2_mask(*reinterpret_cast<const __half2*>(&w), l); };
        const uint32_t m = (ge(r.x) & 0x00020001u) | (ge(r.y) & 0x00080004u) | (ge(r.z) & 0x00200010u) | (ge(r.w) & 0x00800040u);
        return (m | m >> 16) & 0xffu;
    }
    static __device__ __forceinline__ F2 two(uint32_t w) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        return {f.x, f.y};
    }
    static __device__ __forceinline__ void get(const uint4& r, F2* f) { f[0] = two(r.x), f[1] = two(r.y), f[2] = two(r.z), f[3] = two(r.w); }
    static __device__ __forceinline__ uint32_t one(F2 a) {
        const __half2 h = __floats2half2_rn(a.x, a.y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ uint4 put(const F2* f) { return make_uint4(one(f[0]), one(f[1]), one(f[2]), one(f[3])); }
};

// A row as 16-byte chunks from the 16-byte boundary at or before its start: chunk v holds columns
// v * E - head .. Whole chunks are one access; the first and last, where the row covers them in part, go element
// by element, with -infinity in the other places. Nothing outside the row is touched.
template <typename T> struct Row {
    static constexpr int E = 16 / sizeof(T);
    const T* base;  // of chunk 0, before the row's start by `head` elements
    int head, end;  // the row's columns are elements head .. end - 1 of the chunks
    __device__ __forceinline__ Row(const T* x, int64_t vocab) {
        head = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
        base = reinterpret_cast<const T*>(reinterpret_cast<uintptr_t>(x) & ~(uintptr_t)15);
        end = head + (int)vocab;
    }
    __device__ __forceinline__ int chunks() const { return (int)(((int64_t)end + E - 1) / E); }
    __device__ __forceinline__ bool whole(int v) const { return v >= (head ? 1 : 0) && v < end / E; }
    __device__ __forceinline__ uint4 load(int v, int stop) const {
        if (v < stop && whole(v)) return *reinterpret_cast<const uint4*>(base + (int64_t)v * E);
        uint4 r = make_uint4(Chunk<T>::MASKED, Chunk<T>::MASKED, Chunk<T>::MASKED, Chunk<T>::MASKED);
        if (v < stop) {
            T t[E];
            memcpy(t, &r, 16);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int64_t i = (int64_t)v * E + e;
                if (i >= head && i < end) t[e] = base[i];
            }
            memcpy(&r, t, 16);
        }
        return r;
    }
    // Chunks v0 + u * apart + at, u < N, of a step that begins at chunk v0 (the same for all its threads) and
    // spans N * apart of them; false for a step at the row's edge, where some are masked.
    template <int N> __device__ __forceinline__ bool step(uint4 (&r)[N], int v0, int at, int apart, int stop) const {
        const int whole_end = min(stop, end / E), next = v0 + N * apart;
        const uint4* q = reinterpret_cast<const uint4*>(base) + v0 + at;
        if ((v0 > 0 || head == 0) && next <= whole_end) {
#pragma unroll
            for (int u = 0; u < N; ++u) r[u] = q[u * apart];
            return true;
        }
        if ((v0 > 0 || head == 0) && whole_end == stop) {  // every chunk whole or outside
#pragma unroll
            for (int u = 0; u < N; ++u) {
                r[u] = make_uint4(Chunk<T>::MASKED, Chunk<T>::MASKED, Chunk<T>::MASKED, Chunk<T>::MASKED);
                if (v0 + u * apart + at < stop) r[u] = q[u * apart];
            }
        } else {
#pragma unroll
            for (int u = 0; u < N; ++u) r[u] = load(v0 + u * apart + at, stop);
        }
        return false;
    }
};

// ---- the most probable tokens -------------------------------------------------------------------
// A warp keeps its best keys sorted, the i-th best in lane i (0: none yet).
// 32 values, one a lane, into descending order
template <typename K> __device__ __forceinline__ K sort32(K a, int lane) {
#pragma unroll
    for (int n = 2; n <= 32; n *= 2)
#pragma unroll
        for (int o = n / 2; o; o /= 2) {
            const K b = __shfl_xor_sync(0xffffffffu, a, o);
            const bool up = ((lane & n) == 0) == ((lane & o) == 0);  // this lane keeps the larger one
            a = up == (a > b) ? a : b;
        }
    return a;
}
// The k-th largest of 32 values, or a smaller one where some are equal: a bound that at least k reach.
__device__ __forceinline__ uint32_t kth32(uint32_t a, int k, int lane) {
    if (k > 8) return __shfl_sync(0xffffffffu, sort32(a, lane), k - 1);
    uint32_t m = 0;
    for (int i = 0; i < k; ++i) {
        m = __reduce_max_sync(0xffffffffu, a);
        if (a == m) a = 0;
    }
    return m;
}
// the 32 largest of two descending lists, descending
template <typename K> __device__ __forceinline__ K merge32(K a, K b, int lane) {
    b = __shfl_xor_sync(0xffffffffu, b, 31);
    a = a > b ? a : b;
#pragma unroll
    for (int o = 16; o; o /= 2) {
        b = __shfl_xor_sync(0xffffffffu, a, o);
        a = ((lane & o) == 0) == (a > b) ? a : b;
    }
    return a;
}
// the lists of all warps of the CTA into warp 0's (every thread calls it)
template <int NW, typename K> __device__ __forceinline__ K merge_warps(K a, K (*buf)[32], int warp, int lane) {
#pragma unroll
    for (int n = NW / 2; n; n /= 2) {
        if (warp >= n && warp < 2 * n) buf[warp][lane] = a;
        __syncthreads();
        if (warp < n) a = merge32(a, buf[warp + n][lane], lane);
    }
    return a;
}
// one key for the whole warp into a list of `top`
__device__ __forceinline__ unsigned long long insert(unsigned long long list, unsigned long long key, int lane) {
    const int at = __popc(__ballot_sync(0xffffffffu, list > key));
    const unsigned long long up = __shfl_up_sync(0xffffffffu, list, 1);
    return lane < at ? list : lane == at ? key : up;
}

// ---- forward --------------------------------------------------------------------------------------
// Sums of a part of a row: sum 2^t and sum t 2^t over t = (logit - max) * c, c = log2(e) / temperature.
struct Sums {
    float max, z, s;
    int bad;  // a NaN or +infinity is among the logits
};
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b, float c) {
    Sums r;
    r.max = fmaxf(a.max, b.max);
    const float da = fmaxf(__fmul_rn(__fsub_rn(a.max, r.max), c), EXP_FLOOR), db = fmaxf(__fmul_rn(__fsub_rn(b.max, r.max), c), EXP_FLOOR);
    const float fa = exp2_fast(da), fb = exp2_fast(db);
    r.z = fmaf(a.z, fa, __fmul_rn(b.z, fb));
    r.s = fmaf(fmaf(a.z, da, a.s), fa, __fmul_rn(fmaf(b.z, db, b.s), fb));
    r.bad = a.bad | b.bad;
    return r;
}
__device__ __forceinline__ Sums join_warp(Sums a, float c) {
    const float max = unordered(__reduce_max_sync(0xffffffffu, ordered(a.max)));
    const float d = fmaxf(__fmul_rn(__fsub_rn(a.max, max), c), EXP_FLOOR), f = exp2_fast(d);
    a.s = __fmul_rn(fmaf(a.z, d, a.s), f);
    a.z = __fmul_rn(a.z, f);
    a.max = max;
    a.bad = __any_sync(0xffffffffu, a.bad);
#pragma unroll
    for (int o = 16; o; o /= 2) {
        a.z = __fadd_rn(a.z, __shfl_xor_sync(0xffffffffu, a.z, o));
        a.s = __fadd_rn(a.s, __shfl_xor_sync(0xffffffffu, a.s, o));
    }
    return a;
}

// What a split of a row leaves in the workspace for the one that joins them.
struct Part {
    Sums sums;
    unsigned long long keys[TOP_MAX];
};

// A row's given token and its logit, read before the pass so that the row's end does not wait for them.
struct Given {
    int64_t token = -1;
    float logit = 0.f;
    template <typename T> __device__ __forceinline__ void read(const LogprobArgs& p, int64_t row, const T* x) {
        if (!p.logprob) return;
        token = p.tokens[row];
        if (token >= 0 && token < p.vocab) logit = Elem<T>::get(x[token]);
    }
};

// A row's results from its sums.
struct RowLog {
    Sums a;
    bool empty;
    float inv_t, logz;
    __device__ __forceinline__ RowLog(const LogprobArgs& p, const Sums& s) : a(s), empty(s.max == -INFINITY), inv_t(p.inv_t), logz(logf(s.z)) {}
    __device__ __forceinline__ float of(float v) const {
        return a.bad ? nan_f() : empty ? -INFINITY : __fsub_rn(__fmul_rn(__fsub_rn(v, a.max), inv_t), logz);
    }
    // by one thread
    __device__ __forceinline__ void write(const LogprobArgs& p, int64_t row, const Given& given) const {
        if (p.logprob)
            p.logprob[row] = given.token >= p.vocab ? nan_f() : given.token < 0 ? (a.bad ? nan_f() : 0.f) : of(given.logit);
        if (p.entropy)
            p.entropy[row] = a.bad ? nan_f() : empty ? 0.f : fmaxf(__fsub_rn(logz, __fmul_rn(__fdiv_rn(a.s, a.z), LN2)), 0.f);
        if (p.lse) p.lse[row] = a.bad ? nan_f() : empty ? -INFINITY : __fadd_rn(__fmul_rn(a.max, inv_t), logz);
        if (p.row_max) p.row_max[row] = a.bad ? nan_f() : a.max;
        if (p.log_sum) p.log_sum[row] = a.bad ? nan_f() : empty ? 0.f : logz;
    }
    __device__ __forceinline__ void write_top(const LogprobArgs& p, int64_t row, int i, unsigned long long key) const {
        p.top_token[row * p.top + i] = a.bad ? -1 : (int64_t)key_col(key);
        p.top_logprob[row * p.top + i] = of(key_val(key));
    }
};

// Results of one row, by one warp that holds its sums and its best keys.
__device__ __forceinline__ void write_row(const LogprobArgs& p, int64_t row, const Sums& a, unsigned long long list, const Given& given, int lane) {
    const RowLog log(p, a);
    if (lane == 0) log.write(p, row, given);
    if (p.top == 0) return;
    const int have = min(__popc(__ballot_sync(0xffffffffu, list != 0)), p.top);
    if (have < p.top) {
        // Fewer columns than alternatives are not masked, and all of those are in the list: the lowest
        // masked columns follow. They are among the first 64, of which the list holds at most 31.
        bool in0 = lane >= p.vocab, in1 = lane + 32 >= p.vocab;
        for (int i = 0; i < have; ++i) {
            const uint32_t col = key_col(__shfl_sync(0xffffffffu, list, i));
            in0 |= col == (uint32_t)lane;
            in1 |= col == (uint32_t)lane + 32;
        }
        unsigned long long left = __ballot_sync(0xffffffffu, !in0) | (unsigned long long)__ballot_sync(0xffffffffu, !in1) << 32;
        for (int i = have; i < lane; ++i) left &= left - 1;  // the (lane - have)-th of them
        if (lane >= have) list = top_key(-INFINITY, (uint32_t)(__ffsll((long long)left) - 1));
    }
    if (lane < p.top) log.write_top(p, row, lane, list);
}

// The sums of one thread, against the largest of its logits so far: that one's term is 2^0 = 1 exactly, so the sum of
// exponentials is never below 1, and no t 2^t is larger than the entropy's own terms. (A reference that may lag the maximum saves
// most of the raises, but the sum of t 2^t is then a difference of larger numbers: with a lag of up to 2^40 the entropy of
// rows sure of their token was off by 6e-7 (rms) instead of 1e-7, and some of their log probabilities were above 0.)
struct Running {
    float max = -INFINITY;
    F2 z = {0.f, 0.f}, s = {0.f, 0.f};
    int bad = 0;
    // before logits up to m (NaN: one of them is) are added
    __device__ __forceinline__ void raise(float m, float c) {
        if (!(m <= max)) {
            bad |= !(m < INFINITY);
            const float d = fmaxf(__fmul_rn(__fsub_rn(max, m), c), EXP_FLOOR), f = exp2_fast(d);
            s = {__fmul_rn(fmaf(z.x, d, s.x), f), __fmul_rn(fmaf(z.y, d, s.y), f)};
            z = {__fmul_rn(z.x, f), __fmul_rn(z.y, f)};
            max = fmaxf(max, m);
        }
    }
    // CLAMP: masked logits may be among them; t is kept at EXP_FLOOR there, where 2^t is 0
    template <typename T, bool CLAMP> __device__ __forceinline__ void add(const uint4& raw, float c) {
        constexpr int E = 16 / sizeof(T);
        F2 f[E / 2];
        Chunk<T>::get(raw, f);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
            F2 t = mul2(add2(f[e], {-max, -max}), {c, c});
            if (CLAMP) t = {fmaxf(t.x, EXP_FLOOR), fmaxf(t.y, EXP_FLOOR)};
            const F2 q = {exp2_fast(t.x), exp2_fast(t.y)};
            z = add2(z, q);
            s = fma2(q, t, s);
        }
    }
    // A step's chunks, by all lanes of a warp; the first `n` of them are not empty for all. The clamp costs a fifth
    // of the arithmetic and only masks need it: the row's edge has some, and elsewhere a masked logit
    // makes s NaN (0 * -infinity), and the step is then taken again, and the warp's later ones, with it.
    template <typename T, int N> __device__ __forceinline__ void step(const uint4 (&raw)[N], int n, float c, bool edge, bool& clamp) {
        if (!clamp && !edge) {
            const F2 z0 = z, s0 = s;
#pragma unroll
            for (int u = 0; u < N; ++u) add<T, false>(raw[u], c);
            const float t = __fadd_rn(s.x, s.y);
            clamp = __any_sync(0xffffffffu, t != t);
            if (!clamp) return;
            z = z0, s = s0;
        }
#pragma unroll
        for (int u = 0; u < N; ++u)
            if (u < n) add<T, true>(raw[u], c);
    }
    __device__ __forceinline__ Sums sums() const { return {max, __fadd_rn(z.x, z.y), __fadd_rn(s.x, s.y), bad}; }
};

// The largest float below the value of a bound's key, so that `logit > limit_of(bound)` lets in equal logits
// at lower columns; -infinity for no bound.
__device__ __forceinline__ float limit_of(unsigned long long bound) {
    const uint32_t o = (uint32_t)(bound >> 32);
    return !bound ? -INFINITY : unordered(o == 0x80000000u ? 0x7ffffffeu : o - 1);  // below 0 comes -0
}

// Into a warp's list: the keys (0: none) of 32 lanes that are above the bound.
__device__ __forceinline__ void take(unsigned long long& list, unsigned long long& bound, unsigned long long key, int top, int lane) {
    unsigned some = __ballot_sync(0xffffffffu, key > bound);
    if (__popc(some) > 6) {  // six insertions cost what a sort of the 32 does
        list = merge32(list, sort32(key > bound ? key : 0ull, lane), lane);
        some = 0;
    }
    while (some) {
        const unsigned long long k = __shfl_sync(0xffffffffu, key, __ffs((int)some) - 1);
        some &= some - 1;
        list = insert(list, k, lane);
    }
    const unsigned long long k = __shfl_sync(0xffffffffu, list, top - 1);
    bound = k > bound ? k : bound;
}

// One pass over the logits. NW warps to a row, or to one of `splits` parts of it; where a warp has a row to itself, four to a
// CTA. Each step of a thread is a group of U chunks; the groups' maxima stay in shared memory, so that after the
// pass only the groups that can hold one of the best are read again: those whose maximum reaches the k-th largest of
// the threads' maxima, about k of them. Lists kept during the pass took 530 us for 4096 x 131072 bf16 top 20, this 194
// (5.5 TB/s), and 168 (6.4 TB/s) without alternatives; what is left of the difference is the chain at a row's end,
// which the other CTAs of an SM cover in part. Few rows in parts: 1 x 131072 top 20 in 7.8 us, the latency of two rounds to memory
// and of joining the parts. (Times in this file: of the kernel, in a graph of calls on inputs larger than L2 together.)
constexpr int LP_U = 4;
// Most steps of a part: a CTA's groups fit its shared memory, and longer rows are faster on more warps (4096 x 131072 bf16 top
// 20: 194 us on 4, 217 on 2, 201 on 8).
template <typename T> int lp_steps(int nw) { return nw < 8 ? 40 : sizeof(T) == 4 ? 28 : 32; }

constexpr int KEYS = 64;  // candidates that are ranked against one another

template <int NW> struct RowShared {
    unsigned long long keys[NW][32];
    uint32_t maxima[NW][32];
    Sums sums[NW];
    unsigned long long found[KEYS], ranked[32];
    unsigned long long bound;
    int queued, nfound, last;
};

template <int NW> __device__ __forceinline__ void row_sync() {
    if constexpr (NW == 1) __syncwarp();
    else __syncthreads();
}

template <typename T, int NW, bool AHEAD>
__global__ void __launch_bounds__(NW == 1 ? 128 : NW * 32, NW == 1 ? (AHEAD ? 6 : 8) : (AHEAD ? 24 : 32) / NW) k_token_logprobs(const LogprobArgs p) {
    TB_GRID_DEP_ENTRY();
    constexpr int E = 16 / sizeof(T), U = LP_U, NT = NW * 32, ROWS = NW == 1 ? 4 : 1;
    __shared__ RowShared<NW> shared[ROWS];
    extern __shared__ __align__(16) unsigned char dyn[];  // with top > 0: each row's group maxima, then its queue of groups
    RowShared<NW>& sh = shared[NW == 1 ? threadIdx.x >> 5 : 0];
    T (*const group_max)[NT] = reinterpret_cast<T (*)[NT]>(dyn + (NW == 1 ? threadIdx.x >> 5 : 0) * p.steps * NT * (sizeof(T) + 2));
    uint16_t* const queue = reinterpret_cast<uint16_t*>(group_max + p.steps);

    const int lane = threadIdx.x & 31, warp = NW == 1 ? 0 : threadIdx.x >> 5, tid = warp * 32 + lane;
    const int64_t unit = NW == 1 ? (int64_t)blockIdx.x * ROWS + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
    const int64_t row = NW == 1 ? unit : unit / p.splits;
    if (NW == 1 && row >= p.rows) return;
    const int split = NW == 1 ? 0 : (int)(unit - row * p.splits);
    const T* x = static_cast<const T*>(p.logits) + row * p.stride;
    const Row<T> r(x, p.vocab);
    const int chunks = r.chunks(), per = NW == 1 ? chunks : (int)(((int64_t)chunks + p.splits - 1) / p.splits);
    const int begin = (int)min((int64_t)chunks, (int64_t)split * per), stop = min(chunks, begin + per);
    const float c = __fmul_rn(LOG2E, p.inv_t);

    Given given;
    if (warp == 0) given.read(p, row, x);
    if (tid == 0) sh.queued = sh.nfound = 0;

    Running a;
    int steps = 0;
    bool clamp = false;
    uint4 raw[U];
    [[maybe_unused]] uint4 next[U];
    [[maybe_unused]] bool next_whole = false;
    if (AHEAD) next_whole = r.step(next, begin, tid, NT, stop);
    for (int v0 = begin; v0 < stop; v0 += NT * U, ++steps) {
        bool whole;
        if constexpr (AHEAD) {  // the next step's loads run under this step's sums
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = next[u];
            whole = next_whole;
            if (v0 + NT * U < stop) next_whole = r.step(next, v0 + NT * U, tid, NT, stop);
        } else {
            whole = r.step(raw, v0, tid, NT, stop);
        }
        const float m = Chunk<T>::vmax(raw);
        if (p.top) group_max[steps][tid] = Elem<T>::put(m);  // exact: m is one of the logits
        a.raise(m, c);
        a.template step<T>(raw, (stop - v0 + NT - 1) / NT, c, !whole, clamp);
    }
    Sums w = join_warp(a.sums(), c);
    unsigned long long list = 0;
    if (NW > 1 && lane == 0) sh.sums[warp] = w;
    if (p.top) {
        uint32_t o = ordered(a.max);
        if constexpr (NW > 1) {
            o = sort32(o, lane);
            o = merge_warps<NW>(o, sh.maxima, warp, lane);
            if (warp == 0) {
                o = __shfl_sync(0xffffffffu, o, p.top - 1);
                if (lane == 0) sh.bound = unordered(o) > -INFINITY ? (unsigned long long)o << 32 : 0;
            }
        } else {
            o = kth32(o, p.top, lane);
            if (lane == 0) sh.bound = unordered(o) > -INFINITY ? (unsigned long long)o << 32 : 0;
        }
        row_sync<NW>();
        unsigned long long bound = sh.bound;
        const float limit = limit_of(bound);
        auto queue_groups = [&] {
            for (int i = 0; i < steps; ++i)
                if (Elem<T>::get(group_max[i][tid]) > limit) queue[atomicAdd(&sh.queued, 1)] = (uint16_t)(i * NT + tid);
            row_sync<NW>();
            return sh.queued;
        };
        // the groups q, q + NW, .. < q + 4 NW of the queue, an element a lane, four loads at once; every lane takes part
        // in f, also those past a group's U * E
        static_assert(U * E <= 32, "a group is read by one warp at a time");
        auto read_groups = [&](int n, auto f) {
            for (int q = warp; q < n; q += 4 * NW) {
                float l[4];
                int at[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int g = queue[min(q + j * NW, n - 1)];
                    const int v = begin + (g / NT) * NT * U + (lane / E) * NT + g % NT;
                    at[j] = v * E + lane % E;
                    const bool in = q + j * NW < n && lane < U * E && v < stop && at[j] >= r.head && at[j] < r.end;
                    l[j] = in ? Elem<T>::get(r.base[at[j]]) : -INFINITY;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (q + j * NW < n) f(l[j] > limit ? top_key(l[j], (uint32_t)(at[j] - r.head)) : 0ull);
            }
        };
        auto found = [&](unsigned long long key) {
            const int i = atomicAdd(&sh.nfound, 1);
            if (i < KEYS) sh.found[i] = key;
        };
        int groups = -1;
        if (steps == 1 && bound) {  // the logits are still in registers
            const float v = key_val(bound);
            if (a.max >= v) {
                uint32_t some = 0;  // bit u * E + e
#pragma unroll
                for (int u = 0; u < U; ++u) some |= Chunk<T>::at_least(raw[u], v) << u * E;
                while (some) {
                    const int i = __ffs((int)some) - 1;
                    some &= some - 1;
                    const int at = (begin + (i / E) * NT + tid) * E + i % E;
                    found(top_key(Elem<T>::get(r.base[at]), (uint32_t)(at - r.head)));
                }
            }
        } else {
            groups = queue_groups();
            read_groups(groups, [&](unsigned long long key) {
                if (key) found(key);
            });
        }
        row_sync<NW>();
        const int n = sh.nfound;
        if (n <= KEYS) {
            // few: each is placed by the number of larger ones
            if (warp == 0) {
                const unsigned long long k0 = lane < n ? sh.found[lane] : 0, k1 = lane + 32 < n ? sh.found[lane + 32] : 0;
                int r0 = 0, r1 = 0;
                for (int i = 0; i < n; ++i) {
                    const unsigned long long k = sh.found[i];
                    r0 += k > k0;
                    r1 += k > k1;
                }
                if (lane < n && r0 < 32) sh.ranked[r0] = k0;
                if (lane + 32 < n && r1 < 32) sh.ranked[r1] = k1;
                __syncwarp();
                list = lane < min(n, p.top) ? sh.ranked[lane] : 0;
            }
        } else {
            // many equal logits, or few distinct ones: through the warps' sorted lists
            if (groups < 0) groups = queue_groups();
            read_groups(groups, [&](unsigned long long key) { take(list, bound, key, p.top, lane); });
            if (lane >= p.top) list = 0;
            if constexpr (NW > 1) list = merge_warps<NW>(list, sh.keys, warp, lane);
        }
    } else {
        row_sync<NW>();
    }
    if constexpr (NW > 1) {
        if (warp == 0) w = join_warp(lane < NW ? sh.sums[lane] : Sums{-INFINITY, 0.f, 0.f, 0}, c);
        if (p.splits > 1) {
            Part* part = p.parts + row * p.splits;
            if (warp == 0) {
                if (lane == 0) part[split].sums = w;
                part[split].keys[lane] = list;
                __threadfence();
                __syncwarp();
                if (lane == 0) {
                    sh.last = atomicAdd(&p.counters[row], 1) == p.splits - 1;
                    if (sh.last) p.counters[row] = 0;  // ready for the next launch
                }
            }
            __syncthreads();
            if (!sh.last) return;
            __threadfence();
            w = {-INFINITY, 0.f, 0.f, 0};
            list = 0;
            for (int i = warp; i < p.splits; i += NW) {
                w = join(w, {__ldcg(&part[i].sums.max), __ldcg(&part[i].sums.z), __ldcg(&part[i].sums.s), __ldcg(&part[i].sums.bad)}, c);
                if (p.top) list = merge32(list, __ldcg(&part[i].keys[lane]), lane);
            }
            if (lane == 0) sh.sums[warp] = w;
            __syncthreads();
            if (p.top) list = merge_warps<NW>(list, sh.keys, warp, lane);
            if (warp == 0) w = join_warp(lane < NW ? sh.sums[lane] : Sums{-INFINITY, 0.f, 0.f, 0}, c);
        }
    }
    if (warp == 0) write_row(p, row, w, list, given, lane);
}

// ---- forward, short rows ----------------------------------------------------------------------------
// L lanes to a row of up to SHORT_U chunks a lane and up to SHORT_TOP alternatives, all of it in registers: 32 / L rows share a
// warp's instructions for what comes after the logits (joining the sums, ranking, logarithms), which are most of
// a short row's work and bound it: 16384 x 1000 f16 in 14.9 us with top 5 (2.2 TB/s), 10.0 without.
constexpr int SHORT_U = 8, SHORT_TOP = 8, SHORT_KEYS = 32;

template <int L, typename V, typename F> __device__ __forceinline__ V group_reduce(V v, F f) {
#pragma unroll
    for (int o = L / 2; o; o /= 2) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

template <typename T, int L> __global__ void __launch_bounds__(128, 7) k_token_logprobs_short(const LogprobArgs p) {
    TB_GRID_DEP_ENTRY();
    constexpr int E = 16 / sizeof(T), U = SHORT_U, G = 32 / L;
    __shared__ unsigned long long found[4][G][SHORT_KEYS];
    __shared__ int nfound[4][G];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gl = lane % L, group = lane / L;
    const int64_t mine = ((int64_t)blockIdx.x * 4 + warp) * G + group, row = min(mine, p.rows - 1);  // every lane stays for the shuffles
    const bool active = mine < p.rows;
    const T* x = static_cast<const T*>(p.logits) + row * p.stride;
    const Row<T> r(x, p.vocab);
    const int stop = r.chunks();
    const float c = __fmul_rn(LOG2E, p.inv_t);

    uint4 raw[U];
    if (__all_sync(0xffffffffu, r.head == 0 && r.end % E == 0)) {
        const uint4* q = reinterpret_cast<const uint4*>(r.base) + gl;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            raw[u] = make_uint4(Chunk<T>::MASKED, Chunk<T>::MASKED, Chunk<T>::MASKED, Chunk<T>::MASKED);
            if (u * L + gl < stop) raw[u] = q[u * L];
        }
    } else {
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = r.load(u * L + gl, stop);
    }
    Given given;
    if (gl == 0) given.read(p, row, x);
    if (gl == 0) nfound[warp][group] = 0;

    const float own = Chunk<T>::vmax(raw);  // NaN if one of the lane's is
    Running a;
    const float most = group_reduce<L>(own, max_nan);
    a.bad = !(most < INFINITY);
    a.max = a.bad ? 0.f : most;
    bool clamp = __any_sync(0xffffffffu, most == -INFINITY);
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u * L + gl >= stop) continue;
            if (clamp) a.add<T, true>(raw[u], c);
            else a.add<T, false>(raw[u], c);
        }
        if (clamp) break;
        const float t = __fadd_rn(a.s.x, a.s.y);
        clamp = __any_sync(0xffffffffu, t != t);  // masked logits: again, with the clamp
        if (!clamp) break;
        a.z = a.s = {0.f, 0.f};
    }
    const auto add = [](float v, float w) { return __fadd_rn(v, w); };
    const Sums w = {most, group_reduce<L>(__fadd_rn(a.z.x, a.z.y), add), group_reduce<L>(__fadd_rn(a.s.x, a.s.y), add), a.bad};
    const RowLog log(p, w);
    if (gl == 0 && active) log.write(p, row, given);
    if (p.top == 0) return;

    // the k-th largest of the lanes' maxima bounds the k-th best from below
    uint32_t best = ordered(own), bound = 0;
    for (int i = 0; i < p.top; ++i) {
        bound = group_reduce<L>(best, [](uint32_t v, uint32_t w) { return max(v, w); });
        if (best == bound) best = 0;
    }
    const float least = bound > ordered(-INFINITY) && !a.bad ? unordered(bound) : Chunk<T>::LOWEST;
    uint32_t some[2] = {0, 0};  // bit u * E + e
#pragma unroll
    for (int u = 0; u < U; ++u) some[u * E / 32] |= Chunk<T>::at_least(raw[u], least) << u * E % 32;
    const int n = group_reduce<L>(__popc(some[0]) + __popc(some[1]), [](int v, int w) { return v + w; });
    unsigned long long* keys = found[warp][group];
    __syncwarp();
    if (n <= SHORT_KEYS) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            while (some[h]) {
                const int i = __ffs((int)some[h]) - 1 + 32 * h;
                some[h] &= some[h] - 1;
                const int at = (i / E * L + gl) * E + i % E;
                keys[atomicAdd(&nfound[warp][group], 1)] = top_key(Elem<T>::get(r.base[at]), (uint32_t)(at - r.head));
            }
    }
    __syncwarp();
    if (n <= SHORT_KEYS) {
        for (int i = gl; i < n; i += L) {
            const unsigned long long k = keys[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += keys[j] > k;
            if (rank < p.top && active) log.write_top(p, row, rank, k);
        }
        if (n < p.top && gl == 0 && active) {  // fewer columns than alternatives are not masked: the lowest masked ones follow
            uint32_t col = 0;
            for (int i = n; i < p.top; ++i, ++col) {
                for (int j = 0; j < n; ++j)
                    if (key_col(keys[j]) == col) ++col, j = -1;
                log.write_top(p, row, i, top_key(-INFINITY, col));
            }
        }
    }
    // many equal logits: the next best by another pass, for all the warp's rows or none
    const bool many = n > SHORT_KEYS;
    if (__any_sync(0xffffffffu, many)) {
        unsigned long long last = ~0ull;
        for (int i = 0; i < p.top; ++i) {
            unsigned long long k = 0;
            if (many)
                for (int64_t j = gl; j < p.vocab; j += L) {
                    const unsigned long long t = top_key(Elem<T>::get(x[j]), (uint32_t)j);
                    if (t < last && t > k) k = t;
                }
            last = group_reduce<L>(k, [](unsigned long long v, unsigned long long w) { return v > w ? v : w; });
            if (many && gl == 0 && active) log.write_top(p, row, i, last);
        }
    }
}

template <typename T> int launch_logprobs(tb_ctx* ctx, LogprobArgs p) {
    constexpr int E = 16 / sizeof(T);
    // 16-byte chunks that a row touches at most
    const bool aligned = aligned16(p.logits) && (p.rows == 1 || p.stride % E == 0);
    const int64_t chunks = ceil_div(p.vocab + (aligned ? 0 : E - 1), E);
    const int64_t step = 32 * LP_U;                   // chunks a step of one warp
    // Warps per row: the fewest (a row's end keeps few of them busy) that put 20 warps on every SM and leave a part
    // within lp_steps() steps. Measured with 1 / 2 / 4 / 8 warps, us: 8192 x 2048 bf16 top 5 16.6 / 22.1 / 35 / 65, 4096 x 32000 60 / 59 / 62 /
    // 82, 1000 x 16000 16.2 / 16.2 / 12.9 / 15.8, 777 x 30001 f32 - / 27.0 / 20.7 / 24.4.
    // Short rows share warps where they fill the GPU that way, or need no alternatives (else a warp to a row has the shorter
    // chain, and finds more of them): 16384 x 1000 f16 top 5 in 14.9 us and 20.5 with a warp each, 16384 x 80 7.0 and
    // 17.3, 60000 x 10 14.4 and 64; 200 x 200 4.6 and 4.0.
    const int lanes = chunks <= 4 * SHORT_U && p.top <= 4 ? 4 : chunks <= 8 * SHORT_U ? 8 : chunks <= 16 * SHORT_U ? 16 : 32;
    if (chunks <= lanes * SHORT_U && p.top <= SHORT_TOP && (p.top == 0 || p.rows * lanes / 32 >= 8 * ctx->sm_count)) {
        auto run = [&](auto n) {
            return launch_early(ctx, "k_token_logprobs_short", k_token_logprobs_short<T, decltype(n)::value>, dim3((unsigned)ceil_div(p.rows, 128 / lanes)),
                                dim3(128), 0, p);
        };
        switch (lanes) {
        case 4: return run(std::integral_constant<int, 4>());
        case 8: return run(std::integral_constant<int, 8>());
        case 16: return run(std::integral_constant<int, 16>());
        default: return run(std::integral_constant<int, 32>());
        }
    }
    int nw = 1;
    while (nw < 8 && chunks > step * nw && (p.rows * nw < 20 * ctx->sm_count || chunks > step * nw * lp_steps<T>(nw))) nw *= 2;
    // With 8, few rows go in parts: of one step while all of them have an SM each, else of two steps at least and two CTAs
    // to an SM at most (1 x 131072 bf16 top 20 7.7 us in 16 parts, 8.1 in 8; 48 x 50001 f32 top 5 10.4 in 6, 11.4 in 12). Joining them
    // costs what up to 6 steps take (8 x 32000 bf16 top 5 6.3 whole, 7.4 in 4 parts; 5 x 60000 8.5 whole, 7.4 in 8).
    const int64_t steps = ceil_div(chunks, step * nw), sms = ctx->sm_count;
    int64_t splits = 1;
    if (nw == 8) {
        if (steps > 6) splits = p.rows * steps <= sms ? steps : std::min(ceil_div(steps, 2), 2 * sms / p.rows);
        splits = std::max<int64_t>({1, std::min<int64_t>(splits, 256), ceil_div(steps, lp_steps<T>(nw))});
    }
    p.splits = (int)splits;
    // From 3 steps on the next step's loads are taken under this one's sums (777 x 50001 f32 31 -> 28 us), with 24 warps to an SM
    // instead of 32: not where that makes a second wave (4096 x 32000 with a warp a row 59 -> 67 us).
    const int64_t warps = p.rows * splits * nw;
    const bool ahead = ceil_div(steps, splits) >= 3 && (warps <= 24 * sms || warps > 32 * sms);
    p.steps = (int)ceil_div(steps, p.splits);
    if (p.rows * p.splits > 2147483647) return fail(TB_ERR_UNSUPPORTED, "token logprobs: too many rows");
    if (p.splits > 1) {
        // partial results and counters (the context's own, always left at 0, are too few for many long rows)
        const size_t parts = (size_t)(p.rows * p.splits) * sizeof(Part);
        const bool own = p.rows > ctx->tile_cnt_len;
        const int r = ensure_workspace(ctx, parts + (own ? p.rows * sizeof(int) : 0));
        if (r != TB_OK) return r;
        p.parts = static_cast<Part*>(ctx->ws);
        p.counters = ctx->tile_cnt;
        if (own) {
            p.counters = reinterpret_cast<int*>(static_cast<char*>(ctx->ws) + parts);
            TB_CHECK_CUDA(cudaMemsetAsync(p.counters, 0, p.rows * sizeof(int), ctx->stream));
        }
    }
    const size_t smem = p.top ? (size_t)(nw == 1 ? 4 : nw) * 32 * p.steps * (sizeof(T) + 2) : 0;
    const dim3 grid((unsigned)(nw == 1 ? ceil_div(p.rows, 4) : p.rows * p.splits)), block((unsigned)(nw == 1 ? 128 : nw * 32));
    auto run = [&](auto n, auto a) {
        return launch_early(ctx, "k_token_logprobs", k_token_logprobs<T, decltype(n)::value, decltype(a)::value>, grid, block, smem, p);
    };
    auto pick = [&](auto n) { return ahead ? run(n, std::true_type()) : run(n, std::false_type()); };
    switch (nw) {
    case 1: return pick(std::integral_constant<int, 1>());
    case 2: return pick(std::integral_constant<int, 2>());
    case 4: return pick(std::integral_constant<int, 4>());
    default: return pick(std::integral_constant<int, 8>());
    }
}

// ---- gradient ---------------------------------------------------------------------------------------
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
    int64_t parts;  // CTAs per row
};

// d = (a (delta - p) - b p (log p + h)) / T, log p = (l - max) / T - log_sum. Memory bound: 4096 x 131072 bf16 in
// 308 us (7.0 TB/s); a copy of as many bytes takes 333, in a second of copies. A CTA takes 4 x 256 chunks of a row, or (WARP) each
// of its warps a row of up to 4 x 32. In place is safe: a thread writes the chunks that it has read.
template <typename T, bool WARP> __global__ void __launch_bounds__(256) k_token_logprobs_bwd(const LogprobBwdArgs p) {
    TB_GRID_DEP_ENTRY();
    constexpr int E = 16 / sizeof(T), U = 4, NT = WARP ? 32 : 256;
    const int64_t row = WARP ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : (int64_t)blockIdx.x / p.parts;
    if (row >= p.rows) return;
    const int part = WARP ? 0 : (int)((int64_t)blockIdx.x - row * p.parts);
    const int tid = WARP ? threadIdx.x & 31 : threadIdx.x;
    const T* x = static_cast<const T*>(p.logits) + row * p.stride;
    T* d = static_cast<T*>(p.dlogits) + row * p.d_stride;
    const Row<T> r(x, p.vocab);
    const int stop = r.chunks(), v0 = part * NT * U + tid;
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = r.load(v0 + u * NT, stop);

    const float m = p.row_max[row], logz = p.log_sum[row];
    const int64_t tok = p.g_logprob && p.tokens ? p.tokens[row] : -1;
    const float a = tok >= 0 ? p.g_logprob[row] : 0.f, b = p.g_entropy ? p.g_entropy[row] : 0.f;
    const float h = p.g_entropy ? p.entropy[row] : 0.f;
    const bool empty = m == -INFINITY, bad = logz != logz || tok >= p.vocab;
    const float at = __fmul_rn(a, p.inv_t), bt = __fmul_rn(b, p.inv_t), ct = __fmul_rn(fmaf(b, h, a), p.inv_t);
    // log p in bits: t = (l - max) c - log2 of the sum; d = -2^t (b ln 2 / T t + (a + b h) / T) + delta a / T
    const float c = __fmul_rn(LOG2E, p.inv_t), bits = __fmul_rn(-LOG2E, logz), bl = __fmul_rn(-LN2, bt);
    const F2 nm = {-m, -m}, cc = {c, c}, nz = {bits, bits}, b2 = {bl, bl}, c2 = {-ct, -ct};
    const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int v = v0 + u * NT;
        if (v >= stop) continue;
        F2 f[E / 2];
        Chunk<T>::get(raw[u], f);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
            F2 t = fma2(add2(f[e], nm), cc, nz);
            t = {fmaxf(t.x, EXP_FLOOR), fmaxf(t.y, EXP_FLOOR)};
            f[e] = mul2({exp2_fast(t.x), exp2_fast(t.y)}, fma2(b2, t, c2));
        }
        const int64_t i0 = (int64_t)v * E - r.head;
        if (tok >= i0 && tok < i0 + E) {
#pragma unroll
            for (int e = 0; e < E / 2; ++e) {
                if (tok == i0 + 2 * e) f[e].x = __fadd_rn(f[e].x, at);
                if (tok == i0 + 2 * e + 1) f[e].y = __fadd_rn(f[e].y, at);
            }
        }
        if (empty || bad) {
            const float fill = bad ? nan_f() : 0.f;
#pragma unroll
            for (int e = 0; e < E / 2; ++e) f[e] = {fill, fill};
        }
        const uint4 out = Chunk<T>::put(f);
        if (same && r.whole(v)) {
            *reinterpret_cast<uint4*>(d + i0) = out;
        } else {
            T t[E];
            memcpy(t, &out, 16);
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (i0 + e >= 0 && i0 + e < p.vocab) d[i0 + e] = t[e];
        }
    }
}

template <typename T> int launch_bwd(tb_ctx* ctx, LogprobBwdArgs p) {
    constexpr int E = 16 / sizeof(T);
    const bool aligned = aligned16(p.logits) && (p.rows == 1 || p.stride % E == 0);
    const int64_t chunks = ceil_div(p.vocab + (aligned ? 0 : E - 1), E);
    if (chunks <= 32 * 4)
        return launch_early(ctx, "k_token_logprobs_bwd", k_token_logprobs_bwd<T, true>, dim3((unsigned)ceil_div(p.rows, 8)), dim3(256), 0, p);
    p.parts = ceil_div(chunks, 256 * 4);
    if (p.rows * p.parts > 2147483647) return fail(TB_ERR_UNSUPPORTED, "token logprobs: more than 2^31 parts of rows");
    return launch_early(ctx, "k_token_logprobs_bwd", k_token_logprobs_bwd<T, false>, dim3((unsigned)(p.rows * p.parts)), dim3(256), 0, p);
}

int check_logits(int64_t rows, int64_t vocab, const void* logits, int64_t type, int64_t stride, float temperature) {
    if (rows < 0 || vocab <= 0 || rows > 2147483647 || vocab > 2147483000) return fail(TB_ERR_INVALID, "token logprobs: bad shape");
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
    if (!aligned_to(4, {logprob, entropy, lse, row_max, log_sum, top_logprob}) || !aligned_to(8, {tokens, top_token}))
        return fail(TB_ERR_INVALID, "token logprobs: misaligned pointer");
    LogprobArgs p{rows, vocab, logits, stride, tokens, 1.f / temperature, (int)top, tokens ? logprob : nullptr, entropy, lse, row_max, log_sum, top_logprob, top_token, 0, 1, nullptr, nullptr};
    return elem_dispatch(type, [&](auto t) { return launch_logprobs<decltype(t)>(ctx, p); });
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
    if ((uintptr_t)dlogits % elem_size(type) || !aligned_to(4, {row_max, log_sum, entropy, g_logprob, g_entropy}) || !aligned_to(8, {tokens}))
        return fail(TB_ERR_INVALID, "token logprobs: misaligned pointer");
    if (dlogits == logits && rows > 1 && d_stride != stride) return fail(TB_ERR_INVALID, "token logprobs: in place with another row stride");
    const LogprobBwdArgs p{rows, vocab, logits, stride, tokens, 1.f / temperature, row_max, log_sum, entropy, g_logprob, g_entropy, dlogits, d_stride, 1};
    return elem_dispatch(type, [&](auto t) { return launch_bwd<decltype(t)>(ctx, p); });
}

}  // extern "C"

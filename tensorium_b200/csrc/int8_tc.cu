// int8_tc.cu -- the int8 product on the tensor cores (tcgen05.mma kind::i8, int32 sums in TMEM).
//
// Output channels are the MMA's M and tokens its N: a weight tile is 128 (a CTA pair: 256) channels x
// 128 bytes of k, and the token tile can be as narrow as the batch is, down to 16, so a decoding
// batch streams each weight byte through the tensor core once without padding the work to 128
// tokens. TMEM lane = channel: a thread keeps one channel's scale and bias in registers and a
// warp's 32 lanes write 32 consecutive channels of a token. Both operands arrive by TMA as K-major
// 128-byte swizzled rows; TMA fills zeros past k, m and n, so no size needs padding. int32 sums are
// exact in any order, which is what lets k be split freely.
//
// k_int8_stream: one CTA per SM on tiles of 128 channels x up to 128 tokens. One SM takes weights at 58 GB/s at most, with 5 as
// with 10 stages in flight, and 148 of them at 43 GB/s each, which is the HBM's rate (32 x n x 16384, whole tiles, weights larger than L2 in
// turn: 40 to 42 us for 18, 37 and 74 tiles, 43 for 111, 53 for 148). So a few long tiles are shared out by k, to
// 128 bytes evenly: the CTAs of a tile leave int32 sums in the workspace, and the last of them to finish adds them.
// k_int8_pair: persistent CTA pairs (cta_group::2) on 256 x 256 tiles with two accumulators in
// TMEM, so the epilogue of one tile runs under the products of the next.
//
// Every wait is bounded; on a timeout the kernel sets the context's status word, lets copies in
// flight land, frees TMEM and returns.
#include "conv_tc.cuh"
#include "int8.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cstring>
#include <mutex>

namespace tbi {
namespace {

constexpr int I8_BK = 128;             // bytes of k per stage: one swizzled row
constexpr int I8_W_BYTES = 128 * I8_BK;  // weight tile of a stage and CTA

struct I8Maps {
    CUtensorMap w;  // (k, channel), box 128 x 128
    CUtensorMap a;  // (k, token), box 128 x the CTA's share of the token tile
};

// instruction descriptor: S32 accumulate, S8 A and B, both K-major, M x N
__host__ __device__ constexpr uint32_t idesc_i8(int M, int N) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// K-major, 128-byte swizzle: rows of 128 bytes along k, 8-row groups 1024 bytes apart
__device__ __forceinline__ uint64_t desc_k_sw128(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}

template <int CTAS>
__device__ __forceinline__ void mma_i8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CTAS == 1)
        asm volatile(
            "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
            "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate));
    else
        asm volatile(
            "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
            "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate));
}

// waits for the kernel before this one (and its writes) when launched with programmatic serialization
__device__ __forceinline__ void grid_dep_wait() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }

// What a thread of the epilogue keeps of its channel.
template <typename T> struct Channel {
    bool in;
    float scale, bias;
    T* y;
    __device__ Channel(const Int8Args& p, int64_t ch) : in(ch < p.n) {
        scale = in ? __ldg(p.w_scales + ch) : 0.f;
        bias = in && p.bias ? __ldg(p.bias + ch) : 0.f;
        y = static_cast<T*>(p.y) + ch;
    }
    // N consecutive tokens from `token`: every value first, then every store, so that the chains of
    // one thread overlap (an epilogue warp has a scheduler almost to itself)
    template <int N> __device__ __forceinline__ void store(const Int8Args& p, int64_t token, const float* a_scales, const int* acc) const {
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __fmul_rn(__int2float_rn(acc[i]), __fmul_rn(a_scales[i], scale));
        if (p.bias) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = __fadd_rn(v[i], bias);
        }
        if (p.act != TB_ACT_LINEAR) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = tb_activate_dev(v[i], p.act);
        }
        T* to = y + token * p.y_stride;
        const int64_t left = in ? p.m - token : 0;
        if (left >= N) {
#pragma unroll
            for (int i = 0; i < N; ++i) to[i * p.y_stride] = Elem<T>::put(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < left) to[i * p.y_stride] = Elem<T>::put(v[i]);
        }
    }
};

// ---- one CTA on 128 channels x up to 128 tokens -----------------------------------------------------
constexpr int I8S_MAX_STAGES = 12, I8S_THREADS = 320;
constexpr int I8S_SMEM = 216 * 1024;

struct StreamArgs {
    int bt;        // tokens of a tile: a multiple of 16 up to 128
    int stages;
    int tiles_m, tiles, ktiles;
    bool share;    // the tiles are shared out by units of 128 bytes of k, else they are taken whole
    int* partial;  // [2 x CTA][bt / 4][128 channels][4 tokens]
    int* counters; // per shared tile: CTAs that have left their sums, left at 0
};

// A CTA's work in order: its range of the shared tiles' units, or every gridDim.x-th whole tile.
struct StreamWork {
    bool share;
    int at, end, step, ktiles;  // unit and end of the range, or tile and number of tiles
    int tile, kb, ke;           // the current piece
    __device__ StreamWork(const StreamArgs& a) : share(a.share), at(blockIdx.x), end(a.tiles), step(gridDim.x), ktiles(a.ktiles) {
        if (share) {
            const int64_t units = (int64_t)a.tiles * a.ktiles;
            at = (int)(units * blockIdx.x / gridDim.x);
            end = (int)(units * (blockIdx.x + 1) / gridDim.x);
        }
    }
    __device__ __forceinline__ bool take() {
        if (at >= end) return false;
        if (share) {
            tile = at / ktiles;
            kb = at - tile * ktiles;
            ke = min(ktiles, kb + end - at);
            at += ke - kb;
        } else {
            tile = at, kb = 0, ke = ktiles;
            at += step;
        }
        return true;
    }
};

template <typename T>
__global__ void __launch_bounds__(I8S_THREADS, 1) k_int8_stream(const __grid_constant__ I8Maps maps, const Int8Args p, const StreamArgs g,
                                                                 int* status) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const unsigned sbase = ((unsigned)__cvta_generic_to_shared(smem_raw) + 1023u) & ~1023u;
    __shared__ __align__(8) uint64_t full_bar[I8S_MAX_STAGES], empty_bar[I8S_MAX_STAGES], tfull_bar[2], tempty_bar[2], drain_bar;
    __shared__ uint32_t tmem_base;
    __shared__ volatile int abort_flag;
    __shared__ int last;
    __shared__ __align__(16) float a_scales[2][128];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int bt = g.bt, stages = g.stages;
    const int stage_bytes = I8_W_BYTES + bt * I8_BK;

    int pre = 0;
    if (tid == 0) {
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(&maps.w)) : "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(&maps.a)) : "memory");
        for (int s = 0; s < stages; ++s) {
            tc::mbar_init(&full_bar[s], 1);
            tc::mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            tc::mbar_init(&tfull_bar[b], 1);
            tc::mbar_init(&tempty_bar[b], 8);  // one arrival per epilogue warp
        }
        tc::mbar_init(&drain_bar, 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        // the first stages' weights at once: they do not depend on the kernel before
        for (StreamWork w(g); pre < stages && w.take();)
            for (int kt = w.kb; kt < w.ke && pre < stages; ++kt, ++pre) {
                tc::mbar_arrive_expect_tx(&full_bar[pre], stage_bytes);
                tc::tma_load_2d(sbase + pre * stage_bytes, &maps.w, &full_bar[pre], kt * I8_BK, w.tile / g.tiles_m * 128);
            }
    }
    if (warp == 1) tc::tmem_alloc(&tmem_base, 256);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem0 = tmem_base;

    if (warp == 0) {
        if (lane == 0) {
            grid_dep_wait();
            int it = 0, st = 0, ph = 1;  // ph: parity of the stage's last release
            bool ok = true;
            for (StreamWork w(g); ok && w.take();) {
                const int w_row = w.tile / g.tiles_m * 128, a_row = w.tile % g.tiles_m * bt;
                for (int kt = w.kb; kt < w.ke; ++kt, ++it) {
                    const unsigned sw = sbase + st * stage_bytes;
                    if (it >= pre) {
                        if (!tc::mbar_wait_bounded(&empty_bar[st], ph, &abort_flag, status, 931)) {
                            ok = false;
                            break;
                        }
                        tc::mbar_arrive_expect_tx(&full_bar[st], stage_bytes);
                        tc::tma_load_2d(sw, &maps.w, &full_bar[st], kt * I8_BK, w_row);
                    }
                    tc::tma_load_2d(sw + I8_W_BYTES, &maps.a, &full_bar[st], kt * I8_BK, a_row);
                    if (++st == stages) st = 0, ph ^= 1;
                }
            }
            // the copies land before the CTA ends, after an abort too: the last use of every stage
            for (int i = max(0, it - stages); i < it; ++i) tc::mbar_wait_limit(&full_bar[i % stages], (i / stages) & 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = idesc_i8(128, bt);
            int st = 0, ph = 0, n = 0;
            bool ok = true, issued = false;
            for (StreamWork w(g); ok && w.take(); ++n) {
                const int buf = n & 1, u = n >> 1;
                if (u > 0 && !tc::mbar_wait_bounded(&tempty_bar[buf], (u - 1) & 1, &abort_flag, status, 932)) break;
                tc::tc_fence_after();
                const uint32_t d = tmem0 + buf * 128;
                for (int kt = w.kb; kt < w.ke; ++kt) {
                    if (!tc::mbar_wait_bounded(&full_bar[st], ph, &abort_flag, status, 933)) {
                        ok = false;
                        break;
                    }
                    tc::tc_fence_after();
                    const unsigned sw = sbase + st * stage_bytes;
#pragma unroll
                    for (int kk = 0; kk < I8_BK / 32; ++kk)
                        mma_i8<1>(d, desc_k_sw128(sw + kk * 32), desc_k_sw128(sw + I8_W_BYTES + kk * 32), idesc, (kt > w.kb || kk) ? 1u : 0u);
                    issued = true;
                    tc::mma_commit(&empty_bar[st]);
                    if (++st == stages) st = 0, ph ^= 1;
                }
                if (ok) tc::mma_commit(&tfull_bar[buf]);
            }
            if (issued) {  // every MMA has finished before TMEM is freed
                tc::mma_commit(&drain_bar);
                tc::mbar_wait_limit(&drain_bar, 0);
            }
        }
        __syncwarp();
    } else {
        grid_dep_wait();  // a_scales
        const int quarter = warp & 3, half = (warp - 2) >> 2, ch = quarter * 32 + lane, et = tid - 64;
        const int64_t units = (int64_t)g.tiles * g.ktiles;
        int n = 0;
        for (StreamWork w(g); w.take(); ++n) {
            const int buf = n & 1, u = n >> 1;
            const int64_t m0 = (int64_t)(w.tile % g.tiles_m) * bt;
            if (et < bt) a_scales[buf][et] = m0 + et < p.m ? p.a_scales[m0 + et] : 0.f;
            const Channel<T> c(p, (int64_t)(w.tile / g.tiles_m) * 128 + ch);
            const bool ok = !abort_flag && tc::mbar_wait_bounded(&tfull_bar[buf], u & 1, &abort_flag, status, 934);
            if (tc::epi_any(!ok)) break;  // tcgen05.ld is warp-collective: the epilogue warps leave together
            tc::tc_fence_after();
            const uint32_t taddr = tmem0 + buf * 128 + ((uint32_t)(quarter * 32) << 16);
            const bool whole = w.kb == 0 && w.ke == g.ktiles;
            // this CTA's sums of a shared tile: slot 0 where its piece begins inside the tile, 1 where it ends there
            int4* slot = reinterpret_cast<int4*>(g.partial) + (int64_t)(2 * blockIdx.x + (w.kb == 0)) * bt * 32 + ch;
#pragma unroll 1
            for (int c0 = half * 16; c0 < bt; c0 += 32) {
                uint32_t r[16];
                tc::tmem_ld16_issue(taddr + c0, r);
                tc::tmem_wait16(r);
                if (whole) {
                    c.template store<16>(p, m0 + c0, a_scales[buf] + c0, reinterpret_cast<int*>(r));
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        __stcg(slot + (c0 / 4 + i) * 128, make_int4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]));
                }
            }
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&tempty_bar[buf]);
            if (whole) continue;
            // the last of the tile's CTAs to get here adds their sums (int32: the same in any order)
            const int64_t u0 = (int64_t)w.tile * g.ktiles;
            const int first = (int)(((u0 + 1) * gridDim.x - 1) / units), end = (int)(((u0 + g.ktiles) * gridDim.x - 1) / units) + 1;
            __threadfence();
            tc::epi_sync();
            if (et == 0) {
                last = atomicAdd(&g.counters[w.tile], 1) == end - first - 1;
                if (last) g.counters[w.tile] = 0;  // ready for the next launch
            }
            tc::epi_sync();
            if (!last) continue;
            __threadfence();
#pragma unroll 1
            for (int c0 = half * 16; c0 < bt; c0 += 32) {
                int r[16] = {};
#pragma unroll 2
                for (int j = first; j < end; ++j) {
                    const int4* q = reinterpret_cast<const int4*>(g.partial) + (int64_t)(2 * j + (j == first)) * bt * 32 + ch;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int4 v = __ldcg(q + (c0 / 4 + i) * 128);
                        r[4 * i] += v.x, r[4 * i + 1] += v.y, r[4 * i + 2] += v.z, r[4 * i + 3] += v.w;
                    }
                }
                c.template store<16>(p, m0 + c0, a_scales[buf] + c0, r);
            }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 1) tc::tmem_dealloc(tmem0, 256);
}

// ---- CTA pairs ----------------------------------------------------------------------------------
constexpr int I8P_STAGES = 6, I8P_STAGE_BYTES = 2 * I8_W_BYTES, I8P_THREADS = 320;
constexpr int I8P_SMEM = I8P_STAGES * I8P_STAGE_BYTES + 1024;
constexpr int I8P_GROUP = 8;  // token tiles that are walked together through all channels (L2 reuse)

__device__ __forceinline__ void i8p_tile(int64_t t, int64_t tiles_m, int64_t tiles_n, int64_t* mt, int64_t* nt) {
    const int64_t per = (int64_t)I8P_GROUP * tiles_n, g = t / per, r = t - g * per;
    const int64_t rows = min((int64_t)I8P_GROUP, tiles_m - g * I8P_GROUP);
    *nt = r / rows;
    *mt = g * I8P_GROUP + (r - *nt * rows);
}

template <typename T>
__global__ void __launch_bounds__(I8P_THREADS, 1) k_int8_pair(const __grid_constant__ I8Maps maps, const Int8Args p, int* status) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const unsigned sbase = ((unsigned)__cvta_generic_to_shared(smem_raw) + 1023u) & ~1023u;
    __shared__ __align__(8) uint64_t full_bar[I8P_STAGES], empty_bar[I8P_STAGES], tfull_bar[2], tempty_bar[2], drain_bar;
    __shared__ uint32_t tmem_base;
    __shared__ volatile int abort_flag;
    __shared__ __align__(16) float a_scales[8][128];  // each epilogue warp's tokens

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)tc::cluster_rank();
    const int64_t first = blockIdx.x / 2, step = gridDim.x / 2;
    const int64_t tiles_m = (p.m + 255) / 256, tiles_n = (p.n + 255) / 256, tiles = tiles_m * tiles_n;
    const int ktiles = (int)((p.k + I8_BK - 1) / I8_BK);

    if (tid == 0) {
        for (int s = 0; s < I8P_STAGES; ++s) {
            tc::mbar_init(&full_bar[s], 1);
            tc::mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            tc::mbar_init(&tfull_bar[b], 1);
            tc::mbar_init(&tempty_bar[b], 16);  // the epilogue warps of both CTAs
        }
        tc::mbar_init(&drain_bar, 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 1) tc::tmem_alloc_g<2>(&tmem_base, 512);
    tc::tc_fence_before();
    __syncthreads();
    tc::cluster_sync();  // the peer's barriers exist before anything signals them
    tc::tc_fence_after();
    const uint32_t tmem0 = tmem_base;

    if (warp == 0) {
        if (lane == 0) {
            grid_dep_wait();
            int it = 0;
            bool ok = true;
            for (int64_t t = first; ok && t < tiles; t += step) {
                int64_t mt, nt;
                i8p_tile(t, tiles_m, tiles_n, &mt, &nt);
                const int w_row = (int)(nt * 256) + rank * 128, a_row = (int)(mt * 256) + rank * 128;
                for (int kt = 0; kt < ktiles; ++kt, ++it) {
                    const int st = it % I8P_STAGES, use = it / I8P_STAGES;
                    if (use > 0 && !tc::mbar_wait_bounded(&empty_bar[st], (use - 1) & 1, &abort_flag, status, 941)) {
                        ok = false;
                        break;
                    }
                    if (rank == 0) tc::mbar_arrive_expect_tx(&full_bar[st], 2 * I8P_STAGE_BYTES);
                    const unsigned sw = sbase + st * I8P_STAGE_BYTES;
                    tc::tma_load_2d_g<2>(sw, &maps.w, &full_bar[st], kt * I8_BK, w_row);
                    tc::tma_load_2d_g<2>(sw + I8_W_BYTES, &maps.a, &full_bar[st], kt * I8_BK, a_row);
                }
            }
            // an abort: the copies of both CTAs land (they are counted on the even CTA) before either ends
            if (!ok && rank == 0)
                for (int j = it > I8P_STAGES ? it - I8P_STAGES : 0; j < it; ++j)
                    tc::mbar_wait_limit(&full_bar[j % I8P_STAGES], (j / I8P_STAGES) & 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            constexpr uint32_t idesc = idesc_i8(256, 256);
            int it = 0, tl = 0;
            bool ok = true, issued = false;
            for (int64_t t = first; ok && t < tiles; t += step, ++tl) {
                const int buf = tl & 1, u = tl >> 1;
                if (u > 0 && !tc::mbar_wait_bounded(&tempty_bar[buf], (u - 1) & 1, &abort_flag, status, 942)) break;
                tc::tc_fence_after();
                const uint32_t d = tmem0 + buf * 256;
                for (int kt = 0; kt < ktiles; ++kt, ++it) {
                    const int st = it % I8P_STAGES, use = it / I8P_STAGES;
                    if (!tc::mbar_wait_bounded(&full_bar[st], use & 1, &abort_flag, status, 943)) {
                        ok = false;
                        break;
                    }
                    tc::tc_fence_after();
                    const unsigned sw = sbase + st * I8P_STAGE_BYTES;
#pragma unroll
                    for (int kk = 0; kk < I8_BK / 32; ++kk)
                        mma_i8<2>(d, desc_k_sw128(sw + kk * 32), desc_k_sw128(sw + I8_W_BYTES + kk * 32), idesc, (kt || kk) ? 1u : 0u);
                    issued = true;
                    tc::mma_commit_g<2>(&empty_bar[st]);
                }
                if (ok) tc::mma_commit_g<2>(&tfull_bar[buf]);
            }
            if (issued) {  // every MMA has finished before TMEM is freed
                tc::mma_commit_g<2>(&drain_bar);
                tc::mbar_wait_limit(&drain_bar, 0);
            }
        }
        __syncwarp();
    } else {
        grid_dep_wait();  // a_scales
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        int tl = 0;
        for (int64_t t = first; t < tiles; t += step, ++tl) {
            int64_t mt, nt;
            i8p_tile(t, tiles_m, tiles_n, &mt, &nt);
            const int buf = tl & 1, u = tl >> 1;
            const int64_t m0 = mt * 256 + half * 128;
            float* sa = a_scales[warp - 2];
            __syncwarp();
            for (int i = lane; i < 128; i += 32) sa[i] = m0 + i < p.m ? p.a_scales[m0 + i] : 0.f;
            __syncwarp();
            const bool ok = !abort_flag && tc::mbar_wait_bounded(&tfull_bar[buf], u & 1, &abort_flag, status, 944);
            if (tc::epi_any(!ok)) break;  // tcgen05.ld is warp-collective: the epilogue warps leave together
            tc::tc_fence_after();
            const Channel<T> c(p, nt * 256 + rank * 128 + quarter * 32 + lane);
            const uint32_t taddr = tmem0 + buf * 256 + half * 128 + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
            for (int c0 = 0; c0 < 128; c0 += 16) {
                uint32_t r[16];
                tc::tmem_ld16_issue(taddr + c0, r);
                tc::tmem_wait16(r);
                c.template store<16>(p, m0 + c0, sa + c0, reinterpret_cast<int*>(r));
            }
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) {  // the accumulator is free: told to the CTA that issues the MMAs
                if (rank == 0) tc::mbar_arrive(&tempty_bar[buf]);
                else tc::mbar_arrive_cluster(&tempty_bar[buf], 0);
            }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::cluster_sync();  // neither CTA ends, or frees its TMEM, while the other's MMAs or signals use it
    tc::tc_fence_after();
    if (warp == 1) tc::tmem_dealloc_g<2>(tmem0, 512);
}

// ---- host side -------------------------------------------------------------------------------------
PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    });
    return fn;
}

// int8 rows of k bytes, box of 128 bytes x `box_rows`, 128-byte swizzle, zeros out of bounds. The
// copies start at multiples of 128 bytes of k.
int encode_rows(CUtensorMap* m, const int8_t* base, int64_t k, int64_t rows, int64_t stride, int box_rows) {
    auto enc = map_encoder();
    if (!enc) return fail(TB_ERR_CUDA, "int8 product: cuTensorMapEncodeTiled is not available");
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)(rows > 1 ? stride : round_up(k, 16))};
    const cuuint32_t box[2] = {I8_BK, (cuuint32_t)box_rows}, es[2] = {1, 1};
    CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(base), dims, strides, box, es,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(TB_ERR_CUDA, "int8 product: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return TB_OK;
}

// Launches KERNEL with a cluster and, after the quantizer, programmatic serialization. max_smem: the
// most dynamic shared memory that any launch of this kernel asks for.
template <auto KERNEL, typename... Args>
int launch_cluster(tb_ctx* ctx, const char* what, dim3 grid, int threads, int smem, int max_smem, dim3 cluster, bool early,
                   Args&&... args) {
    static std::atomic<bool> done[64];  // the attribute is set once per kernel and device
    if (ctx->device >= 64 || !done[ctx->device].load(std::memory_order_acquire)) {
        cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, max_smem);
        if (e != cudaSuccess) return cuda_fail(e, what);
        if (ctx->device < 64) done[ctx->device].store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (cluster.x * cluster.y * cluster.z > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster.x;
        attr[n].val.clusterDim.y = cluster.y;
        attr[n].val.clusterDim.z = cluster.z;
        ++n;
    }
    if (early) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = (unsigned)n;
    cudaError_t e = cudaLaunchKernelEx(&cfg, KERNEL, std::forward<Args>(args)...);
    if (e != cudaSuccess) return cuda_fail(e, what);
    return check_launch(what);
}

// Tokens of a shared tile: up to 128, in as many equal tiles as it takes.
int shared_tokens(int64_t m) { return (int)round_up(ceil_div(m, ceil_div(m, 128)), 16); }

// How a product is run: the fastest of three by what they were measured to take, us, for `ktiles` steps of 128 bytes
// of k. Whole tiles of one CTA, 4.5 + 0.34 a step and wave: an SM takes that for a step's 16 KB of weights whatever its tokens
// (0.28 where few SMs have a tile, 0.38 where all have); so the tokens go in as many tiles as one wave holds, which shortens the epilogues (128 x
// 4096 x 4096: 13.6 on tiles of 32 tokens, 14.6 of 128). One wave of tiles at most, shared out by k evenly over all SMs: 6 and
// 0.04 a token of the tile more, to leave and add the partial sums (32 x 4096 x 16384: 20 shared, 41 whole; 128 x
// 4096 x 4096: 18 shared). Tiles of CTA pairs, 7.5 + 0.36 a step and wave for four times the work (1000 x 4096 x
// 4096: 19, and 25 in whole tiles; 512 x 4096 x 4096: 18 and 16).
struct Plan {
    int bt;        // tokens of a tile of the single-CTA kernel, 0 for pairs
    bool share;
    int64_t grid;
};

Plan plan(const tb_ctx* ctx, int64_t m, int64_t n, int64_t k) {
    const int64_t sms = ctx->sm_count, ktiles = ceil_div(k, I8_BK), tiles_n = ceil_div(n, 128), least = ceil_div(m, 128);
    const int64_t most = std::max(least, std::min(ceil_div(m, 16), sms / tiles_n));
    const int bt = (int)round_up(ceil_div(m, most), 16), sk_bt = shared_tokens(m);
    const int64_t tiles = ceil_div(m, bt) * tiles_n, sk_tiles = least * tiles_n, sk_grid = std::min(sms, ceil_div(sk_tiles * ktiles, 4));
    const double whole = 4.5 + 0.34 * (double)(ktiles * ceil_div(tiles, sms));
    const bool can_share = sk_tiles < sms && sk_grid > sk_tiles;
    const double shared = can_share ? 10.5 + 0.04 * sk_bt + 0.34 * (double)(sk_tiles * ktiles) / (double)sk_grid : 1e30;
    const double pair = m > 128 ? 7.5 + 0.36 * (double)(ktiles * ceil_div(ceil_div(m, 256) * ceil_div(n, 256), sms / 2)) : 1e30;
    if (pair < whole && pair < shared) return {0, false, 0};
    if (tiles * ktiles >= ((int64_t)1 << 30)) return {0, false, 0};  // the single-CTA kernel counts in 32 bits
    return shared < whole ? Plan{sk_bt, true, sk_grid} : Plan{bt, false, std::min(tiles, sms)};
}

// `scratch`: where the workspace is free
int launch_stream(tb_ctx* ctx, const Int8Args& p, int64_t y_type, bool early, const Plan& plan, size_t scratch) {
    const int bt = plan.bt;
    const int64_t tiles_m = ceil_div(p.m, bt), tiles = tiles_m * ceil_div(p.n, 128);
    I8Maps maps;
    int r = encode_rows(&maps.w, p.w, p.k, p.n, p.w_stride, 128);
    if (r == TB_OK) r = encode_rows(&maps.a, p.a, p.k, p.m, p.a_stride, bt);
    if (r != TB_OK) return r;
    StreamArgs g = {};
    g.bt = bt;
    g.stages = (int)std::min<int64_t>(I8S_MAX_STAGES, (I8S_SMEM - 1024) / (I8_W_BYTES + bt * I8_BK));
    g.tiles_m = (int)tiles_m;
    g.tiles = (int)tiles;
    g.ktiles = (int)ceil_div(p.k, I8_BK);
    g.share = plan.share;
    if (g.share) {
        const size_t need = scratch + (size_t)plan.grid * 2 * bt * 128 * 4;
        if (need > ctx->ws_bytes && scratch) return fail(TB_ERR_STATE, "int8 product: workspace not reserved");
        if ((r = ensure_workspace(ctx, need)) != TB_OK) return r;
        g.partial = reinterpret_cast<int*>(static_cast<char*>(ctx->ws) + scratch);
        g.counters = ctx->tile_cnt;
    }
    const int smem = g.stages * (I8_W_BYTES + bt * I8_BK) + 1024;
    return elem_dispatch(y_type, [&](auto t) {
        return launch_cluster<k_int8_stream<decltype(t)>>(ctx, "k_int8_stream", dim3((unsigned)plan.grid), I8S_THREADS, smem, I8S_SMEM, dim3(1, 1, 1),
                                                          early, maps, p, g, ctx->d_status);
    });
}

int launch_pair(tb_ctx* ctx, const Int8Args& p, int64_t y_type, bool early) {
    I8Maps maps;
    int r = encode_rows(&maps.w, p.w, p.k, p.n, p.w_stride, 128);
    if (r == TB_OK) r = encode_rows(&maps.a, p.a, p.k, p.m, p.a_stride, 128);
    if (r != TB_OK) return r;
    const int64_t tiles = ceil_div(p.m, 256) * ceil_div(p.n, 256);
    const unsigned grid = (unsigned)(2 * std::min<int64_t>(tiles, ctx->sm_count / 2));
    return elem_dispatch(y_type, [&](auto t) {
        return launch_cluster<k_int8_pair<decltype(t)>>(ctx, "k_int8_pair", dim3(grid), I8P_THREADS, I8P_SMEM, I8P_SMEM, dim3(2, 1, 1),
                                                        early, maps, p, ctx->d_status);
    });
}

}  // namespace

size_t int8_gemm_scratch(const tb_ctx* ctx, int64_t m) { return (size_t)ctx->sm_count * 2 * shared_tokens(m) * 128 * 4; }

int int8_gemm_tc(tb_ctx* ctx, const Int8Args& p, int64_t y_type, bool early, size_t scratch) {
    const Plan pl = plan(ctx, p.m, p.n, p.k);
    return pl.bt ? launch_stream(ctx, p, y_type, early, pl, scratch) : launch_pair(ctx, p, y_type, early);
}

}  // namespace tbi

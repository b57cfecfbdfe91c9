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
// k_int8_stream: one tile per CTA; a cluster of CTAs along k shares a tile when the tiles alone do
// not fill the GPU, and sums its int32 partials through distributed shared memory, each CTA a part
// of the tokens.
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

__device__ __forceinline__ void st_cluster(unsigned local, unsigned rank, int v) {
    unsigned remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(remote) : "r"(local), "r"(rank));
    asm volatile("st.shared::cluster.s32 [%0], %1;\n" ::"r"(remote), "r"(v) : "memory");
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }
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

constexpr int I8_MAX_STAGES = 8;
constexpr int I8_STREAM_SMEM = 112 * 1024;  // two CTAs per SM

template <typename T, int BT>
__global__ void __launch_bounds__(192) k_int8_stream(const __grid_constant__ I8Maps maps, const Int8Args p, const int stages,
                                                     int* status) {
    constexpr int STAGE_BYTES = I8_W_BYTES + BT * I8_BK;
    constexpr int COLS = BT < 32 ? 32 : BT;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const unsigned sbase = ((unsigned)__cvta_generic_to_shared(smem_raw) + 1023u) & ~1023u;
    __shared__ __align__(8) uint64_t full_bar[I8_MAX_STAGES], empty_bar[I8_MAX_STAGES], done_bar;
    __shared__ uint32_t tmem_base;
    __shared__ volatile int abort_flag;
    __shared__ __align__(16) float a_scales[BT];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int splits = gridDim.z, z = blockIdx.z;
    const int64_t n0 = (int64_t)blockIdx.x * 128, m0 = (int64_t)blockIdx.y * BT;
    const int ktiles = (int)((p.k + I8_BK - 1) / I8_BK);
    const int kb = (int)((int64_t)ktiles * z / splits), ke = (int)((int64_t)ktiles * (z + 1) / splits);

    if (tid == 0) {
        for (int s = 0; s < stages; ++s) {
            tc::mbar_init(&full_bar[s], 1);
            tc::mbar_init(&empty_bar[s], 1);
        }
        tc::mbar_init(&done_bar, 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 1) tc::tmem_alloc(&tmem_base, COLS);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    if (splits > 1) cluster_arrive();  // waited for before the first remote store: every CTA has started
    const uint32_t tmem0 = tmem_base;

    if (warp == 0) {
        if (lane == 0) {
            // weights of the first stages before the tokens: they do not depend on the kernel before
            const int pre = min(stages, ke - kb);
            for (int j = 0; j < pre; ++j) {
                tc::mbar_arrive_expect_tx(&full_bar[j], STAGE_BYTES);
                tc::tma_load_2d(sbase + j * STAGE_BYTES, &maps.w, &full_bar[j], (kb + j) * I8_BK, (int)n0);
            }
            grid_dep_wait();
            int j = 0;
            for (; j < ke - kb; ++j) {
                const int st = j % stages, use = j / stages;
                const unsigned sw = sbase + st * STAGE_BYTES;
                if (use > 0) {
                    if (!tc::mbar_wait_bounded(&empty_bar[st], (use - 1) & 1, &abort_flag, status, 931)) break;
                    tc::mbar_arrive_expect_tx(&full_bar[st], STAGE_BYTES);
                    tc::tma_load_2d(sw, &maps.w, &full_bar[st], (kb + j) * I8_BK, (int)n0);
                }
                tc::tma_load_2d(sw + I8_W_BYTES, &maps.a, &full_bar[st], (kb + j) * I8_BK, (int)m0);
            }
            // the copies land before the CTA ends, after an abort too: the last use of every stage
            for (int i = max(0, j - stages); i < j; ++i) tc::mbar_wait_limit(&full_bar[i % stages], (i / stages) & 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            bool issued = false;
            for (int j = 0; j < ke - kb; ++j) {
                const int st = j % stages, use = j / stages;
                if (!tc::mbar_wait_bounded(&full_bar[st], use & 1, &abort_flag, status, 932)) break;
                tc::tc_fence_after();
                const unsigned sw = sbase + st * STAGE_BYTES;
#pragma unroll
                for (int kk = 0; kk < I8_BK / 32; ++kk)
                    mma_i8<1>(tmem0, desc_k_sw128(sw + kk * 32), desc_k_sw128(sw + I8_W_BYTES + kk * 32), idesc_i8(128, BT),
                              (j || kk) ? 1u : 0u);
                issued = true;
                tc::mma_commit(&empty_bar[st]);
            }
            if (issued) {  // also after an abort: no MMA runs on when TMEM is freed
                tc::mma_commit(&done_bar);
                tc::mbar_wait_limit(&done_bar, 0);
            }
        }
        __syncwarp();
    }
    const int quarter = warp & 3, ch = quarter * 32 + lane;
    const uint32_t taddr = tmem0 + ((uint32_t)(quarter * 32) << 16);
    bool ok = true;
    if (warp >= 2) {
        grid_dep_wait();
        for (int i = ch; i < BT; i += 128) a_scales[i] = m0 + i < p.m ? p.a_scales[m0 + i] : 0.f;
        asm volatile("bar.sync 1, 128;\n" ::: "memory");
        ok = tc::mbar_wait_bounded(&done_bar, 0, &abort_flag, status, 933);
        ok = __all_sync(0xffffffffu, ok && !abort_flag);
        tc::tc_fence_after();
    }
    if (splits == 1) {
        if (warp >= 2 && ok) {
            const Channel<T> c(p, n0 + ch);
#pragma unroll 1
            for (int c0 = 0; c0 < BT; c0 += 16) {
                uint32_t r[16];
                tc::tmem_ld16_issue(taddr + c0, r);
                tc::tmem_wait16(r);
                c.template store<16>(p, m0 + c0, a_scales + c0, reinterpret_cast<int*>(r));
            }
        }
    } else {
        // each CTA of the cluster sums its share of the tile's tokens: [source][token][channel] in its
        // own buffer behind the stages, filled by every CTA
        const int share = BT / splits;
        const unsigned red = sbase + stages * STAGE_BYTES;
        cluster_wait();
        if (warp >= 2 && ok) {
#pragma unroll 1
            for (int c0 = 0; c0 < BT; c0 += 16) {
                uint32_t r[16];
                tc::tmem_ld16_issue(taddr + c0, r);
                tc::tmem_wait16(r);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int c = c0 + i, to = c / share;
                    st_cluster(red + ((z * share + c - to * share) * 128 + ch) * 4, to, (int)r[i]);
                }
            }
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (warp >= 2 && ok) {
            const Channel<T> c(p, n0 + ch);
            const int* buf = reinterpret_cast<const int*>(smem_raw + (red - (unsigned)__cvta_generic_to_shared(smem_raw))) + ch;
            for (int i = 0; i < share; i += 2) {  // shares are powers of two from 2 on
                int acc[2] = {0, 0};
#pragma unroll 4
                for (int s = 0; s < splits; ++s)
                    for (int u = 0; u < 2; ++u) acc[u] += buf[(s * share + i + u) * 128];
                c.template store<2>(p, m0 + z * share + i, a_scales + z * share + i, acc);
            }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 1) tc::tmem_dealloc(tmem0, COLS);
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

template <int BT> int launch_stream(tb_ctx* ctx, const Int8Args& p, int64_t y_type, bool early, int splits) {
    constexpr int stage = I8_W_BYTES + BT * I8_BK;
    I8Maps maps;
    int r = encode_rows(&maps.w, p.w, p.k, p.n, p.w_stride, 128);
    if (r == TB_OK) r = encode_rows(&maps.a, p.a, p.k, p.m, p.a_stride, BT);
    if (r != TB_OK) return r;
    // two CTAs per SM, so that one's set-up and epilogue run under the other's products
    const int red = splits > 1 ? BT * 512 : 0;
    const int stages = std::min<int>(I8_MAX_STAGES, (I8_STREAM_SMEM - 1024 - red) / stage);
    const int smem = stages * stage + red + 1024;
    const dim3 grid((unsigned)ceil_div(p.n, 128), (unsigned)ceil_div(p.m, BT), (unsigned)splits);
    return elem_dispatch(y_type, [&](auto t) {
        return launch_cluster<k_int8_stream<decltype(t), BT>>(ctx, "k_int8_stream", grid, 192, smem, I8_STREAM_SMEM,
                                                              dim3(1, 1, (unsigned)splits), early, maps, p, stages, ctx->d_status);
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

int int8_gemm_tc(tb_ctx* ctx, const Int8Args& p, int64_t y_type, bool early) {
    const int64_t sms = ctx->sm_count;
    // pairs once their tiles occupy two thirds of the SMs
    if (p.m > 128 && ceil_div(p.m, 256) * ceil_div(p.n, 256) * 2 * 3 >= sms * 2) return launch_pair(ctx, p, y_type, early);
    const int bt = p.m <= 16 ? 16 : p.m <= 32 ? 32 : p.m <= 64 ? 64 : 128;
    if (ceil_div(p.m, bt) > 65535) return launch_pair(ctx, p, y_type, early);
    const int64_t tiles = ceil_div(p.n, 128) * ceil_div(p.m, bt), ktiles = ceil_div(p.k, I8_BK);
    // k in up to 8 parts while there are fewer CTAs than two per SM, parts of 4 stages at least
    int splits = 1;
    while (splits < 8 && splits * 2 <= bt && tiles * splits * 2 <= sms * 2 && ktiles >= splits * 2 * 4) splits *= 2;
    switch (bt) {
    case 16: return launch_stream<16>(ctx, p, y_type, early, splits);
    case 32: return launch_stream<32>(ctx, p, y_type, early, splits);
    case 64: return launch_stream<64>(ctx, p, y_type, early, splits);
    default: return launch_stream<128>(ctx, p, y_type, early, splits);
    }
}

}  // namespace tbi

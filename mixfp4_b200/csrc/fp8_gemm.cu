// Product of E4M3 operands with an fp32 scale per block of 128 along K (rows of x: one per row, weight: one per 128 x 128):
//   y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in block b} qx[m, k] qw[n, k]
//
// A block's products are added by the tensor core (tcgen05.mma kind::f8f6f4, four instructions of 32 K) into a buffer of
// tensor memory of its own; the scales are fp32, so no instruction applies them, and the epilogue warps take every finished
// buffer into registers: acc += partial * (sx sw).  Two to four buffers keep the tensor core busy meanwhile.
//
// Two arrangements of the same pipeline:
//   wide     the 128 lanes of tensor memory are rows of x, the columns 128 or 256 rows of the weight.  A thread owns a
//            row of x and columns of one weight block: its scale is one number a block.
//   swapped  (up to 64 rows of x) the lanes are weight rows, the columns 16, 32 or 64 rows of x, so that no tensor time
//            and no bandwidth is spent on rows that are not there; a block's scales come as a row of shared memory.
//
//   warps 0 .. E-1   epilogue (E = 4, or 8 with 128 columns and more)
//   warp E           producer: per block of 128 K a box of both operands (128-byte swizzle) and the scales of x
//   warp E + 1       tensor memory, MMA issue
//
// Work split: an item is a tile of y.  A cluster of c CTAs (1, 2, 4 or 8) takes items in turn; its CTAs cut the blocks of K
// in c runs, send their sums of 128 / c lanes to each CTA's shared memory and each CTA adds its lanes' in rank order: one launch,
// no workspace, deterministic.  Every wait is bounded and reports through the caller's status word.

#include <mutex>

#include "common.cuh"
#include "fp8.cuh"
#include "tcgen05.cuh"

namespace mixfp4 {
namespace {

constexpr int kMaxStages = 12;
constexpr uint32_t kSmemMax = 227 * 1024;

struct Fp8Args {
    const float* sx;                     // [blocks][ldsx]
    const float* sw;                     // [ceil(n / 128)][blocks]
    void* y;
    int64_t ldsx, ldy;
    int m, n, blocks;
    int x_tiles, items, cluster, stages, out_dtype;
    bool y_vec;                          // rows of y are 16-byte aligned
    int* status;
};

template <int kCols, bool kSwap>
struct Fp8Cfg {
    static constexpr int kEpi = kCols > 64 ? 8 : 4;                     // epilogue warps
    static constexpr int kPer = kCols * 4 / kEpi;                       // columns of a thread
    static constexpr int kThreads = (kEpi + 2) * 32;
    static constexpr uint32_t kABytes = 128 * 128, kBBytes = kCols * 128, kStage = kABytes + kBBytes;
    static constexpr int kScales = kSwap ? kCols : 128;                 // scales of x in a block
    static constexpr int kBufs = kCols > 128 ? 2 : 4;
    static constexpr uint32_t kBufCols = kCols < 32 ? 32 : kCols, kTmemCols = kBufs * kBufCols;
    // D fp32, A and B E4M3, both K-major
    static constexpr uint32_t kInstrDesc = (1u << 4) | ((uint32_t)(kCols >> 3) << 17) | ((128u >> 4) << 24);
    static constexpr uint32_t kPitch = kCols + 4;                       // floats of a lane in the exchange: lanes 16 bytes apart in the banks
};

struct Fp8Layout {
    uint32_t scales, exchange, bars, misc, bytes;
};
template <int kCols, bool kSwap>
__host__ __device__ inline Fp8Layout fp8_layout(int stages, int cluster) {
    using C = Fp8Cfg<kCols, kSwap>;
    Fp8Layout l;
    l.scales = (uint32_t)stages * C::kStage;
    l.exchange = l.scales + (uint32_t)stages * C::kScales * 4u;
    l.bars = l.exchange + (cluster > 1 ? 128u * C::kPitch * 4u : 0u);
    l.misc = l.bars + (2 * kMaxStages + 2 * 4 + 2) * 8;
    l.bytes = l.misc + 16 + 1024;                                       // + alignment slack
    return l;
}

__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// kN columns of this warp's 32 lanes, without the wait.
template <int kN>
__device__ __forceinline__ void tmem_load(uint32_t taddr, float (&r)[kN]);
template <>
__device__ __forceinline__ void tmem_load<16>(uint32_t taddr, float (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
          "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
        : "r"(taddr) : "memory");
}
// The values may be used after this; they pass through it so that no use moves above it.
template <int kN>
__device__ __forceinline__ void tmem_wait(float (&r)[kN]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < kN; ++i) asm volatile("" : "+f"(r[i]));
}

__device__ __forceinline__ float lds_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ float4 lds_f32x4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
    return remote;
}
__device__ __forceinline__ void st_peer(uint32_t remote, float a, float b, float c, float d) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(remote), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}
__device__ __forceinline__ void arrive_peer(uint32_t remote_bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote_bar) : "memory");
}
__device__ __forceinline__ bool try_wait_cluster(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// mbar_wait on arrivals from other CTAs of the cluster.
__device__ __forceinline__ bool wait_cluster(uint32_t bar, uint32_t parity, const WaitCtx& ctx, int code) {
    if (try_wait_cluster(bar, parity)) return true;
    const uint64_t t0 = global_timer_ns();
    uint32_t spins = 0;
    while (!try_wait_cluster(bar, parity)) {
        if ((++spins & 63u) == 0) {
            if (*ctx.abort_flag) return false;
            if (spins > kMinSpins && global_timer_ns() - t0 > ctx.limit_ns) {
                *ctx.abort_flag = 1;
                if (ctx.status) atomicCAS(ctx.status, 0, code);
                return false;
            }
        }
    }
    return true;
}

__device__ __forceinline__ void store_one(const Fp8Args& a, int64_t row, int64_t col, float v) {
    const int64_t at = row * a.ldy + col;
    if (a.out_dtype == MIXFP4_F32) static_cast<float*>(a.y)[at] = v;
    else if (a.out_dtype == MIXFP4_BF16) static_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(v);
    else static_cast<__half*>(a.y)[at] = __float2half_rn(v);
}
// kN consecutive columns of a row, 16 bytes at a time where the whole run is inside and aligned.
template <int kN>
__device__ __forceinline__ void store_run(const Fp8Args& a, int64_t row, int64_t col, const float (&v)[kN]) {
    static_assert(kN % 8 == 0, "a run is stored in 16-byte pieces");
    if (!a.y_vec || col + kN > a.n) {
#pragma unroll
        for (int j = 0; j < kN; ++j)
            if (col + j < a.n) store_one(a, row, col + j, v[j]);
    } else if (a.out_dtype == MIXFP4_F32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(a.y) + row * a.ldy + col);
#pragma unroll
        for (int j = 0; j < kN; j += 4) p[j / 4] = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    } else {
        uint4* p = reinterpret_cast<uint4*>(static_cast<__half*>(a.y) + row * a.ldy + col);
#pragma unroll
        for (int j = 0; j < kN; j += 8) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float lo = v[j + 2 * i], hi = v[j + 2 * i + 1];
                if (a.out_dtype == MIXFP4_BF16) {
                    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
                    w[i] = *reinterpret_cast<const uint32_t*>(&b);
                } else {
                    const __half2 h = __floats2half2_rn(lo, hi);
                    w[i] = *reinterpret_cast<const uint32_t*>(&h);
                }
            }
            p[j / 8] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

template <int kCols, bool kSwap>
__global__ void __launch_bounds__(Fp8Cfg<kCols, kSwap>::kThreads, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const Fp8Args a) {
    using C = Fp8Cfg<kCols, kSwap>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;        // the same offset in every CTA of the cluster
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const Fp8Layout L = fp8_layout<kCols, kSwap>(a.stages, a.cluster);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int rank = (int)cluster_ctarank();
    auto full = [&](int s) { return base + L.bars + s * 8; };
    auto empty = [&](int s) { return base + L.bars + (kMaxStages + s) * 8; };
    auto acc_full = [&](int b) { return base + L.bars + (2 * kMaxStages + b) * 8; };
    auto acc_empty = [&](int b) { return base + L.bars + (2 * kMaxStages + 4 + b) * 8; };
    const uint32_t sums_in = base + L.bars + (2 * kMaxStages + 8) * 8, sums_out = sums_in + 8;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + L.misc + 8);
    const WaitCtx ctx{abort_flag, a.status};

    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1 + C::kEpi); }
        for (int b = 0; b < C::kBufs; ++b) { mbar_init(acc_full(b), 1); mbar_init(acc_empty(b), C::kEpi); }
        mbar_init(sums_in, (uint32_t)a.cluster * C::kEpi);              // every warp of every CTA of the cluster has sent
        mbar_init(sums_out, (uint32_t)a.cluster * C::kEpi);             // ... and has added its share of what was sent
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_proxy();
    }
    if (warp == C::kEpi + 1) tmem_alloc(base + L.misc, C::kTmemCols);
    tcgen05_fence_before();
    __syncthreads();
    if (a.cluster > 1) cluster_sync_all();
    tcgen05_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gen + L.misc);

    // this CTA's run of the blocks of K; items of the cluster
    const int k0 = a.blocks * rank / a.cluster, k1 = a.blocks * (rank + 1) / a.cluster;
    const int step = (int)gridDim.x / a.cluster, first = (int)blockIdx.x / a.cluster;

    if (warp == C::kEpi) {
        if (lane == 0) {
            // Weights never depend on the kernel before (the quantizer of x): the first round of stages asks for them ahead of the wait.
            int s = 0, ahead = 0;
            uint32_t ph = 0;
            auto weights = [&](int item, int kb, int st) {
                mbar_arrive_expect_tx(full(st), C::kStage + C::kScales * 4);
                const uint32_t dst = base + st * C::kStage + (kSwap ? 0u : C::kABytes);
                tma_load_2d(dst, &map_w, full(st), kb * 128, item / a.x_tiles * (kSwap ? 128 : kCols));
            };
            for (int item = first; item < a.items && ahead < a.stages; item += step)
                for (int kb = k0; kb < k1 && ahead < a.stages; ++kb) weights(item, kb, ahead++);
            asm volatile("griddepcontrol.wait;" ::: "memory");
            asm volatile("fence.proxy.async.global;" ::: "memory");     // ordinary stores of that kernel, read by TMA
            bool ok = true;
            for (int item = first; item < a.items && ok; item += step) {
                const int x0 = item % a.x_tiles * (kSwap ? kCols : 128);
                for (int kb = k0; kb < k1; ++kb) {
                    if (ahead > 0) --ahead;
                    else {
                        ok = mbar_wait(empty(s), ph ^ 1, ctx, 21);
                        if (!ok) break;
                        weights(item, kb, s);
                    }
                    tma_load_2d(base + s * C::kStage + (kSwap ? C::kABytes : 0u), &map_x, full(s), kb * 128, x0);
                    bulk_load(base + L.scales + s * (C::kScales * 4), a.sx + (int64_t)kb * a.ldsx + x0, C::kScales * 4, full(s));
                    if (++s == a.stages) { s = 0; ph ^= 1; }
                }
            }
        }
    } else if (warp == C::kEpi + 1) {
        if (lane == 0) {
            int s = 0, b = 0;
            uint32_t ph = 0, bph = 0;
            bool ok = true;
            for (int item = first; item < a.items && ok; item += step) {
                for (int kb = k0; kb < k1; ++kb) {
                    ok = mbar_wait(acc_empty(b), bph ^ 1, ctx, 22) && mbar_wait(full(s), ph, ctx, 23);
                    if (!ok) break;
                    tcgen05_fence_after();
                    const uint64_t da = make_smem_desc(base + s * C::kStage), db = make_smem_desc(base + s * C::kStage + C::kABytes);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        umma_f8(tmem + b * C::kBufCols, da + 2u * k, db + 2u * k, C::kInstrDesc, k != 0 ? 1u : 0u);
                    umma_commit(empty(s));
                    umma_commit(acc_full(b));
                    if (++s == a.stages) { s = 0; ph ^= 1; }
                    if (++b == C::kBufs) { b = 0; bph ^= 1; }
                }
            }
        }
    } else {
        const int quad = warp & 3, half = warp >> 2;                    // lanes 32 quad .., columns half * kPer ..
        const int tl = quad * 32 + lane;
        int s = 0, b = 0;
        uint32_t ph = 0, bph = 0, xph = 0;
        bool ok = true;
        for (int item = first; item < a.items && ok; item += step) {
            const int x0 = item % a.x_tiles * (kSwap ? kCols : 128), w0 = item / a.x_tiles * (kSwap ? 128 : kCols);
            const int wb = (w0 + (kSwap ? 0 : half * C::kPer)) / 128;   // weight block of this thread's columns
            const float* sw = a.sw + (int64_t)min(wb, (a.n - 1) / 128) * a.blocks;
            float acc[C::kPer];
#pragma unroll
            for (int j = 0; j < C::kPer; ++j) acc[j] = 0.0f;
            float sw_next = k0 < k1 ? __ldg(sw + k0) : 0.0f;
            for (int kb = k0; kb < k1; ++kb) {
                const float sw_now = sw_next;
                if (kb + 1 < k1) sw_next = __ldg(sw + kb + 1);
                ok = __all_sync(0xffffffffu, mbar_wait(acc_full(b), bph, ctx, 24) && mbar_wait(full(s), ph, ctx, 25));
                if (!ok) break;
                tcgen05_fence_after();
                const uint32_t sc = base + L.scales + s * (C::kScales * 4);
                const float row_scale = kSwap ? 0.0f : lds_f32(sc + tl * 4) * sw_now;
                const uint32_t src = tmem + ((uint32_t)(quad * 32) << 16) + b * C::kBufCols + half * C::kPer;
#pragma unroll
                for (int c = 0; c < C::kPer; c += 16) {
                    float v[16];
                    tmem_load<16>(src + c, v);
                    float4 sj[4];
                    if constexpr (kSwap) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) sj[q] = lds_f32x4(sc + (c + 4 * q) * 4);
                    }
                    tmem_wait(v);
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float f = kSwap ? reinterpret_cast<const float*>(sj)[j] * sw_now : row_scale;
                        acc[c + j] = fmaf(v[j], f, acc[c + j]);
                    }
                }
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) { mbar_arrive(acc_empty(b)); mbar_arrive(empty(s)); }
                if (++s == a.stages) { s = 0; ph ^= 1; }
                if (++b == C::kBufs) { b = 0; bph ^= 1; }
            }
            if (!ok) break;
            if (a.cluster == 1) {
                if constexpr (kSwap) {
                    if (w0 + tl < a.n) {
#pragma unroll
                        for (int j = 0; j < C::kPer; ++j)
                            if (x0 + j < a.m) store_one(a, x0 + j, w0 + tl, acc[j]);
                    }
                } else if (x0 + tl < a.m) {
                    store_run(a, x0 + tl, w0 + half * C::kPer, acc);
                }
                continue;
            }
            // Sums of lanes [r 128/c, (r+1) 128/c) to rank r, slot of this rank: [source][lane][column].
            const int share = 128 / a.cluster;
            const uint32_t xbuf = base + L.exchange;
            ok = __all_sync(0xffffffffu, wait_cluster(sums_out, xph ^ 1, ctx, 26));
            if (!ok) break;
            const uint32_t dst = peer_addr(xbuf + (((uint32_t)rank * share + tl % share) * C::kPitch + half * C::kPer) * 4, tl / share);
#pragma unroll
            for (int j = 0; j < C::kPer; j += 4) st_peer(dst + j * 4, acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
            asm volatile("fence.acq_rel.cluster;" ::: "memory");
            __syncwarp();
            if (lane < a.cluster) arrive_peer(peer_addr(sums_in, lane));
            ok = __all_sync(0xffffffffu, wait_cluster(sums_in, xph, ctx, 27));
            if (!ok) break;
            xph ^= 1;
            const int groups = kCols / 4;                               // four columns of a lane at a time
            for (int i = threadIdx.x; i < share * groups; i += C::kEpi * 32) {
                const int l = kSwap ? i % share : i / groups, c = (kSwap ? i / share : i % groups) * 4;
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (int r = 0; r < a.cluster; ++r) {
                    const float4 v = lds_f32x4(xbuf + (((uint32_t)r * share + l) * C::kPitch + c) * 4);
                    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
                }
                const float e[4] = {sum.x, sum.y, sum.z, sum.w};
                const int tile_lane = rank * share + l;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int64_t row = kSwap ? x0 + c + j : x0 + tile_lane, col = kSwap ? w0 + tile_lane : w0 + c + j;
                    if (row < a.m && col < a.n) store_one(a, row, col, e[j]);
                }
            }
            __syncwarp();
            if (lane < a.cluster) arrive_peer(peer_addr(sums_out, lane));
        }
    }
    // Every role has stopped issuing.  Without an expired wait all copies have landed and all MMAs are done; after one they
    // get a millisecond (hundreds of times what a block takes) before tensor memory is freed and the CTA leaves.
    tcgen05_fence_before();
    __syncthreads();
    if (*abort_flag) {
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 1000000ull) {}
    }
    if (warp == C::kEpi + 1) {
        tcgen05_fence_after();
        tmem_dealloc(tmem, C::kTmemCols);
    }
    if (a.cluster > 1) cluster_sync_all();                              // no CTA leaves while its peers still send to it
}

// ------------------------------------------------------------------------- host side
constexpr int kMaxDevices = 64, kMaxClusterLog = 3;

// Clusters of 1, 2, 4 and 8 CTAs that the current device runs at once, asked once per device and kernel.
template <int kCols, bool kSwap>
int active_clusters(int (&out)[kMaxClusterLog + 1]) {
    static std::mutex lock;
    static int known[kMaxDevices][kMaxClusterLog + 1];
    static bool have[kMaxDevices];
    int dev = 0;
    MIXFP4_CUDA_CHECK(cudaGetDevice(&dev));
    if (dev < 0 || dev >= kMaxDevices) return MIXFP4_E_UNSUPPORTED;
    std::lock_guard<std::mutex> guard(lock);
    if (!have[dev]) {
        const auto kernel = fp8_gemm_kernel<kCols, kSwap>;
        MIXFP4_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemMax));
        for (int c = 0; c <= kMaxClusterLog; ++c) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(1u << c);
            cfg.blockDim = dim3(Fp8Cfg<kCols, kSwap>::kThreads);
            cfg.dynamicSmemBytes = kSmemMax;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = 1u << c;
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            int n = 0;
            if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
                (void)cudaGetLastError();                               // a cluster size the device does not take
                n = 0;
            }
            known[dev][c] = n;
        }
        have[dev] = true;
    }
    for (int c = 0; c <= kMaxClusterLog; ++c) out[c] = known[dev][c];
    return MIXFP4_OK;
}

struct Fp8Problem {
    const uint8_t* x;
    int64_t ldx;
    const uint8_t* w;
    int64_t ldw, k;
    bool dependent;                      // the kernel before is the quantizer of x
};

int encode_codes(EncodeTiledFn fn, CUtensorMap* map, const uint8_t* p, int64_t rows, int64_t k, int64_t ld, uint32_t box_rows) {
    cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
    cuuint32_t box[2] = {128, box_rows}, elem[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(p), dims, strides, box, elem,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? MIXFP4_OK : record_error_text("cuTensorMapEncodeTiled failed for an fp8 operand");
}

// Microseconds that an arrangement would take: rounds of items times blocks in a run.  Per block: what the weights of one SM
// take from HBM, or the tensor core and the epilogue; per item: filling and draining the pipeline, an exchange.
template <int kCols, bool kSwap>
float fp8_cost(const Fp8Args& a, int cluster_log, const int* clusters) {
    const int c = 1 << cluster_log;
    if (clusters[cluster_log] < 1 || c > a.blocks || (kCols > 128 && c > 1)) return 1e30f;
    const int64_t lanes = kSwap ? a.n : a.m, cols = kSwap ? a.m : a.n;
    const int64_t items = (lanes + 127) / 128 * ((cols + kCols - 1) / kCols);
    const int64_t rounds = (items + clusters[cluster_log] - 1) / clusters[cluster_log];
    const float block = kSwap ? 0.38f : kCols == 128 ? 0.24f : 0.36f;
    return (float)rounds * (block * (float)((a.blocks + c - 1) / c) + (c > 1 ? 1.5f : 0.7f));
}

template <int kCols, bool kSwap>
int launch_fp8(Fp8Args a, const Fp8Problem& p, int cluster_log, const int* clusters, cudaStream_t st) {
    using C = Fp8Cfg<kCols, kSwap>;
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return record_error_text("cuTensorMapEncodeTiled is not available");
    CUtensorMap map_x, map_w;
    if (const int rc = encode_codes(fn, &map_x, p.x, a.m, p.k, p.ldx, kSwap ? kCols : 128)) return rc;
    if (const int rc = encode_codes(fn, &map_w, p.w, a.n, p.k, p.ldw, kSwap ? 128 : kCols)) return rc;
    a.cluster = 1 << cluster_log;
    a.x_tiles = (a.m + (kSwap ? kCols : 128) - 1) / (kSwap ? kCols : 128);
    const int64_t items = (int64_t)a.x_tiles * ((a.n + (kSwap ? 128 : kCols) - 1) / (kSwap ? 128 : kCols));
    if (items > 0x3fffffff) return MIXFP4_E_SHAPE;
    a.items = (int)items;
    a.stages = kMaxStages;
    while (fp8_layout<kCols, kSwap>(a.stages, a.cluster).bytes > kSmemMax) --a.stages;
    const int n = a.items < clusters[cluster_log] ? a.items : clusters[cluster_log];
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(n * a.cluster));
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = fp8_layout<kCols, kSwap>(a.stages, a.cluster).bytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)a.cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.dependent ? 2 : 1;
    const auto kernel = fp8_gemm_kernel<kCols, kSwap>;
    MIXFP4_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, map_x, map_w, a));
    return check_launch("fp8_gemm_kernel");
}

struct Fp8Choice {
    float cost = 1e30f;
    int cols = 0, cluster_log = 0;
    int clusters[kMaxClusterLog + 1] = {};
};
template <int kCols, bool kSwap>
int consider(const Fp8Args& a, Fp8Choice& best) {
    int clusters[kMaxClusterLog + 1];
    if (const int rc = active_clusters<kCols, kSwap>(clusters)) return rc;
    for (int c = 0; c <= kMaxClusterLog; ++c) {
        const float t = fp8_cost<kCols, kSwap>(a, c, clusters);
        if (t < best.cost) {
            best.cost = t; best.cols = kCols; best.cluster_log = c;
            for (int i = 0; i <= kMaxClusterLog; ++i) best.clusters[i] = clusters[i];
        }
    }
    return MIXFP4_OK;
}

int fp8_gemm(const Fp8Args& a, const Fp8Problem& p, cudaStream_t st) {
    Fp8Choice best;
    int rc;
    if (a.m <= 16) rc = consider<16, true>(a, best);
    else if (a.m <= 32) rc = consider<32, true>(a, best);
    else if (a.m <= 64) rc = consider<64, true>(a, best);
    else if (!(rc = consider<128, false>(a, best))) rc = consider<256, false>(a, best);
    if (rc) return rc;
    switch (best.cols) {
        case 16: return launch_fp8<16, true>(a, p, best.cluster_log, best.clusters, st);
        case 32: return launch_fp8<32, true>(a, p, best.cluster_log, best.clusters, st);
        case 64: return launch_fp8<64, true>(a, p, best.cluster_log, best.clusters, st);
        case 128: return launch_fp8<128, false>(a, p, best.cluster_log, best.clusters, st);
        case 256: return launch_fp8<256, false>(a, p, best.cluster_log, best.clusters, st);
        default: return MIXFP4_E_UNSUPPORTED;
    }
}

constexpr int64_t kMaxSide = 0x7fffff00;

int check_product(const uint8_t* w, int64_t ldw, const float* sw, int64_t m, int64_t n, int64_t k, const void* y, int out_dtype,
                  int64_t ldy) {
    if (!w || !sw || !y) return MIXFP4_E_NULL;
    if (out_dtype != MIXFP4_BF16 && out_dtype != MIXFP4_F16 && out_dtype != MIXFP4_F32) return MIXFP4_E_DTYPE;
    if (m <= 0 || n <= 0 || k <= 0 || m > kMaxSide || n > kMaxSide || k > kMaxSide || ldw < k || ldy < n) return MIXFP4_E_SHAPE;
    if (!aligned(w, 16) || ldw % 16 != 0 || !aligned(sw, 4)) return MIXFP4_E_ALIGN;
    return MIXFP4_OK;
}

Fp8Args make_args(const float* sx, int64_t ldsx, const float* sw, int64_t m, int64_t n, int64_t k, void* y, int out_dtype,
                  int64_t ldy, int* status) {
    Fp8Args a = {};
    a.sx = sx; a.sw = sw; a.y = y; a.ldsx = ldsx; a.ldy = ldy;
    a.m = (int)m; a.n = (int)n; a.blocks = (int)((k + kFp8Block - 1) / kFp8Block);
    a.out_dtype = out_dtype; a.status = status;
    a.y_vec = aligned(y, 16) && ldy * (out_dtype == MIXFP4_F32 ? 4 : 2) % 16 == 0;
    return a;
}

}  // namespace
}  // namespace mixfp4

using namespace mixfp4;

extern "C" int mixfp4_fp8_gemm(const uint8_t* x, int64_t ldx, const float* x_scales, int64_t lds, const uint8_t* w, int64_t ldw,
                               const float* w_scales, int64_t m, int64_t n, int64_t k, void* y, int out_dtype, int64_t ldy,
                               int* status, void* stream) {
    if (!x || !x_scales) return MIXFP4_E_NULL;
    if (const int rc = check_product(w, ldw, w_scales, m, n, k, y, out_dtype, ldy)) return rc;
    if (ldx < k || lds < fp8_scale_rows(m)) return MIXFP4_E_SHAPE;
    if (!aligned(x, 16) || ldx % 16 != 0 || !aligned(x_scales, 16) || lds % 4 != 0) return MIXFP4_E_ALIGN;
    return fp8_gemm(make_args(x_scales, lds, w_scales, m, n, k, y, out_dtype, ldy, status), Fp8Problem{x, ldx, w, ldw, k, false},
                    static_cast<cudaStream_t>(stream));
}

extern "C" int64_t mixfp4_fp8_workspace_bytes(int64_t m, int64_t k) {
    if (m <= 0 || k <= 0) return 0;
    const int64_t kp = padded_k(k);
    return (m * kp + 15) / 16 * 16 + fp8_scale_rows(m) * (kp / kFp8Block) * 4;
}

extern "C" int mixfp4_fp8_linear(const void* x, int dtype, int64_t m, int64_t ldx, const uint8_t* w, int64_t ldw,
                                 const float* w_scales, int64_t n, int64_t k, void* y, int out_dtype, int64_t ldy,
                                 void* workspace, int64_t workspace_bytes, int* status, void* stream) {
    if (!x) return MIXFP4_E_NULL;
    if (const int rc = check_product(w, ldw, w_scales, m, n, k, y, out_dtype, ldy)) return rc;
    if (!workspace || workspace_bytes < mixfp4_fp8_workspace_bytes(m, k)) return MIXFP4_E_WORKSPACE;
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    const int64_t kp = padded_k(k), lds = fp8_scale_rows(m);
    float* scales = reinterpret_cast<float*>(codes + (m * kp + 15) / 16 * 16);
    if (const int rc = fp8_check_rows(x, dtype, m, k, ldx, codes, kp, scales, lds)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (const int rc = fp8_quantize_rows(x, dtype, m, k, ldx, codes, kp, scales, lds, st)) return rc;
    return fp8_gemm(make_args(scales, lds, w_scales, m, n, k, y, out_dtype, ldy, status), Fp8Problem{codes, kp, w, ldw, k, true}, st);
}

// Product of E4M3 operands with an fp32 scale per block of 128 along K (rows of x: one per row, weight: one per 128 x 128):
//   y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in block b} qx[m, k] qw[n, k]
//
// A block's products are added by the tensor core (tcgen05.mma kind::f8f6f4, four instructions of 32 K) into a buffer of
// tensor memory of its own; the scales are fp32, so no instruction applies them, and the epilogue warps take every finished
// buffer into registers: acc += partial * (sx sw).  Two to four buffers keep the tensor core busy meanwhile.
//
// Three arrangements of the same pipeline:
//   swapped  (up to 64 rows of x) the lanes of tensor memory are 128 weight rows, the columns 16, 32 or 64 rows of x, so that no
//            tensor time and no bandwidth is spent on rows that are not there; a block's scales come as a row of shared memory.
//   wide     the lanes are 128 rows of x, the columns 128 rows of the weight.  A thread owns a row of x and columns of one
//            weight block: its scale is one number a block.
//   pairs    256 x 256 for two CTAs (further down).
//
//   warps 0 .. E-1   epilogue (E = 4, 8 from 64 columns on)
//   warp E           producer: per block of 128 K a box of both operands (128-byte swizzle) and the scales of x
//   warp E + 1       tensor memory, MMA issue
//
// What bounds it.  One token, 128256 x 4096: HBM (79 us, 6.7 TB/s).  Few rows: a fixed 5 to 6 us (launch, set-up, first loads,
// exchange) beside the weights' bytes; 48 x 14336 x 4096 (15.7 us, 3.8 TB/s) also that items are whole tiles, so that its 112 keep 112 of
// 148 SMs busy: a choice of this split, not a limit (tiles cut along K between neighbouring clusters would use all).
// Many rows: 4096 x 14336 x 4096 242 us, 1.99 PFLOP/s, in a burst and 284 us under the power cap (1.67 GHz); a block takes about 1060 cycles
// of a pair for 512 of MMA, the rest is the way of a buffer from the MMA's end through the epilogue back to the issuer.
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
    const void* x;                       // dense rows, where the kernel quantizes them itself
    int64_t ldx;
    int x_dtype;
    bool x_vec;
    const float* sx;                     // [blocks][ldsx]
    const float* sw;                     // [ceil(n / 128)][blocks]
    void* y;
    int64_t ldsx, ldy;
    int m, n, k, blocks;
    int x_tiles, items, cluster, stages, out_dtype;
    bool early_weights;                  // the kernel before writes x and nothing else of this one's: weights are asked for ahead of it
    bool y_vec;                          // rows of y are whole 32-byte sectors
    int* status;
};

// kOwn: x is dense and quantized by every CTA, its run of K for all rows, into shared memory.
template <int kCols, bool kSwap, bool kOwn>
struct Fp8Cfg {
    static constexpr int kEpi = kCols >= 64 ? 8 : 4;                    // epilogue warps
    static constexpr int kPer = kCols * 4 / kEpi;                       // columns of a thread
    static constexpr int kThreads = (kEpi + 2) * 32;
    static constexpr uint32_t kABytes = 128 * 128, kBBytes = kCols * 128, kStage = kABytes + (kOwn ? 0 : kBBytes);
    static constexpr int kScales = kSwap && !kOwn ? kCols : 0;          // scales of x in a stage
    static constexpr int kBufs = 4;
    static constexpr uint32_t kBufCols = kCols < 32 ? 32 : kCols, kTmemCols = kBufs * kBufCols;
    // D fp32, A and B E4M3, both K-major
    static constexpr uint32_t kInstrDesc = (1u << 4) | ((uint32_t)(kCols >> 3) << 17) | ((128u >> 4) << 24);
};

// Rows of y that are off their sectors leave through a patch of 32 rows x kPatchCols columns a warp, so that a store's lanes are
// neighbouring columns.
constexpr int kPatchCols = 16, kPatchPitch = kPatchCols + 1;
constexpr uint32_t kPatchBytes = 32 * kPatchPitch * 4;

struct Fp8Layout {
    uint32_t own, own_scales, scales, exchange, patches, bars, misc, bytes;
};
template <int kCols, bool kSwap, bool kOwn>
__host__ __device__ inline Fp8Layout fp8_layout(int stages, int cluster, int blocks, bool y_vec) {
    using C = Fp8Cfg<kCols, kSwap, kOwn>;
    const uint32_t run = kOwn ? (uint32_t)((blocks + cluster - 1) / cluster) : 0u;
    Fp8Layout l;
    l.own = (uint32_t)stages * C::kStage;
    l.own_scales = l.own + run * C::kBBytes;
    l.scales = l.own_scales + run * kCols * 4u;
    l.exchange = l.scales + (uint32_t)stages * C::kScales * 4u;
    l.patches = l.exchange + (cluster > 1 ? (128u + cluster) * (kCols / 4) * 16u : 0u);
    l.bars = l.patches + (kSwap || cluster > 1 || y_vec ? 0u : C::kEpi * kPatchBytes);
    l.misc = l.bars + (2 * kMaxStages + 2 * 4 + 3) * 8;
    l.bytes = (l.misc + 16 + 1024 + 7) & ~7u;                           // + alignment slack
    return l;
}

// The single-warp roles run converged, and their issuing instructions take the elected lane as a predicate: the code around
// them stays uniform, their operands in uniform registers.  (A branch for one lane took three times as long a block.)
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p;
}
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, const WaitCtx& ctx, int code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, ctx, code));
}
__device__ __forceinline__ void expect_if(uint32_t lead, uint32_t bar, uint32_t bytes) {
    asm volatile(
        "{\n\t.reg .pred l;\n\tsetp.ne.u32 l, %0, 0;\n\t"
        "@l mbarrier.arrive.expect_tx.shared::cta.b64 _, [%1], %2;\n\t}"
        ::"r"(lead), "r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_load_if(uint32_t lead, uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    asm volatile(
        "{\n\t.reg .pred l;\n\tsetp.ne.u32 l, %0, 0;\n\t"
        "@l cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%1], [%2, {%4, %5}], [%3];\n\t}"
        ::"r"(lead), "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void bulk_load_if(uint32_t lead, uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred l;\n\tsetp.ne.u32 l, %0, 0;\n\t"
        "@l cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%1], [%2], %3, [%4];\n\t}"
        ::"r"(lead), "r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void umma_f8_if(uint32_t lead, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, l;\n\t"
        "setp.ne.b32 p, %5, 0;\n\tsetp.ne.u32 l, %0, 0;\n\t"
        "@l tcgen05.mma.cta_group::1.kind::f8f6f4 [%1], %2, %3, %4, p;\n\t}"
        ::"r"(lead), "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_commit_if(uint32_t lead, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred l;\n\tsetp.ne.u32 l, %0, 0;\n\t"
        "@l tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}"
        ::"r"(lead), "r"(bar) : "memory");
}
// 16 or 32 columns of this warp's 32 lanes, without the wait.
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// A loaded column passes through this after the wait, so that no use of it moves above.
template <int kN>
__device__ __forceinline__ void tmem_landed(uint32_t (&r)[kN]) {
#pragma unroll
    for (int i = 0; i < kN; ++i) asm volatile("" : "+r"(r[i]));
}
template <int kRegs>
__device__ __forceinline__ void take_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs)); }
template <int kRegs>
__device__ __forceinline__ void give_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs)); }

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

// f(y) with the output's type.  Around whole loops: a kernel of few rows runs its stores once, and what it fetches of its code on the
// way counts.
template <typename F>
__device__ __forceinline__ void with_output(const Fp8Args& a, F&& f) {
    if (a.out_dtype == MIXFP4_BF16) f(static_cast<__nv_bfloat16*>(a.y));
    else if (a.out_dtype == MIXFP4_F32) f(static_cast<float*>(a.y));
    else f(static_cast<__half*>(a.y));
}
template <typename T>
__device__ __forceinline__ void put(T* p, float v) { *p = Elem<T>::round(v); }
// 32 aligned bytes, a whole sector of the L2.
__device__ __forceinline__ void st_sector(void* p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
// kN consecutive columns of this lane's row, row0 + lane, by a whole warp.  A sector at a time where rows of y are whole sectors;
// otherwise through the warp's patch (4096 x 4099 x 4096 bf16: 95 us, 4096 x 1000 x 4096: 26 us; each thread storing its row's
// columns one by one, 32 sectors an instruction: 231 us and 61 us).
template <int kN>
__device__ __forceinline__ void store_run(const Fp8Args& a, int64_t row0, int64_t col, const float (&v)[kN], float* patch) {
    static_assert(kN % 16 == 0 && kPatchCols == 16, "a run is stored in sectors");
    const int lane = threadIdx.x & 31;
    const int64_t row = row0 + lane;
    if (!a.y_vec) {
#pragma unroll
        for (int c = 0; c < kN; c += kPatchCols) {
#pragma unroll
            for (int j = 0; j < kPatchCols; ++j) patch[lane * kPatchPitch + j] = v[c + j];
            __syncwarp();
            const int j = lane % kPatchCols;
            if (col + c + j < a.n) {
                with_output(a, [&](auto* y) {
#pragma unroll 8
                    for (int i = lane / kPatchCols; i < 32; i += 32 / kPatchCols)
                        if (row0 + i < a.m) put(y + (row0 + i) * a.ldy + col + c + j, patch[i * kPatchPitch + j]);
                });
            }
            __syncwarp();
        }
    } else if (row >= a.m) {
        return;
    } else if (a.out_dtype == MIXFP4_F32) {
        float* p = static_cast<float*>(a.y) + row * a.ldy + col;
#pragma unroll
        for (int j = 0; j < kN; j += 8) {
            if (col + j >= a.n) break;
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[j + i]);
            st_sector(p + j, w);
        }
    } else {
        __half* p = static_cast<__half*>(a.y) + row * a.ldy + col;
#pragma unroll
        for (int j = 0; j < kN; j += 16) {
            if (col + j >= a.n) break;
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float lo = v[j + 2 * i], hi = v[j + 2 * i + 1];
                if (a.out_dtype == MIXFP4_BF16) {
                    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
                    w[i] = *reinterpret_cast<const uint32_t*>(&b);
                } else {
                    const __half2 h = __floats2half2_rn(lo, hi);
                    w[i] = *reinterpret_cast<const uint32_t*>(&h);
                }
            }
            st_sector(p + j, w);
        }
    }
}

// acc += columns src .. of this warp's lanes * f, the next 32 columns on their way while 32 are added; given_back() once the
// last have landed.  (One multiplication at a time: the packed form of two needs its operands in aligned pairs, and the moves
// that bring the loaded columns there cost more than it saves.)
template <int kPer, typename Done>
__device__ __forceinline__ void add_scaled(uint32_t src, float f, float (&acc)[kPer], Done&& given_back) {
    uint32_t v[2][32];
    tmem_load(src, v[0]);
#pragma unroll
    for (int c = 0; c < kPer; c += 32) {
        tmem_wait();
        tmem_landed(v[(c / 32) & 1]);
        if (c + 32 < kPer) tmem_load(src + c + 32, v[(c / 32 + 1) & 1]);
        else given_back();
#pragma unroll
        for (int j = 0; j < 32; ++j) acc[c + j] = fmaf(__uint_as_float(v[(c / 32) & 1][j]), f, acc[c + j]);
    }
}
// The same with a scale for every column, at sc in shared memory, times sw.
template <int kPer, typename Done>
__device__ __forceinline__ void add_scaled_by_column(uint32_t src, uint32_t sc, float sw, float (&acc)[kPer], Done&& given_back) {
    constexpr int kLoad = kPer < 32 ? kPer : 32;
    uint32_t v[kPer / kLoad][kLoad];
    float4 sj[kPer / 4];
#pragma unroll
    for (int c = 0; c < kPer; c += kLoad) tmem_load(src + c, v[c / kLoad]);
#pragma unroll
    for (int q = 0; q < kPer / 4; ++q) sj[q] = lds_f32x4(sc + q * 16);
    tmem_wait();
#pragma unroll
    for (int c = 0; c < kPer; c += kLoad) tmem_landed(v[c / kLoad]);
#pragma unroll
    for (int q = 0; q < kPer / 4; ++q)                              // the scales have been read before the stage is given back
        asm volatile("" : "+f"(sj[q].x), "+f"(sj[q].y), "+f"(sj[q].z), "+f"(sj[q].w));
    given_back();
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const float4 four = sj[j / 4];
        const float f = (j % 4 == 0 ? four.x : j % 4 == 1 ? four.y : j % 4 == 2 ? four.z : four.w) * sw;
        acc[j] = fmaf(__uint_as_float(v[j / kLoad][j % kLoad]), f, acc[j]);
    }
}

// Rows of x and blocks k0 .. k1 of K: codes as the B operand of the product (kCols rows of 128 bytes a block, swizzled), scales
// as [block][kCols].  Rows that x does not have stay as they are: they make columns that nobody stores.  A group of eight lanes
// takes four blocks at a time, all loads before the first is used.
template <int kCols, typename T>
__device__ __forceinline__ void quantize_own(const Fp8Args& a, uint8_t* codes, float* scales, int k0, int k1, int thread, int threads) {
    constexpr int kAhead = 4;
    const T* x = static_cast<const T*>(a.x);
    const int sub = thread % kLanesPerRow, groups = (k1 - k0) * a.m, step = threads / kLanesPerRow;
    for (int first = 0; first < groups; first += kAhead * step) {
        Raw<T> v[kAhead];
        int block[kAhead], row[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int g = first + i * step + thread / kLanesPerRow;
            block[i] = g / a.m;
            row[i] = g - block[i] * a.m;
            load16(x + row[i] * a.ldx, (int64_t)(k0 + block[i]) * kFp8Block + sub * kLaneElems, g < groups ? a.k : 0, a.x_vec, v[i]);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            uint32_t most = largest_of(v[i]);
#pragma unroll
            for (int d = 1; d < kLanesPerRow; d *= 2) most = larger<T>(most, __shfl_xor_sync(0xffffffffu, most, d));
            if (first + i * step + thread / kLanesPerRow >= groups) continue;
            const float s = block_scale(magnitude<T>(most));
            const int at = block[i] * kCols + row[i];
            *reinterpret_cast<uint4*>(codes + at * 128 + ((sub ^ (row[i] & 7)) * 16)) = encode16(v[i], s);
            if (sub == 0) scales[at] = s;
        }
    }
}

template <int kCols, bool kSwap, bool kOwn>
__global__ void __launch_bounds__(Fp8Cfg<kCols, kSwap, kOwn>::kThreads, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const Fp8Args a) {
    using C = Fp8Cfg<kCols, kSwap, kOwn>;
    constexpr bool kRingScales = kSwap && !kOwn;                        // a stage holds scales of x: it waits for the epilogue
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;        // the same offset in every CTA of the cluster
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const Fp8Layout L = fp8_layout<kCols, kSwap, kOwn>(a.stages, a.cluster, a.blocks, a.y_vec);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int rank = (int)cluster_ctarank();
    auto full = [&](int s) { return base + L.bars + s * 8; };
    auto empty = [&](int s) { return base + L.bars + (kMaxStages + s) * 8; };
    auto acc_full = [&](int b) { return base + L.bars + (2 * kMaxStages + b) * 8; };
    auto acc_empty = [&](int b) { return base + L.bars + (2 * kMaxStages + 4 + b) * 8; };
    const uint32_t sums_in = base + L.bars + (2 * kMaxStages + 8) * 8, sums_out = sums_in + 8, x_ready = sums_in + 16;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + L.misc + 8);
    const WaitCtx ctx{abort_flag, a.status};

    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), kRingScales ? 1 + C::kEpi : 1); }
        for (int b = 0; b < C::kBufs; ++b) { mbar_init(acc_full(b), 1); mbar_init(acc_empty(b), C::kEpi); }
        mbar_init(sums_in, (uint32_t)a.cluster * C::kEpi);              // every warp of every CTA of the cluster has sent
        mbar_init(sums_out, (uint32_t)a.cluster * C::kEpi);             // ... and has added its share of what was sent
        if constexpr (kOwn) mbar_init(x_ready, C::kEpi);
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
    // Everything above runs under the tail of the kernel before, whatever it is; the next one's may run under this one's.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (!a.early_weights) asm volatile("griddepcontrol.wait;" ::: "memory");

    // this CTA's run of the blocks of K; items of the cluster
    const int k0 = a.blocks * rank / a.cluster, k1 = a.blocks * (rank + 1) / a.cluster;
    const int step = (int)gridDim.x / a.cluster, first = (int)blockIdx.x / a.cluster;

    if (warp == C::kEpi) {
        // Weights never depend on the kernel before (the quantizer of x): the first round of stages asks for them ahead of the wait.
        const uint32_t lead = elect_one();
        int s = 0, ahead = 0;
        uint32_t ph = 0;
        auto weights = [&](int row, int kb, int st) {
            expect_if(lead, full(st), C::kStage + C::kScales * 4);
            tma_load_if(lead, base + st * C::kStage + (kSwap ? 0u : C::kABytes), &map_w, full(st), kb * 128, row);
        };
        for (int item = first; item < a.items && ahead < a.stages; item += step)
            for (int kb = k0; kb < k1 && ahead < a.stages; ++kb) weights(item / a.x_tiles * (kSwap ? 128 : kCols), kb, ahead++);
        asm volatile("griddepcontrol.wait;" ::: "memory");
        asm volatile("fence.proxy.async.global;" ::: "memory");         // ordinary stores of that kernel, read by TMA
        bool ok = true;
        for (int item = first; item < a.items && ok; item += step) {
            const int wt = item / a.x_tiles, w_row = wt * (kSwap ? 128 : kCols), x_row = (item - wt * a.x_tiles) * (kSwap ? kCols : 128);
            for (int kb = k0; kb < k1; ++kb) {
                if (ahead > 0) --ahead;
                else {
                    ok = warp_wait(empty(s), ph ^ 1, ctx, 21);
                    if (!ok) break;
                    weights(w_row, kb, s);
                }
                if constexpr (!kOwn) tma_load_if(lead, base + s * C::kStage + (kSwap ? C::kABytes : 0u), &map_x, full(s), kb * 128, x_row);
                if constexpr (kRingScales)
                    bulk_load_if(lead, base + L.scales + s * (C::kScales * 4), a.sx + (int64_t)kb * a.ldsx + x_row, C::kScales * 4, full(s));
                if (++s == a.stages) { s = 0; ph ^= 1; }
            }
        }
    } else if (warp == C::kEpi + 1) {
        const uint32_t lead = elect_one();
        const uint64_t a_desc = make_smem_desc(base), b_desc = make_smem_desc(base + (kOwn ? L.own : C::kABytes));
        int s = 0, b = 0;
        uint32_t ph = 0, bph = 0;
        bool ok = true;
        if constexpr (kOwn) ok = warp_wait(x_ready, 0, ctx, 20);
        for (int item = first; item < a.items && ok; item += step) {
            for (int kb = k0; kb < k1; ++kb) {
                ok = warp_wait(full(s), ph, ctx, 23) && warp_wait(acc_empty(b), bph ^ 1, ctx, 22);
                if (!ok) break;
                tcgen05_fence_after();
                const uint64_t at = (uint64_t)(s * (C::kStage >> 4)), b_at = kOwn ? (uint64_t)((kb - k0) * (C::kBBytes >> 4)) : at;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    umma_f8_if(lead, tmem + b * C::kBufCols, a_desc + at + 2u * k, b_desc + b_at + 2u * k, C::kInstrDesc, k != 0 ? 1u : 0u);
                umma_commit_if(lead, empty(s));
                umma_commit_if(lead, acc_full(b));
                if (++s == a.stages) { s = 0; ph ^= 1; }
                if (++b == C::kBufs) { b = 0; bph ^= 1; }
            }
        }
    } else {
        if constexpr (!kSwap) asm volatile("griddepcontrol.wait;" ::: "memory");     // the scales are the kernel before's
        const int quad = warp & 3, half = warp >> 2;                    // lanes 32 quad .., columns half * kPer ..
        const int tl = quad * 32 + lane;
        if constexpr (kOwn) {
            uint8_t* codes = gen + L.own;
            float* scales = reinterpret_cast<float*>(gen + L.own_scales);
            if (a.x_dtype == MIXFP4_BF16) quantize_own<kCols, __nv_bfloat16>(a, codes, scales, k0, k1, threadIdx.x, C::kEpi * 32);
            else if (a.x_dtype == MIXFP4_F16) quantize_own<kCols, __half>(a, codes, scales, k0, k1, threadIdx.x, C::kEpi * 32);
            else quantize_own<kCols, float>(a, codes, scales, k0, k1, threadIdx.x, C::kEpi * 32);
            fence_async_proxy();                                        // the tensor core reads the codes
            __syncwarp();
            if (lane == 0) mbar_arrive(x_ready);
            mbar_wait(x_ready, 0, ctx, 28);                             // the other warps' scales; what expires shows below
        }
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
            // Swapped: the weight's scales of 32 blocks, a lane each.  Wide: both scales on their way kFar blocks ahead, in registers
            // that take turns (moving one on would wait for it); they are not a stage's, since one that stays until its scales have
            // been read keeps the operands behind it waiting.  No more copies of the loop's body than that: its code is fetched once
            // for few blocks (48 x 14336 x 4096 with four copies 15.9 us, with one 15.7; 1 x 14336 x 4096 12.7 and 12.4).
            constexpr int kFar = kSwap ? 1 : 2;
            const float *sx = a.sx + min(x0 + tl, a.m - 1) + k0 * a.ldsx, *sw_at = sw + k0;
            float sx_far[kFar], sw_far[kFar], sw_lanes = 0.0f;
            auto fetch_scales = [&](int i, bool more) {
                if constexpr (!kSwap) {
                    if (more) {
                        sw_far[i] = __ldg(sw_at);
                        sx_far[i] = __ldcg(sx);
                    }
                    ++sw_at;
                    sx += a.ldsx;
                }
            };
#pragma unroll
            for (int i = 0; i < kFar; ++i) fetch_scales(i, k0 + i < k1);
            for (int kb0 = k0; kb0 < k1 && ok; kb0 += kFar)
#pragma unroll
            for (int turn = 0; turn < kFar; ++turn) {
                const int kb = kb0 + turn;
                if (kb >= k1) break;
                if (kSwap && (kb - k0) % 32 == 0) sw_lanes = kb + lane < k1 ? __ldg(sw + kb + lane) : 0.0f;
                const float sw_now = kSwap ? __shfl_sync(0xffffffffu, sw_lanes, (kb - k0) % 32) : sw_far[turn];
                const float row_scale = kSwap ? 0.0f : sx_far[turn] * sw_now;
                fetch_scales(turn, kb + kFar < k1);
                ok = __all_sync(0xffffffffu, mbar_wait(acc_full(b), bph, ctx, 24) && (!kRingScales || mbar_wait(full(s), ph, ctx, 25)));
                if (!ok) break;
                tcgen05_fence_after();
                const uint32_t sc = half * (C::kPer * 4) + base + (kOwn ? L.own_scales + (kb - k0) * (kCols * 4) : L.scales + s * (C::kScales * 4));
                const uint32_t src = tmem + ((uint32_t)(quad * 32) << 16) + b * C::kBufCols + half * C::kPer;
                auto given_back = [&]() {
                    tcgen05_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(acc_empty(b));
                        if constexpr (kRingScales) mbar_arrive(empty(s));
                    }
                };
                if constexpr (kSwap) add_scaled_by_column(src, sc, sw_now, acc, given_back);
                else add_scaled(src, row_scale, acc, given_back);
                if (++s == a.stages) { s = 0; ph ^= 1; }
                if (++b == C::kBufs) { b = 0; bph ^= 1; }
            }
            if (!ok) break;
            if (a.cluster == 1) {
                if constexpr (kSwap) {
                    if (w0 + tl < a.n)
                        with_output(a, [&](auto* y) {
                            const int row = x0 + half * C::kPer;
                            y += row * a.ldy + w0 + tl;
#pragma unroll
                            for (int j = 0; j < C::kPer; ++j, y += a.ldy)
                                if (row + j < a.m) put(y, acc[j]);
                        });
                } else {
                    store_run<C::kPer>(a, x0 + quad * 32, w0 + half * C::kPer, acc, reinterpret_cast<float*>(gen + L.patches + warp * kPatchBytes));
                }
                continue;
            }
            // Sums of lanes [r 128/c, (r+1) 128/c) to rank r, slot of this rank: [source][four columns][lane], so that the lanes of a
            // store to a peer write side by side (100 x 4096 x 4096 10.3 us; lanes a row of the tile apart 11.6); a lane more between
            // the fours, for reads along the columns.
            const int share = 128 / a.cluster;
            const uint32_t pitch = (share + 1) * 16u, slot = pitch * (kCols / 4);
            const uint32_t xbuf = base + L.exchange;
            ok = __all_sync(0xffffffffu, wait_cluster(sums_out, xph ^ 1, ctx, 26));
            if (!ok) break;
            const uint32_t dst = peer_addr(xbuf + rank * slot + half * (C::kPer / 4) * pitch + tl % share * 16u, tl / share);
#pragma unroll
            for (int j = 0; j < C::kPer; j += 4) st_peer(dst + j / 4 * pitch, acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
            asm volatile("fence.acq_rel.cluster;" ::: "memory");
            __syncwarp();
            if (lane < a.cluster) arrive_peer(peer_addr(sums_in, lane));
            ok = __all_sync(0xffffffffu, wait_cluster(sums_in, xph, ctx, 27));
            if (!ok) break;
            xph ^= 1;
            const int groups = kCols / 4;                               // four columns of a lane at a time
            with_output(a, [&](auto* y) {
#pragma unroll 1
                for (int i = threadIdx.x; i < share * groups; i += C::kEpi * 32) {
                    const int l = kSwap ? i % share : i / groups, c = (kSwap ? i / share : i % groups) * 4;
                    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
                    for (int r = 0; r < a.cluster; ++r) {
                        const float4 v = lds_f32x4(xbuf + r * slot + c / 4 * pitch + l * 16u);
                        sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
                    }
                    const float e[4] = {sum.x, sum.y, sum.z, sum.w};
                    const int row = x0 + (kSwap ? c : rank * share + l), col = w0 + (kSwap ? rank * share + l : c);
                    auto* p = y + row * a.ldy + col;
#pragma unroll
                    for (int j = 0; j < 4; ++j, p += kSwap ? a.ldy : 1)
                        if (row + (kSwap ? j : 0) < a.m && col + (kSwap ? 0 : j) < a.n) put(p, e[j]);
                }
            });
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

// ------------------------------------------------------------------- CTA pairs
// A tile of 256 x 256 for two CTAs: 128 rows of x and half of the weight rows each, one tcgen05.mma.cta_group::2 over both (M
// 256, N 256).  A CTA fetches 32 KB a block for 128 x 256 products, where one alone would fetch 48 (4096 x 14336 x 4096: pairs 242 us,
// 128 x 256 on single CTAs 325, 128 x 128 273; the pairs' own pace without their epilogue's reads 197).  The even CTA (the leader)
// issues; its full barriers count both CTAs' bytes, its commits release stages and report buffers in both, its acc_empty counts
// both CTAs' epilogue warps.
constexpr uint32_t kLeaderMask = 0xFEFFFFFFu;        // clears the CTA-rank bit of a shared::cluster address
constexpr int kPairEpi = 8, kPairThreads = (kPairEpi + 4) * 32, kPairStages = 6, kPairBufs = 2;
constexpr uint32_t kPairHalf = 128 * 128, kPairStage = 2 * kPairHalf, kPairPatches = kPairStages * kPairStage, kPairBars = kPairPatches + kPairEpi * kPatchBytes;
constexpr uint32_t kPairMisc = kPairBars + (2 * kPairStages + 2 * kPairBufs) * 8, kPairBytes = kPairMisc + 16 + 1024;
constexpr uint32_t kPairInstrDesc = (1u << 4) | ((256u >> 3) << 17) | ((256u >> 4) << 24);

__device__ __forceinline__ void tma_load_pair_if(uint32_t lead, uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    asm volatile(
        "{\n\t.reg .pred l;\n\tsetp.ne.u32 l, %0, 0;\n\t"
        "@l cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%1], [%2, {%4, %5}], [%3];\n\t}"
        ::"r"(lead), "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar & kLeaderMask), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void umma_f8_pair_if(uint32_t lead, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, l;\n\t"
        "setp.ne.b32 p, %5, 0;\n\tsetp.ne.u32 l, %0, 0;\n\t"
        "@l tcgen05.mma.cta_group::2.kind::f8f6f4 [%1], %2, %3, %4, p;\n\t}"
        ::"r"(lead), "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(kPairInstrDesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_commit_pair_if(uint32_t lead, uint32_t bar) {     // arrives in both CTAs
    const uint16_t mask = 3;
    asm volatile(
        "{\n\t.reg .pred l;\n\tsetp.ne.u32 l, %0, 0;\n\t"
        "@l tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%1], %2;\n\t}"
        ::"r"(lead), "r"(bar), "h"(mask) : "memory");
}

__global__ void __launch_bounds__(kPairThreads, 1)
fp8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const Fp8Args a) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;        // the same offset in both CTAs
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int rank = (int)cluster_ctarank();
    auto full = [&](int s) { return base + kPairBars + s * 8; };
    auto empty = [&](int s) { return base + kPairBars + (kPairStages + s) * 8; };
    auto acc_full = [&](int b) { return base + kPairBars + (2 * kPairStages + b) * 8; };
    auto acc_empty = [&](int b) { return base + kPairBars + (2 * kPairStages + kPairBufs + b) * 8; };
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + kPairMisc + 8);
    const WaitCtx ctx{abort_flag, a.status};

    if (threadIdx.x == 0) {
        for (int s = 0; s < kPairStages; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        for (int b = 0; b < kPairBufs; ++b) { mbar_init(acc_full(b), 1); mbar_init(acc_empty(b), 2 * kPairEpi); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_proxy();
    }
    if (warp == kPairEpi + 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + kPairMisc), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    cluster_sync_all();
    tcgen05_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gen + kPairMisc);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (!a.early_weights) asm volatile("griddepcontrol.wait;" ::: "memory");
    const int step = (int)gridDim.x / 2, first = (int)blockIdx.x / 2, blocks = a.blocks;

    // 3 x 128 threads start with 168 registers each; 2 x 224 + 56 is the same sum
    if (warp >= kPairEpi) {
        give_registers<56>();
        if (warp == kPairEpi) {
            const uint32_t lead = elect_one(), lead0 = rank == 0 ? lead : 0u;
            int s = 0, ahead = 0;
            uint32_t ph = 0;
            auto weights = [&](int row, int kb, int st) {
                expect_if(lead0, full(st), 2 * kPairStage);
                tma_load_pair_if(lead, base + st * kPairStage + kPairHalf, &map_w, full(st), kb * 128, row);
            };
            // the first round of stages: weights ahead of the wait for the quantizer
            for (int item = first; item < a.items && ahead < kPairStages; item += step)
                for (int kb = 0; kb < blocks && ahead < kPairStages; ++kb) weights(item / a.x_tiles * 256 + rank * 128, kb, ahead++);
            asm volatile("griddepcontrol.wait;" ::: "memory");
            asm volatile("fence.proxy.async.global;" ::: "memory");
            bool ok = true;
            for (int item = first; item < a.items && ok; item += step) {
                const int wt = item / a.x_tiles, w_row = wt * 256 + rank * 128, x_row = (item - wt * a.x_tiles) * 256 + rank * 128;
                for (int kb = 0; kb < blocks; ++kb) {
                    if (ahead > 0) --ahead;
                    else {
                        ok = warp_wait(empty(s), ph ^ 1, ctx, 31);
                        if (!ok) break;
                        weights(w_row, kb, s);
                    }
                    tma_load_pair_if(lead, base + s * kPairStage, &map_x, full(s), kb * 128, x_row);
                    if (++s == kPairStages) { s = 0; ph ^= 1; }
                }
            }
        } else if (warp == kPairEpi + 1 && rank == 0) {
            const uint32_t lead = elect_one();
            const uint64_t a_desc = make_smem_desc(base), b_desc = make_smem_desc(base + kPairHalf);
            int s = 0, b = 0;
            uint32_t ph = 0, bph = 0;
            bool ok = true;
            for (int item = first; item < a.items && ok; item += step) {
                for (int kb = 0; kb < blocks; ++kb) {
                    ok = warp_wait(full(s), ph, ctx, 34) && warp_wait(acc_empty(b), bph ^ 1, ctx, 33);
                    if (!ok) break;
                    tcgen05_fence_after();
                    const uint64_t at = (uint64_t)(s * (kPairStage >> 4));
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        umma_f8_pair_if(lead, tmem + b * 256, a_desc + at + 2u * k, b_desc + at + 2u * k, k != 0 ? 1u : 0u);
                    umma_commit_pair_if(lead, empty(s));
                    umma_commit_pair_if(lead, acc_full(b));
                    if (++s == kPairStages) { s = 0; ph ^= 1; }
                    if (++b == kPairBufs) { b = 0; bph ^= 1; }
                }
            }
        }
    } else {
        take_registers<224>();
        asm volatile("griddepcontrol.wait;" ::: "memory");              // the scales of x are the kernel before's
        const int quad = warp & 3, half = warp >> 2;                    // lanes 32 quad .., columns 128 half ..
        const uint32_t src = tmem + ((uint32_t)(quad * 32) << 16) + half * 128;
        int b = 0;
        uint32_t bph = 0;
        bool ok = true;
        for (int item = first; item < a.items && ok; item += step) {
            const int wt = item / a.x_tiles, w0 = wt * 256 + half * 128;
            const int row = (item - wt * a.x_tiles) * 256 + rank * 128 + quad * 32 + lane;
            const float* sw = a.sw + (int64_t)min(w0 / 128, (a.n - 1) / 128) * blocks;
            const float* sx = a.sx + min(row, a.m - 1);
            float acc[128];
#pragma unroll
            for (int j = 0; j < 128; ++j) acc[j] = 0.0f;
            constexpr int kFar = 4;                                     // scales on their way, as above
            float sx_far[kFar], sw_far[kFar];
            auto fetch_scales = [&](int i, bool more) {
                if (more) {
                    sw_far[i] = __ldg(sw);
                    sx_far[i] = __ldcg(sx);
                }
                ++sw;
                sx += a.ldsx;
            };
#pragma unroll
            for (int i = 0; i < kFar; ++i) fetch_scales(i, i < blocks);
            for (int kb4 = 0; kb4 < blocks && ok; kb4 += kFar)
#pragma unroll
            for (int turn = 0; turn < kFar; ++turn) {
                const int kb = kb4 + turn;
                if (kb >= blocks) break;
                const float f = sx_far[turn] * sw_far[turn];
                fetch_scales(turn, kb + kFar < blocks);
                ok = __all_sync(0xffffffffu, mbar_wait(acc_full(b), bph, ctx, 35));
                if (!ok) break;
                tcgen05_fence_after();
                add_scaled(src + b * 256, f, acc, [&]() {
                    tcgen05_fence_before();
                    __syncwarp();
                    if (lane == 0)
                        asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(acc_empty(b) & kLeaderMask) : "memory");
                });
                if (++b == kPairBufs) { b = 0; bph ^= 1; }
            }
            if (ok) store_run(a, row - lane, w0, acc, reinterpret_cast<float*>(gen + kPairPatches + warp * kPatchBytes));
        }
    }
    // Both CTAs stay until the pair is done: the leader's MMAs read the peer's shared memory, the peer arrives on its barriers.
    tcgen05_fence_before();
    __syncthreads();
    if (*abort_flag) {
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 1000000ull) {}
    }
    cluster_sync_all();
    if (warp == kPairEpi + 1) {
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// ------------------------------------------------------------------------- host side
constexpr int kMaxDevices = 64, kMaxClusterLog = 3;

// Clusters of 1, 2, 4 and 8 CTAs that the current device runs at once, asked once per device and kernel.
struct ActiveClusters {
    std::mutex lock;
    int known[kMaxDevices][kMaxClusterLog + 1];
    bool have[kMaxDevices];
};
int active_clusters(ActiveClusters& of, const void* kernel, int threads, uint32_t smem, int (&out)[kMaxClusterLog + 1]) {
    int dev = 0;
    MIXFP4_CUDA_CHECK(cudaGetDevice(&dev));
    if (dev < 0 || dev >= kMaxDevices) return MIXFP4_E_UNSUPPORTED;
    std::lock_guard<std::mutex> guard(of.lock);
    if (!of.have[dev]) {
        MIXFP4_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        for (int c = 0; c <= kMaxClusterLog; ++c) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(1u << c);
            cfg.blockDim = dim3((unsigned)threads);
            cfg.dynamicSmemBytes = smem;
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
            of.known[dev][c] = n;
        }
        of.have[dev] = true;
    }
    for (int c = 0; c <= kMaxClusterLog; ++c) out[c] = of.known[dev][c];
    return MIXFP4_OK;
}

struct Fp8Problem {
    const uint8_t* x;
    int64_t ldx;
    const uint8_t* w;
    int64_t ldw, k;
    bool dependent;                      // the kernel before is the quantizer of x
    bool own;                            // x is dense: the product quantizes it
};

int encode_codes(EncodeTiledFn fn, CUtensorMap* map, const uint8_t* p, int64_t rows, int64_t k, int64_t ld, uint32_t box_rows) {
    cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
    cuuint32_t box[2] = {128, box_rows}, elem[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(p), dims, strides, box, elem,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? MIXFP4_OK : record_error_text("cuTensorMapEncodeTiled failed for an fp8 operand");
}

struct Fp8Choice {
    float cost = 1e30f;
    int cols = 0, cluster_log = 0, active = 0;
};
// An arrangement's cost in microseconds, up to what all have in common: rounds of items times blocks of K in a run.  Per block: what
// the weights of one SM take from HBM, or the tensor core and the epilogue; per item: filling and draining the pipeline, an
// exchange.  It picks, us on the device, * the choice:
//     1 x 1024 x 4096     clusters of 1 9.4   2 7.7    4 6.1    8 5.7*
//     1 x 4096 x 4096                1 9.6    2 8.9    4 8.1*   8 12.8
//    16 x 4096 x 14336               1 27.2   2 17.8   4 14.9*  8 21.2
//    48 x 14336 x 4096               1 16.0*  2 21.4   4 28.2
//   100 x 4096 x 4096    wide        1 12.6   2 11.4   4 10.3*  pairs 20.9
//   512 x 4096 x 4096                1 13.8*  2 21.0            pairs 21.7
//   333 x 1000 x 1500                1 9.3    2 7.9    4 7.8*   pairs 14.8
//   300 x 14337 x 4096               1 42.2*  2 48.9            pairs 49.7
//  1024 x 4096 x 4096                1 24.0   2 40.7            pairs 22.3*
//  2048 x 4096 x 4096                1 43.8   2 66.5            pairs 40.4*
template <int kCols, bool kSwap, bool kOwn>
int consider(const Fp8Args& a, Fp8Choice& best) {
    static ActiveClusters active;
    int clusters[kMaxClusterLog + 1];
    const auto kernel = fp8_gemm_kernel<kCols, kSwap, kOwn>;
    if (const int rc = active_clusters(active, reinterpret_cast<const void*>(kernel), Fp8Cfg<kCols, kSwap, kOwn>::kThreads, kSmemMax, clusters))
        return rc;
    const int64_t lanes = kSwap ? a.n : a.m, cols = kSwap ? a.m : a.n;
    const int64_t items = (lanes + 127) / 128 * ((cols + kCols - 1) / kCols);
    for (int log = 0; log <= kMaxClusterLog; ++log) {
        const int c = 1 << log;
        if (clusters[log] < 1 || c > a.blocks) continue;
        const int64_t rounds = (items + clusters[log] - 1) / clusters[log];
        const float block = kSwap ? 0.38f : 0.30f;
        const float cost = (float)rounds * (block * (float)((a.blocks + c - 1) / c) + (c > 1 ? 1.5f : 0.7f));
        if (cost < best.cost) best = Fp8Choice{cost, kCols, log, clusters[log]};
    }
    return MIXFP4_OK;
}
int consider_pair(const Fp8Args& a, Fp8Choice& best) {
    static ActiveClusters active;
    int clusters[kMaxClusterLog + 1];
    if (const int rc = active_clusters(active, reinterpret_cast<const void*>(fp8_pair_kernel), kPairThreads, kPairBytes, clusters)) return rc;
    if (clusters[1] < 1) return MIXFP4_OK;
    const int64_t items = (int64_t)((a.m + 255) / 256) * ((a.n + 255) / 256), rounds = (items + clusters[1] - 1) / clusters[1];
    const float cost = (float)rounds * (0.36f * (float)a.blocks + (a.y_vec ? 1.5f : 5.5f));     // stores through the patches show
    if (cost < best.cost) best = Fp8Choice{cost, 256, 1, clusters[1]};
    return MIXFP4_OK;
}

int launch_clusters(const void* kernel, int cluster, int n, int threads, uint32_t smem, const Fp8Problem& p, const CUtensorMap& map_x,
                    const CUtensorMap& map_w, const Fp8Args& a, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(n * cluster));
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    void* args[] = {const_cast<CUtensorMap*>(&map_x), const_cast<CUtensorMap*>(&map_w), const_cast<Fp8Args*>(&a)};
    MIXFP4_CUDA_CHECK(cudaLaunchKernelExC(&cfg, kernel, args));
    return check_launch("fp8 product");
}

// Maps with boxes of x_box rows of x and w_box rows of the weight; items of `tile` rows each.
int launch_fp8(Fp8Args a, const Fp8Problem& p, const Fp8Choice& c, int x_box, int w_box, int x_tile, int w_tile, const void* kernel,
               int threads, uint32_t smem, cudaStream_t st) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return record_error_text("cuTensorMapEncodeTiled is not available");
    a.early_weights = p.dependent;
    CUtensorMap map_x, map_w;
    if (const int rc = encode_codes(fn, &map_w, p.w, a.n, p.k, p.ldw, (uint32_t)w_box)) return rc;
    if (p.own) map_x = map_w;                                           // not used
    else if (const int rc = encode_codes(fn, &map_x, p.x, a.m, p.k, p.ldx, (uint32_t)x_box)) return rc;
    a.x_tiles = (a.m + x_tile - 1) / x_tile;
    const int64_t items = (int64_t)a.x_tiles * ((a.n + w_tile - 1) / w_tile);
    if (items > 0x3fffffff) return MIXFP4_E_SHAPE;
    a.items = (int)items;
    return launch_clusters(kernel, 1 << c.cluster_log, a.items < c.active ? a.items : c.active, threads, smem, p, map_x, map_w, a, st);
}
template <int kCols, bool kSwap, bool kOwn>
int launch_single(Fp8Args a, const Fp8Problem& p, const Fp8Choice& c, cudaStream_t st) {
    a.cluster = 1 << c.cluster_log;
    a.stages = kMaxStages;
    while (fp8_layout<kCols, kSwap, kOwn>(a.stages, a.cluster, a.blocks, a.y_vec).bytes > kSmemMax) --a.stages;
    const auto kernel = fp8_gemm_kernel<kCols, kSwap, kOwn>;
    constexpr int kX = kSwap ? kCols : 128, kW = kSwap ? 128 : kCols;
    return launch_fp8(a, p, c, kX, kW, kX, kW, reinterpret_cast<const void*>(kernel), Fp8Cfg<kCols, kSwap, kOwn>::kThreads,
                      fp8_layout<kCols, kSwap, kOwn>(a.stages, a.cluster, a.blocks, a.y_vec).bytes, st);
}
template <int kCols, bool kOwn>
int few_rows(const Fp8Args& a, const Fp8Problem& p, cudaStream_t st) {
    Fp8Choice best;
    if (const int rc = consider<kCols, true, kOwn>(a, best)) return rc;
    return best.cols ? launch_single<kCols, true, kOwn>(a, p, best, st) : MIXFP4_E_UNSUPPORTED;
}

int fp8_gemm(const Fp8Args& a, const Fp8Problem& p, cudaStream_t st) {
    if (a.m <= 16) return p.own ? few_rows<16, true>(a, p, st) : few_rows<16, false>(a, p, st);
    if (a.m <= 32) return p.own ? few_rows<32, true>(a, p, st) : few_rows<32, false>(a, p, st);
    if (a.m <= 64) return p.own ? few_rows<64, true>(a, p, st) : few_rows<64, false>(a, p, st);
    Fp8Choice best;
    if (const int rc = consider<128, false, false>(a, best)) return rc;
    if (const int rc = consider_pair(a, best)) return rc;
    switch (best.cols) {
        case 128: return launch_single<128, false, false>(a, p, best, st);
        case 256: return launch_fp8(a, p, best, 128, 128, 256, 256, reinterpret_cast<const void*>(fp8_pair_kernel), kPairThreads, kPairBytes, st);
        default: return MIXFP4_E_UNSUPPORTED;
    }
}

constexpr int64_t kMaxSide = 0x7fffff00;

int check_product(const uint8_t* w, int64_t ldw, const float* sw, int64_t m, int64_t n, int64_t k, const void* y, int out_dtype,
                  int64_t ldy) {
    if (!w || !sw || !y) return MIXFP4_E_NULL;
    if (out_dtype != MIXFP4_BF16 && out_dtype != MIXFP4_F16 && out_dtype != MIXFP4_F32) return MIXFP4_E_DTYPE;
    if (m <= 0 || n <= 0 || k <= 0 || m > kMaxSide || n > kMaxSide || k > kMaxSide || ldw < k || ldy < n) return MIXFP4_E_SHAPE;
    if (!aligned(w, 16) || ldw % 16 != 0 || !aligned(sw, 4) || !aligned(y, fp8_elem_bytes(out_dtype))) return MIXFP4_E_ALIGN;
    return MIXFP4_OK;
}

Fp8Args make_args(const float* sx, int64_t ldsx, const float* sw, int64_t m, int64_t n, int64_t k, void* y, int out_dtype,
                  int64_t ldy, int* status) {
    Fp8Args a = {};
    a.sx = sx; a.sw = sw; a.y = y; a.ldsx = ldsx; a.ldy = ldy;
    a.m = (int)m; a.n = (int)n; a.k = (int)k; a.blocks = (int)((k + kFp8Block - 1) / kFp8Block);
    a.out_dtype = out_dtype; a.status = status;
    a.y_vec = aligned(y, 32) && ldy * fp8_elem_bytes(out_dtype) % 32 == 0 && n * fp8_elem_bytes(out_dtype) % 32 == 0;
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
    return fp8_gemm(make_args(x_scales, lds, w_scales, m, n, k, y, out_dtype, ldy, status), Fp8Problem{x, ldx, w, ldw, k, false, false},
                    static_cast<cudaStream_t>(stream));
}

extern "C" int64_t mixfp4_fp8_workspace_bytes(int64_t m, int64_t k) {
    if (m <= 0 || k <= 0 || fp8_quantizes_itself(m, k)) return 0;
    const int64_t kp = padded_k(k);
    return (m * kp + 15) / 16 * 16 + fp8_scale_rows(m) * (kp / kFp8Block) * 4;
}

extern "C" int mixfp4_fp8_linear(const void* x, int dtype, int64_t m, int64_t ldx, const uint8_t* w, int64_t ldw,
                                 const float* w_scales, int64_t n, int64_t k, void* y, int out_dtype, int64_t ldy,
                                 void* workspace, int64_t workspace_bytes, int* status, void* stream) {
    if (!x) return MIXFP4_E_NULL;
    if (const int rc = check_product(w, ldw, w_scales, m, n, k, y, out_dtype, ldy)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Fp8Args a = make_args(nullptr, 0, w_scales, m, n, k, y, out_dtype, ldy, status);
    if (fp8_quantizes_itself(m, k)) {
        if (dtype != MIXFP4_BF16 && dtype != MIXFP4_F16 && dtype != MIXFP4_F32) return MIXFP4_E_DTYPE;
        if (ldx < k) return MIXFP4_E_SHAPE;
        if (!aligned(x, fp8_elem_bytes(dtype))) return MIXFP4_E_ALIGN;
        a.x = x; a.ldx = ldx; a.x_dtype = dtype;
        a.x_vec = aligned(x, 16) && ldx * fp8_elem_bytes(dtype) % 16 == 0;
        return fp8_gemm(a, Fp8Problem{nullptr, 0, w, ldw, k, false, true}, st);
    }
    if (!workspace || workspace_bytes < mixfp4_fp8_workspace_bytes(m, k)) return MIXFP4_E_WORKSPACE;
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    const int64_t kp = padded_k(k), lds = fp8_scale_rows(m);
    float* scales = reinterpret_cast<float*>(codes + (m * kp + 15) / 16 * 16);
    if (const int rc = fp8_check_rows(x, dtype, m, k, ldx, codes, kp, scales, lds)) return rc;
    if (const int rc = fp8_quantize_rows(x, dtype, m, k, ldx, codes, kp, scales, lds, st)) return rc;
    a.sx = scales;
    a.ldsx = lds;
    return fp8_gemm(a, Fp8Problem{codes, kp, w, ldw, k, true, false}, st);
}

// One token a row from logits: temperature, top-k, top-p, min-p, and a random number that the caller brings.
//   w_i   = exp((x_i - max x) / T)                      T = 0: the first of the largest logits
//   order   by value, largest first, equal values by index
//   kept    the first k; of those the shortest run whose weights reach p times theirs; of those every w_i >= min_p
//   token   the first index, in the vocabulary's order, at which the kept weights add up to more than u times their sum
//
// Nothing is sorted.  A cluster of CTAs holds a row in shared memory (one HBM read) and narrows the cut down by
// histograms: 512 bins of equal width over the logits that have a weight at all, then 512 bins of the keys (a monotone
// integer of the value) in the bin that the cut falls in, until that bin is one value; equal values are counted off by
// index.  Every CTA adds the cluster's histograms up for itself: one cluster barrier a step, none to hand a result round.
// Where the first histogram leaves at most 256 candidates for a top-k (the usual settings), one CTA takes them all and
// compares each with each.
//
// Sums.  The set of kept tokens and the token itself hang on comparisons of sums over the vocabulary, so weights are
// integers: W = round(2^44 w), w in double precision.  Integer sums do not depend on their order, so neither do the
// results, and 2^19 of them fit 63 bits.  A weight below 2^-45 of the largest counts as none.  Shared memory adds 32-bit
// words only, so a bin's sum is two words, and whoever overflows the low one adds the carry to the high one: one addition
// for all but the largest few thousandths of the weights.
//
// What bounds it.  A row of a small batch takes a dozen dependent steps (passes over shared memory, cluster barriers), and code
// that runs once or twice: instruction fetch counts, so every pass has one copy (unrolled passes, 86 KB of code, took 70 us for
// one row of 128256 logits with top-k and top-p; this takes 12 to 13).  Large batches without a top-k (64 mixed rows of 128256 57 to 61
// us): instruction issue, 166 thread instructions a logit of a top-p, of which the weights are about half.  They are computed in fp64 for
// every logit, once for the histogram and once for the sums (a pass with all of them 14 us for the 64 K elements of an SM), although
// logits of 16 bits have a few thousand values: fewer are possible.  The rest are the histogram's additions in shared memory.
// Measured and not kept: lists of a warp's few elements of interest, sorting the candidates, sums of what a top-p cannot reach
// beside the histogram, a first histogram over the topmost bf16 keys instead of equal widths (each more code than it saved time:
// 64 mixed rows 4 to 14 us more).

#include <float.h>

#include "common.cuh"

namespace mixfp4 {
namespace {

constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32, kBinsLog = 9, kBins = 1 << kBinsLog;
static_assert(kBins == kSampleThreads, "a thread owns a bin");
constexpr int kMaxRanks = 8;
constexpr int64_t kMaxSlice = 65536, kMaxVocab = kMaxRanks * kMaxSlice - 128;
constexpr int kOneLog = 44;
constexpr double kOne = 17592186044416.0;                // 2^44
constexpr int kSteps = 64;                               // of an octave, in the table of the exponential
constexpr float kSpan = 31.5f;                           // weights vanish at 45 ln 2 = 31.2
// Below 2^-160 the smallest difference of two fp32 numbers, 2^-149, is 2^11 temperatures: only the largest logits have a weight, at
// this one as at any smaller, whose reciprocal need not be finite.
constexpr double kLeastTemperature = 0x1p-160;
constexpr float kNegInf = -__builtin_huge_valf();

typedef unsigned long long u64;

// Ordinary loads: what they read may have been written while this kernel was already running.
template <typename T>
__device__ __forceinline__ T ld_global(const T* p) { return *p; }

template <typename T, typename All>
struct Setting {                                         // a value for each row, or one for all
    const T* each;
    All all;
    __device__ All of(int64_t row) const { return each ? (All)ld_global(each + row) : all; }
};
struct SampleArgs {
    const void* logits;
    int64_t ld;
    int vocab, ranks;
    const float* uniform;
    Setting<float, double> temperature, top_p, min_p;
    Setting<int, int> top_k;
    long long* token;
    float* logprob;                                      // optional
};

template <typename T>
struct Row;                                              // keys: larger value, larger key; zero of either sign is one value
template <>
struct Row<float> {
    static __device__ uint32_t key(float x) {
        const uint32_t b = __float_as_uint(x + 0.0f);
        return b & 0x80000000u ? ~b : b | 0x80000000u;
    }
};
template <typename T>
struct Row {
    static __device__ uint32_t key(float x) {
        const T t = Elem<T>::round(x + 0.0f);
        const uint32_t b = *reinterpret_cast<const uint16_t*>(&t);
        return b & 0x8000u ? b ^ 0xffffu : b | 0x8000u;
    }
};

// What the CTAs of a cluster tell one another; two sets in turn, so that a set is written again only after a barrier that
// every reader of it has passed.
struct Slots {
    float largest[kMaxRanks], least_of_groups[kMaxRanks];
    uint32_t count[kMaxRanks];
    u64 mass[kMaxRanks];
};
constexpr uint32_t kFew = 256;
struct Shared {
    u64 mass[2][kBins];                                  // per bin, as two words
    uint32_t count[2][kBins];
    double octave[kSteps];                               // 2^(j / kSteps)
    u64 few[kFew], few_weight[kFew];                     // candidates: key, then the index turned round
    Slots slots[2];
    u64 warp_mass[kSampleWarps];
    uint32_t warp_count[kSampleWarps];
    float warp_max[kSampleWarps], warp_least[kSampleWarps];
    u64 found_before;
    uint32_t found_bin, found_size, few_count;
};

__device__ __forceinline__ uint32_t shared_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t of_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ uint32_t ld_rank32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ u64 ld_rank64(uint32_t addr) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void st_rank32(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void st_rank64(uint32_t addr, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t add_rank32(uint32_t addr, uint32_t v) {
    uint32_t was;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(was) : "r"(addr), "r"(v) : "memory");
    return was;
}
// The cluster's first barrier in two halves: no CTA touches a peer's shared memory before the peer is known to run, which
// nothing but a barrier of the cluster tells.  Begun at the kernel's start, ended ahead of the first store to a peer: the row's
// loads lie between.
__device__ __forceinline__ void started(int ranks) {
    if (ranks > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void all_started(int ranks) {
    __syncwarp();
    if (ranks > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void meet(int ranks) {        // all threads of the cluster; writes before are seen after
    __syncwarp();
    if (ranks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    else __syncthreads();
}
// Sum over this lane and those before it.
__device__ __noinline__ u64 add_up(u64 v) {
#pragma unroll 1
    for (int d = 1; d < 32; d *= 2) {
        const u64 o = __shfl_up_sync(0xffffffffu, v, d);
        if ((int)(threadIdx.x & 31) >= d) v += o;
    }
    return v;
}
// A prefix of the sorted row: everything above `value`, and the first `ties` of those equal to it.
struct Cut {
    float value;
    uint32_t ties, equal;                                // equal: how many there are
};

// Out of line: once a row, and long.
__device__ __noinline__ double log_of(u64 total) { return log((double)total / kOne); }
__device__ __noinline__ double octave_step(int j) { return exp2((double)j / kSteps); }
// 16 bytes at a row's end: the elements [0, n) of it from index i, -inf around them.
template <typename T>
__device__ __noinline__ uint4 fetch_end(const T* row, int i, int n) {
    uint4 u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int j = 0; j < 16 / (int)sizeof(T); ++j) e[j] = i + j >= 0 && i + j < n ? row[i + j] : Elem<T>::round(kNegInf);
    return u;
}

template <typename T, bool kResident>
struct Sampler {
    static constexpr int kPer = 16 / sizeof(T);          // elements of a granule: 16 aligned bytes
    const SampleArgs& a;
    Shared& s;
    uint4* held;                                         // kResident: the slice's granules
    const T* row;
    int skew, first, c0, c1;                             // first granule of this CTA; this warp's quads
    int warp, lane, rank, hist_turn;
    float largest, floor_x;                              // below floor_x nothing has a weight
    double top;                                          // the largest, if that is finite
    double inv_t, steps_t;                               // 1 / T, kSteps log2(e) / T
    float bin_scale;

    // Granule g holds the indices g * kPer - skew ..: granules start on 16-byte boundaries, the row need not.  NaN and what
    // lies outside the row count as -inf (the larger of NaN and a number is the number).
    __device__ uint4 fetch(int g) const {
        const int i = g * kPer - skew;
        uint4 u = i >= 0 && i + kPer <= a.vocab ? ld_global(reinterpret_cast<const uint4*>(row + i)) : fetch_end(row, i, a.vocab);
        if constexpr (sizeof(T) == 4) {
            float* e = reinterpret_cast<float*>(&u);
#pragma unroll
            for (int j = 0; j < kPer; ++j) e[j] = fmaxf(e[j], kNegInf);
        } else {
            auto clean = [](uint32_t w) {
                if constexpr (Elem<T>::kDtype == MIXFP4_BF16) {
                    const __nv_bfloat162 c = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&w), __float2bfloat162_rn(kNegInf));
                    return *reinterpret_cast<const uint32_t*>(&c);
                } else {
                    const __half2 c = __hmax2(*reinterpret_cast<__half2*>(&w), __float2half2_rn(kNegInf));
                    return *reinterpret_cast<const uint32_t*>(&c);
                }
            };
            u = make_uint4(clean(u.x), clean(u.y), clean(u.z), clean(u.w));
        }
        return u;
    }
    // Quad c, four elements from index 4 c - skew.  A warp's pass takes a quad a lane at a time: code for four elements is short,
    // and four weights at once hide the latency of their operations.
    __device__ void get(int c, float (&x)[4]) const {
        constexpr int kQuads = kPer / 4;
        const T* e;
        uint4 u;
        if constexpr (kResident) {
            if constexpr (sizeof(T) == 4) {
                u = held[c - first];
            } else {
                const uint2 half = reinterpret_cast<const uint2*>(held)[c - first * kQuads];
                u.x = half.x; u.y = half.y;
            }
            e = reinterpret_cast<const T*>(&u);
        } else {
            u = fetch(c / kQuads);
            if (kQuads > 1 && c % kQuads) { u.x = u.z; u.y = u.w; }
            e = reinterpret_cast<const T*>(&u);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = Elem<T>::load(e + j);
    }

    // 2^44 w for x >= floor_x: y = log2(w) in steps of an octave, rounded to a whole step by an addition that leaves no fraction
    // bits; the rest of at most half a step by its series (the next term is 4e-14), the step from the table, the octave into
    // the exponent.  To the nearest integer: below 2^52, an addition of 2^52 leaves it in the low bits.
    __device__ u64 weight(float x) const {
        const double y = ((double)fminf(x, FLT_MAX) - top) * steps_t;
        const double shifted = y + 0x1.8p52;
        const int i = __double2loint(shifted);
        const double r = y - (shifted - 0x1.8p52);
        constexpr double c = 0.69314718055994530942 / kSteps;
        double e = c * c * c * c / 24;
        e = fma(e, r, c * c * c / 6);
        e = fma(e, r, c * c / 2);
        e = fma(e, r, c);
        e = fma(e, r, 1.0) * s.octave[i & (kSteps - 1)];
        static_assert(kSteps == 1 << 6, "the shift below");
        e = __hiloint2double(__double2hiint(e) + (((i >> 6) + kOneLog) << 20), __double2loint(e));
        return (u64)__double_as_longlong(e + 0x1p52) & 0xfffffffffffffull;
    }
    // Bin of equal width, rising as the value falls (rounded operations are monotone).  The conversion takes what is too
    // large to its own largest value, and infinity less infinity, a NaN, to 0.
    __device__ uint32_t linear(float x) const { return min(__float2uint_rz((largest - x) * bin_scale), (uint32_t)kBins - 1); }

    __device__ void clear(int which) {
        s.count[which][threadIdx.x] = 0;
        s.mass[which][threadIdx.x] = 0;
    }
    __device__ void put(uint32_t bin, bool counted, u64 w) {
        if (counted) atomicAdd(&s.count[hist_turn][bin], 1u);
        if (w) {
            uint32_t* words = reinterpret_cast<uint32_t*>(&s.mass[hist_turn][bin]);
            const uint32_t low = (uint32_t)w, was = atomicAdd(words, low);
            const uint32_t high = (uint32_t)(w >> 32) + (was + low < was);
            if (high) atomicAdd(words + 1, high);
        }
    }
    // The count or the mass that a cut by mass has to reach, out of `total`.
    __device__ static u64 share_of(double p, u64 total) {
        const double want = ceil(fmax(p, 0.0) * (double)total);
        return want < 1.0 ? 1ull : min((u64)want, total);
    }
    // The cluster's histogram, a bin a thread, and the first bin at which the running count (or mass) reaches the goal: into
    // s.found_*: the bin (kBins: none), what lies before it, its count.  goal 0: the share p of the mass without `out` of it.
    __device__ u64 find(bool by_mass, u64 before, u64 goal, double p, u64 out) {
        meet(a.ranks);
        clear(hist_turn ^ 1);                            // every CTA is past its reads of that one
        u64 own = 0;
        const uint32_t at_count = shared_addr(&s.count[hist_turn][threadIdx.x]), at_mass = shared_addr(&s.mass[hist_turn][threadIdx.x]);
        u64 h[kMaxRanks];                                // all of them asked for before the first is used
#pragma unroll
        for (int r = 0; r < kMaxRanks; ++r) {
            h[r] = 0;
            if (r < a.ranks) {
                if (by_mass) h[r] = ld_rank64(of_rank(at_mass, r));
                else h[r] = ld_rank32(of_rank(at_count, r));
            }
        }
#pragma unroll
        for (int r = 0; r < kMaxRanks; ++r) own += h[r];
        const int turn = hist_turn;
        hist_turn ^= 1;
        const u64 up = add_up(own);
        if (lane == 31) s.warp_mass[warp] = up;
        if (threadIdx.x == 0) s.found_bin = kBins;
        __syncthreads();
        u64 ahead = add_up(lane < kSampleWarps ? s.warp_mass[lane] : 0);      // the warps' sums, added up by every warp
        if (goal == 0) goal = share_of(p, before + __shfl_sync(0xffffffffu, ahead, 31) - out);
        ahead = __shfl_sync(0xffffffffu, ahead, warp > 0 ? warp - 1 : 0);
        const u64 hi = before + (warp > 0 ? ahead : 0) + up, lo = hi - own;
        if (lo < goal && goal <= hi) {
            uint32_t n = (uint32_t)own;
            if (by_mass) {
                n = 0;
#pragma unroll 1
                for (int r = 0; r < a.ranks; ++r) n += ld_rank32(of_rank(shared_addr(&s.count[turn][threadIdx.x]), r));
            }
            s.found_bin = threadIdx.x;
            s.found_before = lo;
            s.found_size = n;
        }
        __syncthreads();
        return goal;
    }
    __device__ static float value_of(uint32_t key) {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
        } else {
            const uint16_t b = (uint16_t)(key & 0x8000u ? key & 0x7fffu : key ^ 0xffffu);
            return Elem<T>::load(reinterpret_cast<const T*>(&b));
        }
    }
    __device__ u64 block_sum(u64 v) {
#pragma unroll
        for (int d = 16; d > 0; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
        if (lane == 0) s.warp_mass[warp] = v;
        __syncthreads();
        u64 all = lane < kSampleWarps ? s.warp_mass[lane] : 0;
#pragma unroll
        for (int d = 16; d > 0; d /= 2) all += __shfl_xor_sync(0xffffffffu, all, d);
        __syncthreads();
        return all;
    }
    __device__ u64 target_of(double u, u64 total) const {
        const double want = u > 0.0 ? u * (double)total : 0.0;
        return want < (double)total ? min((u64)want, total - 1) : total - 1;
    }
    __device__ void answer(int64_t r, int index, float x, bool greedy, u64 total) const {
        a.token[r] = index;
        if (a.logprob) a.logprob[r] = greedy ? 0.0f : (float)((x == largest ? 0.0 : ((double)x - top) * inv_t) - log_of(total));
    }

    // At most kFew candidates, the elements from `from` on in the linear bins up to `bin`, as they were counted: rank 0 takes them all, two threads to each, and
    // adds up what goes before it, by value and then, of the kept ones, by index.
    __device__ void choose_from_few(int64_t r, float from, uint32_t bin, uint32_t k, double p, u64 lowest, double u) {
        const uint32_t count_at = of_rank(shared_addr(&s.few_count), 0), few_at = of_rank(shared_addr(s.few), 0);
#pragma unroll 1
        for (int c = c0 + lane; c < c1; c += 32) {
            float x[4];
            get(c, x);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!(x[j] >= from) || linear(x[j]) > bin) continue;
                const uint32_t at = add_rank32(count_at, 1), index = (uint32_t)(c * 4 + j - skew);
                if (at < kFew) st_rank64(few_at + at * 8, (u64)Row<T>::key(x[j]) << 32 | (uint32_t)~index);
            }
        }
        constexpr uint32_t kParts = kSampleThreads / kFew;
        meet(a.ranks);
        if (rank != 0) return;
        const uint32_t n = min(s.few_count, kFew), i = threadIdx.x / kParts, part = threadIdx.x % kParts;
        if (threadIdx.x < n) s.few_weight[threadIdx.x] = weight(value_of((uint32_t)(s.few[threadIdx.x] >> 32)));
        __syncthreads();
        const u64 order = i < n ? s.few[i] : 0, w = i < n ? s.few_weight[i] : 0;
        const float x = value_of((uint32_t)(order >> 32));
        auto join = [](u64 v) {
#pragma unroll
            for (int d = 1; d < (int)kParts; d *= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
            return v;
        };
        u64 mass = 0;
        uint32_t ahead = 0;
#pragma unroll 2
        for (uint32_t j = part; j < n; j += kParts) {
            const bool before = s.few[j] > order;
            mass += before ? s.few_weight[j] : 0;
            ahead += before;
        }
        mass = join(mass);
        ahead = (uint32_t)join(ahead);
        bool kept = i < n && ahead < k;
        const u64 of_k = block_sum(kept && part == 0 ? w : 0);
        kept = kept && (!(p < 1.0) || mass < share_of(p, of_k)) && w >= lowest;
        if (part == 0 && i < n) s.few_weight[i] = kept ? w : 0;
        const u64 total = block_sum(kept && part == 0 ? w : 0), goal = target_of(u, total);
        u64 at = 0;
#pragma unroll 2
        for (uint32_t j = part; j < n; j += kParts) at += (uint32_t)s.few[j] > (uint32_t)order ? s.few_weight[j] : 0;      // a lower index
        at = join(at);
        if (part == 0 && kept && goal >= at && goal < at + w) answer(r, (int)~(uint32_t)order, x, false, total);
    }

    __device__ void run(int64_t r) {
        const int ranks = a.ranks;
        started(ranks);
        // the row's granules, the cluster's share, the warps' shares: contiguous, so that indices rise with rank, warp, lane
        const int granules = (a.vocab + skew + kPer - 1) / kPer, per_rank = (granules + ranks - 1) / ranks;
        first = min(rank * per_rank, granules);
        const int end = min(first + per_rank, granules), per_warp = (end - first + kSampleWarps - 1) / kSampleWarps;
        const int g0 = min(first + warp * per_warp, end), g1 = min(g0 + per_warp, end);
        c0 = g0 * (kPer / 4);
        c1 = g1 * (kPer / 4);
        hist_turn = 0;
        clear(0);
        clear(1);
        if (threadIdx.x < kSteps) s.octave[threadIdx.x] = octave_step(threadIdx.x);
        if (threadIdx.x == 0) s.few_count = 0;
        // Nothing of the caller's has been read so far: up to here the kernel runs under the tail of the one before.
        asm volatile("griddepcontrol.wait;" ::: "memory");
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        const double t = a.temperature.of(r), p = a.top_p.of(r), u = (double)ld_global(a.uniform + r);
        const int k = a.top_k.of(r);
        const bool greedy = !(t > 0.0);
        const u64 lowest = greedy ? 0 : (u64)__double2ll_rn(fmin(fmax(a.min_p.of(r), 0.0), 1.0) * kOne);

        float most = kNegInf;
        constexpr int kAhead = 4;                        // granules of a lane on their way at once
        // Past the warp's share a lane takes its own last granule once more: lanes' maxima are of elements of their own.
        const int own_last = g0 + lane + (g1 - 1 - g0 - lane) / 32 * 32;
#pragma unroll 1
        for (int g = g0 + lane; g < g1; g += 32 * kAhead) {
            uint4 v[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) v[i] = fetch(min(g + 32 * i, own_last));
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                if constexpr (kResident) held[min(g + 32 * i, own_last) - first] = v[i];
#pragma unroll
                for (int j = 0; j < kPer; ++j) most = fmaxf(most, Elem<T>::load(reinterpret_cast<const T*>(&v[i]) + j));
            }
        }
        // The largest; and the least of the maxima of so many groups of lanes that there are k of them at least.  No two groups have
        // an element in common, so no fewer than k elements reach it, and a top-k need not look below.
        const int groups = kSampleWarps * ranks;
        float least = k <= groups * 32 ? most : kNegInf;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
            if (groups * (16 / d) >= k) least = most;
        }
#pragma unroll
        for (int d = 1; d < 32; d *= 2) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, d));
        if (lane == 0) {
            s.warp_max[warp] = most;
            s.warp_least[warp] = least;
        }
        all_started(ranks);
        __syncthreads();
        if (warp == 0) {
            most = s.warp_max[lane % kSampleWarps];
            least = s.warp_least[lane % kSampleWarps];
#pragma unroll
            for (int d = 16; d > 0; d /= 2) {
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
                least = fminf(least, __shfl_xor_sync(0xffffffffu, least, d));
            }
            if (lane < ranks) {
                st_rank32(of_rank(shared_addr(&s.slots[0].largest[rank]), lane), __float_as_uint(most));
                st_rank32(of_rank(shared_addr(&s.slots[0].least_of_groups[rank]), lane), __float_as_uint(least));
            }
        }
        meet(ranks);
        largest = kNegInf;
        float reached_by_k = -kNegInf;
#pragma unroll 1
        for (int q = 0; q < ranks; ++q) {
            largest = fmaxf(largest, s.slots[0].largest[q]);
            reached_by_k = fminf(reached_by_k, s.slots[0].least_of_groups[q]);
        }
        top = (double)fminf(largest, FLT_MAX);
        if (largest == kNegInf) {                        // nothing to choose from
            if (rank == 0 && threadIdx.x == 0) {
                a.token[r] = -1;
                if (a.logprob) a.logprob[r] = kNegInf;
            }
            return;
        }
        inv_t = greedy ? 1.0 : 1.0 / t;
        steps_t = inv_t * (kSteps * 1.4426950408889634074);
        bin_scale = (float)fmin((double)kBins / kSpan * inv_t, 1e38);
        floor_x = greedy || isinf(largest) ? largest : fmaxf((float)(top - kSpan * t), -FLT_MAX);

        // The cut, first by count, then by mass within what that kept; each by linear bins, then by keys in the bin found.
        Cut cut{floor_x, 0, 0};                          // everything
        if (greedy) cut = Cut{largest, 1, 0xffffffffu};
#pragma unroll 1
        for (int stage = k > 0 && k < a.vocab ? 0 : 1; stage < (greedy ? 0 : p < 1.0 ? 2 : 1); ++stage) {
            const bool by_mass = stage == 1;
            // the mass of the equal values that the cut by count leaves out
            const u64 out = by_mass && cut.equal > cut.ties ? (u64)(cut.equal - cut.ties) * weight(cut.value) : 0;
            const float from = by_mass ? cut.value : fmaxf(cut.value, reached_by_k);
            u64 goal = by_mass ? 0 : (u64)k, before = 0;
            uint32_t bin = 0, lo = 0, hi = 0;
#pragma unroll 1
            for (int level = 0; level < 5; ++level) {    // 32 bits of a key, 9 a level
                const uint32_t span = hi - lo;
                const int shift = span < (uint32_t)kBins ? 0 : 32 - kBinsLog - __clz(span);
#pragma unroll 1
                for (int c = c0 + lane; c < c1; c += 32) {
                    float x[4];
                    get(c, x);
                    if (!(x[0] >= from || x[1] >= from || x[2] >= from || x[3] >= from)) continue;
                    if (level == 0) {                    // most of them count: four at once
                        u64 w[4] = {};
                        if (by_mass) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) w[j] = weight(fmaxf(x[j], floor_x));
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (x[j] >= from) put(linear(x[j]), !by_mass, w[j]);
                        continue;
                    }
                    uint32_t hits = 0;                   // few do: one at a time
#pragma unroll
                    for (int j = 0; j < 4; ++j) hits |= x[j] >= from && linear(x[j]) == bin ? 1u << j : 0u;
#pragma unroll 1
                    for (; hits; hits &= hits - 1) {
                        const float v = hits & 1 ? x[0] : hits & 2 ? x[1] : hits & 4 ? x[2] : x[3];
                        const uint32_t key = Row<T>::key(v);
                        if (key >= lo && key <= hi) put((hi - key) >> shift, true, by_mass ? weight(v) : 0);
                    }
                }
                goal = find(by_mass, before, goal, p, out);
                const uint32_t b = s.found_bin;
                before = s.found_before;
                const uint32_t size = s.found_size;
                if (b == (uint32_t)kBins) break;         // fewer than k have a weight: all of them stay
                if (level == 0) {
                    if (!by_mass && before + size <= kFew) return choose_from_few(r, from, b, (uint32_t)k, p, lowest, u);
                    // keys that the bin can hold: its edges, moved out by more than rounding moved them
                    bin = b;
                    const float width = 1.0f / bin_scale;
                    const float x_hi = largest - (float)bin * width * 0.9999f, x_lo = largest - ((float)bin + 1.0f) * width * 1.0001f;
                    // (an edge that overflows bounds nothing: differences and temperatures near the largest float)
                    hi = Row<T>::key(bin == 0 || !(x_hi > -FLT_MAX) ? largest : fminf(x_hi + fabsf(largest) * 1e-6f, largest));
                    lo = isinf(largest) ? hi : Row<T>::key(cut.value);
                    if (bin < (uint32_t)kBins - 1) lo = max(lo, Row<T>::key(x_lo - fabsf(largest) * 1e-6f));
                } else {
                    hi -= b << shift;
                    if (shift == 0) {
                        const u64 w = by_mass ? weight(value_of(hi)) : 1;
                        cut = Cut{value_of(hi), (uint32_t)((goal - before + w - 1) / w), size};      // equal weights: as many as are needed
                        break;
                    }
                    if (hi - lo >= 1u << shift) lo = hi - (1u << shift) + 1;
                }
                __syncthreads();                         // found_* has been read
            }
            __syncthreads();
        }

        // equal values before this warp's
        uint32_t ties_before = 0, ties_here = 0;
        const bool some = cut.ties < cut.equal;          // not all of them are kept
        if (some) {
#pragma unroll 1
            for (int c = c0 + lane; c < c1; c += 32) {
                float x[4];
                get(c, x);
#pragma unroll
                for (int j = 0; j < 4; ++j) ties_here += x[j] == cut.value;
            }
            ties_here = __reduce_add_sync(0xffffffffu, ties_here);
            if (lane == 0) s.warp_count[warp] = ties_here;
            __syncthreads();
            const uint32_t up = (uint32_t)add_up(lane < kSampleWarps ? s.warp_count[lane] : 0);
            if (warp == 0) {
                const uint32_t all = __shfl_sync(0xffffffffu, up, 31);
                if (lane < ranks) st_rank32(of_rank(shared_addr(&s.slots[1].count[rank]), lane), all);
            }
            ties_before = __shfl_sync(0xffffffffu, up, warp > 0 ? warp - 1 : 0);
            if (warp == 0) ties_before = 0;
            meet(ranks);
#pragma unroll 1
            for (int q = 0; q < rank; ++q) ties_before += s.slots[1].count[q];
        }
        const bool cut_here = some && ties_before < cut.ties && ties_before + ties_here > cut.ties;
        // Twice over the warp's elements: every warp adds its kept weights up, then the one whose sum the target falls in looks
        // for the token.  One copy of the code for both.
        u64 before = 0, goal = 0, total = 0;
#pragma unroll 1
        for (int look = 0; look < 2; ++look) {
            u64 sum = 0;
            uint32_t running = 0;
#pragma unroll 1
            for (int c = c0; c < c1; c += 32) {
                const bool in = c + lane < c1;
                float x[4];
                get(min(c + lane, c1 - 1), x);
                bool hit[4], equal[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    hit[j] = in && x[j] >= cut.value;
                    equal[j] = hit[j] && x[j] == cut.value;
                }
                if (!__any_sync(0xffffffffu, hit[0] || hit[1] || hit[2] || hit[3])) continue;
                if (some) {
                    uint32_t tie = ties_before;
                    if (cut_here) {                      // equal values of this warp before this lane's
                        const uint32_t n = equal[0] + equal[1] + equal[2] + equal[3], up = (uint32_t)add_up(n);
                        tie += running + up - n;
                        running += __shfl_sync(0xffffffffu, up, 31);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        hit[j] = hit[j] && !(equal[j] && tie >= cut.ties);
                        tie += equal[j];
                    }
                }
                u64 w[4], mine = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    w[j] = weight(fmaxf(x[j], floor_x));
                    if (!hit[j] || w[j] < lowest) w[j] = 0;
                    mine += w[j];
                }
                if (look == 0) {
                    sum += mine;
                    continue;
                }
                const u64 up = add_up(mine);
                u64 at = before + up - mine;
                before += __shfl_sync(0xffffffffu, up, 31);
                if (goal >= at && goal < at + mine) {
                    int index = 0;
                    float value = 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (goal >= at && goal < at + w[j]) { index = j; value = x[j]; }
                        at += w[j];
                    }
                    answer(r, (c + lane) * 4 + index - skew, value, greedy, total);
                }
                if (goal < before) break;
            }
            if (look == 1) break;
#pragma unroll
            for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            if (lane == 0) s.warp_mass[warp] = sum;
            __syncthreads();
            const u64 up = add_up(lane < kSampleWarps ? s.warp_mass[lane] : 0);
            if (warp == 0) {
                const u64 all = __shfl_sync(0xffffffffu, up, 31);
                if (lane < ranks) st_rank64(of_rank(shared_addr(&s.slots[0].mass[rank]), lane), all);
            }
            before = __shfl_sync(0xffffffffu, up, warp > 0 ? warp - 1 : 0);
            if (warp == 0) before = 0;
            meet(ranks);
#pragma unroll 1
            for (int q = 0; q < ranks; ++q) {
                if (q < rank) before += s.slots[0].mass[q];
                total += s.slots[0].mass[q];
            }
            goal = target_of(u, total);
            if (goal < before || goal >= before + sum) break;          // another warp's
        }
    }
};

template <typename T, bool kResident>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const SampleArgs a) {
    __shared__ __align__(16) Shared s;
    extern __shared__ __align__(16) uint8_t sample_smem[];
    const int64_t r = blockIdx.x / a.ranks;
    const T* row = static_cast<const T*>(a.logits) + r * a.ld;
    Sampler<T, kResident> one{a, s};
    one.held = reinterpret_cast<uint4*>(sample_smem);
    one.row = row;
    one.skew = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    one.warp = threadIdx.x >> 5;
    one.lane = threadIdx.x & 31;
    one.rank = (int)(blockIdx.x % a.ranks);
    one.run(r);
    meet(a.ranks);                                       // no CTA leaves while its peers still read its histograms
}

constexpr size_t kSampleSmem = 227 * 1024 - sizeof(Shared) - 1024;
template <typename T, bool kResident>
int launch_sample(const SampleArgs& a, int64_t rows, size_t smem, cudaStream_t st) {
    static unsigned long long configured = 0;            // one per instantiation, one bit per device
    if (const int rc = ensure_dynamic_smem(sample_kernel<T, kResident>, (int)kSampleSmem, configured)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * a.ranks));
    cfg.blockDim = dim3(kSampleThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)a.ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    // One that starts under the tail of the kernel before gets the SMs in the order in which they fall free, two CTAs to each:
    // only where every CTA would have an SM to itself anyway (64 mixed rows of 128256, 256 CTAs: 61 us without, 67 us with it).
    cfg.attrs = attr;
    cfg.numAttrs = rows * a.ranks <= 148 ? 2 : 1;
    const auto kernel = sample_kernel<T, kResident>;
    MIXFP4_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, a));
    return check_launch("sample_kernel");
}

template <typename T>
int sample(SampleArgs& a, int64_t rows, cudaStream_t st) {
    constexpr int kPer = 16 / sizeof(T);
    auto slice = [&](int ranks) { return ((int64_t)a.vocab + 2 * kPer - 2) / kPer / ranks + 1; };      // granules of a CTA, at most
    // CTAs to a row: up to 96 in all, of two thousand elements each at least; up to 256, which share SMs, where each still has
    // eight thousand; more where the slice would be too long.  Top-k and top-p / top-p alone, us, by CTAs a row:
    //     1 x 4096      1: 8.3 / 11.2   2: 8.6 / 10.9   4: 8.9 / 12.4   8: 9.3 / 15.0
    //    16 x 32000     2: 12.9 / 26.2  4: 11.1 / 19.6  8: 12.1 / 22.0
    //    37 x 32000     1: 16.7 / 43.4  2: 13.2 / 27.3  4: 13.7 / 26.5  8: 21.6 / 39.3
    //    64 x 32000     1: 16.8 / 45.4  2: 13.4 / 28.3  4: 14.7 / 27.8
    //    32 x 128256    4: 17.8 / 51.8  8: 17.6 / 45.2
    int ranks = 1;
    while (ranks < kMaxRanks && a.vocab / (ranks * 2) >= 2048 &&
           (rows * ranks * 2 <= 96 || rows * ranks * 2 <= 256 && a.vocab / (ranks * 2) >= 8192))
        ranks *= 2;
    while (ranks < kMaxRanks && (slice(ranks) * 16 > (int64_t)kSampleSmem || slice(ranks) * kPer > kMaxSlice)) ranks *= 2;
    a.ranks = ranks;
    const size_t smem = (size_t)slice(ranks) * 16;
    return smem <= kSampleSmem ? launch_sample<T, true>(a, rows, smem, st) : launch_sample<T, false>(a, rows, 0, st);
}

}  // namespace
}  // namespace mixfp4

using namespace mixfp4;

extern "C" int64_t mixfp4_sample_max_vocab(void) { return kMaxVocab; }

extern "C" int mixfp4_sample(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t ld, const float* uniform,
                             const float* temperature, double temperature_all, const int* top_k, int top_k_all,
                             const float* top_p, double top_p_all, const float* min_p, double min_p_all, int64_t* token,
                             float* logprob, void* stream) {
    if (!logits || !uniform || !token) return MIXFP4_E_NULL;
    if (rows <= 0 || rows > 0x7fffffff / kMaxRanks || vocab <= 0 || ld < vocab) return MIXFP4_E_SHAPE;
    if (vocab > kMaxVocab) return MIXFP4_E_TOO_LARGE;
    const int bytes = dtype == MIXFP4_F32 ? 4 : 2;
    if (dtype != MIXFP4_BF16 && dtype != MIXFP4_F16 && dtype != MIXFP4_F32) return MIXFP4_E_DTYPE;
    if (!aligned(logits, bytes) || !aligned(uniform, 4) || !aligned(token, 8) || !aligned(temperature, 4) || !aligned(top_k, 4) ||
        !aligned(top_p, 4) || !aligned(min_p, 4) || !aligned(logprob, 4))
        return MIXFP4_E_ALIGN;
    SampleArgs a = {};
    a.logits = logits; a.ld = ld; a.vocab = (int)vocab; a.uniform = uniform;
    if (temperature_all > 0.0 && temperature_all < kLeastTemperature) temperature_all = kLeastTemperature;
    a.temperature = {temperature, temperature_all}; a.top_k = {top_k, top_k_all};
    a.top_p = {top_p, top_p_all}; a.min_p = {min_p, min_p_all};
    a.token = reinterpret_cast<long long*>(token); a.logprob = logprob;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case MIXFP4_BF16: return sample<__nv_bfloat16>(a, rows, st);
        case MIXFP4_F16: return sample<__half>(a, rows, st);
        default: return sample<float>(a, rows, st);
    }
}

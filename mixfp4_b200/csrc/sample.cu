// One token a row from logits: temperature, top-k, top-p, min-p, and a random number that the caller brings.
//   w_i   = exp((x_i - max x) / T)                      T = 0: the first of the largest logits
//   order   by value, largest first, equal values by index
//   kept    the first k; of those the shortest run whose weights reach p times theirs; of those every w_i >= min_p
//   token   the first index, in the vocabulary's order, at which the kept weights add up to more than u times their sum
//
// Nothing is sorted.  A cluster of CTAs holds a row in shared memory (one HBM read) and narrows the cut down by
// histograms: 1024 bins of equal width over the logits that have a weight at all, then 1024 bins of the keys (a monotone
// integer of the value) in the bin that the cut falls in, until that bin is one value; equal values are counted off by
// index.  Every CTA adds the cluster's histograms up for itself: one cluster barrier a step, none to hand a result round.
//
// Sums.  The set of kept tokens and the token itself hang on comparisons of sums over the vocabulary, so weights are
// integers: W = round(2^44 w), w in double precision.  Integer sums do not depend on their order, so neither do the
// results, and 2^19 of them fit 63 bits.  A weight below 2^-45 of the largest counts as none.  Shared memory adds 32-bit
// words only, so a bin's sum is kept as three limbs of 16 bits, which 65536 values cannot overflow: the largest slice of a CTA.

#include <mutex>

#include "common.cuh"

namespace mixfp4 {
namespace {

constexpr int kSampleThreads = 1024, kSampleWarps = kSampleThreads / 32, kBins = 1024;
static_assert(kBins == kSampleThreads, "a thread owns a bin");
constexpr int kMaxRanks = 8;
constexpr int64_t kMaxSlice = 65536, kMaxVocab = kMaxRanks * kMaxSlice - 128;
constexpr double kOne = 17592186044416.0;                // 2^44
constexpr float kSpan = 31.5f;                           // weights vanish at 45 ln 2 = 31.2
constexpr float kNegInf = -__builtin_huge_valf();

typedef unsigned long long u64;

template <typename T, typename All>
struct Setting {                                         // a value for each row, or one for all
    const T* each;
    All all;
    __device__ All of(int64_t row) const { return each ? (All)__ldg(each + row) : all; }
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
    float largest[kMaxRanks];
    uint32_t count[kMaxRanks];
    u64 mass[kMaxRanks];
};
struct Shared {
    uint4 hist[2][kBins];                                // per bin: count, three limbs of the weights' sum
    Slots slots[2];
    u64 warp_mass[kSampleWarps];
    uint32_t warp_count[kSampleWarps];
    float warp_max[kSampleWarps];
    u64 found_mass;
    uint32_t found_count, found_bin, found_size;
    u64 total_mass;
};

__device__ __forceinline__ uint32_t shared_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t of_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ uint4 ld_rank(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void st_rank32(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void st_rank64(uint32_t addr, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ void meet(int ranks) {        // all threads of the cluster; writes before are seen after
    if (ranks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    else __syncthreads();
}

// A prefix of the sorted row: everything with a larger key than `key`, and the first `ties` of those equal to it.
struct Cut {
    uint32_t key, ties, equal;                           // equal: how many there are
};

template <typename T, bool kResident>
struct Sampler {
    static constexpr int kPer = 16 / sizeof(T);          // elements of a granule: 16 aligned bytes
    const SampleArgs& a;
    Shared& s;
    uint4* held;                                         // kResident: the slice's granules
    const T* row;
    int skew, granules, g0, g1;                          // granules of the row; this warp's
    int warp, lane, rank, turn, hist_turn;
    float largest;
    double inv_t;
    float bin_scale;

    // Element j of granule g has index g * kPer + j - skew: granules start on 16-byte boundaries, the row need not.
    __device__ void fetch(int g, float (&v)[kPer]) const {
        const int first = g * kPer - skew;
        if (first >= 0 && first + kPer <= a.vocab) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(row + first));
            const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
            for (int j = 0; j < kPer; ++j) v[j] = Elem<T>::load(e + j);
        } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j) v[j] = first + j >= 0 && first + j < a.vocab ? Elem<T>::load(row + first + j) : kNegInf;
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (isnan(v[j])) v[j] = kNegInf;
    }
    __device__ void get(int g, int base, float (&v)[kPer]) const {
        if constexpr (kResident) {
            const uint4 u = held[g - base];
            const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
            for (int j = 0; j < kPer; ++j) v[j] = Elem<T>::load(e + j);
        } else {
            fetch(g, v);
        }
    }
    int base;                                            // first granule of this CTA

    // f(value, index) for this warp's elements in the order of a granule's elements; lanes take granules in turn.
    template <typename F>
    __device__ void each(F&& f) const {
        for (int g = g0 + lane; g < g1; g += 32) {
            float v[kPer];
            get(g, base, v);
#pragma unroll
            for (int j = 0; j < kPer; ++j) f(v[j], g * kPer + j - skew);
        }
    }

    __device__ double weight(float x) const { return x == largest ? 1.0 : exp(((double)x - (double)largest) * inv_t); }
    __device__ u64 fixed(float x) const { return (u64)__double2ll_rn(weight(x) * kOne); }
    // Bin of equal width, rising as the value falls (rounded operations are monotone); kBins and more: no weight.
    __device__ uint32_t linear(float x) const {
        if (x == kNegInf) return kBins;
        const float d = x == largest ? 0.0f : largest - x;
        return (uint32_t)fminf(d * bin_scale, (float)kBins);
    }

    __device__ void clear(int which) {
        s.hist[which][threadIdx.x] = make_uint4(0, 0, 0, 0);
    }
    __device__ void put(int which, uint32_t bin, bool masses, float x) {
        uint32_t* h = reinterpret_cast<uint32_t*>(&s.hist[which][bin]);
        atomicAdd(h, 1u);
        if (masses) {
            const u64 w = fixed(x);
            atomicAdd(h + 1, (uint32_t)(w & 0xffffu));
            atomicAdd(h + 2, (uint32_t)(w >> 16) & 0xffffu);
            atomicAdd(h + 3, (uint32_t)(w >> 32));
        }
    }
    // The cluster's histogram, a bin a thread, and the first bin at which the running count (or mass) reaches `goal`: into
    // s.found_*: the bin, what lies before it, its size.  total_mass: of all bins.  goal 0 looks for the mass's total only.
    __device__ void find(bool by_mass, u64 before_count, u64 before_mass, u64 goal) {
        meet(a.ranks);
        clear(hist_turn ^ 1);                            // every CTA is past its reads of that one
        uint32_t count = 0;
        u64 mass = 0;
        const uint32_t at = shared_addr(&s.hist[hist_turn][threadIdx.x]);
        for (int r = 0; r < a.ranks; ++r) {
            const uint4 h = a.ranks > 1 ? ld_rank(of_rank(at, r)) : s.hist[hist_turn][threadIdx.x];
            count += h.x;
            mass += (u64)h.y + ((u64)h.z << 16) + ((u64)h.w << 32);
        }
        hist_turn ^= 1;
        uint32_t c = count;
        u64 m = mass;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const uint32_t oc = __shfl_up_sync(0xffffffffu, c, d);
            const u64 om = __shfl_up_sync(0xffffffffu, m, d);
            if (lane >= d) { c += oc; m += om; }
        }
        if (lane == 31) { s.warp_count[warp] = c; s.warp_mass[warp] = m; }
        if (threadIdx.x == 0) s.found_bin = kBins;
        __syncthreads();
        u64 pc = before_count, pm = before_mass, all = before_mass;
        for (int w = 0; w < kSampleWarps; ++w) {
            if (w < warp) { pc += s.warp_count[w]; pm += s.warp_mass[w]; }
            all += s.warp_mass[w];
        }
        const u64 hi_c = pc + c, hi_m = pm + m, lo_c = hi_c - count, lo_m = hi_m - mass;
        const bool here = by_mass ? lo_m < goal && goal <= hi_m : lo_c < goal && goal <= hi_c;
        if (here) { s.found_bin = threadIdx.x; s.found_count = (uint32_t)lo_c; s.found_mass = lo_m; s.found_size = count; }
        if (threadIdx.x == 0) s.total_mass = all;
        __syncthreads();
    }

    // From the linear bin s.found_bin down to one value.  `from`: only keys of at least that.
    __device__ Cut narrow(bool by_mass, u64 goal, uint32_t from) {
        const uint32_t bin = s.found_bin;
        u64 count = s.found_count, mass = s.found_mass;
        uint32_t size = s.found_size;
        // keys that the bin can hold: its edges, moved out by more than rounding moved them
        const float width = 1.0f / bin_scale;
        const float x_hi = largest - (float)bin * width * 0.9999f, x_lo = largest - ((float)bin + 1.0f) * width * 1.0001f;
        uint32_t hi = Row<T>::key(bin == 0 ? largest : fminf(x_hi + fabsf(largest) * 1e-6f, largest));
        uint32_t lo = isinf(largest) ? hi : Row<T>::key(x_lo - fabsf(largest) * 1e-6f);
        if (lo < from) lo = from;
        __syncthreads();                                 // found_* has been read
        for (int level = 0; level < 4; ++level) {        // 32 bits, 10 a level
            const uint32_t span = hi - lo;
            const int shift = span < (uint32_t)kBins ? 0 : 22 - __clz(span);
            const int which = hist_turn;
            each([&](float x, int) {
                if (linear(x) != bin) return;
                const uint32_t k = Row<T>::key(x);
                if (k >= lo && k <= hi) put(which, (hi - k) >> shift, by_mass, x);
            });
            find(by_mass, count, mass, goal);
            const uint32_t b = s.found_bin;
            count = s.found_count; mass = s.found_mass; size = s.found_size;
            __syncthreads();
            hi -= b << shift;
            if (shift == 0) break;
            const uint32_t width_keys = 1u << shift;
            if (hi - lo >= width_keys) lo = hi - width_keys + 1;
        }
        Cut cut;
        cut.key = hi;
        cut.equal = size;
        cut.ties = (uint32_t)(goal - count);
        if (by_mass) {                                   // equal weights: as many as are needed
            const u64 w = fixed(value_of(hi));
            cut.ties = (uint32_t)((goal - mass + w - 1) / w);
        }
        return cut;
    }
    __device__ static float value_of(uint32_t key) {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
        } else {
            const uint16_t b = (uint16_t)(key & 0x8000u ? key & 0x7fffu : key ^ 0xffffu);
            return Elem<T>::load(reinterpret_cast<const T*>(&b));
        }
    }

    __device__ void run(int64_t r) {
        const int ranks = a.ranks;
        // the row's granules, the cluster's share, the warps' shares: contiguous, so that indices rise with rank, warp, lane
        const int per_rank = (granules + ranks - 1) / ranks;
        base = min(rank * per_rank, granules);
        const int end = min(base + per_rank, granules), per_warp = (end - base + kSampleWarps - 1) / kSampleWarps;
        g0 = min(base + warp * per_warp, end);
        g1 = min(g0 + per_warp, end);
        turn = 0;
        hist_turn = 0;
        clear(0);
        clear(1);

        float top = kNegInf;
        for (int g = g0 + lane; g < g1; g += 32) {
            float v[kPer];
            fetch(g, v);
            if constexpr (kResident) {
                T e[kPer];
#pragma unroll
                for (int j = 0; j < kPer; ++j) e[j] = Elem<T>::round(v[j]);
                held[g - base] = *reinterpret_cast<const uint4*>(e);
            }
#pragma unroll
            for (int j = 0; j < kPer; ++j) top = fmaxf(top, v[j]);
        }
#pragma unroll
        for (int d = 16; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        if (lane == 0) s.warp_max[warp] = top;
        __syncthreads();
        if (warp == 0) {
            top = s.warp_max[lane];
#pragma unroll
            for (int d = 16; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            if (lane < ranks) st_rank32(of_rank(shared_addr(&s.slots[0].largest[rank]), lane), __float_as_uint(top));
        }
        meet(ranks);
        turn = 1;
        largest = kNegInf;
        for (int q = 0; q < ranks; ++q) largest = fmaxf(largest, s.slots[0].largest[q]);

        if (largest == kNegInf) {                        // nothing to choose from
            if (rank == 0 && threadIdx.x == 0) {
                a.token[r] = -1;
                if (a.logprob) a.logprob[r] = kNegInf;
            }
            return;
        }
        const double t = a.temperature.of(r);
        const bool greedy = !(t > 0.0);
        inv_t = greedy ? 1.0 : 1.0 / t;
        bin_scale = greedy ? 1.0f : (float)fmin((double)kBins / (kSpan * t), 1e38);
        const int k = a.top_k.of(r);
        const double p = a.top_p.of(r), lowest = greedy ? 0.0 : fmin(a.min_p.of(r), 1.0);
        Cut cut{0, 0, 0};                                // key 0: everything
        if (greedy) {
            cut = Cut{Row<T>::key(largest), 1, 0xffffffffu};
        } else {
            if (k > 0 && k < a.vocab) {
                each([&](float x, int) {
                    const uint32_t bin = linear(x);
                    if (bin < (uint32_t)kBins) put(hist_turn, bin, false, x);
                });
                find(false, 0, 0, (u64)k);
                if (s.found_bin < (uint32_t)kBins) cut = narrow(false, (u64)k, 0);      // else fewer than k have a weight
            }
            if (p < 1.0) {
                each([&](float x, int) {
                    const uint32_t bin = linear(x);
                    if (bin < (uint32_t)kBins && Row<T>::key(x) >= cut.key) put(hist_turn, bin, true, x);
                });
                // two looks at the same histogram: the sum, then the bin
                find(true, 0, 0, 0);
                u64 total = s.total_mass;
                if (cut.key) total -= (u64)(cut.equal - cut.ties) * fixed(value_of(cut.key));
                const double want = ceil(fmax(p, 0.0) * (double)total);
                u64 goal = want < 1.0 ? 1 : (u64)want;
                if (goal > total) goal = total;
                hist_turn ^= 1;                          // the same one again
                find(true, 0, 0, goal);
                cut = narrow(true, goal, cut.key);
            }
        }

        // equal values before this warp's
        uint32_t ties_before = 0, ties_here = 0;
        const bool some = cut.ties < cut.equal;          // not all of them are kept
        if (some) {
            each([&](float x, int) { ties_here += x > kNegInf && Row<T>::key(x) == cut.key; });
            ties_here = __reduce_add_sync(0xffffffffu, ties_here);
            __syncthreads();
            if (lane == 0) s.warp_count[warp] = ties_here;
            __syncthreads();
            if (warp == 0) {
                const uint32_t sum = __reduce_add_sync(0xffffffffu, s.warp_count[lane]);
                if (lane < ranks) st_rank32(of_rank(shared_addr(&s.slots[turn].count[rank]), lane), sum);
            }
            meet(ranks);
            for (int q = 0; q < rank; ++q) ties_before += s.slots[turn].count[q];
            for (int w = 0; w < warp; ++w) ties_before += s.warp_count[w];
            turn ^= 1;
        }
        // the weight of an element if it is kept; ties of this warp that come before it
        auto kept = [&](float x, uint32_t tie) -> u64 {
            if (x == kNegInf) return 0;
            const uint32_t key = Row<T>::key(x);
            if (key < cut.key || (some && key == cut.key && ties_before + tie >= cut.ties)) return 0;
            const double w = weight(x);
            return w >= lowest ? (u64)__double2ll_rn(w * kOne) : 0;
        };
        // Elements of a step (32 granules) before this lane's that are equal to the cut's value.
        auto tie_rank = [&](const float (&v)[kPer], bool in, uint32_t& running) -> uint32_t {
            uint32_t n = 0;
#pragma unroll
            for (int j = 0; j < kPer; ++j) n += in && v[j] > kNegInf && Row<T>::key(v[j]) == cut.key;
            uint32_t up = n;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const uint32_t o = __shfl_up_sync(0xffffffffu, up, d);
                if (lane >= d) up += o;
            }
            const uint32_t mine = running + up - n;
            running += __shfl_sync(0xffffffffu, up, 31);
            return mine;
        };
        const bool cut_here = some && ties_before < cut.ties && ties_before + ties_here > cut.ties;
        u64 sum = 0;
        uint32_t running = 0;
        for (int g = g0; g < g1; g += 32) {
            const bool in = g + lane < g1;
            float v[kPer];
            if (in) get(g + lane, base, v);
            uint32_t tie = cut_here ? tie_rank(v, in, running) : 0;
            if (in) {
#pragma unroll
                for (int j = 0; j < kPer; ++j) {
                    sum += kept(v[j], tie);
                    if (cut_here) tie += v[j] > kNegInf && Row<T>::key(v[j]) == cut.key;
                }
            }
        }
#pragma unroll
        for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        __syncthreads();
        if (lane == 0) s.warp_mass[warp] = sum;
        __syncthreads();
        if (warp == 0) {
            u64 all = s.warp_mass[lane];
#pragma unroll
            for (int d = 16; d > 0; d /= 2) all += __shfl_xor_sync(0xffffffffu, all, d);
            if (lane < ranks) st_rank64(of_rank(shared_addr(&s.slots[turn].mass[rank]), lane), all);
        }
        meet(ranks);
        u64 total = 0, before = 0;
        for (int q = 0; q < ranks; ++q) {
            if (q < rank) before += s.slots[turn].mass[q];
            total += s.slots[turn].mass[q];
        }
        for (int w = 0; w < warp; ++w) before += s.warp_mass[w];
        const double u = (double)__ldg(a.uniform + r);
        const double want = u > 0.0 ? u * (double)total : 0.0;
        const u64 goal = want < (double)total ? min((u64)want, total - 1) : total - 1;
        if (goal < before || goal >= before + sum) return;          // another warp's
        // this warp holds the token: lanes' sums of a step, then the elements of the lane
        running = 0;
        for (int g = g0; g < g1; g += 32) {
            const bool in = g + lane < g1;
            float v[kPer];
            if (in) get(g + lane, base, v);
            uint32_t tie = cut_here ? tie_rank(v, in, running) : 0;
            u64 w[kPer], mine = 0;
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                w[j] = in ? kept(v[j], tie) : 0;
                if (cut_here) tie += in && v[j] > kNegInf && Row<T>::key(v[j]) == cut.key;
                mine += w[j];
            }
            u64 up = mine;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const u64 o = __shfl_up_sync(0xffffffffu, up, d);
                if (lane >= d) up += o;
            }
            u64 at = before + up - mine;
            before += __shfl_sync(0xffffffffu, up, 31);
            if (goal >= at && goal < at + mine) {
#pragma unroll
                for (int j = 0; j < kPer; ++j) {
                    if (goal >= at && goal < at + w[j]) {
                        a.token[r] = (long long)(g + lane) * kPer + j - skew;
                        if (a.logprob)
                            a.logprob[r] = greedy ? 0.0f
                                                  : (float)((v[j] == largest ? 0.0 : ((double)v[j] - (double)largest) * inv_t) -
                                                            log((double)total / kOne));
                    }
                    at += w[j];
                }
            }
            if (goal < before) break;
        }
    }
};

template <typename T, bool kResident>
__global__ void __launch_bounds__(kSampleThreads, 1) sample_kernel(const SampleArgs a) {
    __shared__ __align__(16) Shared s;
    extern __shared__ __align__(16) uint8_t sample_smem[];
    const int64_t r = blockIdx.x / a.ranks;
    const T* row = static_cast<const T*>(a.logits) + r * a.ld;
    Sampler<T, kResident> one{a, s};
    one.held = reinterpret_cast<uint4*>(sample_smem);
    one.row = row;
    one.skew = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    one.granules = (a.vocab + one.skew + one.kPer - 1) / one.kPer;
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
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)a.ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const auto kernel = sample_kernel<T, kResident>;
    MIXFP4_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, a));
    return check_launch("sample_kernel");
}

template <typename T>
int sample(SampleArgs& a, int64_t rows, cudaStream_t st) {
    constexpr int kPer = 16 / sizeof(T);
    auto slice = [&](int ranks) { return ((int64_t)a.vocab + 2 * kPer - 2) / kPer / ranks + 1; };      // granules of a CTA, at most
    // as many CTAs to a row as keep the SMs busy, a thousand elements each at least; more where the slice would be too long
    int ranks = 1;
    while (ranks < kMaxRanks && rows * ranks * 2 <= 148 && a.vocab / (ranks * 2) >= 1024) ranks *= 2;
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
    if (!aligned(logits, bytes) || !aligned(uniform, 4) || !aligned(token, 8)) return MIXFP4_E_ALIGN;
    SampleArgs a = {};
    a.logits = logits; a.ld = ld; a.vocab = (int)vocab; a.uniform = uniform;
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

// Sampling of the next token from what temperature, top-k, top-p and min-p leave of a distribution, and the logits with all
// else at -infinity.
//
// A cluster takes a row and keeps it in the shared memory of its CTAs, so that the logits are read once however many passes
// the row needs:
//     weight  W = 2^44 * 2^((x - max) * log2(e) / T), as a whole number
//     kept    the tokens from the largest on (the lowest index of equals first): top_k of them, then as many as it takes
//             until their sum reaches top_p of those, none below min_p of the largest
//     token   the first index at which the running sum of the kept exceeds u times their sum
// A set that is kept is always "all logits above a key, and those at the key up to an index". Top-k lists what lies above a bound
// that bins of the threads' largest logits give; top-p sums 1024 bins of the distance to the maximum and lists the bin in which
// the border lies. A list of up to 1024 logits is in every CTA, which finds the border in it by itself. Where that does not come
// down to a list, the key is found by counts or sums over 128 bins at a time, of the distance and then of the bits of the keys
// that are left. What each CTA keeps is known from bins and list: only the CTA that has the token adds weights up by index.
//
// Weights are evaluated in 64 bits and summed as whole numbers: borders are compared exactly, and neither the cluster's
// size nor the order of atomics has a say. With weights in 32 bits a running sum is off by some 1e-8, and a tail of 100,000
// tokens of 1e-6 each is off by a token once in a hundred draws.
//
// What bounds it: one row is a chain of barriers of its cluster (some 0.7 us each with what they wait for) and passes over
// 8 to 44 logits a thread; of many rows, some 45 are on the GPU at a time, as many as its shared memory holds, so their chains
// and the 64-bit weights (15 instructions, 7.5 clocks a warp and SM) are the time, not HBM. 256 rows of 131,072 (20.5 us of
// HBM): temperature 0 48 us, top-k 40 with top-p 78, no truncation 113, a nucleus of 0.9 197; one row 4, 8, 8 and 15.
#include "cache.cuh"

using namespace nb;

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 128;
constexpr int kFine = 1024;                       // bins of the nucleus, in groups of 32
constexpr int kFew = 256;                         // logits of top-k that are ordered one by one
constexpr int kFewer = 64;                        // the same where one of a list is looked for
constexpr int kSparse = 16;                       // of a lane's 32 logits: with more than these in a lane, all of the warp's are weighed
constexpr int kList = 1024;                       // logits that every CTA has a list of
constexpr int kStep = kThreads * 4;               // a CTA's part of a row is a multiple of this: a thread has whole units of four
constexpr int kMaxUnits = 22;                     // of a thread: 188 KB a CTA
constexpr int kMaxRanks = 16;                     // CTAs of a cluster
constexpr int kMaxVocab = 8 * kMaxUnits * kStep;
constexpr int kRowsAtOnce = 1 << 20;
static_assert(32 * kMaxUnits * kMaxUnits < 65536, "a unit's owner by multiplication");
static_assert(kMaxVocab <= 1 << 19, "sums of weights, 2^44 at most, fit 63 bits");
static_assert(kMaxRanks == kWarps && kMaxRanks % 4 == 0 && 2 * kFew <= kThreads && 4 * kBins == kThreads, "two threads to a logit that is ordered, four to a bin");

struct SampleArgs {
    const float *logits, *uniforms, *temperature, *top_p, *min_p;
    const int *top_k;
    float *out;
    int *token;
    int per, rows, vocab, units;
    unsigned inverse;  // of units, in 65536ths and rounded up: right for all of a warp's 32 * units, since 32 * 22 * 22 < 65536
    __device__ __forceinline__ int owner_of(int unit) const { return (int)(unit * inverse >> 16); }
};

using Whole = unsigned long long;

// What the CTAs of a cluster read of each other.
struct Shared {
    Whole ends[kMaxRanks];             // key of the largest logit; inverted, the lowest of the threads' largest, or its index
    int last[2];
    Whole total[2][kMaxRanks];         // by the parity of the exchange: a CTA may be one ahead
    unsigned hist[2][2][kBins];        // by the parity of the pass: counts, or the low and high words of sums
    Whole list[kList];                 // key and inverted index: the larger is the better
    int listed, lists[kMaxRanks];      // of this CTA's list and of all
    union {
        unsigned fine[2][kFine];       // words of sums
        Whole entry[kList];            // from here on a CTA's own: these once all have read the bins, with a barrier between
        Whole bins[4][kBins];
    };
    union {
        Whole entry_weight[kFew];
        Whole read[kMaxRanks][kFine / 32];  // sums of the CTAs' groups of bins, then of a group's bins; until entries are ordered
    };
    Whole warp_sum[kWarps];
    Whole found, kept_sum;
    int few;
    unsigned warp_most[kWarps], warp_least[kWarps];
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
// The address of a variable of this CTA in CTA `rank`.
__device__ __forceinline__ uint32_t at_rank(const void *p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ unsigned peer_load(uint32_t a) {
    unsigned x;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(a) : "memory");
    return x;
}
__device__ __forceinline__ Whole peer_load64(uint32_t a) {
    Whole x;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(x) : "r"(a) : "memory");
    return x;
}
__device__ __forceinline__ void peer_store(uint32_t a, unsigned x) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(x) : "memory"); }
__device__ __forceinline__ void peer_store(uint32_t a, Whole x) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(x) : "memory"); }
// The larger, or NaN if one is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// Whole numbers in the order of the floats.
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned b = __float_as_uint(x);
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(unsigned k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
constexpr unsigned kNone = 0x007fffffu;       // key of -infinity
constexpr unsigned kMinusZero = 0x7fffffffu;  // of -0, which no logit is
constexpr float kLowest = -3.402823466e38f;

__device__ __forceinline__ Whole warp_sum(Whole x) {
#pragma unroll
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}
__device__ __forceinline__ Whole warp_scan(Whole x) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const Whole y = __shfl_up_sync(0xffffffffu, x, d);
        if ((threadIdx.x & 31) >= d) x += y;
    }
    return x;
}

// One CTA's view of a row. A thread has units of four neighbouring logits, all of its units next to each other, so the
// threads' order is the indices' order; in shared memory threads are an odd number of units apart, which keeps their reads
// off each other's banks.
struct Row {
    const float4 *mine;  // the thread's units; what lies outside the row is -infinity
    int units;           // of a thread
    int index;           // of its first logit (may be negative, where the row does not start on 16 bytes)
    uint32_t rank, ranks;
    float most, zero;    // the largest logit; below `zero` weights are 0
    double top, c;       // log2(e) / T
    unsigned key;        // kept: logits above the key, and those at it up to index `last`
    int last;
    bool settled;        // whether it is known already what the CTAs' kept weights add up to
    bool known;          // whether all threads' shares add up to those that this CTA keeps
    Whole share;
    int ahead;           // logits of the first CTA that lie before the row
    unsigned inverse;    // of units

    // The CTA that has a logit.
    __device__ __forceinline__ int rank_of(int i) const { return (int)(((unsigned)(i + ahead) / kStep) * inverse >> 16); }
    // f(x, index) for every logit of the thread.
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
#pragma unroll 2
        for (int j = 0; j < units; j++) {
            const float4 x = mine[j];
            const int at = index + 4 * j;
            f(x.x, at), f(x.y, at + 1), f(x.z, at + 2), f(x.w, at + 3);
        }
    }
    // f(x, index) for two of those from low to high at a time (-infinity where there is none). They are looked for first, 32
    // logits at a time: a warp then takes as many turns as its fullest lane has logits, and not one for every place at which
    // some lane has one. (A list of a warp's logits that its lanes share evenly takes longer than it saves: nucleus of 0.98 at
    // temperature 1, 34 us in all against 53.)
    template <typename F>
    __device__ __forceinline__ void some(float low, float high, F f) const {
        for (int j0 = 0; j0 < units; j0 += 8) two_by_two(between(j0, low, high), j0, f);
    }
    // Which of the 32 logits from unit j0 on lie between low and high. With low alone: up to the largest.
    __device__ __forceinline__ unsigned between(int j0, float low, float high) const {
        return which(j0, [=](float x) { return x >= low && x <= high; });
    }
    __device__ __forceinline__ unsigned from(int j0, float low) const {
        return which(j0, [=](float x) { return x >= low; });
    }
    template <typename P>
    __device__ __forceinline__ unsigned which(int j0, P is) const {
        unsigned found = 0;
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j0 + j < units) {
                const float4 x = mine[j0 + j];
                found |= (is(x.x) ? 1u << (4 * j) : 0) | (is(x.y) ? 2u << (4 * j) : 0) | (is(x.z) ? 4u << (4 * j) : 0) | (is(x.w) ? 8u << (4 * j) : 0);
            }
        return found;
    }
    template <typename F>
    __device__ __forceinline__ void two_by_two(unsigned found, int j0, F f) const {
        while (found) {
            float x[2];
            int at[2];
            const int a = __ffs(found) - 1;
            found &= found - 1;
            const int b = found ? __ffs(found) - 1 : a;
            const float *from = reinterpret_cast<const float *>(mine + j0);
            x[0] = from[a], x[1] = found ? from[b] : -INFINITY;
            found &= found - 1;
            at[0] = index + 4 * j0 + a, at[1] = index + 4 * j0 + b;
            f(x, at);
        }
    }
    // f(x, index, weight) for four neighbouring logits at a time, where some of the warp's are at or above low (and weigh something).
    template <typename F>
    __device__ __forceinline__ void each_weight(float low, F f) const {
        weights_of(0, units, fmaxf(low, zero), f);
    }
    template <typename F>
    __device__ __forceinline__ void weights_of(int j0, int j1, float low, F f) const {
#pragma unroll 2
        for (int j = j0; j < j1; j++) {
            const float4 x = mine[j];
            if (!__any_sync(0xffffffffu, fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)) >= low)) continue;
            const float y[4] = {x.x, x.y, x.z, x.w};
            const Whole w[4] = {weigh(x.x), weigh(x.y), weigh(x.z), weigh(x.w)};
            f(y, index + 4 * j, w);
        }
    }
    // The thread's sum of the weights that are kept. Few of 32 logits are taken two by two (256 rows of 131,072, nucleus of 0.9: 246 us
    // with all weighed, 230 so; no truncation 123 and 125).
    __device__ __forceinline__ Whole kept_sum() const {
        Whole sum = 0;
        const float low = floor(), weighs = fmaxf(low, zero);
        for (int j0 = 0; j0 < units; j0 += 8) {
            const unsigned found = key == kNone ? ~0u : from(j0, weighs);
            if (__reduce_max_sync(0xffffffffu, __popc(found)) <= kSparse)
                two_by_two(found, j0, [&](const float (&x)[2], const int (&at)[2]) {
                    const Whole w[2] = {weigh(x[0]), weigh(x[1])};
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        if (kept_of_floor(x[e], at[e])) sum += w[e];
                });
            else
                weights_of(j0, min(units, j0 + 8), weighs, [&](const float (&x)[4], int at, const Whole (&w)[4]) {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (kept_of_floor(x[e], at + e)) sum += w[e];
                });
        }
        return sum;
    }
    // Of logits from floor() up, and -infinity: those that are kept.
    __device__ __forceinline__ bool kept_of_floor(float x, int i) const { return x > floor() || (x == floor() && i <= last); }
    __device__ __forceinline__ bool keeps(float x, int i) const {
        const unsigned k = key_of(x);
        return k > key || (k == key && i <= last);
    }
    // The lowest logit that may be kept, or -infinity.
    __device__ __forceinline__ float floor() const { return of_key(key); }

    // 2^44 * 2^((x - most) * c), rounded. The polynomial of degree 9 is 2^f's Chebyshev fit on [-1/2, 1/2] (off by less than
    // 2^-46 there, and by 2^-45.6 of its value at most).
    __device__ __forceinline__ Whole weigh(float x) const {
        const double t = ((double)fmaxf(x, zero) - top) * c;
        constexpr double kRound = 6755399441055744.0 + 44.0, kUnit = 4503599627370496.0;  // 1.5 * 2^52 (the last bits: n + 44), 2^52
        const double n = t + kRound, f = t - (n - kRound);
        double p = 1.0205905413765595e-07;
        p = fma(p, f, 1.325964524488711e-06);
        p = fma(p, f, 1.5252672924850737e-05);
        p = fma(p, f, 1.540343375125101e-04);
        p = fma(p, f, 1.3333558200794592e-03);
        p = fma(p, f, 9.618129193934313e-03);
        p = fma(p, f, 5.550410866465167e-02);
        p = fma(p, f, 2.402265069564034e-01);
        p = fma(p, f, 6.931471805599462e-01);
        p = fma(p, f, 1.0000000000000135);
        const double v = __hiloint2double(__double2hiint(p) + (__double2loint(n) << 20), __double2loint(p)) + kUnit;
        const Whole w = (Whole)__double_as_longlong(v) & 0xfffffffffffffull;
        return x >= zero ? w : 0;
    }
};

// Of the threads' sums: the warps' to s.warp_sum, the CTAs' to s.total of all. Ends with a barrier of the cluster.
// `along` is called by all threads once all are here, before that barrier.
template <typename F>
__device__ __forceinline__ void share_sums(Shared &s, const Row &r, Whole x, int turn, F along) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    x = warp_sum(x);
    if (lane == 0) s.warp_sum[warp] = x;
    __syncthreads();
    along();
    if (warp == 0) {
        const Whole all = warp_sum(lane < kWarps ? s.warp_sum[lane] : 0);
        if (lane < r.ranks) peer_store(at_rank(&s.total[turn & 1][r.rank], lane), all);
    }
    cluster_sync();
}
__device__ __forceinline__ void share_sums(Shared &s, const Row &r, Whole x, int turn) {
    share_sums(s, r, x, turn, [] {});
}
// Totals of the CTAs before this one, and of all.
__device__ __forceinline__ Whole sums_before(const Shared &s, const Row &r, int turn, Whole &all) {
    Whole before = 0;
    all = 0;
#pragma unroll 1
    for (uint32_t i0 = 0; i0 < r.ranks; i0 += 4)
#pragma unroll
        for (uint32_t i = i0; i < i0 + 4; i++) {
            const Whole x = i < r.ranks ? s.total[turn & 1][i] : 0;
            if (i < r.rank) before += x;
            all += x;
        }
    return before;
}
// The index at which the running sum of f (in the order of indices) reaches `target`, for the one warp that holds it; -1 for
// all others. `mine`: the thread's sum; after share_sums of it.
template <typename F>
__device__ int reach(const Shared &s, const Row &r, Whole mine, Whole before, Whole target, F f) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Whole of_warp = lane < kWarps ? s.warp_sum[lane] : 0, upto = warp_scan(of_warp) + before;
    const unsigned past = __ballot_sync(0xffffffffu, lane < kWarps && upto >= target);
    if (!past || __ffs(past) - 1 != warp) return -1;
    const Whole base = __shfl_sync(0xffffffffu, upto - of_warp, warp);
    if (base >= target) return -1;  // (an earlier CTA's)
    const Whole here = warp_scan(mine) + base;
    const int l = __ffs(__ballot_sync(0xffffffffu, here >= target)) - 1;
    // the warp goes through that lane's logits, 32 at a time
    Whole run = __shfl_sync(0xffffffffu, here - mine, l);
    const float *x = reinterpret_cast<const float *>(r.mine + (l - lane) * (r.units | 1));
    const int first = r.index + (l - lane) * 4 * r.units;
    for (int i = 0; i < 4 * r.units; i += 32) {
        const int at = i + lane;
        const Whole w = at < 4 * r.units ? f(x[at], first + at) : 0, till = warp_scan(w) + run;
        const unsigned hit = __ballot_sync(0xffffffffu, till >= target);
        if (hit) return first + i + __ffs(hit) - 1;
        run = __shfl_sync(0xffffffffu, till, 31);
    }
    return -1;
}

// The bin, thread tid's for tid < kBins, at which the running sum of `mine` reaches `target`, and the sum before it, to all
// threads; -1 where it is not reached.
struct Bin {
    int bin;
    Whole before;
};
__device__ __forceinline__ Bin reach_bin(Shared &s, Whole mine, Whole target) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Whole upto_warp = warp_scan(mine);
    if (lane == 31) s.warp_sum[warp] = upto_warp;
    if (tid == 0) s.found = ~0ull;
    __syncthreads();
    const Whole of_warp = lane < kWarps ? s.warp_sum[lane] : 0, warps_upto = warp_scan(of_warp);
    const Whole upto = upto_warp + __shfl_sync(0xffffffffu, warps_upto - of_warp, warp);
    if (upto >= target && upto - mine < target) s.found = tid, s.kept_sum = upto - mine;
    __syncthreads();
    return {(int)s.found, s.kept_sum};
}
// Adds to a sum of two words. Shared memory has no addition of 64 bits of its own (one that tries again and again takes 61
// clocks a warp over 64 bins, two words 5.6, three parts that need no carry 7.5).
__device__ __forceinline__ void add_words(unsigned &low, unsigned &high, Whole w) {
    const unsigned before = atomicAdd(&low, (unsigned)w);
    unsigned carried;
    asm("{.reg .u32 t;\n add.cc.u32 t, %1, %2;\n addc.u32 %0, %3, 0;}" : "=r"(carried) : "r"(before), "r"((unsigned)w), "r"((unsigned)(w >> 32)));
    atomicAdd(&high, carried);
}
__device__ __forceinline__ Whole words(unsigned low, unsigned high) { return (Whole)high << 32 | low; }
// A histogram counts, or adds up weights.
using Hist = unsigned[2][kBins];
template <bool SUM>
__device__ __forceinline__ void add_to(Hist &hist, int bin, Whole w) {
    if (SUM) add_words(hist[0][bin], hist[1][bin], w);
    else atomicAdd(&hist[0][bin], 1u);
}
// One histogram of all CTAs' added up: bin tid's, for tid < kBins. Four threads to a bin read, a quarter of the CTAs' each.
template <bool SUM>
__device__ __forceinline__ Whole all_bins(Shared &s, const Row &r, const Hist &hist) {
    const int bin = threadIdx.x % kBins, group = threadIdx.x / kBins;
    constexpr int N = SUM ? 2 : 1;
    Whole sum = 0;
#pragma unroll 1
    for (uint32_t q0 = group; q0 < r.ranks; q0 += 8) {
        unsigned part[2][N];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < N; e++) part[i][e] = q0 + 4 * i < r.ranks ? peer_load(at_rank(&hist[e][bin], q0 + 4 * i)) : 0;
        sum += (Whole)part[0][0] + part[1][0];
        if constexpr (SUM) sum += (Whole)(part[0][1] + part[1][1]) << 32;
    }
    s.bins[group][bin] = sum;
    __syncthreads();
    return threadIdx.x < kBins ? (s.bins[0][bin] + s.bins[1][bin]) + (s.bins[2][bin] + s.bins[3][bin]) : 0;
}
// Keys from low to high, and of these the logits whose distance from the largest falls into `bin` (-1: any).
struct Range {
    unsigned low, high;
    float most, scale;
    int last_bin, bin;
    // Up to where its logits are looked for. Keys that end at -0's end below 0, which as a float is not above it.
    __device__ __forceinline__ float highest() const { return of_key(high == kMinusZero ? high - 1 : high); }
    __device__ __forceinline__ int bin_of(float x) const { return min(last_bin, (int)((most - x) * scale)); }
    __device__ __forceinline__ bool has(float x) const { return bin < 0 || bin_of(x) == bin; }  // of those between low and high
    // Only what is in distance bin b. The keys' limits are wider than the bin by more than bin_of rounds.
    __device__ __forceinline__ void take_bin(int b) {
        const double width = 1.0f / scale;
        if (b < last_bin) low = max(low, key_of(__double2float_rd((double)most - (b + 1) * 1.000001 * width)));
        if (b) high = min(high, key_of(__double2float_ru((double)most - b * 0.999999 * width)));
        bin = b;
    }
    // Only key bin b of those that are 2^shift keys wide, from high on downwards.
    __device__ __forceinline__ void take_keys(int b, int shift) {
        high -= (unsigned)b << shift;
        const unsigned span = (1u << shift) - 1;
        low = high - low > span ? high - span : low;
    }
    __device__ __forceinline__ int shift() const { return max(0, 25 - __clz(high - low)); }  // (high - low) >> shift < kBins
};

// The kept logits in a range, of all CTAs and in any order, in s.entry. Returns their number; more than kList are not listed.
// s.listed is zero before.
__device__ int gather(Shared &s, const Row &r, const Range &in) {
    r.some(of_key(max(in.low, kNone + 1)), in.highest(), [&](const float (&x)[2], const int (&at)[2]) {
#pragma unroll
        for (int e = 0; e < 2; e++)
            if (r.kept_of_floor(x[e], at[e]) && in.has(x[e])) {
                const int to = atomicAdd(&s.listed, 1);
                if (to < kList) s.list[to] = (Whole)key_of(x[e]) << 32 | (unsigned)~at[e];
            }
    });
    __syncthreads();
    if (threadIdx.x < r.ranks) peer_store(at_rank(&s.lists[r.rank], threadIdx.x), (unsigned)s.listed);
    cluster_sync();
    // a lane has a CTA's number, and where its part of the list begins
    const int lane = threadIdx.x & 31, n = lane < r.ranks ? s.lists[lane] : 0;
    int upto = n;
#pragma unroll
    for (int d = 1; d < kMaxRanks; d <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += x;
    }
    const int all = __shfl_sync(0xffffffffu, upto, kMaxRanks - 1);
    if (all > kList) return all;
    for (int i0 = threadIdx.x & ~31; i0 < all; i0 += kThreads) {
        const int i = i0 + lane;
        int q = 0, from = 0;
#pragma unroll
        for (int e = 0; e < kMaxRanks - 1; e++) {
            const int end = __shfl_sync(0xffffffffu, upto, e);
            if (i >= end) q = e + 1, from = end;
        }
        if (i < all) s.entry[i] = peer_load64(at_rank(&s.list[i - from], q));
    }
    __syncthreads();
    return all;
}
// Weights of the n entries, and for entry tid/2 the number and the weights of the better ones. n is at most kFew.
__device__ __forceinline__ int order(Shared &s, const Row &r, int n, Whole &above) {
    const int tid = threadIdx.x;
    if (tid < n) s.entry_weight[tid] = r.weigh(of_key((unsigned)(s.entry[tid] >> 32)));
    __syncthreads();
    int better = 0;
    above = 0;
    if ((tid & ~31) / 2 < n) {  // whole warps
        const Whole me = s.entry[min(tid / 2, n - 1)];
#pragma unroll 4
        for (int j = tid & 1; j < n; j += 2) {
            const bool b = s.entry[j] > me;
            better += b;
            above += b ? s.entry_weight[j] : 0;
        }
        better += __shfl_xor_sync(0xffffffffu, better, 1);
        above += __shfl_xor_sync(0xffffffffu, above, 1);
    }
    return better;
}
// Of the n entries (they are the kept logits in a range): the one at which the running count, or sum, from the best on reaches
// `target`. `hist` is zero before and after. In every CTA by itself.
template <bool SUM>
__device__ Whole nth_entry(Shared &s, const Row &r, int n, Range in, Whole target, Hist &hist) {
    const int tid = threadIdx.x;
    static_assert(kList == 2 * kThreads, "two entries to a thread");
    while (n > kFewer && in.low < in.high) {
        Whole mine[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            mine[i] = tid + i * kThreads < n ? s.entry[tid + i * kThreads] : 0;
            if (mine[i]) {
                const int bin = (int)((in.high - (unsigned)(mine[i] >> 32)) >> in.shift());
                add_to<SUM>(hist, bin, SUM ? r.weigh(of_key((unsigned)(mine[i] >> 32))) : 1);
            }
        }
        __syncthreads();
        if (tid == 0) s.few = 0;
        Whole sum = 0;
        if (tid < kBins) {
            sum = words(hist[0][tid], hist[1][tid]);  // (counts: the high words are zero)
            hist[0][tid] = hist[1][tid] = 0;
        }
        const Bin b = reach_bin(s, sum, target);
        const int shift = in.shift();
        target -= b.before;
        in.take_keys(b.bin, shift);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const unsigned k = (unsigned)(mine[i] >> 32);
            if (mine[i] && k >= in.low && k <= in.high) s.entry[atomicAdd(&s.few, 1)] = mine[i];
        }
        __syncthreads();
        n = s.few;
    }
    if (n <= kFewer) {
        Whole above;
        const int better = order(s, r, n, above);
        if (!(tid & 1) && tid / 2 < n && (SUM ? above < target && above + s.entry_weight[tid / 2] >= target : (Whole)better + 1 == target))
            s.found = s.entry[tid / 2];
        __syncthreads();
        return s.found;
    }
    // equal logits: by their index alone
    if (SUM) {
        const Whole one = r.weigh(of_key(in.low));
        target = (target + one - 1) / one;
    }
    for (int i = tid; i < n; i += kThreads) {
        int better = 0;
        const Whole me = s.entry[i];
        for (int j = 0; j < n; j++) better += s.entry[j] > me;
        if ((Whole)better + 1 == target) s.found = me;
    }
    __syncthreads();
    return s.found;
}

// The kept set ends at a listed entry. SUM: the threads' shares of what this CTA has in better bins are summed up; its own
// list is the rest.
template <bool SUM>
__device__ __forceinline__ void keep_to(const Shared &s, Row &r, Whole worst) {
    r.key = (unsigned)(worst >> 32), r.last = (int)~(unsigned)worst;
    if constexpr (SUM) {
        for (int i = threadIdx.x; i < s.listed; i += kThreads)
            if (s.list[i] >= worst) r.share += r.weigh(of_key((unsigned)(s.list[i] >> 32)));
        r.known = true;
    }
}

// Narrows the kept set to its largest logits: of those in a range, `target` (SUM: as many as it takes until their weights reach
// it). linear: the first bins are distances.
template <bool SUM>
__device__ void narrow(Shared &s, Row &r, Whole target, Range in, bool linear, int &pass, int &turn) {
    const int tid = threadIdx.x, lane = tid & 31;
    for (; linear || in.low < in.high; linear = false) {
        const int shift = in.shift();
        Hist &hist = s.hist[pass & 1], &other = s.hist[~pass & 1];  // (zeros)
        r.some(of_key(max(in.low, kNone + 1)), in.highest(), [&](const float (&x)[2], const int (&at)[2]) {
            const Whole w[2] = {SUM ? r.weigh(x[0]) : 1, SUM ? r.weigh(x[1]) : 1};
#pragma unroll
            for (int e = 0; e < 2; e++)
                if (r.kept_of_floor(x[e], at[e]) && in.has(x[e]))
                    add_to<SUM>(hist, linear ? in.bin_of(x[e]) : (int)((in.high - key_of(x[e])) >> shift), w[e]);
        });
        cluster_sync();
        const Whole mine = all_bins<SUM>(s, r, hist);
        // the other histogram, and the list, were read before this pass's barrier
        for (int i = tid; i < 2 * kBins; i += kThreads) other[0][i] = 0;
        if (tid == 0) s.listed = 0;
        pass++;
        const Bin b = reach_bin(s, mine, target);
        if (b.bin < 0) return;  // all of them
        target -= b.before;
        if (SUM && tid < b.bin) r.share += words(hist[0][tid], hist[1][tid]);
        if (linear) in.take_bin(b.bin);
        else in.take_keys(b.bin, shift);
        const int n = gather(s, r, in);
        if (n <= kList) {
            keep_to<SUM>(s, r, nth_entry<SUM>(s, r, n, in, target, other));
            return;
        }
    }
    // more equal logits than are listed: the first ones
    const Whole one = SUM ? r.weigh(of_key(in.low)) : 1;
    if (SUM) target = (target + one - 1) / one;
    auto tie = [&](float x, int index) { return (Whole)(key_of(x) == in.low && r.keeps(x, index)); };
    Whole n = 0, all;
    r.each([&](float x, int index) { n += tie(x, index); });
    share_sums(s, r, n, turn);
    const Whole before = sums_before(s, r, turn, all);
    turn++;
    const int index = reach(s, r, n, before, target, tie);
    if (index >= 0 && lane < r.ranks) peer_store(at_rank(&s.last[SUM], lane), (unsigned)index);
    cluster_sync();
    r.key = in.low;
    r.last = s.last[SUM];
}

// The whole number that a sum must reach to be at least p of `all`.
__device__ __forceinline__ Whole share_of(float p, Whole all) {
    const Whole share = p > 0.0f ? __double2ull_rz((double)p * 18446744073709551616.0) : 0;
    return max(__umul64hi(share, all) + (share * all != 0), 1ull);
}
// How far below the largest weight, in octaves, a logit must lie so that all of them there together are less than what top-p
// leaves out. The sum is one largest weight at least.
__device__ __forceinline__ float octaves_of(float p, int vocab) { return log2f((float)vocab) - log2f(1.0f - fmaxf(p, 0.0f)) + 1.0f; }

// The kept set ends where the n entries' weights, from the best on, reach `target`. With `settle`, s.total[turn & 1] has what the
// CTAs keep besides, and has all of it after.
__device__ __forceinline__ void cut_list(Shared &s, Row &r, int n, const Range &in, Whole target, bool settle, int pass, int turn) {
    const int tid = threadIdx.x;
    Whole mine[2];
#pragma unroll
    for (int i = 0; i < 2; i++) mine[i] = tid + i * kThreads < n ? s.entry[tid + i * kThreads] : 0;
    Hist &hist = s.hist[pass & 1];
    const Whole worst = nth_entry<true>(s, r, n, in, target, hist);
    r.key = (unsigned)(worst >> 32), r.last = (int)~(unsigned)worst;
    if (!settle) return;
#pragma unroll
    for (int i = 0; i < 2; i++)
        if (mine[i] >= worst) {
            const int q = r.rank_of((int)~(unsigned)mine[i]);
            add_words(hist[0][q], hist[1][q], r.weigh(of_key((unsigned)(mine[i] >> 32))));
        }
    __syncthreads();
    if (tid < r.ranks) s.total[turn & 1][tid] += words(hist[0][tid], hist[1][tid]);
    __syncthreads();
    r.settled = true;
}

// Top-p of a kept set of kList logits at most, all of which every CTA then has.
__device__ void listed_nucleus(Shared &s, Row &r, float p, bool settle, int pass, int turn) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    cluster_sync();  // others have read this CTA's list
    if (tid == 0) s.listed = 0;
    if (tid < r.ranks) s.total[turn & 1][tid] = 0;
    __syncthreads();
    const Range in = {r.key, key_of(r.most), r.most, 0.0f, 0, -1};
    const int n = gather(s, r, in);
    Whole sum = 0;
    for (int i = tid; i < n; i += kThreads) sum += r.weigh(of_key((unsigned)(s.entry[i] >> 32)));
    sum = warp_sum(sum);
    if (lane == 0) s.warp_sum[warp] = sum;
    __syncthreads();
    const Whole all = warp_sum(lane < kWarps ? s.warp_sum[lane] : 0);
    cut_list(s, r, n, in, share_of(p, all), settle, pass, turn);
}

// Top-p of a whole row: the sum of all weights and the bins of those that may matter, none of which lie below `end`, in one pass.
// s.fine is zero before. Where it comes down to a list, what the CTAs keep is in s.total[turn & 1] (for `settle`).
__device__ void nucleus(Shared &s, Row &r, float p, float end, bool settle, int &pass, int &turn) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    Range in = {key_of(end), key_of(r.most), r.most, fminf((kFine - 0.001f) / (r.most - end), 1e30f), kFine - 1, -1};
    Whole sum = 0;
    r.each_weight(-INFINITY, [&](const float (&x)[4], int, const Whole (&w)[4]) {
        sum += (w[0] + w[1]) + (w[2] + w[3]);
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (x[e] >= end) {
                const int bin = (int)((in.most - x[e]) * in.scale);  // bin_of: kFine is not reached
                add_words(s.fine[0][bin], s.fine[1][bin], w[e]);
            }
    });
    share_sums(s, r, sum, turn, [&] {  // and the sums of groups of 32 bins
#pragma unroll
        for (int g = warp; g < kFine / 32; g += kWarps) {
            const Whole of_group = warp_sum(words(s.fine[0][32 * g + lane], s.fine[1][32 * g + lane]));
            if (lane < r.ranks) peer_store(at_rank(&s.read[r.rank][g], lane), of_group);
        }
    });
    Whole all;
    sums_before(s, r, turn, all);
    turn++;
    Whole target = share_of(p, all);
    // the group, then the bin in it, by every warp
    auto find = [&]() {
        Whole mine = 0;
#pragma unroll 1
        for (uint32_t q0 = 0; q0 < r.ranks; q0 += 8)
#pragma unroll
            for (uint32_t q = q0; q < q0 + 8; q++) mine += q < r.ranks ? s.read[q][lane] : 0;
        const Whole upto = warp_scan(mine);
        const unsigned past = __ballot_sync(0xffffffffu, upto >= target);
        if (!past) return -1;
        const int l = __ffs(past) - 1;
        target -= __shfl_sync(0xffffffffu, upto - mine, l);
        return l;
    };
    const int group = find();
    if (group < 0) return;  // all of them
    // a warp reads one CTA's
    Whole better = 0, of_bin = 0;
    if (warp < r.ranks) {
        better = lane < group ? s.read[warp][lane] : 0;
        const unsigned low = peer_load(at_rank(&s.fine[0][32 * group + lane], warp)), high = peer_load(at_rank(&s.fine[1][32 * group + lane], warp));
        of_bin = words(low, high);
    }
    __syncthreads();
    if (warp < r.ranks) s.read[warp][lane] = of_bin;
    __syncthreads();
    const int bin = find();
    if (settle && warp < r.ranks) {
        better = warp_sum(better + (lane < bin ? of_bin : 0));
        if (lane == 0) s.total[turn & 1][warp] = better;
    }
    in.take_bin(32 * group + bin);
    const int n = gather(s, r, in);
    if (n > kList) {
        if (settle && tid == 0) r.share = s.total[turn & 1][r.rank];
        narrow<true>(s, r, target, in, false, pass, turn);
        return;
    }
    cut_list(s, r, n, in, target, settle, pass, turn);
}

// Bins a quarter wide around the logits that models give, and the lowest logit of one. They serve to leave out most logits
// early, before the largest is known: logits that lie elsewhere (log-probabilities, for instance) are passed over once more. 40 lower
// or higher, 256 rows of 131,072 with top-k 40 and top-p 0.95 take 178 us for 78, with top-k 200 and min-p 154 for 121, with top-k 1000 and
// top-p 0.8 209 for 178; one row 17 for 8.4, 14 for 11, 20 for 18.5.
__device__ __forceinline__ int plain_bin(float x) { return (int)fminf(fmaxf((24.0f - x) * 4.0f, 0.0f), (float)(kBins - 1)); }
__device__ __forceinline__ float plain_edge(int bin) { return 24.0f - 0.25f * (bin + 1) - 1e-4f; }
// A lower bound of the k-th largest logit, from bins of each thread's largest, in s.hist[0] (k logits are at least as large as
// the k-th largest of these); -infinity where there is none. many: so many logits are above it for sure that a list
// will hardly do.
__device__ float bound_of(Shared &s, const Row &r, int k, bool &many, int &pass) {
    const Whole count = all_bins<false>(s, r, s.hist[pass & 1]);
    pass++;  // (the next pass clears this histogram)
    const Bin b = reach_bin(s, count, k);
    many = __syncthreads_or((int)threadIdx.x == b.bin && b.before + count > kList / 2);
    return b.bin < 0 || b.bin == kBins - 1 ? -INFINITY : plain_edge(b.bin);
}

// One row, by one cluster.
__device__ __forceinline__ void do_row(const SampleArgs &a, Shared &s, float4 *part, Row &r, int row, int next) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, stride = a.units | 1;
    const int user = row / a.per;
    const float *const x0 = a.logits + (size_t)row * a.vocab;
    const int ahead = (int)(reinterpret_cast<uintptr_t>(x0) >> 2 & 3);  // logits between a multiple of 16 bytes and the row
    const int start = (int)r.rank * a.units * kStep - ahead;
    r.index = start + tid * 4 * a.units;
    r.ahead = ahead, r.inverse = a.inverse;
    const float t = a.temperature ? a.temperature[user] : 1.0f, p = a.top_p ? a.top_p[user] : 1.0f, least = a.min_p ? a.min_p[user] : 0.0f;
    // (min-p above 1 leaves the token that is always kept, and of equals that is the first: what top-k leaves with 1)
    const int asked = a.top_k ? a.top_k[user] : 0, k = least > 1.0f ? 1 : asked;
    const float u = a.uniforms ? a.uniforms[row] : 0.0f;

    // ---- the row, and its largest logit. A warp copies its threads' units, neighbouring ones at a time.
    float most = -INFINITY;
    __syncwarp();  // (its lanes are done with the row before)
    {
        float4 *const to = part + warp * 32 * stride;
        const int from = start + warp * 32 * 4 * a.units;
        for (int j0 = 0; j0 < a.units; j0 += 8) {
            float4 x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int at = (j0 + j) * 32 + lane, i = from + 4 * at;
                x[j] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                if (j0 + j < a.units) {
                    if (i >= 0 && i + 3 < a.vocab) x[j] = __ldcs(reinterpret_cast<const float4 *>(x0 + i));
                    else {
                        if (i >= 0 && i < a.vocab) x[j].x = x0[i];
                        if (i + 1 >= 0 && i + 1 < a.vocab) x[j].y = x0[i + 1];
                        if (i + 2 >= 0 && i + 2 < a.vocab) x[j].z = x0[i + 2];
                        if (i + 3 >= 0 && i + 3 < a.vocab) x[j].w = x0[i + 3];
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j0 + j < a.units) {
                    const int at = (j0 + j) * 32 + lane, owner = a.owner_of(at);
                    x[j].x += 0.0f, x[j].y += 0.0f, x[j].z += 0.0f, x[j].w += 0.0f;  // -0 is 0: equals go by their index
                    to[owner * stride + (at - owner * a.units)] = x[j];
                    most = max_nan(max_nan(max_nan(most, x[j].x), max_nan(x[j].y, x[j].z)), x[j].w);
                }
        }
    }
    if (next < a.rows) {  // the cluster's next row comes to L2 meanwhile
        const float *const x1 = a.logits + (size_t)next * a.vocab;
        for (int i = max(0, start) + tid * 32; i < min(a.vocab, start + a.units * kStep); i += kThreads * 32)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(x1 + i));
    }
    const float threads_most = most;
    const double octaves_per_logit = 1.4426950408889634 / (t > 0.0f ? (double)t : 1.0), logits_per_octave = 0.6931471805599453 * (t > 0.0f ? (double)t : 1.0);
    const double nucleus_below = p < 1.0f ? fminf(octaves_of(p, a.vocab), 46.0f) * logits_per_octave : 0.0;
    const double min_below = least > 0.0f ? (double)t * log((double)least) : 0.0;
    // ---- the largest logit of all (as a key: a NaN's is above all), with temperature 0 its lowest index too. For top-k, bins of the
    // threads' largest go along.
    unsigned top = key_of(most), low = most > -INFINITY ? top : ~0u;  // the lowest: of the threads' largest
    top = __reduce_max_sync(0xffffffffu, top);
    low = __reduce_min_sync(0xffffffffu, low);
    if (lane == 0) s.warp_most[warp] = top, s.warp_least[warp] = low;
    // (what this CTA's memory held of the row before is read by others until they are here)
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    const bool cut_k = k > 0 && k < a.vocab && t > 0.0f;
    for (int i = tid; i < 2 * 2 * kBins; i += kThreads) s.hist[0][0][i] = 0;
    if (!cut_k && p < 1.0f)
        for (int i = tid; i < 2 * kFine; i += kThreads) s.fine[0][i] = 0;
    if (tid == 0) s.listed = 0;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, lane < kWarps ? s.warp_most[lane] : 0);
    low = __reduce_min_sync(0xffffffffu, lane < kWarps ? s.warp_least[lane] : ~0u);
    if (t == 0.0f) {
        unsigned index = 0x7fffffff;
        r.some(of_key(top), of_key(top), [&](const float (&x)[2], const int (&at)[2]) {
#pragma unroll
            for (int e = 0; e < 2; e++)
                if (x[e] == of_key(top)) index = min(index, (unsigned)at[e]);
        });
        index = __reduce_min_sync(0xffffffffu, index);
        if (lane == 0) s.warp_sum[warp] = index;
        __syncthreads();
        low = __reduce_min_sync(0xffffffffu, lane < kWarps ? (unsigned)s.warp_sum[lane] : 0x7fffffffu);
    } else if (cut_k && threads_most > -INFINITY) {
        atomicAdd(&s.hist[0][0][plain_bin(threads_most)], 1u);
    }
    if (warp == 0 && lane < r.ranks) peer_store(at_rank(&s.ends[r.rank], lane), (Whole)top << 32 | ~low);
    cluster_sync();
    // of equal keys the lowest index; without temperature 0, the lowest of all
    const Whole of_rank = lane < r.ranks ? s.ends[lane] : 0;
    const unsigned most_key = __reduce_max_sync(0xffffffffu, (unsigned)(of_rank >> 32)), least_key = __reduce_min_sync(0xffffffffu, ~(unsigned)of_rank);
    most = of_key(most_key);
    const float lowest = least_key == ~0u ? most : of_key(least_key);
    const bool refused = !(most > -INFINITY && most < INFINITY) || !(t >= 0.0f && t < INFINITY) || p != p || least != least || u != u;

    // ---- what is kept
    auto bins_down_to = [&](float x) { return fminf(kBins / (most - x), 1e30f); };
    int turn = 0, pass = 0;
    r.most = most;
    r.top = most;
    r.c = octaves_per_logit;
    r.zero = fmaxf((float)(r.top - 46.0 * logits_per_octave), kLowest);
    r.share = 0, r.known = r.settled = false;
    r.key = kNone, r.last = -0x7fffffff;  // (what lies outside the row has indices from -3 on)
    const unsigned min_key = [&]() -> unsigned {  // of the lowest logit that min_p leaves
        if (!(least > 0.0f)) return 0;
        const double border = r.top + min_below;
        return border >= r.top ? key_of(most) : key_of(__double2float_ru(border));
    }();
    int token = -1;  // where it is known already
    if (refused) {
    } else if (t == 0.0f) {  // the largest logit, the lowest index of equals
        r.key = most_key, r.last = (int)~__reduce_max_sync(0xffffffffu, (unsigned)(of_rank >> 32) == most_key ? (unsigned)of_rank : 0);
        token = r.last;
    } else {
        bool done = false;
        if (cut_k) {
            int n = kList + 1;
            bool many;
            const float bound = bound_of(s, r, k, many, pass);
            const Range upward = {key_of(bound), key_of(most), most, 0.0f, 0, -1};
            if (!many && bound > -INFINITY) n = gather(s, r, upward);
            if (n <= kFew) {
                // few enough: all of the rest is in every CTA's own memory
                Whole above;
                const int better = order(s, r, n, above), held = min(k, n), me = tid / 2;
                const bool one = !(tid & 1) && me < n;
                if (one && better == held - 1) s.kept_sum = above + s.entry_weight[me];
                __syncthreads();
                bool stays = one && better < k;
                if (p < 1.0f) {
                    const Whole target = share_of(p, s.kept_sum);
                    stays = stays && above < target;
                }
                stays = stays && (unsigned)(s.entry[min(me, n - 1)] >> 32) >= min_key;
                const int kept = __syncthreads_count(stays);
                if (one && better == kept - 1) s.found = s.entry[me], s.kept_sum = above + s.entry_weight[me];
                __syncthreads();
                const Whole worst = s.found;
                r.key = (unsigned)(worst >> 32), r.last = (int)~(unsigned)worst;
                done = true;
                if (a.token) {
                    // among what is kept, the weights at lower indices
                    const float v = fminf(fmaxf(u, 0.0f), 0.99999994f);
                    const Whole aim = __umul64hi(__double2ull_rz((double)v * 18446744073709551616.0), s.kept_sum) + 1;
                    if ((tid & ~31) / 2 < n) {
                        const Whole entry = s.entry[min(me, n - 1)];
                        Whole before = 0;
                        for (int j = tid & 1; j < n; j += 2) {
                            const Whole e = s.entry[j];
                            if (e >= worst && (unsigned)e > (unsigned)entry) before += s.entry_weight[j];
                        }
                        before += __shfl_xor_sync(0xffffffffu, before, 1);
                        if (one && entry >= worst && before < aim && before + s.entry_weight[me] >= aim && r.rank == 0)
                            a.token[row] = (int)~(unsigned)entry;
                    }
                    return;
                }
            } else if (n <= kList) {
                keep_to<false>(s, r, nth_entry<false>(s, r, n, upward, min(k, n), s.hist[pass & 1]));
            } else {
                narrow<false>(s, r, k, {key_of(bound), key_of(most), most, bins_down_to(fmaxf(bound, lowest)), kBins - 1, -1}, true, pass, turn);
            }
        }
        if (!done && p < 1.0f) {
            const float end = fmaxf((float)(r.top - nucleus_below), kLowest);
            if (r.key == kNone) {
                if (cut_k) {
                    for (int i = tid; i < 2 * kFine; i += kThreads) s.fine[0][i] = 0;
                    __syncthreads();
                }
                nucleus(s, r, p, end, a.token, pass, turn);
            } else if (k <= kList) {
                listed_nucleus(s, r, p, a.token, pass, turn);
            } else {
                Whole all;
                share_sums(s, r, r.kept_sum(), turn);
                sums_before(s, r, turn, all);
                turn++;
                narrow<true>(s, r, share_of(p, all), {max(key_of(end), r.key), key_of(most), most, bins_down_to(fmaxf(end, r.floor())), kBins - 1, -1},
                             true, pass, turn);
            }
        }
        if (!done && min_key > r.key) {
            r.key = min_key, r.last = 0x7fffffff;
            turn += r.settled;  // (others may be at the next exchange already)
            r.known = r.settled = false;
        }
    }

    // ---- the token, or the logits
    if (a.token) {
        if (refused || t == 0.0f) {
            if (r.rank == 0 && tid == 0) a.token[row] = token;
            return;
        }
        auto mine = [&](float x, int index) { return r.keeps(x, index) ? r.weigh(x) : 0; };
        Whole sum = 0, all;
        if (!r.settled) {
            sum = r.known ? r.share : r.kept_sum();
            share_sums(s, r, sum, turn);
        }
        const Whole before = sums_before(s, r, turn, all);
        // the first running sum above u * all is the first that reaches the whole number after it
        const float v = fminf(fmaxf(u, 0.0f), 0.99999994f);
        const Whole aim = __umul64hi(__double2ull_rz((double)v * 18446744073709551616.0), all) + 1;
        if (r.settled || r.known) {  // by index, in the one CTA that has the token
            if (before >= aim || before + s.total[turn & 1][r.rank] < aim) return;
            sum = r.kept_sum();
            const Whole of_warp = warp_sum(sum);
            if (lane == 0) s.warp_sum[warp] = of_warp;
            __syncthreads();
        }
        const int index = reach(s, r, sum, before, aim, mine);
        if (index >= 0 && lane == 0) a.token[row] = index;
        return;
    }
    float *const out = a.out + (size_t)row * a.vocab;
    const float other = refused ? __int_as_float(0x7fc00000) : -INFINITY;
    const bool whole = !((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(x0)) & 15);
    const float4 *const from = part + warp * 32 * stride;
    for (int j = 0; j < a.units; j++) {
        const int at = j * 32 + lane, owner = a.owner_of(at), i = start + (warp * 32 * a.units + at) * 4;
        float4 x = from[owner * stride + (at - owner * a.units)];
        x.x = !refused && r.keeps(x.x, i) ? x.x : other;
        x.y = !refused && r.keeps(x.y, i + 1) ? x.y : other;
        x.z = !refused && r.keeps(x.z, i + 2) ? x.z : other;
        x.w = !refused && r.keeps(x.w, i + 3) ? x.w : other;
        if (whole && i >= 0 && i + 3 < a.vocab) __stcs(reinterpret_cast<float4 *>(out + i), x);
        else {
            if (i >= 0 && i < a.vocab) out[i] = x.x;
            if (i + 1 >= 0 && i + 1 < a.vocab) out[i + 1] = x.y;
            if (i + 2 >= 0 && i + 2 < a.vocab) out[i + 2] = x.z;
            if (i + 3 >= 0 && i + 3 < a.vocab) out[i + 3] = x.w;
        }
    }
}

__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ SampleArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    float4 *const part = reinterpret_cast<float4 *>(smem);
    Shared &s = *reinterpret_cast<Shared *>(part + kThreads * (a.units | 1));
    Row r;
    r.rank = cluster_rank(), r.ranks = cluster_size();
    r.units = a.units;
    r.mine = part + threadIdx.x * (a.units | 1);
    asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");  // a CTA's memory is there for others once it runs
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int clusters = gridDim.x / r.ranks;
    for (int row = blockIdx.x / r.ranks; row < a.rows; row += clusters) {
        do_row(a, s, part, r, row, row + clusters);
        // (nothing is handed over: others' memory was read, and what was read is used. A release would wait for the row's stores.)
        asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
    }
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");  // no CTA ends while others read its memory
}

constexpr int smem_of(int units) { return kThreads * (units | 1) * 16 + (int)sizeof(Shared); }
static_assert(smem_of(kMaxUnits) <= 232448, "shared memory");

int launch(SampleArgs &a, int rows) {
    // up to three logits may lie before a row that does not start on 16 bytes
    const bool aligned = !(reinterpret_cast<uintptr_t>(a.logits) & 15) && a.vocab % 4 == 0;
    const int long_row = a.vocab + (aligned ? 0 : 3);
    // Clusters of more CTAs take less time for a row, but fewer of them fit: as many as these, by what cudaOccupancyMaxActiveClusters
    // says of one B200 (another part's may be others, and then the choice is not the fastest), two CTAs to an SM (up to half its
    // memory each) or one. A row takes about as long for its fixed steps as for seven units of a thread, and 1.4 times as long
    // where CTAs share an SM. A nucleus of 0.9 with the number of CTAs that this takes, and
    // with others: 14 rows of 131,072 8 (21.7 us) or 16 (24.3); 17 rows 13 (26) or 8 (27.9); 256 rows 6 (200) or 8 (209);
    // 37 rows of 50,001 7 (22.4) or 4 (25.4); 60 rows of 200,000 9 (75) or 8 (103).
    static constexpr short kTwo[kMaxRanks] = {296, 148, 93, 71, 56, 45, 37, 33, 30, 26, 21, 21, 17, 14, 14, 14};
    static constexpr short kOne[kMaxRanks] = {148, 74, 45, 33, 26, 22, 15, 15, 15, 11, 7, 7, 7, 7, 7, 7};
    int ranks = 1, clusters = 1;
    long long best = 0;
    for (int n = 1; n <= kMaxRanks; n++) {
        const int units = ((long_row + n - 1) / n + kStep - 1) / kStep;
        if (units > kMaxUnits) continue;
        const bool half = smem_of(units) <= 115200;
        const int one = kOne[n - 1], fit = half ? kTwo[n - 1] : one, rest = rows % fit;
        const long long time = (long long)(7 + units) * ((long long)(rows / fit) * (half ? 7 : 5) + (rest > one ? 7 : rest ? 5 : 0));
        if (!best || time < best) best = time, ranks = n, clusters = rows < fit ? rows : fit, a.units = units;
    }
    const int smem = smem_of(a.units);
    // (the kernel's limits are the same in every call: another thread's, for a row of another length, may come before this launch)
    if (int rc = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_of(kMaxUnits))) return rc;
    if (int rc = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) return rc;
    a.inverse = 65535 / a.units + 1;
    a.rows = rows;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = launch_stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ranks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cfg.gridDim = dim3((unsigned)(clusters * ranks));
    return cudaLaunchKernelEx(&cfg, sample_kernel, a);
}

template <typename... T>
bool unaligned(const T *...p) { return ((reinterpret_cast<uintptr_t>(p) | ...) & 3) != 0; }

int settings(SampleArgs &a, const float *logits, const float *temperature, const int *top_k, const float *top_p, const float *min_p, int per,
             int rows, int vocab) {
    if (!logits || unaligned(logits, temperature, top_k, top_p, min_p) || per < 1 || rows < 1 || rows > kRowsAtOnce || vocab < 1 || vocab > kMaxVocab - 3)
        return cudaErrorInvalidValue;
    a.logits = logits;
    a.temperature = temperature;
    a.top_k = top_k;
    a.top_p = top_p;
    a.min_p = min_p;
    a.per = per;
    a.vocab = vocab;
    a.uniforms = nullptr;
    a.token = nullptr;
    a.out = nullptr;
    return 0;
}

}  // namespace

extern "C" int qg_sample(int *token, const float *logits, const float *uniforms, const float *temperature, const int *top_k, const float *top_p,
                         const float *min_p, int per, int rows, int vocab) {
    SampleArgs a;
    if (int rc = settings(a, logits, temperature, top_k, top_p, min_p, per, rows, vocab)) return rc;
    if (!token || !uniforms || unaligned(token, uniforms)) return cudaErrorInvalidValue;
    a.token = token;
    a.uniforms = uniforms;
    return launch(a, rows);
}

extern "C" int qg_truncate_logits(float *out, const float *logits, const float *temperature, const int *top_k, const float *top_p,
                                  const float *min_p, int per, int rows, int vocab) {
    SampleArgs a;
    if (int rc = settings(a, logits, temperature, top_k, top_p, min_p, per, rows, vocab)) return rc;
    if (!out || unaligned(out)) return cudaErrorInvalidValue;
    // a row is read before it is written, but rows are at work in any order
    const size_t bytes = (size_t)rows * vocab * sizeof(float);
    const uintptr_t x = reinterpret_cast<uintptr_t>(logits), y = reinterpret_cast<uintptr_t>(out);
    if (x != y && x < y + bytes && y < x + bytes) return cudaErrorInvalidValue;
    a.out = out;
    return launch(a, rows);
}

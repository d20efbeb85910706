// Sampling of the next token from what temperature, top-k, top-p and min-p leave of a distribution, and the logits with all
// else at -infinity.
//
// A cluster takes a row and keeps it in the shared memory of its CTAs, so that the logits are read once however many passes
// the row needs:
//     weight  W = 2^44 * 2^((x - max) * log2(e) / T), as a whole number
//     kept    the tokens from the largest on (the lowest index of equals first): top_k of them, then as many as it takes
//             until their sum reaches top_p of those, none below min_p of the largest
//     token   the first index at which the running sum of the kept exceeds u times their sum
// A set that is kept is always "all logits above a key, and those at the key up to an index". The key is found by counts (top-k)
// or sums (top-p) over 1024 bins, first of the distance to the maximum, then of the bits of the keys that are left.
//
// Weights are evaluated in 64 bits and summed as whole numbers: borders are compared exactly, and neither the cluster's
// size nor the order of atomics has a say. With weights in 32 bits a running sum is off by some 1e-8, and a tail of 100,000
// tokens of 1e-6 each is off by a token once in a hundred draws.
#include "cache.cuh"

using namespace nb;

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 1024;
constexpr int kPiece = 128;                       // logits that a warp takes at a time: four to a lane
constexpr int kStep = kWarps * kPiece;            // a CTA's part of a row is a multiple of this
constexpr int kMaxPart = 24 * kStep;              // 192 KB
constexpr int kMaxRanks = 8;                      // CTAs of a cluster
constexpr int kMaxVocab = kMaxRanks * kMaxPart;   // the sum of 2^44 for each still fits 63 bits
constexpr int kRowsAtOnce = 1 << 20;
static_assert(kMaxVocab <= 1 << 19, "sums of weights");

struct SampleArgs {
    const float *logits, *uniforms, *temperature, *top_p, *min_p;
    const int *top_k;
    float *out;
    int *token;
    int per, vocab, part;  // part: logits of a CTA
};

struct Top {
    float most;
    int odd;  // a NaN or +infinity
};
// What the CTAs of a cluster tell each other.
struct Shared {
    Top top[kMaxRanks];
    unsigned long long total[2][kMaxRanks];  // by the parity of the exchange: a CTA may be one ahead
    unsigned long long before;               // of the bin that was found
    unsigned long long warp_sum[kWarps];
    unsigned bin, count;
    int index[kMaxRanks];
    int last;                                // of the ties that are kept
    float warp_most[kWarps];
    int warp_odd[kWarps];
    unsigned hist[4][kBins];                 // counts; sums as 15 + 15 + 14 bits
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
__device__ __forceinline__ void peer_store(uint32_t a, unsigned x) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(x) : "memory"); }
__device__ __forceinline__ void peer_store(uint32_t a, unsigned long long x) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(x) : "memory");
}

// Whole numbers in the order of the floats.
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned b = __float_as_uint(x);
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(unsigned k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
constexpr unsigned kNone = 0x007fffffu;  // key of -infinity

// 2^44 * 2^((x - most) * c), rounded; c = log2(e) / T. The polynomial of degree 9 is 2^f's Chebyshev fit on [-1/2, 1/2]
// (error 2^-46).
__device__ __forceinline__ unsigned long long weight(float x, double most, double c) {
    const double t = ((double)x - most) * c;
    if (!(t > -46.0)) return 0;  // less than half a unit
    constexpr double kRound = 6755399441055744.0, kUnit = 4503599627370496.0;  // 1.5 * 2^52, 2^52
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
    const double v = __hiloint2double(__double2hiint(p) + ((__double2loint(n) + 44) << 20), __double2loint(p)) + kUnit;
    return (unsigned long long)__double_as_longlong(v) & 0xfffffffffffffull;
}

__device__ __forceinline__ unsigned long long warp_sum(unsigned long long x) {
#pragma unroll
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}
__device__ __forceinline__ unsigned long long warp_scan(unsigned long long x) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, x, d);
        if ((threadIdx.x & 31) >= d) x += y;
    }
    return x;
}

// One CTA's view of a row.
struct Row {
    const float *part;  // its logits, in shared memory; what lies outside the row is -infinity
    int pieces;         // of each warp
    int start;          // index of the first logit (may be negative, where the row does not start on 16 bytes)
    uint32_t rank, ranks;
    float most;
    double top, c;
    unsigned key;       // kept: logits above the key, and those at it up to index `last`
    int last;

    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll 2
        for (int i = 0; i < pieces; i++) {
            const int at = (warp * pieces + i) * kPiece + lane * 4;
            const float4 x = *reinterpret_cast<const float4 *>(part + at);
            f(x.x, start + at), f(x.y, start + at + 1), f(x.z, start + at + 2), f(x.w, start + at + 3);
        }
    }
    __device__ __forceinline__ bool keeps(float x, int index) const {
        const unsigned k = key_of(x);
        return k > key || (k == key && index <= last);
    }
    __device__ __forceinline__ unsigned long long weigh(float x) const { return weight(x, top, c); }
};

// Of 64-bit sums of the threads: the warps' to s.warp_sum, the CTAs' to s.total[turn] of all. Ends with a barrier of the
// cluster.
__device__ __forceinline__ void share_sums(Shared &s, const Row &r, unsigned long long x, int turn) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    x = warp_sum(x);
    if (lane == 0) s.warp_sum[warp] = x;
    __syncthreads();
    if (warp == 0) {
        const unsigned long long all = warp_sum(lane < kWarps ? s.warp_sum[lane] : 0);
        if (lane < r.ranks) peer_store(at_rank(&s.total[turn & 1][r.rank], lane), all);
    }
    cluster_sync();
}
// Totals of the CTAs before this one, and of all.
__device__ __forceinline__ unsigned long long sums_before(const Shared &s, const Row &r, int turn, unsigned long long &all) {
    unsigned long long before = 0;
    all = 0;
    for (uint32_t i = 0; i < r.ranks; i++) {
        const unsigned long long x = s.total[turn & 1][i];
        if (i < r.rank) before += x;
        all += x;
    }
    return before;
}
// The index at which the running sum of f (in the order of indices) reaches `target`, for the one warp that holds it; -1 for
// all others. After share_sums of the same f.
template <typename F>
__device__ int reach(const Shared &s, const Row &r, unsigned long long before, unsigned long long target, F f) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned long long mine = lane < kWarps ? s.warp_sum[lane] : 0, upto = warp_scan(mine) + before;
    const unsigned past = __ballot_sync(0xffffffffu, lane < kWarps && upto >= target);
    if (!past || __ffs(past) - 1 != warp) return -1;
    unsigned long long base = __shfl_sync(0xffffffffu, upto - mine, warp);
    if (base >= target) return -1;  // (an earlier CTA's)
    for (int i = 0; i < r.pieces; i++) {
        const int at = (warp * r.pieces + i) * kPiece + lane * 4;
        const float4 x = *reinterpret_cast<const float4 *>(r.part + at);
        const unsigned long long w[4] = {f(x.x, r.start + at), f(x.y, r.start + at + 1), f(x.z, r.start + at + 2), f(x.w, r.start + at + 3)};
        const unsigned long long four = w[0] + w[1] + w[2] + w[3], here = warp_scan(four) + base;
        const unsigned hit = __ballot_sync(0xffffffffu, here >= target);
        if (hit) {
            const int l = __ffs(hit) - 1;
            unsigned long long run = here - four;
            int index = r.start + at;
#pragma unroll
            for (int e = 0; e < 3; e++) {
                run += w[e];
                if (run < target) index++;
                else break;
            }
            return __shfl_sync(0xffffffffu, index, l);
        }
        base = __shfl_sync(0xffffffffu, here, 31);
    }
    return -1;
}

// The lowest key whose logit has a distance bin of at most `bin`. Each round, the lanes try 32 keys.
__device__ unsigned lowest_key(float most, float scale, int bin) {
    const int lane = threadIdx.x & 31;
    const unsigned high = key_of(most);
    unsigned a = 0;
    for (int shift = 27; shift >= 0; shift = shift ? max(shift - 5, 0) : -1) {
        const unsigned long long k = a + ((unsigned long long)lane << shift);
        const bool below = lane == 0 || (k < high && (k <= kNone || min(kBins - 1, (int)((most - of_key((unsigned)k)) * scale)) > bin));
        a += (unsigned)(__popc(__ballot_sync(0xffffffffu, below)) - 1) << shift;
    }
    return a + 1;
}

// Narrows the kept set to its largest logits: `target` of them (SUM: as many as it takes until their weights reach it).
// `octaves`: bins of the first pass reach so far below the largest weight.
template <bool SUM>
__device__ void narrow(Shared &s, Row &r, unsigned long long target, float octaves, int &turn) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int bins = kBins / r.ranks, bin0 = r.rank * bins;  // that this CTA adds up
    const float scale = fminf((float)((kBins - 1) / (double)octaves * r.c), 1e30f);
    const unsigned lowest = r.key;
    unsigned low = r.key, high = key_of(r.most);
    bool linear = true;
    while (linear || low < high) {
        const int shift = linear ? 0 : max(0, 22 - __clz(high - low));  // (high - low) >> shift < kBins
        for (int i = tid; i < 4 * kBins; i += kThreads) s.hist[0][i] = 0;
        __syncthreads();
        r.each([&](float x, int index) {
            const unsigned k = key_of(x);
            if (k < low || k > high || !r.keeps(x, index)) return;
            const int bin = linear ? min(kBins - 1, (int)((r.most - x) * scale)) : (int)((high - k) >> shift);
            atomicAdd(&s.hist[0][bin], 1u);
            if (SUM) {
                const unsigned long long w = r.weigh(x);
                atomicAdd(&s.hist[1][bin], (unsigned)w & 0x7fffu);
                atomicAdd(&s.hist[2][bin], (unsigned)(w >> 15) & 0x7fffu);
                atomicAdd(&s.hist[3][bin], (unsigned)(w >> 30));
            }
        });
        cluster_sync();
        // this CTA's bins over all CTAs, one bin to a thread and pass; warps' sums go through s.warp_sum
        unsigned long long upto[2], mine[2];
        unsigned count[2];
        unsigned long long sum = 0;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int b = 2 * tid + i;
            mine[i] = 0, count[i] = 0;
            if (b < bins) {
                unsigned long long part[3] = {0, 0, 0};
                for (uint32_t q = 0; q < r.ranks; q++) {
                    const uint32_t a = at_rank(&s.hist[0][bin0 + b], q);
                    count[i] += peer_load(a);
                    if (SUM)
                        for (int e = 0; e < 3; e++) part[e] += peer_load(a + (e + 1) * kBins * 4);
                }
                mine[i] = SUM ? part[0] + (part[1] << 15) + (part[2] << 30) : count[i];
            }
            sum += mine[i];
        }
        share_sums(s, r, sum, turn);
        unsigned long long all;
        unsigned long long before = sums_before(s, r, turn, all);
        turn++;
        if (all < target) return;  // all of them
        for (int i = 0; i < warp; i++) before += s.warp_sum[i];
        before += warp_scan(sum) - sum;
        upto[0] = before + mine[0], upto[1] = upto[0] + mine[1];
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (upto[i] >= target && upto[i] - mine[i] < target)
                for (uint32_t q = 0; q < r.ranks; q++) {
                    peer_store(at_rank(&s.bin, q), (unsigned)(bin0 + 2 * tid + i));
                    peer_store(at_rank(&s.count, q), count[i]);
                    peer_store(at_rank(&s.before, q), upto[i] - mine[i]);
                }
        cluster_sync();
        const int bin = s.bin;
        const bool whole = s.count == 1 || (!SUM && s.count == target - s.before);
        target -= s.before;
        if (linear) {
            if (bin) high = min(high, lowest_key(r.most, scale, bin - 1) - 1);
            low = max(low, lowest_key(r.most, scale, bin));
            linear = false;
        } else {
            high -= (unsigned)bin << shift;
            const unsigned span = (1u << shift) - 1;
            low = high - low > span ? high - span : low;
        }
        if (whole) {  // the bin ends the set
            if (low > lowest) r.last = 0x7fffffff;  // (at the lowest key fewer may have been kept before)
            r.key = low;
            return;
        }
    }
    // equal logits: the first ones
    const unsigned long long each = SUM ? r.weigh(of_key(low)) : 1;
    if (SUM) target = (target + each - 1) / each;
    auto tie = [&](float x, int index) { return (unsigned long long)(key_of(x) == low && r.keeps(x, index)); };
    unsigned long long n = 0;
    r.each([&](float x, int index) { n += tie(x, index); });
    share_sums(s, r, n, turn);
    unsigned long long all;
    const unsigned long long before = sums_before(s, r, turn, all);
    turn++;
    const int index = reach(s, r, before, target, tie);
    if (index >= 0 && lane < r.ranks) peer_store(at_rank(&s.last, lane), (unsigned)index);
    cluster_sync();
    r.key = low;
    r.last = s.last;
}

__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ SampleArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    float *const part = reinterpret_cast<float *>(smem);
    Shared &s = *reinterpret_cast<Shared *>(part + a.part);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");  // a CTA's memory is there for others once it runs
    Row r;
    r.part = part;
    r.rank = cluster_rank(), r.ranks = cluster_size();
    r.pieces = a.part / kStep;
    const int row = blockIdx.x / r.ranks, user = row / a.per;
    const float *const x0 = a.logits + (size_t)row * a.vocab;
    const int ahead = (int)(reinterpret_cast<uintptr_t>(x0) >> 2 & 3);  // logits between a multiple of 16 bytes and the row
    r.start = (int)r.rank * a.part - ahead;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const float t = a.temperature ? a.temperature[user] : 1.0f, p = a.top_p ? a.top_p[user] : 1.0f, least = a.min_p ? a.min_p[user] : 0.0f;
    const int k = a.top_k ? a.top_k[user] : 0;
    const float u = a.uniforms ? a.uniforms[row] : 0.0f;

    // ---- the row, and its largest logit
    float most = -INFINITY;
    bool odd = false;
#pragma unroll 8
    for (int i = 0; i < r.pieces; i++) {
        const int at = (warp * r.pieces + i) * kPiece + lane * 4, index = r.start + at;
        float4 x = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (index >= 0 && index + 3 < a.vocab) x = __ldcs(reinterpret_cast<const float4 *>(x0 + index));
        else {
            if (index >= 0 && index < a.vocab) x.x = x0[index];
            if (index + 1 >= 0 && index + 1 < a.vocab) x.y = x0[index + 1];
            if (index + 2 >= 0 && index + 2 < a.vocab) x.z = x0[index + 2];
            if (index + 3 >= 0 && index + 3 < a.vocab) x.w = x0[index + 3];
        }
        x.x += 0.0f, x.y += 0.0f, x.z += 0.0f, x.w += 0.0f;  // -0 is 0: equals go by their index
        *reinterpret_cast<float4 *>(part + at) = x;
        most = fmaxf(fmaxf(fmaxf(most, x.x), fmaxf(x.y, x.z)), x.w);
        odd |= !(x.x < INFINITY && x.y < INFINITY && x.z < INFINITY && x.w < INFINITY);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
    odd = __any_sync(0xffffffffu, odd);
    if (lane == 0) s.warp_most[warp] = most, s.warp_odd[warp] = odd;
    __syncthreads();
    if (warp == 0) {
        most = lane < kWarps ? s.warp_most[lane] : -INFINITY;
        odd = lane < kWarps && s.warp_odd[lane];
#pragma unroll
        for (int d = 16; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
        odd = __any_sync(0xffffffffu, odd);
    }
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    if (warp == 0) {
        if (lane < r.ranks) {
            peer_store(at_rank(&s.top[r.rank].most, lane), __float_as_uint(most));
            peer_store(at_rank(&s.top[r.rank].odd, lane), (unsigned)odd);
        }
    }
    cluster_sync();
    most = -INFINITY, odd = false;
    for (uint32_t i = 0; i < r.ranks; i++) most = fmaxf(most, s.top[i].most), odd |= s.top[i].odd != 0;
    const bool refused = odd || most == -INFINITY || !(t >= 0.0f && t < INFINITY) || p != p || least != least || u != u;

    // ---- what is kept
    int turn = 0;
    r.most = most;
    r.top = most;
    r.c = 1.4426950408889634 / (t > 0.0f ? (double)t : 1.0);
    r.key = kNone, r.last = -0x7fffffff;  // (what lies outside the row has indices from -3 on)
    if (!refused) {
        if (t == 0.0f) {  // the largest logit, the lowest index of equals
            int index = 0x7fffffff;
            r.each([&](float x, int at) { if (x == most) index = min(index, at); });
            index = __reduce_min_sync(0xffffffffu, index);
            if (lane == 0) s.warp_odd[warp] = index;
            __syncthreads();
            if (warp == 0) {
                index = __reduce_min_sync(0xffffffffu, lane < kWarps ? s.warp_odd[lane] : 0x7fffffff);
                if (lane < r.ranks) peer_store(at_rank(&s.index[r.rank], lane), (unsigned)index);
            }
            cluster_sync();
            r.key = key_of(most), r.last = 0x7fffffff;
            for (uint32_t i = 0; i < r.ranks; i++) r.last = min(r.last, s.index[i]);
        } else {
            if (k > 0 && k < a.vocab) narrow<false>(s, r, k, 32.0f, turn);
            if (p < 1.0f) {
                unsigned long long sum = 0, all;
                r.each([&](float x, int index) { if (r.keeps(x, index)) sum += r.weigh(x); });
                share_sums(s, r, sum, turn);
                sums_before(s, r, turn, all);
                turn++;
                const unsigned long long share = p > 0.0f ? __double2ull_rz((double)p * 18446744073709551616.0) : 0;
                const unsigned long long target = __umul64hi(share, all) + (share * all != 0);
                // What lies a factor of vocab / (what may be left out) below the largest cannot reach into it.
                const float left = (1.0f - fmaxf(p, 0.0f)) * (float)all * (1.0f / 17592186044416.0f);
                const float octaves = fminf(fmaxf(log2f((float)a.vocab) - log2f(left) + 1.0f, 1.0f), 46.0f);
                narrow<true>(s, r, target > 1 ? target : 1, octaves, turn);
            }
            if (least > 0.0f) {
                const double border = r.top + (double)t * log((double)least);
                const unsigned key = border >= r.top ? key_of(most) : key_of(__double2float_ru(border));
                if (key > r.key) r.key = key, r.last = 0x7fffffff;
            }
        }
    }

    // ---- the token, or the logits
    if (a.token) {
        if (refused) {
            if (r.rank == 0 && tid == 0) a.token[row] = -1;
            return;
        }
        if (t == 0.0f) {
            if (r.rank == 0 && tid == 0) a.token[row] = r.last;
            return;
        }
        auto mine = [&](float x, int index) { return r.keeps(x, index) ? r.weigh(x) : 0; };
        unsigned long long sum = 0, all;
        r.each([&](float x, int index) { sum += mine(x, index); });
        share_sums(s, r, sum, turn);
        const unsigned long long before = sums_before(s, r, turn, all);
        // the first running sum above u * all is the first that reaches the whole number after it
        const float v = fminf(fmaxf(u, 0.0f), 0.99999994f);
        const unsigned long long aim = __umul64hi(__double2ull_rz((double)v * 18446744073709551616.0), all) + 1;
        const int index = reach(s, r, before, aim, mine);
        if (index >= 0 && lane == 0) a.token[row] = index;
        return;
    }
    float *const out = a.out + (size_t)row * a.vocab;
    const float other = refused ? __int_as_float(0x7fc00000) : -INFINITY;
    if (!((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(x0)) & 15)) {
        for (int i = 0; i < r.pieces; i++) {
            const int at = (warp * r.pieces + i) * kPiece + lane * 4, index = r.start + at;
            float4 x = *reinterpret_cast<const float4 *>(part + at);
            x.x = !refused && r.keeps(x.x, index) ? x.x : other;
            x.y = !refused && r.keeps(x.y, index + 1) ? x.y : other;
            x.z = !refused && r.keeps(x.z, index + 2) ? x.z : other;
            x.w = !refused && r.keeps(x.w, index + 3) ? x.w : other;
            if (index >= 0 && index + 3 < a.vocab) __stcs(reinterpret_cast<float4 *>(out + index), x);
            else {
                if (index >= 0 && index < a.vocab) out[index] = x.x;
                if (index + 1 >= 0 && index + 1 < a.vocab) out[index + 1] = x.y;
                if (index + 2 >= 0 && index + 2 < a.vocab) out[index + 2] = x.z;
                if (index + 3 >= 0 && index + 3 < a.vocab) out[index + 3] = x.w;
            }
        }
    } else {
        __syncwarp();
        for (int i = 0; i < 4 * r.pieces; i++) {
            const int at = warp * r.pieces * kPiece + i * 32 + lane, index = r.start + at;
            const float x = part[at];
            if (index >= 0 && index < a.vocab) out[index] = !refused && r.keeps(x, index) ? x : other;
        }
    }
}

int launch(SampleArgs &a, int rows) {
    // three logits may lie before a row that does not start on 16 bytes
    const int long_row = a.vocab + 3;
    int ranks = 1;
    while (ranks < kMaxRanks && (long_row + ranks - 1) / ranks > kStep) ranks *= 2;
    a.part = ((long_row + ranks - 1) / ranks + kStep - 1) / kStep * kStep;
    const int smem = a.part * 4 + (int)sizeof(Shared);
    if (int rc = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows * ranks);
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
    return cudaLaunchKernelEx(&cfg, sample_kernel, a);
}

bool unaligned(const void *p) { return reinterpret_cast<uintptr_t>(p) & 3; }

int settings(SampleArgs &a, const float *logits, const float *temperature, const int *top_k, const float *top_p, const float *min_p, int per,
             int rows, int vocab) {
    if (!logits || unaligned(logits) || per < 1 || rows < 1 || rows > kRowsAtOnce || vocab < 1 || vocab > kMaxVocab - 3)
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
    if (!token || !uniforms) return cudaErrorInvalidValue;
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

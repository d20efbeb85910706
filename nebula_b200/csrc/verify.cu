// Which drafted tokens the target accepts, and the token that follows them.
//
// A logit x becomes t = x * log2(e)/temperature = n + f with n = floor(t), and
// the weight 2^(n - M) * 2^f, M the largest n of the row: 2^f does not depend
// on M, and the power of two is exact, so sums over parts of a row, each
// relative to its own M, come to a common M without rounding, and one pass over
// the logits is enough. Sums are held in 64 bits: a token is a whole number
// that must not depend on their order. So are the weights of drafts and of the
// chunk that the next token is drawn from, down to 2^-1000 of the largest.
//
// Two kernels, the second chained to the first (programmatic launch):
//  - chunk_kernel reads all logits once, 4096 to a CTA, and leaves each chunk's
//    M and sum. Bound by HBM.
//  - walk_kernel, a cluster per sequence: joins the chunks, walks the tree, and
//    draws the next token by finding its chunk among the sums and then its
//    place in that chunk. With drawn drafts the sums of max(p - q, 0) come first,
//    over all CTAs of the cluster. Bound by latency.
#include <cfloat>
#include <cooperative_groups.h>
#include "cache.cuh"

using namespace nb;
namespace cg = cooperative_groups;

namespace {

constexpr int kMaxVocab = 1 << 24;
constexpr int kChunk = 4096;
constexpr int kChunkThreads = 256, kWalkThreads = 512;
constexpr int kDrawnCtas = 8;  // CTAs per sequence that sum max(p - q, 0)

// Of a chunk, or of a row.
struct Stats {
    double sum;  // of the weights, relative to 2^top
    float top;   // M; with temperature 0 the largest logit
    int best;    // with temperature 0 its index, else 0; kNone: no finite logit; kBad: a NaN or +infinity
};
constexpr int kBad = -1, kNone = -2;

struct VerifyArgs {
    int *path, *accepted, *next;
    const float *logits;
    const int *draft, *parents;
    const float *probs, *uniforms;
    float scale;  // log2(e)/temperature; 0: the largest logit takes all
    int tokens, vocab, chunks;
    Stats *stats;   // [rows][chunks]
    double *rest;   // [seqs][chunks]: sums of max(p - q, 0)
};

// t = n + f, the product rounded before the floor; one past the finite range counts as the range's end.
__device__ __forceinline__ float split(float x, float scale, float &frac) {
    const float t = fminf(fmaxf(__fmul_rn(x, scale), -FLT_MAX), FLT_MAX), n = floorf(t);
    frac = t - n;
    return n;
}
__device__ __forceinline__ float ex2(float x) {  // the instruction: |x| <= 1 here, which needs no scaling
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^f * 2^rel for 0 <= f <= 1 and rel <= 0: the power of two goes into the exponent; weights below 2^-126 are zero.
__device__ __forceinline__ float weigh(float f, float rel) {
    return rel < -126.0f ? 0.0f : ex2(f) * __int_as_float(((int)rel + 127) << 23);
}
// 2^rel for rel <= 0, 0 below `least`. Sums come to another M down to 2^-900, single weights are held in 64 bits down to
// 2^-1000: a part of a row whose sum is not zero holds a weight that is not zero, and a uniform of 0 finds it.
constexpr float kLeastSum = -900.0f, kLeastWeight = -1000.0f;
__device__ __forceinline__ double shift_down(float rel, float least = kLeastSum) {
    return rel < least ? 0.0 : __longlong_as_double((long long)((int)rel + 1023) << 52);
}
// Conversions and floor run at an eighth of the rate of additions. Where |M| < 2^20, x*scale + (1.5 * 2^23 - M + b) that
// rounds down is an integer of the last bit, floor(x*scale) - M + b stands in its low bits, and what it leaves of x*scale
// is f: not even x*scale is rounded. Far below M the sum's bits are any, but it compares below.
constexpr float kMagic = 12582912.0f, kNear = 1048576.0f;  // 1.5 * 2^23, 2^20
__device__ __forceinline__ float near_weight(float scale, float k, float x) {  // k: kMagic + 127 - M
    const float u = __fmaf_rd(x, scale, k), g = ex2(__fmaf_rn(x, scale, __fsub_rn(k, u)));
    return u >= kMagic + 1.0f ? g * __int_as_float(__float_as_int(u) << 23) : 0.0f;
}
__device__ __forceinline__ float far_weight(float scale, const Stats &r, float x, int v) {
    if (scale == 0.0f) return v == r.best ? 1.0f : 0.0f;
    if (x == -INFINITY) return 0.0f;
    float f;
    const float n = split(x, scale, f);
    return weigh(f, n - r.top);
}
__device__ __forceinline__ bool is_near(float scale, const Stats &r) { return scale > 0.0f && fabsf(r.top) < kNear; }
// The same weights in 64 bits, what is below 2^-126 too. `near`: 2^f 2^(n - M) put together as the bits of a double.
__device__ __forceinline__ double near_fine(float scale, float k, float x) {  // k: kMagic + 127 - M
    const float u = __fmaf_rd(x, scale, k);
    const unsigned g = __float_as_uint(ex2(__fmaf_rn(x, scale, __fsub_rn(k, u))));  // in [1, 2] where it is used
    const int n = __float_as_int(u) - __float_as_int(kMagic + 127.0f);
    return u >= kMagic + 127.0f + kLeastWeight ? __hiloint2double((int)(g >> 3) + (n + 896) * (1 << 20), (int)(g << 29)) : 0.0;
}
__device__ __forceinline__ double far_fine(float scale, const Stats &r, float x, int v) {
    if (scale == 0.0f) return v == r.best ? 1.0 : 0.0;
    if (x == -INFINITY) return 0.0;
    float f;
    const float rel = split(x, scale, f) - r.top;
    return rel < kLeastWeight ? 0.0 : (double)ex2(f) * shift_down(rel, kLeastWeight);
}
__device__ __forceinline__ double fine_weight(float scale, const Stats &r, float x, int v) {
    return is_near(scale, r) ? near_fine(scale, kMagic + 127.0f - r.top, x) : far_fine(scale, r, x, v);
}
// Of 8 neighbouring values from v on.
__device__ __forceinline__ void weights8(float scale, const Stats &r, float (&x)[8], int v) {
    if (is_near(scale, r)) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = near_weight(scale, kMagic + 127.0f - r.top, x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = far_weight(scale, r, x[i], v + i);
    }
}

__device__ __forceinline__ void fine8(float scale, const Stats &r, const float (&x)[8], int v, double (&w)[8]) {
    if (is_near(scale, r)) {
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = near_fine(scale, kMagic + 127.0f - r.top, x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = far_fine(scale, r, x[i], v + i);
    }
}

// A part of a row brought to the row's M.
__device__ __forceinline__ double brought(const Stats &s, float top) { return s.sum * shift_down(s.top - top); }

// Chunks begin at the row's last 16-byte boundary at or before its start, up to three values before the row, so that a
// thread loads four values at once.
__device__ __forceinline__ int chunk_lead(const float *row) { return (int)(reinterpret_cast<uintptr_t>(row) / 4 % 4); }
// Four values from position v on, those outside the row -infinity.
__device__ __forceinline__ void load4(const float *row, int vocab, int v, float (&x)[4]) {
    if (v >= 0 && v + 4 <= vocab && !(reinterpret_cast<uintptr_t>(row + v) & 15)) {
        *reinterpret_cast<float4 *>(x) = __ldg(reinterpret_cast<const float4 *>(row + v));
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = v + k >= 0 && v + k < vocab ? __ldg(row + v + k) : -INFINITY;
    }
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}
// Floats in order as integers.
__device__ __forceinline__ int ordered(float x) {
    const int b = __float_as_int(x);
    return b < 0 ? b ^ 0x7fffffff : b;
}
__device__ __forceinline__ float warp_max(float x) {
    const int m = __reduce_max_sync(0xffffffffu, ordered(x));
    return __int_as_float(m < 0 ? m ^ 0x7fffffff : m);
}

// NaN if one of them is.
__device__ __forceinline__ float max_nan(float x, float y) {
    float z;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
    return z;
}

// The values of a thread, `most` the largest: the largest n, and the sum of the weights relative to it.
template <int N>
__device__ __forceinline__ void weigh_all(const float (&x)[N], float most, float scale, float &top, double &sum) {
    sum = 0.0;
    const float t = __fmul_rn(most, scale);
    if (t > -kNear && t < kNear) {
        // As near_weight, and 2^f 2^(n - top) put together as the bits of a double: 896 more make the exponent's bias.
        // What is far below (2^f any there, 0, infinity and NaN too) comes to less than 2^-511: nothing beside the largest.
        top = __fsub_rn(__fmaf_rd(most, scale, kMagic), kMagic);
        const float k = kMagic + 896.0f - top;
        const int least = __float_as_int(kMagic);
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float u = __fmaf_rd(x[i], scale, k);
            const unsigned g = __float_as_uint(ex2(__fmaf_rn(x[i], scale, __fsub_rn(k, u))));  // in [1, 2]
            sum += __hiloint2double((int)(g >> 3) + (max(__float_as_int(u), least) << 20), (int)(g << 29));
        }
    } else {
        float f;
        top = most > -INFINITY ? split(most, scale, f) : -INFINITY;
#pragma unroll 1
        for (int i = 0; i < N; i++) {
            float y = -INFINITY;
#pragma unroll
            for (int j = 0; j < N; j++) y = j == i ? x[j] : y;
            if (y > -INFINITY) {
                const float n = split(y, scale, f);
                sum += (double)weigh(f, n - top);
            }
        }
    }
}

// GREEDY: temperature 0, only the largest logit and its lowest index.
// One chunk to a CTA: many short CTAs keep more loads in flight than fewer that go on to a next chunk (all of a step, 12 x
// 17 x 131072 logits: 46 us against 50 with the next chunk's loads ahead). The warps' instructions count next to the
// bytes: at 26 a logit (guarded loads, the product rounded by itself, a maximum per eight) the step took 39.5 us,
// like this 33.8; 128 threads with twice the logits 36.9.
template <bool GREEDY>
__global__ void __launch_bounds__(kChunkThreads) chunk_kernel(const __grid_constant__ VerifyArgs a) {
    constexpr int kWarps = kChunkThreads / 32, kQuads = kChunk / (4 * kChunkThreads);
    __shared__ Stats part[kWarps];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const float *row = a.logits + (size_t)blockIdx.x * a.vocab;
    const int start = (int)blockIdx.y * kChunk - chunk_lead(row), first = start + 4 * (int)threadIdx.x;
    float x[4 * kQuads];
    if (start >= 0 && start + kChunk <= a.vocab) {
        const float4 *at = reinterpret_cast<const float4 *>(row + first);
#pragma unroll
        for (int i = 0; i < kQuads; i++) *reinterpret_cast<float4 *>(&x[4 * i]) = __ldg(at + kChunkThreads * i);
    } else {
#pragma unroll
        for (int i = 0; i < kQuads; i++) load4(row, a.vocab, first + 4 * kChunkThreads * i, *reinterpret_cast<float(*)[4]>(&x[4 * i]));
    }
    float most = x[0];
#pragma unroll
    for (int i = 1; i < 4 * kQuads; i++) most = max_nan(most, x[i]);
    bool bad = __any_sync(0xffffffffu, !(most < INFINITY));
    Stats s = {0.0, -INFINITY, 0};
    if constexpr (GREEDY) {
        int best = 0x7fffffff;
#pragma unroll
        for (int i = 4 * kQuads - 1; i >= 0; i--)
            if (x[i] == most) best = first + 4 * kChunkThreads * (i / 4) + i % 4;
        s.top = warp_max(most + 0.0f);  // -0 and 0 are equals
        s.best = __reduce_min_sync(0xffffffffu, s.top == most ? best : 0x7fffffff);
    } else {
        float top = -INFINITY;
        double sum = 0.0;
        if (!bad) weigh_all(x, most, a.scale, top, sum);
        s.top = warp_max(top);
        if (s.top > -INFINITY) s.sum = warp_sum(sum * shift_down(top - s.top));
    }
    if (!(s.top > -INFINITY)) s.best = kNone;
    if (bad) s.best = kBad;
    if (lane == 0) part[warp] = s;
    __syncthreads();
    if (warp == 0) {
        s = lane < kWarps ? part[lane] : Stats{0.0, -INFINITY, kNone};
        bad = __any_sync(0xffffffffu, s.best == kBad);
        const float m = warp_max(s.best >= 0 ? s.top : -INFINITY);
        const int best = __reduce_min_sync(0xffffffffu, s.best >= 0 && s.top == m ? s.best : 0x7fffffff);
        const double sum = m > -INFINITY && !GREEDY ? warp_sum(s.best >= 0 ? s.sum * shift_down(s.top - m) : 0.0) : 0.0;
        if (lane == 0) a.stats[(size_t)blockIdx.x * a.chunks + blockIdx.y] = {sum, m, bad ? kBad : m > -INFINITY ? best : kNone};
    }
}

// The running sum of x over a warp.
__device__ __forceinline__ double warp_scan(double x) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += up;
    }
    return x;
}
// The lane at which a running sum (`upto`, of parts that are not negative) passes the aim; where rounding leaves none,
// the last that has any weight. -1: no weight at all.
__device__ __forceinline__ int claim(double part, double upto, double aim) {
    const unsigned has = __ballot_sync(0xffffffffu, part > 0.0), passes = __ballot_sync(0xffffffffu, part > 0.0 && aim < upto);
    return passes ? __ffs(passes) - 1 : has ? 31 - __clz(has) : -1;
}

// What refused drafts leave of a row's or a chunk's mass is taken as a difference of 64-bit sums, which are off by some
// 2^-50. Where it comes out below this share of the sum and matters, walk_anew adds up what is there.
constexpr double kSure = 0x1p-20;

// The thread's eight weights of chunk c, without those of the nodes `gone`.
__device__ void weights_without(const VerifyArgs &a, const float *row, const Stats &r, int c, unsigned long long gone,
                                const int *draft, double (&w)[8]) {
    const int v = c * kChunk - chunk_lead(row) + 8 * (int)threadIdx.x;
    float x[8];
    load4(row, a.vocab, v, *reinterpret_cast<float(*)[4]>(&x[0]));
    load4(row, a.vocab, v + 4, *reinterpret_cast<float(*)[4]>(&x[4]));
    fine8(a.scale, r, x, v, w);
    for (unsigned long long m = gone; m; m &= m - 1) {
        const int g = draft[__ffsll(m) - 1] - v;
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (g == i) w[i] = 0.0;
    }
}
// Their sum over chunks c0 .. c1-1, by one CTA.
__device__ double sum_without(const VerifyArgs &a, const float *row, const Stats &r, int c0, int c1, unsigned long long gone,
                              const int *draft, double *sums) {
    double part = 0.0, all = 0.0;
    for (int c = c0; c < c1; c++) {
        double w[8];
        weights_without(a, row, r, c, gone, draft, w);
#pragma unroll
        for (int i = 0; i < 8; i++) part += w[i];
    }
    part = warp_sum(part);
    __syncthreads();
    if (threadIdx.x % 32 == 0) sums[threadIdx.x / 32] = part;
    __syncthreads();
    for (int k = 0; k < kWalkThreads / 32; k++) all += sums[k];
    return all;
}
// The walk for given drafts and the draw of the next token, one step after the other and by sums of what is left. Rare (refused
// drafts hold all but 2^-20 of p), and apart from the other walk: in the way of it 9.0 us became 9.7 (one tree of
// 17 x 131072 logits).
__noinline__ __device__ void walk_anew(const VerifyArgs &a, int seq, const Stats *rows, const unsigned long long *kids, const int *draft,
                                       const double *held, int *path, double *sums) {
    __shared__ int first, last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const size_t base = (size_t)seq * a.tokens;
    int cur = 0, n = 0;
    unsigned long long gone;
    bool ok = true;
    path[0] = 0;
    for (;;) {
        int to = -1;
        gone = 0;
        double held_gone = 0.0;
        for (unsigned long long k = kids[cur]; k; k &= k - 1) {
            const int c = __ffsll(k) - 1;
            ok = (unsigned)draft[c] < (unsigned)a.vocab;
            if (!ok) break;
            double left = rows[cur].sum - held_gone;
            if (gone && left < kSure * rows[cur].sum)
                left = sum_without(a, a.logits + (base + cur) * a.vocab, rows[cur], 0, a.chunks, gone, draft, sums);
            if ((double)a.uniforms[base + c] * left < held[c]) {
                to = c;
                break;
            }
            gone |= 1ull << c;
            held_gone += held[c];
        }
        if (to < 0) break;
        ok = rows[to].best >= 0;
        if (!ok) break;
        cur = to;
        n++;
        path[n] = to;  // all threads write the same
    }
    __syncthreads();
    if (tid < a.tokens) a.path[base + tid] = ok && tid <= n ? path[tid] : -1;
    if (tid == 0) {
        a.accepted[seq] = ok ? n : -1;
        a.next[seq] = -1;
        first = kWalkThreads, last = -1;
    }
    if (!ok) return;
    const float *row = a.logits + (base + cur) * a.vocab;
    const Stats r = rows[cur];
    double *rest = a.rest + (size_t)seq * a.chunks, whole = 0.0, run = 0.0, before = 0.0;
    for (int c = 0; c < a.chunks; c++) {
        const double all = sum_without(a, row, r, c, c + 1, gone, draft, sums);
        if (tid == 0) __stcg(rest + c, all);
        whole += all;
    }
    __syncthreads();
    const double aim = (double)a.uniforms[base] * whole;
    int chunk = -1;
    for (int c = 0; c < a.chunks && (chunk < 0 || run <= aim); c++) {
        const double all = __ldcg(rest + c);
        if (all > 0.0) chunk = c, before = run;
        run += all;
    }
    if (chunk < 0) return;  // not with uniforms below 1
    double w[8], part = 0.0;
    weights_without(a, row, r, chunk, gone, draft, w);
#pragma unroll
    for (int i = 0; i < 8; i++) part += w[i];
    double end = warp_scan(part);
    if (lane == 31) sums[warp] = end;
    __syncthreads();
    end += before;
    for (int k = 0; k < warp; k++) end += sums[k];
    if (part > 0.0) {
        if (aim < end) atomicMin(&first, tid);
        atomicMax(&last, tid);
    }
    __syncthreads();
    if (tid != (first < kWalkThreads ? first : last)) return;
    run = end - part;
    int hit = 0;
    bool past = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if (!past && w[i] > 0.0) hit = i;
        run += w[i];
        past |= run > aim;
    }
    a.next[seq] = chunk * kChunk - chunk_lead(row) + 8 * tid + hit;
}

// DRAWN: the drafts' distributions are given; a cluster of kDrawnCtas CTAs per sequence, otherwise one CTA.
template <bool DRAWN>
__global__ void __launch_bounds__(kWalkThreads) walk_kernel(const __grid_constant__ VerifyArgs a) {
    constexpr int kWarps = kWalkThreads / 32, kCtas = DRAWN ? kDrawnCtas : 1;
    static_assert(kWalkThreads * 8 == kChunk, "eight values of a chunk to a thread");
    // Chunks whose loads are in flight together (four: 7 x 6 x 50001 logits 0.6 us slower, 12 x 17 x
    // 131072 0.7 us faster).
    constexpr int kBatch = 2;
    constexpr double kVisible = 0x1p-126, kCoarse = 0x1p-60;  // weights that 32 bits hold; aims that need the others
    __shared__ Stats rows[kMaxNodes];
    __shared__ double sums[kWarps], batch[DRAWN ? kBatch : 1][kWarps];
    __shared__ unsigned long long kids[kMaxNodes];     // of a node: its children
    __shared__ double held[kMaxNodes];                 // the target's weight of a draft, 0 after an older sibling's equal
    __shared__ unsigned takes[2], bads[2], sane[2], weighty[2], unsure[2];  // nodes as bits
    __shared__ int draft[kMaxNodes], parent[kMaxNodes], path[kMaxNodes], count, at_node, refused, doubt;
    __shared__ float first_uniform;
    const int seq = blockIdx.x / kCtas, rank = blockIdx.x % kCtas, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const size_t base = (size_t)seq * a.tokens;
    const bool greedy = a.scale == 0.0f, node = tid < a.tokens;
    bool sound = true;
    float u = 0.0f;
    if (tid < kMaxNodes) kids[tid] = 0;
    if (node) {
        parent[tid] = a.parents[base + tid];
        draft[tid] = a.draft[base + tid];
        u = a.uniforms[base + tid];
        sound = tid == 0 || (parent[tid] >= -1 && parent[tid] < tid);
    }
    if (tid == 0) first_uniform = u;
    sound = __syncthreads_and(sound);
    const bool used = sound && tid > 0 && node && parent[tid] >= 0, tries = used && (unsigned)draft[tid] < (unsigned)a.vocab;
    const size_t above = tries ? base + parent[tid] : 0;
    const float x = tries ? a.logits[above * a.vocab + draft[tid]] : 0.0f;
    const float guess = DRAWN && tries ? a.probs[(base + tid) * a.vocab + draft[tid]] : 0.0f;
    if (used) atomicOr(&kids[parent[tid]], 1ull << tid);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // ---- the rows' M and total: a warp per row, two rows' first 64 chunks asked for together
    for (int r0 = warp; r0 < a.tokens; r0 += 2 * kWarps) {
        Stats ahead[2][2];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = r0 + i / 2 * kWarps, c = lane + i % 2 * 32;
            ahead[i / 2][i % 2] = r < a.tokens && c < a.chunks ? a.stats[(base + r) * a.chunks + c] : Stats{0.0, -INFINITY, kNone};
        }
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int r = r0 + j * kWarps;
            if (r >= a.tokens) break;
            float top = -INFINITY;
            int best = 0x7fffffff, bad = 0;
            double sum = 0.0;
            auto join = [&](const Stats &s) {
                bad |= s.best == kBad;
                if (s.best < 0) return;
                if (s.top > top) {
                    sum *= shift_down(top - s.top);
                    top = s.top, best = s.best;
                } else if (s.top == top && s.best < best) {
                    best = s.best;
                }
                sum += brought(s, top);
            };
            join(ahead[j][0]);
            join(ahead[j][1]);
            for (int c = lane + 64; c < a.chunks; c += 32) join(a.stats[(base + r) * a.chunks + c]);
            const float m = warp_max(top);
            sum = m > -INFINITY ? warp_sum(sum * shift_down(top - m)) : 0.0;
            best = __reduce_min_sync(0xffffffffu, top == m ? best : 0x7fffffff);
            bad = __any_sync(0xffffffffu, bad);
            if (lane == 0) rows[r] = {greedy ? 1.0 : sum, m, bad ? kBad : m > -INFINITY ? best : kNone};
        }
    }
    __syncthreads();
    // ---- the walk: a thread per node decides whether it would be taken were it reached with all older siblings
    // refused, so that what is left to do one after the other is to follow bits
    if (warp < kMaxNodes / 32) {
        double w = tries ? fine_weight(a.scale, rows[parent[tid]], x, draft[tid]) : 0.0;
        const unsigned long long older = tries ? kids[parent[tid]] & ((1ull << tid) - 1) : 0;
        if constexpr (!DRAWN)
            for (unsigned long long m = older; m; m &= m - 1)
                if (draft[__ffsll(m) - 1] == draft[tid]) w = 0.0;  // a token leaves p once
        held[tid] = w;
        asm volatile("bar.sync 1, 64;" ::: "memory");
        bool take = false, close = false;  // close: the older siblings leave next to nothing
        if (tries) {
            double left = rows[parent[tid]].sum;
            if constexpr (DRAWN) {
                take = w < kVisible ? (double)u * (double)guess < w / left : __fmul_rn(u, guess) < (float)w / (float)left;
            } else {
                for (unsigned long long m = older; m; m &= m - 1) left -= held[__ffsll(m) - 1];
                take = (double)u * left < w;
                close = older && left < kSure * rows[parent[tid]].sum;
            }
        }
        const unsigned t = __ballot_sync(0xffffffffu, take), b = __ballot_sync(0xffffffffu, used && !tries);
        const unsigned s = __ballot_sync(0xffffffffu, node && rows[node ? tid : 0].best >= 0), h = __ballot_sync(0xffffffffu, w > 0.0);
        const unsigned z = __ballot_sync(0xffffffffu, close);
        if (lane == 0) takes[warp] = t, bads[warp] = b, sane[warp] = s, weighty[warp] = h, unsure[warp] = z;
        asm volatile("bar.sync 1, 64;" ::: "memory");
    }
    auto bits = [](const unsigned (&m)[2]) { return m[0] | (unsigned long long)m[1] << 32; };
    if (tid == 0) {
        const unsigned long long taken = bits(takes), bad = bits(bads), good = bits(sane), doubted = bits(unsure);
        unsigned long long met = 0;  // nodes that were tried
        int cur = 0, n = 0;
        bool ok = sound && (good & 1);
        refused = -1;
        path[0] = 0;
        while (ok) {
            const unsigned long long k = kids[cur], first = DRAWN ? k & (~k + 1) : k, t = first & taken;
            if (!t) {
                met |= k;
                ok = !(bad & k) && !(DRAWN && (k & (k - 1)));
                refused = __ffsll(k) - 1;
                break;
            }
            const unsigned long long c = t & (~t + 1);
            met |= k & (c | (c - 1));
            ok = !(bad & k & (c - 1)) && (good & c);
            cur = __ffsll(c) - 1;
            path[++n] = cur;
        }
        at_node = ok ? cur : -1;
        count = ok ? n : -1;
        doubt = (met & doubted) != 0;
    }
    __syncthreads();
    if constexpr (!DRAWN) {
        if (doubt) return walk_anew(a, seq, rows, kids, draft, held, path, sums);
    }
    if (rank == 0) {
        if (tid < a.tokens) a.path[base + tid] = tid <= count ? path[tid] : -1;
        if (tid == 0) a.accepted[seq] = count;
        if (at_node < 0 && tid == 0) a.next[seq] = -1;
    }
    if (at_node < 0) return;  // the same in all CTAs of the cluster

    // ---- what is left of the last node's row
    const float *row = a.logits + (base + at_node) * a.vocab;
    const Stats r = rows[at_node];
    const float total = (float)r.sum, inverse = __frcp_rn(total);
    const float *q = DRAWN && refused >= 0 ? a.probs + (base + refused) * a.vocab : nullptr;
    const int lead = chunk_lead(row);
    const unsigned long long gone = DRAWN ? 0 : kids[at_node] & bits(weighty);  // nodes whose drafts have left p
    // the thread's eight neighbouring values of chunk c
    // (q's rows may lie otherwise on the 16-byte boundaries: twelve values from the boundary before, of which eight from
    // `off` on are the thread's)
    constexpr int kY = DRAWN ? 12 : 8;
    const int off = DRAWN && q ? (chunk_lead(q) - lead) & 3 : 0;
    auto fetch = [&](int c, float (&w)[8], float (&y)[kY]) {
        const int v = c * kChunk - lead + 8 * tid;
        load4(row, a.vocab, v, *reinterpret_cast<float(*)[4]>(&w[0]));
        load4(row, a.vocab, v + 4, *reinterpret_cast<float(*)[4]>(&w[4]));
        if (DRAWN && q) {
            load4(q, a.vocab, v - off, *reinterpret_cast<float(*)[4]>(&y[0]));
            load4(q, a.vocab, v - off + 4, *reinterpret_cast<float(*)[4]>(&y[4]));
            if (off) load4(q, a.vocab, v - off + 8, *reinterpret_cast<float(*)[4]>(&y[8]));
        }
    };
    auto turn = [&](float (&y)[kY]) {
        if constexpr (DRAWN) {
            if (off & 1) {
#pragma unroll
                for (int i = 0; i < kY - 1; i++) y[i] = y[i + 1];
            }
            if (off & 2) {
#pragma unroll
                for (int i = 0; i < 8; i++) y[i] = y[i + 2];
            }
        }
    };
    // With drawn drafts p is a 32-bit number, and weights below 2^-126 are left out: all of them come to less than 2^-102.
    auto left8 = [&](int c, float (&w)[8], float (&y)[kY]) {
        const int v = c * kChunk - lead + 8 * tid;
        turn(y);
        weights8(a.scale, r, w, v);  // none outside the row
#pragma unroll
        for (int i = 0; i < 8; i++) {
            // w/total with one reciprocal for all: from a correctly rounded reciprocal one step on the remainder
            // leads to the correctly rounded quotient (P. Markstein, 1990), w < 2^-100 aside
            const float p = w[i] * inverse;
            w[i] = fmaf(fmaf(-p, total, w[i]), inverse, p);
            if (q) w[i] = v + i >= 0 && v + i < a.vocab ? fmaxf(w[i] - y[i], 0.0f) : 0.0f;
        }
    };
    // Where nothing may be left out: 64-bit weights (with drawn drafts p, the same 32-bit number where it is one).
    auto left8_fine = [&](int c, const float (&x)[8], float (&y)[kY], double (&w)[8]) {
        const int v = c * kChunk - lead + 8 * tid;
        turn(y);
        fine8(a.scale, r, x, v, w);
        if constexpr (DRAWN) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                w[i] = w[i] < kVisible ? w[i] / r.sum : (double)((float)w[i] / total);
                if (q) w[i] = v + i >= 0 && v + i < a.vocab ? fmax(w[i] - (double)y[i], 0.0) : 0.0;
            }
        }
        for (unsigned long long m = gone; m; m &= m - 1) {
            const int g = draft[__ffsll(m) - 1] - v;
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (g == i) w[i] = 0.0;
        }
    };
    auto fine_sum = [&](int c) -> double {  // of chunk c, by the whole CTA
        float x[8], y[kY];
        double w[8], part = 0.0, all = 0.0;
        fetch(c, x, y);
        left8_fine(c, x, y, w);
#pragma unroll
        for (int i = 0; i < 8; i++) part += w[i];
        part = warp_sum(part);
        __syncthreads();
        if (lane == 0) sums[warp] = part;
        __syncthreads();
        for (int k = 0; k < kWarps; k++) all += sums[k];
        return all;
    };
    double *rest = a.rest + (size_t)seq * a.chunks;
    // ---- the chunk that holds the aim: every warp finds it for itself, a lane takes neighbouring chunks
    const int per = (a.chunks + 31) / 32, c0 = min(lane * per, a.chunks), c1 = min(c0 + per, a.chunks);
    constexpr int kKept = 4;  // a lane's first chunks, whose sums stay in registers
    unsigned close = 0;       // those of which refused drafts leave next to nothing, as bits (the others: bit kKept)
    auto chunk_sum = [&](int c) -> double {
        if constexpr (DRAWN) {
            return __ldcg(rest + c);
        } else {
            const Stats s = a.stats[(base + at_node) * a.chunks + c];
            if (greedy) return s.best == r.best ? 1.0 : 0.0;
            const double all = s.best >= 0 ? brought(s, r.top) : 0.0;
            double w = all;
            for (unsigned long long m = gone; m; m &= m - 1) {
                const int g = __ffsll(m) - 1;
                if ((draft[g] + lead) / kChunk == c) w -= held[g];
            }
            close |= (unsigned)(w < kSure * all) << min(c - c0, kKept);
            return fmax(w, 0.0);
        }
    };
    double whole = 0.0, upto = 0.0, sum = 0.0, kept[kKept];
    bool fine = !DRAWN;
    for (;;) {
        if constexpr (DRAWN) {
            const int full = (a.vocab + lead + kChunk - 1) / kChunk;  // chunks that hold values: all, or all but the last
            for (int b0 = rank; b0 < full && !fine; b0 += kBatch * kCtas) {
                float w[kBatch][8], y[kBatch][kY];
#pragma unroll
                for (int i = 0; i < kBatch; i++) fetch(b0 + i * kCtas, w[i], y[i]);  // -infinity past the row's end
#pragma unroll
                for (int i = 0; i < kBatch; i++) {
                    if (b0 + i * kCtas >= full) break;
                    left8(b0 + i * kCtas, w[i], y[i]);
                    double part = 0.0;
#pragma unroll
                    for (int k = 0; k < 8; k++) part += (double)w[i][k];
                    part = warp_sum(part);
                    if (lane == 0) batch[i][warp] = part;
                }
                __syncthreads();
                if (tid < kBatch && b0 + tid * kCtas < full) {
                    double all = 0.0;
                    for (int k = 0; k < kWarps; k++) all += batch[tid][k];
                    __stcg(rest + b0 + tid * kCtas, all);
                }
                __syncthreads();
            }
            for (int b = rank; b < full && fine; b += kCtas) {
                const double all = fine_sum(b);
                if (tid == 0) __stcg(rest + b, all);
            }
            if (rank == 0 && tid == 0 && full < a.chunks) __stcg(rest + full, 0.0);
            cg::this_cluster().sync();  // the sums are there
        }
        sum = 0.0;
#pragma unroll
        for (int k = 0; k < kKept; k++) kept[k] = c0 + k < c1 ? chunk_sum(c0 + k) : 0.0;
#pragma unroll
        for (int k = 0; k < kKept; k++) sum += kept[k];
        for (int c = c0 + kKept; c < c1; c++) sum += chunk_sum(c);
        upto = warp_scan(sum);
        whole = __shfl_sync(0xffffffffu, upto, 31);
        if constexpr (!DRAWN) {
            break;
        } else {
            if (!fine && !greedy && (double)first_uniform * whole < kCoarse) fine = true;  // the weights left out matter
            else if (q && !(whole > 0.0)) q = nullptr;  // the draft's distribution covers the target's: draw from the target's
            else break;
            cg::this_cluster().sync();  // the sums were read
        }
    }
    if (rank) return;
    const double aim = (double)first_uniform * whole;
    const int owner = claim(sum, upto, aim);
    // Chunks with next to nothing left do not count beside the others, unless the aim is as small (or one is chosen, below).
    // All warps say the same.
    if constexpr (!DRAWN) {
        if (aim < kSure * r.sum && __any_sync(0xffffffffu, close)) return walk_anew(a, seq, rows, kids, draft, held, path, sums);
    }
    if (owner < 0) {  // not met: a row with a distribution has weight left, for what was refused was not all of it
        if (tid == 0) a.next[seq] = -1;
        return;
    }
    int c = c0;
    double before = upto - sum;
    if (lane == owner) {
        double run = before;
        bool past = false;
        auto look = [&](int k, double w) {
            if (!past && w > 0.0) c = k, before = run;
            run += w;
            past |= run > aim;
        };
#pragma unroll
        for (int k = 0; k < kKept; k++) look(c0 + k, kept[k]);
        for (int k = c0 + kKept; k < c1 && !past; k++) look(k, chunk_sum(k));
    }
    if constexpr (!DRAWN) {
        if (__any_sync(0xffffffffu, lane == owner && close >> min(c - c0, kKept) & 1))
            return walk_anew(a, seq, rows, kids, draft, held, path, sums);
    }
    c = __shfl_sync(0xffffffffu, c, owner);
    before = __shfl_sync(0xffffffffu, before, owner);
    // ---- the place in the chunk
    float x8[8], y[kY];
    double w[8], part = 0.0;
    fetch(c, x8, y);
    if (fine) {
        left8_fine(c, x8, y, w);
    } else {
        left8(c, x8, y);
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = x8[i];
    }
#pragma unroll
    for (int i = 0; i < 8; i++) part += w[i];
    double end = warp_scan(part);
    __syncthreads();
    if (lane == 31) sums[warp] = end;
    __syncthreads();
    const double theirs = lane < kWarps ? sums[lane] : 0.0, ends = before + warp_scan(theirs);
    if (claim(theirs, ends, aim) != warp) return;
    end += __shfl_sync(0xffffffffu, ends - theirs, warp);
    if (lane != claim(part, end, aim)) return;
    double run = end - part;
    int hit = 0;
    bool past = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if (!past && w[i] > 0.0) hit = i;
        run += w[i];
        past |= run > aim;
    }
    a.next[seq] = c * kChunk - lead + 8 * tid + hit;
}

template <bool DRAWN>
int launch_walk(const VerifyArgs &a, int seqs) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(seqs * (DRAWN ? kDrawnCtas : 1));
    cfg.blockDim = dim3(kWalkThreads);
    cfg.stream = launch_stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = DRAWN ? kDrawnCtas : 1;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, walk_kernel<DRAWN>, a);
}

int chunks_of(int vocab) { return (vocab + 3 + kChunk - 1) / kChunk; }  // a row may begin up to three values into its first

}  // namespace

extern "C" int qg_verify_workspace_bytes(int seqs, int tokens, int vocab, size_t *bytes) {
    if (!bytes || seqs < 1 || seqs > kMaxSeqs || tokens < 1 || tokens > kMaxNodes || vocab < 1 || vocab > kMaxVocab)
        return cudaErrorInvalidValue;
    *bytes = (size_t)seqs * chunks_of(vocab) * (tokens * sizeof(Stats) + sizeof(double));
    return cudaSuccess;
}

extern "C" int qg_verify_tree(int *path, int *accepted, int *next, const float *logits, const int *draft, const int *parents,
                              const float *draft_probs, const float *uniforms, double temperature, int seqs, int tokens,
                              int vocab, void *workspace) {
    size_t bytes;
    if (int rc = qg_verify_workspace_bytes(seqs, tokens, vocab, &bytes)) return rc;
    const float scale = temperature > 0 ? (float)(1.0 / temperature * 1.4426950408889634) : 0.0f;
    if (!path || !accepted || !next || !logits || !draft || !parents || !uniforms || !workspace || !(temperature >= 0) ||
        !(scale < INFINITY) || (temperature > 0 && scale == 0.0f) || (reinterpret_cast<uintptr_t>(workspace) & 15))
        return cudaErrorInvalidValue;
    const int chunks = chunks_of(vocab);
    Stats *stats = static_cast<Stats *>(workspace);
    const VerifyArgs a = {path, accepted, next, logits, draft, parents, draft_probs, uniforms, scale, tokens, vocab, chunks, stats,
                          reinterpret_cast<double *>(stats + (size_t)seqs * tokens * chunks)};
    if (int rc = launch_chained(scale == 0.0f ? chunk_kernel<true> : chunk_kernel<false>, dim3(seqs * tokens, chunks), kChunkThreads, a))
        return rc;
    return draft_probs ? launch_walk<true>(a, seqs) : launch_walk<false>(a, seqs);
}

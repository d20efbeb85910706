// Which drafted tokens the target accepts, and the token that follows them.
//
// A logit x becomes t = x * log2(e)/temperature = n + f with n = floor(t), and
// the weight 2^(n - M) * 2^f, M the largest n of the row: 2^f does not depend
// on M, and the power of two is exact, so sums over parts of a row, each
// relative to its own M, come to a common M without rounding, and one pass over
// the logits is enough. Sums are held in 64 bits: a token is a whole number
// that must not depend on their order.
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
constexpr int kChunk = 4096, kThreads = 256, kPer = kChunk / kThreads;
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

// t = n + f. The product is rounded before the floor (no fused multiply-add), so that f is the same everywhere; one
// past the finite range counts as the range's end.
__device__ __forceinline__ float split(float x, float scale, float &frac) {
    const float t = fminf(fmaxf(__fmul_rn(x, scale), -FLT_MAX), FLT_MAX), n = floorf(t);
    frac = t - n;
    return n;
}
// 2^f * 2^rel for 0 <= f <= 1 and rel <= 0: the power of two goes into the exponent; weights below 2^-126 are zero.
__device__ __forceinline__ float weigh(float f, float rel) {
    return rel < -126.0f ? 0.0f : exp2f(f) * __int_as_float(((int)rel + 127) << 23);
}
// 2^rel for rel <= 0 (0 below the range), to bring a sum to another M.
__device__ __forceinline__ double shift_down(float rel) {
    return rel < -1000.0f ? 0.0 : __longlong_as_double((long long)((int)rel + 1023) << 52);
}
__device__ __forceinline__ float weight(float scale, const Stats &r, float x, int v) {
    if (scale == 0.0f) return v == r.best ? 1.0f : 0.0f;
    if (x == -INFINITY) return 0.0f;
    float f;
    const float n = split(x, scale, f);
    return weigh(f, n - r.top);
}

// Two parts of a row as one. The order of equal logits: the lower index.
__device__ __forceinline__ Stats join(const Stats &a, const Stats &b, bool greedy) {
    Stats r;
    if (a.best == kBad || b.best == kBad) return {0.0, 0.0f, kBad};
    if (a.best == kNone) return b;
    if (b.best == kNone) return a;
    if (greedy) return a.top > b.top || (a.top == b.top && a.best < b.best) ? a : b;
    r.top = fmaxf(a.top, b.top);
    r.sum = a.sum * shift_down(a.top - r.top) + b.sum * shift_down(b.top - r.top);
    r.best = 0;
    return r;
}
__device__ __forceinline__ Stats shuffled(const Stats &a, int d) {
    return {__shfl_xor_sync(0xffffffffu, a.sum, d), __shfl_xor_sync(0xffffffffu, a.top, d), __shfl_xor_sync(0xffffffffu, a.best, d)};
}
__device__ __forceinline__ Stats warp_join(Stats a, bool greedy) {
#pragma unroll
    for (int d = 16; d; d >>= 1) a = join(a, shuffled(a, d), greedy);
    return a;
}

// Chunks begin at the row's first 16-byte boundary at or before its start (when the logits are 16-byte aligned), so a
// thread loads four values at once; `v` of the first is then up to three before the row.
__device__ __forceinline__ int chunk_lead(const float *row) { return (int)(reinterpret_cast<uintptr_t>(row) / 4 % 4); }

// The thread's kPer values of chunk c; out: their positions in the row are first + 4*kThreads*(i/4) + i%4, those
// outside the row -infinity.
__device__ __forceinline__ void load_chunk(const float *row, int vocab, int c, float (&x)[kPer], int &first, float outside) {
    first = c * kChunk - chunk_lead(row) + 4 * (int)threadIdx.x;
#pragma unroll
    for (int i = 0; i < kPer / 4; i++) {
        const int v = first + 4 * kThreads * i;
        if (v >= 0 && v + 4 <= vocab) {
            *reinterpret_cast<float4 *>(x + 4 * i) = __ldg(reinterpret_cast<const float4 *>(row + v));
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) x[4 * i + k] = v + k >= 0 && v + k < vocab ? __ldg(row + v + k) : outside;
        }
    }
}
__device__ __forceinline__ int place(int first, int i) { return first + 4 * kThreads * (i / 4) + i % 4; }

template <bool GREEDY>
__global__ void __launch_bounds__(kThreads) chunk_kernel(const VerifyArgs a) {
    __shared__ Stats part[kThreads / 32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int c = blockIdx.x % a.chunks, row = blockIdx.x / a.chunks;
    float x[kPer];
    int first;
    load_chunk(a.logits + (size_t)row * a.vocab, a.vocab, c, x, first, -INFINITY);
    bool bad = false;
    Stats s = {0.0, -INFINITY, kNone};
    if (GREEDY) {
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            bad |= !(x[i] < INFINITY);
            if (x[i] > s.top) s.top = x[i], s.best = place(first, i);
        }
    } else {
        float n[kPer];
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            bad |= !(x[i] < INFINITY);
            n[i] = -INFINITY;
            if (x[i] > -INFINITY) n[i] = split(x[i], a.scale, x[i]);
            s.top = fmaxf(s.top, n[i]);
        }
        if (s.top > -INFINITY) {
            s.best = 0;
#pragma unroll
            for (int i = 0; i < kPer; i++) s.sum += (double)(n[i] > -INFINITY ? weigh(x[i], n[i] - s.top) : 0.0f);
        }
    }
    if (bad) s.best = kBad;
    s = warp_join(s, GREEDY);
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kThreads / 32; w++) s = join(s, part[w], GREEDY);
        a.stats[blockIdx.x] = s;
    }
}

// The running sum of x over the CTA's threads, and its total.
__device__ double block_scan(double x, double *buf, double &total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += up;
    }
    __syncthreads();
    if (lane == 31) buf[warp] = x;
    __syncthreads();
    total = 0.0;
    double before = 0.0;
    for (int w = 0; w < kThreads / 32; w++) {
        before = w == warp ? total : before;
        total += buf[w];
    }
    return before + x;
}

// The first thread whose running sum passes the aim, or where rounding leaves none the last that has any weight; -1: no
// weight at all. (`has`: the thread has weight.)
__device__ int claim(bool has, bool passes, int *buf) {
    if (threadIdx.x == 0) buf[0] = kThreads, buf[1] = -1;
    __syncthreads();
    if (has && passes) atomicMin(&buf[0], (int)threadIdx.x);
    if (has) atomicMax(&buf[1], (int)threadIdx.x);
    __syncthreads();
    return buf[0] < kThreads ? buf[0] : buf[1];
}

// DRAWN: the drafts' distributions are given; a cluster of kDrawnCtas CTAs per sequence, otherwise one CTA.
template <bool DRAWN>
__global__ void __launch_bounds__(kThreads) walk_kernel(const VerifyArgs a) {
    __shared__ Stats rows[kMaxNodes];
    __shared__ double buf[kThreads / 32];
    __shared__ float mine[kMaxNodes], guess[kMaxNodes], uniform[kMaxNodes], values[kChunk + kChunk / 16];
    __shared__ int draft[kMaxNodes], parent[kMaxNodes], gone[kMaxNodes], path[kMaxNodes], n_gone, count, at_node, refused, picked, found[2];
    __shared__ double before_chunk;
    constexpr int kCtas = DRAWN ? kDrawnCtas : 1;
    const int seq = blockIdx.x / kCtas, rank = blockIdx.x % kCtas, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const size_t base = (size_t)seq * a.tokens;
    const bool greedy = a.scale == 0.0f;
    bool sound = true;
    if (tid < a.tokens) {
        parent[tid] = a.parents[base + tid];
        draft[tid] = a.draft[base + tid];
        uniform[tid] = a.uniforms[base + tid];
        sound = tid == 0 || (parent[tid] >= -1 && parent[tid] < tid);
    }
    sound = __syncthreads_and(sound);
    const bool tries = sound && tid > 0 && tid < a.tokens && parent[tid] >= 0 && (unsigned)draft[tid] < (unsigned)a.vocab;
    const size_t above = tries ? base + parent[tid] : 0;
    const float x = tries ? a.logits[above * a.vocab + draft[tid]] : 0.0f;
    if (DRAWN && tries) guess[tid] = a.probs[(base + tid) * a.vocab + draft[tid]];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int r = warp; r < a.tokens; r += kThreads / 32) {
        Stats s = {0.0, -INFINITY, kNone};
        for (int c = lane; c < a.chunks; c += 32) s = join(s, a.stats[(base + r) * a.chunks + c], greedy);
        s = warp_join(s, greedy);
        if (greedy) s.sum = 1.0;
        if (lane == 0) rows[r] = s;
    }
    __syncthreads();
    if (tries) mine[tid] = weight(a.scale, rows[parent[tid]], x, draft[tid]);  // the target's weight of each draft
    __syncthreads();
    if (tid == 0) {
        int cur = 0, n = 0, child = -1, left_out = 0;
        bool ok = sound && rows[0].best >= 0;
        double left = rows[0].sum;
        path[0] = 0;
        for (int c = 1; ok && c < a.tokens; c++) {  // children come after their parent
            if (parent[c] != cur) continue;
            if ((unsigned)draft[c] >= (unsigned)a.vocab || (DRAWN && child >= 0)) {
                ok = false;
                break;
            }
            float w = mine[c];
            bool take;
            if (DRAWN) {
                take = __fmul_rn(uniform[c], guess[c]) < w / (float)rows[cur].sum;
            } else {
                for (int g = 0; g < left_out; g++)
                    if (gone[g] == draft[c]) w = 0.0f;
                take = (double)uniform[c] * left < (double)w;
            }
            if (take) {
                cur = c;
                path[++n] = c;
                child = -1;
                left_out = 0;
                ok = rows[c].best >= 0;
                left = rows[c].sum;
            } else {
                child = c;
                if (w > 0.0f) gone[left_out++] = draft[c];
                left -= (double)w;
            }
        }
        at_node = ok ? cur : -1;
        refused = child;
        n_gone = DRAWN ? 0 : left_out;
        count = ok ? n : -1;
        picked = -1;
    }
    __syncthreads();
    if (rank == 0) {
        if (tid < a.tokens) a.path[base + tid] = tid <= count ? path[tid] : -1;
        if (tid == 0) a.accepted[seq] = count;
        if (at_node < 0 && tid == 0) a.next[seq] = -1;
    }
    if (at_node < 0) return;  // the same in all CTAs of the cluster

    const float *row = a.logits + (base + at_node) * a.vocab;
    const Stats r = rows[at_node];
    const float total = (float)r.sum;
    const float *q = DRAWN && refused >= 0 ? a.probs + (base + refused) * a.vocab : nullptr;
    // what is left of token v's weight
    auto left = [&](float x, int v) -> float {
        float w = weight(a.scale, r, x, v);
        if constexpr (DRAWN) {
            w /= total;
            return q ? fmaxf(w - __ldg(q + v), 0.0f) : w;
        } else {
            for (int g = 0; g < n_gone; g++)
                if (gone[g] == v) w = 0.0f;
            return w;
        }
    };
    double *rest = a.rest + (size_t)seq * a.chunks;
    // ---- the chunks' sums, and the chunk that holds the aim
    const int per = (a.chunks + kThreads - 1) / kThreads, c0 = tid * per, c1 = min(c0 + per, a.chunks);
    double whole = 0.0, upto = 0.0, sum = 0.0;
    auto chunk_sum = [&](int c) -> double {
        if constexpr (DRAWN) return __ldcg(rest + c);
        const Stats s = a.stats[(base + at_node) * a.chunks + c];
        if (greedy) return s.best == r.best ? 1.0 : 0.0;
        double w = s.best >= 0 ? s.sum * shift_down(s.top - r.top) : 0.0;
        const int lead = chunk_lead(row);
        for (int g = 0; g < n_gone; g++)
            if ((gone[g] + lead) / kChunk == c) w -= (double)weight(a.scale, r, row[gone[g]], gone[g]);
        return fmax(w, 0.0);
    };
    for (;;) {
        if constexpr (DRAWN) {
            for (int c = rank; c < a.chunks; c += kCtas) {
                float v[kPer];
                int first;
                load_chunk(row, a.vocab, c, v, first, -INFINITY);
                double part = 0.0;
#pragma unroll
                for (int i = 0; i < kPer; i++) {
                    const int at = place(first, i);
                    if (at >= 0 && at < a.vocab) part += (double)left(v[i], at);
                }
                double all;
                block_scan(part, buf, all);
                if (tid == 0) __stcg(rest + c, all);
            }
            cg::this_cluster().sync();  // the sums are there (and were read, before they are written again)
        }
        sum = 0.0;
        for (int c = c0; c < c1; c++) sum += chunk_sum(c);
        upto = block_scan(sum, buf, whole);
        if (!DRAWN || whole > 0.0 || !q) break;
        q = nullptr;  // the draft's distribution covers the target's: draw from the target's
        cg::this_cluster().sync();
    }
    if (rank) return;
    const double aim = (double)uniform[0] * whole;
    if (tid == claim(sum > 0.0, aim < upto, found)) {
        double run = upto - sum;
        for (int c = c0; c < c1; c++) {
            const double w = chunk_sum(c);
            if (w > 0.0) picked = c, before_chunk = run;
            run += w;
            if (run > aim) break;
        }
    }
    __syncthreads();
    const int c = picked;  // a row with a distribution has weight left (what was refused was not all of it)
    if (c < 0) {
        if (tid == 0) a.next[seq] = -1;
        return;
    }
    // ---- the place in the chunk: 16 values in a row to a thread
    {
        float v[kPer];
        int first;
        load_chunk(row, a.vocab, c, v, first, -INFINITY);
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int at = place(first, i), in = at - first + 4 * tid;
            values[in + in / 16] = at >= 0 && at < a.vocab ? left(v[i], at) : 0.0f;
        }
    }
    __syncthreads();
    const double before = before_chunk;
    double part = 0.0, all;
#pragma unroll
    for (int i = 0; i < 16; i++) part += (double)values[17 * tid + i];
    const double end = before + block_scan(part, buf, all);
    if (tid == claim(part > 0.0, aim < end, found)) {
        double run = end - part;
        int hit = 0;
        for (int i = 0; i < 16; i++) {
            const float w = values[17 * tid + i];
            if (w > 0.0f) hit = i;
            run += (double)w;
            if (run > aim) break;
        }
        a.next[seq] = 16 * tid + hit + c * kChunk - chunk_lead(row);
    }
}

template <bool DRAWN>
int launch_walk(const VerifyArgs &a, int seqs) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(seqs * (DRAWN ? kDrawnCtas : 1));
    cfg.blockDim = dim3(kThreads);
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
    const unsigned grid = (unsigned)((size_t)seqs * tokens * chunks);
    if (scale == 0.0f) chunk_kernel<true><<<grid, kThreads, 0, launch_stream>>>(a);
    else chunk_kernel<false><<<grid, kThreads, 0, launch_stream>>>(a);
    if (int rc = cudaGetLastError()) return rc;
    return draft_probs ? launch_walk<true>(a, seqs) : launch_walk<false>(a, seqs);
}

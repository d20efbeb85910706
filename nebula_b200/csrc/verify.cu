// Which drafted tokens the target accepts, and the token that follows them.
//
// A logit x becomes t = x * log2(e)/temperature = n + f with n = floor(t), and
// the weight 2^(n - M) * 2^f, M the largest n of the row: 2^f does not depend
// on M, and the power of two is exact, so partial sums over parts of a row can
// be brought to a common M without rounding. Sums are held in 64 bits.
#include <cfloat>
#include "cache.cuh"

using namespace nb;

namespace {

constexpr int kMaxVocab = 1 << 24;

struct RowStats {
    double total;
    float top;   // M
    int best;    // index of the largest logit, or -1: the row has no distribution
};

struct VerifyArgs {
    int *path, *accepted, *next;
    const float *logits;
    const int *draft, *parents;
    const float *probs, *uniforms;
    float scale;  // log2(e)/temperature; 0: the largest logit takes all
    int tokens, vocab;
    RowStats *stats;
};

// t = n + f. The product is rounded before the floor (no fused multiply-add), so that f is the same everywhere; one
// past the finite range counts as the range's end.
__device__ __forceinline__ float split(float x, float scale, float &frac) {
    const float t = fminf(fmaxf(__fmul_rn(x, scale), -FLT_MAX), FLT_MAX), n = floorf(t);
    frac = exp2f(t - n);
    return n;
}
// 2^rel for rel <= 0; weights below 2^-126 of the largest are zero.
__device__ __forceinline__ float pow2(float rel) {
    return rel < -126.0f ? 0.0f : __int_as_float(((int)rel + 127) << 23);
}
__device__ __forceinline__ float weight(const VerifyArgs &a, const RowStats &r, const float *row, int v) {
    if (a.scale == 0.0f) return v == r.best ? 1.0f : 0.0f;
    const float x = row[v];
    if (x == -INFINITY) return 0.0f;
    float f;
    const float n = split(x, a.scale, f);
    return f * pow2(n - r.top);
}

template <typename T, typename F>
__device__ T block_reduce(T x, T *buf, F f) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int d = 16; d; d >>= 1) x = f(x, __shfl_xor_sync(0xffffffffu, x, d));
    __syncthreads();
    if (lane == 0) buf[warp] = x;
    __syncthreads();
    x = buf[0];
    for (int w = 1; w < (int)blockDim.x / 32; w++) x = f(x, buf[w]);
    return x;
}

__global__ void __launch_bounds__(1024) row_stats_kernel(const VerifyArgs a) {
    __shared__ double buf[32];
    const float *row = a.logits + (size_t)blockIdx.x * a.vocab;
    // the largest logit and its lowest index, as one ordered 64-bit value
    long long best = 0;
    bool bad = false;
    for (int v = threadIdx.x; v < a.vocab; v += blockDim.x) {
        const float x = row[v];
        bad |= !(x < INFINITY);
        const int b = __float_as_int(x + 0.0f);  // -0 and 0 are equals
        const unsigned key = b < 0 ? ~(unsigned)b : (unsigned)b | 0x80000000u;
        const long long both = (long long)(((unsigned long long)key << 31) | (unsigned)(0x7fffffff - v));
        best = both > best ? both : best;
    }
    bad = __syncthreads_or(bad);
    best = block_reduce(best, reinterpret_cast<long long *>(buf), [](long long x, long long y) { return x > y ? x : y; });
    const int index = 0x7fffffff - (int)(best & 0x7fffffff);
    float f;
    const float top = a.scale == 0.0f ? 0.0f : split(row[index], a.scale, f);
    bad = bad || !(fabsf(row[index]) < INFINITY);
    RowStats r = {1.0, top, bad ? -1 : index};
    if (!bad && a.scale != 0.0f) {
        double sum = 0.0;
        for (int v = threadIdx.x; v < a.vocab; v += blockDim.x) sum += (double)weight(a, r, row, v);
        r.total = block_reduce(sum, buf, [](double x, double y) { return x + y; });
    }
    if (threadIdx.x == 0) a.stats[blockIdx.x] = r;
}

// One CTA per sequence: one thread walks the tree, then the CTA draws from what is left of the last node's row.
__global__ void __launch_bounds__(1024) walk_kernel(const VerifyArgs a) {
    __shared__ double prefix[1024];
    __shared__ int gone[kMaxNodes], n_gone, at_node, refused, picked;
    const int seq = blockIdx.x, tid = threadIdx.x;
    const size_t base = (size_t)seq * a.tokens;
    int *path = a.path + base;
    for (int i = tid; i < a.tokens; i += blockDim.x) path[i] = -1;
    __syncthreads();
    if (tid == 0) {
        const int *parents = a.parents + base, *draft = a.draft + base;
        int cur = 0, count = 0, child = -1;
        bool ok = a.stats[base].best >= 0;
        for (int c = 1; c < a.tokens; c++) ok = ok && parents[c] >= -1 && parents[c] < c;
        n_gone = 0;
        if (ok) path[0] = 0;
        for (int c = 1; ok && c < a.tokens; c++) {  // children of a node come after it
            if (parents[c] != cur) continue;
            const int tok = draft[c];
            if ((unsigned)tok >= (unsigned)a.vocab || (a.probs && child >= 0)) {
                ok = false;
                break;
            }
            const RowStats r = a.stats[base + cur];
            float w = weight(a, r, a.logits + (base + cur) * a.vocab, tok);
            bool take;
            if (a.probs) {
                take = __fmul_rn(a.uniforms[base + c], a.probs[(base + c) * a.vocab + tok]) < w / (float)r.total;
            } else {
                double left = r.total;
                for (int g = 0; g < n_gone; g++) {
                    left -= (double)weight(a, r, a.logits + (base + cur) * a.vocab, gone[g]);
                    if (gone[g] == tok) w = 0.0f;
                }
                take = (double)a.uniforms[base + c] * left < (double)w;
            }
            if (take) {
                cur = c;
                path[++count] = c;
                child = -1;
                n_gone = 0;
                ok = a.stats[base + c].best >= 0;
            } else {
                child = c;
                bool known = false;
                for (int g = 0; g < n_gone; g++) known |= gone[g] == tok;
                if (!known) gone[n_gone++] = tok;
            }
        }
        if (a.probs && child >= 0) {
            for (int c = child + 1; c < a.tokens; c++) ok = ok && parents[c] != cur;
        }
        at_node = ok ? cur : -1;
        refused = a.probs ? child : -1;
        if (a.probs) n_gone = 0;
        a.accepted[seq] = ok ? count : -1;
        if (!ok) {
            a.next[seq] = -1;
            for (int i = 0; i < a.tokens; i++) path[i] = -1;
        }
    }
    __syncthreads();
    if (at_node < 0) return;
    const float *row = a.logits + (base + at_node) * a.vocab;
    const RowStats r = a.stats[base + at_node];
    const int per = (a.vocab + 1023) / 1024, first = tid * per, last = min(first + per, a.vocab);
    const float total = (float)r.total;
    for (int pass = refused >= 0 ? 0 : 1; pass < 2; pass++) {
        const float *q = pass == 0 ? a.probs + (base + refused) * a.vocab : nullptr;
        auto left = [&](int v) -> double {
            float w = weight(a, r, row, v);
            if (q) return (double)fmaxf(w / total - q[v], 0.0f);
            for (int g = 0; g < n_gone; g++)
                if (gone[g] == v) w = 0.0f;
            return (double)(a.probs ? w / total : w);
        };
        double sum = 0.0;
        for (int v = first; v < last; v++) sum += left(v);
        // inclusive running sums over the threads' parts
        prefix[tid] = sum;
        __syncthreads();
        for (int d = 1; d < 1024; d <<= 1) {
            const double up = tid >= d ? prefix[tid - d] : 0.0;
            __syncthreads();
            prefix[tid] += up;
            __syncthreads();
        }
        const double whole = prefix[1023];
        if (!(whole > 0.0) && pass == 0) {
            __syncthreads();
            continue;  // the draft's distribution covers the target's: draw from the target's
        }
        const double aim = (double)a.uniforms[base] * whole;
        if (tid == 0) picked = -1;
        __syncthreads();
        double run = tid ? prefix[tid - 1] : 0.0;
        if (run <= aim && aim < prefix[tid]) {
            int pick = -1;
            for (int v = first; v < last; v++) {
                const double w = left(v);
                if (w > 0.0) pick = v;
                run += w;
                if (run > aim) break;
            }
            picked = pick;
        }
        __syncthreads();
        if (tid == 0) a.next[seq] = picked;
        break;
    }
}

}  // namespace

extern "C" int qg_verify_workspace_bytes(int seqs, int tokens, int vocab, size_t *bytes) {
    if (!bytes || seqs < 1 || seqs > kMaxSeqs || tokens < 1 || tokens > kMaxNodes || vocab < 1 || vocab > kMaxVocab)
        return cudaErrorInvalidValue;
    *bytes = (size_t)seqs * tokens * sizeof(RowStats);
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
    const VerifyArgs a = {path, accepted, next, logits, draft, parents, draft_probs, uniforms, scale, tokens, vocab,
                          static_cast<RowStats *>(workspace)};
    row_stats_kernel<<<seqs * tokens, 1024, 0, launch_stream>>>(a);
    if (int rc = cudaGetLastError()) return rc;
    walk_kernel<<<seqs, 1024, 0, launch_stream>>>(a);
    NB_CHECK_LAUNCH();
}

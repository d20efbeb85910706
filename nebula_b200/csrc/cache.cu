// What enters the paged cache and what stays there: the query/key preparation
// that stores a step's keys and values, and the commit of the accepted nodes.
#include <cooperative_groups.h>
#include "cache.cuh"

using namespace nb;
namespace cg = cooperative_groups;

namespace {

__global__ void rope_table_kernel(float2 *table, int positions, int half, double base) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (long long)positions * half) return;
    const int p = (int)(i / half), f = (int)(i % half);
    double s, c;
    sincos(p * pow(base, -(double)f / half), &s, &c);
    table[i] = make_float2((float)c, (float)s);
}

struct PrepArgs {
    CacheView c;
    float *q_out;
    const float *q, *k, *v, *q_weight, *k_weight;
    const float2 *rope;
    const int *offsets;
    int q_stride, k_stride, v_stride, rope_positions, half, tokens, q_heads, rows;
    float eps;
};

// One warp per (row, head): query heads, then key heads, then value heads.
// Lane l holds values l + 32j. The partner of a rotated value may sit in any
// lane (rotary is any even number), so the normalised head goes through the
// warp's part of shared memory.
template <int D>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const PrepArgs a) {
    constexpr int N = D / 32;
    __shared__ float head[8][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int heads = a.q_heads + 2 * a.c.kv_heads;
    const long long item = (long long)blockIdx.x * 8 + warp;
    if (item >= (long long)a.rows * heads) return;
    const int row = (int)(item / heads), h = (int)(item % heads);
    const int seq = row / a.tokens, node = row % a.tokens;
    const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + a.c.kv_heads;
    const int kv = is_q ? 0 : (h - a.q_heads) % a.c.kv_heads;

    const int length = a.c.committed(seq, a.tokens);
    const int pos = length + (a.offsets ? a.offsets[row] : node);
    long long at = length < 0 ? -1 : a.c.row(seq, length + node);
    if (a.half && (unsigned)pos >= (unsigned)a.rope_positions) at = -1;
    if (at < 0) {  // the header's refusals: NaN queries, no store
        if (is_q)
            for (int j = 0; j < N; j++)
                a.q_out[((size_t)row * a.q_heads + h) * D + lane + 32 * j] = __int_as_float(0x7fc00000);
        return;
    }
    const float *src = is_q ? a.q + (size_t)row * a.q_stride + (size_t)h * D
                            : (is_v ? a.v + (size_t)row * a.v_stride : a.k + (size_t)row * a.k_stride) + (size_t)kv * D;
    float x[N];
#pragma unroll
    for (int j = 0; j < N; j++) x[j] = src[lane + 32 * j];
    if (!is_v) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < N; j++) sum = fmaf(x[j], x[j], sum);
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        const float inv = rsqrtf(sum * (1.0f / D) + a.eps);
        const float *w = is_q ? a.q_weight : a.k_weight;
#pragma unroll
        for (int j = 0; j < N; j++) {
            x[j] = x[j] * inv * w[lane + 32 * j];
            head[warp][lane + 32 * j] = x[j];
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int i = lane + 32 * j;
            if (i < 2 * a.half) {
                const bool low = i < a.half;
                const float2 t = a.rope[(size_t)pos * a.half + (low ? i : i - a.half)];
                const float other = head[warp][low ? i + a.half : i - a.half];
                x[j] = low ? x[j] * t.x - other * t.y : x[j] * t.x + other * t.y;
            }
        }
    }
    if (is_q) {
#pragma unroll
        for (int j = 0; j < N; j++) a.q_out[((size_t)row * a.q_heads + h) * D + lane + 32 * j] = x[j];
    } else {
        __half *dst = (is_v ? a.c.v : a.c.k) + ((size_t)at * a.c.kv_heads + kv) * D;
#pragma unroll
        for (int j = 0; j < N; j++) dst[lane + 32 * j] = __float2half_rn(x[j]);
    }
}

struct CommitArgs {
    CacheView c;  // layer 0
    size_t layer_bytes;
    int layers, tokens;
    int *lengths_out;
    const int *path, *accepted;
};

constexpr int kCommitCtas = 8;  // one cluster per sequence

// The rows of one sequence move by one cluster; a thread owns a 16-byte column
// of one layer's key or value rows and moves it for every accepted node. path
// ascends, so path[i] >= i: a destination is never a later node's source, and
// a thread that reads nodes in ascending order before it writes them moves
// them as if at once. The length is written after the cluster's barrier, when
// every CTA has read it, so lengths_out may be the cache's own.
__global__ void __cluster_dims__(kCommitCtas, 1, 1) __launch_bounds__(256) cache_commit_kernel(const CommitArgs a) {
    __shared__ long long from[kMaxNodes], to[kMaxNodes];
    __shared__ int moves;
    cg::cluster_group cluster = cg::this_cluster();
    const int seq = blockIdx.x / kCommitCtas, part = blockIdx.x % kCommitCtas;
    const int length = a.c.committed(seq, a.tokens);
    const int n = a.accepted[seq];
    if (threadIdx.x == 0) {
        int m = length >= 0 && n >= 0 && n < a.tokens ? 0 : -1, last = 0;
        for (int i = 1; m >= 0 && i <= n; i++) {
            const int p = a.path[(size_t)seq * a.tokens + i];
            if (p <= last || p >= a.tokens) {
                m = -1;
                break;
            }
            last = p;
            if (p == i) continue;
            from[m] = a.c.row(seq, length + p);
            to[m] = a.c.row(seq, length + i);
            if (from[m] < 0 || to[m] < 0) m = -1;
            else m++;
        }
        moves = m;
    }
    __syncthreads();
    if (moves > 0) {
        const size_t width = (size_t)a.c.kv_heads * a.c.head_dim * sizeof(__half) / 16;  // 16-byte columns of a row
        const size_t columns = width * 2 * a.layers;
        for (size_t col = (size_t)part * 256 + threadIdx.x; col < columns; col += kCommitCtas * 256) {
            const size_t pool = col / width, x = col % width;
            uint4 *base = reinterpret_cast<uint4 *>(reinterpret_cast<char *>(pool & 1 ? a.c.v : a.c.k) +
                                                    (pool >> 1) * a.layer_bytes) + x;
            for (int i = 0; i < moves; i++) base[to[i] * width] = base[from[i] * width];
        }
    }
    cluster.sync();
    if (part == 0 && threadIdx.x == 0) a.lengths_out[seq] = moves >= 0 ? length + n + 1 : a.c.lengths[seq];
}

}  // namespace

extern "C" int qg_rope_table(float *table, int positions, int rotary, double base) {
    if (!table || positions < 1 || rotary < 2 || rotary > 256 || rotary % 2 || !(base > 0)) return cudaErrorInvalidValue;
    const long long n = (long long)positions * (rotary / 2);
    rope_table_kernel<<<(unsigned)((n + 255) / 256), 256, 0, launch_stream>>>(reinterpret_cast<float2 *>(table), positions,
                                                                               rotary / 2, base);
    NB_CHECK_LAUNCH();
}

extern "C" int qg_qk_norm_rope(float *q_out, const qg_kv_cache *cache, int layer, const float *q, int q_stride,
                               const float *k, int k_stride, const float *v, int v_stride, const float *q_weight,
                               const float *k_weight, float eps, const float *rope, int rope_positions, int rotary,
                               const int *offsets, int seqs, int tokens, int q_heads) {
    PrepArgs a;
    if (int rc = cache_view(cache, layer, seqs, tokens, a.c)) return rc;
    const int D = a.c.head_dim;
    if (!q_out || !q || !k || !v || !q_weight || !k_weight || !(eps >= 0.0f) || q_heads < 1 || q_heads > 1024 ||
        rotary < 0 || rotary % 2 || rotary > D || (rotary && (!rope || rope_positions < 1)) ||
        (reinterpret_cast<uintptr_t>(rope) & 7))
        return cudaErrorInvalidValue;
    if (q_stride < q_heads * D || k_stride < a.c.kv_heads * D || v_stride < a.c.kv_heads * D ||
        (q_out == q && q_stride != q_heads * D))
        return cudaErrorInvalidValue;
    a.q_out = q_out;
    a.q = q, a.k = k, a.v = v;
    a.q_weight = q_weight, a.k_weight = k_weight;
    a.rope = reinterpret_cast<const float2 *>(rope);
    a.offsets = offsets;
    a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride;
    a.rope_positions = rope_positions;
    a.half = rotary / 2;
    a.tokens = tokens, a.q_heads = q_heads, a.rows = seqs * tokens;
    a.eps = eps;
    const long long items = (long long)a.rows * (q_heads + 2 * a.c.kv_heads);
    const unsigned grid = (unsigned)((items + 7) / 8);
    if (D == 64) qk_norm_rope_kernel<64><<<grid, 256, 0, launch_stream>>>(a);
    else if (D == 128) qk_norm_rope_kernel<128><<<grid, 256, 0, launch_stream>>>(a);
    else qk_norm_rope_kernel<256><<<grid, 256, 0, launch_stream>>>(a);
    NB_CHECK_LAUNCH();
}

extern "C" int qg_cache_commit(const qg_kv_cache *cache, int *lengths_out, const int *path, const int *accepted, int seqs,
                               int tokens) {
    CommitArgs a;
    if (int rc = cache_view(cache, 0, seqs, tokens, a.c)) return rc;
    if (!lengths_out || !path || !accepted) return cudaErrorInvalidValue;
    a.layer_bytes = cache->layer_bytes;
    a.layers = cache->layers;
    a.tokens = tokens;
    a.lengths_out = lengths_out;
    a.path = path;
    a.accepted = accepted;
    cache_commit_kernel<<<seqs * kCommitCtas, 256, 0, launch_stream>>>(a);
    NB_CHECK_LAUNCH();
}

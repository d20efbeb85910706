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
    int q_stride, k_stride, v_stride, rope_positions, half, tokens, q_heads;
    float eps;
};

// W neighbouring floats; WIDE: in one load. (Not through the read-only path: q may be q_out.)
template <bool WIDE, int W>
__device__ __forceinline__ void load(float (&x)[W], const float *p) {
    if constexpr (W == 4 && WIDE) {
        *reinterpret_cast<float4 *>(x) = *reinterpret_cast<const float4 *>(p);
    } else if constexpr (W == 2 && WIDE) {
        *reinterpret_cast<float2 *>(x) = *reinterpret_cast<const float2 *>(p);
    } else {
#pragma unroll
        for (int e = 0; e < W; e++) x[e] = p[e];
    }
}

// One warp per row and kHeads of its heads: query heads, then key heads, then
// value heads. Lane l holds values W*l .. W*l+W-1 of each 128 (64 for heads of
// 64) of a head. The heads' values are asked for first; the length, the page and
// the table's angles, each of which depends on the one before, arrive meanwhile
// and serve both heads (96 x 17 rows of 24 + 4 heads of 256: 22.6 us; one head to a warp 24.6, four 26.7; with the chained
// launch 20.6). The partner of a rotated value sits in another lane, so the rotated part of the normalised head goes through
// the warp's part of shared memory. For many rows bound by the latency of its loads: 64 registers leave 37 % of the warps, which
// wait for memory most of the time (issue slots 48 %, HBM 30 %); for one verify batch by the launch.
constexpr int kHeads = 2;

// WIDE: all rows of q, k, v, q_out and the weights start on 16-byte boundaries, and the rotated halves and the table's
// rows are whole loads of a lane (before, the instructions took two thirds of the issue slots).
template <int D, bool WIDE>
__global__ void __launch_bounds__(256, 4) qk_norm_rope_kernel(const __grid_constant__ PrepArgs a) {
    constexpr int W = D == 64 ? 2 : 4, N = D / (32 * W);
    __shared__ __align__(16) float head[8][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int heads = a.q_heads + 2 * a.c.kv_heads;
    const int row = blockIdx.x, h0 = ((int)(blockIdx.y * blockDim.x / 32) + warp) * kHeads;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (h0 >= heads) return;
    const int seq = row / a.tokens, node = row - seq * a.tokens;
    float x[kHeads][N][W];
#pragma unroll
    for (int g = 0; g < kHeads; g++) {
        const int h = min(h0 + g, heads - 1), k = h - a.q_heads, v = k - a.c.kv_heads;
        const float *src = k < 0   ? a.q + (size_t)row * a.q_stride + (size_t)h * D
                           : v < 0 ? a.k + (size_t)row * a.k_stride + (size_t)k * D
                                   : a.v + (size_t)row * a.v_stride + (size_t)v * D;
#pragma unroll
        for (int j = 0; j < N; j++) load<WIDE>(x[g][j], src + 32 * W * j + W * lane);
    }
    const int length = a.c.committed(seq, a.tokens);
    const int pos = length + (a.offsets ? a.offsets[row] : node);
    long long at = length < 0 ? -1 : a.c.row(seq, length + node);
    if (a.half && (unsigned)pos >= (unsigned)a.rope_positions) at = -1;
    float2 turn[N][W];
    const float2 *angles = a.rope + (size_t)pos * a.half;
#pragma unroll
    for (int j = 0; j < N; j++) {
        const int i0 = 32 * W * j + W * lane;
        if (at < 0 || i0 >= 2 * a.half) continue;
        if constexpr (WIDE) {
#pragma unroll
            for (int e = 0; e < W; e += 2)
                *reinterpret_cast<float4 *>(&turn[j][e]) = __ldg(reinterpret_cast<const float4 *>(angles + (i0 < a.half ? i0 : i0 - a.half) + e));
        } else {
#pragma unroll
            for (int e = 0; e < W; e++)
                if (i0 + e < 2 * a.half) turn[j][e] = __ldg(angles + (i0 + e < a.half ? i0 + e : i0 + e - a.half));
        }
    }
#pragma unroll
    for (int g = 0; g < kHeads; g++) {
        const int h = h0 + g, k = h - a.q_heads, v = k - a.c.kv_heads;
        if (h >= heads) break;
        if (v < 0) {
            const float *weight = (k < 0 ? a.q_weight : a.k_weight) + W * lane;
            float w[N][W], sum = 0.0f;
#pragma unroll
            for (int j = 0; j < N; j++) {
                load<WIDE>(w[j], weight + 32 * W * j);
#pragma unroll
                for (int e = 0; e < W; e++) sum = fmaf(x[g][j][e], x[g][j][e], sum);
            }
#pragma unroll
            for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            const float inv = rsqrtf(sum * (1.0f / D) + a.eps);
            __syncwarp();
#pragma unroll
            for (int j = 0; j < N; j++)
#pragma unroll
                for (int e = 0; e < W; e++) {
                    x[g][j][e] = x[g][j][e] * inv * w[j][e];
                }
#pragma unroll
            for (int j = 0; j < N; j++)
                if (32 * W * j < 2 * a.half) {
                    if constexpr (W == 4) *reinterpret_cast<float4 *>(&head[warp][32 * W * j + W * lane]) = *reinterpret_cast<float4 *>(x[g][j]);
                    else *reinterpret_cast<float2 *>(&head[warp][32 * W * j + W * lane]) = *reinterpret_cast<float2 *>(x[g][j]);
                }
            __syncwarp();
#pragma unroll
            for (int j = 0; j < N; j++) {
                const int i0 = 32 * W * j + W * lane;
                if (i0 >= 2 * a.half) continue;
                if constexpr (WIDE) {
                    const bool low = i0 < a.half;
                    float other[W];
                    load<true>(other, &head[warp][low ? i0 + a.half : i0 - a.half]);
#pragma unroll
                    for (int e = 0; e < W; e++)
                        x[g][j][e] = fmaf(other[e], low ? -turn[j][e].y : turn[j][e].y, x[g][j][e] * turn[j][e].x);
                } else {
#pragma unroll
                    for (int e = 0; e < W; e++) {
                        const int i = i0 + e;
                        if (i >= 2 * a.half) continue;
                        const bool low = i < a.half;
                        const float other = head[warp][low ? i + a.half : i - a.half];
                        const float2 t = turn[j][e];
                        x[g][j][e] = low ? x[g][j][e] * t.x - other * t.y : x[g][j][e] * t.x + other * t.y;
                    }
                }
            }
        }
        if (k < 0) {
            float *out = a.q_out + ((size_t)row * a.q_heads + h) * D + W * lane;
#pragma unroll
            for (int j = 0; j < N; j++) {
                if (at < 0)  // the header's refusals: NaN queries, no store
#pragma unroll
                    for (int e = 0; e < W; e++) x[g][j][e] = __int_as_float(0x7fc00000);
                if constexpr (W == 4 && WIDE) *reinterpret_cast<float4 *>(out + 32 * W * j) = *reinterpret_cast<float4 *>(x[g][j]);
                else
#pragma unroll
                    for (int e = 0; e < W; e++) out[32 * W * j + e] = x[g][j][e];
            }
        } else if (at >= 0) {
            // cache rows are 16-byte aligned
            __half2 *dst = reinterpret_cast<__half2 *>((v < 0 ? a.c.k : a.c.v) + ((size_t)at * a.c.kv_heads + (v < 0 ? k : v)) * D + W * lane);
#pragma unroll
            for (int j = 0; j < N; j++) {
                __half2 y[W / 2];
#pragma unroll
                for (int e = 0; e < W / 2; e++) y[e] = __floats2half2_rn(x[g][j][2 * e], x[g][j][2 * e + 1]);
                if constexpr (W == 4) *reinterpret_cast<uint2 *>(dst + 16 * W * j) = *reinterpret_cast<uint2 *>(y);
                else dst[16 * W * j] = y[0];
            }
        }
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
// them as if at once. Eight are read before they are written: with one at a
// time each move waits for its own load (48 sequences x 24 layers: 45 us, so 32). Nodes
// already in place are a prefix. The length is written after the cluster's
// barrier, when every CTA has read it, so lengths_out may be the cache's own.
// Bound by HBM for many sequences, by the chain length - page - row for one.
__global__ void __cluster_dims__(kCommitCtas, 1, 1) __launch_bounds__(256) cache_commit_kernel(const __grid_constant__ CommitArgs a) {
    __shared__ long long from[kMaxNodes], to[kMaxNodes];
    cg::cluster_group cluster = cg::this_cluster();
    const int seq = blockIdx.x / kCommitCtas, part = blockIdx.x % kCommitCtas, i = threadIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int n = a.accepted[seq];
    const int p = i < a.tokens ? a.path[(size_t)seq * a.tokens + i] : 0;
    const int before = i > 0 && i < a.tokens ? a.path[(size_t)seq * a.tokens + i - 1] : -1;
    const int length = a.c.committed(seq, a.tokens);
    bool sound = length >= 0 && n >= 0 && n < a.tokens, moves = false;
    if (sound && i > 0 && i <= n) {
        // the root is not read: the first draft only has to come after it
        sound = p < a.tokens && p > (i == 1 ? 0 : before);
        if (sound && p != i) {
            from[i] = a.c.row(seq, length + p);
            to[i] = a.c.row(seq, length + i);
            sound = from[i] >= 0 && to[i] >= 0;
            moves = true;
        }
    }
    sound = __syncthreads_and(sound);
    const int count = __syncthreads_count(moves);
    if (sound && count) {
        const size_t width = (size_t)a.c.kv_heads * a.c.head_dim * sizeof(__half) / 16;  // 16-byte columns of a row
        const unsigned columns = (unsigned)(width * 2 * a.layers);
        for (unsigned col = part * 256 + i; col < columns; col += kCommitCtas * 256) {
            const unsigned pool = col / (unsigned)width, x = col % (unsigned)width;
            uint4 *base = reinterpret_cast<uint4 *>(reinterpret_cast<char *>(pool & 1 ? a.c.v : a.c.k) +
                                                    (pool >> 1) * a.layer_bytes) + x;
            for (int m = n - count + 1; m <= n; m += 8) {
                uint4 v[8];
#pragma unroll
                for (int k = 0; k < 8; k++)
                    if (m + k <= n) v[k] = base[from[m + k] * width];
#pragma unroll
                for (int k = 0; k < 8; k++)
                    if (m + k <= n) base[to[m + k] * width] = v[k];
            }
        }
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    cluster.sync();
    if (part == 0 && i == 0) a.lengths_out[seq] = sound ? length + n + 1 : a.c.lengths[seq];
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
    a.tokens = tokens, a.q_heads = q_heads;
    a.eps = eps;
    const bool wide = !((reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
                         reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(q_weight) | reinterpret_cast<uintptr_t>(k_weight) |
                         reinterpret_cast<uintptr_t>(rope)) & 15) &&
                      !((q_stride | k_stride | v_stride | a.half) & 3);
    // the warps of a row in as few blocks as hold them, evenly
    const int groups = (q_heads + 2 * a.c.kv_heads + kHeads - 1) / kHeads, blocks = (groups + 7) / 8;
    const dim3 grid(seqs * tokens, blocks);
    const int threads = 32 * ((groups + blocks - 1) / blocks);
    const auto kernel = D == 64    ? wide ? qk_norm_rope_kernel<64, true> : qk_norm_rope_kernel<64, false>
                        : D == 128 ? wide ? qk_norm_rope_kernel<128, true> : qk_norm_rope_kernel<128, false>
                                   : wide ? qk_norm_rope_kernel<256, true> : qk_norm_rope_kernel<256, false>;
    return launch_chained(kernel, grid, threads, a);
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
    // A chained launch hides what the kernel before leaves of the launch (one sequence 3.6 us in place of 4.4 to 5.1); with
    // more clusters than the GPU takes at once it only adds (48 sequences 32.6 us in place of 31.4).
    if (seqs * kCommitCtas <= kSms) return launch_chained(cache_commit_kernel, dim3(seqs * kCommitCtas), 256, a);
    cache_commit_kernel<<<seqs * kCommitCtas, 256, 0, launch_stream>>>(a);
    NB_CHECK_LAUNCH();
}

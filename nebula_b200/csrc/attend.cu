// Attention of drafted tokens (a tree) over the paged cache.
#include "cache.cuh"

using namespace nb;

namespace {

struct AttendArgs {
    CacheView c;
    float *out;
    const float *q;
    const uint64_t *tree;
    float scale;
    int tokens, q_heads;
};

constexpr int kWarps = 8;

// One CTA per (row, query head); warps take keys in turn with a running
// maximum and sum, and join at the end. Every 32 keys the sums join those of
// the keys before: one running sum over thousands of small weights beside a
// large one would round each of them in the same direction.
template <int D>
__global__ void __launch_bounds__(32 * kWarps) tree_attention_kernel(const AttendArgs a) {
    constexpr int N = D / 32;
    __shared__ float acc[kWarps][D], top[kWarps], total[kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = blockIdx.x, h = blockIdx.y, seq = row / a.tokens, node = row % a.tokens;
    const int kv = h / (a.q_heads / a.c.kv_heads);
    const int length = a.c.committed(seq, a.tokens);
    const uint64_t seen = a.tree ? a.tree[row] : node == 63 ? ~0ull : (2ull << node) - 1;
    float q[N], o[N], far_o[N], m = -INFINITY, l = 0.0f, far_l = 0.0f;
#pragma unroll
    for (int j = 0; j < N; j++) {
        q[j] = a.q[((size_t)row * a.q_heads + h) * D + lane + 32 * j] * a.scale;
        o[j] = far_o[j] = 0.0f;
    }
    bool bad = length < 0;
    const int n = bad ? 0 : length + a.tokens;
    int taken = 0;
    for (int p = warp; p < n; p += kWarps) {
        const long long at = a.c.row(seq, p);
        if (at < 0) {
            bad = true;
            continue;
        }
        if (p >= length && !(seen >> (p - length) & 1)) continue;
        const __half *k = a.c.k + ((size_t)at * a.c.kv_heads + kv) * D, *v = a.c.v + ((size_t)at * a.c.kv_heads + kv) * D;
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < N; j++) s = fmaf(q[j], __half2float(k[lane + 32 * j]), s);
#pragma unroll
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        const float mx = fmaxf(m, s);
        const float keep = m == -INFINITY ? 0.0f : expf(m - mx), w = s == -INFINITY ? 0.0f : expf(s - mx);
        const bool join = (++taken & 31) == 0;
        l = l * keep + w;
        far_l = far_l * keep + (join ? l : 0.0f);
        l = join ? 0.0f : l;
#pragma unroll
        for (int j = 0; j < N; j++) {
            o[j] = fmaf(w, __half2float(v[lane + 32 * j]), o[j] * keep);
            far_o[j] = far_o[j] * keep + (join ? o[j] : 0.0f);
            o[j] = join ? 0.0f : o[j];
        }
        m = mx;
    }
#pragma unroll
    for (int j = 0; j < N; j++) acc[warp][lane + 32 * j] = o[j] + far_o[j];
    if (lane == 0) {
        top[warp] = m;
        total[warp] = l + far_l;
    }
    bad = __syncthreads_or(bad);
    float mx = -INFINITY, sum = 0.0f;
    for (int w = 0; w < kWarps; w++) mx = fmaxf(mx, top[w]);
    for (int w = 0; w < kWarps; w++) sum += top[w] == -INFINITY ? total[w] : total[w] * expf(top[w] - mx);
    for (int i = threadIdx.x; i < D; i += 32 * kWarps) {
        float v = 0.0f;
        for (int w = 0; w < kWarps; w++) v += top[w] == -INFINITY ? acc[w][i] : acc[w][i] * expf(top[w] - mx);
        v = sum == 0.0f ? 0.0f : v / sum;
        a.out[((size_t)row * a.q_heads + h) * D + i] = bad ? __int_as_float(0x7fc00000) : v;
    }
}

}  // namespace

extern "C" int qg_attention_workspace_bytes(int seqs, int tokens, int q_heads, int kv_heads, int head_dim, size_t *bytes) {
    if (!bytes || seqs < 1 || seqs > kMaxSeqs || tokens < 1 || tokens > kMaxNodes || kv_heads < 1 || kv_heads > 1024 ||
        q_heads < kv_heads || q_heads > 1024 || q_heads % kv_heads || (head_dim != 64 && head_dim != 128 && head_dim != 256))
        return cudaErrorInvalidValue;
    *bytes = 256;
    return cudaSuccess;
}

extern "C" int qg_tree_attention(float *out, const float *q, const qg_kv_cache *cache, int layer, const uint64_t *tree,
                                 float scale, int seqs, int tokens, int q_heads, void *workspace) {
    AttendArgs a;
    if (int rc = cache_view(cache, layer, seqs, tokens, a.c)) return rc;
    if (!out || !q || !workspace || q_heads < a.c.kv_heads || q_heads > 1024 || q_heads % a.c.kv_heads ||
        ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(workspace)) & 15) ||
        (reinterpret_cast<uintptr_t>(tree) & 7))
        return cudaErrorInvalidValue;
    a.out = out;
    a.q = q;
    a.tree = tree;
    a.scale = scale;
    a.tokens = tokens;
    a.q_heads = q_heads;
    const dim3 grid(seqs * tokens, q_heads);
    if (a.c.head_dim == 64) tree_attention_kernel<64><<<grid, 32 * kWarps, 0, launch_stream>>>(a);
    else if (a.c.head_dim == 128) tree_attention_kernel<128><<<grid, 32 * kWarps, 0, launch_stream>>>(a);
    else tree_attention_kernel<256><<<grid, 32 * kWarps, 0, launch_stream>>>(a);
    NB_CHECK_LAUNCH();
}

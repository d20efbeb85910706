// The paged key/value cache of the verify step (qg_kv_cache) as kernels see it.
#pragma once
#include "common.cuh"

namespace nb {

constexpr int kMaxSeqs = 1024;
constexpr int kMaxNodes = 64;  // one 64-bit mask per node
constexpr int kSms = 148;      // of a B200; no kernel needs its CTAs to run at the same time beyond a cluster

struct CacheView {
    __half *k, *v;  // one layer's pools
    const int *table;
    const int *lengths;
    int pages, shift, table_pages, kv_heads, head_dim;

    __host__ __device__ int page_tokens() const { return 1 << shift; }
    // Committed tokens of a sequence, or -1 when its length leaves no room for its nodes.
    __device__ int committed(int seq, int tokens) const {
        const int n = lengths[seq];
        return n >= 0 && n <= (table_pages << shift) - tokens ? n : -1;
    }
    // Pool row of a position (64 bits: a pool may hold more than 2^31 values), or -1 for a page outside the pool.
    __device__ long long row(int seq, int pos) const {
        const int page = table[(size_t)seq * table_pages + (pos >> shift)];
        if ((unsigned)page >= (unsigned)pages) return -1;
        return ((long long)page << shift) + (pos & (page_tokens() - 1));
    }
};

// A launch that may begin while the stream's previous kernel ends; the kernel waits (griddepcontrol.wait) before it touches
// memory.
template <typename Args>
inline int launch_chained(void (*kernel)(Args), dim3 grid, int threads, const Args &args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = launch_stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args);
}

// Checks what the header asks of a cache and a batch; cudaErrorInvalidValue before any launch.
inline int cache_view(const qg_kv_cache *c, int layer, int seqs, int tokens, CacheView &view) {
    if (!c || !c->k || !c->v || !c->page_table || !c->lengths || seqs < 1 || seqs > kMaxSeqs || tokens < 1 ||
        tokens > kMaxNodes)
        return cudaErrorInvalidValue;
    if (c->layers < 1 || layer < 0 || layer >= c->layers || c->pages < 1 || c->table_pages < 1 || c->kv_heads < 1 ||
        c->kv_heads > 1024 || (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256))
        return cudaErrorInvalidValue;
    int shift = 4;
    while (shift <= 8 && (1 << shift) != c->page_tokens) shift++;
    if (shift > 8) return cudaErrorInvalidValue;
    // pool rows are 32-bit coordinates, and so is the end of the 128 keys that a sequence's last position lies in
    if (((long long)c->pages << shift) > 0x7fffffffll || ((long long)c->table_pages << shift) > 0x7fffff80ll)
        return cudaErrorInvalidValue;
    const size_t pool = ((size_t)c->pages << shift) * c->kv_heads * c->head_dim * sizeof(__half);
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) return cudaErrorInvalidValue;
    if (c->layers > 1 && (c->layer_bytes < pool || c->layer_bytes % 16)) return cudaErrorInvalidValue;
    view.k = reinterpret_cast<__half *>(static_cast<char *>(c->k) + layer * c->layer_bytes);
    view.v = reinterpret_cast<__half *>(static_cast<char *>(c->v) + layer * c->layer_bytes);
    view.table = c->page_table;
    view.lengths = c->lengths;
    view.pages = c->pages;
    view.shift = shift;
    view.table_pages = c->table_pages;
    view.kv_heads = c->kv_heads;
    view.head_dim = c->head_dim;
    return 0;
}

}  // namespace nb

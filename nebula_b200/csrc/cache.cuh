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
    const int *held;  // entries of a row that are its sequence's pages, or NULL: all
    int pages, shift, table_pages;
    short kv_heads, head_dim;  // 16 bits: 8 bytes more of arguments cost a commit of one sequence 0.35 of 3.9 us

    __host__ __device__ int page_tokens() const { return 1 << shift; }
    // Committed tokens of a sequence, or -1 when its length leaves no room for its nodes: in the table, or on the pages that it
    // has. What its row names behind those may be another sequence's by now.
    __device__ int committed(int seq, int tokens) const {
        // (A load under a predicate: as a branch it takes registers that the attention's roles do not have. One sequence of 98k
        // keys and heads of 256 106.5 us, so 102.9, and 103.1 without the check.)
        const int n = lengths[seq];
        int room;
        asm volatile("{.reg .pred p;\n setp.ne.u64 p, %1, 0;\n mov.b32 %0, %3;\n @p ld.global.b32 %0, [%2];}"
                     : "=r"(room)
                     : "l"(held), "l"(held + seq), "r"(table_pages));
        return n >= 0 && (unsigned)room <= (unsigned)table_pages && n <= (room << shift) - tokens ? n : -1;
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

// log2 of a page's tokens: 16, 32, 64, 128 or 256; -1 for others.
inline int page_shift(int page_tokens) {
    for (int shift = 4; shift <= 8; shift++)
        if (1 << shift == page_tokens) return shift;
    return -1;
}
// Pool rows are 32-bit coordinates, and so is the end of the 128 keys that a sequence's last position lies in.
inline bool pool_too_large(int pages, int table_pages, int shift) {
    return ((long long)pages << shift) > 0x7fffffffll || ((long long)table_pages << shift) > 0x7fffff80ll;
}

// Checks what the header asks of a cache and a batch; cudaErrorInvalidValue before any launch.
inline int cache_view(const qg_kv_cache *c, int layer, int seqs, int tokens, CacheView &view) {
    if (!c || !c->k || !c->v || !c->page_table || !c->lengths || seqs < 1 || seqs > kMaxSeqs || tokens < 1 ||
        tokens > kMaxNodes)
        return cudaErrorInvalidValue;
    if (c->layers < 1 || layer < 0 || layer >= c->layers || c->pages < 1 || c->table_pages < 1 || c->kv_heads < 1 ||
        c->kv_heads > 1024 || (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256))
        return cudaErrorInvalidValue;
    // (a caller that knows nothing of held may not have set it)
    const bool has_held = c->page_tokens & QG_CACHE_HELD;
    const int shift = page_shift(c->page_tokens & ~QG_CACHE_HELD);
    if (has_held && (!c->held || (reinterpret_cast<uintptr_t>(c->held) & 3))) return cudaErrorInvalidValue;
    if (shift < 0 || pool_too_large(c->pages, c->table_pages, shift)) return cudaErrorInvalidValue;
    const size_t pool = ((size_t)c->pages << shift) * c->kv_heads * c->head_dim * sizeof(__half);
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) return cudaErrorInvalidValue;
    if (c->layers > 1 && (c->layer_bytes < pool || c->layer_bytes % 16)) return cudaErrorInvalidValue;
    view.k = reinterpret_cast<__half *>(static_cast<char *>(c->k) + layer * c->layer_bytes);
    view.v = reinterpret_cast<__half *>(static_cast<char *>(c->v) + layer * c->layer_bytes);
    view.table = c->page_table;
    view.lengths = c->lengths;
    view.held = has_held ? c->held : nullptr;
    view.pages = c->pages;
    view.shift = shift;
    view.table_pages = c->table_pages;
    view.kv_heads = (short)c->kv_heads;
    view.head_dim = (short)c->head_dim;
    return 0;
}

}  // namespace nb

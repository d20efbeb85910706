// The pages of a cache for many sequences, handed out and taken back on the GPU: page tables and the map from a step's new
// positions to pool rows, from nothing but lengths.
//
// Free pages are a stack. One cluster does a call: a thread per sequence, so every CTA makes the same prefix sum of what the
// sequences need (or give back) in its own shared memory, then takes its share of the entries to write. What the call
// changes and all CTAs read (pages held, the stack's height) is written after a barrier of the cluster. Bound by latency:
// launch, one trip for the lengths, one for the stack or the table, the barrier. Where there are many slots to write a second
// kernel does it on the whole GPU, from the page tables that the first one has left (700 sequences of up to 512 new positions:
// releasing and reserving 17 us with one kernel each, 12 with the third). Four sequences of 17: 7 us for both calls.
#include "cache.cuh"

using namespace nb;

namespace {

constexpr int kThreads = 1024;      // one per sequence
constexpr int kPagesCluster = 8;    // CTAs where there is more than kOneCta to write
constexpr long long kOneCta = 4096;
constexpr int kChunk = 256;         // slots that a warp takes at a time
constexpr long long kWide = 65536;  // slots that get a kernel of their own
static_assert(kThreads >= kMaxSeqs, "a thread per sequence");

struct PagesArgs {
    int *table, *held, *stack, *height;
    int pages, shift, table_pages;
    int *slots, *out;
    const int *lengths, *counts;
    int seqs, tokens, shared;
};

struct Need {
    int held;    // pages before the call
    int first;   // of all sequences' pages, which are this one's
    int count;   // pages taken or given back
    int length;  // positions before the new ones
    int fresh;   // new positions, or -1: none of them has a place
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

// Sum over the threads up to this one, and over all. 64 bits: what sequences ask for is bounded by their tables, not by the
// pool.
__device__ long long block_scan(long long x, long long &all) {
    __shared__ long long sums[kThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long upto = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += y;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    long long before = 0;
    all = 0;
    const long long mine = sums[lane];
    before = lane < warp ? mine : 0;
    all = mine;
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, d);
        all += __shfl_xor_sync(0xffffffffu, all, d);
    }
    return before + upto;
}

// The sequence whose pages hold page `at` of all: the last one that starts at or before it.
__device__ __forceinline__ int owner(const Need *need, int seqs, int at) {
    int lo = 0, hi = seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (need[mid].first <= at) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(kThreads, 1) reserve_kernel(const __grid_constant__ PagesArgs a) {
    __shared__ Need need[kThreads];
    const int s = threadIdx.x, rank = cluster_rank(), ranks = cluster_size();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int height = *a.height;
    if ((unsigned)height > (unsigned)a.pages) height = 0;
    int length = 0, fresh = 0, held = 0, wanted = 0, out = -1;
    if (s < a.seqs) {
        length = a.lengths[s], held = a.held[s], fresh = a.counts ? a.counts[s] : a.tokens;
        const long long end = (long long)length + fresh;
        if (length < 0 || fresh < 0 || fresh > a.tokens || end > (long long)a.table_pages << a.shift || (unsigned)held > (unsigned)a.table_pages) fresh = -1;
        else wanted = max(0, (int)((end + (1 << a.shift) - 1) >> a.shift) - held), out = wanted;
    }
    long long all;
    const long long upto = block_scan(wanted, all);
    if (fresh >= 0 && wanted && upto > height) fresh = -1, wanted = 0, out = -2;
    // Sequences that get pages come before all that are refused for want of them, so theirs are the stack's first ones. The
    // others' places are those after them all: `owner` finds none of these.
    const int first = (int)min(upto - wanted, (long long)height);
    need[s] = {held, first, wanted, length, fresh};
    long long given;
    __syncthreads();  // (block_scan's own sums)
    block_scan(wanted, given);
    __syncthreads();
    if (ranks > 1) cluster_sync();  // every CTA has read what rank 0 changes
    if (rank == 0) {
        if (s < a.seqs) {
            a.out[s] = out;
            if (wanted) a.held[s] = held + wanted;
        }
        if (s == 0 && given) *a.height = height - (int)given;
    }
    // Page i of all those given is the i-th from the stack's top.
    for (int i = rank * kThreads + s; i < (int)given; i += ranks * kThreads) {
        const int q = owner(need, a.seqs, i);
        a.table[(size_t)q * a.table_pages + need[q].held + (i - need[q].first)] = a.stack[height - 1 - i];
    }
    if (!a.slots) return;
    const int chunks = (a.tokens + kChunk - 1) / kChunk, lane = s & 31, mask = (1 << a.shift) - 1;
    for (int u = rank * (kThreads / 32) + (s >> 5); u < a.seqs * chunks; u += ranks * (kThreads / 32)) {
        const int q = u / chunks, from = (u - q * chunks) * kChunk, to = min(from + kChunk, a.tokens);
        const Need n = need[q];
        const int *row = a.table + (size_t)q * a.table_pages;
#pragma unroll 4
        for (int i = from + lane; i < to; i += 32) {
            int slot = -1;
            if (i < n.fresh) {
                const int at = n.length + i, p = at >> a.shift;
                const int page = p < n.held ? row[p] : a.stack[height - 1 - (n.first + p - n.held)];
                if ((unsigned)page < (unsigned)a.pages) slot = page << a.shift | (at & mask);
            }
            a.slots[(size_t)q * a.tokens + i] = slot;
        }
    }
}

__global__ void __launch_bounds__(kThreads, 1) release_kernel(const __grid_constant__ PagesArgs a) {
    __shared__ Need need[kThreads];
    const int s = threadIdx.x, rank = cluster_rank(), ranks = cluster_size();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int height = *a.height;
    int stay = 0, gone = 0, out = -1;
    if (s < a.seqs) {
        const int held = a.held[s];
        const long long keep = ((long long)max(0, a.lengths[s]) + (1 << a.shift) - 1) >> a.shift;
        if ((unsigned)held <= (unsigned)a.table_pages) {
            stay = (int)min(max(keep, (long long)a.shared), (long long)held);
            out = gone = held - stay;
        }
    }
    long long all;
    const long long upto = block_scan(gone, all);
    const bool fits = height >= 0 && height + all <= a.pages;  // more than the pool has: some page is given back twice
    if (!fits && gone) out = -1;
    need[s] = {stay, (int)min(upto - gone, (long long)a.pages), gone, 0, 0};
    __syncthreads();
    if (ranks > 1) cluster_sync();  // every CTA has read what rank 0 changes
    if (rank == 0) {
        if (s < a.seqs) {
            a.out[s] = out;
            if (fits && gone) a.held[s] = stay;
        }
        if (s == 0 && fits && all) *a.height = height + (int)all;
    }
    if (!fits) return;
    // Page i of all those given back becomes the i-th from the stack's new top.
    for (int i = rank * kThreads + s; i < (int)all; i += ranks * kThreads) {
        const int q = owner(need, a.seqs, i);
        a.stack[height + (int)all - 1 - i] = a.table[(size_t)q * a.table_pages + need[q].held + (i - need[q].first)];
    }
}

// The slots alone, four at a time where that is how they lie, after reserve_kernel.
__global__ void __launch_bounds__(256) slots_kernel(const __grid_constant__ PagesArgs a) {
    const int lane = threadIdx.x & 31, chunks = (a.tokens + kChunk - 1) / kChunk, u = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int q = u / chunks, from = (u - q * chunks) * kChunk, to = min(from + kChunk, a.tokens), mask = (1 << a.shift) - 1;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (q >= a.seqs) return;
    const int fresh = a.out[q] < 0 ? 0 : a.counts ? a.counts[q] : a.tokens, length = fresh ? a.lengths[q] : 0;
    const int *row = a.table + (size_t)q * a.table_pages;
    int *slots = a.slots + (size_t)q * a.tokens;
    auto slot = [&](int page, int at) { return (unsigned)page < (unsigned)a.pages ? page << a.shift | (at & mask) : -1; };
    if (!(a.tokens & 3) && !(reinterpret_cast<uintptr_t>(a.slots) & 15)) {
#pragma unroll
        for (int i = from + 4 * lane; i < to; i += 128) {
            int4 x = {-1, -1, -1, -1};
            if (i < fresh) {
                const int at = length + i, last = length + min(i + 3, fresh - 1);  // (on two pages at most)
                const int first_page = at >> a.shift, p0 = row[first_page], p1 = row[last >> a.shift];
                auto one = [&](int k) { return at + k > last ? -1 : slot((at + k) >> a.shift == first_page ? p0 : p1, at + k); };
                x = make_int4(one(0), one(1), one(2), one(3));
            }
            *reinterpret_cast<int4 *>(slots + i) = x;
        }
    } else {
#pragma unroll 4
        for (int i = from + lane; i < to; i += 32) slots[i] = i < fresh ? slot(row[(length + i) >> a.shift], length + i) : -1;
    }
}

template <typename... T>
bool unaligned(const T *...p) { return ((reinterpret_cast<uintptr_t>(p) | ...) & 3) != 0; }

// n values at p.
struct Span {
    const int *p;
    size_t n;
    bool meets(const Span &o) const { return p && o.p && p < o.p + o.n && o.p < p + n; }
};
// What a call writes besides the pool's arrays must not be one of these or of the inputs, not even in part: sequences' results are
// written while others' inputs are read.
bool meets_pool(const Span &x, const qg_page_pool *p, int seqs) {
    return x.meets({p->page_table, (size_t)seqs * p->table_pages}) || x.meets({p->held, (size_t)seqs}) || x.meets({p->free_pages, (size_t)p->pages}) ||
           x.meets({p->free_count, 1});
}

int pages_args(const qg_page_pool *p, int *out, const int *lengths, int seqs, PagesArgs &a) {
    if (!p || !p->page_table || !p->held || !p->free_pages || !p->free_count || !out || !lengths || seqs < 1 || seqs > kMaxSeqs ||
        p->pages < 1 || p->table_pages < 1 || unaligned(p->page_table, p->held, p->free_pages, p->free_count, out, lengths))
        return cudaErrorInvalidValue;
    a.shift = page_shift(p->page_tokens);
    if (a.shift < 0 || pool_too_large(p->pages, p->table_pages, a.shift)) return cudaErrorInvalidValue;
    const Span results = {out, (size_t)seqs};
    if (results.meets({lengths, (size_t)seqs}) || meets_pool(results, p, seqs)) return cudaErrorInvalidValue;
    a.table = p->page_table;
    a.held = p->held;
    a.stack = p->free_pages;
    a.height = p->free_count;
    a.pages = p->pages;
    a.table_pages = p->table_pages;
    a.slots = nullptr;
    a.out = out;
    a.lengths = lengths;
    a.counts = nullptr;
    a.seqs = seqs;
    a.tokens = a.shared = 0;
    return 0;
}

// `entries`: what there may be to write. A cluster's barrier and its CTAs' launch cost as much as one CTA's writes of some
// thousands of them (both calls, one CTA and eight: 64 sequences of 17 slots 10.2 and 11.3 us, 300 of 17 12.9 and 8.6).
int launch(void (*kernel)(PagesArgs), const PagesArgs &a, long long entries) {
    const int ranks = entries > kOneCta ? kPagesCluster : 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ranks);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = launch_stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ranks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace

extern "C" int qg_pages_reserve(const qg_page_pool *pool, int *slots, int *taken, const int *lengths, const int *counts, int seqs,
                                int tokens) {
    PagesArgs a;
    if (int rc = pages_args(pool, taken, lengths, seqs, a)) return rc;
    if (tokens < 1 || tokens > 1 << 30 || (long long)seqs * tokens > 0x7fffffffll || unaligned(slots, counts)) return cudaErrorInvalidValue;
    const Span results = {taken, (size_t)seqs}, places = {slots, (size_t)seqs * tokens}, asked = {counts, (size_t)seqs};
    if (results.meets(asked) || places.meets(asked) || places.meets(results) || places.meets({lengths, (size_t)seqs}) || meets_pool(places, pool, seqs))
        return cudaErrorInvalidValue;
    const bool wide = slots && (long long)seqs * tokens > kWide;
    a.slots = wide ? nullptr : slots;
    a.counts = counts;
    a.tokens = tokens;
    if (int rc = launch(reserve_kernel, a, slots && !wide ? (long long)seqs * tokens : (long long)seqs * 16)) return rc;
    if (!wide) return cudaSuccess;
    a.slots = slots;
    const long long warps = (long long)seqs * ((tokens + kChunk - 1) / kChunk);
    return launch_chained(slots_kernel, dim3((unsigned)((warps + 7) / 8)), 256, a);
}

extern "C" int qg_pages_release(const qg_page_pool *pool, int *freed, const int *lengths, int shared_pages, int seqs) {
    PagesArgs a;
    if (int rc = pages_args(pool, freed, lengths, seqs, a)) return rc;
    if (shared_pages < 0 || shared_pages > a.table_pages) return cudaErrorInvalidValue;
    a.shared = shared_pages;
    return launch(release_kernel, a, (long long)seqs * 16);
}

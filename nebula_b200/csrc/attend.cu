// Attention of drafted tokens (a tree) over the paged cache, on tcgen05.
//
// For one sequence and key/value head, the queries of all nodes and of the
// group's heads are the rows of one matrix product: rows (node, head of the
// group), 128 to a tile. A CTA streams 64 keys at a time:
//     S = Q K^T          tcgen05, Q and K in shared memory, S in tensor memory
//     P = 2^(c S - m)    one thread per row, m the row's running maximum
//     O = P V            tcgen05, P in tensor memory, V in shared memory
//     acc = acc * 2^(m_old - m) + O     in registers
// and out = acc / sum(P). F32 results need more than one F16 product: Q is
// scaled by a power of two per row and split into F16 hi + lo (22 bits), P
// likewise, and both planes go into the same accumulator; K and V are F16 as
// they are. O starts anew with every 64 keys and is added up in registers,
// because an accumulation on the tensor cores does not round to nearest: one
// accumulator over thousands of keys would drift towards zero.
//
// Work is cut into units of 64 keys of one (sequence, head, row tile), and the
// CTAs take equal contiguous ranges of them, so one long sequence fills the
// GPU as well as many short ones. A range that covers an item only in part
// leaves its unnormalised sum, maximum and total in the workspace; a second
// kernel joins the parts in order.
//
// What a row must not see: scores are replaced before the maximum, and the
// value rows of the nodes' tiles are cleaned in shared memory (P = 0 would not
// keep a NaN or infinity out of a product); nodes whose values are not finite
// are added by hand to the rows that see them.
#include <cuda.h>
#include <cstring>
#include "cache.cuh"
#include "moe_tc.cuh"

using namespace nb;

namespace {

constexpr int kRows = 128;       // rows per tile (MMA M)
constexpr int kKeys = 64;        // keys per unit
constexpr int kMaxCtas = 148;    // SMs of a B200: one CTA each
constexpr int kThreads = 512;
// Registers per thread after the split; the four warpgroups' sum is what the
// CTA was launched with (4 * 128).
constexpr int kRegsControl = 48, kRegsSoftmax = 112, kRegsAcc = 176;
static_assert(kRegsControl + kRegsSoftmax + 2 * kRegsAcc <= 4 * (65536 / kThreads), "register split");
constexpr float kPScale = 32768.0f;  // P as F16: 2^15 at the maximum, so that small weights keep their bits

struct AttendArgs {
    CacheView c;
    float *out;
    const float *q;
    const uint64_t *tree;
    float scale;  // |scale| * log2(e)
    float sign;   // of scale, folded into Q
    int seqs, tokens, q_heads, group, row_tiles, part_rows;
    int box;      // rows of one TMA box: a page, at most kKeys
    int *err;
    float *part_acc;   // [2 * kMaxCtas][part_rows][D]
    float2 *part_ml;   // [2 * kMaxCtas][part_rows]
};

template <int D>
struct Cfg {
    static constexpr int kChunks = D / 64;                  // 128-byte wide column blocks
    static constexpr int kPlane = kChunks * kRows * 128;    // one plane of Q
    static constexpr int kStage = kChunks * kKeys * 128;    // 64 keys or values
    static constexpr int kStages = D == 256 ? 3 : 8;
    static constexpr int kSmem = 2 * kPlane + kStages * kStage + 2048 + 1024;
    // tensor memory columns: O, two S, two P (hi and lo, two values a column)
    static constexpr int kS = 256, kP = 384;
};

struct Shared {
    float val[2][kRows];    // rescaling factors, and at an item's end the totals: softmax -> accumulators
    float q_scale[kRows];
    uint64_t full[8], empty[8], s_full[2], s_empty[2], p_full[2], p_empty[2], v_full[2], v_empty[2], o_full, o_empty, q_full, drain;
    uint64_t odd_nodes;     // nodes whose values are not finite: softmax warps only
    uint64_t odd_msg[2];    // the same, posted with an item's totals
    long long unit0, unit1, base;
    int seq0;
    uint32_t tmem;
    int abort;
};
static_assert(sizeof(Shared) <= 2048, "shared bookkeeping");

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Every wait is bounded: 2^17 attempts of at most 20 us (about 2.6 s), then the
// CTA stops and the workspace's error word makes every row NaN.
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, volatile int *abort, int *err) {
    if (mbar_try_wait(bar, parity)) return true;
    for (int i = 0; i < (1 << 17); i++) {
        if (mbar_try_wait_sleep(bar, parity, kWaitHintNs)) return true;
        if (*abort) return false;
    }
    *abort = 1;
    atomicOr(err, 4);
    return false;
}
// The same by a whole warp, with one answer for all its lanes.
__device__ __forceinline__ bool wait_warp(uint64_t *bar, uint32_t parity, volatile int *abort, int *err) {
    return __all_sync(0xffffffffu, wait(bar, parity, abort, err));
}
// For what is already in flight: not cut short by the stop flag.
__device__ __forceinline__ void wait_drain(uint64_t *bar, uint32_t parity) {
    for (int i = 0; i < (1 << 17); i++)
        if (mbar_try_wait_sleep(bar, parity, kWaitHintNs)) return;
}
__device__ __forceinline__ void tma_2d(void *dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
            "r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}
// Shared-memory operand with 128-byte swizzle. K-major (Q, K: rows of 64
// values): groups of 8 rows 1024 bytes apart. MN-major (V as it lies, rows are
// keys): groups of 8 keys 1024 bytes apart, blocks of 64 columns `lead` apart.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)((lead >> 4) & 0x3FFF) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// F16 operands, F32 accumulator; bit 16: B is MN-major.
constexpr uint32_t idesc(int n, bool b_mn) {
    return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(id), "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
        "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]),
          "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]),
          "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]),
          "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void group_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ bool group_any(int id, int n, bool x) {
    int r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.or.pred q, %2, %3, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"((int)x), "r"(id), "r"(n) : "memory");
    return r != 0;
}

// ---- the division of the work ---------------------------------------------

// Units of one (sequence, head, row tile); 0: the sequence is refused.
__device__ __forceinline__ int units_of(const AttendArgs &a, int seq) {
    const int n = a.c.committed(seq, a.tokens);
    return n < 0 ? 0 : (n + a.tokens + kKeys - 1) / kKeys;
}
// One warp: units of all sequences, of those before `seq`, or (find) the
// sequence that holds unit `at` and the units before it.
__device__ long long sum_units(const AttendArgs &a, int seqs, int per) {
    const int lane = threadIdx.x & 31;
    long long sum = 0;
    for (int s = lane; s < seqs; s += 32) sum += (long long)units_of(a, s) * per;
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    return sum;
}
__device__ int find_unit(const AttendArgs &a, int per, long long at, long long &base) {
    const int lane = threadIdx.x & 31;
    base = 0;
    for (int s0 = 0; s0 < a.seqs; s0 += 32) {
        const int s = s0 + lane;
        const long long mine = s < a.seqs ? (long long)units_of(a, s) * per : 0;
        long long upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += x;
        }
        const unsigned past = __ballot_sync(0xffffffffu, base + upto > at);
        if (past) {
            const int l = __ffs(past) - 1;
            base += __shfl_sync(0xffffffffu, upto - mine, l);
            return s0 + l;
        }
        base += __shfl_sync(0xffffffffu, upto, 31);
    }
    return a.seqs;
}
// CTA c of g takes units [c*w/g, (c+1)*w/g).
__device__ __forceinline__ long long range_start(long long c, long long w, int g) { return c * w / g; }
__device__ __forceinline__ int cta_of(long long unit, long long w, int g) { return (int)(((unit + 1) * g + w - 1) / w) - 1; }

// One CTA's part of one item.
struct Item {
    int seq, kv, tile, first, count, units, length;
    long long start;  // the item's first unit
};
struct Walk {
    long long at, end, base;
    int seq;
    __device__ Walk(const Shared &s) : at(s.unit0), end(s.unit1), base(s.base), seq(s.seq0) {}
    __device__ bool next(const AttendArgs &a, Item &it) {
        if (at >= end) return false;
        const int per = a.c.kv_heads * a.row_tiles;
        for (;;) {
            it.units = units_of(a, seq);
            if (at < base + (long long)it.units * per) break;
            base += (long long)it.units * per;
            seq++;
        }
        const long long in = at - base;
        const int index = (int)(in / it.units);
        it.seq = seq;
        it.kv = index / a.row_tiles;
        it.tile = index % a.row_tiles;
        it.first = (int)(in - (long long)index * it.units);
        it.count = (int)min((long long)(it.units - it.first), end - at);
        it.length = a.c.lengths[seq];
        it.start = at - it.first;
        at += it.count;
        return true;
    }
};

// The ring's order within an item of n units: K0, K1, V0, K2, V1, ..., V(n-1).
__device__ __forceinline__ uint32_t k_index(int j) { return j ? 2 * j - 1 : 0; }
__device__ __forceinline__ uint32_t v_index(int j, int n) { return j == n - 1 ? 2 * n - 1 : 2 * j + 2; }

template <int D>
__global__ void __launch_bounds__(kThreads, 1) tree_attention_kernel(const __grid_constant__ AttendArgs a,
                                                                     const __grid_constant__ CUtensorMap k_map,
                                                                     const __grid_constant__ CUtensorMap v_map) {
    using C = Cfg<D>;
    extern __shared__ unsigned char raw[];
    unsigned char *smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    unsigned char *q_smem = smem, *ring = smem + 2 * C::kPlane;
    Shared &s = *reinterpret_cast<Shared *>(ring + C::kStages * C::kStage);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    volatile int *abort = &s.abort;

    if (warp == 0) {
        const int per = a.c.kv_heads * a.row_tiles;
        const long long w = sum_units(a, a.seqs, per);
        const int g = (int)min((long long)gridDim.x, w);
        long long base = 0, u0 = 0, u1 = 0;
        int seq = 0;
        if ((int)blockIdx.x < g) {
            u0 = range_start(blockIdx.x, w, g);
            u1 = range_start(blockIdx.x + 1, w, g);
            seq = find_unit(a, per, u0, base);
        }
        if (lane == 0) {
            s.unit0 = u0, s.unit1 = u1, s.base = base, s.seq0 = seq;
            s.abort = 0;
            s.odd_nodes = 0;
            for (int i = 0; i < C::kStages; i++) mbar_init(&s.full[i], 1), mbar_init(&s.empty[i], 1);
            for (int i = 0; i < 2; i++) {
                mbar_init(&s.s_full[i], 1), mbar_init(&s.s_empty[i], 4);
                mbar_init(&s.p_full[i], 4), mbar_init(&s.p_empty[i], 1);
                mbar_init(&s.v_full[i], 4), mbar_init(&s.v_empty[i], 8);
            }
            mbar_init(&s.o_full, 1), mbar_init(&s.o_empty, 8), mbar_init(&s.q_full, 8), mbar_init(&s.drain, 2);
            fence_mbar_init();
        }
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s.tmem)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = s.tmem;
    Walk walk(s);
    Item it;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
        if (warp == 0 && lane == 0) {
            // ------------------------------------------------ producer: pages to the ring
            uint32_t idx = 0;
            bool ok = true;
            const int page = a.c.page_tokens();
            while (ok && walk.next(a, it)) {
                const int n = it.length + a.tokens;
                const int *table = a.c.table + (size_t)it.seq * a.c.table_pages;
                for (int i = 0; ok && i < 2 * it.count; i++, idx++) {
                    // i-th of K0, K1, V0, K2, V1, ...
                    const bool is_k = i == 0 || (i & 1 && i != 2 * it.count - 1);
                    const int j = is_k ? (i + 1) / 2 : (i == 2 * it.count - 1 ? it.count - 1 : i / 2 - 1);
                    const int st = idx % C::kStages;
                    if (idx >= C::kStages) ok = wait(&s.empty[st], (idx / C::kStages - 1) & 1, abort, a.err);
                    if (!ok) break;
                    const int pos = (it.first + j) * kKeys;
                    const int boxes = (min(kKeys, n - pos) + a.box - 1) / a.box;  // none past the last position
                    mbar_arrive_expect_tx(&s.full[st], boxes * a.box * 128 * C::kChunks);
                    for (int b = 0; b < boxes; b++) {
                        const int p = pos + b * a.box;
                        int id = table[p >> a.c.shift];
                        if ((unsigned)id >= (unsigned)a.c.pages) id = 0;  // the accumulators make the row NaN
                        const int y = (id << a.c.shift) + (p & (page - 1));
                        for (int c = 0; c < C::kChunks; c++)
                            tma_2d(ring + st * C::kStage + c * kKeys * 128 + b * a.box * 128, is_k ? &k_map : &v_map,
                                   it.kv * D + c * 64, y, &s.full[st]);
                    }
                }
            }
            if (!ok)  // the copies in flight land before the CTA ends
                for (uint32_t i = idx > C::kStages ? idx - C::kStages : 0; i < idx; i++)
                    wait_drain(&s.full[i % C::kStages], (i / C::kStages) & 1);
        } else if (warp == 1 && lane == 0) {
            // ------------------------------------------------ S = Q K^T
            uint32_t ring0 = 0, tile = 0, item = 0;
            bool ok = true;
            while (ok && walk.next(a, it)) {
                ok = wait(&s.q_full, item & 1, abort, a.err);
                for (int j = 0; ok && j < it.count; j++, tile++) {
                    const uint32_t idx = ring0 + k_index(j), st = idx % C::kStages, buf = tile & 1;
                    ok = wait(&s.full[st], (idx / C::kStages) & 1, abort, a.err) &&
                         (tile < 2 || wait(&s.s_empty[buf], (tile / 2 - 1) & 1, abort, a.err));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t d = tmem + C::kS + buf * kKeys;
                    const uint32_t kb = smem_u32(ring + st * C::kStage), qb = smem_u32(q_smem);
#pragma unroll
                    for (int p = 0; p < 2; p++)
#pragma unroll
                        for (int c = 0; c < C::kChunks; c++)
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                mma_ss(d, operand(qb + (1 - p) * C::kPlane + c * kRows * 128 + k * 32, 16),
                                       operand(kb + c * kKeys * 128 + k * 32, 16), idesc(kKeys, false), p + c + k > 0);
                    commit(&s.empty[st]);
                    commit(&s.s_full[buf]);
                }
                ring0 += 2 * it.count;
                item++;
            }
            commit(&s.drain);
            wait_drain(&s.drain, 0);
        } else if (warp == 2 && lane == 0) {
            // ------------------------------------------------ O = P V
            uint32_t ring0 = 0, tile = 0;
            bool ok = true;
            while (ok && walk.next(a, it)) {
                for (int j = 0; ok && j < it.count; j++, tile++) {
                    const uint32_t idx = ring0 + v_index(j, it.count), st = idx % C::kStages, buf = tile & 1;
                    ok = wait(&s.full[st], (idx / C::kStages) & 1, abort, a.err) &&
                         (tile < 1 || wait(&s.o_empty, (tile - 1) & 1, abort, a.err)) &&
                         wait(&s.p_full[buf], (tile / 2) & 1, abort, a.err);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t p0 = tmem + C::kP + buf * kKeys, vb = smem_u32(ring + st * C::kStage);
#pragma unroll
                    for (int p = 0; p < 2; p++)
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            mma_ts(tmem, p0 + (1 - p) * (kKeys / 2) + k * 8, operand(vb + k * 2048, kKeys * 128), idesc(D, true),
                                   p + k > 0);
                    commit(&s.empty[st]);
                    commit(&s.p_empty[buf]);
                    commit(&s.o_full);
                }
                ring0 += 2 * it.count;
            }
            commit(&s.drain);
            wait_drain(&s.drain, 0);
        }
    } else if (warp < 8) {
        // ---------------------------------------------------- softmax: one thread per row
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        const int row = tid - 128;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // tensor memory lane of the warp's first row, in bits 16+
        uint32_t ring0 = 0, tile = 0, item = 0, msg = 0;
        bool ok = true;
        while (ok && walk.next(a, it)) {
            ok = wait_warp(&s.q_full, item & 1, abort, a.err);
            const float c = s.q_scale[row];
            const int r = it.tile * kRows + row, node = r / a.group;
            uint64_t mask = 0;
            if (node < a.tokens) {
                mask = a.tree ? a.tree[(size_t)it.seq * a.tokens + node] : ~0ull >> (63 - node);
                if (a.tokens < 64) mask &= (1ull << a.tokens) - 1;
            }
            float m = -INFINITY, l = 0.0f, l_low = 0.0f;
            for (int j = 0; ok && j < it.count; j++, tile++) {
                const uint32_t buf = tile & 1;
                ok = wait_warp(&s.s_full[buf], (tile / 2) & 1, abort, a.err);
                if (!ok) break;
                tc_fence_after();
                float x[2][32];
                tmem_ld32(tmem + lanes + C::kS + buf * kKeys, x[0]);
                tmem_ld32(tmem + lanes + C::kS + buf * kKeys + 32, x[1]);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive(&s.s_empty[buf]);
                const int pos = (it.first + j) * kKeys, past = it.length - pos;  // keys of this unit before the nodes
                const bool tail = past < kKeys;
                if (tail) {
                    const uint64_t seen = (past > 0 ? (1ull << past) - 1 : 0) |
                                          (past > 0 ? mask << past : past > -64 ? mask >> -past : 0);
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t bits = (uint32_t)(seen >> (32 * h));
#pragma unroll
                        for (int i = 0; i < 32; i++) x[h][i] = bits >> i & 1 ? x[h][i] : -INFINITY;
                    }
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 32; i++) {
                    top[i & 1] = fmaxf(top[i & 1], x[0][i]);
                    top[2 + (i & 1)] = fmaxf(top[2 + (i & 1)], x[1][i]);
                }
                const float m_new = fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * c);
                const float keep = m == -INFINITY ? 0.0f : ex2(m - m_new);
                const float off = m_new == -INFINITY ? 0.0f : m_new;
                m = m_new;
                // the factor goes to the accumulators
                const uint32_t slot = msg & 1;
                if (msg >= 2) ok = wait_warp(&s.v_empty[slot], (msg / 2 - 1) & 1, abort, a.err);
                if (!ok) break;
                s.val[slot][row] = keep;
                __syncwarp();
                if (lane == 0) arrive(&s.v_full[slot]);
                msg++;
                if (tile >= 2) ok = wait_warp(&s.p_empty[buf], (tile / 2 - 1) & 1, abort, a.err);
                if (!ok) break;
                tc_fence_after();
                const uint32_t p_cols = tmem + lanes + C::kP + buf * kKeys;
                float2 sum[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
                const float2 c2 = {c, c}, off2 = {-off, -off}, up2 = {kPScale, kPScale};
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float2 t = __ffma2_rn({x[h][2 * i], x[h][2 * i + 1]}, c2, off2);
                        const float2 p = __fmul2_rn({ex2(t.x), ex2(t.y)}, up2);
                        sum[i & 1] = __fadd2_rn(sum[i & 1], p);
                        hi[i] = pack_half(p.x, p.y);
                        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi[i]));
                        lo[i] = pack_half(p.x - f.x, p.y - f.y);
                    }
                    tmem_st16(p_cols + 16 * h, hi);
                    tmem_st16(p_cols + kKeys / 2 + 16 * h, lo);
                }
                // the running total, with what its rounding lost
                const float add = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                l *= keep;
                const float y = add - l_low * keep, next = l + y;
                l_low = (next - l) - y;
                l = next;
                if (tail) {
                    // Values past the last position become 0; those of nodes 0 where they are not finite.
                    const uint32_t idx = ring0 + v_index(j, it.count), st = idx % C::kStages;
                    ok = wait_warp(&s.full[st], (idx / C::kStages) & 1, abort, a.err);
                    if (!ok) break;
                    const int end = past + a.tokens;  // first row of the unit that holds no value
                    uint64_t odd = 0;
                    for (int u = row; u < kKeys * C::kChunks * 8; u += 128) {
                        const int key = (u >> 3) & (kKeys - 1);
                        if (key < past) continue;
                        uint4 *p = reinterpret_cast<uint4 *>(ring + st * C::kStage) + u;
                        uint4 v = key < end ? *p : make_uint4(0, 0, 0, 0);
                        uint32_t *wd = &v.x;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            if ((wd[e] & 0x7c00u) == 0x7c00u) wd[e] &= 0xffff0000u, odd |= 1ull << (key - past);
                            if ((wd[e] & 0x7c000000u) == 0x7c000000u) wd[e] &= 0x0000ffffu, odd |= 1ull << (key - past);
                        }
                        *p = v;
                    }
                    if (odd) atomicOr(reinterpret_cast<unsigned long long *>(&s.odd_nodes), (unsigned long long)odd);
                    fence_proxy_async();
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive(&s.p_full[buf]);
            }
            // the item's totals
            const uint32_t slot = msg & 1;
            if (ok && msg >= 2) ok = wait_warp(&s.v_empty[slot], (msg / 2 - 1) & 1, abort, a.err);
            ok = !group_any(1, 128, !ok);  // the four warps stop together; odd_nodes is complete
            if (!ok) break;
            s.val[slot][row] = l;
            if (row == 0) {
                s.odd_msg[slot] = s.odd_nodes;
                s.odd_nodes = 0;
            }
            if (it.count != it.units && row < a.part_rows)
                a.part_ml[(size_t)(2 * blockIdx.x + (it.start > s.unit0)) * a.part_rows + row] = make_float2(m, l);
            __syncwarp();
            if (lane == 0) arrive(&s.v_full[slot]);
            msg++;
            ring0 += 2 * it.count;
            item++;
            group_sync(2, 128);  // odd_nodes is empty again
        }
    } else {
        // ---------------------------------------------------- Q, and the accumulators: rows x half of the columns
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsAcc));
        constexpr int H = D / 2, V = D / 32;
        const int w = warp - 8, row = (warp & 3) * 32 + lane, col0 = (w >> 2) * H;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;
        uint32_t tile = 0, msg = 0;
        bool ok = true;
        while (ok && walk.next(a, it)) {
            // ---- Q of this item: warp w prepares rows 16w .. 16w+15, lane l values V*l .. V*l+V-1
            bool bad = false;
            {
                float x[16][V];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int r = it.tile * kRows + w * 16 + i, node = r / a.group;
                    const float *src = a.q + (((size_t)it.seq * a.tokens + node) * a.q_heads + it.kv * a.group + r % a.group) * D + lane * V;
#pragma unroll
                    for (int e = 0; e < V; e += 2) {
                        const float2 f = node < a.tokens ? *reinterpret_cast<const float2 *>(src + e) : make_float2(0.0f, 0.0f);
                        x[i][e] = f.x, x[i][e + 1] = f.y;
                    }
                }
                // pages of the item, checked meanwhile
                const int last = min((it.first + it.count) * kKeys, it.length + a.tokens) - 1;
                for (int p = ((it.first * kKeys) >> a.c.shift) + (tid - 256); p <= last >> a.c.shift; p += 256)
                    bad |= (unsigned)a.c.table[(size_t)it.seq * a.c.table_pages + p] >= (unsigned)a.c.pages;
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int r = w * 16 + i;
                    float mx = 0.0f;
#pragma unroll
                    for (int e = 0; e < V; e++) mx = fmaxf(mx, fabsf(x[i][e]));
#pragma unroll
                    for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                    float up, inv;
                    pow2_scale(mx, up, inv);
                    if (lane == 0) s.q_scale[r] = fmaxf(a.scale * inv, 1e-44f);  // never 0: -infinity stays what it is
                    up *= a.sign;
                    uint32_t hi[V / 2], lo[V / 2];
#pragma unroll
                    for (int e = 0; e < V / 2; e++) {
                        const float p = x[i][2 * e] * up, q = x[i][2 * e + 1] * up;
                        hi[e] = pack_half(p, q);
                        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi[e]));
                        lo[e] = pack_half(p - f.x, q - f.y);
                    }
                    const int at = lane * V, unit = (at % 64) / 8;
                    unsigned char *dst = q_smem + (at / 64) * kRows * 128 + r * 128 + ((unit ^ (r & 7)) << 4) + (at % 8) * 2;
#pragma unroll
                    for (int e = 0; e < V / 2; e++) {
                        reinterpret_cast<uint32_t *>(dst)[e] = hi[e];
                        reinterpret_cast<uint32_t *>(dst + C::kPlane)[e] = lo[e];
                    }
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) arrive(&s.q_full);
            }
            float2 acc[H / 2];
#pragma unroll
            for (int i = 0; i < H / 2; i++) acc[i] = make_float2(0.0f, 0.0f);
            for (int j = 0; ok && j < it.count; j++, tile++, msg++) {
                const uint32_t slot = msg & 1;
                ok = wait_warp(&s.v_full[slot], (msg / 2) & 1, abort, a.err);
                if (!ok) break;
                const float keep = s.val[slot][row];
                __syncwarp();
                if (lane == 0) arrive(&s.v_empty[slot]);
                ok = wait_warp(&s.o_full, tile & 1, abort, a.err);
                if (!ok) break;
                tc_fence_after();
                const float2 keep2 = {keep, keep};
#pragma unroll
                for (int b = 0; b < H / 32; b++) {
                    float x[32];
                    tmem_ld32(tmem + lanes + col0 + 32 * b, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; i++) acc[16 * b + i] = __ffma2_rn(acc[16 * b + i], keep2, {x[2 * i], x[2 * i + 1]});
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive(&s.o_empty);
            }
            const uint32_t slot = msg & 1;
            if (ok) ok = wait_warp(&s.v_full[slot], (msg / 2) & 1, abort, a.err);
            ok = !group_any(3, 256, !ok);  // the eight warps stop together
            if (!ok) break;
            const float total = s.val[slot][row];
            uint64_t odd = s.odd_msg[slot];
            __syncwarp();
            if (lane == 0) arrive(&s.v_empty[slot]);
            msg++;
            bad = group_any(4, 256, bad);
            const int r = it.tile * kRows + row, node = r / a.group;
            if (node < a.tokens) {
                if (odd) {  // rare: values that are not finite, for the rows that see them
                    odd &= a.tree ? a.tree[(size_t)it.seq * a.tokens + node] : ~0ull >> (63 - node);
                    while (odd) {
                        const int nd = __ffsll((long long)odd) - 1;
                        odd &= odd - 1;
                        const long long at = a.c.row(it.seq, it.length + nd);
                        if (at < 0) continue;
                        const __half *v = a.c.v + ((size_t)at * a.c.kv_heads + it.kv) * D + col0;
    #pragma unroll
                        for (int i = 0; i < H / 2; i++) {
                            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(v + 2 * i));
                            if (!(fabsf(f.x) < INFINITY)) acc[i].x += f.x;
                            if (!(fabsf(f.y) < INFINITY)) acc[i].y += f.y;
                        }
                    }
                }
                const bool whole = it.count == it.units;
                float mul = whole ? (total == 0.0f ? 0.0f : 1.0f / total) : 1.0f;
                if (bad) mul = __int_as_float(0x7fc00000);
                float *dst = whole ? a.out + (((size_t)it.seq * a.tokens + node) * a.q_heads + it.kv * a.group + r % a.group) * D + col0
                                   : a.part_acc + ((size_t)(2 * blockIdx.x + (it.start > s.unit0)) * a.part_rows + row) * D + col0;
    #pragma unroll
                for (int i = 0; i < H / 4; i++)
                    reinterpret_cast<float4 *>(dst)[i] =
                        make_float4(acc[2 * i].x * mul, acc[2 * i].y * mul, acc[2 * i + 1].x * mul, acc[2 * i + 1].y * mul);
            }
        }
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

// Joins the parts of items that several CTAs share, one warp per (row, head);
// refused sequences, and every row after an error, become NaN.
template <int D>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ AttendArgs a, int ctas) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31;
    const int id = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (id >= a.seqs * a.tokens * a.q_heads) return;
    const int h = id % a.q_heads, row = id / a.q_heads, seq = row / a.tokens;
    const int kv = h / a.group, r = (row % a.tokens) * a.group + h % a.group, tile = r / kRows;
    const int per = a.c.kv_heads * a.row_tiles;
    const long long w = sum_units(a, a.seqs, per);
    const int units = units_of(a, seq);
    const long long start = sum_units(a, seq, per) + (long long)(kv * a.row_tiles + tile) * units;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    float *out = a.out + (size_t)id * D + lane * V;
    if (units == 0 || *(volatile int *)a.err) {
        for (int e = 0; e < V; e++) out[e] = __int_as_float(0x7fc00000);
        return;
    }
    const int g = (int)min((long long)ctas, w);
    const int c0 = cta_of(start, w, g), c1 = cta_of(start + units - 1, w, g);
    if (c0 == c1) return;
    float m = -INFINITY, l = 0.0f, acc[V];
    for (int e = 0; e < V; e++) acc[e] = 0.0f;
    for (int c = c0; c <= c1; c++) m = fmaxf(m, __ldcg(&a.part_ml[(size_t)(2 * c + (start > range_start(c, w, g))) * a.part_rows + r % kRows].x));
    for (int c = c0; c <= c1; c++) {
        const size_t at = (size_t)(2 * c + (start > range_start(c, w, g))) * a.part_rows + r % kRows;
        const float2 ml = __ldcg(a.part_ml + at);
        const float f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - m);
        l += f == 0.0f && ml.y == 0.0f ? 0.0f : f * ml.y;
        const float *p = a.part_acc + at * D + lane * V;
#pragma unroll
        for (int e = 0; e < V; e++) acc[e] = fmaf(f, __ldcg(p + e), acc[e]);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    for (int e = 0; e < V; e++) out[e] = acc[e] * inv;
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// One layer's pool as rows of kv_heads*head_dim halves, read 64 values x box rows at a time.
int pool_map(CUtensorMap *m, const CacheView &c, const __half *pool, int box) {
    static EncodeTiled fn = nullptr;
    if (!fn) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return cudaErrorNotSupported;
        fn = reinterpret_cast<EncodeTiled>(p);
    }
    const cuuint64_t inner = (cuuint64_t)c.kv_heads * c.head_dim;
    const cuuint64_t dims[2] = {inner, (cuuint64_t)c.pages << c.shift}, strides[1] = {inner * sizeof(__half)};
    const cuuint32_t boxes[2] = {64, (cuuint32_t)box}, step[2] = {1, 1};
    const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<__half *>(pool), dims, strides, boxes, step,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : cudaErrorInvalidValue;
}

int part_rows(int tokens, int group) { return tokens * group < kRows ? tokens * group : kRows; }

size_t ml_bytes(int rows) { return (size_t)2 * kMaxCtas * rows * sizeof(float2); }

template <int D>
int launch(const AttendArgs &a, const CUtensorMap &k_map, const CUtensorMap &v_map) {
    if (int rc = cudaFuncSetAttribute(tree_attention_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmem)) return rc;
    // no more CTAs than the longest sequences that the table allows could use
    const long long most = (long long)a.seqs * a.c.kv_heads * a.row_tiles * ((((long long)a.c.table_pages << a.c.shift) + kKeys - 1) / kKeys);
    const int ctas = (int)(most < kMaxCtas ? most : kMaxCtas);
    tree_attention_kernel<D><<<ctas, kThreads, Cfg<D>::kSmem, launch_stream>>>(a, k_map, v_map);
    if (int rc = cudaGetLastError()) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((a.seqs * a.tokens * a.q_heads + 7) / 8));
    cfg.blockDim = dim3(256);
    cfg.stream = launch_stream;
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = pdl;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, join_kernel<D>, a, ctas);
}

}  // namespace

extern "C" int qg_attention_workspace_bytes(int seqs, int tokens, int q_heads, int kv_heads, int head_dim, size_t *bytes) {
    if (!bytes || seqs < 1 || seqs > kMaxSeqs || tokens < 1 || tokens > kMaxNodes || kv_heads < 1 || kv_heads > 1024 ||
        q_heads < kv_heads || q_heads > 1024 || q_heads % kv_heads || (head_dim != 64 && head_dim != 128 && head_dim != 256))
        return cudaErrorInvalidValue;
    const int rows = part_rows(tokens, q_heads / kv_heads);
    *bytes = 256 + ml_bytes(rows) + (size_t)2 * kMaxCtas * rows * head_dim * sizeof(float);
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
    a.sign = scale < 0 ? -1.0f : 1.0f;
    a.scale = (scale < 0 ? -scale : scale) * 1.4426950408889634f;
    a.seqs = seqs;
    a.tokens = tokens;
    a.q_heads = q_heads;
    a.group = q_heads / a.c.kv_heads;
    a.row_tiles = (tokens * a.group + kRows - 1) / kRows;
    a.part_rows = part_rows(tokens, a.group);
    a.box = a.c.page_tokens() < kKeys ? a.c.page_tokens() : kKeys;
    a.err = static_cast<int *>(workspace);
    a.part_ml = reinterpret_cast<float2 *>(static_cast<char *>(workspace) + 256);
    a.part_acc = reinterpret_cast<float *>(static_cast<char *>(workspace) + 256 + ml_bytes(a.part_rows));
    CUtensorMap k_map, v_map;
    if (int rc = pool_map(&k_map, a.c, a.c.k, a.box)) return rc;
    if (int rc = pool_map(&v_map, a.c, a.c.v, a.box)) return rc;
    if (a.c.head_dim == 64) return launch<64>(a, k_map, v_map);
    if (a.c.head_dim == 128) return launch<128>(a, k_map, v_map);
    return launch<256>(a, k_map, v_map);
}

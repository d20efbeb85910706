// Attention of drafted tokens (a tree) over the paged cache, on tcgen05.
//
// For one sequence and key/value head, the queries of all nodes and of the
// group's heads are the rows of one matrix product: rows (node, head of the
// group), 128 to a tile. A CTA streams 128 keys at a time:
//     S = Q K^T          tcgen05, Q and K in shared memory, S in tensor memory
//     P = 2^(c S - m)    one thread per row, m the row's running maximum
//     O = P V            tcgen05, P in tensor memory, V in shared memory
//     acc = acc * 2^(m_old - m) + O     in registers
// and out = acc / sum(P). F32 results need more than one F16 product: Q is
// scaled by a power of two per row and split into F16 hi + lo (22 bits), P
// likewise, and both planes go into the same accumulator; K and V are F16 as
// they are. O starts anew with every 128 keys and is added up in registers,
// because an accumulation on the tensor cores does not round to nearest: one
// accumulator over thousands of keys would drift towards zero.
//
// Work is cut into units of 128 keys of one (sequence, head, row tile), and the
// CTAs take equal contiguous ranges of them, so one long sequence fills the
// GPU as well as many short ones. A range that covers an item only in part
// leaves its unnormalised sum, maximum and total in the workspace; a second
// kernel joins the parts in order.
//
// What a row must not see: scores are replaced before the maximum, and the
// value rows of the nodes' tiles are cleaned in shared memory (P = 0 would not
// keep a NaN or infinity out of a product); nodes whose values are not finite
// are added by hand to the rows that see them.
//
// One token whose query heads share a key head by four at most has a kernel
// without tensor cores (token_attention_kernel): its arithmetic hides behind
// HBM, and nothing is handed from one role to another.
//
// Sequences that begin alike (qg_shared_attention): the prefix is one more
// sequence at the head of the line, whose rows are those of all sequences, and
// the join adds its parts to each sequence's own. A key of the prefix is read
// once for 128 or 256 rows, so the tensor cores bound it: with both planes of
// Q and P 4 rows heads keys values FLOP count twice (48 x 5 rows, 32,768 shared,
// heads of 256: 243 us at the rate of one library product, 330 measured, 389
// in a loop under the power cap).
#include <cuda.h>
#include <cstring>
#include "cache.cuh"
#include "moe_tc.cuh"

using namespace nb;

namespace {

constexpr int kRows = 128;       // rows per tile (MMA M)
constexpr int kKeys = 128;       // keys per unit (MMA N of S: with 64 the re-reads of Q bound the shared memory)
constexpr int kMaxCtas = kSms;   // one CTA each
constexpr int kThreads = 512;
constexpr int kNotes = 3 * 1024;  // bytes for the roles' shared bookkeeping
// Registers per thread after the split; the four warpgroups' sum is what the
// CTA was launched with (4 * 128).
constexpr int kRegsControl = 48, kRegsSoftmax = 112, kRegsAcc = 176;
static_assert(kRegsControl + kRegsSoftmax + 2 * kRegsAcc <= 4 * (65536 / kThreads), "register split");
constexpr float kPScale = 32768.0f;  // P as F16: 2^15 at the maximum, so that small weights keep their bits
// c x - m is one instruction whose product is not rounded; m is. Up to this |m| the two differ by 2^-4 at most; far above it
// P at the maximum would be beyond F16, or nothing. There the scores are taken relative to the largest before they are scaled.
constexpr float kFar = 1048576.0f;  // 2^20

struct AttendArgs {
    CacheView c;
    float *out;
    const float *q;
    const uint64_t *tree;
    float scale;  // |scale| * log2(e)
    float sign;   // of scale, folded into Q
    int seqs, tokens, q_heads, group, row_tiles, tile_rows, part_rows, copies;
    int k_box, v_box;  // rows of one TMA box: a page, at most a piece's keys
    int k_blocks;      // column blocks of a box of keys
    int *err;
    float *part_acc;   // [2 * kMaxCtas][part_rows][D]
    float2 *part_ml;   // [2 * kMaxCtas][part_rows]
    // with a shared prefix:
    float tile_scale;    // scale, and what makes up for the tensor cores' sums
    const int *shared;
    int all_tiles;       // row tiles of all sequences' rows together
    float *prefix_acc;   // [row][q_heads][D], [row][q_heads]: of prefix items that one CTA did as a whole
    float2 *prefix_ml;
    float2 *own_ml;      // the same of sequences' items, whose sums are in out
    float *own_part_acc;  // parts of sequences' items: part_acc, or where their line is one of its own
    float2 *own_part_ml;  // [2 * kGroups * kMaxCtas][kFewRows]
    int own_part_rows;
    // for the join: the slots before each sequence's, all of the sequences' line, all of the prefix's (the same line, or one of its
    // own); own_length of each sequence, the common positions, the CTAs (or groups) of both lines
    long long *starts;   // [seqs + 2]
    int *lengths;        // [seqs + 3]
};

constexpr int kChunk = 32;       // keys per step of the softmax

// D: values of a head. MR: rows of Q that are kept. PAIR: two CTAs on neighbouring SMs (a cluster) work on 256 rows with
// MMAs that span both (cta_group::2): each has its 128 rows of Q, S, P and O, and half of the keys' rows and of the
// values' columns, which the tensor cores of both read. The rings hold twice the keys, and L2 delivers each key once for
// 256 rows: heads of 256 need 128 KB for 128 rows of Q, and the 96 KB left are too few for keys and values of one CTA
// (98k keys x 204 rows in a sustained loop, power-capped at 1.59 GHz: 102 us, with two row tiles apart 109.5; at the first
// calls' 1.97 GHz 88 and 95).
template <int D, int MR, bool PAIR>
struct Cfg {
    static constexpr int kChunks = D / 64;                  // 128-byte wide column blocks
    static constexpr int kBlock = MR * 128;                 // one of them, of one plane of Q
    static constexpr int kPlane = kChunks * kBlock;
    // The rings' pieces: kKBlocks column blocks of kKeyRows keys, or kVBlocks column blocks of kVKeys values; kPieces for
    // a unit's keys or values.
    static constexpr int kPiece = 16384, kKeyRows = PAIR ? kKeys / 2 : kKeys, kKBlocks = kPiece / (128 * kKeyRows);
    static constexpr int kVBlocks = PAIR ? kChunks / 2 : kChunks, kVKeys = kPiece / (128 * kVBlocks);
    static constexpr int kPieces = kChunks / kKBlocks;
    static_assert(kPieces * kVKeys == kKeys, "as many pieces of values as of keys");
    // Two places for Q where there is room: the next item's is prepared while this one's is in use.
    static constexpr int kQBufs = 4 * kPlane <= 131072 ? 2 : 1;
    static constexpr int kKStages = (232448 - kNotes - kQBufs * 2 * kPlane) / (2 * kPiece), kVStages = kKStages;
    static constexpr int kSmem = kQBufs * 2 * kPlane + (kKStages + kVStages) * kPiece + kNotes;
    static constexpr int kOBufs = D == 256 ? 1 : 2;
    static constexpr int kS = 256;  // tensor memory columns: O (twice where it fits), then two of S (P takes its place)
    // A warp that issued MMAs stalls at its next wait until they have read their operands, and the tensor cores run dry:
    // so where the rings have room the issuers wait for two pieces at once (16 x 2 tokens, up to 8191 keys of heads of 128:
    // 85.2 -> 83.6 us at full clock, no difference under the power cap; heads of 256 have no room: 98k keys 102 -> 105 us,
    // 4097 keys 23.8 -> 24.4). P comes in kParts
    // parts of a unit.
    static constexpr int kGroup = D == 128 ? 2 : 1, kParts = kPieces / kGroup, kPartKeys = kKeys / kParts;
    static constexpr int kTileRows = PAIR ? 2 * kRows : kRows;
};

// The slots of one CTA (or pair), and where the first of them lies.
struct Plan {
    long long slot0, slot1;
    int seq0, length0, kv0, tile0, pos0;
    int common, source;  // positions that are read once for all sequences, and the sequence whose pages tell where
};

struct Shared : Plan {
    float val[2][kRows];    // rescaling factors, and at an item's end the totals: softmax -> accumulators
    float q_scale[2][kRows];  // at an item's end the maxima
    uint64_t k_full[7], k_empty[7], v_full[7], v_empty[7], s_full[2], p_full[2][4], pv_done[2], msg_full[2], msg_empty[2], o_full[2], o_empty[2], q_full[2], q_all, landed[2], clean[2], drain;
    int pages[2][2][8];     // of the units that the producers are at: keys, values
    uint64_t odd_nodes[2];  // nodes whose values are not finite: of this item, and of the next (a pair's other CTA may be there)
    uint32_t tmem;
    int abort;
};
static_assert(sizeof(Shared) <= kNotes, "shared bookkeeping");

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// At the same place in the pair's leading CTA (its own, without a pair).
template <bool PAIR>
__device__ __forceinline__ void arrive_leader(uint64_t *bar) {
    if constexpr (PAIR)
        asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, 0;\n\t"
                     "mbarrier.arrive.shared::cluster.b64 _, [a];\n\t}" ::"r"(smem_u32(bar)) : "memory");
    else arrive(bar);
}
// In both CTAs of a pair.
template <bool PAIR>
__device__ __forceinline__ void arrive_both(uint64_t *bar) {
    arrive_leader<PAIR>(bar);
    if constexpr (PAIR)
        asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, 1;\n\t"
                     "mbarrier.arrive.shared::cluster.b64 _, [a];\n\t}" ::"r"(smem_u32(bar)) : "memory");
}
// When this thread's MMAs so far are done: an arrival here, or in both CTAs of a pair.
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t *bar) {
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
    else asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void commit_both(uint64_t *bar) {
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                         smem_u32(bar)),
                     "h"((uint16_t)3)
                     : "memory");
    else commit<false>(bar);
}
// All threads of the CTA, or of the pair.
template <bool PAIR>
__device__ __forceinline__ void sync_all() {
    if constexpr (PAIR) {
        asm volatile("barrier.cluster.arrive.release;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    } else {
        __syncthreads();
    }
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
// Box at pool row y, 64-column block z, into this CTA's memory; its bytes count at the leading CTA's barrier.
template <bool PAIR>
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap *map, int y, int z, uint32_t bar) {
    if constexpr (PAIR)  // bit 24 of a shared::cluster address tells the CTAs of a pair apart
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
                "r"(dst),
            "l"(map), "r"(0), "r"(y), "r"(z), "r"(bar & 0xFEFFFFFFu)
            : "memory");
    else asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
            "r"(dst),
        "l"(map), "r"(0), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// Shared-memory operand with 128-byte swizzle. K-major (Q, K: rows of 64
// values): groups of 8 rows 1024 bytes apart. MN-major (V as it lies, rows are
// keys): groups of 8 keys 1024 bytes apart, blocks of 64 columns `lead` apart.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)((lead >> 4) & 0x3FFF) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// F16 operands, F32 accumulator; bit 16: B is MN-major.
template <bool PAIR>
constexpr uint32_t idesc(int n, bool b_mn) {
    return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)((PAIR ? 2 : 1) * kRows >> 4) << 24);
}
template <bool PAIR>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool acc) {
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(id), "r"((uint32_t)acc)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(id), "r"((uint32_t)acc)
            : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, bool acc) {
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
            "r"(a), "l"(b), "r"(id), "r"((uint32_t)acc)
            : "memory");
    else
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

// With a shared prefix (SHARED) the line of work begins with the prefix, as one more sequence (-1) whose rows are those of all
// sequences and whose keys are `common` positions, a whole number of units and pages; the sequences' own items hold what
// comes after. Their lengths below count from there.
__device__ __forceinline__ long long warp_sum(long long x) {
#pragma unroll
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}
// Positions that all sequences share as asked for, 0: none, -1: more than a table has (every sequence is refused).
template <bool SHARED>
__device__ __forceinline__ int asked_shared(const AttendArgs &a) {
    if constexpr (!SHARED) return 0;
    const int n = *a.shared;
    return n > a.c.table_pages << a.c.shift ? -1 : max(n, 0);
}
template <bool SHARED>
__device__ __forceinline__ int committed(const AttendArgs &a, int seq, int shared) {
    const int n = a.c.committed(seq, a.tokens);
    return SHARED && (shared < 0 || n < shared) ? -1 : n;
}
// One warp: the first sequence that is not refused, or -1.
__device__ __forceinline__ int first_live(const AttendArgs &a, int shared) {
    for (int s0 = 0; s0 < a.seqs; s0 += 32) {
        const int s = s0 + (threadIdx.x & 31);
        const unsigned live = __ballot_sync(0xffffffffu, s < a.seqs && committed<true>(a, s, shared) >= 0);
        if (live) return s0 + __ffs(live) - 1;
    }
    return -1;
}
__device__ __forceinline__ int common_of(const AttendArgs &a, int shared, int source) {
    return shared <= 0 || source < 0 ? 0 : shared & ~(max(kKeys, a.c.page_tokens()) - 1);
}
// A sequence's committed positions after the common ones.
template <bool SHARED>
__device__ __forceinline__ int own_length(const AttendArgs &a, int seq, int shared, int common) {
    const int n = committed<SHARED>(a, seq, shared);
    return n < 0 ? -1 : n - common;
}

// Units of one (sequence, head, row tile); 0: the sequence is refused (length -1).
__device__ __forceinline__ int units_of(const AttendArgs &a, int length) {
    return length < 0 ? 0 : (length + a.tokens + kKeys - 1) / kKeys;
}
// What an item costs besides its units, in units: Q, the first unit's latency and the store (about 2 us). The ranges
// divide the sum of both; an item's first kItemCost slots stand for it and hold no unit. (When only units counted: 16 x 2
// tokens, 512 to 8191 keys of heads of 128 92.1 -> 97.3 us, 5 x 5 tokens of heads of 64 18.5 -> 19.5.)
// With a shared prefix a CTA of heads of 256 often goes from one item to another, with one place for Q (in units, 1, 3 and 5:
// 8 x 17 rows, 8,192 shared 92, 70, 68 us; 48 x 5, 32,768 shared 380, 329, 337; 32 single tokens, 4,096 shared 44, 41, 57).
template <int D, bool SHARED>
constexpr int kItemCost = D == 256 ? (SHARED ? 3 : 1) : 2;
template <int D, bool SHARED>
__device__ __forceinline__ int slots_of(const AttendArgs &a, int length) {
    return length < 0 ? 0 : units_of(a, length) + kItemCost<D, SHARED>;
}
// Slots of the prefix, and those of one of its items.
template <int D>
__device__ __forceinline__ int prefix_slots(int common) { return common / kKeys + kItemCost<D, true>; }
template <int D>
__device__ __forceinline__ long long prefix_line(const AttendArgs &a, int common) {
    return common ? (long long)prefix_slots<D>(common) * a.c.kv_heads * a.all_tiles : 0;
}
// One warp: slots of the sequences before `seqs`.
template <int D, bool SHARED>
__device__ long long sum_slots(const AttendArgs &a, int seqs, int per, int shared, int common) {
    long long sum = 0;
    for (int s = threadIdx.x & 31; s < seqs; s += 32) sum += (long long)slots_of<D, SHARED>(a, own_length<SHARED>(a, s, shared, common)) * per;
    return warp_sum(sum);
}
// One warp: the sequence that holds slot `at`, its length and the slots before it. `len`: the lane's own sequence
// among the first 32.
template <int D, bool SHARED>
__device__ int find_slot(const AttendArgs &a, int per, long long at, int len, int shared, int common, long long &base, int &length) {
    const int lane = threadIdx.x & 31;
    base = 0;
    for (int s0 = 0; s0 < a.seqs; s0 += 32) {
        if (s0) len = s0 + lane < a.seqs ? own_length<SHARED>(a, s0 + lane, shared, common) : -1;
        const long long mine = (long long)slots_of<D, SHARED>(a, len) * per;
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
            length = __shfl_sync(0xffffffffu, len, l);
            return s0 + l;
        }
        base += __shfl_sync(0xffffffffu, upto, 31);
    }
    return a.seqs;
}
// Quotients that nearly always fit 32 bits.
__device__ __forceinline__ long long quotient(long long x, long long y) {
    return (x | y) >> 32 ? x / y : (long long)((uint32_t)x / (uint32_t)y);
}
// CTA c of g takes slots [c*w/g, (c+1)*w/g).
__device__ __forceinline__ long long range_start(long long c, long long w, int g) { return quotient(c * w, g); }
__device__ __forceinline__ int cta_of(long long slot, long long w, int g) { return (int)quotient((slot + 1) * g + w - 1, w) - 1; }

// One CTA's part of one item.
struct Item {
    int seq, kv, tile, first, count, units, length;
    long long start;  // the slot of the item's first unit
};
template <int D, bool SHARED>
struct Walk {
    long long at, end;
    int seq, length, kv, tile, pos;  // pos: slot within the item
    const Plan &p;
    __device__ Walk(const Plan &s)
        : at(s.slot0), end(s.slot1), seq(s.seq0), length(s.length0), kv(s.kv0), tile(s.tile0), pos(s.pos0), p(s) {}
    __device__ bool next(const AttendArgs &a, Item &it) {
        const int from = max(pos, kItemCost<D, SHARED>);
        if (at + (from - pos) >= end) return false;
        it.seq = seq, it.kv = kv, it.tile = tile, it.first = from - kItemCost<D, SHARED>, it.length = length;
        it.units = SHARED && seq < 0 ? length / kKeys : units_of(a, length);
        it.start = at - pos + kItemCost<D, SHARED>;
        at += from - pos;
        it.count = (int)min((long long)(it.units - it.first), end - at);
        at += it.count;
        pos = 0;  // the item after it, should there be one
        if (++tile == (SHARED && seq < 0 ? a.all_tiles : a.row_tiles)) {
            tile = 0;
            if (++kv == a.c.kv_heads) {
                kv = 0;
                do
                    if (++seq < a.seqs) length = own_length<SHARED>(a, seq, SHARED ? asked_shared<SHARED>(a) : 0, SHARED ? p.common : 0);
                while (seq < a.seqs && length < 0);
            }
        }
        return true;
    }
};

// One warp: what the join needs to find every row's parts. `line`: slots before the first sequence's.
template <int D>
__device__ void tell_join(const AttendArgs &a, int shared, int common, long long line, long long own_w, long long prefix_w, int own_g, int prefix_g) {
    const int lane = threadIdx.x & 31;
    for (int s0 = 0; s0 < a.seqs; s0 += 32) {
        const int q = s0 + lane, own = q < a.seqs ? own_length<true>(a, q, shared, common) : -1;
        const long long mine = (long long)slots_of<D, true>(a, own) * a.c.kv_heads * a.row_tiles;
        long long upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += x;
        }
        if (q < a.seqs) a.starts[q] = line + upto - mine, a.lengths[q] = own;
        line += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) {
        a.starts[a.seqs] = own_w, a.starts[a.seqs + 1] = prefix_w;
        int *to = a.lengths + a.seqs;
        to[0] = common, to[1] = own_g, to[2] = prefix_g;
    }
}

// One warp: the slots of CTA (or pair) `team`.
template <int D, bool SHARED>
__device__ __forceinline__ void plan(const AttendArgs &a, Plan &s, int team, int teams) {
    const int lane = threadIdx.x & 31;
    const int per = a.c.kv_heads * a.row_tiles;
    const int shared = asked_shared<SHARED>(a), source = SHARED ? first_live(a, shared) : 0, common = SHARED ? common_of(a, shared, source) : 0;
    const int len = lane < a.seqs ? own_length<SHARED>(a, lane, shared, common) : -1;
    const long long line = SHARED ? prefix_line<D>(a, common) : 0;
    long long w = (long long)slots_of<D, SHARED>(a, len) * per, base = 0, u0 = 0, u1 = 0;
    int seq = 0, length = len;
    if (a.seqs > 1) {
        for (int q = lane + 32; q < a.seqs; q += 32) w += (long long)slots_of<D, SHARED>(a, own_length<SHARED>(a, q, shared, common)) * per;
        w = warp_sum(w);
    }
    w += line;
    const int g = (int)min((long long)teams, w);  // (one sequence: right in lane 0)
    if (team < g) {
        u0 = range_start(team, w, g);
        u1 = range_start(team + 1, w, g);
        if (u0 < line) seq = -1, length = common;
        else if (a.seqs > 1) seq = find_slot<D, SHARED>(a, per, u0 - line, len, shared, common, base, length), base += line;
        else base = line;
    }
    if (lane == 0) {
        const int slots = SHARED && seq < 0 ? prefix_slots<D>(common) : max(1, slots_of<D, SHARED>(a, length)), index = (int)quotient(u0 - base, slots);
        const int tiles = SHARED && seq < 0 ? a.all_tiles : a.row_tiles;
        s.slot0 = u0, s.slot1 = u1, s.seq0 = seq, s.length0 = length;
        s.kv0 = index / tiles, s.tile0 = index % tiles;
        s.pos0 = (int)(u0 - base - (long long)index * slots);
        s.common = common, s.source = source;
    }
    if (SHARED && team == 0 && blockIdx.x == 0) tell_join<D>(a, shared, common, line, w, w, g, g);
}

// Of an item: the rows of q that are its own, counted from its first sequence's; where its keys begin; whose pages they are on.
template <bool SHARED>
__device__ __forceinline__ int rows_of(const AttendArgs &a, const Item &it) {
    return (SHARED && it.seq < 0 ? a.seqs * a.tokens : a.tokens) * a.group;
}
template <bool SHARED>
__device__ __forceinline__ int base_of(const Plan &s, const Item &it) { return SHARED && it.seq >= 0 ? s.common : 0; }
template <bool SHARED>
__device__ __forceinline__ int pages_of(const Plan &s, const Item &it) { return SHARED && it.seq < 0 ? s.source : it.seq; }
template <bool SHARED>
__device__ __forceinline__ int nodes_of(const AttendArgs &a, const Item &it) { return SHARED && it.seq < 0 ? 0 : a.tokens; }
// Row r of the item in q and out, in heads.
template <bool SHARED>
__device__ __forceinline__ size_t head_of(const AttendArgs &a, const Item &it, int r) {
    const int node = r / a.group;
    return ((size_t)(SHARED ? max(it.seq, 0) : it.seq) * a.tokens + node) * a.q_heads + it.kv * a.group + (r - node * a.group);
}

// Keys that unit j of an item's part holds.
template <bool SHARED>
__device__ __forceinline__ int keys_of(const AttendArgs &a, const Item &it, int j) {
    return min(kKeys, it.length + nodes_of<SHARED>(a, it) - (it.first + j) * kKeys);
}
// Where key `row` of a piece of values starts: boxes of v_box keys, in each the column blocks one after the other.
template <int NC>
__device__ __forceinline__ uint32_t value_at(const AttendArgs &a, int row) {
    return ((row & ~(a.v_box - 1)) * NC + (row & (a.v_box - 1))) * 128;
}
// Pieces of values of an item's part: a last unit that is not full has fewer.
template <class C, bool SHARED>
__device__ __forceinline__ uint32_t value_pieces(const AttendArgs &a, const Item &it) {
    return (it.count - 1) * C::kPieces + (keys_of<SHARED>(a, it, it.count - 1) + C::kVKeys - 1) / C::kVKeys;
}

// Nodes whose values are not finite, in the notes of both CTAs of a pair: each sees half of the columns. The other CTA may
// still be at the item before (it has given O back, but not yet read and cleared its notes), so notes are kept by the item's
// parity; two items apart they cannot be, for the unit between them takes both CTAs' O. The fence brings the note to the
// other CTA before the values are reported clean.
template <bool PAIR>
__device__ __forceinline__ void mark_odd(uint64_t *notes, uint64_t nodes) {
    if constexpr (!PAIR) {
        atomicOr(reinterpret_cast<unsigned long long *>(notes), (unsigned long long)nodes);
    } else {
#pragma unroll
        for (int r = 0; r < 2; r++)
            asm volatile("{\n\t.reg .b32 a;\n\t.reg .b64 x;\n\tmapa.shared::cluster.u32 a, %0, %2;\n\t"
                         "atom.relaxed.cluster.shared::cluster.or.b64 x, [a], %1;\n\t}" ::"r"(smem_u32(notes)),
                         "l"(nodes), "r"(r)
                         : "memory");
        asm volatile("fence.acq_rel.cluster;" ::: "memory");
    }
}

// PLANNED: the plan is in shared memory already.
template <int D, int MR, bool PAIR, bool SHARED, bool PLANNED>
__device__ __forceinline__ void attend_tiles(const AttendArgs &a, const CUtensorMap &k_map, const CUtensorMap &v_map) {
    using C = Cfg<D, MR, PAIR>;
    static_assert(!PAIR || C::kOBufs == 1, "mark_odd: a unit takes both CTAs' O of the unit before");
    const int copies = D == 256 || SHARED ? 1 : a.copies;
    constexpr int NC = C::kChunks, NK = C::kKStages, NV = C::kVStages, VK = C::kVKeys, QB = C::kQBufs, OB = C::kOBufs, VB = C::kVBlocks, NP = C::kPieces, KB = C::kKBlocks;
    constexpr int kPeers = PAIR ? 2 : 1;  // CTAs that work on one item
    const int team = blockIdx.x / kPeers, rank = blockIdx.x % kPeers, teams = gridDim.x / kPeers;
    extern __shared__ __align__(1024) unsigned char smem[];  // swizzled tiles start on multiples of 1024
    unsigned char *q_smem = smem, *k_ring = smem + QB * 2 * C::kPlane, *v_ring = k_ring + NK * C::kPiece;
    Shared &s = *reinterpret_cast<Shared *>(v_ring + NV * C::kPiece);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    volatile int *abort = &s.abort;

    if (warp == 0) {
        if constexpr (!PLANNED) {
            asm volatile("griddepcontrol.wait;" ::: "memory");
            plan<D, SHARED>(a, s, team, teams);
        }
    } else if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s.tmem)));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s.tmem)));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
    } else if (warp == 2 && lane == 0) {
        s.abort = 0;
        s.odd_nodes[0] = s.odd_nodes[1] = 0;
        for (int i = 0; i < NK; i++) mbar_init(&s.k_full[i], 1), mbar_init(&s.k_empty[i], 1);
        for (int i = 0; i < NV; i++) mbar_init(&s.v_full[i], 1), mbar_init(&s.v_empty[i], 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&s.s_full[i], 1), mbar_init(&s.pv_done[i], 1);
            mbar_init(&s.msg_full[i], 4), mbar_init(&s.msg_empty[i], 8);
            for (int z = 0; z < C::kParts; z++) mbar_init(&s.p_full[i][z], 4 * kPeers);
            mbar_init(&s.o_full[i], 1), mbar_init(&s.o_empty[i], 8 * kPeers), mbar_init(&s.q_full[i], 8);
            mbar_init(&s.landed[i], 1), mbar_init(&s.clean[i], 8 * kPeers);
        }
        mbar_init(&s.q_all, 8 * kPeers);
        mbar_init(&s.drain, 2);
        fence_mbar_init();
    } else if (warp == 3 && lane == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map));
        asm volatile("prefetch.tensormap [%0];" ::"l"(&v_map));
    }
    // Every role goes to its code first and meets the others there: instructions that are not yet in the SM's caches
    // arrive while the plan is made.
    tc_fence_before();
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
        sync_all<PAIR>();
        tc_fence_after();
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        const uint32_t tmem = s.tmem;
        Walk<D, SHARED> walk(s);
        Item it;
        if (warp == 0 || warp == 3) {
            // ------------------------------------------------ producers: pages to the rings, keys (warp 0), values (warp 3)
            // A warp issues its copies one after the other (134 cycles for a 2 KB box, 440 for 8 KB, measured), 15-23
            // bytes per cycle and SM; HBM delivers 25, so it takes two of them.
            // The warp looks a unit's pages up one unit ahead (a lane each); one lane issues the boxes. A box of values has
            // all its column blocks side by side; keys want all rows of a block together.
            const bool is_k = warp == 0;
            const int page = a.c.page_tokens(), per_unit = max(1, kKeys >> a.c.shift);
            const int box = is_k ? a.k_box : a.v_box, piece = is_k ? C::kKeyRows : VK, blocks = is_k ? a.k_blocks : VB, bytes = box * 128 * blocks;
            const uint32_t ring = smem_u32(is_k ? k_ring : v_ring), places = is_k ? NK : NV;
            uint64_t *full = is_k ? s.k_full : s.v_full, *empty = is_k ? s.k_empty : s.v_empty;
            const CUtensorMap *map = is_k ? &k_map : &v_map;
            uint32_t st = 0, round = 0, unit = 0;
            bool ok = true;
            while (ok && walk.next(a, it)) {
                const int base = base_of<SHARED>(s, it), n = base + it.length + nodes_of<SHARED>(a, it);
                const int *table = a.c.table + (size_t)pages_of<SHARED>(s, it) * a.c.table_pages;
                auto look_up = [&](int j) {  // page of keys l*page.. of unit j, for lane l
                    const int p = ((base + (it.first + j) * kKeys) >> a.c.shift) + lane;
                    const int id = lane < per_unit && p <= (n - 1) >> a.c.shift ? table[p] : 0;
                    return (unsigned)id < (unsigned)a.c.pages ? id : 0;  // the accumulators make the row NaN
                };
                int ids = look_up(0);
                for (int j = 0; ok && j < it.count; j++, unit++) {
                    int *pages = s.pages[!is_k][unit & 1];
                    if (lane < 8) pages[lane] = ids;
                    __syncwarp();
                    if (j + 1 < it.count) ids = look_up(j + 1);
                    const int pos = base + (it.first + j) * kKeys, keys = keys_of<SHARED>(a, it, j);
                    const int pieces = is_k ? NP : (keys + VK - 1) / VK;
                    for (int c = 0; c < pieces; c++) {
                        if (round) ok = wait_warp(&empty[st], (round - 1) & 1, abort, a.err);
                        if (!ok) break;
                        if (elect_one()) {
                            const int key0 = is_k ? rank * C::kKeyRows : c * VK;  // the piece's first key within the unit
                            auto boxes_from = [&](int key) { return (min(piece, keys - key) + box - 1) / box; };
                            const int boxes = boxes_from(key0);  // none past the last position
                            const uint32_t bar = smem_u32(&full[st]);
                            const int sweeps = is_k ? KB / blocks : 1;  // over the piece's column blocks
                            if (!PAIR) mbar_arrive_expect_tx(&full[st], sweeps * boxes * bytes);
                            else if (rank == 0)  // what both CTAs will bring
                                mbar_arrive_expect_tx(&full[st], sweeps * (boxes + (is_k ? max(0, boxes_from(C::kKeyRows)) : boxes)) * bytes);
                            for (int sw = 0; sw < sweeps; sw++) {
                                uint32_t dst = ring + st * C::kPiece + sw * C::kKeyRows * 128;
                                int p = pos + key0;
                                for (int b = 0; b < boxes; b++, p += box, dst += bytes)
                                    tma_3d<PAIR>(dst, map, (pages[(p >> a.c.shift) - (pos >> a.c.shift)] << a.c.shift) + (p & (page - 1)),
                                                 it.kv * NC + (is_k ? c * KB + sw * blocks : rank * VB), bar);
                            }
                        }
                        __syncwarp();
                        if (++st == places) st = 0, round++;
                    }
                }
            }
            if (!ok && lane == 0)  // the copies in flight land before the CTA ends
                for (uint32_t i = 0; i < places; i++)
                    if ((i < st || round) && rank == 0) wait_drain(&full[i], (i < st ? round : round - 1) & 1);
            if (!SHARED && !is_k)  // rows of refused sequences (with a shared prefix, the join's)
                for (int q = blockIdx.x; q < a.seqs; q += gridDim.x)
                    if (a.c.committed(q, a.tokens) < 0)
                        for (size_t i = lane; i < (size_t)a.tokens * a.q_heads * D; i += 32)
                            a.out[(size_t)q * a.tokens * a.q_heads * D + i] = __int_as_float(0x7fc00000);
        } else if (warp == 1 && rank == 0 && elect_one()) {
            // ------------------------------------------------ S = Q K^T
            uint32_t st = 0, round = 0, tile = 0, item = 0;
            bool ok = true;
            const uint64_t q_lo = operand(smem_u32(q_smem) + C::kPlane, 16);
            const uint64_t q_hi = operand(smem_u32(q_smem), 16);
            while (ok && walk.next(a, it)) {
                const uint32_t qb = item % QB;
                ok = PAIR ? wait(&s.q_all, item & 1, abort, a.err) : wait(&s.q_full[qb], item / QB & 1, abort, a.err);
                for (int j = 0; ok && j < it.count; j++, tile++) {
                    const uint32_t buf = tile & 1, d = tmem + C::kS + buf * kKeys;
                    if (tile >= 2) ok = wait(&s.pv_done[buf], (tile / 2 - 1) & 1, abort, a.err);
#pragma unroll 1
                    for (int c0 = 0; ok && c0 < NP; c0 += C::kGroup) {
                        uint32_t at = st, turn = round;
#pragma unroll
                        for (int c = 0; c < C::kGroup; c++) {
                            ok = ok && wait(&s.k_full[at], turn & 1, abort, a.err);
                            if (++at == NK) at = 0, turn++;
                        }
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll
                        for (int c = 0; c < C::kGroup; c++) {
#pragma unroll
                            for (int e = 0; e < KB; e++) {
                                const uint64_t kd = operand(smem_u32(k_ring + st * C::kPiece + e * C::kKeyRows * 128), 16);
                                const uint64_t qd = qb * (2 * C::kPlane / 16) + ((c0 + c) * KB + e) * (C::kBlock / 16);
#pragma unroll
                                for (int k = 0; k < 4; k++)
                                    mma_ss<PAIR>(d, q_lo + qd + 2 * k, kd + 2 * k, idesc<PAIR>(kKeys, false), c0 + c + e + k > 0);
#pragma unroll
                                for (int k = 0; k < 4; k++) mma_ss<PAIR>(d, q_hi + qd + 2 * k, kd + 2 * k, idesc<PAIR>(kKeys, false), true);
                            }
                            commit_both<PAIR>(&s.k_empty[st]);
                            if (++st == NK) st = 0, round++;
                        }
                    }
                    if (ok) commit_both<PAIR>(&s.s_full[buf]);
                }
                item++;
            }
            commit<PAIR>(&s.drain);
            wait_drain(&s.drain, 0);
        } else if (warp == 2 && rank == 0 && elect_one()) {
            // ------------------------------------------------ O = P V
            uint32_t st = 0, round = 0, tile = 0, lands = 0, cleans = 0;  // (at most two parts between landed and clean)
            // descriptor steps for 16 and 32 keys within a piece: a box of 16 or 32 keys ends with them
            const uint32_t step16 = value_at<VB>(a, 16) / 16, step32 = value_at<VB>(a, 32) / 16;
            bool ok = true;
            while (ok && walk.next(a, it)) {
                for (int j = 0; ok && j < it.count; j++, tile++) {
                    const uint32_t buf = tile & 1, p0 = tmem + C::kS + buf * kKeys, ob = tile % OB, o = tmem + ob * D;
                    const int keys = keys_of<SHARED>(a, it, j), past = it.length - (it.first + j) * kKeys;
                    if (tile >= OB) ok = wait(&s.o_empty[ob], (tile / OB - 1) & 1, abort, a.err);
                    // the pieces of part z; where it holds nodes, the accumulator warps are told to clean their values
                    uint32_t at = st, turn = round;
                    auto take = [&](int z) {
                        const int n = min(C::kPartKeys, keys - z * C::kPartKeys);
                        for (int c = 0; c * VK < n; c++) {
                            ok = ok && wait(&s.v_full[at], turn & 1, abort, a.err);
                            if (++at == NV) at = 0, turn++;
                        }
                        if (ok && n > 0 && (z + 1) * C::kPartKeys > past) arrive_both<PAIR>(&s.landed[lands++ & 1]);
                    };
                    if (past < kKeys) take(0);
#pragma unroll 1
                    for (int z = 0; ok && z < C::kParts; z++) {
                        // Past the last key there is nothing to multiply, but the softmax writes there too, and must be
                        // done before S takes the place again.
                        const int key0 = z * C::kPartKeys, end = min(key0 + C::kPartKeys, keys);
                        if (past >= kKeys) take(z);
                        else if (z + 1 < C::kParts) take(z + 1);  // a part ahead, so that the cleaning is not waited for
                        if (ok && key0 < end && key0 + C::kPartKeys > past) {
                            ok = wait(&s.clean[cleans & 1], cleans / 2 & 1, abort, a.err);
                            cleans++;
                        }
                        ok = ok && wait(&s.p_full[buf][z], (tile / 2) & 1, abort, a.err);
                        if (!ok) break;
                        tc_fence_after();
                        uint64_t vd = operand(smem_u32(v_ring + st * C::kPiece), a.v_box * 128);
                        uint32_t p = p0 + key0;  // 32 keys: 16 columns of hi, 16 of lo
#pragma unroll 1
                        for (int key = key0; key < end; key += 32) {
                            mma_ts<PAIR>(o, p + 16, vd, idesc<PAIR>(D, true), key > 0);
                            mma_ts<PAIR>(o, p, vd, idesc<PAIR>(D, true), true);
                            if (key + 16 < end) {
                                mma_ts<PAIR>(o, p + 24, vd + step16, idesc<PAIR>(D, true), true);
                                mma_ts<PAIR>(o, p + 8, vd + step16, idesc<PAIR>(D, true), true);
                            }
                            p += 32, vd += step32;
                            if ((key + 32) % VK == 0 || key + 32 >= keys) {
                                commit_both<PAIR>(&s.v_empty[st]);
                                if (++st == NV) st = 0, round++;
                                vd = operand(smem_u32(v_ring + st * C::kPiece), a.v_box * 128);
                            }
                        }
                    }
                    if (!ok) break;
                    commit<PAIR>(&s.pv_done[buf]);
                    commit_both<PAIR>(&s.o_full[ob]);
                }
            }
            commit<PAIR>(&s.drain);
            wait_drain(&s.drain, 0);
        }
    } else if (warp < 8) {
        // ---------------------------------------------------- softmax: one thread per row
        // With few rows (a.copies 2 or 4) Q lies in the tile several times, and each copy takes its share of a unit's
        // keys: a running maximum and total of its own, P = 0 for the others' keys, joined at the end of the item.
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        sync_all<PAIR>();
        tc_fence_after();
        const uint32_t tmem = s.tmem;
        Walk<D, SHARED> walk(s);
        Item it;
        const int row = tid - 128, span = MR / copies, copy = row / span, chunks = kKeys / kChunk / copies;
        const int h0 = copy * chunks, h1 = h0 + chunks;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // tensor memory lane of the warp's first row, in bits 16+
        uint32_t tile = 0, item = 0, msg = 0;
        bool ok = true;
        while (ok && walk.next(a, it)) {
            const int row0 = it.tile * C::kTileRows + rank * kRows, node = (row0 + row % span) / a.group;
            const bool live = row < MR && row0 + (row & ~31) % span < rows_of<SHARED>(a, it);  // the warp has rows
            uint64_t mask = 0;
            if (!(SHARED && it.seq < 0) && node < a.tokens) {
                mask = a.tree ? a.tree[(size_t)it.seq * a.tokens + node] : ~0ull >> (63 - node);
                if (a.tokens < 64) mask &= (1ull << a.tokens) - 1;
            }
            const uint32_t qb = item % QB;
            ok = wait_warp(&s.q_full[qb], item / QB & 1, abort, a.err);
            const float c = s.q_scale[qb][row];
            float most = -INFINITY, m = -INFINITY, l = 0.0f, l_low = 0.0f;  // most: the largest score as it is; m = c * most
            for (int j = 0; ok && j < it.count; j++, tile++) {
                const uint32_t buf = tile & 1, cols = tmem + lanes + C::kS + buf * kKeys;
                const int past = it.length - (it.first + j) * kKeys;  // keys of this unit before the nodes
                const bool tail = past < kKeys;
                const int held = (keys_of<SHARED>(a, it, j) + kChunk - 1) / kChunk;  // chunks that hold keys; the product leaves out the others
                // which of keys 32h .. 32h+31 the row sees, in a unit that holds nodes
                auto seen = [&](int h) -> uint32_t {
                    const int at = past - 32 * h;  // keys of the chunk before the nodes
                    if (at >= 32) return ~0u;
                    const uint32_t before = at > 0 ? (1u << at) - 1 : 0;
                    return before | (uint32_t)(at > 0 ? mask << at : at > -64 ? mask >> -at : 0);
                };
                ok = wait_warp(&s.s_full[buf], (tile / 2) & 1, abort, a.err);
                if (!ok) break;
                tc_fence_after();
                float keep = 0.0f, off = 0.0f;
                if (live) {
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
                    for (int h = h0; h < min(h1, held); h++) {
                        float x[32];
                        tmem_ld32(cols + 32 * h, x);
                        tmem_wait_ld();
                        if (tail) {
                            const uint32_t bits = seen(h);
#pragma unroll
                            for (int i = 0; i < 32; i++) x[i] = bits >> i & 1 ? x[i] : -INFINITY;
                        }
#pragma unroll
                        for (int i = 0; i < 32; i++) top[i & 3] = fmaxf(top[i & 3], x[i]);
                    }
                    const float here = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), m_new = fmaxf(m, here * c);
                    most = fmaxf(most, here);
                    keep = m == -INFINITY ? 0.0f : ex2(m - m_new);
                    off = m_new == -INFINITY ? 0.0f : m_new;
                    m = m_new;
                }
                // the factor goes to the accumulators
                const uint32_t slot = msg & 1;
                if (msg >= 2) ok = wait_warp(&s.msg_empty[slot], (msg / 2 - 1) & 1, abort, a.err);
                if (!ok) break;
                s.val[slot][row] = keep;
                __syncwarp();
                if (lane == 0) arrive(&s.msg_full[slot]);
                msg++;
                if (__builtin_expect(__any_sync(0xffffffffu, fabsf(off) >= kFar), 0)) {  // (in the chunks' way instead: 98k keys 103 -> 105 us)
                    float base = 0.0f;
                    if (fabsf(off) >= kFar) base = most, off = 0.0f;
#pragma unroll 1
                    for (int h = h0; h < min(h1, held); h++) {
                        float x[32];
                        tmem_ld32(cols + 32 * h, x);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; i++) x[i] -= base;
                        tmem_st16(cols + 32 * h, reinterpret_cast<const uint32_t(&)[16]>(x[0]));
                        tmem_st16(cols + 32 * h + 16, reinterpret_cast<const uint32_t(&)[16]>(x[16]));
                    }
                    tmem_wait_st();
                }
                float2 sum[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
                const float2 c2 = {c, c}, off2 = {-off, -off}, up2 = {kPScale, kPScale};
#pragma unroll 1
                for (int h = 0; h < kKeys / kChunk; h++) {
                    // P takes the place of 32 scores: 16 columns of hi, 16 of lo
                    uint32_t hi[16], lo[16];
                    if (h >= held) {
                    } else if (h >= h0 && h < h1) {
                        if (live) {
                            float x[32];
                            tmem_ld32(cols + 32 * h, x);
                            tmem_wait_ld();
                            if (tail) {
                                const uint32_t bits = seen(h);
#pragma unroll
                                for (int i = 0; i < 32; i++) x[i] = bits >> i & 1 ? x[i] : -INFINITY;
                            }
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                const float2 t = __ffma2_rn({x[2 * i], x[2 * i + 1]}, c2, off2);
                                const float2 p = __fmul2_rn({ex2(t.x), ex2(t.y)}, up2);
                                sum[i & 1] = __fadd2_rn(sum[i & 1], p);
                                hi[i] = pack_half(p.x, p.y);
                                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi[i]));
                                const float2 d = __fadd2_rn(p, {-f.x, -f.y});
                                lo[i] = pack_half(d.x, d.y);
                            }
                            tmem_st16(cols + 32 * h, hi);
                            tmem_st16(cols + 32 * h + 16, lo);
                            tmem_wait_st();
                        }
                    } else if (live) {
#pragma unroll
                        for (int i = 0; i < 16; i++) hi[i] = 0;
                        tmem_st16(cols + 32 * h, hi);
                        tmem_st16(cols + 32 * h + 16, hi);
                        tmem_wait_st();
                    }
                    if ((h + 1) * kChunk % C::kPartKeys) continue;
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_leader<PAIR>(&s.p_full[buf][h * kChunk / C::kPartKeys]);
                }
                // the running total, with what its rounding lost
                const float add = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                l *= keep;
                const float y = add - l_low * keep, next = l + y;
                l_low = (next - l) - y;
                l = next;
            }
            // the item's totals
            const uint32_t slot = msg & 1;
            if (ok && msg >= 2) ok = wait_warp(&s.msg_empty[slot], (msg / 2 - 1) & 1, abort, a.err);
            ok = !group_any(1, 128, !ok);  // the four warps stop together
            if (!ok) break;
            s.val[slot][row] = l;
            s.q_scale[qb][row] = m;
            __syncwarp();
            if (lane == 0) arrive(&s.msg_full[slot]);
            msg++;
            item++;
        }
    } else {
        // ---------------------------------------------------- Q, and the accumulators: rows x half of the columns
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsAcc));
        sync_all<PAIR>();
        tc_fence_after();
        const uint32_t tmem = s.tmem;
        Walk<D, SHARED> walk(s);
        Item it;
        constexpr int H = D / 2, V = D / 32;
        const int w = warp - 8, row = (warp & 3) * 32 + lane, col0 = (w >> 2) * H, span = MR / copies;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;
        uint32_t piece0 = 0, tile = 0, msg = 0, cleans = 0, items = 0;
        // Every round prepares Q of one item and works through one: the same, or with two places for Q the one before.
        Item nx;
        size_t where_nx = 0, where = 0;
        bool ok = true, more = walk.next(a, nx), left = false;
        for (uint32_t round = 0; ok && (more || left); round++) {
            if (more) {
                // Warp w prepares, and at the end stores, rows w, w+8, ...; lane i < 16 knows where row w+8i lies in q
                // and out. Rows past the last are left as they are: no one reads their results.
                const int row0 = nx.tile * C::kTileRows + rank * kRows, rows = min(kRows, rows_of<SHARED>(a, nx) - row0);
                {
                    const int r = row0 + w + 8 * (lane & 15);
                    where_nx = r < rows_of<SHARED>(a, nx) ? head_of<SHARED>(a, nx, r) * D : 0;
                }
                const uint32_t qb = round % QB;
                unsigned char *q_to = q_smem + qb * 2 * C::kPlane;
                // lane l holds values V*l .. V*l+V-1 of four rows; the next four are asked for meanwhile
                float next[4][V];
                auto ask = [&](int i0) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float *src = a.q + __shfl_sync(0xffffffffu, where_nx, i0 + i & 15) + lane * V;
                        if constexpr (V == 2) {
                            *reinterpret_cast<float2 *>(next[i]) = __ldg(reinterpret_cast<const float2 *>(src));
                        } else {
#pragma unroll
                            for (int e = 0; e < V; e += 4) *reinterpret_cast<float4 *>(next[i] + e) = __ldg(reinterpret_cast<const float4 *>(src + e));
                        }
                    }
                };
                ask(0);
#pragma unroll 1
                for (int i0 = 0; w + 8 * i0 < rows; i0 += 4) {
                    float x[4][V];
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int e = 0; e < V; e++) x[i][e] = next[i][e];
                    if (w + 8 * (i0 + 4) < rows) ask(i0 + 4);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int r = w + 8 * (i0 + i);
                        if (r >= rows) break;
                        float mx = 0.0f;
#pragma unroll
                        for (int e = 0; e < V; e++) mx = fmaxf(mx, fabsf(x[i][e]));
                        // of values that are not negative the bit patterns have the same order
                        mx = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mx)));
                        float up, inv;
                        pow2_scale(mx, up, inv);
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
                        for (int rr = r; rr < MR; rr += span) {
                            if (lane == 0) s.q_scale[qb][rr] = fmaxf((SHARED ? a.tile_scale : a.scale) * inv, 1e-44f);  // never 0: -infinity stays what it is
                            unsigned char *dst = q_to + (at / 64) * C::kBlock + rr * 128 + ((unit ^ (rr & 7)) << 4) + (at % 8) * 2;
                            if constexpr (V == 8) {
                                *reinterpret_cast<uint4 *>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                                *reinterpret_cast<uint4 *>(dst + C::kPlane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                            } else if constexpr (V == 4) {
                                *reinterpret_cast<uint2 *>(dst) = make_uint2(hi[0], hi[1]);
                                *reinterpret_cast<uint2 *>(dst + C::kPlane) = make_uint2(lo[0], lo[1]);
                            } else {
                                *reinterpret_cast<uint32_t *>(dst) = hi[0];
                                *reinterpret_cast<uint32_t *>(dst + C::kPlane) = lo[0];
                            }
                        }
                    }
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) arrive(&s.q_full[qb]);
                if (PAIR && lane == 0) arrive_leader<PAIR>(&s.q_all);
            }
            if (QB == 2 && !left) {  // the first round only prepares
                it = nx, where = where_nx, left = more;
                more = more && walk.next(a, nx);
                continue;
            }
            if (QB == 1) it = nx, where = where_nx;
            const uint32_t qb = QB == 2 ? (round - 1) % 2 : 0;
            const int row0 = it.tile * C::kTileRows + rank * kRows, rows = min(kRows, rows_of<SHARED>(a, it) - row0);
            const bool live = (row & ~31) % span < rows && row < MR;  // the warp has rows
            unsigned char *stage = q_smem + qb * 2 * C::kPlane;
            // pages of the item, checked
            bool bad = false;
            const int base = base_of<SHARED>(s, it);
            const int last = base + min((it.first + it.count) * kKeys, it.length + nodes_of<SHARED>(a, it)) - 1;
#pragma unroll 1
            for (int p = ((base + it.first * kKeys) >> a.c.shift) + (tid - 256); p <= last >> a.c.shift; p += 256)
                bad |= (unsigned)a.c.table[(size_t)pages_of<SHARED>(s, it) * a.c.table_pages + p] >= (unsigned)a.c.pages;
            float2 acc[H / 2];
#pragma unroll
            for (int i = 0; i < H / 2; i++) acc[i] = make_float2(0.0f, 0.0f);
#pragma unroll 1
            for (int j = 0; ok && j < it.count; j++, tile++, msg++) {
                const uint32_t slot = msg & 1;
                ok = wait_warp(&s.msg_full[slot], (msg / 2) & 1, abort, a.err);
                if (!ok) break;
                const float keep = s.val[slot][row];
                __syncwarp();
                if (lane == 0) arrive(&s.msg_empty[slot]);
                const int past = it.length - (it.first + j) * kKeys;  // keys of the unit before the nodes
                if (past < kKeys) {
                    // Values past the last position become 0 up to a multiple of 32; those of nodes 0 where they are
                    // not finite.
                    const int end = min(kKeys, past + a.tokens);
                    for (int z = max(past, 0) / C::kPartKeys; ok && z * C::kPartKeys < end; z++) {
                        ok = wait_warp(&s.landed[cleans & 1], cleans / 2 & 1, abort, a.err);
                        if (!ok) break;
                        const int key0 = max(past, z * C::kPartKeys) & ~31, key1 = min(end, (z + 1) * C::kPartKeys);
                        uint64_t odd = 0;
                        for (int k0 = key0; k0 < key1; k0 += 32) {
                            unsigned char *v0 = v_ring + (piece0 + j * NP + k0 / VK) % NV * C::kPiece;
#pragma unroll 1
                            for (int u = tid - 256; u < 32 * 8 * VB; u += 256) {
                                const int key = k0 + ((u >> 3) & 31);
                                if (key < past) continue;
                                uint4 *p = reinterpret_cast<uint4 *>(v0 + value_at<VB>(a, key % VK) + (u >> 8) * a.v_box * 128 + (u & 7) * 16);
                                uint4 v = key < end ? *p : make_uint4(0, 0, 0, 0);
                                uint32_t *wd = &v.x;
#pragma unroll
                                for (int e = 0; e < 4; e++) {
                                    if ((wd[e] & 0x7c00u) == 0x7c00u) wd[e] &= 0xffff0000u, odd |= 1ull << (key - past);
                                    if ((wd[e] & 0x7c000000u) == 0x7c000000u) wd[e] &= 0x0000ffffu, odd |= 1ull << (key - past);
                                }
                                *p = v;
                            }
                        }
                        if (odd) mark_odd<PAIR>(&s.odd_nodes[PAIR ? items & 1 : 0], odd);
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) arrive_leader<PAIR>(&s.clean[cleans & 1]);
                        cleans++;
                    }
                    if (!ok) break;
                }
                const uint32_t ob = tile % OB;
                ok = wait_warp(&s.o_full[ob], tile / OB & 1, abort, a.err);
                if (!ok) break;
                if (live) {
                    tc_fence_after();
                    const float2 keep2 = {keep, keep};
#pragma unroll
                    for (int b = 0; b < H / 32; b++) {
                        float x[32];
                        tmem_ld32(tmem + lanes + ob * D + col0 + 32 * b, x);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; i++) acc[16 * b + i] = __ffma2_rn(acc[16 * b + i], keep2, {x[2 * i], x[2 * i + 1]});
                    }
                    tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) arrive_leader<PAIR>(&s.o_empty[ob]);
            }
            const uint32_t slot = msg & 1;
            if (ok) ok = wait_warp(&s.msg_full[slot], (msg / 2) & 1, abort, a.err);
            const bool whole = it.count == it.units;
            // The rows go through Q's place, 16-byte units turned by the row's low bits, so that whole rows are stored.
            if (ok && live) {
                unsigned char *mine = stage + (size_t)row * D * 4;
                float mul = 1.0f;
                if (!SHARED && copies == 1 && whole) {
                    const float total = s.val[slot][row];
                    mul = total == 0.0f ? 0.0f : 1.0f / total;
                }
#pragma unroll
                for (int i = 0; i < H / 4; i++)
                    *reinterpret_cast<float4 *>(mine + (((col0 / 4 + i) ^ (row & 7)) << 4)) =
                        make_float4(acc[2 * i].x * mul, acc[2 * i].y * mul, acc[2 * i + 1].x * mul, acc[2 * i + 1].y * mul);
                uint64_t odd = row % span < rows && !(SHARED && it.seq < 0) ? *(volatile uint64_t *)&s.odd_nodes[PAIR ? items & 1 : 0] : 0;
                if (odd) {  // rare: values that are not finite, for the rows that see them
                    const int node = (row0 + row % span) / a.group;
                    odd &= a.tree ? a.tree[(size_t)it.seq * a.tokens + node] : ~0ull >> (63 - node);
                    while (odd) {
                        const int nd = __ffsll((long long)odd) - 1;
                        odd &= odd - 1;
                        const long long at = a.c.row(it.seq, base + it.length + nd);
                        // (only in the copy of Q that has the key: another may see nothing, and its sums be left out by a 0)
                        if (at < 0 || (it.length + nd) % kKeys * copies / kKeys != row / span) continue;
                        const __half *v = a.c.v + ((size_t)at * a.c.kv_heads + it.kv) * D + col0;
#pragma unroll 1
                        for (int i = 0; i < H; i++) {
                            const float f = __half2float(v[i]);
                            if (!(fabsf(f) < INFINITY))
                                *reinterpret_cast<float *>(mine + (((col0 + i) / 4 ^ (row & 7)) << 4) + (i & 3) * 4) += f;
                        }
                    }
                }
            }
            bad = group_any(3, 256, bad);
            ok = !group_any(4, 256, !ok);  // the eight warps stop together
            if (!ok) break;
            if (tid == 256) s.odd_nodes[PAIR ? items & 1 : 0] = 0;
            const size_t part = (size_t)(2 * team + (it.start > s.slot0)) * a.part_rows + rank * kRows;
            const float nan = __int_as_float(0x7fc00000);
            if (copies == 1) {
                // whole items with a shared prefix wait in out, or in the prefix's rows, for the join
                float *const rows_to = SHARED && it.seq < 0 ? a.prefix_acc : a.out;
                if ((SHARED || !whole) && col0 == 0 && row < rows) {
                    float2 *ml = a.part_ml + part + row;
                    if (SHARED && whole) ml = (it.seq < 0 ? a.prefix_ml : a.own_ml) + head_of<SHARED>(a, it, row0 + row);
                    *ml = make_float2(s.q_scale[qb][row], s.val[slot][row]);
                }
#pragma unroll 4
                for (int i = 0; w + 8 * i < rows; i++) {
                    const int r = w + 8 * i;
                    const size_t at = __shfl_sync(0xffffffffu, where, i);
                    float *dst = whole ? rows_to + at : a.part_acc + (part + r) * D;
#pragma unroll
                    for (int u = lane; u < D / 4; u += 32) {
                        float4 v = *reinterpret_cast<const float4 *>(stage + (size_t)r * D * 4 + ((u ^ (r & 7)) << 4));
                        if (bad) v = make_float4(nan, nan, nan, nan);
                        reinterpret_cast<float4 *>(dst)[u] = v;
                    }
                }
            } else {
                // the copies' maxima and totals become one
#pragma unroll 1
                for (int i = 0; w + 8 * i < rows; i++) {
                    const int r = w + 8 * i;
                    const size_t at = __shfl_sync(0xffffffffu, where, i);
                    float m = -INFINITY, l = 0.0f, f[4];
                    for (int k = 0; k < copies; k++) m = fmaxf(m, s.q_scale[qb][r + k * span]);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        f[k] = 0.0f;
                        if (k < copies) {
                            const float mk = s.q_scale[qb][r + k * span], lk = s.val[slot][r + k * span];
                            f[k] = mk == -INFINITY ? lk : ex2(mk - m);  // lk is 0 (nothing seen) or NaN
                            l += f[k] * lk;
                        }
                    }
                    float mul = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
                    if (bad) mul = nan;
                    float *dst = whole ? a.out + at : a.part_acc + (part + r) * D;
                    if (!whole && lane == 0) a.part_ml[part + r] = make_float2(m, l);
#pragma unroll
                    for (int u = lane; u < D / 4; u += 32) {
                        float4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            if (k < copies) {
                                const float4 x = *reinterpret_cast<const float4 *>(stage + (size_t)(r + k * span) * D * 4 + ((u ^ (r & 7)) << 4));
                                v.x += f[k] * x.x, v.y += f[k] * x.y, v.z += f[k] * x.z, v.w += f[k] * x.w;
                            }
                        reinterpret_cast<float4 *>(dst)[u] = make_float4(v.x * mul, v.y * mul, v.z * mul, v.w * mul);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) arrive(&s.msg_empty[slot]);
            msg++, items++;
            piece0 += value_pieces<C, SHARED>(a, it);
            group_sync(4, 256);  // Q's place is free again
            if (QB == 2) it = nx, where = where_nx, left = more;
            more = more && walk.next(a, nx);
        }
    }
    sync_all<PAIR>();  // (a pair's CTA stays until the other's MMAs and arrivals are over)
    if (warp == 1) {
        tc_fence_after();
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(s.tmem));
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(s.tmem));
    }
}

template <int D, int MR, bool PAIR, bool SHARED>
__global__ void __launch_bounds__(kThreads, 1) tree_attention_kernel(const __grid_constant__ AttendArgs a,
                                                                     const __grid_constant__ CUtensorMap k_map,
                                                                     const __grid_constant__ CUtensorMap v_map) {
    attend_tiles<D, MR, PAIR, SHARED, false>(a, k_map, v_map);
}

// ---- one token and at most four heads to a key head ---------------------------

// So few rows need no tensor cores: a value of the cache costs five instructions or so, and the SM has time for them while
// HBM delivers it. Warp w of 16 takes keys 8w .. 8w+7 of every unit, on its own from memory to registers: its copies go to
// its own part of shared memory, kStages units ahead, and a lane reads only what it copied itself, so there is no barrier
// before an item's end. Lane l holds 8 values of a key, D/8 lanes a key. The 8 x 4 partial products of a lane are added up
// over the lanes in a butterfly that leaves one score to a lane; softmax runs per warp, and an item's 16 maxima, totals and
// sums become one at its end. The division of the work and the join are the other kernel's. Bound by HBM (16 single tokens
// of 32 heads, 8 key heads of 128, 285 MB: 62 us, on the tensor cores 88).
constexpr int kFewWarps = 16, kFewRows = 4;
template <int D>
struct Few {
    static constexpr int kLanes = D / 8, kPer = 32 / kLanes, kLoads = 8 / kPer;  // lanes a key, keys a load, loads of 8 keys
    static constexpr int kStage = 2 * kLoads * 512, kStages = D == 128 ? 3 : 6;
    static constexpr int kRing = kFewWarps * kStages * kStage, kSmem = kRing + kFewWarps * kFewRows * D * 4;
    static_assert(kLoads * kFewRows == kLanes, "a score to a lane");
    // the kernel's own variables lie before, up to the next multiple of 1024
    static_assert(kSmem + (sizeof(Plan) + kFewWarps * kFewRows * sizeof(float2) + 1023) / 1024 * 1024 <= 232448, "shared memory");
};

__device__ __forceinline__ void eight(const unsigned char *p, float (&x)[8], bool none = false) {
    const uint4 y = none ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4 *>(p);
    const uint32_t z[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&z[i]));
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
}

template <int D>
__global__ void __launch_bounds__(32 * kFewWarps, 1) token_attention_kernel(const __grid_constant__ AttendArgs a) {
    using C = Few<D>;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ Plan s;
    __shared__ float2 ml[kFewWarps][kFewRows];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, team = blockIdx.x;
    const int key = lane / C::kLanes, dim = lane % C::kLanes * 8;
    const float nan = __int_as_float(0x7fc00000);
    if (warp == 0) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        plan<D, false>(a, s, team, gridDim.x);
    }
    __syncthreads();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    for (int q = team; q < a.seqs; q += gridDim.x)  // rows of refused sequences
        if (a.c.committed(q, 1) < 0)
            for (int i = tid; i < a.q_heads * D; i += 32 * kFewWarps) a.out[(size_t)q * a.q_heads * D + i] = nan;
    unsigned char *const ring = smem + warp * C::kStages * C::kStage + lane * 16;
    float *const sums = reinterpret_cast<float *>(smem + C::kRing);
    const size_t width = (size_t)a.c.kv_heads * D;
    Walk<D, false> walk(s);
    Item it;
    while (walk.next(a, it)) {
        const int all = it.length + 1, n = it.length + (a.tree ? (int)(a.tree[it.seq] & 1) : 1);  // keys there, keys seen
        const int first = it.first * kKeys + 8 * warp;
        const int *table = a.c.table + (size_t)it.seq * a.c.table_pages;
        bool bad = false;
        int page = 0;
        auto issue = [&](int t) {
            if (t < it.count) {
                if (!(t & 31)) {  // the pages of the next 32 units, a lane each
                    const int at = first + (t + lane) * kKeys;
                    page = t + lane < it.count && at < all ? table[at >> a.c.shift] : 0;
                    if ((unsigned)page >= (unsigned)a.c.pages) bad = true, page = 0;
                }
                const int p = __shfl_sync(0xffffffffu, page, t & 31), base = first + t * kKeys;
                if (base < all) {  // (the 8 rows lie in one page)
                    const size_t row = ((size_t)p << a.c.shift) + (base & (a.c.page_tokens() - 1)) + key;
                    const size_t off = row * width + (size_t)it.kv * D + dim;
                    const uint32_t to = smem_u32(ring + t % C::kStages * C::kStage);
#pragma unroll
                    for (int i = 0; i < C::kLoads; i++)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i * 512), "l"(a.c.k + off + i * C::kPer * width) : "memory");
#pragma unroll
                    for (int i = 0; i < C::kLoads; i++)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + (C::kLoads + i) * 512), "l"(a.c.v + off + i * C::kPer * width) : "memory");
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int t = 0; t < C::kStages - 1; t++) issue(t);
        float q[kFewRows][8], acc[kFewRows][8], m = -INFINITY, l = 0.0f;  // m and l: of row lane % 4
#pragma unroll
        for (int r = 0; r < kFewRows; r++) {
            const float *src = a.q + ((size_t)it.seq * a.q_heads + it.kv * a.group + min(r, a.group - 1)) * D + dim;
#pragma unroll
            for (int e = 0; e < 8; e += 4) *reinterpret_cast<float4 *>(&q[r][e]) = *reinterpret_cast<const float4 *>(src + e);
#pragma unroll
            for (int e = 0; e < 8; e++) q[r][e] *= a.scale * a.sign, acc[r][e] = 0.0f;
        }
#pragma unroll 1
        for (int t = 0; t < it.count; t++) {
            __syncwarp();  // what was read from the place of the unit before is read
            issue(t + C::kStages - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 1) : "memory");
            const int base = first + t * kKeys;
            if (base >= all) break;  // and so are the units after it
            const unsigned char *k = ring + t % C::kStages * C::kStage, *v = k + C::kLoads * 512;
            float x[C::kLanes];
#pragma unroll
            for (int i = 0; i < C::kLoads; i++) {
                float f[8];
                eight(k + i * 512, f);
#pragma unroll
                for (int r = 0; r < kFewRows; r++) {
                    float dot = q[r][0] * f[0];
#pragma unroll
                    for (int e = 1; e < 8; e++) dot = fmaf(q[r][e], f[e], dot);
                    x[i * kFewRows + r] = dot;
                }
            }
#pragma unroll
            for (int o = C::kLanes / 2; o; o >>= 1) {
#pragma unroll
                for (int j = 0; j < o; j++) {
                    const float mine = lane & o ? x[j + o] : x[j], other = lane & o ? x[j] : x[j + o];
                    x[j] = mine + __shfl_xor_sync(0xffffffffu, other, o);
                }
            }
            // the lane's score: row lane % 4 and key
            const int at = base + lane % C::kLanes / kFewRows * C::kPer + key;
            const float score = at < n ? x[0] : -INFINITY;
            float top = score;
#pragma unroll
            for (int o = kFewRows; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            top = fmaxf(m, top);
            if (__any_sync(0xffffffffu, top > m)) {
                const float keep = m == -INFINITY ? 0.0f : ex2(m - top);
                l *= keep;
                m = top;
#pragma unroll
                for (int r = 0; r < kFewRows; r++) {
                    const float f = __shfl_sync(0xffffffffu, keep, r);
#pragma unroll
                    for (int e = 0; e < 8; e++) acc[r][e] *= f;
                }
            }
            const float p = ex2(score - (m == -INFINITY ? 0.0f : m));
            l += p;
#pragma unroll
            for (int i = 0; i < C::kLoads; i++) {
                float f[8];
                eight(v + i * 512, f, base + i * C::kPer + key >= n);  // unseen values are any: P = 0 would not keep a NaN out
#pragma unroll
                for (int r = 0; r < kFewRows; r++) {
                    const float w = __shfl_sync(0xffffffffu, p, key * C::kLanes + i * kFewRows + r);
#pragma unroll
                    for (int e = 0; e < 8; e++) acc[r][e] = fmaf(w, f[e], acc[r][e]);
                }
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        // ---- the warps' parts become one
#pragma unroll
        for (int o = kFewRows; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
        for (int r = 0; r < kFewRows; r++) {
#pragma unroll
            for (int e = 0; e < 8; e++)
#pragma unroll
                for (int o = C::kLanes; o < 32; o <<= 1) acc[r][e] += __shfl_xor_sync(0xffffffffu, acc[r][e], o);
            if (key == 0)
#pragma unroll
                for (int e = 0; e < 8; e += 4)
                    *reinterpret_cast<float4 *>(&sums[(warp * kFewRows + r) * D + dim + e]) = *reinterpret_cast<float4 *>(&acc[r][e]);
        }
        if (lane < kFewRows) ml[warp][lane] = make_float2(m, l);
        bad = __syncthreads_or(bad);
        const bool whole = it.count == it.units;
        const size_t part = (size_t)(2 * team + (it.start > s.slot0)) * a.part_rows;
        for (int i = tid; i < a.group * D; i += 32 * kFewWarps) {
            const int r = i / D, d = i % D;
            float most = -INFINITY, total = 0.0f, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kFewWarps; w++) most = fmaxf(most, ml[w][r].x);
#pragma unroll
            for (int w = 0; w < kFewWarps; w++) {
                const float2 x = ml[w][r];
                const float f = x.x == -INFINITY ? x.y : ex2(x.x - most);  // its total is 0 (nothing seen) or NaN
                total += f * x.y;
                sum = fmaf(f, sums[(w * kFewRows + r) * D + d], sum);
            }
            if (bad) sum = nan;
            if (whole) {
                a.out[((size_t)it.seq * a.q_heads + it.kv * a.group + r) * D + d] = total == 0.0f && !bad ? 0.0f : sum / total;
            } else {
                a.part_acc[(part + r) * D + d] = sum;
                if (d == 0) a.part_ml[part + r] = make_float2(most, total);
            }
        }
        __syncthreads();
    }
}

// The same with a shared prefix, for the sequences' own keys: these are few, and an item's start and end would be most of its
// time. So a CTA works on four items at once: a group of four warps on one, warp w of them on keys 8w .. 8w+7 of every 32.
constexpr int kGroups = 4, kGroupWarps = kFewWarps / kGroups, kGroupKeys = 8 * kGroupWarps;
struct GroupNotes {
    Plan plan[kGroups];
    float2 ml[kFewWarps][kFewRows];
};
template <int D>
__device__ __forceinline__ void attend_tokens(const AttendArgs &a, unsigned char *smem, GroupNotes &notes, int team) {
    using C = Few<D>;
    constexpr int kSteps = kKeys / kGroupKeys;  // to a unit
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = warp / kGroupWarps, tid = threadIdx.x % (32 * kGroupWarps);
    const int key = lane / C::kLanes, dim = lane % C::kLanes * 8;
    const float nan = __int_as_float(0x7fc00000);
    const Plan &s = notes.plan[group];
    float2 (*const ml)[kFewRows] = notes.ml + group * kGroupWarps;
    unsigned char *const ring = smem + warp * C::kStages * C::kStage + lane * 16;
    float *const sums = reinterpret_cast<float *>(smem + C::kRing) + group * kGroupWarps * kFewRows * D;
    const size_t width = (size_t)a.c.kv_heads * D;
    const int base0 = s.common;  // where the items' positions begin
    Walk<D, true> walk(s);
    Item it;
    while (walk.next(a, it)) {
        const int all = it.length + 1, n = it.length + (a.tree ? (int)(a.tree[it.seq] & 1) : 1);  // keys there, keys seen
        const int first = it.first * kKeys + 8 * (warp % kGroupWarps), steps = it.count * kSteps;
        const int *table = a.c.table + (size_t)it.seq * a.c.table_pages;
        bool bad = false;
        int page = 0;
        auto issue = [&](int t) {
            if (t < steps) {
                if (!(t & 31)) {  // the pages of the next 32 steps, a lane each
                    const int at = first + (t + lane) * kGroupKeys;
                    page = t + lane < steps && at < all ? table[(base0 + at) >> a.c.shift] : 0;
                    if ((unsigned)page >= (unsigned)a.c.pages) bad = true, page = 0;
                }
                const int p = __shfl_sync(0xffffffffu, page, t & 31), base = first + t * kGroupKeys;
                if (base < all) {  // (the 8 rows lie in one page)
                    const size_t row = ((size_t)p << a.c.shift) + (base & (a.c.page_tokens() - 1)) + key;
                    const size_t off = row * width + (size_t)it.kv * D + dim;
                    const uint32_t to = smem_u32(ring + t % C::kStages * C::kStage);
#pragma unroll
                    for (int i = 0; i < C::kLoads; i++)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i * 512), "l"(a.c.k + off + i * C::kPer * width) : "memory");
#pragma unroll
                    for (int i = 0; i < C::kLoads; i++)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + (C::kLoads + i) * 512), "l"(a.c.v + off + i * C::kPer * width) : "memory");
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int t = 0; t < C::kStages - 1; t++) issue(t);
        float q[kFewRows][8], acc[kFewRows][8], m = -INFINITY, l = 0.0f;  // m and l: of row lane % 4
#pragma unroll
        for (int r = 0; r < kFewRows; r++) {
            const float *src = a.q + ((size_t)it.seq * a.q_heads + it.kv * a.group + min(r, a.group - 1)) * D + dim;
#pragma unroll
            for (int e = 0; e < 8; e += 4) *reinterpret_cast<float4 *>(&q[r][e]) = *reinterpret_cast<const float4 *>(src + e);
#pragma unroll
            for (int e = 0; e < 8; e++) q[r][e] *= a.scale * a.sign, acc[r][e] = 0.0f;
        }
#pragma unroll 1
        for (int t = 0; t < steps; t++) {
            __syncwarp();  // what was read from the place of the unit before is read
            issue(t + C::kStages - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 1) : "memory");
            const int base = first + t * kGroupKeys;
            if (base >= all) break;  // and so are the steps after it
            const unsigned char *k = ring + t % C::kStages * C::kStage, *v = k + C::kLoads * 512;
            float x[C::kLanes];
#pragma unroll
            for (int i = 0; i < C::kLoads; i++) {
                float f[8];
                eight(k + i * 512, f);
#pragma unroll
                for (int r = 0; r < kFewRows; r++) {
                    float dot = q[r][0] * f[0];
#pragma unroll
                    for (int e = 1; e < 8; e++) dot = fmaf(q[r][e], f[e], dot);
                    x[i * kFewRows + r] = dot;
                }
            }
#pragma unroll
            for (int o = C::kLanes / 2; o; o >>= 1) {
#pragma unroll
                for (int j = 0; j < o; j++) {
                    const float mine = lane & o ? x[j + o] : x[j], other = lane & o ? x[j] : x[j + o];
                    x[j] = mine + __shfl_xor_sync(0xffffffffu, other, o);
                }
            }
            // the lane's score: row lane % 4 and key
            const int at = base + lane % C::kLanes / kFewRows * C::kPer + key;
            const float score = at < n ? x[0] : -INFINITY;
            float top = score;
#pragma unroll
            for (int o = kFewRows; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            top = fmaxf(m, top);
            if (__any_sync(0xffffffffu, top > m)) {
                const float keep = m == -INFINITY ? 0.0f : ex2(m - top);
                l *= keep;
                m = top;
#pragma unroll
                for (int r = 0; r < kFewRows; r++) {
                    const float f = __shfl_sync(0xffffffffu, keep, r);
#pragma unroll
                    for (int e = 0; e < 8; e++) acc[r][e] *= f;
                }
            }
            const float p = ex2(score - (m == -INFINITY ? 0.0f : m));
            l += p;
#pragma unroll
            for (int i = 0; i < C::kLoads; i++) {
                float f[8];
                eight(v + i * 512, f, base + i * C::kPer + key >= n);  // unseen values are any: P = 0 would not keep a NaN out
#pragma unroll
                for (int r = 0; r < kFewRows; r++) {
                    const float w = __shfl_sync(0xffffffffu, p, key * C::kLanes + i * kFewRows + r);
#pragma unroll
                    for (int e = 0; e < 8; e++) acc[r][e] = fmaf(w, f[e], acc[r][e]);
                }
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        // ---- the group's parts become one
#pragma unroll
        for (int o = kFewRows; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
        for (int r = 0; r < kFewRows; r++) {
#pragma unroll
            for (int e = 0; e < 8; e++)
#pragma unroll
                for (int o = C::kLanes; o < 32; o <<= 1) acc[r][e] += __shfl_xor_sync(0xffffffffu, acc[r][e], o);
            if (key == 0)
#pragma unroll
                for (int e = 0; e < 8; e += 4)
                    *reinterpret_cast<float4 *>(&sums[(warp % kGroupWarps * kFewRows + r) * D + dim + e]) = *reinterpret_cast<float4 *>(&acc[r][e]);
        }
        if (lane < kFewRows) ml[warp % kGroupWarps][lane] = make_float2(m, l);
        bad = group_any(1 + group, 32 * kGroupWarps, bad);
        const bool whole = it.count == it.units;
        const size_t part = (size_t)(2 * (team + group) + (it.start > s.slot0)) * kFewRows;
        for (int i = tid; i < a.group * D; i += 32 * kGroupWarps) {
            const int r = i / D, d = i % D;
            float most = -INFINITY, total = 0.0f, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kGroupWarps; w++) most = fmaxf(most, ml[w][r].x);
#pragma unroll
            for (int w = 0; w < kGroupWarps; w++) {
                const float2 x = ml[w][r];
                const float f = x.x == -INFINITY ? x.y : ex2(x.x - most);  // its total is 0 (nothing seen) or NaN
                total += f * x.y;
                sum = fmaf(f, sums[(w * kFewRows + r) * D + d], sum);
            }
            sum *= kPScale, total *= kPScale;  // as the prefix's parts are
            if (bad) sum = nan;
            // all of it is for the join
            const size_t at = (size_t)it.seq * a.q_heads + it.kv * a.group + r;
            *((whole ? a.out + at * D : a.own_part_acc + (part + r) * D) + d) = sum;
            if (d == 0) *(whole ? a.own_ml + at : a.own_part_ml + part + r) = make_float2(most, total);
        }
        group_sync(1 + group, 32 * kGroupWarps);
    }
}

// With a shared prefix: the first CTAs do the prefix on the tensor cores, the others the sequences without them. Each has a line
// of its own, and they share the GPU by what the lines take.
// Time of a slot of either line, relatively (64 users, 4,112 shared, in us, 1 to 1, 2 to 1, 3 to 1 and 4 to 1: 32/8 heads of 128 71, 53,
// 51, 55; 10/10 of 128 77, 53, 49, 54; 16/4 of 64 45, 37, 34, 34, with 16,384 shared 58, 51, 50, 48).
constexpr int kPrefixUnit = 3, kTokenUnit = 1;
template <int D>
__global__ void __launch_bounds__(kThreads, 1) shared_token_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ CUtensorMap k_map,
                                                                   const __grid_constant__ CUtensorMap v_map) {
    using C = Cfg<D, 128, false>;
    static_assert(kThreads == 32 * kFewWarps && sizeof(GroupNotes) <= kNotes && Few<D>::kSmem <= C::kSmem - kNotes, "one CTA for both");
    extern __shared__ __align__(1024) unsigned char smem[];
    GroupNotes &notes = *reinterpret_cast<GroupNotes *>(smem + C::kSmem - kNotes);  // (the first plan is where the tiles' plan is, too)
    const int warp = threadIdx.x >> 5, group = warp / kGroupWarps;
    if (warp % kGroupWarps == 0) {  // a plan for each group, or for the CTA
        asm volatile("griddepcontrol.wait;" ::: "memory");
        const int lane = threadIdx.x & 31, cta = blockIdx.x, ctas = gridDim.x, per = a.c.kv_heads;
        const int shared = asked_shared<true>(a), source = first_live(a, shared), common = common_of(a, shared, source);
        const int len = lane < a.seqs ? own_length<true>(a, lane, shared, common) : -1;
        const long long prefix = prefix_line<D>(a, common), own = sum_slots<D, true>(a, a.seqs, per, shared, common);
        const long long c1 = prefix * kPrefixUnit, c2 = own * kTokenUnit;
        const int split = prefix ? max(1, min(ctas - 1, (int)((ctas * c1 + (c1 + c2) / 2) / (c1 + c2)))) : 0;
        const int prefix_g = (int)min((long long)split, prefix), own_g = (int)min((long long)(ctas - split) * kGroups, own);
        const bool first = cta < split;
        const int g = first ? prefix_g : own_g;
        const int team = first ? cta : (cta - split) * kGroups + group;
        const long long w = first ? prefix : own;
        long long base = 0, u0 = 0, u1 = 0;
        int seq = first ? -1 : 0, length = common;
        if (team < g) {
            u0 = range_start(team, w, g);
            u1 = range_start(team + 1, w, g);
            if (!first) seq = find_slot<D, true>(a, per, u0, len, shared, common, base, length);
        }
        if (lane == 0 && (!first || group == 0)) {
            Plan &s = notes.plan[group];
            const int slots = first ? prefix_slots<D>(common) : max(1, slots_of<D, true>(a, length)), index = (int)quotient(u0 - base, slots);
            const int tiles = first ? a.all_tiles : 1;
            s.slot0 = u0, s.slot1 = u1, s.seq0 = seq, s.length0 = length;
            s.kv0 = index / tiles, s.tile0 = index % tiles;
            s.pos0 = (int)(u0 - base - (long long)index * slots);
            s.common = common, s.source = first ? source : split;
        }
        if (cta == 0 && warp == 0) tell_join<D>(a, shared, common, 0, own, prefix, own_g, prefix_g);
    }
    __syncthreads();
    if (notes.plan[0].seq0 < 0) {
        attend_tiles<D, 128, false, true, true>(a, k_map, v_map);
    } else {
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        attend_tokens<D>(a, smem, notes, ((int)blockIdx.x - notes.plan[0].source) * kGroups);
    }
}

// Joins the parts of items that several CTAs share, and makes every row NaN
// after an error: one CTA per (row, head). Warps take every eighth part, so all
// loads of a row are in flight at once; their sums join in order.
template <int D>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ AttendArgs a, int teams) {
    constexpr int V = D / 32;
    __shared__ float sums[8][D];
    __shared__ float2 totals[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int id = blockIdx.x, h = id % a.q_heads, row = id / a.q_heads, seq = row / a.tokens;
    const int kv = h / a.group, r = (row % a.tokens) * a.group + h % a.group, tile = r / a.tile_rows;
    const int per = a.c.kv_heads * a.row_tiles;
    const int units = units_of(a, a.c.committed(seq, a.tokens));
    const long long w = sum_slots<D, false>(a, a.seqs, per, 0, 0);
    const long long start = (seq ? sum_slots<D, false>(a, seq, per, 0, 0) : 0) + (long long)(kv * a.row_tiles + tile) * (units + kItemCost<D, false>) + kItemCost<D, false>;
    const int g = (int)min((long long)teams, w);
    const int c0 = units ? cta_of(start, w, g) : 0, parts = units ? cta_of(start + units - 1, w, g) - c0 + 1 : 0;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    float *out = a.out + (size_t)id * D;
    if (*(volatile int *)a.err) {
        for (int i = threadIdx.x; i < D; i += 256) out[i] = __int_as_float(0x7fc00000);
        return;
    }
    if (parts < 2) return;
    // Every warp has its own maximum; kFly parts are asked for before the first is used.
    constexpr int kFly = 5;
    float m = -INFINITY, l = 0.0f, acc[V];
#pragma unroll
    for (int e = 0; e < V; e++) acc[e] = 0.0f;
    const bool late = start > range_start(c0, w, g);  // the first part is its CTA's second
    for (int p0 = warp; p0 < parts; p0 += 8 * kFly) {
        float2 ml[kFly];
        float x[kFly][V], top = m;
#pragma unroll
        for (int i = 0; i < kFly; i++) {
            const int p = p0 + 8 * i;
            ml[i] = make_float2(-INFINITY, 0.0f);
            if (p < parts) {
                const size_t at = (size_t)(2 * (c0 + p) + (p == 0 && late)) * a.part_rows + r % a.tile_rows;
                const float *src = a.part_acc + at * D + lane * V;
                ml[i] = __ldcg(a.part_ml + at);
                if constexpr (V == 2) {
                    *reinterpret_cast<float2 *>(x[i]) = __ldcg(reinterpret_cast<const float2 *>(src));
                } else {
#pragma unroll
                    for (int e = 0; e < V; e += 4) *reinterpret_cast<float4 *>(x[i] + e) = __ldcg(reinterpret_cast<const float4 *>(src + e));
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kFly; i++) top = fmaxf(top, ml[i].x);
        const float keep = m == -INFINITY ? 1.0f : ex2(m - top);  // (what there is without a maximum is 0 or NaN)
        m = top;
        l *= keep;
#pragma unroll
        for (int e = 0; e < V; e++) acc[e] *= keep;
#pragma unroll
        for (int i = 0; i < kFly; i++) {
            if (p0 + 8 * i >= parts) continue;
            const float f = ml[i].x == -INFINITY ? ml[i].y : ex2(ml[i].x - m);  // its total is 0 (nothing seen) or NaN
            l += f * ml[i].y;
#pragma unroll
            for (int e = 0; e < V; e++) acc[e] = fmaf(f, x[i][e], acc[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < V; e++) sums[warp][lane * V + e] = acc[e];
    if (lane == 0) totals[warp] = make_float2(m, l);
    __syncthreads();
    m = -INFINITY, l = 0.0f;
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; k++) m = fmaxf(m, totals[k].x);
#pragma unroll
    for (int k = 0; k < 8; k++) {
        f[k] = totals[k].x == -INFINITY ? totals[k].y : ex2(totals[k].x - m);
        l += f[k] * totals[k].y;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    for (int i = threadIdx.x; i < D; i += 256) {
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++) v = fmaf(f[k], sums[k][i], v);
        out[i] = v * inv;
    }
}

// With a shared prefix every row has parts: the prefix's, then its sequence's own. What a CTA did as a whole is in the rows of
// prefix_acc or out. WARPS warps to a (row, head): eight where there are so few rows that each may have many parts, otherwise one,
// so that all rows are under way at once (the whole call, in us, with eight and with one: 8 x 17 rows of 24 heads, 8,192 shared
// 88 and 70; two single tokens of 24 heads, 30,016 shared 39 and 69; eight of 32 heads, 8,192 shared 39 and 47).
template <int D, int WARPS>
__global__ void __launch_bounds__(256) join_shared_kernel(const __grid_constant__ AttendArgs a) {
    constexpr int V = D / 32, kFly = 4;  // parts that are asked for before the first is used
    __shared__ float sums[8][D];
    __shared__ float2 totals[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int id = WARPS == 1 ? blockIdx.x * 8 + warp : blockIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (id >= a.seqs * a.tokens * a.q_heads) return;  // (whole warps, and no barrier with WARPS 1)
    const int h = id % a.q_heads, row = id / a.q_heads, seq = row / a.tokens, kv = h / a.group, r = (row - seq * a.tokens) * a.group + h % a.group;
    const long long w = a.starts[a.seqs], all_w = a.starts[a.seqs + 1], first = a.starts[seq];
    const int *said = a.lengths + a.seqs;
    const int own = a.lengths[seq], common = said[0], g = said[1], all_g = said[2], units = units_of(a, own);
    float *out = a.out + (size_t)id * D;
    if (*(volatile int *)a.err || own < 0) {
        for (int i = WARPS == 1 ? lane : threadIdx.x; i < D; i += 32 * WARPS) out[i] = __int_as_float(0x7fc00000);
        return;
    }
    const long long start = first + (long long)(kv * a.row_tiles + r / a.tile_rows) * (units + kItemCost<D, true>) + kItemCost<D, true>;
    const int c0 = cta_of(start, w, g), parts = cta_of(start + units - 1, w, g) - c0 + 1;
    // the prefix's parts of this row
    const int all_r = row * a.group + h % a.group;
    const long long all_start = (long long)(kv * a.all_tiles + all_r / a.tile_rows) * prefix_slots<D>(common) + kItemCost<D, true>;
    const int p0 = common ? cta_of(all_start, all_w, all_g) : 0, before = common ? cta_of(all_start + common / kKeys - 1, all_w, all_g) - p0 + 1 : 0;
    // the first part is its CTA's second
    const bool late = start > range_start(c0, w, g), all_late = common && all_start > range_start(p0, all_w, all_g);
    const int count = before + parts;
    // where part p of the row is
    auto part = [&](int p, const float *&acc, const float2 *&ml) {
        const bool prefix = p < before;
        if ((prefix ? before : parts) == 1) {
            acc = (prefix ? a.prefix_acc : a.out) + (size_t)id * D, ml = (prefix ? a.prefix_ml : a.own_ml) + id;
            return;
        }
        const int q = prefix ? p : p - before;
        const size_t at = (size_t)(2 * ((prefix ? p0 : c0) + q) + (q == 0 && (prefix ? all_late : late))) * (prefix ? a.part_rows : a.own_part_rows) +
                          (prefix ? all_r : r) % a.tile_rows;
        acc = (prefix ? a.part_acc : a.own_part_acc) + at * D, ml = (prefix ? a.part_ml : a.own_part_ml) + at;
    };
    float m = -INFINITY, l = 0.0f, acc[V];
#pragma unroll
    for (int e = 0; e < V; e++) acc[e] = 0.0f;
    for (int from = WARPS == 1 ? 0 : warp; from < count; from += WARPS * kFly) {
        float2 ml[kFly];
        float x[kFly][V], top = m;
#pragma unroll
        for (int i = 0; i < kFly; i++) {
            const int p = from + WARPS * i;
            ml[i] = make_float2(-INFINITY, 0.0f);
            if (p < count) {
                const float *src;
                const float2 *totals_at;
                part(p, src, totals_at);
                src += lane * V;
                ml[i] = __ldcg(totals_at);
                if constexpr (V == 2) {
                    *reinterpret_cast<float2 *>(x[i]) = __ldcg(reinterpret_cast<const float2 *>(src));
                } else {
#pragma unroll
                    for (int e = 0; e < V; e += 4) *reinterpret_cast<float4 *>(x[i] + e) = __ldcg(reinterpret_cast<const float4 *>(src + e));
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kFly; i++) top = fmaxf(top, ml[i].x);
        const float keep = m == -INFINITY ? 1.0f : ex2(m - top);  // (what there is without a maximum is 0 or NaN)
        m = top;
        l *= keep;
#pragma unroll
        for (int e = 0; e < V; e++) acc[e] *= keep;
#pragma unroll
        for (int i = 0; i < kFly; i++) {
            if (from + WARPS * i >= count) continue;
            const float f = ml[i].x == -INFINITY ? ml[i].y : ex2(ml[i].x - m);  // its total is 0 (nothing seen) or NaN
            l += f * ml[i].y;
#pragma unroll
            for (int e = 0; e < V; e++) acc[e] = fmaf(f, x[i][e], acc[e]);
        }
    }
    if constexpr (WARPS == 1) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int e = 0; e < V; e++) acc[e] *= inv;
        float *to = out + lane * V;
        if constexpr (V == 2) {
            *reinterpret_cast<float2 *>(to) = *reinterpret_cast<float2 *>(acc);
        } else {
#pragma unroll
            for (int e = 0; e < V; e += 4) *reinterpret_cast<float4 *>(to + e) = *reinterpret_cast<float4 *>(acc + e);
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; e++) sums[warp][lane * V + e] = acc[e];
        if (lane == 0) totals[warp] = make_float2(m, l);
        __syncthreads();
        m = -INFINITY, l = 0.0f;
        float f[8];
#pragma unroll
        for (int k = 0; k < 8; k++) m = fmaxf(m, totals[k].x);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            f[k] = totals[k].x == -INFINITY ? totals[k].y : ex2(totals[k].x - m);
            l += f[k] * totals[k].y;
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        for (int i = threadIdx.x; i < D; i += 256) {
            float v = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; k++) v = fmaf(f[k], sums[k][i], v);
            out[i] = v * inv;
        }
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// One layer's pool as [column blocks of 64 values][rows][64], read in boxes of box rows and `blocks` column blocks.
int pool_map(CUtensorMap *m, const CacheView &c, const __half *pool, int box, int blocks) {
    static EncodeTiled fn = nullptr;
    if (!fn) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return cudaErrorNotSupported;
        fn = reinterpret_cast<EncodeTiled>(p);
    }
    const cuuint64_t width = (cuuint64_t)c.kv_heads * c.head_dim;
    const cuuint64_t dims[3] = {64, (cuuint64_t)c.pages << c.shift, width / 64}, strides[2] = {width * sizeof(__half), 128};
    const cuuint32_t boxes[3] = {64, (cuuint32_t)box, (cuuint32_t)blocks}, step[3] = {1, 1, 1};
    const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half *>(pool), dims, strides, boxes, step,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : cudaErrorInvalidValue;
}

int part_rows(int tokens, int group) { return tokens * group < kRows ? tokens * group : kRows; }

constexpr unsigned kFewJoined = 4 * kSms;  // rows that get eight warps each

size_t ml_bytes(int rows) { return (size_t)2 * kMaxCtas * rows * sizeof(float2); }

// The attention kernel and the join, chained to what runs before. Peers: CTAs that work on one item.
template <int D, bool SHARED, typename... A>
int launch(const AttendArgs &a, void (*kernel)(A...), int peers, int threads, int smem, const A &...args) {
    if (int rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) return rc;
    // no more CTAs than the longest sequences that the table allows could use
    const long long units = (((long long)a.c.table_pages << a.c.shift) + kKeys - 1) / kKeys;
    const long long most = ((long long)a.seqs * a.row_tiles + (SHARED ? a.all_tiles : 0)) * a.c.kv_heads * (units + kItemCost<D, SHARED>);
    const int teams = (int)(most < kMaxCtas / peers ? most : kMaxCtas / peers);  // (two at least with SHARED: items cost more than a slot)
    cudaLaunchConfig_t cfg = {};
    cfg.stream = launch_stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = peers;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = peers > 1 ? 2 : 1;
    cfg.gridDim = dim3(teams * peers);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    if (int rc = cudaLaunchKernelEx(&cfg, kernel, args...)) return rc;
    cfg.numAttrs = 1;
    const unsigned rows = (unsigned)(a.seqs * a.tokens * a.q_heads);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    if constexpr (!SHARED) {
        cfg.gridDim = dim3(rows);
        return cudaLaunchKernelEx(&cfg, join_kernel<D>, a, teams);
    } else {
        cfg.gridDim = dim3(rows <= kFewJoined ? rows : (rows + 7) / 8);
        return rows <= kFewJoined ? cudaLaunchKernelEx(&cfg, join_shared_kernel<D, 8>, a) : cudaLaunchKernelEx(&cfg, join_shared_kernel<D, 1>, a);
    }
}
template <int D, int MR, bool PAIR, bool SHARED>
int launch_tiles(const AttendArgs &a, const CUtensorMap &k_map, const CUtensorMap &v_map) {
    return launch<D, SHARED>(a, tree_attention_kernel<D, MR, PAIR, SHARED>, PAIR ? 2 : 1, kThreads, Cfg<D, MR, PAIR>::kSmem, a, k_map, v_map);
}
template <int D>
int launch_token(const AttendArgs &a) {
    return launch<D, false>(a, token_attention_kernel<D>, 1, 32 * kFewWarps, Few<D>::kSmem, a);
}

// Checks of both attentions' arguments, and what follows from them alone.
int attend_args(AttendArgs &a, float *out, const float *q, const qg_kv_cache *cache, int layer, const uint64_t *tree, float scale, int seqs,
                int tokens, int q_heads, void *workspace) {
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
    if (!(a.scale < INFINITY)) return cudaErrorInvalidValue;
    a.seqs = seqs;
    a.tokens = tokens;
    a.q_heads = q_heads;
    a.group = q_heads / a.c.kv_heads;
    a.tile_scale = a.scale;
    a.shared = nullptr;
    a.all_tiles = 0;
    a.prefix_acc = nullptr;
    a.prefix_ml = a.own_ml = nullptr;
    a.own_part_acc = nullptr;
    a.own_part_ml = nullptr;
    a.own_part_rows = 0;
    a.starts = nullptr;
    a.lengths = nullptr;
    a.err = static_cast<int *>(workspace);
    a.part_ml = reinterpret_cast<float2 *>(static_cast<char *>(workspace) + 256);
    return 0;
}
// Tiles of 128 rows, or of 256 for a pair, and the boxes of keys and values that go with them. `rows`: of the tallest item.
void tiles(AttendArgs &a, int rows, bool pair) {
    a.tile_rows = pair ? 2 * kRows : kRows;
    a.row_tiles = (a.tokens * a.group + a.tile_rows - 1) / a.tile_rows;
    a.part_rows = rows < a.tile_rows ? rows : a.tile_rows;
    const int page = a.c.page_tokens(), k_rows = pair ? kKeys / 2 : kKeys, v_blocks = a.c.head_dim / (pair ? 128 : 64);
    const int v_rows = 16384 / (128 * v_blocks);
    a.k_box = page < k_rows ? page : k_rows;
    a.k_blocks = pair && a.k_box == k_rows ? 2 : 1;
    a.v_box = page < v_rows ? page : v_rows;
}
int maps(const AttendArgs &a, bool pair, CUtensorMap &k_map, CUtensorMap &v_map) {
    if (int rc = pool_map(&k_map, a.c, a.c.k, a.k_box, a.k_blocks)) return rc;
    return pool_map(&v_map, a.c, a.c.v, a.v_box, a.c.head_dim / (pair ? 128 : 64));
}
bool bad_sizes(int seqs, int tokens, int q_heads, int kv_heads, int head_dim) {
    return seqs < 1 || seqs > kMaxSeqs || tokens < 1 || tokens > kMaxNodes || kv_heads < 1 || kv_heads > 1024 || q_heads < kv_heads ||
           q_heads > 1024 || q_heads % kv_heads || (head_dim != 64 && head_dim != 128 && head_dim != 256);
}
constexpr size_t kFewParts = (size_t)2 * kGroups * kMaxCtas * kFewRows;  // rows of the parts of sequences' own lines
constexpr long long kMaxShared = 1 << 24;  // rows and heads of a batch with a shared prefix

}  // namespace

extern "C" int qg_attention_workspace_bytes(int seqs, int tokens, int q_heads, int kv_heads, int head_dim, size_t *bytes) {
    if (!bytes || bad_sizes(seqs, tokens, q_heads, kv_heads, head_dim)) return cudaErrorInvalidValue;
    const int rows = part_rows(tokens, q_heads / kv_heads);
    *bytes = 256 + ml_bytes(rows) + (size_t)2 * kMaxCtas * rows * head_dim * sizeof(float);
    return cudaSuccess;
}

extern "C" int qg_tree_attention(float *out, const float *q, const qg_kv_cache *cache, int layer, const uint64_t *tree,
                                 float scale, int seqs, int tokens, int q_heads, void *workspace) {
    AttendArgs a;
    if (int rc = attend_args(a, out, q, cache, layer, tree, scale, seqs, tokens, q_heads, workspace)) return rc;
    // Few rows: heads of 64 and 128 values, whose units take little time, share a unit's keys among copies of Q; heads of
    // 256 keep only 64 rows of Q, and the room goes to the rings. Many rows of heads of 256: pairs of CTAs.
    const int rows = tokens * a.group;
    const bool pair = a.c.head_dim == 256 && rows > kRows;
    a.copies = a.c.head_dim == 256 || rows > 64 ? 1 : a.c.head_dim == 128 || rows > 32 ? 2 : 4;
    tiles(a, rows, pair);
    a.part_acc = reinterpret_cast<float *>(static_cast<char *>(workspace) + 256 + ml_bytes(part_rows(tokens, a.group)));
    // One token, at most four heads to a key head of up to 128 values: no tensor cores (16 tokens, 32/8 heads of 128: 62 us
    // against 88). Heads of 256 leave no room for copies ahead.
    if (rows <= kFewRows && tokens == 1 && a.c.head_dim <= 128) return a.c.head_dim == 64 ? launch_token<64>(a) : launch_token<128>(a);
    CUtensorMap k_map, v_map;
    if (int rc = maps(a, pair, k_map, v_map)) return rc;
    if (a.c.head_dim == 64) return launch_tiles<64, 128, false, false>(a, k_map, v_map);
    if (a.c.head_dim == 128) return rows <= 32 ? launch_tiles<128, 64, false, false>(a, k_map, v_map) : launch_tiles<128, 128, false, false>(a, k_map, v_map);
    if (pair) return launch_tiles<256, 128, true, false>(a, k_map, v_map);
    return rows <= 64 ? launch_tiles<256, 64, false, false>(a, k_map, v_map) : launch_tiles<256, 128, false, false>(a, k_map, v_map);
}

extern "C" int qg_shared_attention_workspace_bytes(int seqs, int tokens, int q_heads, int kv_heads, int head_dim, size_t *bytes) {
    if (!bytes || bad_sizes(seqs, tokens, q_heads, kv_heads, head_dim) || (long long)seqs * tokens * q_heads > kMaxShared)
        return cudaErrorInvalidValue;
    const int rows = part_rows(seqs * tokens, q_heads / kv_heads);
    const size_t heads = ((size_t)seqs * tokens * q_heads + 1) & ~(size_t)1;
    *bytes = 256 + ml_bytes(rows) + (size_t)2 * kMaxCtas * rows * head_dim * sizeof(float) + heads * (2 * sizeof(float2) + head_dim * sizeof(float)) +
             (kMaxSeqs + 2) * sizeof(long long) + (kMaxSeqs + 4) * sizeof(int) + kFewParts * (sizeof(float2) + head_dim * sizeof(float));
    return cudaSuccess;
}

extern "C" int qg_shared_attention(float *out, const float *q, const qg_kv_cache *cache, int layer, const int *shared, const uint64_t *tree,
                                   float scale, int seqs, int tokens, int q_heads, void *workspace) {
    AttendArgs a;
    if (int rc = attend_args(a, out, q, cache, layer, tree, scale, seqs, tokens, q_heads, workspace)) return rc;
    if (!shared || (reinterpret_cast<uintptr_t>(shared) & 3) || (long long)seqs * tokens * q_heads > kMaxShared) return cudaErrorInvalidValue;
    const float *const q_end = q + (size_t)seqs * tokens * q_heads * a.c.head_dim, *const out_end = out + (q_end - q);
    if (out < q_end && q < out_end) return cudaErrorInvalidValue;  // out holds parts of rows while others' queries are read
    const int rows = seqs * tokens * a.group, d = a.c.head_dim;  // of the prefix
    const bool pair = d == 256 && rows > kRows;
    a.copies = 1;
    // The tensor cores cut off what does not fit when they add to S: two planes of d/16 steps each take half a unit in the last
    // place, 0.72 * 2^-24 on average over the mantissas, of a running sum that is half of the final one on average (both of random
    // keys and queries; sums that cancel lose less). So their scores are too small by d/16 * 0.72 * 2^-24, which their scale makes
    // up for (24/2 heads of 256, 8,192 shared: errors against 64 bits 1.8e-6 -> 0.95e-6; 16/4 of 64 0.58 -> 0.39e-6). Scores that
    // attend_tokens adds up lose nothing and have the scale as it is.
    a.tile_scale = (float)((double)a.scale * (1.0 + d / 16 * 0.72 / 16777216.0));
    tiles(a, rows, pair);
    a.shared = shared;
    a.all_tiles = (rows + a.tile_rows - 1) / a.tile_rows;
    const int held = part_rows(seqs * tokens, a.group);
    const size_t heads = ((size_t)seqs * tokens * q_heads + 1) & ~(size_t)1;
    a.part_acc = reinterpret_cast<float *>(static_cast<char *>(workspace) + 256 + ml_bytes(held));
    a.prefix_acc = a.part_acc + (size_t)2 * kMaxCtas * held * d;
    a.prefix_ml = reinterpret_cast<float2 *>(a.prefix_acc + heads * d);
    a.own_ml = a.prefix_ml + heads;
    a.starts = reinterpret_cast<long long *>(a.own_ml + heads);
    a.lengths = reinterpret_cast<int *>(a.starts + kMaxSeqs + 2);
    CUtensorMap k_map, v_map;
    if (int rc = maps(a, pair, k_map, v_map)) return rc;
    a.own_part_acc = a.part_acc;
    a.own_part_ml = a.part_ml;
    a.own_part_rows = a.part_rows;
    // One token, at most four heads to a key head of up to 128 values: as without a prefix, the sequences' own keys need no
    // tensor cores.
    const bool few = tokens == 1 && a.group <= kFewRows && d <= 128;
    if (few) {
        a.own_part_ml = reinterpret_cast<float2 *>(a.lengths + kMaxSeqs + 4);
        a.own_part_acc = reinterpret_cast<float *>(a.own_part_ml + kFewParts);
        a.own_part_rows = kFewRows;
    }
    if (few && d == 64)
        return launch<64, true>(a, shared_token_kernel<64>, 1, kThreads, Cfg<64, 128, false>::kSmem, a, k_map, v_map);
    if (few)
        return launch<128, true>(a, shared_token_kernel<128>, 1, kThreads, Cfg<128, 128, false>::kSmem, a, k_map, v_map);
    if (d == 64) return launch_tiles<64, 128, false, true>(a, k_map, v_map);
    if (d == 128) return launch_tiles<128, 128, false, true>(a, k_map, v_map);
    if (pair) return launch_tiles<256, 128, true, true>(a, k_map, v_map);
    return rows <= 64 ? launch_tiles<256, 64, false, true>(a, k_map, v_map) : launch_tiles<256, 128, false, true>(a, k_map, v_map);
}

// Decode attention over blocks that a group of sequences shares: every member's queries against the group's shared
// keys and values, which are read once for the group instead of once per sequence.
//
// For one kv head, a group of m sequences with g query heads each has m * g query rows over the same keys, so what is a
// matrix-vector product per sequence becomes a matrix product, S = Q K^T and O = P V, for the tensor cores:
//   read  2 * P * head_dim * 2 bytes of K and V per kv head (P shared tokens),
//   compute 4 * m * g * P * head_dim flops (half as many again for the rests of P, below).
// Up to about 170 rows the bytes take longer than these products at the rates of a copy and of a large matrix product
// (256 without the rests); beyond, the tensor cores and the exponentials bound it.
//
// Three launches.  prefix_kernel attends over the shared blocks, own_kernel over each sequence's own blocks, beside it
// on what it leaves of an SM; both leave partial results, which join_kernel joins.
//
// prefix_kernel: one CTA per SM takes an even share of the step's units -- a unit is one tile of 128 keys for one
// (group, kv head, pair of row tiles), of fewer where the blocks' size shares no factor of 8 with it: as many whole
// blocks as fit, copied one by one (16 groups with blocks of 5 tokens: 55 us, of 16 tokens 51; by whole contexts 916)
// -- regardless of where groups and heads begin and end.  A row tile is as many whole members as fit 128 rows
// (tcgen05's M).  Two warpgroups of softmax, one per accumulator pair in TMEM, take turns with the tensor cores: while
// one exponentiates its scores, the MMAs of the other run.  Exponentiating at the same time gains nothing: with two
// score buffers of 64 keys each, which keep both at it, 256 sequences over 16384 tokens took 176 us instead of 148;
// with a quarter of the exponentials as a polynomial on the FMA pipe 150 (all three with P in one 16-bit number).
//   two row tiles:  the warpgroups take one tile each and every key tile; K and V are read once for 256 rows.
//   one row tile:   both warpgroups take the same rows, one the even, the other the odd key tiles, so that the wait for
//                   a tile's exponentials is covered by the other tile; they leave two partial results.
// Scores S and accumulators O live in TMEM (S0, S1 at columns 0 and 128, O0, O1 at 256 and 256 + head_dim); the
// probabilities P overwrite S as 16-bit numbers and are the A operand of the second product straight from TMEM.  A
// thread owns one row: the running maximum and sum need no exchange.  O is rescaled only when a row's maximum has grown
// by more than 2^3 (fp16) or 2^8 (bf16) since its last rescaling: P, O and the sum have one scale, so nothing is lost.
// P is kept as a part and a rest of the pools' 16-bit type each, as the own parts and the decode attention keep it: the
// two products with V hold 16 (bf16) or 22 (fp16) bits of each weight, and the output's only rounding that counts is
// its own.  With one 16-bit number each the weights' roundings were as large as a bf16 output's (1.66e-3 against 64
// bits became 2.3e-3, relative to all outputs' size 1e-4 became 2.5e-3), and an fp32 output held no more.  It costs
// half of the tensor cores' work on top: 16 groups 46.9 -> 51.9 us, 512 samples 71.2 -> 78.7, 256 over 16384 154.9 ->
// 186.4, 4 beams the same.
//
// Measured, 32 query and 8 kv heads of 128, bf16: a pair of row tiles takes 5260 clocks per key tile, of which the
// matrix products are 3070 (3750 and 2050 with P in one 16-bit number); starting (groups, table, first tiles) takes
// 12000 clocks, writing the partial results 5000 to 8000.  512 sequences over 2048 shared tokens and up to 100 own
// ones: 79 us (prefix_kernel alone 49, the own parts alone 31, joining 13, each with cold caches); 256 over 16384, up
// to 512 own: 172 us (119, 63, 12); 4 beams over 2048, 24 own: 18 us.
// prefix_kernel leaves shared memory unused on purpose: with 224 KB instead of 192 the L1, which the own parts' loads
// go through, shrinks to 28 KB, and the first two calls took 85 and 174 us where they took 72 and 149.
// The own parts are cut alike, into at most 8 each: a long one beside many short ones, or few long ones, are slower
// than by kvp_paged_attention, whose partition follows the lengths (2 sequences of 30000 own tokens: 320 us against
// 105; 255 of 100 beside one of 30000: 1227 against 96; 64 of 8192 over 2048 shared ones: 400 against 363).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "attention_common.h"
#include "kvp_device.cuh"

namespace kvpd {

constexpr int kKeys = 128;         // keys per tile
constexpr int kRows = 128;         // rows per tile: M of the MMA
constexpr int kPrefixThreads = 352;  // 8 softmax warps, the MMA warp, the warps that load K (and Q) and V
constexpr int kTmemCols = 512;
// Most tokens of a table row: places are 32-bit numbers, and those of the tiles that are looked up ahead lie up to 300
// behind the row's end.
constexpr long long kPrefixTokens = (1LL << 31) - 1024;
// The weight of a row's reference score is represented by 2^kLift: fp16 numbers, a part and its rest, end at 2^-25, and
// of many keys far below the largest one the numerator would lose what the sum of the weights holds.
template <class KV>
constexpr float kLift = std::is_same<KV, __half>::value ? 12.f : 0.f;
constexpr int kPrefixLimit = 512;  // at most 128 registers a thread: five of own_kernel's single warps fit beside a CTA

// What joins a (sequence, kv head): partial rows of query head 0 begin at row0, and 256 further for each CTA before the
// first of the span at pair_at (-1: nothing is shared); `parts` per CTA, `rows` apart.
struct OwnMeta {
    long long row0, pair_at;
    int parts, rows, fine, unused;
};

struct PrefixParams {
    const int32_t* tables;
    const int32_t* lens;
    const int32_t* prefix_blocks;
    const int32_t* group_starts;
    int32_t* status;
    int32_t* unsorted;  // a group starts before the one ahead: they overlap, and nobody's partial rows are their own
    // first and last CTA of each (group, kv head, pair), at its first row's (member, kv head)
    int2* spans;
    float2* part_ml;           // partial rows: (maximum in log2 units, sum)
    float* part_o;
    OwnMeta* own_meta;         // of each (sequence, kv head)
    float2* own_ml;            // own parts, own_parts rows per (sequence, query head)
    float* own_o;
    const void* q;
    const void* k_cache;
    const void* v_cache;
    void* out;
    long long num_blocks;
    long long wait_limit;
    int num_seqs, num_groups, nh, kvh, g, max_blocks, B, Bshift, run, runs, oob_row;
    int mt;                    // members per row tile
    int keys;                  // keys that a tile holds: 128, or as many whole blocks as fit
    int own_parts;             // warps that share a (sequence, kv head)'s own tokens
    int bf16, out_dtype, ctas;  // ctas: prefix_kernel's
    float sl2;
};

// ---------------------------------------------------------------- tcgen05
__device__ __forceinline__ void tmem_alloc(uint32_t smem_dst) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst), "n"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t base) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "n"(kTmemCols));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// D (TMEM) = or += A (shared memory) * B (shared memory); operands by the low and high words of their descriptors.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                       uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "mov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n\t}" ::"r"(d),
        "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(static_cast<uint32_t>(add))
        : "memory");
}
// D (TMEM) = or += A (TMEM) * B (shared memory)
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(static_cast<uint32_t>(add))
        : "memory");
}
// 32 columns of this warp's 32 lanes, one row per thread.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// Waits for the loads so far; r: what the last one fills, so that no use of it is moved before the wait.
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15])::"memory");
    asm volatile(""
                 : "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                   "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                   "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One 32-byte sector of global memory.
__device__ __forceinline__ void store_sector(float* p, const uint32_t* v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// Shared-memory operand in the 128-byte swizzle: rows of 64 elements, 8-row atoms of 1024 bytes.
//   along the rows (K-major: Q and K): atoms follow each other at 1024 bytes; a 16-element step is 32 bytes further.
//   across them (MN-major: V, whose rows are the keys the product sums over): atoms of 8 keys at 1024 bytes (stride),
//   64-dim columns at the column tile's size (leading); a 16-key step is 2048 bytes further.
// The low word holds the address (in 16-byte units, so a step is an addition) and the leading distance, the high word
// the stride, the version and the swizzle.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t leading_bytes) {
    return ((addr & 0x3ffffu) >> 4) | ((leading_bytes >> 4) << 16);
}
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
// kind::f16, fp32 accumulator, A and B both bf16 or both fp16; b_mn: B is MN-major.
__device__ __forceinline__ uint32_t mma_desc(int bf16, int n, bool b_mn) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kRows >> 4) << 24);
}

// Scores of keys from `valid` on become -inf.
__device__ __forceinline__ void mask_keys(uint32_t (&s)[32], int valid) {
    if (valid >= 32) return;
#pragma unroll
    for (int i = 0; i < 32; ++i)
        if (i >= valid) s[i] = 0xff800000u;
}

// A row's largest score; its first 32 scores are on their way to s[0] again when it returns.
__device__ __forceinline__ float row_max(uint32_t addr, uint32_t (&s)[2][32], int valid) {
    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    tmem_ld32(addr, s[0]);
#pragma unroll 1
    for (int h = 0; h < 4; h += 2) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            tmem_wait_ld(s[b]);
            tmem_ld32(addr + ((h + b + 1) & 3) * 32, s[b ^ 1]);
            mask_keys(s[b], valid - (h + b) * 32);
#pragma unroll
            for (int e = 0; e < 32; e += 2)
                top[(e >> 1) & 3] = fmaxf(fmaxf(top[(e >> 1) & 3], __uint_as_float(s[b][e])),
                                          __uint_as_float(s[b][e + 1]));
        }
    }
    return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}
__device__ __forceinline__ float exp2_unit(float x) {  // free to be moved, unlike fast_exp2
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// A partial row's maximum and sum as they are left for joining.  Where every score was NaN the maximum, which passes
// over them, is still -inf, the mark of a part without keys: the row has to become NaN, not to go without these keys.
template <class KV>
__device__ __forceinline__ float2 partial(float m, float l) {
    return make_float2(m == -INFINITY && l != l ? 0.f : m - kLift<KV>, l);
}
// ---------------------------------------------------------------- units
// Units of a group: kv heads x pairs of row tiles x key tiles.  A group with a bad range or a bad block count has none.
struct Group {
    int start, members, blocks, pairs, ktiles;
    __device__ __forceinline__ long long units(int kvh) const { return static_cast<long long>(kvh) * pairs * ktiles; }
};
__device__ __forceinline__ Group load_group(const PrefixParams& p, int gi) {
    Group r;
    r.start = __ldg(p.group_starts + gi);
    const int end = __ldg(p.group_starts + gi + 1);
    r.members = 0;
    r.blocks = 0;
    if (r.start >= 0 && end > r.start && end <= p.num_seqs) {
        r.members = end - r.start;
        const int b = __ldg(p.prefix_blocks + r.start);
        if (b > 0 && b <= p.max_blocks) r.blocks = b;
    }
    r.pairs = (r.members + 2 * p.mt - 1) / (2 * p.mt);
    const long long last = static_cast<long long>(r.blocks) * p.B + p.keys - 1;
    r.ktiles = static_cast<int>(p.keys == kKeys ? last / kKeys : last / p.keys);
    return r;
}

__device__ __forceinline__ long long floor_div(long long a, long long b, long long c) {  // a * b / c, a * b < 2^53
    const long long n = a * b;
    long long q = static_cast<long long>(static_cast<double>(n) / static_cast<double>(c));
    if (q * c > n) --q;
    else if ((q + 1) * c <= n) ++q;
    return q;
}
// CTA c of G owns units [c T / G, (c + 1) T / G).
__device__ __forceinline__ long long first_unit(int c, long long T, int G) {
    // c <= 1023
    if (T < (1 << 22)) return static_cast<unsigned>(c) * static_cast<unsigned>(T) / static_cast<unsigned>(G);
    return floor_div(c, T, G);
}

// One stretch of a CTA's units: key tiles [k0, k0 + n) of (group, kv head, pair).
struct Work {
    int start, head, member0, k0, n, ktiles, tokens;  // member0: the pair's first member, within the group
    int rows0, rows1;                         // rows of the two row tiles; rows1 == 0: one row tile, key tiles in turn
    long long pair_at;   // the pair's place among all (member, kv head) rows of the batch
    long long part_row;
};

struct WorkList {
    Group grp;
    long long first, t, end;  // the group's first unit, the next unit, the CTA's last
    int gi, cta;
    __device__ __forceinline__ bool next(const PrefixParams& p, Work& w) {
        if (t >= end) return false;
        while (t >= first + grp.units(p.kvh)) {
            first += grp.units(p.kvh);
            grp = load_group(p, ++gi);
        }
        const long long rel = t - first;
        const int triple = static_cast<int>(
            rel < (1LL << 32) ? static_cast<unsigned>(rel) / static_cast<unsigned>(grp.ktiles) : rel / grp.ktiles);
        w.k0 = static_cast<int>(rel - static_cast<long long>(triple) * grp.ktiles);
        w.n = static_cast<int>(min(static_cast<long long>(grp.ktiles - w.k0), end - t));
        t += w.n;
        w.start = grp.start;
        w.head = triple / grp.pairs;
        w.member0 = (triple - w.head * grp.pairs) * 2 * p.mt;
        w.ktiles = grp.ktiles;
        w.tokens = grp.blocks * p.B;
        const int left = grp.members - w.member0;
        w.rows0 = min(left, p.mt) * p.g;
        w.rows1 = min(max(left - p.mt, 0), p.mt) * p.g;
        // two partial rows per (member, head) row of the batch, 256 more per CTA: a stretch's rows are its own
        w.pair_at = static_cast<long long>(grp.start) * p.kvh + static_cast<long long>(w.head) * grp.members +
            w.member0;
        w.part_row = 2LL * p.g * w.pair_at + static_cast<long long>(cta) * 2 * kRows;
        return true;
    }
};

// Where a CTA's units begin: the total, the group that holds the CTA's first unit and that group's first unit.
struct Start {
    long long total, first;
    int group;
    bool unsorted;  // nothing is done then
};
// Up to 32 groups: every warp by itself, a lane per group.
__device__ __forceinline__ Start find_start_few(const PrefixParams& p, Group* grp) {
    const int lane = threadIdx.x & 31;
    const Group mine = lane < p.num_groups ? load_group(p, lane) : Group{0, 0, 0, 0, 0};
    const long long u = mine.units(p.kvh);
    long long x = u;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, off);
        if (lane >= off) x += y;
    }
    Start s{__shfl_sync(0xffffffffu, x, 31), 0, 0, false};
    const int next = __shfl_down_sync(0xffffffffu, mine.start, 1);
    if (__any_sync(0xffffffffu, lane + 1 < p.num_groups && next < mine.start)) return Start{0, 0, 0, true};
    const int G = static_cast<int>(min(static_cast<long long>(gridDim.x), s.total));
    if (static_cast<int>(blockIdx.x) >= G) return s;
    const long long at = first_unit(blockIdx.x, s.total, G);
    s.group = __ffs(__ballot_sync(0xffffffffu, x - u <= at && at < x)) - 1;
    s.first = __shfl_sync(0xffffffffu, x - u, s.group);
    grp->start = __shfl_sync(0xffffffffu, mine.start, s.group);
    grp->members = __shfl_sync(0xffffffffu, mine.members, s.group);
    grp->blocks = __shfl_sync(0xffffffffu, mine.blocks, s.group);
    grp->pairs = __shfl_sync(0xffffffffu, mine.pairs, s.group);
    grp->ktiles = __shfl_sync(0xffffffffu, mine.ktiles, s.group);
    return s;
}
// More: the CTA together, a thread per group and kPrefixThreads groups at a time.
__device__ __forceinline__ Start find_start(const PrefixParams& p, long long* warp_sum, Start* found, Group* grp) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // all of a chunk; *mine: what lies before this thread
    auto scan = [&](long long u, long long carry, long long* mine) {
        long long x = u;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, off);
            if (lane >= off) x += y;
        }
        if (lane == 31) warp_sum[warp] = x;
        __syncthreads();
        long long before = carry, all = 0;
        for (int w = 0; w < kPrefixThreads / 32; ++w) {
            const long long s = warp_sum[w];
            if (w < warp) before += s;
            all += s;
        }
        *mine = before + x - u;
        __syncthreads();
        return all;
    };
    auto units_of = [&](int gi) { return gi < p.num_groups ? load_group(p, gi).units(p.kvh) : 0ll; };
    bool back = false;
    for (int gi = static_cast<int>(threadIdx.x); gi + 1 < p.num_groups; gi += kPrefixThreads)
        back = back || __ldg(p.group_starts + gi + 1) < __ldg(p.group_starts + gi);
    if (__syncthreads_or(back)) return Start{0, 0, 0, true};
    long long total = 0, mine = 0;
    for (int g0 = 0; g0 < p.num_groups; g0 += kPrefixThreads)
        total += scan(units_of(g0 + static_cast<int>(threadIdx.x)), total, &mine);
    const int G = static_cast<int>(min(static_cast<long long>(gridDim.x), total));
    if (static_cast<int>(blockIdx.x) >= G) return Start{total, 0, 0, false};
    const long long at = first_unit(blockIdx.x, total, G);
    long long carry = 0;
    for (int g0 = 0; g0 < p.num_groups; g0 += kPrefixThreads) {
        const int gi = g0 + static_cast<int>(threadIdx.x);
        const long long u = units_of(gi);
        carry += scan(u, carry, &mine);
        if (u > 0 && mine <= at && at < mine + u) *found = Start{total, mine, gi, false};
    }
    __syncthreads();
    *grp = load_group(p, found->group);
    return *found;
}

// ---------------------------------------------------------------- the kernel
struct PrefixShared {
    uint64_t full[2][8], empty[2][8];  // the rings' slots: K, V
    uint64_t q_full, q_free, s_full[2], p_full[2][2], o_full[2], drain;  // p_full: P's first and second 64 keys
    uint32_t tmem;
    int abort;
    Start found;
    long long warp_sum[kPrefixThreads / 32];
};

// Bounded wait that also ends once another role of the CTA gave up.
__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, const PrefixParams& p, PrefixShared& sh) {
    const uint32_t b = smem_u32(bar);
    if (mbar_try_wait(b, parity)) return true;
    const long long t0 = clock64();
    while (true) {
        for (int i = 0; i < 32; ++i)
            if (mbar_try_wait(b, parity)) return true;
        if (*reinterpret_cast<volatile int*>(&sh.abort)) return false;
        if (clock64() - t0 > p.wait_limit) {
            report(p.status, KVP_STATUS_TIMEOUT);
            *reinterpret_cast<volatile int*>(&sh.abort) = 1;
            return false;
        }
    }
}

// The same for a whole warp, with one answer for all lanes.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const PrefixParams& p, PrefixShared& sh) {
    return __all_sync(0xffffffffu, wait_or_abort(bar, parity, p, sh));
}

// A place in the ring of tiles: its slot and the parity of the slot's current use.
struct Cursor {
    int slot;
    uint32_t parity;
    __device__ __forceinline__ Cursor next(int slots) const {
        return slot + 1 == slots ? Cursor{0, parity ^ 1u} : Cursor{slot + 1, parity};
    }
};

template <int D, class KV>
__global__ void __launch_bounds__(kPrefixLimit, 1)
    prefix_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                  const __grid_constant__ CUtensorMap vmap, const PrefixParams p) {
    using Tr = F16Traits<KV>;
    constexpr int NCH = D / 64;                      // 64-element columns of a head
    constexpr uint32_t kCol = kKeys * 128;           // bytes of one such column of a tile
    constexpr uint32_t kTile = NCH * kCol;           // one tile of Q, K or V
    constexpr uint32_t kO = 256;                     // TMEM column of the first accumulator
    // How far (log2) a score may exceed the maximum that P, O and the sum refer to: P, which starts at 2^kLift, has to
    // stay below the type's largest value, and O below fp32's, which a bf16 V may come near to by itself (with 2^40
    // values of 2^88 became infinite).
    constexpr float kFar = std::is_same<KV, __half>::value ? 3.f : 8.f;
    __shared__ PrefixShared sh;
    extern __shared__ uint8_t dyn[];
    const uint32_t base = (smem_u32(dyn) + 1023u) & ~1023u;
    // Slots of K and of V, beside two query tiles: 192 KB in all at head_dim 128, 144 KB at 64.
    constexpr int kSlotsK = D == 128 ? 2 : 4, kSlotsV = D == 128 ? 2 : 3;
    const uint32_t ring_k = base + 2 * kTile, ring_v = ring_k + kSlotsK * kTile;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        sh.abort = 0;
        for (int s = 0; s < 8; ++s) {
            mbar_init(smem_u32(&sh.full[0][s]), 1);
            mbar_init(smem_u32(&sh.empty[0][s]), 1);
            mbar_init(smem_u32(&sh.full[1][s]), 1);
            mbar_init(smem_u32(&sh.empty[1][s]), 1);
        }
        mbar_init(smem_u32(&sh.q_full), 1);
        mbar_init(smem_u32(&sh.q_free), 1);
        for (int t = 0; t < 2; ++t) {
            mbar_init(smem_u32(&sh.s_full[t]), 1);
            mbar_init(smem_u32(&sh.p_full[t][0]), 4);
            mbar_init(smem_u32(&sh.p_full[t][1]), 4);
            mbar_init(smem_u32(&sh.o_full[t]), 1);
        }
        mbar_init(smem_u32(&sh.drain), 1);
        fence_barrier_init();
    }
    if (warp == 10 && lane == 0) {
        prefetch_tensormap(&qmap);
        prefetch_tensormap(&kmap);
        prefetch_tensormap(&vmap);
    }
    // Nothing is read or written before the kernels ahead are done, and no tensor memory is held while waiting for
    // them.  The kernels behind start only once every CTA here has its own: one of them that takes tensor memory while
    // it waits for this kernel could otherwise keep it from ever getting any.
    griddep_wait();
    if (p.keys < kKeys) {  // rows of V that no copy fills: their weights are zero, and so have they to be
        const int words = (kKeys - p.keys) * 8;  // of 16 bytes
        for (int i = threadIdx.x; i < words * NCH * kSlotsV; i += kPrefixThreads) {
            const uint32_t to = ring_v + (i / words) * kCol + p.keys * 128 + (i % words) * 16;
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(to), "r"(0) : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 8) {
        tmem_alloc(smem_u32(&sh.tmem));
        griddep_launch_dependents();
    }
    WorkList list;
    const Start from =
        p.num_groups <= 32 ? find_start_few(p, &list.grp) : find_start(p, sh.warp_sum, &sh.found, &list.grp);
    const int cta = blockIdx.x, G = static_cast<int>(min(static_cast<long long>(gridDim.x), from.total));
    if (cta == 0 && threadIdx.x == 0) {
        *p.unsorted = from.unsorted;
        if (from.unsorted) report(p.status, KVP_STATUS_BAD_LEN);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (cta >= G) {  // more CTAs than units
        if (warp == 8) tmem_free(sh.tmem);
        return;
    }
    list.cta = cta;
    list.t = first_unit(cta, from.total, G);
    list.end = first_unit(cta + 1, from.total, G);
    list.gi = from.group;
    list.first = from.first;
    const uint32_t tmem = sh.tmem;
    Work w;

    if (warp >= 9) {
        // ------------------------------------------------------------ loads: K and the queries, and V
        // Each lane issues one copy (a run of tokens within a block, 64 dims); the copies of a warp's lanes are issued
        // one after the other, at about 60 clocks each, which is why K and V have a warp each.
        const int v = warp - 9, slots = v ? kSlotsV : kSlotsK;
        const uint32_t ring = v ? ring_v : ring_k;
        const CUtensorMap* map = v ? &vmap : &kmap;
        bool ok = true;
        Cursor at{0, 0u};
        int loaded = 0, queries = 0;  // tiles and query loads issued
        while (ok && list.next(p, w)) {
            const int32_t* trow = p.tables + static_cast<long long>(w.start) * p.max_blocks;
            // The pool row of a run of a tile; for the runs of a lane's own, looked up a tile ahead, so that the
            // table's latency is past when it is needed.
            const int run = lane / NCH, c = lane - run * NCH;
            auto row_at = [&](int kt, int run) {
                const int tok = kt * p.keys + run * p.run;
                // zeros behind the shared tokens
                if (run >= p.runs || tok >= w.tokens || kt >= w.k0 + w.n) return p.oob_row;
                const int bi = p.Bshift >= 0 ? tok >> p.Bshift : tok / p.B;
                const int blk = __ldg(trow + bi);
                if (blk >= 0 && blk < p.num_blocks) return blk * p.B + (tok - bi * p.B);
                report(p.status, KVP_STATUS_BAD_BLOCK);
                return p.oob_row;
            };
            auto row_of = [&](int kt) { return row_at(kt, run); };
            int row = row_of(w.k0);
            if (v == 0) {  // queries, once the previous stretch's products have read theirs
                if (queries > 0) ok = warp_wait(&sh.q_free, (queries - 1) & 1, p, sh);
                if (!ok) break;
                ++queries;
                if (lane == 0) {
                    const uint32_t bar = smem_u32(&sh.q_full);
                    const int tiles = w.rows1 ? 2 : 1;
                    mbar_arrive_expect_tx(bar, static_cast<uint32_t>(tiles * NCH * p.mt * p.g) * 128u);
                    for (int t = 0; t < tiles; ++t)
                        for (int k = 0; k < NCH; ++k)
                            tma_load_3d(base + t * kTile + k * kCol, &qmap, bar, k * 64, w.head * p.g,
                                        w.start + w.member0 + t * p.mt);
                }
                __syncwarp();
            }
            for (int j = 0; ok && j < w.n; ++j) {
                const int next_row = row_of(w.k0 + j + 1);
                if (loaded >= slots && !(ok = warp_wait(&sh.empty[v][at.slot], at.parity ^ 1u, p, sh))) break;
                const uint32_t bar = smem_u32(&sh.full[v][at.slot]);
                if (lane == 0) mbar_arrive_expect_tx(bar, static_cast<uint32_t>(p.keys) * NCH * 128u);
                __syncwarp();
                if (run < p.runs)
                    tma_load_3d(ring + at.slot * kTile + c * kCol + static_cast<uint32_t>(run * p.run) * 128u, map, bar,
                                c * 64, w.head, row);
                for (int i = 32 + lane; i < p.runs * NCH; i += 32)  // small blocks: more runs than lanes
                    tma_load_3d(ring + at.slot * kTile + (i % NCH) * kCol +
                                static_cast<uint32_t>(i / NCH * p.run) * 128u, map, bar,
                                i % NCH * 64, w.head, row_at(w.k0 + j, i / NCH));
                row = next_row;
                at = at.next(slots);
                ++loaded;
            }
        }
        // Nothing may be in flight into this CTA's shared memory when it ends: all is consumed, unless a wait gave up.
        if ((!ok || *reinterpret_cast<volatile int*>(&sh.abort)) && lane == 0) {
            for (int s = 0; s < slots; ++s) {
                const int n = loaded > s ? (loaded - s - 1) / slots + 1 : 0;  // tiles loaded into slot s
                if (n > 0) mbar_wait(smem_u32(&sh.full[v][s]), static_cast<uint32_t>((n - 1) & 1), p.wait_limit);
            }
            if (queries > 0) mbar_wait(smem_u32(&sh.q_full), static_cast<uint32_t>((queries - 1) & 1), p.wait_limit);
        }
        __syncwarp();
    } else if (warp == 8) {
        // ------------------------------------------------------------ MMAs, one thread
        // One thread for both warpgroups keeps their products one after the other, and with them the turns of the
        // warpgroups: issued by two threads the products of both ran side by side, both softmaxes waited for them and
        // then ran at the same time, 4950 clocks for a pair of tiles.
        if (lane == 0) {
            const uint32_t qk_desc = mma_desc(p.bf16, kKeys, false);
            const uint32_t pv_desc = mma_desc(p.bf16, D, true);
            bool ok = true;
            Cursor kat{0, 0u}, vat{0, 0u};
            // parities of the next queries and of the next P tile of each warpgroup
            uint32_t seg = 0, turn0 = 0, turn1 = 0;
            const uint32_t q_lo = desc_lo(base, 16), k_lo = desc_lo(ring_k, 16), v_lo = desc_lo(ring_v, kCol);
            auto qk = [&](int t, int qt, int slot) {
                const uint32_t q = q_lo + qt * (kTile >> 4), k = k_lo + static_cast<uint32_t>(slot) * (kTile >> 4);
#pragma unroll
                for (int c = 0; c < NCH; ++c)
#pragma unroll
                    for (int s = 0; s < 4; ++s)
                        mma_ss(tmem + t * kKeys, q + ((c * kCol + s * 32) >> 4), kDescHi,
                               k + ((c * kCol + s * 32) >> 4), kDescHi,
                               qk_desc, c + s > 0);
                tc_commit(smem_u32(&sh.s_full[t]));
            };
            auto wait_k = [&] { return wait_or_abort(&sh.full[0][kat.slot], kat.parity, p, sh); };
            auto done_k = [&] {
                tc_commit(smem_u32(&sh.empty[0][kat.slot]));
                kat = kat.next(kSlotsK);
            };
            while (ok && list.next(p, w)) {
                const bool two = w.rows1 > 0;
                const int ahead = two ? 1 : 2;
                ok = wait_or_abort(&sh.q_full, seg & 1, p, sh);
                for (int i = 0; ok && i < min(ahead, w.n); ++i) {
                    if (!(ok = wait_k())) break;
                    tc_fence_after();
                    for (int t = two ? 0 : i; t <= (two ? 1 : i); ++t) qk(t, two ? t : 0, kat.slot);
                    done_k();
                }
                for (int j = 0; ok && j < w.n; ++j) {
                    const bool more = j + ahead < w.n;
                    if (!(ok = wait_or_abort(&sh.full[1][vat.slot], vat.parity, p, sh))) break;
                    for (int t = two ? 0 : j & 1; t <= (two ? 1 : j & 1); ++t) {
                        const uint32_t turn = (t ? turn1 : turn0) & 1;
                        if (t) ++turn1; else ++turn0;
                        const uint32_t v = v_lo + static_cast<uint32_t>(vat.slot) * (kTile >> 4);
                        const bool add = j >= ahead;
#pragma unroll
                        for (int half = 0; half < 2; ++half) {  // the first half runs while the second's P is computed
                            if (ok) ok = wait_or_abort(&sh.p_full[t][half], turn, p, sh);
                            if (!ok) break;
                            tc_fence_after();
#pragma unroll
                            for (int s = half * 4; s < half * 4 + 4; ++s) {
                                const uint32_t at = tmem + t * kKeys + s * 16;
                                mma_ts(tmem + kO + t * D, at, v + s * (2048 >> 4), kDescHi, pv_desc, add || s > 0);
                                mma_ts(tmem + kO + t * D, at + 8, v + s * (2048 >> 4), kDescHi, pv_desc, true);
                            }
                        }
                        if (!ok) break;
                        if (more) {
                            if (!(ok = wait_k())) break;
                            qk(t, two ? t : 0, kat.slot);
                        }
                    }
                    if (!ok) break;
                    tc_commit(smem_u32(&sh.empty[1][vat.slot]));
                    vat = vat.next(kSlotsV);
                    if (more) done_k();
                }
                if (ok) {
                    // Only to a warpgroup that has a tile here: its own P gates the next stretch's products, so this
                    // barrier never completes twice before it has looked.  One without a tile would be gated by
                    // nothing.
                    tc_commit(smem_u32(&sh.o_full[0]));
                    if (two || w.n > 1) tc_commit(smem_u32(&sh.o_full[1]));
                    tc_commit(smem_u32(&sh.q_free));
                }
                ++seg;
            }
            // every MMA has to be done before the accumulators and the shared memory are given up
            tc_commit(smem_u32(&sh.drain));
            if (!mbar_wait(smem_u32(&sh.drain), 0, p.wait_limit)) report(p.status, KVP_STATUS_TIMEOUT);
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------ softmax: warpgroup t, one row per thread
        const int t = warp >> 2;
        const int row = threadIdx.x & 127;
        const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // 32 lanes per warp, in bits 16 and up
        const uint32_t s_addr = tmem + lanes + t * kKeys, o_addr = tmem + lanes + kO + t * D;
        bool ok = true;
        int uses = 0, seg = 0;  // tiles, and stretches in which this warpgroup has some
        while (ok && list.next(p, w)) {
            const bool two = w.rows1 > 0;
            const int rows = two && t ? w.rows1 : w.rows0;
            const bool busy = (warp & 3) * 32 < rows;  // else this warp's lanes hold no row: it only keeps step
            float m = -INFINITY, l = 0.f;              // maximum (scaled, log2) the accumulator refers to, sum
            const int j0 = two ? 0 : t, dj = two ? 1 : 2;
            for (int j = j0; j < w.n; j += dj) {
                if (!(ok = warp_wait(&sh.s_full[t], uses & 1, p, sh))) break;
                ++uses;
                if (busy) {
                    tc_fence_after();
                    const int valid = min(w.tokens - (w.k0 + j) * p.keys, p.keys);
                    // The row's maximum, then the exponentials, the scores read twice and 32 at a time: loops, not one
                    // long stretch of code, whose way through the instruction caches cost a launch 10 us.
                    uint32_t s[2][32];
                    const float mx = row_max(s_addr, s, valid) * p.sl2;
                    if (j == j0) {
                        m = mx;  // the first product overwrites the accumulator
                    } else if (__any_sync(0xffffffffu, mx > m + kFar)) {
                        const float mn = fmaxf(m, mx), f = mn == -INFINITY ? 1.f : fast_exp2(m - mn);
                        m = mn;
                        l *= f;
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            tmem_ld32(o_addr + c, s[1]);
                            tmem_wait_ld(s[1]);
#pragma unroll
                            for (int i = 0; i < 32; ++i) s[1][i] = __float_as_uint(__uint_as_float(s[1][i]) * f);
                            tmem_st32(o_addr + c, s[1]);
                        }
                    }
                    const float ref = (m == -INFINITY ? 0.f : m) - kLift<KV>;
                    const uint64_t scale2 = pack2(p.sl2, p.sl2), ref2 = pack2(-ref, -ref);
                    uint64_t sum[2] = {0ull, 0ull};
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) {
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            // P takes the place of scores that are in registers: of each 16 keys 8 columns of 16-bit
                            // parts, then 8 of the rests
                            const int h = half * 2 + b;
                            tmem_wait_ld(s[b]);
                            if (h < 3) tmem_ld32(s_addr + (h + 1) * 32, s[b ^ 1]);
                            mask_keys(s[b], valid - h * 32);
#pragma unroll
                            for (int k = 0; k < 32; k += 16) {
                                uint32_t pk[16];
#pragma unroll
                                for (int i = 0; i < 8; ++i) {
                                    const float2 x = unpack2(fma2(
                                        pack2(__uint_as_float(s[b][k + 2 * i]), __uint_as_float(s[b][k + 2 * i + 1])),
                                            scale2, ref2));
                                    const float2 e = make_float2(exp2_unit(x.x), exp2_unit(x.y));
                                    sum[i & 1] = add2(sum[i & 1], pack2(e.x, e.y));
                                    pk[i] = Tr::pack(e.x, e.y);
                                    pk[8 + i] = Tr::pack(e.x - Tr::unpack_lo(pk[i]), e.y - Tr::unpack_hi(pk[i]));
                                }
                                tmem_st16(s_addr + h * 32 + k, pk);
                            }
                        }
                        tmem_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[t][half]));
                    }
                    const float2 both = unpack2(add2(sum[0], sum[1]));
                    l += both.x + both.y;
                } else if (lane == 0) {
                    mbar_arrive(smem_u32(&sh.p_full[t][0]));
                    mbar_arrive(smem_u32(&sh.p_full[t][1]));
                }
                __syncwarp();
            }
            if (!ok) break;
            const bool some = two || t < w.n;
            if (some) {
                if (!(ok = warp_wait(&sh.o_full[t], seg & 1, p, sh))) break;
                ++seg;
            }
            if (threadIdx.x == 0) {
                if (w.k0 == 0) p.spans[w.pair_at].x = cta;
                if (w.k0 + w.n == w.ktiles) p.spans[w.pair_at].y = cta;
            }
            if (busy) {
                tc_fence_after();
                const long long r0 = w.part_row + (t ? w.rows0 : 0) + row;
                if (row < rows) p.part_ml[r0] = partial<KV>(m, l);
                if (some) {
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        uint32_t o[32];
                        tmem_ld32(o_addr + c, o);
                        tmem_wait_ld(o);
                        if (row < rows) {
#pragma unroll
                            for (int i = 0; i < 32; i += 8) store_sector(p.part_o + r0 * D + c + i, o + i);
                        }
                    }
                }
                tc_fence_before();
            }
            __syncwarp();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_free(tmem);
    }
}

// ---------------------------------------------------------------- own parts
// 1 to 8 single warps, which wait for nothing from each other, share the own tokens of a (sequence, kv head), 16 at a
// time.  Bound by HBM, and by latency where the own parts are short, which most of them are: a warp takes K and V from
// global memory straight into the registers of its matrix instructions, without a pipeline to fill and drain.  Alone it
// takes 20 us at 512 sequences with up to 100 own tokens, 44 us at 256 with up to 512 (6.5 TB/s), 31 and 63 with cold
// caches.  CTAs of four warps that also joined their results with the shared part's took 42 and 71 us; clusters of
// eight such CTAs, where pairs are few, 19.2 us for the whole call at 4 beams instead of 16.2.
//   S^T[tokens x heads] = K Q^T:  a lane holds 8 neighbouring dims of a token's K (one 16-byte load); the sum over dims
//                                 does not care for their order, so these are the dims of two steps, for K and Q alike.
//   O^T[dims x heads] += V^T P^T: a lane holds 8 neighbouring dims of four tokens' V and pairs up two tokens' halves;
//                                 the rows of the instruction are dims in an order of their own.  P^T by an 8 x 8
//                                 transposition.
// The heads are the 8 columns of the instruction (NT times, for more than 8): as its 16 rows they took twice the
// instructions and accumulators, and twice the time at head_dim 128.  With more than 8 heads per kv head and head_dim
// 128 the kernel spills 140 bytes of registers, else at most 16; ten warps an SM, which need no spills, took 116 us
// instead of 113 (256 sequences, 64 query and 4 kv heads, 256 shared and 512 own tokens).

// Four partial results (maximum, sum; four columns of the output) at a time, folded into what there is.  One with the
// maximum -inf is nothing, and its columns may never have been written.
struct Fold {
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    __device__ __forceinline__ void add(const float2 (&ml)[4], const float4 (&x)[4]) {
        const float mn = fmaxf(fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), m);
        if (mn == -INFINITY) return;
        const float f = fast_exp2(m - mn);
        m = mn;
        l *= f;
        o.x *= f;
        o.y *= f;
        o.z *= f;
        o.w *= f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool some = ml[i].x != -INFINITY;
            const float w = fast_exp2(ml[i].x - mn);
            l += ml[i].y * w;
            o.x += some ? x[i].x * w : 0.f;
            o.y += some ? x[i].y * w : 0.f;
            o.z += some ? x[i].z * w : 0.f;
            o.w += some ? x[i].w * w : 0.f;
        }
    }
};

__device__ __forceinline__ void store_out(const PrefixParams& p, size_t at, const float4& o, float inv) {
    const float y[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    if (p.out_dtype == KVP_DTYPE_F32)
        *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = make_float4(y[0], y[1], y[2], y[3]);
    else
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) =
            p.out_dtype == KVP_DTYPE_F16 ? make_uint2(F16Traits<__half>::pack(y[0], y[1]),
                                                      F16Traits<__half>::pack(y[2], y[3]))
                                         : make_uint2(F16Traits<__nv_bfloat16>::pack(y[0], y[1]),
                                                      F16Traits<__nv_bfloat16>::pack(y[2], y[3]));
}

// Partial rows k0 .. k0 + 3 of the `count` that the shared part left of a query head.
struct SharedParts {
    long long row0 = 0;
    int count = 0, parts = 1, rows = 0;
    __device__ __forceinline__ void load(const PrefixParams& p, int j, int D, int col, int k0, float2 (&ml)[4],
                                         float4 (&x)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = k0 + i;
            const long long r = row0 + j + (parts == 2 ? static_cast<long long>(k >> 1) * 2 * kRows + (k & 1) * rows
                                                       : static_cast<long long>(k) * 2 * kRows);
            ml[i] = k < count ? __ldcg(&p.part_ml[r]) : make_float2(-INFINITY, 0.f);
            x[i] = k < count ? __ldcg(reinterpret_cast<const float4*>(p.part_o + r * D + col))
                : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
};

__device__ __forceinline__ SharedParts shared_parts(const PrefixParams& p, const OwnMeta& m) {
    SharedParts s;
    if (m.pair_at < 0) return s;
    const int2 span = __ldcg(p.spans + m.pair_at);
    const int first = min(max(span.x, 0), p.ctas - 1);  // (a wait that ran out may have left them unwritten)
    s.row0 = m.row0 + static_cast<long long>(first) * 2 * kRows;
    s.count = (min(max(span.y, first), p.ctas - 1) - first + 1) * m.parts;
    s.parts = m.parts;
    s.rows = m.rows;
    return s;
}

// NT: groups of 8 query heads per kv head.  Its inputs were written before prefix_kernel, which lets this kernel start
// once it has waited for the kernels ahead; so nothing is waited for, but for the last CTA, through which join_kernel
// waits for the shared part.
template <int D, class KV, int NT>
__global__ void __launch_bounds__(32, NT == 1 ? 16 : 12) own_kernel(const PrefixParams p) {
    using Tr = F16Traits<KV>;
    constexpr int NI = D / 32;   // 16-byte pieces of a row that a lane of four holds
    constexpr int NH = D / 64;   // and that a lane of eight holds
    griddep_launch_dependents();
    const int lane = threadIdx.x, gid = lane >> 2, c4 = lane & 3;
    const int item = static_cast<int>(blockIdx.x) / p.own_parts,
        rank = static_cast<int>(blockIdx.x) - item * p.own_parts;
    const int seq = item / p.kvh, h = item - seq * p.kvh;
    const int len = __ldg(p.lens + seq), pb = __ldg(p.prefix_blocks + seq);
    const long long nblk = (static_cast<long long>(len) + p.B - 1) / p.B;
    bool fine = len >= 1 && nblk <= p.max_blocks && pb >= 0 && static_cast<long long>(pb) * p.B <= len;
    const int own = fine ? len - pb * p.B : 0;
    const int32_t* trow = p.tables + static_cast<long long>(seq) * p.max_blocks + (fine ? pb : 0);
    const int tiles = (own + 15) >> 4, stride = p.own_parts;

    // queries of head 8 nt + gid
    uint4 qr[NT][NI];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int j = 8 * nt + gid;
        const uint4* src = reinterpret_cast<const uint4*>(
            static_cast<const KV*>(p.q) + (static_cast<long long>(seq) * p.nh + h * p.g + min(j, p.g - 1)) * D +
                c4 * 8);
#pragma unroll
        for (int i = 0; i < NI; ++i) qr[nt][i] = j < p.g ? __ldg(src + i * 4) : make_uint4(0u, 0u, 0u, 0u);
    }
    // the pool row of token `lane % 16` of a tile; -1: none (behind the context, or a block outside the pool)
    auto row_of = [&](int tile) {
        const int tok = tile * 16 + (lane & 15);
        if (tok >= own) return -1;
        const int bi = p.Bshift >= 0 ? tok >> p.Bshift : tok / p.B;
        const int blk = __ldg(trow + bi);
        if (blk >= 0 && blk < p.num_blocks) return blk * p.B + (tok - bi * p.B);
        report(p.status, KVP_STATUS_BAD_BLOCK);
        return -1;
    };
    float o[NT][D / 16][4];
    float m[NT][2], l[NT][2];  // of heads 8 nt + 2 c4, + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
    }
    uint4 kr[2][NI], vr[4][NH];
    auto load_k = [&](int row) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int x = __shfl_sync(0xffffffffu, row, gid + 8 * r);
            const uint4* src = reinterpret_cast<const uint4*>(static_cast<const KV*>(p.k_cache) +
                                                              (static_cast<long long>(max(x, 0)) * p.kvh + h) * D +
                                                                  c4 * 8);
#pragma unroll
            for (int i = 0; i < NI; ++i) kr[r][i] = x >= 0 ? __ldg(src + i * 4) : make_uint4(0u, 0u, 0u, 0u);
        }
    };
    auto load_v = [&](int row) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int x = __shfl_sync(0xffffffffu, row, 2 * c4 + (r & 1) + (r >> 1) * 8);
            const uint4* src = reinterpret_cast<const uint4*>(static_cast<const KV*>(p.v_cache) +
                                                              (static_cast<long long>(max(x, 0)) * p.kvh + h) * D +
                                                                  gid * 8);
#pragma unroll
            for (int i = 0; i < NH; ++i) vr[r][i] = x >= 0 ? __ldg(src + i * 8) : make_uint4(0u, 0u, 0u, 0u);
        }
    };
    // The next tile's K is on its way as soon as this one's scores are there, its V as soon as this one's is used.
    {
        const int row = row_of(rank);
        load_k(row);
        load_v(row);
    }
    int row = row_of(rank + stride);
    if (rank == 0) {  // meanwhile: the sequence's group, the last one that starts at or before it, 32 candidates a step
        int lo = 0;
        for (int n = p.num_groups; n > 1;) {
            const int step = (n + 31) >> 5;
            const unsigned below = __ballot_sync(0xffffffffu, lane * step < n &&
                                                 __ldg(p.group_starts + lo + lane * step) <= seq);
            const int k = below ? 31 - __clz(below) : 0;
            lo += k * step;
            n = min(step, n - k * step);
        }
        const Group grp = load_group(p, lo);
        fine = fine && grp.start <= seq && seq < grp.start + grp.members && grp.blocks == pb;
        OwnMeta meta = {0, -1, 1, 0, fine, 0};
        if (fine && grp.ktiles > 0) {
            const int member = seq - grp.start, member0 = member / (2 * p.mt) * 2 * p.mt, left = grp.members - member0;
            meta.pair_at = static_cast<long long>(grp.start) * p.kvh + static_cast<long long>(h) * grp.members +
                member0;
            meta.row0 = 2LL * p.g * meta.pair_at + (member - member0) * p.g;  // two row tiles: one after the other
            if (left <= p.mt) {  // one: the even and the odd key tiles'
                meta.parts = 2;
                meta.rows = left * p.g;
            }
        }
        if (lane == 0) {
            p.own_meta[item] = meta;
            if (!fine && h == 0) report(p.status, KVP_STATUS_BAD_LEN);
        }
    }
    for (int tile = rank; tile < tiles; tile += stride) {
        const bool in0 = tile * 16 + gid < own, in1 = tile * 16 + gid + 8 < own;
        uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            // scores of tokens gid, gid + 8 for heads 2 c4, 2 c4 + 1
            float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const uint32_t a0[4] = {kr[0][i].x, kr[1][i].x, kr[0][i].y, kr[1][i].y};
                mma16816<KV>(s, a0, qr[nt][i].x, qr[nt][i].y);
                const uint32_t a1[4] = {kr[0][i].z, kr[1][i].z, kr[0][i].w, kr[1][i].w};
                mma16816<KV>(s, a1, qr[nt][i].z, qr[nt][i].w);
            }
            if (nt == NT - 1) load_k(row);
            // softmax over the tokens of the tile, which eight lanes share
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                s[e] = in0 ? s[e] * p.sl2 : -INFINITY;
                s[2 + e] = in1 ? s[2 + e] * p.sl2 : -INFINITY;
                float mx = fmaxf(s[e], s[2 + e]);
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
                const float mn = fmaxf(m[nt][e], mx), ref = mn == -INFINITY ? 0.f : mn, f = fast_exp2(m[nt][e] - ref);
                m[nt][e] = mn;
                s[e] = fast_exp2(s[e] - (ref - kLift<KV>));
                s[2 + e] = fast_exp2(s[2 + e] - (ref - kLift<KV>));
                l[nt][e] = l[nt][e] * f + (s[e] + s[2 + e]);
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    o[nt][i][e] *= f;
                    o[nt][i][2 + e] *= f;
                }
            }
            // P as a 16-bit part and a 16-bit rest: the memory leaves time for both, and the result keeps close to fp32
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const uint32_t hi = Tr::pack(s[2 * r], s[2 * r + 1]);
                ph[nt][r] = movmatrix_trans(hi);
                pl[nt][r] = movmatrix_trans(Tr::pack(s[2 * r] - Tr::unpack_lo(hi), s[2 * r + 1] - Tr::unpack_hi(hi)));
            }
        }
#pragma unroll
        for (int i = 0; i < NH; ++i) {
            const uint32_t w[4][4] = {{vr[0][i].x, vr[0][i].y, vr[0][i].z, vr[0][i].w},
                                      {vr[1][i].x, vr[1][i].y, vr[1][i].z, vr[1][i].w},
                                      {vr[2][i].x, vr[2][i].y, vr[2][i].z, vr[2][i].w},
                                      {vr[3][i].x, vr[3][i].y, vr[3][i].z, vr[3][i].w}};
#pragma unroll
            for (int t = 0; t < 4; ++t) {  // rows r and r + 8 are dims 64 i + 8 r + 2 t and the one behind it
                const uint32_t a[4] = {__byte_perm(w[0][t], w[1][t], 0x5410u), __byte_perm(w[0][t], w[1][t], 0x7632u),
                                       __byte_perm(w[2][t], w[3][t], 0x5410u), __byte_perm(w[2][t], w[3][t], 0x7632u)};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma16816<KV>(o[nt][i * 4 + t], a, ph[nt][0], ph[nt][1]);
                    mma16816<KV>(o[nt][i * 4 + t], a, pl[nt][0], pl[nt][1]);
                }
            }
        }
        load_v(row);
        row = row_of(tile + 2 * stride);
    }
    {  // a lane holds dims 64 i + 8 gid .. + 7 of heads 2 c4, 2 c4 + 1
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float sum = l[nt][e];
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                const int j = 8 * nt + 2 * c4 + e;
                if (j >= p.g) continue;
                const long long row = (static_cast<long long>(seq) * p.nh + h * p.g + j) * p.own_parts + rank;
                if (gid == 0) p.own_ml[row] = partial<KV>(m[nt][e], sum);
                if (rank >= tiles) continue;  // nothing, and its columns are not used
#pragma unroll
                for (int i = 0; i < NH; ++i)
#pragma unroll
                    for (int t = 0; t < 4; t += 2)
                        *reinterpret_cast<float4*>(p.own_o + row * D + 64 * i + 8 * gid + 2 * t) =
                            make_float4(o[nt][i * 4 + t][e], o[nt][i * 4 + t][2 + e], o[nt][i * 4 + t + 1][e],
                                        o[nt][i * 4 + t + 1][2 + e]);
            }
    }
    if (blockIdx.x == gridDim.x - 1) griddep_wait();
}

// The own parts and the shared part's partial rows: a thread folds four columns of a (sequence, query head).  Bound by
// the partial rows' way through L2, and three latencies.
template <int D>
__global__ void __launch_bounds__(256) join_kernel(const PrefixParams p) {
    griddep_launch_dependents();
    const long long at = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    const long long row = at / (D / 4);
    const int col = static_cast<int>(at % (D / 4)) * 4;
    if (row >= static_cast<long long>(p.num_seqs) * p.nh) return;
    const unsigned item = static_cast<unsigned>(row) / static_cast<unsigned>(p.g);
    const int j = static_cast<int>(static_cast<unsigned>(row) - item * static_cast<unsigned>(p.g));
    griddep_wait();
    const int32_t unsorted = __ldcg(p.unsorted);
    const OwnMeta meta = p.own_meta[item];
    float2 ml[4];
    float4 x[4];
    auto own_part = [&](int k0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool some = k0 + i < p.own_parts;
            const long long r = row * p.own_parts + k0 + i;
            ml[i] = some ? __ldcg(&p.own_ml[r]) : make_float2(-INFINITY, 0.f);
            x[i] = some ? __ldcg(reinterpret_cast<const float4*>(p.own_o + r * D + col))
                : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    };
    own_part(0);  // on their way while the place of the others is looked up
    const SharedParts shared = shared_parts(p, meta);
    Fold all;
    all.add(ml, x);
    if (p.own_parts > 4) {
        own_part(4);
        all.add(ml, x);
    }
    for (int k0 = 0; k0 < shared.count; k0 += 4) {
        shared.load(p, j, D, col, k0, ml, x);
        all.add(ml, x);
    }
    const bool fine = meta.fine && !unsorted;
    store_out(p, static_cast<size_t>(row) * D + col, fine ? all.o : make_float4(0.f, 0.f, 0.f, 0.f),
              fine ? 1.f / all.l : 0.f);
}

}  // namespace kvpd

namespace kvpi {
namespace {

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// The decode attention over whole contexts with the same arguments.
kvp_attn_args whole_contexts(const kvp_prefix_args& a) {
    kvp_attn_args w;
    std::memset(&w, 0, sizeof(w));
    w.q = a.q;
    w.q_dtype = a.q_dtype;
    w.k_cache = a.k_cache;
    w.v_cache = a.v_cache;
    w.kv_dtype = a.kv_dtype;
    w.num_blocks = a.num_blocks;
    w.block_tables = a.block_tables;
    w.seq_lens = a.seq_lens;
    w.out = a.out;
    w.out_dtype = a.out_dtype;
    w.num_seqs = a.num_seqs;
    w.num_heads = a.num_heads;
    w.kv_heads = a.kv_heads;
    w.head_dim = a.head_dim;
    w.block_size = a.block_size;
    w.max_blocks = a.max_blocks;
    w.scale = a.scale;
    w.workspace = a.workspace;
    w.workspace_bytes = a.workspace_bytes;
    w.status = a.status;
    return w;
}

// Warps an SM that own parts are split into at least: 16 is what its registers hold.  Half as many took 186 us at 256
// sequences with up to 512 own tokens instead of 171 (twice as many 170); twice as many 82 us at 512 with up to 100
// instead of 79, four times 90, for the parts that join_kernel has to read.
constexpr long long kOwnWarps = 16;

struct PrefixPlan {
    bool shared = false;  // else the plain decode attention over every sequence's whole context
    size_t spans = 0, ml = 0, o = 0, meta = 0, own_ml = 0, own_o = 0, bytes = 0;
    int mt = 1, run = 8, keys = 0;
    int own_parts = 1;
};

int gcd_of(int a, int b) { return b ? gcd_of(b, a % b) : a; }

int plan_prefix(const kvp_prefix_args* a, PrefixPlan* pl) {
    if (!a) return fail(KVP_EINVAL, "null arguments");
    if (!valid_dtype(a->q_dtype) || !valid_dtype(a->kv_dtype) || !valid_dtype(a->out_dtype))
        return fail(KVP_EINVAL, "unsupported dtype");
    if (a->num_seqs < 0 || a->num_groups < 0 || (a->num_seqs > 0 && a->num_groups < 1) || a->num_groups > a->num_seqs)
        return fail(KVP_EINVAL, "bad num_seqs / num_groups");
    if (a->num_blocks < 1 || a->block_size < 1 || a->max_blocks < 1)
        return fail(KVP_EINVAL, "bad num_blocks / block_size / max_blocks");
    kvp_attn_args w = whole_contexts(*a);
    if (a->num_seqs == 0) return KVP_OK;
    if (a->kv_dtype == KVP_DTYPE_F32) return KVP_OK;
    // The shared kernel's tiles hold 128 keys, copied in runs of at least 8 within a block; of blocks that have no such
    // runs, as many whole ones as fit.
    pl->run = gcd_of(a->block_size, kvpd::kKeys);
    pl->keys = kvpd::kKeys;
    if (pl->run < 8) {
        pl->run = a->block_size;
        pl->keys = kvpd::kKeys / a->block_size * a->block_size;  // 0: none fits
    }
    AttnPlan whole;
    const int rc = plan_attention(w, true, &whole);
    if (rc != KVP_OK) return rc;
    pl->bytes = whole.ws_bytes;
    if (aligned16(a->q)) {  // unaligned queries may need more, which a size asked for without buffers has to cover
        w.q = reinterpret_cast<const void*>(uintptr_t{2});
        if (plan_attention(w, true, &whole) == KVP_OK) pl->bytes = std::max(pl->bytes, whole.ws_bytes);
        else clear_error();
    }
    pl->shared = (a->head_dim == 64 || a->head_dim == 128) && a->q_dtype == a->kv_dtype && pl->keys > 0 &&
        aligned16(a->q) &&
                 aligned16(a->out) && static_cast<long long>(a->num_seqs) * a->kv_heads <= (1LL << 27) &&
                 static_cast<long long>(a->max_blocks) * a->block_size <= kvpd::kPrefixTokens;
    if (!pl->shared) return KVP_OK;
    const size_t rows = static_cast<size_t>(a->num_seqs) * a->num_heads;
    const size_t parts = 2 * rows + static_cast<size_t>(sm_count()) * 2 * kvpd::kRows;
    pl->mt = kvpd::kRows / (a->num_heads / a->kv_heads);
    pl->spans = 256;  // behind the word that tells of unsorted groups
    pl->ml = pl->spans + up256(static_cast<size_t>(a->num_seqs) * a->kv_heads * 8);
    pl->o = pl->ml + up256(parts * 8);
    // (the largest of all: where q or out are not aligned the other path runs in the same workspace)
    pl->meta = pl->o + up256(parts * a->head_dim * 4);
    const long long items = static_cast<long long>(a->num_seqs) * a->kv_heads;
    while (pl->own_parts < 8 && items * pl->own_parts < sm_count() * kOwnWarps) pl->own_parts *= 2;
    pl->own_ml = pl->meta + up256(static_cast<size_t>(a->num_seqs) * a->kv_heads * sizeof(kvpd::OwnMeta));
    pl->own_o = pl->own_ml + up256(rows * pl->own_parts * 8);
    pl->bytes = std::max(pl->bytes, pl->own_o + rows * pl->own_parts * a->head_dim * 4);
    return KVP_OK;
}

int encode_3d(CUtensorMap* map, int dtype, const void* base, const cuuint64_t (&dims)[3],
              const cuuint64_t (&strides)[2], const cuuint32_t (&box)[3]) {
    auto fn = encode_fn();
    if (!fn) return fail(KVP_ECUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint32_t one[3] = {1, 1, 1};
    const CUtensorMapDataType type =
        dtype == KVP_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const CUresult r = fn(map, type, 3, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(KVP_ECUDA, "cuTensorMapEncodeTiled failed with code " + std::to_string(r));
    return KVP_OK;
}

// A launch that may start before the one ahead has ended.
template <class... P>
int launch_early(void (*fn)(P...), unsigned grid, unsigned threads, size_t smem, cudaStream_t s, const char* what,
                 const P&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, fn, args...), what);
}

template <int D, class KV>
int launch_prefix(const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, kvpd::PrefixParams p,
                  cudaStream_t s) {
    auto fn = &kvpd::prefix_kernel<D, KV>;
    const int rc = allow_smem(reinterpret_cast<const void*>(fn));
    if (rc != KVP_OK) return rc;
    constexpr size_t tile = static_cast<size_t>(kvpd::kKeys) * D * 2;
    return launch_early(fn, static_cast<unsigned>(p.ctas), kvpd::kPrefixThreads, 1024 + (2 + (D == 128 ? 4 : 7)) * tile,
                        s, "shared prefix launch",
                        qm, km, vm, p);
}

template <int D, class KV>
int launch_own(const kvpd::PrefixParams& p, cudaStream_t s) {
    auto fn = p.g > 8 ? &kvpd::own_kernel<D, KV, 2> : &kvpd::own_kernel<D, KV, 1>;
    const unsigned warps = static_cast<unsigned>(p.num_seqs) * static_cast<unsigned>(p.kvh) *
        static_cast<unsigned>(p.own_parts);
    const int rc = launch_early(fn, warps, 32, 0, s, "own part launch", p);
    if (rc != KVP_OK) return rc;
    const long long threads = static_cast<long long>(p.num_seqs) * p.nh * (D / 4);
    return launch_early(&kvpd::join_kernel<D>, static_cast<unsigned>((threads + 255) / 256), 256, 0, s, "join launch",
                        p);
}

template <int D, class KV>
int launch_both(const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, const kvpd::PrefixParams& p,
                cudaStream_t s) {
    const int rc = launch_prefix<D, KV>(qm, km, vm, p, s);
    return rc != KVP_OK ? rc : launch_own<D, KV>(p, s);
}

}  // namespace
}  // namespace kvpi

extern "C" KVP_API size_t kvp_prefix_workspace_size(const kvp_prefix_args* a) {
    kvpi::clear_error();
    kvpi::PrefixPlan pl;
    return kvpi::plan_prefix(a, &pl) == KVP_OK ? pl.bytes : 0;
}

extern "C" KVP_API int kvp_prefix_attention(const kvp_prefix_args* a, void* stream) {
    using namespace kvpi;
    clear_error();
    PrefixPlan pl;
    int rc = plan_prefix(a, &pl);
    if (rc != KVP_OK || a->num_seqs == 0) return rc;
    if (!a->q || !a->k_cache || !a->v_cache || !a->block_tables || !a->seq_lens || !a->prefix_blocks ||
        !a->group_starts || !a->out)
        return fail(KVP_EINVAL, "null buffer");
    if (pl.bytes > 0 && (!a->workspace || a->workspace_bytes < pl.bytes))
        return fail(KVP_ENOSPACE, "workspace smaller than kvp_prefix_workspace_size()");
    if ((reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0)
        return fail(KVP_EINVAL, "workspace must be 256-byte aligned");
    if (!pl.shared) {
        const kvp_attn_args w = whole_contexts(*a);
        return kvp_paged_attention(&w, stream);
    }
    if (!aligned16(a->k_cache) || !aligned16(a->v_cache)) return fail(KVP_EINVAL, "K/V pools must be 16-byte aligned");
    if (a->num_blocks > 0x7fffffffLL / a->block_size)
        return fail(KVP_EINVAL, "num_blocks * block_size must stay below 2^31");
    const long long rows = a->num_blocks * a->block_size;
    const int g = a->num_heads / a->kv_heads;
    const cuuint64_t D = static_cast<cuuint64_t>(a->head_dim);
    CUtensorMap qm, km, vm;
    {
        const cuuint64_t dims[3] = {D, static_cast<cuuint64_t>(a->num_heads), static_cast<cuuint64_t>(a->num_seqs)};
        const cuuint64_t strides[2] = {D * 2, D * 2 * a->num_heads};
        const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(g), static_cast<cuuint32_t>(pl.mt)};
        rc = encode_3d(&qm, a->kv_dtype, a->q, dims, strides, box);
        if (rc != KVP_OK) return rc;
    }
    {
        const cuuint64_t dims[3] = {D, static_cast<cuuint64_t>(a->kv_heads), static_cast<cuuint64_t>(rows)};
        const cuuint64_t strides[2] = {D * 2, D * 2 * a->kv_heads};
        const cuuint32_t box[3] = {64, 1, static_cast<cuuint32_t>(pl.run)};
        rc = encode_3d(&km, a->kv_dtype, a->k_cache, dims, strides, box);
        if (rc != KVP_OK) return rc;
        rc = encode_3d(&vm, a->kv_dtype, a->v_cache, dims, strides, box);
        if (rc != KVP_OK) return rc;
    }
    char* ws = static_cast<char*>(a->workspace);
    kvpd::PrefixParams p;
    std::memset(&p, 0, sizeof(p));
    p.tables = a->block_tables;
    p.lens = a->seq_lens;
    p.prefix_blocks = a->prefix_blocks;
    p.group_starts = a->group_starts;
    p.status = a->status;
    p.unsorted = reinterpret_cast<int32_t*>(ws);
    p.spans = reinterpret_cast<int2*>(ws + pl.spans);
    p.part_ml = reinterpret_cast<float2*>(ws + pl.ml);
    p.part_o = reinterpret_cast<float*>(ws + pl.o);
    p.own_meta = reinterpret_cast<kvpd::OwnMeta*>(ws + pl.meta);
    p.own_ml = reinterpret_cast<float2*>(ws + pl.own_ml);
    p.own_o = reinterpret_cast<float*>(ws + pl.own_o);
    p.q = a->q;
    p.k_cache = a->k_cache;
    p.v_cache = a->v_cache;
    p.out = a->out;
    p.num_blocks = a->num_blocks;
    p.wait_limit = kvpd::kWaitLimitCycles;
    p.num_seqs = a->num_seqs;
    p.num_groups = a->num_groups;
    p.nh = a->num_heads;
    p.kvh = a->kv_heads;
    p.g = g;
    p.max_blocks = a->max_blocks;
    p.B = a->block_size;
    p.Bshift = -1;
    if ((a->block_size & (a->block_size - 1)) == 0)
        for (p.Bshift = 0; (1 << p.Bshift) < a->block_size;) ++p.Bshift;
    p.run = pl.run;
    p.keys = pl.keys;
    p.runs = pl.keys / pl.run;
    p.oob_row = static_cast<int>(rows);
    p.mt = pl.mt;
    p.own_parts = pl.own_parts;
    p.bf16 = a->kv_dtype == KVP_DTYPE_BF16;
    p.out_dtype = a->out_dtype;
    p.ctas = sm_count();
    p.sl2 = (a->scale > 0.f ? a->scale : 1.0f / std::sqrt(static_cast<float>(a->head_dim))) * 1.4426950408889634f;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a->head_dim == 64)
        rc = p.bf16 ? launch_both<64, __nv_bfloat16>(qm, km, vm, p, s) : launch_both<64, __half>(qm, km, vm, p, s);
    else
        rc = p.bf16 ? launch_both<128, __nv_bfloat16>(qm, km, vm, p, s) : launch_both<128, __half>(qm, km, vm, p, s);
    return rc;
}

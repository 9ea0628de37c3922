// Beam selection: of all continuations (beam, token) of a request, the `select` best by
//     value = score[beam] + logit[beam][token] - log(sum over tokens of exp(logit[beam][.])),
// ties to the lower beam, then the lower token.  One read of the logits, two launches.
//
// beam_scan_kernel (bound by HBM): a warp takes its share of one row, 512 logits a step, three steps in flight.  It
// keeps a running maximum and sum of exponentials per lane, and its best `select` logits as a list sorted over its 32
// lanes; within a row the order of the values is the order of the logits, so no logarithm is needed here.  The list
// starts from the lanes' own maxima of the first step (one sort); of the rest only what passes the list's last entry --
// or that of another warp of the CTA, which works on the same row -- costs more than one vote per step, and is inserted
// with a ballot and a shift.  Entries are 64-bit keys (ordered logit, ~token): all different, so ties fall to the lower
// token however the row is cut.  512 rows of 128000 fp32 logits, select 16: 262 MB in 61 us (4.3 TB/s), the issue slots
// 63% busy: about 100 instructions a step of 512 logits, and as many again for what passes into the lists.
//
// beam_pick_kernel (bound by latency): one CTA per request joins each beam's segments -- their sums in 64 bits, their
// lists by bitonic merges -- and takes the best head of the beams' lists `select` times, comparing values in 64 bits,
// so that no 32-bit rounding of a value decides.  A beam's own continuations are in the exact order of their logits.
// Between beams the log-sums' errors remain, whose terms lanes and warps add in fp32: at most (16 + 34 s) 2^-24 with s
// steps a warp, 1.7e-5 at 8 steps; values that lie nearer to each other than twice that may change places.  About 8 us,
// most of it the way from the partial sums to the first choice.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kvp_device.cuh"
#include "kvp_internal.h"

namespace kvpd {

constexpr int kBeamMost = 32;    // beams and selected continuations per request: a warp's lanes
constexpr int kBeamSegs = 32;    // segments of a row
constexpr int kBeamLane = 16;    // logits a lane takes at once
constexpr int kBeamStep = 32 * kBeamLane;
constexpr int kBeamRing = 3;     // steps of a warp in flight
constexpr int kBeamWarps = 4;    // warps per CTA of the scan, all on one row
constexpr int kBeamShows = 6;    // times a CTA's warps compare their lists
constexpr int kPickWarps = 16;
constexpr int kBeamTokenBits = 26;

struct BeamParams {
    const void* logits;
    const float* scores;
    float* out_scores;
    int32_t* out_parents;
    int32_t* out_tokens;
    float2* seg_ml;             // [rows][segs] maximum and sum of exp(logit - maximum)
    unsigned long long* keys;   // [rows][segs][select]
    int32_t* status;
    long long row_stride;       // elements
    int batch, beams, vocab, select, segs;
    int seg_steps;              // most steps of a warp
};

__device__ __forceinline__ uint32_t ordered32(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered32(uint32_t o) {
    return __uint_as_float(o ^ ((o & 0x80000000u) ? 0x80000000u : 0xffffffffu));
}
// Key of a logit; 0 is "no entry" (below every key, that of -inf included).  -0 counts as 0.
__device__ __forceinline__ unsigned long long beam_key(float x, int token) {
    return (static_cast<unsigned long long>(ordered32(x + 0.f)) << 32) | static_cast<uint32_t>(~token);
}

// Sorts one key per lane, largest in lane 0 (bitonic).
__device__ __forceinline__ unsigned long long warp_sort_desc(unsigned long long v, int lane) {
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1) {
            const unsigned long long w = __shfl_xor_sync(0xffffffffu, v, j);
            const bool keep_max = ((lane & j) == 0) == ((lane & k) == 0);
            v = keep_max ? (v > w ? v : w) : (v < w ? v : w);
        }
    return v;
}

// Two lists sorted over the lanes, largest first, become the 32 largest of both.
__device__ __forceinline__ unsigned long long warp_merge_desc(unsigned long long a, unsigned long long b, int lane) {
    const unsigned long long r = __shfl_xor_sync(0xffffffffu, b, 31);
    unsigned long long v = a > r ? a : r;  // a bitonic sequence of the 32 largest
#pragma unroll
    for (int j = 16; j > 0; j >>= 1) {
        const unsigned long long w = __shfl_xor_sync(0xffffffffu, v, j);
        v = (lane & j) == 0 ? (v > w ? v : w) : (v < w ? v : w);
    }
    return v;
}

// One step of a row, 16 logits per lane: element e of a lane is token at + ((e / N) * 32 + lane) * N + e % N - shift.
// Vec: 16-byte loads, where all rows of a request lie alike against 16-byte boundaries.  Else single loads of
// neighbouring tokens by neighbouring lanes: with an odd vocabulary the rows start at different offsets, and vectors
// would group the sums of two equal rows differently, so that their tie fell to a rounding.
template <class T, bool Vec>
struct BeamStep {
    static constexpr int N = 1;
    T u[kBeamLane];
    __device__ __forceinline__ void load(const T* p, int lane) {
#pragma unroll
        for (int j = 0; j < kBeamLane; ++j) u[j] = __ldcs(p + j * 32 + lane);
    }
    __device__ __forceinline__ void get(float (&x)[kBeamLane]) const {
#pragma unroll
        for (int j = 0; j < kBeamLane; ++j) x[j] = one(u + j);
    }
    static __device__ __forceinline__ float one(const T* p) {
        if constexpr (sizeof(T) == 4) return *p;
        else return F16Traits<T>::to_float(*p);
    }
};
template <class T>
struct BeamStep<T, true> {
    static constexpr int N = 16 / sizeof(T);       // logits of a vector
    static constexpr int kVecs = kBeamLane / N;    // vectors of a lane
    static __device__ __forceinline__ float one(const T* p) { return BeamStep<T, false>::one(p); }
};
// A warp's steps on their way, each lane's vectors in places of its own: copied asynchronously, so that three steps are
// in flight without registers, and read back by the lane that asked for them.
template <class T>
struct BeamRing {
    using Step = BeamStep<T, true>;
    uint32_t at;  // this lane's first place
    __device__ __forceinline__ void load(int slot, const T* p, int lane) const {
#pragma unroll
        for (int j = 0; j < Step::kVecs; ++j)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                         :
                         : "r"(at + static_cast<uint32_t>(slot * Step::kVecs + j) * 512u),
                           "l"(p + (j * 32 + lane) * Step::N)
                         : "memory");
    }
    static __device__ __forceinline__ void close() { asm volatile("cp.async.commit_group;" ::: "memory"); }
    static __device__ __forceinline__ void wait() {
        asm volatile("cp.async.wait_group %0;" ::"n"(kBeamRing - 1) : "memory");
    }
    __device__ __forceinline__ void get(int slot, float (&x)[kBeamLane]) const {
#pragma unroll
        for (int j = 0; j < Step::kVecs; ++j) {
            uint32_t w[4];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                         : "r"(at + static_cast<uint32_t>(slot * Step::kVecs + j) * 512u)
                         : "memory");
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 4) {
                    x[4 * j + i] = __uint_as_float(w[i]);
                } else {
                    x[8 * j + 2 * i] = F16Traits<T>::unpack_lo(w[i]);
                    x[8 * j + 2 * i + 1] = F16Traits<T>::unpack_hi(w[i]);
                }
            }
        }
    }
};

// A beam takes part when its score is finite; -inf is a beam that is not in use.
__device__ __forceinline__ bool beam_live(float score) { return score > -INFINITY && score < INFINITY; }

// Maxima of each group of eight, and of all.
__device__ __forceinline__ float max_of(const float (&x)[kBeamLane], float (&group)[kBeamLane / 8]) {
    float top = -INFINITY;
#pragma unroll
    for (int g = 0; g < kBeamLane / 8; ++g) {
        const float a = fmaxf(fmaxf(x[8 * g], x[8 * g + 1]), x[8 * g + 2]);
        const float b = fmaxf(fmaxf(x[8 * g + 3], x[8 * g + 4]), x[8 * g + 5]);
        group[g] = fmaxf(fmaxf(a, b), fmaxf(x[8 * g + 6], x[8 * g + 7]));
        top = fmaxf(top, group[g]);
    }
    return top;
}
// Sum of exp(x - ref), two at a time: the difference is taken first, so that the large terms, whose difference is
// small, are exact to the exponential's own error.
__device__ __forceinline__ float expsum(const float (&x)[kBeamLane], float ref) {
    const uint64_t back = pack2(-ref, -ref), log2e = pack2(1.4426950408889634f, 1.4426950408889634f);
    uint64_t t[2] = {0ull, 0ull};
#pragma unroll
    for (int i = 0; i < kBeamLane / 2; ++i) {
        const float2 d = unpack2(mul2(add2(pack2(x[2 * i], x[2 * i + 1]), back), log2e));
        t[i & 1] = add2(t[i & 1], pack2(fast_exp2(d.x), fast_exp2(d.y)));
    }
    const float2 r = unpack2(add2(t[0], t[1]));
    return r.x + r.y;
}
__device__ __forceinline__ float exp_of(float d) { return fast_exp2(d * 1.4426950408889634f); }

// Named barrier 1 + k, with a constant number: a number from a register would claim all sixteen for each CTA, and four
// CTAs an SM would be the most.
__device__ __forceinline__ void barrier_of(int k, bool only_arrive, int threads) {
    auto at = [&](auto id) {
        if (only_arrive)
            asm volatile("bar.arrive %0, %1;" ::"n"(decltype(id)::value), "r"(threads) : "memory");
        else
            asm volatile("bar.sync %0, %1;" ::"n"(decltype(id)::value), "r"(threads) : "memory");
    };
    switch (k) {
        case 0: at(std::integral_constant<int, 1>{}); break;
        case 1: at(std::integral_constant<int, 2>{}); break;
        case 2: at(std::integral_constant<int, 3>{}); break;
        case 3: at(std::integral_constant<int, 4>{}); break;
        case 4: at(std::integral_constant<int, 5>{}); break;
        default: at(std::integral_constant<int, 6>{}); break;
    }
}

template <class T, bool Vec>
__global__ void __launch_bounds__(kBeamWarps * 32, 7) beam_scan_kernel(const BeamParams p) {
    using Step = BeamStep<T, Vec>;
    constexpr int N = Step::N;
    __shared__ unsigned long long floor_key;  // no entry below it is among the row's best `select`
    __shared__ unsigned long long shown[kBeamShows][kBeamWarps][32];
    __shared__ __align__(16) uint8_t steps[Vec ? kBeamWarps * kBeamRing * kBeamStep * sizeof(T) : 16];
    BeamRing<T> ring;
    ring.at = smem_u32(steps) + (threadIdx.x >> 5) * (kBeamRing * kBeamStep * sizeof(T)) + (threadIdx.x & 31) * 16;
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int groups = (p.segs + kBeamWarps - 1) / kBeamWarps;  // CTAs per row
    const long long row = blockIdx.x / groups;
    const int warp = threadIdx.x >> 5;
    const int seg = static_cast<int>(blockIdx.x - row * groups) * kBeamWarps + warp;
    const int partners = min(kBeamWarps, p.segs - (seg - warp));  // warps of this CTA that have a segment
    const long long item = row * p.segs + seg;
    if (threadIdx.x == 0) floor_key = 0ull;
    __syncthreads();
    if (seg >= p.segs) return;
    unsigned long long* out = p.keys + item * p.select;
    const float score = __ldg(p.scores + row);
    if (!beam_live(score)) {
        // every continuation of this beam has the value -inf: the lowest tokens stand for it
        if (seg == 0 && lane == 0 && score != -INFINITY) report(p.status, KVP_STATUS_BAD_VALUE);
        if (lane < p.select) out[lane] = seg == 0 && lane < p.vocab ? beam_key(-INFINITY, lane) : 0ull;
        if (lane == 0) p.seg_ml[item] = make_float2(-INFINITY, 0.f);
        return;
    }
    const T* base = static_cast<const T*>(p.logits) + row * p.row_stride;
    // Steps start at 16-byte boundaries: token = place - shift.  A row's warps take its steps in turn, so that at any
    // time they read one stretch of memory.
    const int shift = Vec ? static_cast<int>((reinterpret_cast<uintptr_t>(base) & 15u) / sizeof(T)) : 0;
    const int end = p.vocab + shift, first = seg * kBeamStep, ahead = p.segs * kBeamStep;
    const int n = first < end ? (end - first - 1) / ahead + 1 : 0;  // steps of this warp
    // those that lie inside the row from end to end
    const int f0 = first < shift ? 1 : 0, f1 = n > 0 && first + (n - 1) * ahead + kBeamStep > end ? n - 1 : n;
    auto at_edge = [&](int place, float (&x)[kBeamLane]) {  // a row's first or last step; the elements that exist
        unsigned live = 0u;
#pragma unroll
        for (int e = 0; e < kBeamLane; ++e) {
            const int tok = place + (e / N) * 32 * N + e % N;
            const bool in = tok >= 0 && tok < p.vocab;
            x[e] = in ? Step::one(base + tok) : -INFINITY;
            if (in) live |= 1u << e;
        }
        return live;
    };
    bool bad = false;
    auto ban = [&](float (&x)[kBeamLane]) {  // NaN and +inf count as -inf
#pragma unroll
        for (int e = 0; e < kBeamLane; ++e)
            if (!(x[e] < INFINITY)) {
                x[e] = -INFINITY;
                bad = true;
            }
    };
    constexpr unsigned kAll = (1u << kBeamLane) - 1u;
    const T* next = base + (first - shift);  // the step to ask for next
    int asked = 0, slot = 0;
    Step raw;
    auto ask = [&](int to) {
        if (asked >= f0 && asked < f1) {
            if constexpr (Vec) ring.load(to, next, lane);
            else raw.load(next, lane);
        }
        if constexpr (Vec) ring.close();
        next += ahead;
        ++asked;
    };
#pragma unroll
    for (int k = 0; k < (Vec ? kBeamRing : 1); ++k) ask(k);
    float m = -INFINITY, sum = 0.f;
    unsigned long long best = 0ull, least = 0ull;  // the list (one entry per lane); what an entry has to exceed
    // The same as a value and a token.  An equal value counts only before that token, which lies ahead only where
    // another warp set the floor.
    float lv = -INFINITY;
    int ltok = 0x7fffffff;
    auto refresh = [&] {
        if (least) {
            lv = unordered32(static_cast<uint32_t>(least >> 32));
            ltok = static_cast<int>(~static_cast<uint32_t>(least));
        }
    };
    // After steps 1, 2, 4, ... the warps show their lists; the first one joins them and raises the floor for all.  Each
    // such moment has its own barrier and its own place, so the other warps only arrive and go on.  Every warp of the
    // CTA that has a share takes part in all of them.
    int show = 0, shows = 0;
    if (partners > 1)
        while (shows < kBeamShows && (1 << shows) < p.seg_steps) ++shows;
    auto compare = [&] {
        shown[show][warp][lane] = best;
        __threadfence_block();
        __syncwarp();
        barrier_of(show, warp > 0, partners * 32);
        if (warp == 0) {
            unsigned long long all = best;
            for (int i = 1; i < partners; ++i) all = warp_merge_desc(all, shown[show][i][lane], lane);
            if (lane == p.select - 1) *reinterpret_cast<volatile unsigned long long*>(&floor_key) = all;
        }
        ++show;
    };
    // The list starts from each lane's best of the first step.
    unsigned done = 0u;  // elements of the first step that it holds already
    if (n > 0) {
        float x[kBeamLane], group[kBeamLane / 8];
        unsigned live = kAll;
        const int place = first + lane * N - shift;
        if constexpr (Vec) ring.wait();
        if (f0 > 0 || f1 == 0) {
            live = at_edge(place, x);
        } else {
            if constexpr (Vec) ring.get(0, x);
            else raw.get(x);
        }
        ban(x);
        const float top = max_of(x, group);
        int arg = kBeamLane - 1;
#pragma unroll
        for (int e = kBeamLane - 1; e >= 0; --e)
            if (x[e] == top && ((live >> e) & 1u)) arg = e;
        best = warp_sort_desc((live >> arg) & 1u ? beam_key(top, place + (arg / N) * 32 * N + arg % N) : 0ull, lane);
        done = 1u << arg;
        least = __shfl_sync(0xffffffffu, best, p.select - 1);
        refresh();
    }
    for (int i = 0; i < n; ++i) {
        float x[kBeamLane], group[kBeamLane / 8];
        unsigned live = kAll;
        const int at = first + i * ahead - shift, place = at + lane * N;  // tokens: the step's and this lane's first
        if constexpr (Vec) ring.wait();
        if (i >= f0 && i < f1) {
            if constexpr (Vec) ring.get(slot, x);
            else raw.get(x);
        } else {
            live = at_edge(place, x);
        }
        ask(slot);
        slot = slot + 1 == kBeamRing ? 0 : slot + 1;
        float top = max_of(x, group);
        float mn = fmaxf(m, top);
        float add = expsum(x, mn > -INFINITY ? mn : 0.f);
        // A NaN or a +inf among them shows here: each term is at most 1 else.  (Asked of the whole warp, so that what
        // is rare is branched over and not predicated.)
        if (__any_sync(0xffffffffu, !(add <= static_cast<float>(kBeamLane)))) {
            ban(x);
            top = max_of(x, group);
            mn = fmaxf(m, top);
            add = expsum(x, mn > -INFINITY ? mn : 0.f);
        }
        if (mn > -INFINITY) {
            sum = sum * exp_of(m - mn) + add;
            m = mn;
        }
        unsigned long long known = *reinterpret_cast<volatile unsigned long long*>(&floor_key);
        if (__any_sync(0xffffffffu, known > least)) {
            known = __shfl_sync(0xffffffffu, known, 0);  // written at any time: the lanes take the same one
            least = known > least ? known : least;
            refresh();
        }
        const bool ties = at < ltok;
        if (__any_sync(0xffffffffu, top > lv || (ties && top == lv))) {
#pragma unroll
            for (int g = 0; g < kBeamLane / 8; ++g) {
                if (!__any_sync(0xffffffffu, group[g] > lv || (ties && group[g] == lv))) continue;
                unsigned pass = 0u;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (x[8 * g + e] > lv) pass |= 1u << e;
                if (ties) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (x[8 * g + e] == lv) pass |= 1u << e;
                }
                pass &= (live & ~done) >> (8 * g);
                while (__any_sync(0xffffffffu, pass != 0u)) {
                    const int e = __ffs(pass) - 1;  // -1: nothing left in this lane
                    float t[4], v;  // element e: a tree of selections instead of an array in memory
#pragma unroll
                    for (int k = 0; k < 4; ++k) t[k] = e & 4 ? x[8 * g + k + 4] : x[8 * g + k];
                    v = e & 2 ? (e & 1 ? t[3] : t[2]) : (e & 1 ? t[1] : t[0]);
                    const int el = 8 * g + e;
                    const unsigned long long key = pass ? beam_key(v, place + (el / N) * 32 * N + el % N) : 0ull;
                    pass &= pass - 1u;
                    unsigned who = __ballot_sync(0xffffffffu, key > least);
                    while (who) {
                        const int src = __ffs(who) - 1;
                        who &= who - 1u;
                        const unsigned long long in = __shfl_sync(0xffffffffu, key, src);
                        if (in <= least) continue;
                        const int rank = __popc(__ballot_sync(0xffffffffu, best > in));
                        const unsigned long long up = __shfl_up_sync(0xffffffffu, best, 1);
                        best = lane < rank ? best : lane == rank ? in : up;
                        const unsigned long long own = __shfl_sync(0xffffffffu, best, p.select - 1);
                        least = own > least ? own : least;
                    }
                }
                refresh();
            }
        }
        done = 0u;
        if (show < shows && i + 1 == 1 << show) compare();
    }
    while (show < shows) compare();  // a warp with fewer steps: its partners wait for as many
    float top = m;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    float total = top > -INFINITY ? sum * exp_of(m - top) : 0.f;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
    if (lane == 0) p.seg_ml[item] = make_float2(top, total);
    if (lane < p.select) out[lane] = best;
    if (bad) report(p.status, KVP_STATUS_BAD_VALUE);
}

__global__ void __launch_bounds__(kPickWarps * 32) beam_pick_kernel(const BeamParams p) {
    __shared__ unsigned long long part[kPickWarps][32];
    __shared__ unsigned long long value[kBeamMost][32];  // [beam][entry]
    __shared__ int token[kBeamMost][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long row0 = static_cast<long long>(blockIdx.x) * p.beams;
    const int per = max(1, kPickWarps / p.beams);  // warps that share a beam's lists
    auto fold = [&](unsigned long long best, unsigned long long k) {  // only a list whose head gets in
        const bool in = __shfl_sync(0xffffffffu, k, 0) > __shfl_sync(0xffffffffu, best, p.select - 1);
        return in ? warp_merge_desc(best, k, lane) : best;
    };
    griddep_wait();
    for (int b0 = 0; b0 < p.beams; b0 += kPickWarps) {
        const int b = b0 + warp / per, sub = warp % per;
        const bool mine = b < p.beams && warp < per * p.beams;
        const float score = mine ? __ldg(p.scores + row0 + b) : 0.f;
        double lse = 0.0;
        if (mine) {
            const long long item0 = (row0 + b) * p.segs;
            unsigned long long best = 0ull;
            for (int s0 = sub; s0 < p.segs; s0 += 4 * per) {
                unsigned long long k[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int seg = s0 + i * per;
                    k[i] = seg < p.segs && lane < p.select ? __ldcg(p.keys + (item0 + seg) * p.select + lane) : 0ull;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) best = fold(best, k[i]);
            }
            part[warp][lane] = best;
            if (sub == 0) {  // the beam's sums of exponentials, in 64 bits
                float2 ml[kBeamSegs / 32];
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < kBeamSegs / 32; ++i) {
                    const int s = i * 32 + lane;
                    ml[i] = s < p.segs ? __ldcg(p.seg_ml + item0 + s) : make_float2(-INFINITY, 0.f);
                    top = fmaxf(top, ml[i].x);
                }
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                double total = 0.0;
#pragma unroll
                for (int i = 0; i < kBeamSegs / 32; ++i)
                    if (ml[i].x > -INFINITY)
                        total += static_cast<double>(ml[i].y) * exp(static_cast<double>(ml[i].x) - top);
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
                lse = top > -INFINITY ? top + log(total) : -static_cast<double>(INFINITY);
            }
        }
        __syncthreads();
        if (mine && sub == 0) {
            unsigned long long best = part[warp][lane];
            for (int i = 1; i < per; ++i) best = fold(best, part[warp + i][lane]);
            // each entry as an ordered value in 64 bits (0: none) and its place
            const float x = unordered32(static_cast<uint32_t>(best >> 32));
            const double v = x > -INFINITY && beam_live(score) ? score + (x - lse) : -static_cast<double>(INFINITY);
            const unsigned long long bits = static_cast<unsigned long long>(__double_as_longlong(v + 0.0));
            value[b][lane] = best && lane < p.select ? bits ^ ((bits >> 63) ? ~0ull : 0x8000000000000000ull) : 0ull;
            token[b][lane] = static_cast<int>(~static_cast<uint32_t>(best));
        }
        __syncthreads();
    }
    if (warp != 0) return;
    // one lane per beam, its best continuation left; the best of these `select` times
    int next = 0, tok = 0;
    unsigned long long val = 0ull;
    auto head = [&] {
        val = lane < p.beams && next < 32 ? value[lane][next] : 0ull;
        tok = lane < p.beams && next < 32 ? token[lane][next] : 0;
    };
    head();
    for (int r = 0; r < p.select; ++r) {
        // the largest value, by its halves; of equal ones the lowest beam, which is the lowest lane
        const uint32_t hi = static_cast<uint32_t>(val >> 32), lo = static_cast<uint32_t>(val);
        const uint32_t h = __reduce_max_sync(0xffffffffu, hi);
        const uint32_t l = __reduce_max_sync(0xffffffffu, hi == h ? lo : 0u);
        if (lane == __ffs(__ballot_sync(0xffffffffu, hi == h && lo == l)) - 1) {
            const unsigned long long b = val ^ ((val >> 63) ? 0x8000000000000000ull : ~0ull);
            const long long at = static_cast<long long>(blockIdx.x) * p.select + r;
            p.out_scores[at] = static_cast<float>(__longlong_as_double(static_cast<long long>(b)));
            p.out_parents[at] = lane;
            p.out_tokens[at] = tok;
            ++next;
            head();
        }
    }
}

}  // namespace kvpd

namespace kvpi {
namespace {

// Segments of a row: about 28 warps for each processor -- what the scan's registers let reside -- in fours, since a
// CTA's warps share what they have found; none shorter than one step.
void plan_beam(const kvp_beam_args& a, int* segs, int* steps) {
    const long long rows = static_cast<long long>(a.batch) * a.beams;
    const long long total = (static_cast<long long>(a.vocab) + 7 + kvpd::kBeamStep - 1) / kvpd::kBeamStep;
    const long long want = (static_cast<long long>(sm_count()) * 28 / std::max<long long>(rows, 1) + 3) / 4 * 4;
    const long long n = std::max<long long>(1, std::min(std::min<long long>(want, kvpd::kBeamSegs), total));
    *steps = static_cast<int>((total + n - 1) / n);
    *segs = static_cast<int>((total + *steps - 1) / *steps);
}

int check_beam(const kvp_beam_args* a) {
    if (!a) return fail(KVP_EINVAL, "null arguments");
    if (!valid_dtype(a->logits_dtype)) return fail(KVP_EINVAL, "unsupported dtype");
    if (a->batch < 0 || a->vocab < 1 || a->beams < 1 || a->select < 1) return fail(KVP_EINVAL, "bad shape");
    if (a->beams > kvpd::kBeamMost || a->select > kvpd::kBeamMost)
        return fail(KVP_EINVAL, "at most 32 beams and 32 selected continuations per request");
    if (a->vocab > (1 << kvpd::kBeamTokenBits)) return fail(KVP_EINVAL, "vocab must be at most 2^26");
    if (static_cast<long long>(a->beams) * a->vocab < a->select)
        return fail(KVP_EINVAL, "fewer continuations than select");
    if (static_cast<long long>(a->batch) * a->beams > (1LL << 24)) return fail(KVP_EINVAL, "too many rows");
    if (a->row_stride != 0 && a->row_stride < a->vocab) return fail(KVP_EINVAL, "row_stride must cover a row");
    return KVP_OK;
}

}  // namespace
}  // namespace kvpi

extern "C" KVP_API size_t kvp_beam_workspace_size(const kvp_beam_args* a) {
    using namespace kvpi;
    clear_error();
    if (check_beam(a) != KVP_OK || a->batch == 0) return 0;
    int segs, steps;
    plan_beam(*a, &segs, &steps);
    const size_t items = static_cast<size_t>(a->batch) * a->beams * segs;
    return (items * 8 + 255) / 256 * 256 + items * a->select * 8;
}

extern "C" KVP_API int kvp_beam_select(const kvp_beam_args* a, void* stream) {
    using namespace kvpi;
    clear_error();
    int rc = check_beam(a);
    if (rc != KVP_OK || a->batch == 0) return rc;
    if (!a->logits || !a->scores || !a->out_scores || !a->out_parents || !a->out_tokens)
        return fail(KVP_EINVAL, "null buffer");
    if (reinterpret_cast<uintptr_t>(a->logits) % dtype_bytes(a->logits_dtype))
        return fail(KVP_EINVAL, "misaligned logits");
    kvpd::BeamParams p;
    plan_beam(*a, &p.segs, &p.seg_steps);
    const size_t items = static_cast<size_t>(a->batch) * a->beams * p.segs;
    const size_t keys_off = (items * 8 + 255) / 256 * 256;
    if (!a->workspace || a->workspace_bytes < keys_off + items * a->select * 8)
        return fail(KVP_ENOSPACE, "workspace smaller than kvp_beam_workspace_size()");
    if ((reinterpret_cast<uintptr_t>(a->workspace) & 15u) != 0)
        return fail(KVP_EINVAL, "workspace must be 16-byte aligned");
    p.logits = a->logits;
    p.scores = a->scores;
    p.out_scores = a->out_scores;
    p.out_parents = a->out_parents;
    p.out_tokens = a->out_tokens;
    p.seg_ml = static_cast<float2*>(a->workspace);
    p.keys = reinterpret_cast<unsigned long long*>(static_cast<char*>(a->workspace) + keys_off);
    p.status = a->status;
    p.row_stride = a->row_stride ? a->row_stride : a->vocab;
    p.batch = a->batch;
    p.beams = a->beams;
    p.vocab = a->vocab;
    p.select = a->select;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const unsigned grid = static_cast<unsigned>(static_cast<size_t>(a->batch) * a->beams *
                                                ((p.segs + kvpd::kBeamWarps - 1) / kvpd::kBeamWarps));
    const bool vec = a->beams == 1 || (p.row_stride * dtype_bytes(a->logits_dtype)) % 16 == 0;
    auto scan = vec ? kvpd::beam_scan_kernel<__nv_bfloat16, true> : kvpd::beam_scan_kernel<__nv_bfloat16, false>;
    if (a->logits_dtype == KVP_DTYPE_F32)
        scan = vec ? kvpd::beam_scan_kernel<float, true> : kvpd::beam_scan_kernel<float, false>;
    else if (a->logits_dtype == KVP_DTYPE_F16)
        scan = vec ? kvpd::beam_scan_kernel<__half, true> : kvpd::beam_scan_kernel<__half, false>;
    scan<<<grid, kvpd::kBeamWarps * 32, 0, s>>>(p);
    rc = cuda_status(cudaGetLastError(), "beam scan launch");
    if (rc != KVP_OK) return rc;
    // the second kernel's launch overlaps the first one's run; it waits for it before its first read
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(a->batch));
    cfg.blockDim = dim3(kvpd::kPickWarps * 32);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, kvpd::beam_pick_kernel, p), "beam pick launch");
}

// Beam selection: of all continuations (beam, token) of a request, the `select` best by
//     value = score[beam] + logit[beam][token] - log(sum over tokens of exp(logit[beam][.])),
// ties to the lower beam, then the lower token.  One read of the logits, two launches.
//
// beam_scan_kernel (bound by HBM): a warp takes one segment of one row.  It keeps a running maximum and sum of
// exponentials per lane, and the segment's best `select` logits as a list sorted over its 32 lanes; within a row the
// order of the values is the order of the logits, so no logarithm is needed here.  The list starts from the lanes' own
// maxima of the first 1024 logits (one sort), so that of the rest only what passes the list's last entry costs more than
// one vote per 256 logits; it is inserted with a ballot and a shift.  Entries are 64-bit keys (ordered logit, ~token):
// all different, so ties fall to the lower token however the segment is cut.
//
// beam_pick_kernel (bound by latency): one CTA per request joins the segments' sums in 64 bits, turns the lists' heads
// into values in 64 bits -- continuations of different beams are ordered by their values, not by a 32-bit rounding --
// and takes the best head `select` times, first within each warp's lists, then over the warps.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "kvp_device.cuh"
#include "kvp_internal.h"

namespace kvpd {

constexpr int kBeamMost = 32;        // beams and selected continuations per request: a warp's lanes
constexpr int kBeamLists = 256;      // lists per request: one per thread of the picking CTA
constexpr int kBeamEntries = 5400;   // and their entries: 42 KB of its shared memory
constexpr int kBeamStep = 1024;      // logits a warp takes at once
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
    int seg_steps;              // kBeamStep logits each
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

template <class T>
struct BeamVec {  // 16-bit logits: 8 per 16-byte vector
    static constexpr int N = 8;
    uint4 u;
    __device__ __forceinline__ void load(const T* p) { u = __ldcs(reinterpret_cast<const uint4*>(p)); }
    __device__ __forceinline__ void get(float (&x)[N]) const {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = F16Traits<T>::unpack_lo(w[i]);
            x[2 * i + 1] = F16Traits<T>::unpack_hi(w[i]);
        }
    }
    static __device__ __forceinline__ float one(const T* p) { return F16Traits<T>::to_float(*p); }
};
template <>
struct BeamVec<float> {
    static constexpr int N = 4;
    float4 u;
    __device__ __forceinline__ void load(const float* p) { u = __ldcs(reinterpret_cast<const float4*>(p)); }
    __device__ __forceinline__ void get(float (&x)[N]) const {
        x[0] = u.x;
        x[1] = u.y;
        x[2] = u.z;
        x[3] = u.w;
    }
    static __device__ __forceinline__ float one(const float* p) { return *p; }
};

// A beam takes part when its score is finite; -inf is a beam that is not in use.
__device__ __forceinline__ bool beam_live(float score) { return score > -INFINITY && score < INFINITY; }

template <class T>
__global__ void __launch_bounds__(128) beam_scan_kernel(const BeamParams p) {
    constexpr int N = BeamVec<T>::N;
    constexpr int NV = kBeamStep / (32 * N);
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31;
    const long long item = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (item >= static_cast<long long>(p.batch) * p.beams * p.segs) return;
    const long long row = item / p.segs;
    const int seg = static_cast<int>(item - row * p.segs);
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
    // vectors start at 16-byte boundaries: token = place - shift
    const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(base) & 15u) / sizeof(T));
    const int end = p.vocab + shift;
    const int first = seg * p.seg_steps * kBeamStep;
    const int last = min(end, first + p.seg_steps * kBeamStep);
    float m = -INFINITY, sum = 0.f;
    unsigned long long best = 0ull, least = 0ull;  // the list (one entry per lane), its entry select - 1
    bool bad = false, seeded = false;
    for (int at = first; at < last; at += kBeamStep) {
        BeamVec<T> raw[NV];
        const bool inside = at >= shift && at + kBeamStep <= end;  // the whole warp's step
        if (inside) {
#pragma unroll
            for (int j = 0; j < NV; ++j) raw[j].load(base + (at + (j * 32 + lane) * N - shift));
        }
        unsigned long long mine = 0ull;  // seeding: this lane's best of the step
#pragma unroll 1
        for (int pass = seeded ? 1 : 0; pass < 2; ++pass) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                float x[N];
                const int place = at + (j * 32 + lane) * N;
                unsigned live = (1u << N) - 1u;
                if (inside) {
                    raw[j].get(x);
                } else {
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const int tok = place + i - shift;
                        const bool in = tok >= 0 && tok < p.vocab;
                        x[i] = in ? BeamVec<T>::one(base + tok) : -INFINITY;
                        if (!in) live &= ~(1u << i);
                    }
                }
                float vm = x[0];
#pragma unroll
                for (int i = 1; i < N; ++i) vm = fmaxf(vm, x[i]);
                // NaN and +inf count as -inf.  A sum shows both: fmaxf drops a NaN, but the sum keeps it.
                float chk = 0.f;
#pragma unroll
                for (int i = 0; i < N; ++i) chk += x[i];
                if (!(chk < INFINITY) || !(vm < INFINITY)) {
                    vm = -INFINITY;
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        if (!(x[i] < INFINITY)) {
                            x[i] = -INFINITY;
                            bad = true;
                        }
                        vm = fmaxf(vm, x[i]);
                    }
                }
                if (pass == 0) {
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const unsigned long long key = (live >> i) & 1u ? beam_key(x[i], place + i - shift) : 0ull;
                        mine = key > mine ? key : mine;
                    }
                    continue;
                }
                const float mn = fmaxf(m, vm);
                if (mn > -INFINITY) {
                    sum *= __expf(m - mn);
                    m = mn;
#pragma unroll
                    for (int i = 0; i < N; ++i) sum += __expf(x[i] - mn);
                }
                const uint32_t least_hi = static_cast<uint32_t>(least >> 32);
                if (!__any_sync(0xffffffffu, ordered32(vm + 0.f) >= least_hi)) continue;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const unsigned long long key = (live >> i) & 1u ? beam_key(x[i], place + i - shift) : 0ull;
                    // entries of the seed come by again: the list never holds a key twice
                    unsigned who = __ballot_sync(0xffffffffu, key > least && key != mine);
                    while (who) {
                        const int src = __ffs(who) - 1;
                        who &= who - 1;
                        const unsigned long long add = __shfl_sync(0xffffffffu, key, src);
                        if (add <= least) continue;
                        const int rank = __popc(__ballot_sync(0xffffffffu, best > add));
                        const unsigned long long up = __shfl_up_sync(0xffffffffu, best, 1);
                        best = lane < rank ? best : lane == rank ? add : up;
                        least = __shfl_sync(0xffffffffu, best, p.select - 1);
                    }
                }
            }
            if (pass == 0) {
                best = warp_sort_desc(mine, lane);
                least = __shfl_sync(0xffffffffu, best, p.select - 1);
                seeded = true;
            }
        }
    }
    float top = m;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    float total = top > -INFINITY ? sum * __expf(m - top) : 0.f;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
    if (lane == 0) p.seg_ml[item] = make_float2(top, total);
    if (lane < p.select) out[lane] = best;
    if (bad) report(p.status, KVP_STATUS_BAD_VALUE);
}

// The best of the warp's heads: (value as two ordered halves, then the lower place); the lane that holds it.
__device__ __forceinline__ int best_lane(uint32_t hi, uint32_t lo, uint32_t place) {
    const uint32_t h = __reduce_max_sync(0xffffffffu, hi);
    const uint32_t l = __reduce_max_sync(0xffffffffu, hi == h ? lo : 0u);
    const bool in = hi == h && lo == l;
    const uint32_t w = __reduce_min_sync(0xffffffffu, in ? place : 0xffffffffu);
    return __ffs(__ballot_sync(0xffffffffu, in && place == w)) - 1;
}

struct BeamEntry {
    uint32_t hi, lo, place;  // ordered 64-bit value (0, 0: none), beam << 26 | token
};

__global__ void __launch_bounds__(kBeamLists) beam_pick_kernel(const BeamParams p) {
    extern __shared__ unsigned long long keys[];  // [lists][select]
    __shared__ double lse[kBeamMost];
    __shared__ BeamEntry won[kBeamLists / 32][kBeamMost];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int lists = p.beams * p.segs, warps = (lists + 31) >> 5;
    const long long list0 = static_cast<long long>(blockIdx.x) * lists;
    griddep_wait();
    for (int i = threadIdx.x; i < lists * p.select; i += blockDim.x) keys[i] = __ldcg(p.keys + list0 * p.select + i);
    // log-sum-exp of each beam, a warp per beam
    for (int b = warp; b < p.beams; b += blockDim.x >> 5) {
        float top = -INFINITY;
        for (int s = lane; s < p.segs; s += 32) top = fmaxf(top, __ldcg(p.seg_ml + list0 + b * p.segs + s).x);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        double total = 0.0;
        if (top > -INFINITY)
            for (int s = lane; s < p.segs; s += 32) {
                const float2 ml = __ldcg(p.seg_ml + list0 + b * p.segs + s);
                if (ml.x > -INFINITY) total += static_cast<double>(ml.y) * exp(static_cast<double>(ml.x) - top);
            }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
        if (lane == 0) lse[b] = top > -INFINITY ? top + log(total) : -static_cast<double>(INFINITY);
    }
    __syncthreads();
    // each lane's list, its head as a value in 64 bits
    BeamEntry e{0u, 0u, 0xffffffffu};
    int next = 0;
    const int list = threadIdx.x, beam = list / p.segs;
    auto head = [&] {
        e = BeamEntry{0u, 0u, 0xffffffffu};
        if (list >= lists || next >= p.select) return;
        const unsigned long long key = keys[list * p.select + next];
        if (!key) return;
        const float x = unordered32(static_cast<uint32_t>(key >> 32));
        const float score = __ldg(p.scores + static_cast<long long>(blockIdx.x) * p.beams + beam);
        const double v = x > -INFINITY && beam_live(score) ? score + (x - lse[beam]) : -static_cast<double>(INFINITY);
        const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(v + 0.0));
        const unsigned long long o = b ^ ((b >> 63) ? ~0ull : 0x8000000000000000ull);
        e = BeamEntry{static_cast<uint32_t>(o >> 32), static_cast<uint32_t>(o),
                      (static_cast<uint32_t>(beam) << kBeamTokenBits) | ~static_cast<uint32_t>(key)};
    };
    if (warp < warps) {
        head();
        for (int r = 0; r < p.select; ++r) {
            const int w = best_lane(e.hi, e.lo, e.place);
            if (lane == w) {
                won[warp][r] = e;
                ++next;
                head();
            }
        }
    }
    __syncthreads();
    if (warp != 0) return;
    next = 0;
    e = lane < warps ? won[lane][0] : BeamEntry{0u, 0u, 0xffffffffu};
    for (int r = 0; r < p.select; ++r) {
        const int w = best_lane(e.hi, e.lo, e.place);
        if (lane == w) {
            const unsigned long long o = (static_cast<unsigned long long>(e.hi) << 32) | e.lo;
            const unsigned long long b = o ^ ((o >> 63) ? 0x8000000000000000ull : ~0ull);
            const long long at = static_cast<long long>(blockIdx.x) * p.select + r;
            p.out_scores[at] = static_cast<float>(__longlong_as_double(static_cast<long long>(b)));
            p.out_parents[at] = static_cast<int32_t>(e.place >> kBeamTokenBits);
            p.out_tokens[at] = static_cast<int32_t>(e.place & ((1u << kBeamTokenBits) - 1u));
            ++next;
            e = next < p.select && lane < warps ? won[lane][next] : BeamEntry{0u, 0u, 0xffffffffu};
        }
    }
}

}  // namespace kvpd

namespace kvpi {
namespace {

// Segments of a row: enough warps to fill the GPU about twice (32 resident warps an SM cover the memory latency with
// four 16-byte loads a lane each), none shorter than one step, and no more lists per request than the picking CTA has
// threads and shared memory for.
void plan_beam(const kvp_beam_args& a, int* segs, int* steps) {
    const long long rows = static_cast<long long>(a.batch) * a.beams;
    const long long total = (static_cast<long long>(a.vocab) + 7 + kvpd::kBeamStep - 1) / kvpd::kBeamStep;
    const long long want = std::max<long long>(1, static_cast<long long>(sm_count()) * 64 / std::max<long long>(rows, 1));
    const long long most = std::min(kvpd::kBeamLists / a.beams, kvpd::kBeamEntries / (a.beams * a.select));
    const long long n = std::min(std::min(want, most), total);
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
    if (!a->logits || !a->scores || !a->out_scores || !a->out_parents || !a->out_tokens) return fail(KVP_EINVAL, "null buffer");
    if (reinterpret_cast<uintptr_t>(a->logits) % dtype_bytes(a->logits_dtype)) return fail(KVP_EINVAL, "misaligned logits");
    kvpd::BeamParams p;
    plan_beam(*a, &p.segs, &p.seg_steps);
    const size_t items = static_cast<size_t>(a->batch) * a->beams * p.segs;
    const size_t keys_off = (items * 8 + 255) / 256 * 256;
    if (!a->workspace || a->workspace_bytes < keys_off + items * a->select * 8)
        return fail(KVP_ENOSPACE, "workspace smaller than kvp_beam_workspace_size()");
    if ((reinterpret_cast<uintptr_t>(a->workspace) & 15u) != 0) return fail(KVP_EINVAL, "workspace must be 16-byte aligned");
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
    const unsigned grid = static_cast<unsigned>((items + 3) / 4);
    if (a->logits_dtype == KVP_DTYPE_F32)
        kvpd::beam_scan_kernel<float><<<grid, 128, 0, s>>>(p);
    else if (a->logits_dtype == KVP_DTYPE_F16)
        kvpd::beam_scan_kernel<__half><<<grid, 128, 0, s>>>(p);
    else
        kvpd::beam_scan_kernel<__nv_bfloat16><<<grid, 128, 0, s>>>(p);
    rc = cuda_status(cudaGetLastError(), "beam scan launch");
    if (rc != KVP_OK) return rc;
    // the second kernel's launch overlaps the first one's run; it waits for it before its first read
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(a->batch));
    cfg.blockDim = dim3(kvpd::kBeamLists);
    cfg.dynamicSmemBytes = static_cast<size_t>(a->beams) * p.segs * a->select * 8;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, kvpd::beam_pick_kernel, p), "beam pick launch");
}

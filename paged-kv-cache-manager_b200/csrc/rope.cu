// One layer's new rows on their way into the cache: RMS norms of the query and key heads, the position rotation,
// the queries (and, where asked for, the keys) written out, keys and values stored into their slots.
//
//   norm (optional, per head):  x <- w * x / sqrt(mean(x^2) + eps)
//   rotation of the first `rot` elements of a head at position p, with c = table[p][i], s = table[p][rot/2 + i]:
//     halves:       (x[i], x[i + rot/2])   <- (x[i] c - x[i + rot/2] s,  x[i + rot/2] c + x[i] s)
//     interleaved:  (x[2i], x[2i + 1])     <- (x[2i] c - x[2i + 1] s,    x[2i + 1] c + x[2i] s)
//
// Byte movement with a few flops per element: bound by HBM for a prompt and by launch latency for a decode step.  A
// thread owns 16 elements of a head as two 8-element vectors, placed so that every rotated pair lies in one
// thread (halves: elements 8u.. and rot/2 + 8u..; interleaved, and the part behind `rot`: 16 in a row), so the
// rotation needs no exchange and the norm one shuffle reduction over the head's lanes.  A lane owns the same element
// offsets in every head, so the token's cos/sin values (fp32, twice the bytes of a head of bf16) are read once
// per warp and stay in registers over its heads.  All arithmetic is fp32; each output is rounded once.
#include <cuda_runtime.h>

#include <algorithm>

#include "kvp_device.cuh"
#include "kvp_internal.h"

namespace kvpd {

struct RopeParams {
    const void* q;
    const void* k;
    const void* v;
    void* q_out;
    void* k_out;
    void* k_cache;
    void* v_cache;
    const int32_t* slots;
    const int32_t* positions;
    const float* table;
    const void* q_norm;
    const void* k_norm;
    int32_t* status;
    long long q_stride, k_stride, v_stride, q_out_stride, k_out_stride;  // elements between tokens
    long long num_slots;                                                // of the cache
    float eps, inv_dim;
    int tokens, nh, kvh, rows;  // rows: head rows per token (nh + kvh, + kvh with a cache)
    int dim, units, rot, interleaved, max_positions, out_dtype, kv_dtype;
    int chunks, per_chunk;  // warps per token and warp iterations of each
};

// 8 consecutive elements as floats, and back.
struct Vec8 {
    float x[8];
};
template <class T>
__device__ __forceinline__ Vec8 unpack8(uint4 u) {
    Vec8 r;
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r.x[2 * i] = F16Traits<T>::unpack_lo(w[i]);
        r.x[2 * i + 1] = F16Traits<T>::unpack_hi(w[i]);
    }
    return r;
}
template <class T>
__device__ __forceinline__ uint4 pack8(const Vec8& a) {
    return make_uint4(F16Traits<T>::pack(a.x[0], a.x[1]), F16Traits<T>::pack(a.x[2], a.x[3]),
                      F16Traits<T>::pack(a.x[4], a.x[5]), F16Traits<T>::pack(a.x[6], a.x[7]));
}

// Raw storage of 8 input elements: loads are issued for several heads before any is unpacked.
template <class T>
struct Raw8 {
    uint4 u;
    __device__ __forceinline__ void load(const T* p) { u = __ldcs(reinterpret_cast<const uint4*>(p)); }
    __device__ __forceinline__ void load_kept(const T* p) { u = __ldg(reinterpret_cast<const uint4*>(p)); }
    __device__ __forceinline__ Vec8 get() const { return unpack8<T>(u); }
};
template <>
struct Raw8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = __ldcs(reinterpret_cast<const float4*>(p));
        b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
    }
    __device__ __forceinline__ void load_kept(const float* p) {
        a = __ldg(reinterpret_cast<const float4*>(p));
        b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    }
    __device__ __forceinline__ Vec8 get() const { return Vec8{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}}; }
};

__device__ __forceinline__ void store8(void* base, long long at, int dtype, const Vec8& a) {
    if (dtype == KVP_DTYPE_F32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + at);
        p[0] = make_float4(a.x[0], a.x[1], a.x[2], a.x[3]);
        p[1] = make_float4(a.x[4], a.x[5], a.x[6], a.x[7]);
    } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + at) =
            dtype == KVP_DTYPE_F16 ? pack8<__half>(a) : pack8<__nv_bfloat16>(a);
    }
}

// LPH: lanes per head, the power of two at or above dim / 16.  U: heads per lane group in flight.
// A long prompt (16384 tokens, 32 + 8 + 8 heads of 128, norms): 411 MB in 82 us, 5.0 TB/s, 77% of a copy's rate, with
// the instructions (270 a warp for 4 heads of 128) taking 64% of the issue slots.  Two heads in flight and six CTAs an
// SM: four heads and five CTAs took 88 us; a coefficient form of norm and rotation in paired operations took fewer
// instructions, but 150 registers and 114 us; a token's rows spread over three warps 104 us, for its position and table
// read thrice.
// A decode step (1 to 256 tokens) takes 2.5 to 3.4 us on the GPU, the latencies of position, table row and heads in
// turn.
template <class T, int LPH, int U>
__global__ void __launch_bounds__(128, sizeof(T) == 4 ? 4 : 6) rope_append_kernel(const RopeParams p) {
    constexpr int HPW = 32 / LPH;  // heads a warp takes at once
    const int lane = threadIdx.x & 31;
    const int u = lane & (LPH - 1);
    const bool on = u < p.units;
    // this lane's two vectors of a head, and where its cos/sin values start in a table row (-1: not rotated)
    int ea = 16 * u, eb = ea + 8, ca = -1;
    if (ea < p.rot) {
        if (p.interleaved) {
            ca = 8 * u;
        } else {
            ea = 8 * u;
            eb = ea + (p.rot >> 1);
            ca = ea;
        }
    }
    const long long items = static_cast<long long>(p.tokens) * p.chunks;
    const long long stride = static_cast<long long>(gridDim.x) * (blockDim.x >> 5);
    const long long it0 = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
    for (long long it = it0; it < items; it += stride) {
        const long long tok = p.chunks == 1 ? it : it / p.chunks;
        const int chunk = static_cast<int>(it - tok * p.chunks);
        const int pos = __ldg(p.positions + tok);
        const int slot = p.slots ? __ldg(p.slots + tok) : -1;
        if (pos < 0) continue;  // padding
        if (pos >= p.max_positions) {
            if (lane == 0 && chunk == 0) report(p.status, KVP_STATUS_BAD_POSITION);
            continue;
        }
        const bool cached = slot >= 0 && slot < p.num_slots;
        if (slot >= 0 && !cached && lane == 0 && chunk == 0) report(p.status, KVP_STATUS_BAD_BLOCK);
        Vec8 c, s;
        if (on && ca >= 0) {
            const float4* t = reinterpret_cast<const float4*>(p.table + static_cast<long long>(pos) * p.rot + ca);
            const float4* t2 = reinterpret_cast<const float4*>(p.table + static_cast<long long>(pos) * p.rot +
                                                               (p.rot >> 1) + ca);
            const float4 c0 = __ldg(t), c1 = __ldg(t + 1), s0 = __ldg(t2), s1 = __ldg(t2 + 1);
            c = Vec8{{c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w}};
            s = Vec8{{s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w}};
        }
        const int row_end = min(p.rows, (chunk + 1) * p.per_chunk * HPW);
        for (int row0 = chunk * p.per_chunk * HPW + lane / LPH; row0 - lane / LPH < row_end; row0 += U * HPW) {
            Raw8<T> ra[U], rb[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int row = row0 + j * HPW;
                if (row < row_end && on) {
                    const T* src = row < p.nh ? static_cast<const T*>(p.q) + tok * p.q_stride + row * p.dim
                                 : row < p.nh + p.kvh
                                     ? static_cast<const T*>(p.k) + tok * p.k_stride + (row - p.nh) * p.dim
                                     : static_cast<const T*>(p.v) + tok * p.v_stride + (row - p.nh - p.kvh) * p.dim;
                    ra[j].load(src + ea);
                    rb[j].load(src + eb);
                }
            }
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int row = row0 + j * HPW;
                const bool live = row < row_end && on;
                const bool is_q = row < p.nh, is_k = !is_q && row < p.nh + p.kvh;
                Vec8 a{}, b{};
                if (live) {
                    a = ra[j].get();
                    b = rb[j].get();
                }
                if (p.q_norm || p.k_norm) {  // the same for the whole grid: every lane takes part in the reduction
                    const void* w = is_q ? p.q_norm : is_k ? p.k_norm : nullptr;
                    float ss = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) ss += a.x[i] * a.x[i] + b.x[i] * b.x[i];
#pragma unroll
                    for (int off = 1; off < LPH; off <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
                    if (w && live) {
                        const float r = rsqrtf(ss * p.inv_dim + p.eps);
                        Raw8<T> wa, wb;
                        wa.load_kept(static_cast<const T*>(w) + ea);
                        wb.load_kept(static_cast<const T*>(w) + eb);
                        const Vec8 fa = wa.get(), fb = wb.get();
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            a.x[i] *= r * fa.x[i];
                            b.x[i] *= r * fb.x[i];
                        }
                    }
                }
                if (!live) continue;
                if (ca >= 0 && (is_q || is_k)) {
                    if (p.interleaved) {
                        // a holds pairs 0..3 of this lane's eight, b pairs 4..7
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float a0 = a.x[2 * i], a1 = a.x[2 * i + 1], b0 = b.x[2 * i], b1 = b.x[2 * i + 1];
                            a.x[2 * i] = a0 * c.x[i] - a1 * s.x[i];
                            a.x[2 * i + 1] = a1 * c.x[i] + a0 * s.x[i];
                            b.x[2 * i] = b0 * c.x[4 + i] - b1 * s.x[4 + i];
                            b.x[2 * i + 1] = b1 * c.x[4 + i] + b0 * s.x[4 + i];
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float x0 = a.x[i], x1 = b.x[i];
                            a.x[i] = x0 * c.x[i] - x1 * s.x[i];
                            b.x[i] = x1 * c.x[i] + x0 * s.x[i];
                        }
                    }
                }
                if (is_q) {
                    const long long at = tok * p.q_out_stride + row * p.dim;
                    store8(p.q_out, at + ea, p.out_dtype, a);
                    store8(p.q_out, at + eb, p.out_dtype, b);
                    continue;
                }
                const int h = row - (is_k ? p.nh : p.nh + p.kvh);
                if (is_k && p.k_out) {
                    const long long at = tok * p.k_out_stride + h * p.dim;
                    store8(p.k_out, at + ea, p.out_dtype, a);
                    store8(p.k_out, at + eb, p.out_dtype, b);
                }
                if (cached) {
                    void* pool = is_k ? p.k_cache : p.v_cache;
                    const long long at = (static_cast<long long>(slot) * p.kvh + h) * p.dim;
                    store8(pool, at + ea, p.kv_dtype, a);
                    store8(pool, at + eb, p.kv_dtype, b);
                }
            }
        }
    }
}

template <class T, int LPH>
int launch_rope(const RopeParams& p0, cudaStream_t s) {
    RopeParams p = p0;
    constexpr int U = 2;
    constexpr int kWarps = 4;
    const int iters = (p.rows + 32 / LPH - 1) / (32 / LPH);  // warp iterations of a token
    // Few tokens: a token's heads are spread over several warps, so that the launch's latency is that of one head;
    // from about 16 warps per SM on one warp keeps its token and reads the cos/sin row once.
    const long long want = static_cast<long long>(kvpi::sm_count()) * 16;
    p.chunks = static_cast<int>(std::min<long long>(iters, std::max<long long>(1, want / p.tokens)));
    p.per_chunk = (iters + p.chunks - 1) / p.chunks;
    p.chunks = (iters + p.per_chunk - 1) / p.per_chunk;
    const long long items = static_cast<long long>(p.tokens) * p.chunks;
    const long long grid = std::min<long long>((items + kWarps - 1) / kWarps,
                                               static_cast<long long>(kvpi::sm_count()) * 16);
    rope_append_kernel<T, LPH, U><<<static_cast<unsigned>(grid), kWarps * 32, 0, s>>>(p);
    return kvpi::cuda_status(cudaGetLastError(), "rope append launch");
}

template <class T>
int launch_rope_lanes(const RopeParams& p, cudaStream_t s) {
    if (p.units <= 1) return launch_rope<T, 1>(p, s);
    if (p.units <= 2) return launch_rope<T, 2>(p, s);
    if (p.units <= 4) return launch_rope<T, 4>(p, s);
    if (p.units <= 8) return launch_rope<T, 8>(p, s);
    return launch_rope<T, 16>(p, s);
}

}  // namespace kvpd

extern "C" KVP_API int kvp_rope_append(const kvp_rope_args* a, void* stream) {
    using namespace kvpi;
    clear_error();
    if (!a) return fail(KVP_EINVAL, "null arguments");
    if (!valid_dtype(a->in_dtype) || !valid_dtype(a->out_dtype)) return fail(KVP_EINVAL, "unsupported dtype");
    if (a->num_tokens < 0 || a->num_heads < 1 || a->kv_heads < 1 || a->max_positions < 1)
        return fail(KVP_EINVAL, "bad shape");
    if (a->head_dim < 16 || a->head_dim > 256 || a->head_dim % 16 != 0)
        return fail(KVP_EINVAL, "head_dim must be a multiple of 16, at most 256");
    if (a->rot_dim < 16 || a->rot_dim > a->head_dim || a->rot_dim % 16 != 0)
        return fail(KVP_EINVAL, "rot_dim must be a multiple of 16, at most head_dim");
    if (static_cast<long long>(a->num_heads) + 2LL * a->kv_heads > (1 << 20)) return fail(KVP_EINVAL, "too many heads");
    const bool cache = a->k_cache != nullptr || a->v_cache != nullptr || a->slots != nullptr;
    if (cache) {
        if (!a->k_cache || !a->v_cache || (a->num_tokens > 0 && (!a->slots || !a->v)))
            return fail(KVP_EINVAL, "v, k_cache, v_cache and slots go together");
        if (!(a->kv_dtype == KVP_DTYPE_F16 || a->kv_dtype == KVP_DTYPE_BF16))
            return fail(KVP_EINVAL, "pool dtype must be fp16 or bf16");
        if (a->block_size < 1 || a->num_blocks < 1 || a->num_blocks > INT64_MAX / a->block_size)
            return fail(KVP_EINVAL, "block_size and num_blocks bound the slots");
        if (!aligned16(a->k_cache) || !aligned16(a->v_cache)) return fail(KVP_EINVAL, "pools must be 16-byte aligned");
    } else if (!a->k_out) {
        return fail(KVP_EINVAL, "the keys need k_out or a cache");
    }
    if (!(a->eps >= 0.f) && (a->q_norm || a->k_norm)) return fail(KVP_EINVAL, "eps must not be negative");
    const long long qrow = static_cast<long long>(a->num_heads) * a->head_dim;
    const long long krow = static_cast<long long>(a->kv_heads) * a->head_dim;
    kvpd::RopeParams p;
    p.q_stride = a->q_stride ? a->q_stride : qrow;
    p.k_stride = a->k_stride ? a->k_stride : krow;
    p.v_stride = a->v_stride ? a->v_stride : krow;
    p.q_out_stride = a->q_out_stride ? a->q_out_stride : qrow;
    p.k_out_stride = a->k_out_stride ? a->k_out_stride : krow;
    const int in_b = dtype_bytes(a->in_dtype), out_b = dtype_bytes(a->out_dtype);
    if (p.q_stride < qrow || p.k_stride < krow || p.q_out_stride < qrow || p.k_out_stride < krow ||
        (cache && p.v_stride < krow))
        return fail(KVP_EINVAL, "token strides must cover a token's heads");
    if ((p.q_stride * in_b) % 16 || (p.k_stride * in_b) % 16 || (cache && (p.v_stride * in_b) % 16) ||
        (p.q_out_stride * out_b) % 16 || (p.k_out_stride * out_b) % 16)
        return fail(KVP_EINVAL, "token strides must be multiples of 16 bytes");
    if (a->num_tokens == 0) return KVP_OK;
    if (!a->q || !a->k || !a->q_out || !a->positions || !a->table) return fail(KVP_EINVAL, "null buffer");
    if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->q_out) || !aligned16(a->k_out) ||
        !aligned16(a->table) || !aligned16(a->q_norm) || !aligned16(a->k_norm))
        return fail(KVP_EINVAL, "buffers must be 16-byte aligned");
    p.q = a->q;
    p.k = a->k;
    p.v = a->v;
    p.q_out = a->q_out;
    p.k_out = a->k_out;
    p.k_cache = a->k_cache;
    p.v_cache = a->v_cache;
    p.slots = a->slots;
    p.positions = a->positions;
    p.table = a->table;
    p.q_norm = a->q_norm;
    p.k_norm = a->k_norm;
    p.status = a->status;
    p.num_slots = cache ? a->num_blocks * static_cast<long long>(a->block_size) : 0;
    p.eps = a->eps;
    p.inv_dim = 1.0f / static_cast<float>(a->head_dim);
    p.tokens = a->num_tokens;
    p.nh = a->num_heads;
    p.kvh = a->kv_heads;
    p.rows = a->num_heads + a->kv_heads * (cache ? 2 : 1);
    p.dim = a->head_dim;
    p.units = a->head_dim / 16;
    p.rot = a->rot_dim;
    p.interleaved = a->interleaved ? 1 : 0;
    p.max_positions = a->max_positions;
    p.out_dtype = a->out_dtype;
    p.kv_dtype = a->kv_dtype;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a->in_dtype == KVP_DTYPE_F32) return kvpd::launch_rope_lanes<float>(p, s);
    if (a->in_dtype == KVP_DTYPE_F16) return kvpd::launch_rope_lanes<__half>(p, s);
    return kvpd::launch_rope_lanes<__nv_bfloat16>(p, s);
}

// The balanced attention kernel over the own parts of sequences in groups: 16-bit pools, queries of their dtype.
#include "attention_kernels.cuh"

namespace kvpd {

template <class KV>
static int launch_own_kv(const kvp_attn_args& a, const kvpi::AttnPlan& pl, const AttnParams& prm, const CUtensorMap& km,
                         const CUtensorMap& vm, cudaStream_t s) {
    const bool wide = prm.g > 8;  // two n-tiles of query heads per kv head
    if (a.head_dim == 64)
        return wide ? launch_own<64, 2, KV>(pl, prm, km, vm, s) : launch_own<64, 1, KV>(pl, prm, km, vm, s);
    if (a.head_dim == 128)
        return wide ? launch_own<128, 2, KV>(pl, prm, km, vm, s) : launch_own<128, 1, KV>(pl, prm, km, vm, s);
    return kvpi::fail(KVP_EINVAL, "unsupported head_dim");
}

int launch_own_parts(const kvp_attn_args& a, const kvpi::AttnPlan& pl, const AttnParams& prm, const CUtensorMap& km,
                     const CUtensorMap& vm, cudaStream_t s) {
    if (!pl.streamk) return kvpi::fail(KVP_EINVAL, "the own parts need the balanced schedule");
    return a.kv_dtype == KVP_DTYPE_F16 ? launch_own_kv<__half>(a, pl, prm, km, vm, s)
                                       : launch_own_kv<__nv_bfloat16>(a, pl, prm, km, vm, s);
}

}  // namespace kvpd

// Attention kernels over a KV cache (kv_attention.cuh holds the mathematics and the measurements).  The Makefile compiles this
// file once per cache format and head dimension, with KV_BITS and KV_DIM set, and once without them for the choice among them.
#ifdef KV_BITS

#include "kv_attention.cuh"
#include "kv_attention_tc.cuh"

namespace kcb {
template <>
int attn_launch<KV_BITS, KV_DIM>(const AttnP& P, bool general, AttnKernel which, cudaStream_t st) {
    return attn_launch_kernels<KV_DIM, KV_BITS>(P, general, which, st);
}
#if KV_BITS == 16 && (KV_DIM == 64 || KV_DIM == 128)
template <>
int attn_launch_tc_dim<KV_DIM>(const AttnP& P, bool general, cudaStream_t st) {
    return attn_launch_tc<KV_DIM, 16>(P, general, st);
}
#endif
#if KV_DIM == 64 || KV_DIM == 128
template <>
unsigned attn_timeouts_of<KV_BITS, KV_DIM>() {
    return attn_timeouts_here();
}
#endif
}  // namespace kcb

#else

#include "common.cuh"
#include "kv_cache.h"

namespace kcb {
template <int BITS>
static int attn_launch_dim(const AttnP& P, int head_dim, bool general, AttnKernel which, cudaStream_t st) {
    switch (head_dim) {
    case 32: return attn_launch<BITS, 32>(P, general, which, st);
    case 64: return attn_launch<BITS, 64>(P, general, which, st);
    case 96: return attn_launch<BITS, 96>(P, general, which, st);
    case 128: return attn_launch<BITS, 128>(P, general, which, st);
    case 256: return attn_launch<BITS, 256>(P, general, which, st);
    }
    return KCB_UNSUPPORTED_OPERATION;
}
int attn_launch_bits(const AttnP& P, int bits, int head_dim, bool general, AttnKernel which, cudaStream_t st) {
    return bits == KCB_CACHE_F16 ? attn_launch_dim<16>(P, head_dim, general, which, st) : attn_launch_dim<4>(P, head_dim, general, which, st);
}
unsigned attn_timeouts() { return attn_timeouts_of<16, 64>() + attn_timeouts_of<16, 128>() + attn_timeouts_of<4, 64>() + attn_timeouts_of<4, 128>(); }
}  // namespace kcb

#endif

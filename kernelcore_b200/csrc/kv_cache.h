// Internal declarations of the KV-cache operators (kv_cache.cu, kv_attention.cu).
#pragma once

#include "../../include/kernelcore_b200.h"

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace kcb {

constexpr int kMaxSmem = 227 * 1024;  // dynamic shared memory a CTA may ask for on sm_100

struct AttnP;
// One instance per cache format and head dimension (kv_attention.cu), and the choice among them.
enum class AttnKernel { rows, tile, tc };
template <int BITS, int D>
int attn_launch(const AttnP& P, bool general, AttnKernel which, cudaStream_t st);
// The tcgen05 kernel for fp16 caches, built for 64 and 128 channels; P.dim may be smaller (the rest is zeros).
template <int D>
int attn_launch_tc_dim(const AttnP& P, bool general, cudaStream_t st);
template <int BITS, int D>
unsigned attn_timeouts_of();
int attn_launch_bits(const AttnP& P, int bits, int head_dim, bool general, AttnKernel which, cudaStream_t st);
unsigned attn_timeouts();  // bounded waits of the attention kernels that expired since load; synchronous

// Bytes of one sequence's keys (or values) in the 4-bit format, and where its parameter plane begins.
inline size_t q4_param_offset(int kv_heads, int head_dim, int capacity) { return static_cast<size_t>(kv_heads) * capacity * (head_dim / 2); }
inline size_t q4_seq_bytes(int kv_heads, int head_dim, int capacity) {
    return (static_cast<size_t>(kv_heads) * capacity * (head_dim / 2 + head_dim / 8) + 15) / 16 * 16;
}

}  // namespace kcb

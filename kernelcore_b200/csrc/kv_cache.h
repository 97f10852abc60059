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
template <int BITS, int D>
int attn_launch(const AttnP& P, bool general, bool tile, cudaStream_t st);
int attn_launch_bits(const AttnP& P, int bits, int head_dim, bool general, bool tile, cudaStream_t st);

// Bytes of one sequence's keys (or values) in the 4-bit format, and where its parameter plane begins.
inline size_t q4_param_offset(int kv_heads, int head_dim, int capacity) { return static_cast<size_t>(kv_heads) * capacity * (head_dim / 2); }
inline size_t q4_seq_bytes(int kv_heads, int head_dim, int capacity) {
    return (static_cast<size_t>(kv_heads) * capacity * (head_dim / 2 + head_dim / 8) + 15) / 16 * 16;
}

}  // namespace kcb

// Attention over a KV cache held in fp16 or in 4 bits, with capped or distance-biased scores and causal, prefix, document
// or additive masks: the kernels, as templates over (head dimension, cache format, general scores).  Included by one
// translation unit per format and head dimension (kv_attention.cu).
//
// Per sequence, kv head and query row (a row is one head of the group at one token), over the visible key slots t:
//     z_t = scale q.k_t;  z_t = cap tanh(z_t / cap);  z_t += bias;   out = sum_t softmax(z)_t v_t
// computed in one pass with the running maximum and sum of the softmax, in base 2 (scores are multiplied by log2 e).
//
// Precision.  Queries, outputs and every sum are fp32, but the products run on the tensor cores, whose operands are fp16:
// a query (scaled per row by a power of two so that its largest element is about 2^11) and a probability (times 2^12) are
// each split into the sum of two fp16 numbers, hi + lo, 22 bits together, and both halves are multiplied.  An fp16 key or
// value is exact as it is, and so is a 4-bit code (code_pair below).  The scale d and the minimum m of a block of 32 channels stay
// outside the products:
//     q.k = sum_b d_b (q_b . code_b) + m_b sum(q_b),       sum_t p_t v_t = sum_t (p_t d_tb) (code_t - 8) + sum_t p_t (m_tb + 8 d_tb).
// Values are taken about the middle of their block: over a long context they average to far less than a block's range, and two
// sums of the range's size that cancel would cost digits (131072 keys: four times the error).
#pragma once

#include "common.cuh"
#include "kv_cache.h"

#include <cuda_fp16.h>

namespace kcb {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPShift = 12.0f;  // probabilities enter the products times 2^12
constexpr int kRowsMax = 32;      // a rows launch takes at most this many query rows per kv head (the join keeps that many sums)

// Everything a launch needs, by value.  Strides are in elements (halves, floats).
struct AttnP {
    const uint8_t* k;
    const uint8_t* v;
    long long k_row, k_head, k_seq, v_row, v_head, v_seq;  // fp16 caches
    long long par_off, seq_bytes;                          // 4-bit caches: offset of the parameter plane, bytes of a sequence
    const float* q;
    float* out;
    long long q_token, q_head, q_seq, o_token, o_head, o_seq;
    const int* n_keys;
    const int* next_pos;
    const int* positions;
    float* weights;
    const int* prefix;
    const int* q_pos;
    const int* q_doc;
    const int* k_doc;
    const unsigned short* mask;
    long long mask_token, mask_seq;
    int dim, cap, n_seqs, n_tokens, heads, kv_heads, group, rows;  // rows = n_tokens * group
    int causal, bias_log2_heads;                      // bias_log2_heads: largest power of two <= heads
    float sc;                                         // score factor: scale * log2 e, or scale / cap with a cap
    float cap_out;                                    // cap * log2 e, 0 without a cap
    float bias_step;                                  // max_bias / bias_log2_heads, 0 without a bias
    int nsplit, row_tiles;
    float* part_o;   // [seq][kv head][split][row][D]
    float2* part_ml; // [seq][kv head][split][row] {maximum, sum}
    float2* final_ml;  // [seq][kv head][row], for the weights of a tile launch, else null
    float* scores;     // [seq][kv head][row][capacity], for the weights of a rows launch, else null (part_ml is written then)
};

// A kernel launched with launch_dependent may start while its predecessor in the stream still runs; it touches nothing that the
// predecessor writes before this wait.  The predecessor lets it start early with the second call.
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dependents_may_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <class... P, class... A>
inline int launch_clusters(void (*kernel)(P...), dim3 grid, int cluster, int threads, size_t smem, cudaStream_t st, A... args) {  // cluster: CTAs along x
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid, cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster), attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = cluster > 1 ? 2 : 1;
    if (cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess) return KCB_SUCCESS;
    cudaGetLastError();
    return KCB_LAUNCH_FAILURE;
}

template <class... P, class... A>
inline int launch_dependent(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, A... args) {
    return launch_clusters(kernel, grid, 1, threads, smem, st, args...);
}

// ---- small device helpers ------------------------------------------------------------------------------------------
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_small(uint32_t dst, const void* src, bool ok) {  // N = 4 or 8 bytes
    asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(ok ? N : 0), "n"(N) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(unsigned (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(unsigned (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
// c += A (16 x 16, row) * B (16 x 8, column), fp16 operands, fp32 sums
__device__ __forceinline__ void mma16816(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two codes out of a word of nibbles as fp16 numbers: code * 2^-10, or (code - 8) * 2^-10; SHIFT: they stand four bits up.
// The nibble's bits are the subnormal number code * 2^-24 (times 16 when shifted), which one multiply-add brings up and moves.
// (The subnormals themselves would multiply exactly too, but the tensor cores align their products as if they were 2^-14: six to
// ten of the sum's 24 bits are lost.)
template <bool SHIFT, bool CENTRED>
__device__ __forceinline__ unsigned code_pair(unsigned w) {
    const unsigned n = w & (SHIFT ? 0x00F000F0u : 0x000F000Fu);
    unsigned r;
    if (CENTRED) asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(n), "r"(SHIFT ? 0x64006400u : 0x74007400u), "r"(0xA000A000u));  // * 2^10 or 2^14, - 2^-7
    else asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(n), "r"(SHIFT ? 0x64006400u : 0x74007400u));
    return r;
}
// Packed fp32 pairs (one instruction for two values, each rounded as the scalar operation).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)), "l"(reinterpret_cast<unsigned long long&>(c)));
    return reinterpret_cast<float2&>(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return reinterpret_cast<float2&>(r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return reinterpret_cast<float2&>(r);
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ unsigned h2_bits(__half2 h) { return *reinterpret_cast<unsigned*>(&h); }
// (x, y) = hi + lo, each a pair of fp16 numbers: hi rounds to nearest, lo holds the next 11 bits
__device__ __forceinline__ void split2(float x, float y, unsigned& hi, unsigned& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 l = fma2(__half22float2(h), both(-1.0f), make_float2(x, y));
    hi = h2_bits(h);
    lo = h2_bits(__floats2half2_rn(l.x, l.y));
}
// Power of two that brings |x| near 2^11, and its inverse; 1 for zero, infinite and NaN rows as far as their exponents allow.
__device__ __forceinline__ void row_scale(float amax, float& up, float& down) {
    const int ex = static_cast<int>((__float_as_uint(amax) >> 23) & 255u);
    const int se = (ex == 0 || ex == 255) ? 127 : min(250, max(4, 265 - ex));
    up = __uint_as_float(static_cast<unsigned>(se) << 23);
    down = __uint_as_float(static_cast<unsigned>(254 - se) << 23);
}
// tanh to fp32 accuracy.  Below 0.55 the odd power series (coefficients B_2n 2^2n (2^2n - 1) / (2n)!, truncated after
// u^15: 2e-8 relative there); above it the library's function.  Capped scores are mostly small against their cap.
__device__ __forceinline__ float tanh_series(float u) {
    const float w = u * u;
    float r = -1.4558344e-3f;
    r = fmaf(r, w, 3.5921280e-3f);
    r = fmaf(r, w, -8.8632355e-3f);
    r = fmaf(r, w, 2.1869488e-2f);
    r = fmaf(r, w, -5.3968254e-2f);
    r = fmaf(r, w, 1.3333333e-1f);
    r = fmaf(r, w, -3.3333333e-1f);
    return fmaf(u * w, r, u);
}
__device__ __forceinline__ float tanh_acc(float u) { return fabsf(u) < 0.55f ? tanh_series(u) : tanhf(u); }
// Values that are not finite, of which a product with a zero weight would make NaN: found 16 bytes at a time, added to a row
// that sees them, and cleared from a tile.
__device__ __forceinline__ bool not_finite2(unsigned w) { return (w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u; }
__device__ __forceinline__ bool not_finite(uint4 v) { return not_finite2(v.x) || not_finite2(v.y) || not_finite2(v.z) || not_finite2(v.w); }
__device__ __forceinline__ void add_not_finite(float& a, float& b, float p, unsigned w) {
    if ((w & 0x7C00u) == 0x7C00u) a = fmaf(p, half_bits_to_float(w & 0xFFFFu), a);
    if ((w & 0x7C000000u) == 0x7C000000u) b = fmaf(p, half_bits_to_float(w >> 16), b);
}
__device__ __forceinline__ void zero_not_finite(uint8_t* chunk) {
    unsigned* w = reinterpret_cast<unsigned*>(chunk);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if ((w[i] & 0x7C00u) == 0x7C00u) w[i] &= 0xFFFF0000u;
        if ((w[i] & 0x7C000000u) == 0x7C000000u) w[i] &= 0x0000FFFFu;
    }
}
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// Slope of the distance bias of a head, times log2 e (1 times log2 e without a slope: an additive mask as it is).
__device__ __forceinline__ float bias_slope(const AttnP& P, int head) {
    if (P.bias_step == 0.0f) return kLog2e;
    const int h = P.bias_log2_heads;
    const float e = head < h ? static_cast<float>(head + 1) * P.bias_step : static_cast<float>(2 * (head - h) + 1) * (0.5f * P.bias_step);
    return exp2f(-e) * kLog2e;
}

// What a query row needs to know of itself when scores are general.
struct RowInfo {
    int pos, doc;
    bool valid;
    float slope;
    const unsigned short* mask;
};
__device__ __forceinline__ int seq_keys(const AttnP& P, int s) { return P.n_keys ? max(0, min(P.n_keys[s], P.cap)) : P.cap; }
__device__ __forceinline__ int row_pos(const AttnP& P, int s, int n, int token) {
    if (P.q_pos) return P.q_pos[static_cast<size_t>(s) * P.n_tokens + token];
    return (P.next_pos ? P.next_pos[s] : n) - P.n_tokens + token;
}
// Slots (= positions) from here on are hidden from a row by causality; `end` bounds it.
__device__ __forceinline__ int causal_limit(int pos, int prefix, int end) { return pos >= end ? end : min(end, max(prefix, pos + 1)); }
__device__ __forceinline__ RowInfo row_info(const AttnP& P, int s, int kvh, int n, int row) {
    RowInfo r;
    r.valid = row < P.rows;
    const int rr = r.valid ? row : 0, token = rr / P.group, head = kvh * P.group + rr % P.group;
    r.pos = row_pos(P, s, n, token);
    r.doc = P.q_doc ? P.q_doc[static_cast<size_t>(s) * P.n_tokens + token] : 0;
    r.slope = bias_slope(P, head);
    r.mask = P.mask ? P.mask + static_cast<size_t>(s) * P.mask_seq + static_cast<size_t>(token) * P.mask_token : nullptr;
    return r;
}
// What a key slot is to every row: its position and document.
struct KeyInfo {
    int pos, doc;
};
__device__ __forceinline__ KeyInfo key_info(const AttnP& P, int s, int kvh, int t, int n) {
    KeyInfo k;
    k.pos = t, k.doc = 0;
    if (t < n) {
        if (P.positions) k.pos = P.positions[(static_cast<size_t>(s) * P.kv_heads + kvh) * P.cap + t];
        if (P.k_doc) k.doc = P.k_doc[static_cast<size_t>(s) * P.cap + t];
    }
    return k;
}
// Base-2 score of a raw product (already times the row's power of two), or -inf where the row does not see the slot.
// GEN = false: no cap, no bias, no mask arrays, slot = position; visible is t < limit (the caller's causal bound).
__device__ __forceinline__ float general_score(const AttnP& P, float z, const RowInfo& r, const KeyInfo& key, int t, int n, int prefix) {
    float y = P.cap_out != 0.0f ? tanh_acc(z) * P.cap_out : z;
    bool see = t < n && r.valid;
    if (P.causal) see = see && (key.pos <= r.pos || key.pos < prefix);
    if (P.q_doc) see = see && key.doc == r.doc;
    if (P.mask) {
        const float add = see ? half_bits_to_float(r.mask[t]) : 0.0f;
        see = see && add != -INFINITY;  // hides whatever the product is
        y += r.slope * add;
    } else if (P.bias_step != 0.0f) {
        y -= r.slope * fabsf(static_cast<float>(r.pos - key.pos));
    }
    return see ? y : -INFINITY;
}

// Which key tiles of [begin, end) hold a document of the query tokens tok0 .. tok1: a bitmap in shared memory, a bit per 2^k tiles
// with k so large that kDocBits bits are enough.
constexpr int kDocBits = 8192;
template <int TK>
struct DocTiles {
    uint32_t* bits;
    int nt;
    __device__ __forceinline__ int shift() const { return nt <= kDocBits ? 0 : 32 - __clz((nt - 1) / kDocBits); }
    __device__ __forceinline__ void clear(int tid, int threads) const {
        for (int i = tid; i < kDocBits / 32; i += threads) bits[i] = 0u;
    }
    __device__ __forceinline__ void find(const AttnP& P, int s, int tok0, int tok1, int begin, int end, int warp, int warps, int lane) const {
        int lo = INT32_MAX, hi = INT32_MIN;
        for (int t = tok0 + lane; t <= tok1; t += 32) {
            const int d = P.q_doc[static_cast<size_t>(s) * P.n_tokens + t];
            lo = min(lo, d), hi = max(hi, d);
        }
        lo = __reduce_min_sync(0xffffffffu, lo), hi = __reduce_max_sync(0xffffffffu, hi);
        const int* kd = P.k_doc + static_cast<size_t>(s) * P.cap;
        const int sh = shift();
        constexpr int kAhead = 8, kPer = TK / 32;  // tiles whose documents are requested at once
        for (int i0 = warp; i0 < nt; i0 += warps * kAhead) {
            int d[kAhead][kPer];
#pragma unroll
            for (int a = 0; a < kAhead; ++a)
#pragma unroll
                for (int k = 0; k < kPer; ++k) {
                    const int t = begin + (i0 + a * warps) * TK + k * 32 + lane;
                    d[a][k] = i0 + a * warps < nt && t < end ? kd[t] : (lo > INT32_MIN ? lo - 1 : hi + 1);
                }
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                bool any = false;
#pragma unroll
                for (int k = 0; k < kPer; ++k) any = any || (d[a][k] >= lo && d[a][k] <= hi);
                const int i = (i0 + a * warps) >> sh;
                if (__any_sync(0xffffffffu, any) && lane == 0) atomicOr(&bits[i / 32], 1u << (i % 32));
            }
        }
    }
    __device__ __forceinline__ int next(int i) const {  // the wanted tile behind tile i, nt if there is none
        const int sh = shift();
        ++i;
        while (i < nt) {
            const int b = i >> sh;
            const uint32_t w = bits[b / 32] >> (b % 32);
            if (w & 1u) break;
            i = (b + (w ? __ffs(w) - 1 : 32 - b % 32)) << sh;
        }
        return min(i, nt);
    }
};

// ---- cache tiles in shared memory -----------------------------------------------------------------------------------
// fp16: rows of D halves, padded by 16 bytes so that the eight rows of an ldmatrix fall into different banks.
// 4 bits: [rows][D / 2] nibbles, then [rows][D / 32] {d, m}: the cache's own order, read without conflicts as it is.
template <int D, int FMT>
struct Tile {
    static constexpr int NB = D / 32;
    static constexpr int kRow = FMT == 16 ? 2 * D + 16 : D / 2;
    static constexpr int kPar = FMT == 16 ? 0 : 4 * NB;
    __host__ __device__ static constexpr int bytes(int rows) { return (rows * (kRow + kPar) + 15) / 16 * 16; }
};
// Copies rows [t0, t0 + ROWS) of one plane (keys or values) of (sequence, head) into a tile; rows at or past `end` become zeros.
// `tid` of `nt` threads share the work; ROWS and the thread count make every loop bound a constant.
template <int D, int FMT, int ROWS, int NT>
__device__ __forceinline__ void load_tile(const AttnP& P, const uint8_t* base, long long row, long long head, long long seq, int s, int kvh, int t0, int end,
                                          uint32_t dst, int tid) {
    using T = Tile<D, FMT>;
    if constexpr (FMT == 16) {
        const __half* src = reinterpret_cast<const __half*>(base) + static_cast<size_t>(s) * seq + static_cast<size_t>(kvh) * head;
        constexpr int kChunks = D / 8;
#pragma unroll
        for (int i = 0; i < (ROWS * kChunks + NT - 1) / NT; ++i) {
            const int x = i * NT + tid;
            if ((ROWS * kChunks) % NT && x >= ROWS * kChunks) break;
            const int r = x / kChunks, ch = x % kChunks;
            const bool ok = t0 + r < end;
            cp16(dst + r * T::kRow + ch * 16, src + static_cast<size_t>(ok ? t0 + r : 0) * row + ch * 8, ok);
        }
    } else {
        const uint8_t* b = base + static_cast<size_t>(s) * P.seq_bytes;
        const uint8_t* rows = b + static_cast<size_t>(kvh) * P.cap * (D / 2);
        constexpr int kChunks = D / 32;  // 16 bytes each
#pragma unroll
        for (int i = 0; i < (ROWS * kChunks + NT - 1) / NT; ++i) {
            const int x = i * NT + tid;
            if ((ROWS * kChunks) % NT && x >= ROWS * kChunks) break;
            const bool ok = t0 + x / kChunks < end;
            cp16(dst + x * 16, rows + (ok ? static_cast<size_t>(t0) * (D / 2) + x * 16 : 0), ok);
        }
        // parameters: 4 NB bytes a row, whose alignment is that of the row
        constexpr int kSz = T::NB % 4 == 0 ? 16 : T::NB % 2 == 0 ? 8 : 4, kPer = T::kPar / kSz;
        const uint8_t* par = b + P.par_off + static_cast<size_t>(kvh) * P.cap * T::kPar;
        const uint32_t pd = dst + ROWS * T::kRow;
#pragma unroll
        for (int i = 0; i < (ROWS * kPer + NT - 1) / NT; ++i) {
            const int x = i * NT + tid;
            if ((ROWS * kPer) % NT && x >= ROWS * kPer) break;
            const bool ok = t0 + x / kPer < end;
            const uint8_t* src = par + (ok ? static_cast<size_t>(t0) * T::kPar + x * kSz : 0);
            if constexpr (kSz == 16) cp16(pd + x * 16, src, ok);
            else cp_small<kSz>(pd + x * kSz, src, ok);
        }
    }
}

// The same for a tile of ROWS slots that are all in use, by one warp: no predicates, and where an address moves on by constants only
// the copies.  (4-bit parameters of narrow heads are not aligned to 16 bytes: those take the form above.)
__device__ __forceinline__ void cp16_all(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
template <int D, int FMT, int ROWS>
__device__ __forceinline__ void load_tile_full(const uint8_t* codes_or_rows, const uint8_t* params, long long row, int t0, uint32_t dst, int lane) {
    using T = Tile<D, FMT>;
    if constexpr (FMT == 16) {
        const __half* src = reinterpret_cast<const __half*>(codes_or_rows);
        constexpr int kChunks = D / 8;
#pragma unroll
        for (int i = 0; i < ROWS * kChunks / 32; ++i) {
            const int x = i * 32 + lane, r = x / kChunks, ch = x % kChunks;
            cp16_all(dst + r * T::kRow + ch * 16, src + static_cast<long long>(t0 + r) * row + ch * 8);
        }
    } else {
        const uint8_t* src = codes_or_rows + static_cast<size_t>(t0) * (D / 2) + lane * 16;
#pragma unroll
        for (int i = 0; i < ROWS * (D / 32) / 32; ++i) cp16_all(dst + (i * 32 + lane) * 16, src + i * 512);
        if constexpr (T::NB % 4 == 0) {
            const uint8_t* par = params + static_cast<size_t>(t0) * T::kPar + lane * 16;
#pragma unroll
            for (int i = 0; i < ROWS * T::kPar / 512; ++i) cp16_all(dst + ROWS * T::kRow + (i * 32 + lane) * 16, par + i * 512);
        }
    }
}

// NW 32-bit words at a 4-byte (or wider, as NW allows) aligned shared address
template <int NW>
__device__ __forceinline__ void lds_words(unsigned (&w)[NW], const uint8_t* p) {
    if (NW % 4 == 0) {
#pragma unroll
        for (int i = 0; i < NW / 4; ++i) {
            const uint4 v = reinterpret_cast<const uint4*>(p)[i];
            w[4 * i] = v.x, w[(4 * i + 1) % NW] = v.y, w[(4 * i + 2) % NW] = v.z, w[(4 * i + 3) % NW] = v.w;
        }
    } else if (NW % 2 == 0) {
#pragma unroll
        for (int i = 0; i < NW / 2; ++i) {
            const uint2 v = reinterpret_cast<const uint2*>(p)[i];
            w[2 * i] = v.x, w[(2 * i + 1) % NW] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < NW; ++i) w[i] = reinterpret_cast<const unsigned*>(p)[i];
    }
}
// A row group's 16-bit pieces, one per block: two blocks to a word (the last word of an odd count half used)
template <int NB>
__device__ __forceinline__ void lds_value_words(unsigned (&w)[(NB + 1) / 2], const uint8_t* p) {
    if (NB % 2 == 0) {
        unsigned t[NB % 2 == 0 ? NB / 2 : 1];
        lds_words(t, p);
#pragma unroll
        for (int i = 0; i < NB / 2; ++i) w[i] = t[i];
    } else {
        const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
        for (int i = 0; i < (NB + 1) / 2; ++i) w[i] = h[2 * i] | (2 * i + 1 < NB ? static_cast<unsigned>(h[2 * i + 1]) << 16 : 0u);
    }
}
// Slot inside a 16-slot block of value j (0..3) of quad lane c: for fp16 the fragment's own order, for 4 bits an order in
// which the four quad lanes read four neighbouring rows at once.
template <int FMT>
__device__ __forceinline__ int slot_of(int c, int j) {
    return FMT == 16 ? (j >> 1) * 8 + 2 * c + (j & 1) : c + 4 * j;
}
// Row of the 16-slot block that column g of n-tile t (0, 1) is, in the same order.
template <int FMT>
__device__ __forceinline__ int row_of_column(int t, int g) {
    return FMT == 16 ? t * 8 + g : t * 8 + (g >> 1) + 4 * (g & 1);
}
// Channels of the pair (first, second) that lane c holds of k-step ks of a query row, one register at a time (reg 0: k = 2c,
// 2c + 1; reg 1: k = 2c + 8, 2c + 9).
template <int FMT>
__device__ __forceinline__ void q_channels(int ks, int reg, int c, int& first, int& second) {
    if (FMT == 16) {
        first = 16 * ks + 8 * reg + 2 * c, second = first + 1;
    } else {  // nibbles (i, i + 4) of word c of block ks / 2, i = 2 (ks % 2) + reg
        first = 32 * (ks >> 1) + 8 * c + 2 * (ks & 1) + reg, second = first + 4;
    }
}
// The factor that 4-bit codes are scaled down by in the products.
template <int FMT>
constexpr float kCodeUp = FMT == 16 ? 1.0f : 1024.0f;

// ---- rows kernel: up to eight rows per CTA, many keys ---------------------------------------------------------------------
// For single tokens.  What bounds it is reading the cache once.  Each of the CTA's four warps works alone on blocks of slots (its own
// copies in flight, its own running maximum), so nothing waits for a neighbour; the eight rows' hi and lo halves are stacked
// into one 16-row fragment, which makes the second half of the precision free of extra products.  16 slots a block for fp16 (whose
// ring then fills the shared memory with eight warps), 32 for 4 bits.
// Measured: 32 sequences of 4096 slots, 32 heads over 8, D = 128: fp16 110 us back to back = 4.9 TB/s (0.31 instructions issued per
// cycle and scheduler: the latency of the ring), 4 bits 67 us = 2.5 TB/s (0.55 on 131072 slots: unpacking).
// MODE 0: scores as they are; 1: with a cap or a distance bias, slot = position; 2: positions, documents or an additive mask too.
// In the first two a row sees the slots below a limit.
constexpr int kRowsWarps = 4;
template <int D, int FMT>
struct RowsCfg {
    static constexpr int kSlots = FMT == 16 ? 16 : 32;
    static constexpr int kBlock = 2 * Tile<D, FMT>::bytes(kSlots);
    static constexpr int kStages = FMT == 16 && D < 128 ? 4 : 3;
    static constexpr int kMerge = kRowsWarps * 8 * (D + 4) * 4;
    static constexpr int kRing = kRowsWarps * kStages * kBlock;
    static constexpr int kSmem = kRing > kMerge ? kRing : kMerge;
};

template <int D, int FMT, int MODE>
__global__ void __launch_bounds__(32 * kRowsWarps, FMT == 16 && D == 128 ? 2 : 1) attn_rows_kernel(const __grid_constant__ AttnP P) {
    using C = RowsCfg<D, FMT>;
    using T = Tile<D, FMT>;
    constexpr int NB = D / 32, KS = D / 16, NT = D / 8, SL = C::kSlots, U = SL / 16;
    extern __shared__ __align__(16) uint8_t sm[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    const int split = blockIdx.x, kvh = blockIdx.y / P.row_tiles, row0 = (blockIdx.y % P.row_tiles) * 8, s = blockIdx.z;
    const int n = seq_keys(P, s);
    grid_dependents_may_launch();
    const int row = row0 + g;
    const bool valid = row < P.rows;
    const int token = (valid ? row : 0) / P.group, head = kvh * P.group + (valid ? row : 0) % P.group;
    const int chunk = (n + P.nsplit * 64 - 1) / (P.nsplit * 64) * 64;
    const int begin = min(n, split * chunk), end = min(n, begin + chunk);

    uint8_t* ring = sm + warp * C::kStages * C::kBlock;
    const uint32_t ring_a = smem_u32(ring);
    const int nblk = (end - begin + SL - 1) / SL, mine = nblk > warp ? (nblk - warp + kRowsWarps - 1) / kRowsWarps : 0;
    const uint8_t *kb, *vb, *kpar = nullptr, *vpar = nullptr;  // this sequence's and head's rows
    if (FMT == 16) {
        kb = P.k + 2 * (static_cast<size_t>(s) * P.k_seq + static_cast<size_t>(kvh) * P.k_head);
        vb = P.v + 2 * (static_cast<size_t>(s) * P.v_seq + static_cast<size_t>(kvh) * P.v_head);
    } else {
        const size_t seq = static_cast<size_t>(s) * P.seq_bytes, at = static_cast<size_t>(kvh) * P.cap;
        kb = P.k + seq + at * (D / 2), vb = P.v + seq + at * (D / 2);
        kpar = P.k + seq + P.par_off + at * T::kPar, vpar = P.v + seq + P.par_off + at * T::kPar;
    }
    constexpr bool kWhole = FMT == 16 ? (SL * D / 8) % 32 == 0 : NB % 4 == 0;
    auto fetch = [&](int i, int stage) {
        if (i < mine) {
            const int t0 = begin + (warp + i * kRowsWarps) * SL;
            const uint32_t dst = ring_a + stage * C::kBlock;
            if (kWhole && t0 + SL <= end) {
                load_tile_full<D, FMT, SL>(kb, kpar, P.k_row, t0, dst, lane);
                load_tile_full<D, FMT, SL>(vb, vpar, P.v_row, t0, dst + T::bytes(SL), lane);
            } else {
                load_tile<D, FMT, SL, 32>(P, P.k, P.k_row, P.k_head, P.k_seq, s, kvh, t0, end, dst, lane);
                load_tile<D, FMT, SL, 32>(P, P.v, P.v_row, P.v_head, P.v_seq, s, kvh, t0, end, dst + T::bytes(SL), lane);
            }
        }
        cp_commit();
    };
#pragma unroll
    for (int i = 0; i < C::kStages - 1; ++i) fetch(i, i);

    // the row's query as hi (registers 0, 2) and lo (1, 3) fragments, scaled; block sums for the minima
    unsigned qf[KS][4];
    float qs[FMT == 16 ? 1 : NB];
    float up, down;
    {
        const float* qp = P.q + static_cast<size_t>(s) * P.q_seq + static_cast<size_t>(token) * P.q_token + static_cast<size_t>(head) * P.q_head;
        float x[KS][4], amax = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                int a, b;
                q_channels<FMT>(ks, r, c, a, b);
                x[ks][2 * r] = valid ? qp[a] : 0.0f, x[ks][2 * r + 1] = valid ? qp[b] : 0.0f;
                amax = fmaxf(amax, fmaxf(fabsf(x[ks][2 * r]), fabsf(x[ks][2 * r + 1])));
            }
        row_scale(quad_max(amax), up, down);
        if (FMT != 16) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float t = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) t += x[2 * b][i] + x[2 * b + 1][i];
                qs[b] = quad_sum(t) * up * (1.0f / kCodeUp<FMT>);
            }
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            split2(x[ks][0] * up, x[ks][1] * up, qf[ks][0], qf[ks][1]);
            split2(x[ks][2] * up, x[ks][3] * up, qf[ks][2], qf[ks][3]);
        }
    }
    const float ysc = P.sc * down * kCodeUp<FMT>;
    RowInfo ri{};
    int limit = valid ? end : 0;
    const int prefix = P.prefix ? P.prefix[s] : 0;
    if (MODE) ri = row_info(P, s, kvh, n, row);
    if (MODE < 2 && P.causal && valid) limit = causal_limit(row_pos(P, s, n, token), prefix, end);
    const bool hides = MODE == 2 || (P.causal && (P.n_tokens > 1 || P.next_pos || P.q_pos));  // slots in use may be hidden from a row

    float o[NT][4], m = -INFINITY, l = 0.0f;
    float2 om[FMT == 16 ? 1 : NB];
#pragma unroll
    for (int j = 0; j < NT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
#pragma unroll
    for (int b = 0; b < (FMT == 16 ? 1 : NB); ++b) om[b] = make_float2(0.0f, 0.0f);

    int stage = 0;
    for (int i = 0; i < mine; ++i) {
        cp_wait<C::kStages - 2>();
        __syncwarp();
        fetch(i + C::kStages - 1, stage == 0 ? C::kStages - 1 : stage - 1);  // into the stage that was read in the last round
        const uint8_t* kt = ring + stage * C::kBlock;
        const uint8_t* vt = kt + T::bytes(SL);
        if (++stage == C::kStages) stage = 0;
        const int t0 = begin + (warp + i * kRowsWarps) * SL;
        float y[U][4];
        if (FMT == 16) {
            float sc[2][4] = {};
#pragma unroll
            for (int k2 = 0; k2 < KS / 2; ++k2)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    unsigned b[4];
                    ldsm4(b, smem_u32(kt) + (t * 8 + (lane & 7)) * T::kRow + k2 * 64 + (lane >> 3) * 16);
                    mma16816(sc[t], qf[2 * k2], b[0], b[1]);
                    mma16816(sc[t], qf[2 * k2 + 1], b[2], b[3]);
                }
#pragma unroll
            for (int j = 0; j < 4; ++j) y[0][j] = sc[j >> 1][j & 1] + sc[j >> 1][2 + (j & 1)];
        } else {
            const uint8_t* kp = kt + SL * T::kRow;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    unsigned w[NB], p0[NB], p1[NB];
                    lds_words(w, kt + (u * 16 + row_of_column<FMT>(t, g)) * T::kRow + c * 4 * NB);
                    lds_words(p0, kp + (u * 16 + t * 8 + c) * T::kPar);
                    lds_words(p1, kp + (u * 16 + t * 8 + c + 4) * T::kPar);
                    float2 acc = make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        const unsigned hi = w[b] >> 8;
                        mma16816(a, qf[2 * b], code_pair<false, false>(w[b]), code_pair<true, false>(w[b]));
                        mma16816(a, qf[2 * b + 1], code_pair<false, false>(hi), code_pair<true, false>(hi));
                        const float2 d0 = __half22float2(*reinterpret_cast<__half2*>(&p0[b])), d1 = __half22float2(*reinterpret_cast<__half2*>(&p1[b]));
                        acc = fma2(make_float2(d0.x, d1.x), add2(make_float2(a[0], a[1]), make_float2(a[2], a[3])), fma2(make_float2(d0.y, d1.y), both(qs[b]), acc));
                    }
                    y[u][2 * t] = acc.x, y[u][2 * t + 1] = acc.y;
                }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int t = t0 + u * 16 + slot_of<FMT>(c, j);
                float& v = y[u][j];
                v *= ysc;
                if (MODE == 2) {
                    v = general_score(P, v, ri, key_info(P, s, kvh, t, end), t, end, prefix);
                } else {
                    if (MODE == 1) {
                        if (P.cap_out != 0.0f) v = tanh_acc(v) * P.cap_out;
                        if (P.bias_step != 0.0f) v -= ri.slope * fabsf(static_cast<float>(ri.pos - t));
                    }
                    if (t >= limit) v = -INFINITY;
                }
                mx = fmaxf(mx, v);
            }
        if (P.scores && valid) {
            float* sp = P.scores + ((static_cast<size_t>(s) * P.kv_heads + kvh) * P.rows + row) * P.cap + t0;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (t0 + u * 16 + slot_of<FMT>(c, j) < end) sp[u * 16 + slot_of<FMT>(c, j)] = y[u][j];
        }
        if (FMT != 16) {
            // p d must stay below fp16's largest number.  With every d below 16 it does; larger scales raise the reference.
            // (The OR is at least the largest d; scales of 2 and more may come here without need, and lose nothing.)
            const uint8_t* pp = vt + SL * T::kRow;
            unsigned big = 0;
#pragma unroll
            for (int x = 0; x < SL * NB / 32; ++x) big |= *reinterpret_cast<const unsigned*>(pp + 4 * (x * 32 + lane));
            if (__any_sync(0xffffffffu, (big & 0x7FFFu) >= 0x4C00u)) {
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        unsigned dm = 0;
#pragma unroll
                        for (int b = 0; b < NB; ++b) dm = max(dm, *reinterpret_cast<const unsigned*>(pp + (u * 16 + slot_of<FMT>(c, j)) * T::kPar + 4 * b) & 0x7FFFu);
                        if (y[u][j] != -INFINITY) mx = fmaxf(mx, y[u][j] + static_cast<float>(max(0, static_cast<int>(dm >> 10) - 18)));
                    }
            }
        }
        mx = quad_max(mx);
        const float mn = fmaxf(m, mx);
        if (__any_sync(0xffffffffu, mn > m)) {
            const float al = mn > m ? ex2(m - mn) : 1.0f;
#pragma unroll
            for (int j = 0; j < NT; ++j) o[j][0] *= al, o[j][1] *= al, o[j][2] *= al, o[j][3] *= al;
            l *= al;
            if (FMT != 16)
#pragma unroll
                for (int b = 0; b < NB; ++b) om[b].x *= al, om[b].y *= al;
            m = mn;
        }
        const float ref = m == -INFINITY ? 0.0f : m - kPShift;
        float p[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                p[u][j] = ex2(y[u][j] - ref);
                l += p[u][j];
            }
        if (FMT == 16) {
            if (hides) {  // an infinity or NaN in a hidden slot must not reach the row as 0 * inf
                bool odd = false;
#pragma unroll
                for (int x = 0; x < (16 * D / 8) / 32; ++x) {
                    const int ch = x * 32 + lane;
                    odd = odd || not_finite(*reinterpret_cast<const uint4*>(vt + ch / (D / 8) * T::kRow + ch % (D / 8) * 16));
                }
                if (__any_sync(0xffffffffu, odd)) {  // rare: such values go to the rows that see them one by one, and become zeros
#pragma unroll 1
                    for (int t = 0; t < 16; ++t) {
                        const float pv = (t & 8) ? ((t & 1) ? p[0][3] : p[0][2]) : ((t & 1) ? p[0][1] : p[0][0]);
                        const float pt = __shfl_sync(0xffffffffu, pv, (lane & 28) + ((t & 7) >> 1));
                        if (pt != 0.0f)
#pragma unroll
                            for (int j = 0; j < NT; ++j) add_not_finite(o[j][0], o[j][1], pt, *reinterpret_cast<const unsigned*>(vt + t * T::kRow + j * 16 + c * 4));
                    }
                    __syncwarp();
#pragma unroll 1
                    for (int x = lane; x < 16 * D / 8; x += 32) zero_not_finite(ring + (vt - ring) + x / (D / 8) * T::kRow + x % (D / 8) * 16);
                    __syncwarp();
                }
            }
            unsigned a[4];
            split2(p[0][0], p[0][1], a[0], a[1]);
            split2(p[0][2], p[0][3], a[2], a[3]);
#pragma unroll
            for (int j = 0; j < NT / 2; ++j) {
                unsigned b[4];
                ldsm4t(b, smem_u32(vt) + ((lane & 7) + ((lane >> 3) & 1) * 8) * T::kRow + j * 32 + (lane >> 4) * 16);
                mma16816(o[2 * j], a, b[0], b[1]);
                mma16816(o[2 * j + 1], a, b[2], b[3]);
            }
        } else {
            const uint8_t* pp = vt + SL * T::kRow;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                unsigned vp[4][NB], w[4][(NB + 1) / 2];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    lds_words(vp[j], pp + (u * 16 + slot_of<FMT>(c, j)) * T::kPar);
                    lds_value_words<NB>(w[j], vt + (u * 16 + c + 4 * j) * T::kRow + g * 2 * NB);
                }
                if (hides) {  // a hidden slot's scales may be anything (slots behind the last are zeros)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int b = 0; b < NB; ++b)
                            if (p[u][j] == 0.0f) vp[j][b] = 0u;
                }
                const float2 p01 = make_float2(p[u][0], p[u][1]), p23 = make_float2(p[u][2], p[u][3]);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    float2 dm[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) dm[j] = __half22float2(*reinterpret_cast<__half2*>(&vp[j][b]));
                    const float2 d01 = make_float2(dm[0].x, dm[1].x), d23 = make_float2(dm[2].x, dm[3].x);
                    om[b] = fma2(p01, fma2(both(8.0f), d01, make_float2(dm[0].y, dm[1].y)), om[b]);
                    om[b] = fma2(p23, fma2(both(8.0f), d23, make_float2(dm[2].y, dm[3].y)), om[b]);
                    const float2 e01 = mul2(p01, d01), e23 = mul2(p23, d23);
                    unsigned a[4];
                    split2(e01.x, e01.y, a[0], a[1]);
                    split2(e23.x, e23.y, a[2], a[3]);
                    const unsigned sel = b & 1 ? 0x7632u : 0x5410u;
                    const unsigned x0 = __byte_perm(w[0][b / 2], w[1][b / 2], sel), x1 = __byte_perm(w[2][b / 2], w[3][b / 2], sel);
                    const unsigned h0 = x0 >> 8, h1 = x1 >> 8;
                    mma16816(o[4 * b], a, code_pair<false, true>(x0), code_pair<false, true>(x1));
                    mma16816(o[4 * b + 1], a, code_pair<true, true>(x0), code_pair<true, true>(x1));
                    mma16816(o[4 * b + 2], a, code_pair<false, true>(h0), code_pair<false, true>(h1));
                    mma16816(o[4 * b + 3], a, code_pair<true, true>(h0), code_pair<true, true>(h1));
                }
            }
        }
    }
    cp_wait<0>();
    l = quad_sum(l);
    __syncthreads();

    // the warps' partial rows through shared memory: [warp][row][D + 4], {m, l} behind the row
    float* buf = reinterpret_cast<float*>(sm);
    float* my = buf + (warp * 8 + g) * (D + 4);
    if (FMT == 16) {
#pragma unroll
        for (int j = 0; j < NT; ++j) *reinterpret_cast<float2*>(my + 8 * j + 2 * c) = make_float2(o[j][0] + o[j][2], o[j][1] + o[j][3]);
    } else {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float mm = quad_sum(om[b].x + om[b].y);
            float r[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                r[i] = fmaf(o[4 * b + i][0] + o[4 * b + i][2], kCodeUp<FMT>, mm);
                r[4 + i] = fmaf(o[4 * b + i][1] + o[4 * b + i][3], kCodeUp<FMT>, mm);
            }
            float4* dst = reinterpret_cast<float4*>(my + 32 * b + 8 * c);
            dst[0] = make_float4(r[0], r[1], r[2], r[3]);
            dst[1] = make_float4(r[4], r[5], r[6], r[7]);
        }
    }
    if (c == 0) my[D] = m, my[D + 1] = l;
    __syncthreads();
    const size_t part = ((static_cast<size_t>(s) * P.kv_heads + kvh) * P.nsplit + split) * P.rows + row0;
    for (int x = tid; x < 8 * (D / 4); x += 32 * kRowsWarps) {
        const int r = x / (D / 4), ch = x % (D / 4) * 4;
        if (row0 + r >= P.rows) continue;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kRowsWarps; ++w) M = fmaxf(M, buf[(w * 8 + r) * (D + 4) + D]);
        float L = 0.0f;
        float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kRowsWarps; ++w) {
            const float* p = buf + (w * 8 + r) * (D + 4);
            if (p[D + 1] == 0.0f) continue;  // saw nothing (a NaN sum goes on)
            const float f = ex2(p[D] - M);
            const float4 v = *reinterpret_cast<const float4*>(p + ch);
            a.x = fmaf(f, v.x, a.x), a.y = fmaf(f, v.y, a.y), a.z = fmaf(f, v.z, a.z), a.w = fmaf(f, v.w, a.w);
            L = fmaf(f, p[D + 1], L);
        }
        if (P.nsplit > 1) {
            *reinterpret_cast<float4*>(P.part_o + (part + r) * D + ch) = a;
        } else {
            const float inv = L > 0.0f || L != L ? 1.0f / L : 0.0f;
            const int tok = (row0 + r) / P.group, hd = kvh * P.group + (row0 + r) % P.group;
            *reinterpret_cast<float4*>(P.out + static_cast<size_t>(s) * P.o_seq + static_cast<size_t>(tok) * P.o_token + static_cast<size_t>(hd) * P.o_head + ch) =
                make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
        }
        if (ch == 0 && (P.nsplit > 1 || P.scores)) P.part_ml[part + r] = make_float2(M, L);
    }
}

// ---- joining the splits of a row -------------------------------------------------------------------------------------------
// By warps (at most 32 splits): one warp per row, eight splits of it in flight.  Else one CTA per row, whose warps take the splits in
// turn and join their sums through shared memory.  Warps where there are at most as many splits as a CTA has warps (8192 rows in two
// splits 3 us, by CTAs 20), or more rows than the GPU holds CTAs of (2048 rows in 9 or 18 splits: the call 26.7 and 28.7 us, by CTAs 30.8
// and 32.8); else CTAs (384 rows in 18 splits: 22.5, by warps 24.6).
constexpr int kMergeWarps = 8;
__device__ __forceinline__ float4* merged_row(const AttnP& P, int s, int kvh, int r) {
    return reinterpret_cast<float4*>(P.out + static_cast<size_t>(s) * P.o_seq + static_cast<size_t>(r / P.group) * P.o_token + static_cast<size_t>(kvh * P.group + r % P.group) * P.o_head);
}
template <int D>
__global__ void __launch_bounds__(32 * kMergeWarps) attn_merge_warps_kernel(const __grid_constant__ AttnP P) {
    constexpr int W = kMergeWarps, Q = (D / 4 + 31) / 32;
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, kvh = blockIdx.y, s = blockIdx.z;
    const int r = blockIdx.x * W + (threadIdx.x >> 5);
    if (r >= P.rows) return;
    const size_t base = (static_cast<size_t>(s) * P.kv_heads + kvh) * P.nsplit;
    const float2 t = lane < P.nsplit ? P.part_ml[(base + lane) * P.rows + r] : make_float2(0.0f, 0.0f);
    const float M = warp_max(t.y != 0.0f ? t.x : -INFINITY), f = t.y != 0.0f ? ex2(t.x - M) : 0.0f, L = warp_sum(t.y != 0.0f ? f * t.y : 0.0f);
    const float inv = L > 0.0f || L != L ? 1.0f / L : 0.0f;
    float4* out = merged_row(P, s, kvh, r);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int x = q * 32 + lane;
        float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
        for (int i0 = 0; i0 < P.nsplit; i0 += W) {
            float4 v[W];
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (i0 + i < P.nsplit && x < D / 4) v[i] = reinterpret_cast<const float4*>(P.part_o + ((base + i0 + i) * P.rows + r) * D)[x];
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const float fi = __shfl_sync(0xffffffffu, f, i0 + i), ly = __shfl_sync(0xffffffffu, t.y, i0 + i);
                if (ly != 0.0f && x < D / 4)  // a split in which the row saw nothing has no sums
                    a.x = fmaf(fi, v[i].x, a.x), a.y = fmaf(fi, v[i].y, a.y), a.z = fmaf(fi, v[i].z, a.z), a.w = fmaf(fi, v[i].w, a.w);
            }
        }
        if (x < D / 4) out[x] = make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
    }
    if (P.final_ml && lane == 0) P.final_ml[(static_cast<size_t>(s) * P.kv_heads + kvh) * P.rows + r] = make_float2(M, L);
}

// After a rows launch that also wants weights, further CTAs (blockIdx.x from `joins` on) turn 2048 slots' scores into weights each:
// weights[t] += sum over the rows of 2^(score - M) / L, the rows in order, no atomics.
constexpr int kWeightSlots = 2048;
template <int D>
__global__ void __launch_bounds__(32 * kMergeWarps) attn_merge_kernel(const __grid_constant__ AttnP P, int joins) {
    constexpr int W = kMergeWarps, Q = (D / 4 + 31) / 32;
    __shared__ float4 acc[W][D / 4];
    __shared__ float2 ml[kRowsMax];
    static_assert(W <= kRowsMax);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = blockIdx.x, kvh = blockIdx.y, s = blockIdx.z;
    grid_dependency_wait();
    if (row >= joins) {
        const int n = seq_keys(P, s), t0 = (row - joins) * kWeightSlots;
        if (t0 >= n) return;
        const size_t sh = static_cast<size_t>(s) * P.kv_heads + kvh;
        for (int r = warp; r < P.rows; r += W) {
            float M = -INFINITY, L = 0.0f;
            for (int i = lane; i < P.nsplit; i += 32) {
                const float2 t = P.part_ml[(sh * P.nsplit + i) * P.rows + r];
                if (t.y == 0.0f) continue;
                const float m = fmaxf(M, t.x);
                L = L * ex2(M - m) + t.y * ex2(t.x - m), M = m;
            }
            const float m = warp_max(M);
            L = warp_sum(M == -INFINITY ? L : L * ex2(M - m));
            if (lane == 0) ml[r] = make_float2(m - kPShift, L != 0.0f ? 1.0f / L : 0.0f);
        }
        __syncthreads();
        float* w = P.weights + sh * P.cap;
        const float* sc = P.scores + sh * P.rows * P.cap;
        constexpr int kPer = kWeightSlots / (32 * W);  // slots per thread, all of a row's scores requested at once
        float sum[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) sum[i] = 0.0f;
        for (int r = 0; r < P.rows; ++r) {
            float y[kPer];
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int t = t0 + i * (32 * W) + threadIdx.x;
                y[i] = t < n ? sc[static_cast<size_t>(r) * P.cap + t] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (y[i] != -INFINITY) sum[i] = fmaf(ex2(y[i] - ml[r].x), ml[r].y, sum[i]);
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int t = t0 + i * (32 * W) + threadIdx.x;
            if (t < n) w[t] += sum[i];
        }
        return;
    }
    const size_t base = (static_cast<size_t>(s) * P.kv_heads + kvh) * P.nsplit;
    float M = -INFINITY;
    for (int i = threadIdx.x & 31; i < P.nsplit; i += 32) {
        const float2 t = P.part_ml[(base + i) * P.rows + row];
        if (t.y != 0.0f) M = fmaxf(M, t.x);
    }
    M = warp_max(M);
    float4 a[Q];
    float L = 0.0f;
#pragma unroll
    for (int q = 0; q < Q; ++q) a[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int i = warp; i < P.nsplit; i += W) {
        const size_t p = (base + i) * P.rows + row;
        const float2 t = P.part_ml[p];
        const float f = t.y != 0.0f ? ex2(t.x - M) : 0.0f;
        L = t.y != 0.0f ? fmaf(f, t.y, L) : L;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            if (q * 32 + lane < D / 4 && t.y != 0.0f) {
                const float4 v = reinterpret_cast<const float4*>(P.part_o + p * D)[q * 32 + lane];
                a[q].x = fmaf(f, v.x, a[q].x), a[q].y = fmaf(f, v.y, a[q].y), a[q].z = fmaf(f, v.z, a[q].z), a[q].w = fmaf(f, v.w, a[q].w);
            }
        }
    }
#pragma unroll
    for (int q = 0; q < Q; ++q)
        if (q * 32 + lane < D / 4) acc[warp][q * 32 + lane] = a[q];
    if (lane == 0) ml[warp] = make_float2(M, L);
    __syncthreads();
    L = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) L += ml[w].y;
    const float inv = L > 0.0f || L != L ? 1.0f / L : 0.0f;
    float4* out = merged_row(P, s, kvh, row);
    for (int x = threadIdx.x; x < D / 4; x += 32 * W) {
        float4 r = acc[0][x];
#pragma unroll
        for (int w = 1; w < W; ++w) {
            const float4 v = acc[w][x];
            r.x += v.x, r.y += v.y, r.z += v.z, r.w += v.w;
        }
        out[x] = make_float4(r.x * inv, r.y * inv, r.z * inv, r.w * inv);
    }
    if (P.final_ml && threadIdx.x == 0) P.final_ml[(static_cast<size_t>(s) * P.kv_heads + kvh) * P.rows + row] = make_float2(M, L);
}

// ---- 16-row fragments: queries in shared memory, scores of a key tile -------------------------------------------------------
// Sixty-four query rows as hi and lo halves in the order of the products' k (for 4 bits the order of the nibbles), each row
// scaled by its power of two; per row the factor that turns a product into a base-2 score and, for 4 bits, the block sums.
template <int D>
struct QTile {
    static constexpr int kRows = 64;
    static constexpr int kRow = 2 * D + 16;
    static constexpr int kLo = kRows * kRow;
    static constexpr int kYsc = 2 * kRows * kRow;
    static constexpr int kSums = kYsc + kRows * 4;                       // [row][NB + 1]: one word more than blocks against bank conflicts
    static constexpr int kBytes = (kSums + kRows * (D / 32 + 1) * 4 + 15) / 16 * 16;
};
// One row by eight lanes: piece i * 8 + l8 of 8 channels into x[i], then scaled and split into the tile.
template <int D>
struct QPieces {
    static constexpr int kCh = D / 8, kPer = (kCh + 7) / 8;
    float x[kPer][8];
};
template <int D>
__device__ __forceinline__ void fetch_q_row(const AttnP& P, int s, int kvh, int row, int l8, QPieces<D>& q) {
    constexpr int kCh = QPieces<D>::kCh;
    const bool ok = row < P.rows;
    const int token = (ok ? row : 0) / P.group, head = kvh * P.group + (ok ? row : 0) % P.group;
    const float* qp = P.q + static_cast<size_t>(s) * P.q_seq + static_cast<size_t>(token) * P.q_token + static_cast<size_t>(head) * P.q_head;
#pragma unroll
    for (int i = 0; i < QPieces<D>::kPer; ++i) {
        const int ch = i * 8 + l8;
        float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f), b = a;
        if (ok && ch < kCh) a = reinterpret_cast<const float4*>(qp)[2 * ch], b = reinterpret_cast<const float4*>(qp)[2 * ch + 1];
        q.x[i][0] = a.x, q.x[i][1] = a.y, q.x[i][2] = a.z, q.x[i][3] = a.w, q.x[i][4] = b.x, q.x[i][5] = b.y, q.x[i][6] = b.z, q.x[i][7] = b.w;
    }
}
template <int D, int FMT>
__device__ __forceinline__ void put_q_row(const AttnP& P, uint8_t* qt, int r, int l8, const QPieces<D>& q) {
    using Q = QTile<D>;
    constexpr int kCh = QPieces<D>::kCh, kPer = QPieces<D>::kPer;
    const float(&x)[kPer][8] = q.x;
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fabsf(x[i][k]));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    float up, down;
    row_scale(amax, up, down);
    if (l8 == 0) reinterpret_cast<float*>(qt + Q::kYsc)[r] = P.sc * down * kCodeUp<FMT>;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int ch = i * 8 + l8;
        if (FMT == 16) {
            if (ch < kCh) {
                uint4 hi, lo;
                split2(x[i][0] * up, x[i][1] * up, hi.x, lo.x);
                split2(x[i][2] * up, x[i][3] * up, hi.y, lo.y);
                split2(x[i][4] * up, x[i][5] * up, hi.z, lo.z);
                split2(x[i][6] * up, x[i][7] * up, hi.w, lo.w);
                *reinterpret_cast<uint4*>(qt + r * Q::kRow + ch * 16) = hi;
                *reinterpret_cast<uint4*>(qt + Q::kLo + r * Q::kRow + ch * 16) = lo;
            }
        } else {
            const int b = ch / 4, c = ch % 4;  // piece c of block b: its four pairs (k, k + 4) go to four k places
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                sum += x[i][k] + x[i][k + 4];
                if (ch < kCh) {
                    unsigned hi, lo;
                    split2(x[i][k] * up, x[i][k + 4] * up, hi, lo);
                    const int at = r * Q::kRow + 2 * (16 * (2 * b + (k >> 1)) + 8 * (k & 1) + 2 * c);
                    *reinterpret_cast<unsigned*>(qt + at) = hi;
                    *reinterpret_cast<unsigned*>(qt + Q::kLo + at) = lo;
                }
            }
            sum = quad_sum(sum);
            if (ch < kCh && c == 0) reinterpret_cast<float*>(qt + Q::kSums)[r * (D / 32 + 1) + b] = sum * up * (1.0f / kCodeUp<FMT>);
        }
    }
}
template <int D, int FMT>
__device__ __forceinline__ void load_q_tile(const AttnP& P, int s, int kvh, int row0, uint8_t* qt, int tid) {
    const int l8 = tid & 7;
#pragma unroll 1
    for (int r = tid >> 3; r < QTile<D>::kRows; r += 16) {
        QPieces<D> q;
        fetch_q_row<D>(P, s, kvh, row0 + r, l8, q);
        put_q_row<D, FMT>(P, qt, r, l8, q);
    }
}
// Products of this warp's 16 rows (row r0 of the query tile on) with NTL n-tiles of 8 slots, from 16-slot block `blk0` of a key
// tile of KROWS slots on.  s[nt][0, 1]: row g, [2, 3]: row g + 8; columns as slot_of gives them.
template <int D, int FMT, int NTL, int KROWS>
__device__ __forceinline__ void scores16(float (&sc)[NTL][4], const uint8_t* qt, int r0, const uint8_t* kt, int blk0, int lane) {
    using Q = QTile<D>;
    using T = Tile<D, FMT>;
    constexpr int NB = D / 32;
    const int g = lane >> 2, c = lane & 3;
    const uint32_t qa = smem_u32(qt) + (r0 + (lane & 15)) * Q::kRow + (lane >> 4) * 16;
#pragma unroll
    for (int nt = 0; nt < NTL; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.0f;
    if (FMT == 16) {
        const uint32_t ka = smem_u32(kt) + (blk0 * 16 + (lane & 7) + (lane >> 4) * 8) * T::kRow + ((lane >> 3) & 1) * 16;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            unsigned ah[4], al[4];
            ldsm4(ah, qa + ks * 32);
            ldsm4(al, qa + Q::kLo + ks * 32);
#pragma unroll
            for (int n2 = 0; n2 < NTL / 2; ++n2) {
                unsigned b[4];
                ldsm4(b, ka + n2 * 16 * T::kRow + ks * 32);
                mma16816(sc[2 * n2], ah, b[0], b[1]);
                mma16816(sc[2 * n2 + 1], ah, b[2], b[3]);
                mma16816(sc[2 * n2], al, b[0], b[1]);
                mma16816(sc[2 * n2 + 1], al, b[2], b[3]);
            }
        }
    } else {
        const uint8_t* kp = kt + KROWS * T::kRow;
        const float* sums = reinterpret_cast<const float*>(qt + Q::kSums) + (r0 + g) * (NB + 1);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            unsigned ah[2][4], al[2][4];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                ldsm4(ah[k], qa + (2 * b + k) * 32);
                ldsm4(al[k], qa + Q::kLo + (2 * b + k) * 32);
            }
            const float s0 = sums[b], s1 = sums[8 * (NB + 1) + b];
#pragma unroll
            for (int nt = 0; nt < NTL; ++nt) {
                const int at = (blk0 + nt / 2) * 16;
                const unsigned w = *reinterpret_cast<const unsigned*>(kt + (at + row_of_column<FMT>(nt & 1, g)) * T::kRow + (c * NB + b) * 4);
                const unsigned hi = w >> 8;
                float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                const unsigned c0 = code_pair<false, false>(w), c1 = code_pair<true, false>(w), c2 = code_pair<false, false>(hi), c3 = code_pair<true, false>(hi);
                mma16816(a, ah[0], c0, c1);
                mma16816(a, al[0], c0, c1);
                mma16816(a, ah[1], c2, c3);
                mma16816(a, al[1], c2, c3);
                const uint8_t* pp = kp + (at + 8 * (nt & 1) + c) * T::kPar + 4 * b;
                const float2 d0 = __half22float2(*reinterpret_cast<const __half2*>(pp)), d1 = __half22float2(*reinterpret_cast<const __half2*>(pp + 4 * T::kPar));
                sc[nt][0] = fmaf(d0.x, a[0], fmaf(d0.y, s0, sc[nt][0])), sc[nt][1] = fmaf(d1.x, a[1], fmaf(d1.y, s0, sc[nt][1]));
                sc[nt][2] = fmaf(d0.x, a[2], fmaf(d0.y, s1, sc[nt][2])), sc[nt][3] = fmaf(d1.x, a[3], fmaf(d1.y, s1, sc[nt][3]));
            }
        }
    }
}

// ---- tile kernel: 64 rows per CTA ---------------------------------------------------------------------------------------------
// For prompts of the shapes that the tcgen05 kernel does not take.  Four warps of 16 rows share every key and value tile; what bounds it is the tensor pipe (two products for
// each of the two contractions).  A tile's value products start from zero and are added to the running output in fp32, so
// the length of the context never meets the rounding of the tensor cores' accumulation.
// Measured: 2048 tokens over 2048 slots, 16 heads over 8, D = 256, no mask: 722 us = 95 TFLOP/s (fp16), 832 us (4 bits).
template <int D, int FMT>
struct TileCfg {
    static constexpr int kKeys = D >= 256 ? 32 : 64;
    static constexpr int kPlane = Tile<D, FMT>::bytes(kKeys);
    static constexpr int kOffKv = QTile<D>::kBytes;
    static constexpr int kOffBits = kOffKv + 4 * kPlane;  // bitmap of the tiles that hold a document of these rows
    static constexpr int kSmem = kOffBits + kDocBits / 8;
    static_assert(kSmem <= kMaxSmem);
};

template <int D, int FMT, bool GEN>
__global__ void __launch_bounds__(128) attn_tile_kernel(const __grid_constant__ AttnP P) {
    using C = TileCfg<D, FMT>;
    using T = Tile<D, FMT>;
    using Q = QTile<D>;
    constexpr int NB = D / 32, NT = D / 8, TK = C::kKeys, NS = TK / 8, KK = TK / 16;
    extern __shared__ __align__(16) uint8_t sm[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    // the last rows see the most keys: they start first
    const int rt = P.row_tiles - 1 - static_cast<int>(blockIdx.x) / P.nsplit, split = blockIdx.x % P.nsplit, kvh = blockIdx.y, s = blockIdx.z;
    const int row0 = rt * Q::kRows;
    const int n = seq_keys(P, s);
    const int chunk = (n + P.nsplit * 64 - 1) / (P.nsplit * 64) * 64;
    const int begin = min(n, split * chunk);
    int end = min(n, begin + chunk);
    const int last_row = min(P.rows, row0 + Q::kRows) - 1;
    const int tok0 = row0 / P.group, tok1 = last_row / P.group;
    const int prefix = GEN && P.prefix ? P.prefix[s] : 0;
    if (P.causal && !P.positions && !P.q_pos)  // no row here sees a slot behind the last token's position or the prefix
        end = max(begin, causal_limit(row_pos(P, s, n, tok1), prefix, end));
    const int nt = (end - begin + TK - 1) / TK;

    const bool docs = GEN && P.q_doc != nullptr;
    const DocTiles<TK> doc_tiles{reinterpret_cast<uint32_t*>(sm + C::kOffBits), nt};
    if (docs) {
        doc_tiles.clear(tid, 128);
        __syncthreads();
        doc_tiles.find(P, s, tok0, tok1, begin, end, warp, 4, lane);
    }
    load_q_tile<D, FMT>(P, s, kvh, row0, sm, tid);
    __syncthreads();
    auto next = [&](int i) { return docs ? doc_tiles.next(i) : i + 1; };  // the tile behind tile i that is wanted
    auto fetch = [&](int i, int stage) {
        if (i < nt) {
            const uint32_t dst = smem_u32(sm) + C::kOffKv + stage * 2 * C::kPlane;
            load_tile<D, FMT, TK, 128>(P, P.k, P.k_row, P.k_head, P.k_seq, s, kvh, begin + i * TK, end, dst, tid);
            load_tile<D, FMT, TK, 128>(P, P.v, P.v_row, P.v_head, P.v_seq, s, kvh, begin + i * TK, end, dst + C::kPlane, tid);
        }
        cp_commit();
    };
    const int ra = row0 + warp * 16 + g, rb = ra + 8;
    RowInfo ia, ib;
    int lima = n, limb = n;
    if (GEN) {
        ia = row_info(P, s, kvh, n, ra), ib = row_info(P, s, kvh, n, rb);
    } else {
        if (P.causal) {
            lima = ra < P.rows ? causal_limit(row_pos(P, s, n, ra / P.group), 0, n) : 0;
            limb = rb < P.rows ? causal_limit(row_pos(P, s, n, rb / P.group), 0, n) : 0;
        }
    }
    const float* yscp = reinterpret_cast<const float*>(sm + Q::kYsc) + warp * 16 + g;
    const float ysa = yscp[0], ysb = yscp[8];
    const bool hides = GEN || P.causal;

    float o[NT][4], oma[FMT == 16 ? 1 : NB], omb[FMT == 16 ? 1 : NB];
    float ma = -INFINITY, mb = -INFINITY, la = 0.0f, lb = 0.0f;
#pragma unroll
    for (int j = 0; j < NT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
#pragma unroll
    for (int b = 0; b < (FMT == 16 ? 1 : NB); ++b) oma[b] = omb[b] = 0.0f;

    int cur = next(-1), stage = 0;
    fetch(cur, 0);
    while (cur < nt) {
        const int nxt = next(cur);
        fetch(nxt, stage ^ 1);
        cp_wait<1>();
        const uint8_t* kt = sm + C::kOffKv + stage * 2 * C::kPlane;
        const uint8_t* vt = kt + C::kPlane;
        const int t0 = begin + cur * TK;
        bool dirty = false;
        if (FMT == 16 && hides) {  // the chunks this thread copied itself: a value that is not finite?
#pragma unroll
            for (int i = 0; i < TK * (D / 8) / 128; ++i) {
                const int x = i * 128 + tid;
                dirty = dirty || not_finite(*reinterpret_cast<const uint4*>(vt + x / (D / 8) * T::kRow + x % (D / 8) * 16));
            }
        }
        if (FMT == 16) dirty = __syncthreads_or(dirty);
        else __syncthreads();

        float sc[NS][4];
        scores16<D, FMT, NS, TK>(sc, sm, warp * 16, kt, 0, lane);
        float xa = -INFINITY, xb = -INFINITY;
#pragma unroll
        for (int j = 0; j < NS; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int t = t0 + (j >> 1) * 16 + slot_of<FMT>(c, 2 * (j & 1) + e);
                if (GEN) {
                    const KeyInfo key = key_info(P, s, kvh, t, end);
                    sc[j][e] = general_score(P, sc[j][e] * ysa, ia, key, t, end, prefix);
                    sc[j][2 + e] = general_score(P, sc[j][2 + e] * ysb, ib, key, t, end, prefix);
                } else {
                    sc[j][e] = t < min(lima, end) ? sc[j][e] * ysa : -INFINITY;
                    sc[j][2 + e] = t < min(limb, end) ? sc[j][2 + e] * ysb : -INFINITY;
                }
                xa = fmaxf(xa, sc[j][e]), xb = fmaxf(xb, sc[j][2 + e]);
            }
        if (FMT != 16) {  // scales of 16 and more raise the reference so that p d stays in fp16's range (see the rows kernel)
            const uint8_t* pp = vt + TK * T::kRow;
            unsigned big = 0;
#pragma unroll
            for (int x = 0; x < (TK * NB + 31) / 32; ++x)
                if (x * 32 + lane < TK * NB) big |= *reinterpret_cast<const unsigned*>(pp + 4 * (x * 32 + lane)) & 0x7FFFu;
            if (__any_sync(0xffffffffu, big >= 0x4C00u)) {
#pragma unroll
                for (int j = 0; j < NS; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        unsigned dm = 0;
                        for (int b = 0; b < NB; ++b)
                            dm = max(dm, *reinterpret_cast<const unsigned*>(pp + ((j >> 1) * 16 + slot_of<FMT>(c, 2 * (j & 1) + e)) * T::kPar + 4 * b) & 0x7FFFu);
                        const float more = static_cast<float>(max(0, static_cast<int>(dm >> 10) - 18));
                        if (sc[j][e] != -INFINITY) xa = fmaxf(xa, sc[j][e] + more);
                        if (sc[j][2 + e] != -INFINITY) xb = fmaxf(xb, sc[j][2 + e] + more);
                    }
            }
        }
        xa = fmaxf(ma, quad_max(xa)), xb = fmaxf(mb, quad_max(xb));
        float fa = xa > ma ? ex2(ma - xa) : 1.0f, fb = xb > mb ? ex2(mb - xb) : 1.0f;
        ma = xa, mb = xb;
        const float refa = ma == -INFINITY ? 0.0f : ma - kPShift, refb = mb == -INFINITY ? 0.0f : mb - kPShift;
        la *= fa, lb *= fb;
#pragma unroll
        for (int j = 0; j < NS; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                sc[j][e] = ex2(sc[j][e] - refa), sc[j][2 + e] = ex2(sc[j][2 + e] - refb);
                la += sc[j][e], lb += sc[j][2 + e];
            }
        if (FMT == 16) {
            if (dirty) {  // rare, the same for the whole CTA: such values go to the rows that see them one by one, and become zeros
                float pl[NS * 4];
#pragma unroll
                for (int x = 0; x < NS * 4; ++x) pl[x] = sc[x >> 2][x & 3];
                fa = fmaxf(fa, 1e-30f), fb = fmaxf(fb, 1e-30f);  // an infinity added now stays one when the output is rescaled below
#pragma unroll 1
                for (int t = 0; t < TK; ++t) {
                    const int at = (t >> 3) * 4 + (t & 1), src = (lane & 28) + ((t & 7) >> 1);
                    const float pa = __shfl_sync(0xffffffffu, pl[at], src), pb = __shfl_sync(0xffffffffu, pl[at + 2], src);
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const unsigned w = *reinterpret_cast<const unsigned*>(vt + t * T::kRow + j * 16 + c * 4);
                        if (pa != 0.0f) add_not_finite(o[j][0], o[j][1], pa, w);
                        if (pb != 0.0f) add_not_finite(o[j][2], o[j][3], pb, w);
                    }
                }
                __syncthreads();
                for (int x = tid; x < TK * (D / 8); x += 128) zero_not_finite(sm + (vt - sm) + x / (D / 8) * T::kRow + x % (D / 8) * 16);
                __syncthreads();
            }
            unsigned ah[KK][4], al[KK][4];
#pragma unroll
            for (int k = 0; k < KK; ++k) {
                split2(sc[2 * k][0], sc[2 * k][1], ah[k][0], al[k][0]);
                split2(sc[2 * k][2], sc[2 * k][3], ah[k][1], al[k][1]);
                split2(sc[2 * k + 1][0], sc[2 * k + 1][1], ah[k][2], al[k][2]);
                split2(sc[2 * k + 1][2], sc[2 * k + 1][3], ah[k][3], al[k][3]);
            }
            const uint32_t va = smem_u32(vt) + ((lane & 7) + ((lane >> 3) & 1) * 8) * T::kRow + (lane >> 4) * 16;
#pragma unroll
            for (int j = 0; j < NT / 2; ++j) {
                float x0[4] = {0.0f, 0.0f, 0.0f, 0.0f}, x1[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < KK; ++k) {
                    unsigned b[4];
                    ldsm4t(b, va + k * 16 * T::kRow + j * 32);
                    mma16816(x0, ah[k], b[0], b[1]);
                    mma16816(x1, ah[k], b[2], b[3]);
                    mma16816(x0, al[k], b[0], b[1]);
                    mma16816(x1, al[k], b[2], b[3]);
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    o[2 * j][e] = fmaf(o[2 * j][e], fa, x0[e]), o[2 * j][2 + e] = fmaf(o[2 * j][2 + e], fb, x0[2 + e]);
                    o[2 * j + 1][e] = fmaf(o[2 * j + 1][e], fa, x1[e]), o[2 * j + 1][2 + e] = fmaf(o[2 * j + 1][2 + e], fb, x1[2 + e]);
                }
            }
        } else {
            const uint8_t* pp = vt + TK * T::kRow;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                unsigned ah[KK][4], al[KK][4];
                float sa = 0.0f, sb = 0.0f;
#pragma unroll
                for (int k = 0; k < KK; ++k) {
                    float da[4], db[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float pa = sc[2 * k + (j >> 1)][j & 1], pb = sc[2 * k + (j >> 1)][2 + (j & 1)];
                        const float2 dm = __half22float2(*reinterpret_cast<const __half2*>(pp + (16 * k + slot_of<FMT>(c, j)) * T::kPar + 4 * b));
                        // a hidden slot's scales may be anything
                        da[j] = pa != 0.0f ? pa * dm.x : 0.0f, db[j] = pb != 0.0f ? pb * dm.x : 0.0f;
                        const float mid = fmaf(8.0f, dm.x, dm.y);
                        sa = pa != 0.0f ? fmaf(pa, mid, sa) : sa, sb = pb != 0.0f ? fmaf(pb, mid, sb) : sb;
                    }
                    split2(da[0], da[1], ah[k][0], al[k][0]);
                    split2(db[0], db[1], ah[k][1], al[k][1]);
                    split2(da[2], da[3], ah[k][2], al[k][2]);
                    split2(db[2], db[3], ah[k][3], al[k][3]);
                }
                oma[b] = fmaf(oma[b], fa, sa), omb[b] = fmaf(omb[b], fb, sb);
                float x[4][4] = {};
#pragma unroll
                for (int k = 0; k < KK; ++k) {
                    unsigned w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const unsigned short*>(vt + (16 * k + c + 4 * j) * T::kRow + (g * NB + b) * 2);
                    const unsigned x0 = w[0] | (w[1] << 16), x1 = w[2] | (w[3] << 16), h0 = x0 >> 8, h1 = x1 >> 8;
                    const unsigned c0[4] = {code_pair<false, true>(x0), code_pair<true, true>(x0), code_pair<false, true>(h0), code_pair<true, true>(h0)};
                    const unsigned c1[4] = {code_pair<false, true>(x1), code_pair<true, true>(x1), code_pair<false, true>(h1), code_pair<true, true>(h1)};
#pragma unroll
                    for (int i = 0; i < 4; ++i) mma16816(x[i], ah[k], c0[i], c1[i]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) mma16816(x[i], al[k], c0[i], c1[i]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        o[4 * b + i][e] = fmaf(o[4 * b + i][e], fa, x[i][e]);
                        o[4 * b + i][2 + e] = fmaf(o[4 * b + i][2 + e], fb, x[i][2 + e]);
                    }
            }
        }
        __syncthreads();
        cur = nxt, stage ^= 1;
    }
    cp_wait<0>();
    la = quad_sum(la), lb = quad_sum(lb);

    const size_t part = ((static_cast<size_t>(s) * P.kv_heads + kvh) * P.nsplit + split) * P.rows;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = h ? rb : ra;
        const float L = h ? lb : la, M = h ? mb : ma;
        float f = 1.0f;
        float* dst;
        if (P.nsplit > 1) {
            dst = P.part_o + (part + row) * D;
        } else {
            f = L > 0.0f || L != L ? 1.0f / L : 0.0f;
            const int tok = row / P.group, head = kvh * P.group + row % P.group;
            dst = P.out + static_cast<size_t>(s) * P.o_seq + static_cast<size_t>(tok) * P.o_token + static_cast<size_t>(head) * P.o_head;
        }
        if (FMT == 16) {
            if (row < P.rows)
#pragma unroll
                for (int j = 0; j < NT; ++j) *reinterpret_cast<float2*>(dst + 8 * j + 2 * c) = make_float2(o[j][2 * h] * f, o[j][2 * h + 1] * f);
        } else {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float mm = quad_sum(h ? omb[b] : oma[b]);
                float r[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    r[i] = fmaf(o[4 * b + i][2 * h], kCodeUp<FMT>, mm) * f;
                    r[4 + i] = fmaf(o[4 * b + i][2 * h + 1], kCodeUp<FMT>, mm) * f;
                }
                if (row < P.rows) {
                    reinterpret_cast<float4*>(dst + 32 * b + 8 * c)[0] = make_float4(r[0], r[1], r[2], r[3]);
                    reinterpret_cast<float4*>(dst + 32 * b + 8 * c)[1] = make_float4(r[4], r[5], r[6], r[7]);
                }
            }
        }
        if (c == 0 && row < P.rows) {
            if (P.nsplit > 1) P.part_ml[part + row] = make_float2(M, L);
            else if (P.final_ml) P.final_ml[(static_cast<size_t>(s) * P.kv_heads + kvh) * P.rows + row] = make_float2(M, L);
        }
    }
}

// ---- attention weights per key ---------------------------------------------------------------------------------------------------
// weights[t] += sum over the rows of a kv head of softmax(z)_t, from the rows' final maximum and sum.  A CTA owns 64 slots and
// goes over all rows in order, so nothing is added atomically and the result does not depend on timing.  Sixteen warps: four blocks of
// 16 slots times the four steps of 16 rows of a query tile, whose successor is on its way from memory meanwhile.  Where there are
// few slots, the CTAs of a cluster take the query tiles in turn, and the first one adds up their sums in order.
// Bounded by issue slots: per 8 scores of a lane 32 products, their 24 fragment loads and some 60 instructions to sum weights.
// Measured: 2048 tokens, 32 heads over 8, D = 128: 500 us (fp16), 750 (4 bits) behind 219 and 381 of attention; 300 tokens, 8 heads over
// 2, over 500 slots 17 us in clusters of 8, 53 without.
template <int D, int FMT>
struct WeightsCfg {
    static constexpr int kThreads = 512;
    static constexpr int kOffK = QTile<D>::kBytes;
    static constexpr int kOffRows = kOffK + Tile<D, FMT>::bytes(64);  // per row: RowInfo, {reference, 1 / sum}
    static constexpr int kOffMl = kOffRows + QTile<D>::kRows * static_cast<int>(sizeof(RowInfo));
    static constexpr int kOffSum = kOffMl + QTile<D>::kRows * 8;      // [step][slot]
    static constexpr int kSmem = kOffSum + 4 * 64 * 4;
    static_assert(kOffRows % 16 == 0 && kOffMl % 8 == 0 && kThreads == 8 * QTile<D>::kRows);
};
// GEN = false: neither cap nor bias, documents or mask.  The two branch-free tests that are left decide by the key's position alone.
template <int D, int FMT, bool GEN>
__global__ void __launch_bounds__(WeightsCfg<D, FMT>::kThreads, D <= 128 ? 2 : 1) attn_weights_kernel(const __grid_constant__ AttnP P, int ranks) {
    using C = WeightsCfg<D, FMT>;
    using Q = QTile<D>;
    extern __shared__ __align__(16) uint8_t sm[];
    const int tid = threadIdx.x, lane = tid & 31, blk = (tid >> 5) & 3, step = tid >> 7, g = lane >> 2, c = lane & 3;
    const int t0 = blockIdx.x / ranks * 64, rank = blockIdx.x % ranks, kvh = blockIdx.y, s = blockIdx.z;
    grid_dependency_wait();
    const int n = seq_keys(P, s);
    if (t0 >= n) return;
    const uint8_t* kt = sm + C::kOffK;
    if (tid < 128) load_tile<D, FMT, 64, 128>(P, P.k, P.k_row, P.k_head, P.k_seq, s, kvh, t0, n, smem_u32(kt), tid);
    cp_commit();
    const int prefix = P.prefix ? P.prefix[s] : 0;
    KeyInfo key[4];
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        key[j] = key_info(P, s, kvh, t0 + blk * 16 + slot_of<FMT>(c, j), n);
        if (!GEN && (!P.causal || key[j].pos < prefix)) key[j].pos = INT32_MIN;  // every row sees it (what lies behind n is not stored)
    }
    int row0 = 0;
    if (P.causal && !P.positions && !P.q_pos && t0 >= prefix) {  // rows in front of the first token that sees slot t0
        const int first = t0 - row_pos(P, s, n, 0);
        if (first > 0) row0 = static_cast<int>(min(static_cast<long long>(P.rows), static_cast<long long>(first) * P.group)) / Q::kRows * Q::kRows;
    }
    row0 += rank * Q::kRows;
    const int stride = ranks * Q::kRows;
    RowInfo* infos = reinterpret_cast<RowInfo*>(sm + C::kOffRows);
    float2* mls = reinterpret_cast<float2*>(sm + C::kOffMl);
    // a thread's part of a query tile: pieces of row tid / 8, and for one of the eight what that row needs to know
    const int qr = tid >> 3, l8 = tid & 7;
    QPieces<D> q;
    RowInfo info{};
    float2 ml{};
    auto fetch = [&](int first) {
        const int row = first + qr;
        fetch_q_row<D>(P, s, kvh, row, l8, q);
        if (l8 == 0) {
            info = row_info(P, s, kvh, n, row);
            ml = info.valid ? P.final_ml[(static_cast<size_t>(s) * P.kv_heads + kvh) * P.rows + row] : make_float2(0.0f, 0.0f);
        }
    };
    if (row0 < P.rows) fetch(row0);
    for (; row0 < P.rows; row0 += stride) {
        put_q_row<D, FMT>(P, sm, qr, l8, q);
        if (l8 == 0) infos[qr] = info, mls[qr] = ml.y != 0.0f ? make_float2(ml.x - kPShift, 1.0f / ml.y) : make_float2(0.0f, 0.0f);
        if (P.rows - row0 > stride) fetch(row0 + stride);
        cp_wait<0>();
        __syncthreads();
        const int r0 = step * 16;
        if (row0 + r0 < P.rows) {
            float sc[2][4];
            scores16<D, FMT, 2, 64>(sc, sm, r0, kt, blk, lane);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = r0 + 8 * h + g;
                const float2 m = mls[r];
                const float ys = reinterpret_cast<const float*>(sm + Q::kYsc)[r];
                if (!GEN) {
                    const int pos = infos[r].pos;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float p = ex2(fmaf(sc[j >> 1][2 * h + (j & 1)], ys, -m.x)) * m.y;
                        sum[j] += key[j].pos <= pos && m.y != 0.0f ? p : 0.0f;
                    }
                    continue;
                }
                const RowInfo ri = infos[r];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float y = general_score(P, sc[j >> 1][2 * h + (j & 1)] * ys, ri, key[j], t0 + blk * 16 + slot_of<FMT>(c, j), n, prefix);
                    sum[j] += y == -INFINITY || m.y == 0.0f ? 0.0f : ex2(y - m.x) * m.y;
                }
            }
        }
        __syncthreads();
    }
    cp_wait<0>();
    float* sums = reinterpret_cast<float*>(sm + C::kOffSum);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float v = sum[j];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        if (g == 0) sums[step * 64 + blk * 16 + slot_of<FMT>(c, j)] = v;
    }
    __syncthreads();
    float all = 0.0f;
    if (tid < 64) all = (sums[tid] + sums[64 + tid]) + (sums[128 + tid] + sums[192 + tid]);
    if (ranks > 1) {
        if (tid < 64) sums[tid] = all;  // (only this thread read that word)
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (rank == 0 && tid < 64)
            for (int i = 1; i < ranks; ++i) {
                float x;
                asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}" : "=f"(x) : "r"(smem_u32(sums + tid)), "r"(i) : "memory");
                all += x;
            }
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");  // their memory is read
    }
    if (rank == 0 && tid < 64 && t0 + tid < n) P.weights[(static_cast<size_t>(s) * P.kv_heads + kvh) * P.cap + t0 + tid] += all;
}

// ---- launches --------------------------------------------------------------------------------------------------------------------
// kv_attention_tc.cuh
template <int D, int FMT>
int attn_launch_tc(const AttnP& P, bool general, cudaStream_t st);

template <int D, int FMT, bool GEN>
int attn_launch_tile(const AttnP& P, cudaStream_t st) {
    constexpr int smem = TileCfg<D, FMT>::kSmem;
    static PerDeviceFlag raised;
    const dim3 grid(P.row_tiles * P.nsplit, P.kv_heads, P.n_seqs);
    if (!raise_dynamic_smem(attn_tile_kernel<D, FMT, GEN>, smem, raised)) return KCB_LAUNCH_FAILURE;
    attn_tile_kernel<D, FMT, GEN><<<grid, 128, smem, st>>>(P);
    return launch_status();
}
template <int D, int FMT, int MODE>
int attn_launch_rows(const AttnP& P, cudaStream_t st) {
    constexpr int smem = RowsCfg<D, FMT>::kSmem;
    static PerDeviceFlag raised;
    if (!raise_dynamic_smem(attn_rows_kernel<D, FMT, MODE>, smem, raised)) return KCB_LAUNCH_FAILURE;
    attn_rows_kernel<D, FMT, MODE><<<dim3(P.nsplit, P.kv_heads * P.row_tiles, P.n_seqs), 32 * kRowsWarps, smem, st>>>(P);
    return launch_status();
}
template <int D, int FMT>
int attn_launch_kernels(const AttnP& P, bool general, AttnKernel which, cudaStream_t st) {
    if (which == AttnKernel::tc) {
        int e = KCB_UNSUPPORTED_OPERATION;
        if constexpr (FMT == 16 && D <= 128) e = attn_launch_tc_dim<D <= 64 ? 64 : 128>(P, general, st);  // 32 and 96: in the next wider kernel
        else if constexpr (D == 64 || D == 128) e = attn_launch_tc<D, FMT>(P, general, st);
        if constexpr (FMT == 16 && D <= 128)
            if (e == KCB_UNSUPPORTED_OPERATION) {  // strides that a tensor map does not take (sequences that share one cache: stride 0)
                AttnP T = P;
                T.row_tiles = (P.rows + QTile<D>::kRows - 1) / QTile<D>::kRows;
                e = attn_launch_tile<D, FMT, true>(T, st);
            }
        if (e != KCB_SUCCESS) return e;
    } else if (which == AttnKernel::tile) {
        int e = KCB_UNSUPPORTED_OPERATION;
        if constexpr (D == 256 || (FMT == 4 && D != 64 && D != 128))  // the shapes that tcgen05 does not take
            e = general ? attn_launch_tile<D, FMT, true>(P, st) : attn_launch_tile<D, FMT, false>(P, st);
        if (e != KCB_SUCCESS) return e;
    } else {
        int e;
        if (P.positions || P.q_doc || P.mask) e = attn_launch_rows<D, FMT, 2>(P, st);
        else if (P.cap_out != 0.0f || P.bias_step != 0.0f) e = attn_launch_rows<D, FMT, 1>(P, st);
        else e = attn_launch_rows<D, FMT, 0>(P, st);
        if (e != KCB_SUCCESS) return e;
    }
    const bool by_warps = P.nsplit <= kMergeWarps || (P.nsplit <= 32 && static_cast<long long>(P.rows) * P.kv_heads * P.n_seqs > 8 * kSmCount);
    if (P.nsplit > 1 && by_warps && !P.scores) {
        const int e = launch_dependent(attn_merge_warps_kernel<D>, dim3((P.rows + kMergeWarps - 1) / kMergeWarps, P.kv_heads, P.n_seqs), 32 * kMergeWarps, 0, st, P);
        if (e != KCB_SUCCESS) return e;
    } else if (P.nsplit > 1 || P.scores) {
        const int joins = P.nsplit > 1 ? P.rows : 0, weights = P.scores ? (P.cap + kWeightSlots - 1) / kWeightSlots : 0;
        const int e = launch_dependent(attn_merge_kernel<D>, dim3(joins + weights, P.kv_heads, P.n_seqs), 32 * kMergeWarps, 0, st, P, joins);
        if (e != KCB_SUCCESS) return e;
    }
    if (P.final_ml) {
        static PerDeviceFlag raised[2];
        const bool gen = P.cap_out != 0.0f || P.bias_step != 0.0f || P.q_doc || P.mask;
        const auto kernel = gen ? attn_weights_kernel<D, FMT, true> : attn_weights_kernel<D, FMT, false>;
        if (!raise_dynamic_smem(kernel, WeightsCfg<D, FMT>::kSmem, raised[gen])) return KCB_LAUNCH_FAILURE;
        const long long blocks = (P.cap + 63) / 64, tiles = (P.rows + QTile<D>::kRows - 1) / QTile<D>::kRows;
        int ranks = 1;  // clusters of up to 8 while the GPU has room for twice the CTAs
        while (ranks < 8 && 2 * ranks <= tiles && 2 * ranks * blocks * P.kv_heads * P.n_seqs <= 2 * kSmCount) ranks *= 2;
        return launch_clusters(kernel, dim3(static_cast<unsigned>(blocks) * ranks, P.kv_heads, P.n_seqs), ranks, WeightsCfg<D, FMT>::kThreads, WeightsCfg<D, FMT>::kSmem, st, P, ranks);
    }
    return KCB_SUCCESS;
}
}  // namespace kcb

// KV cache for long contexts: rows in (fp16 or 4 bits), rows back out, eviction by accumulated attention weight, and the
// host side of the attention entry (kv_attention.cuh).
//
// The 4-bit format.  A block is 32 channels of one row: minimum m = fp16(min x), scale d = fp16((max x - min x) * fp32(1 / 15)),
// code = the integer in 0..15 nearest to (x - m) / d (ties to even), value d code + m.  Per sequence a plane of nibbles
// [kv_heads][capacity][D / 2 bytes], then a plane of parameters [kv_heads][capacity][D / 32]{d, m}: 0.625 bytes a value.
// A row's bytes are grouped for the tensor-core lane that multiplies them: in a key row the 4 bytes of channels 8 c .. 8 c + 7
// of all blocks lie together for c = 0..3, in a value row the 2 bytes of channels 4 g .. 4 g + 3 of all blocks for g = 0..7.

#include "common.cuh"
#include "kv_attention.cuh"
#include "kv_cache.h"

#include <algorithm>
#include <cmath>

namespace kcb {
namespace {

// ---- rows in ---------------------------------------------------------------------------------------------------------------
// Bounded by memory: 4 bytes read and 2 or 0.625 written per value.  Eight lanes hold a block of 32 channels, so a warp reads
// 512 contiguous bytes and reduces minima and maxima in three shuffle steps.
// The code is rounded from the exact quotient: the fp32 quotient decides unless it lies near a half, where fp64 does.
__device__ __forceinline__ unsigned code_of(float x, float m, float d, float inv) {
    const float t = (x - m) * inv;
    float r = rintf(t);
    // t is off by at most 16 * 3 * 2^-24 < 3e-6; between 0.4999 and 0.5001 from an integer the quotient is taken in 64 bits
    if (fabsf(fabsf(t - r) - 0.5f) < 1e-4f) r = static_cast<float>(rint((static_cast<double>(x) - static_cast<double>(m)) / static_cast<double>(d)));
    return static_cast<unsigned>(static_cast<int>(fminf(fmaxf(r, 0.0f), 15.0f)));
}
struct AppendP {
    kcb_kv_cache c;
    const float* k;
    const float* v;
    long long tok, seq, seq_bytes, par_off;
    int n_tokens;
};
__device__ __forceinline__ float cache_value(float x) {  // what a cache can hold: NaN -> 0, the rest within fp16's range
    return x != x ? 0.0f : fminf(fmaxf(x, -65504.0f), 65504.0f);
}
template <int BITS>
__global__ void __launch_bounds__(256) kv_append_rows_kernel(const __grid_constant__ AppendP A) {
    const kcb_kv_cache& c = A.c;
    const int per_row = c.head_dim / 4;  // lanes of four channels
    const long long total = static_cast<long long>(A.n_tokens) * c.kv_heads * per_row * 2;
    const int s = blockIdx.y;
    const int n0 = max(0, c.n_keys[s]);
    const int first_pos = c.next_pos ? c.next_pos[s] : n0;
    for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += static_cast<long long>(gridDim.x) * blockDim.x) {
        const int j = static_cast<int>(i % per_row);
        long long x = i / per_row;
        const int h = static_cast<int>(x % c.kv_heads);
        x /= c.kv_heads;
        const bool val = x >= A.n_tokens;
        const int tok = static_cast<int>(val ? x - A.n_tokens : x);
        const long long t = static_cast<long long>(n0) + tok;
        const float* src = (val ? A.v : A.k) + s * A.seq + tok * A.tok + static_cast<long long>(h) * c.head_dim + 4 * j;
        const float4 f = *reinterpret_cast<const float4*>(src);
        const bool fits = t < c.capacity;  // rows beyond the capacity are dropped
        if (BITS == 16) {
            if (fits) {
                __half* dst = static_cast<__half*>(val ? c.v : c.k) + (val ? c.v_seq : c.k_seq) * s + (val ? c.v_head : c.k_head) * h + (val ? c.v_row : c.k_row) * t + 4 * j;
                *reinterpret_cast<uint2*>(dst) = make_uint2(f32_to_f16_bits(f.x) | (f32_to_f16_bits(f.y) << 16), f32_to_f16_bits(f.z) | (f32_to_f16_bits(f.w) << 16));
            }
        } else {
            const float e[4] = {cache_value(f.x), cache_value(f.y), cache_value(f.z), cache_value(f.w)};
            float lo = fminf(fminf(e[0], e[1]), fminf(e[2], e[3])), hi = fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3]));
            const unsigned who = 0xFFu << (threadIdx.x & 24);  // the block's eight lanes come and go together (total is a multiple of 8)
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) lo = fminf(lo, __shfl_xor_sync(who, lo, o)), hi = fmaxf(hi, __shfl_xor_sync(who, hi, o));
            const __half mh = __float2half_rn(lo), dh = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
            const float m = __half2float(mh), d = __half2float(dh), inv = d > 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
            unsigned w = 0;
            if (d > 0.0f)
#pragma unroll
                for (int k = 0; k < 4; ++k) w |= code_of(e[k], m, d, inv) << (4 * k);
            if (fits) {
                const int nb = c.head_dim / 32, b = j >> 3, jj = j & 7;
                uint8_t* base = static_cast<uint8_t*>(val ? c.v : c.k) + A.seq_bytes * s;
                const long long row = static_cast<long long>(h) * c.capacity + t;
                const int at = val ? (jj * nb + b) * 2 : ((jj >> 1) * nb + b) * 4 + (jj & 1) * 2;
                *reinterpret_cast<unsigned short*>(base + row * (c.head_dim / 2) + at) = static_cast<unsigned short>(w);
                if (jj == 0) *reinterpret_cast<__half2*>(base + A.par_off + (row * nb + b) * 4) = __halves2half2(dh, mh);
            }
        }
        if (j == 0 && !val && fits) {
            const long long at = (static_cast<long long>(s) * c.kv_heads + h) * c.capacity + t;
            if (c.positions) c.positions[at] = first_pos + tok;
            if (c.weights) c.weights[at] = 0.0f;
        }
    }
}
// The counts move on in a launch of their own: every CTA of the rows' launch reads them.
__global__ void kv_count_kernel(int* n_keys, int* next_pos, int n_seqs, int capacity, int n_tokens) {
    for (int s = blockIdx.x * blockDim.x + threadIdx.x; s < n_seqs; s += gridDim.x * blockDim.x) {
        const long long n = static_cast<long long>(max(0, n_keys[s])) + n_tokens;
        const long long p = static_cast<long long>(next_pos ? next_pos[s] : 0) + n_tokens;
        n_keys[s] = static_cast<int>(n < capacity ? n : capacity);
        if (next_pos) next_pos[s] = static_cast<int>(p);
    }
}

// ---- rows out ----------------------------------------------------------------------------------------------------------------
struct ReadP {
    kcb_kv_cache c;
    float* k;
    float* v;
    long long seq_bytes, par_off;
    int first, count;
};
template <int BITS>
__global__ void __launch_bounds__(256) kv_read_rows_kernel(const __grid_constant__ ReadP R) {
    const kcb_kv_cache& c = R.c;
    const int per_row = c.head_dim / 4;
    const long long total = static_cast<long long>(R.count) * c.kv_heads * per_row * 2;
    const int s = blockIdx.y;
    const int n = c.n_keys ? min(max(0, c.n_keys[s]), c.capacity) : c.capacity;
    for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += static_cast<long long>(gridDim.x) * blockDim.x) {
        const int j = static_cast<int>(i % per_row);
        long long x = i / per_row;
        const int h = static_cast<int>(x % c.kv_heads);
        x /= c.kv_heads;
        const bool val = x >= R.count;
        const int r = static_cast<int>(val ? x - R.count : x);
        const long long t = static_cast<long long>(R.first) + r;
        float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (t < n) {
            if (BITS == 16) {
                const __half* src = static_cast<const __half*>(val ? c.v : c.k) + (val ? c.v_seq : c.k_seq) * s + (val ? c.v_head : c.k_head) * h + (val ? c.v_row : c.k_row) * t + 4 * j;
                const uint2 w = *reinterpret_cast<const uint2*>(src);
                f = make_float4(half_bits_to_float(w.x & 0xFFFFu), half_bits_to_float(w.x >> 16), half_bits_to_float(w.y & 0xFFFFu), half_bits_to_float(w.y >> 16));
            } else {
                const int nb = c.head_dim / 32, b = j >> 3, jj = j & 7;
                const uint8_t* base = static_cast<const uint8_t*>(val ? c.v : c.k) + R.seq_bytes * s;
                const long long row = static_cast<long long>(h) * c.capacity + t;
                const int at = val ? (jj * nb + b) * 2 : ((jj >> 1) * nb + b) * 4 + (jj & 1) * 2;
                const unsigned w = *reinterpret_cast<const unsigned short*>(base + row * (c.head_dim / 2) + at);
                const float2 dm = __half22float2(*reinterpret_cast<const __half2*>(base + R.par_off + (row * nb + b) * 4));
                f = make_float4(fmaf(dm.x, static_cast<float>(w & 15u), dm.y), fmaf(dm.x, static_cast<float>(w >> 4 & 15u), dm.y),
                                fmaf(dm.x, static_cast<float>(w >> 8 & 15u), dm.y), fmaf(dm.x, static_cast<float>(w >> 12), dm.y));
            }
        }
        float* dst = (val ? R.v : R.k) + ((static_cast<long long>(s) * R.count + r) * c.kv_heads + h) * c.head_dim + 4 * j;
        *reinterpret_cast<float4*>(dst) = f;
    }
}

// ---- eviction ------------------------------------------------------------------------------------------------------------------
// Which rows stay: one CTA per (sequence, kv head).  A row's key orders first the protected rows (position at or after next_pos -
// recent), then the others by weight; a radix selection over the 32-bit keys finds the keep-th largest, rows that tie with it stay
// from the lowest slot on.  Then the free slots below `keep` and the kept rows at or behind it are listed in ascending order: the
// j-th kept row moves into the j-th free slot, so sources and destinations are disjoint and the rows can move in place, in
// parallel and in any order (the positions beside them say where a row belongs).
constexpr int kSelThreads = 1024;
constexpr int kSelKeys = 50 * 1024;  // keys kept in shared memory; longer caches compute them anew in every pass

struct EvictP {
    kcb_kv_cache c;
    int keep, recent, max_moves;
    int* counts;  // [seq][head]
    int2* moves;  // [seq][head][max_moves] {from, to}
    long long seq_bytes, par_off;
};
__device__ __forceinline__ unsigned weight_key(float w) {
    if (w != w) return 0u;                       // a NaN weight goes first
    if (w == 0.0f) return 0x80000000u;           // both zeros alike
    const unsigned b = __float_as_uint(w);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ int block_scan_exclusive(int v, int* warps, int& total) {  // warps: 33 ints of shared memory
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) warps[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int t = warps[lane], y = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int z = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) y += z;
        }
        warps[lane] = y - t;
        if (lane == 31) warps[32] = y;
    }
    __syncthreads();
    total = warps[32];
    return warps[warp] + x - v;
}
__global__ void __launch_bounds__(kSelThreads) kv_select_kernel(const __grid_constant__ EvictP E) {
    extern __shared__ unsigned keys[];
    __shared__ int hist[256], scan[33], digit, rest;
    const kcb_kv_cache& c = E.c;
    const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
    const size_t sh = static_cast<size_t>(s) * c.kv_heads + h;
    const int n = min(max(0, c.n_keys[s]), c.capacity), keep = E.keep;
    if (n <= keep) {
        if (tid == 0) E.counts[sh] = 0;
        return;
    }
    const int* pos = c.positions + sh * c.capacity;
    const float* w = c.weights + sh * c.capacity;
    const long long from = static_cast<long long>(c.next_pos[s]) - E.recent;
    const bool held = n <= kSelKeys;
    auto make_key = [&](int t) { return pos[t] >= from ? 0xFFFFFFFFu : weight_key(w[t]); };
    auto key_of = [&](int t) { return held ? keys[t] : make_key(t); };
    if (held)
        for (int t = tid; t < n; t += kSelThreads) keys[t] = make_key(t);
    unsigned prefix = 0, mask = 0;
    int need = keep;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        for (int t = tid; t < n; t += kSelThreads) {
            const unsigned k = key_of(t);
            if ((k & mask) == prefix) atomicAdd(&hist[k >> shift & 255u], 1);
        }
        __syncthreads();
        if (tid < 32) {  // from the largest digit down: where does the need-th key fall?
            int sum = 0;
            for (int i = 0; i < 8; ++i) sum += hist[255 - (tid * 8 + i)];
            int before = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, before, o);
                if (tid >= o) before += y;
            }
            before -= sum;
            if (before < need && need <= before + sum) {
                int left = need - before, i = 0;
                while (left > hist[255 - (tid * 8 + i)]) left -= hist[255 - (tid * 8 + i)], ++i;
                digit = 255 - (tid * 8 + i), rest = left;
            }
        }
        __syncthreads();
        prefix |= static_cast<unsigned>(digit) << shift;
        mask |= 255u << shift;
        need = rest;
        __syncthreads();
    }
    // prefix: the keep-th largest key; `need` rows that equal it stay.  Each thread looks after a run of neighbouring slots.
    const int run = (n + kSelThreads - 1) / kSelThreads, t0 = min(n, tid * run), t1 = min(n, t0 + run);
    int ties = 0, total;
    for (int t = t0; t < t1; ++t) ties += key_of(t) == prefix;
    const int tie0 = block_scan_exclusive(ties, scan, total);
    int holes = 0, tails = 0, tie = tie0;
    for (int t = t0; t < t1; ++t) {
        const unsigned k = key_of(t);
        const bool kept = k > prefix || (k == prefix && tie++ < need);
        if (t < keep) holes += !kept;
        else tails += kept;
    }
    int hole = block_scan_exclusive(holes, scan, total);
    int tail = block_scan_exclusive(tails, scan, total);
    if (tid == 0) E.counts[sh] = total;
    int2* mv = E.moves + sh * E.max_moves;
    tie = tie0;
    for (int t = t0; t < t1; ++t) {
        const unsigned k = key_of(t);
        const bool kept = k > prefix || (k == prefix && tie++ < need);
        if (t < keep) {
            if (!kept) mv[hole++].y = t;
        } else if (kept) {
            mv[tail++].x = t;
        }
    }
}
// Bounded by memory: every moved row is read and written once.  One warp per row, keys and values 16 (or, for the parameters of
// narrow heads, 4) bytes a lane.
template <int BITS>
__global__ void __launch_bounds__(256) kv_move_kernel(const __grid_constant__ EvictP E) {
    const kcb_kv_cache& c = E.c;
    const int h = blockIdx.y, s = blockIdx.z, lane = threadIdx.x & 31;
    const size_t sh = static_cast<size_t>(s) * c.kv_heads + h;
    const int count = E.counts[sh];
    if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) c.n_keys[s] = min(max(0, c.n_keys[s]), E.keep);
    for (int j = blockIdx.x * 8 + (threadIdx.x >> 5); j < count; j += gridDim.x * 8) {
        const int2 mv = E.moves[sh * E.max_moves + j];
        if (BITS == 16) {
            const int chunks = c.head_dim / 8;
            for (int x = lane; x < 2 * chunks; x += 32) {
                const bool val = x >= chunks;
                __half* base = static_cast<__half*>(val ? c.v : c.k) + (val ? c.v_seq : c.k_seq) * s + (val ? c.v_head : c.k_head) * h;
                const long long row = val ? c.v_row : c.k_row;
                const int ch = (val ? x - chunks : x) * 8;
                *reinterpret_cast<uint4*>(base + mv.y * row + ch) = *reinterpret_cast<const uint4*>(base + mv.x * row + ch);
            }
        } else {
            const int nb = c.head_dim / 32;
            for (int x = lane; x < 4 * nb; x += 32) {  // per plane: nb chunks of 16 bytes of nibbles, nb words of parameters
                const bool val = x >= 2 * nb;
                const int y = val ? x - 2 * nb : x;
                uint8_t* base = static_cast<uint8_t*>(val ? c.v : c.k) + E.seq_bytes * s;
                const long long from = static_cast<long long>(h) * c.capacity + mv.x, to = static_cast<long long>(h) * c.capacity + mv.y;
                if (y < nb) {
                    *reinterpret_cast<uint4*>(base + to * (16 * nb) + y * 16) = *reinterpret_cast<const uint4*>(base + from * (16 * nb) + y * 16);
                } else {
                    uint8_t* par = base + E.par_off;
                    *reinterpret_cast<unsigned*>(par + to * (4 * nb) + (y - nb) * 4) = *reinterpret_cast<const unsigned*>(par + from * (4 * nb) + (y - nb) * 4);
                }
            }
        }
        if (lane == 0) {
            const size_t at = sh * c.capacity;
            c.positions[at + mv.y] = c.positions[at + mv.x];
            c.weights[at + mv.y] = c.weights[at + mv.x];
        }
    }
}

// ---- host side -----------------------------------------------------------------------------------------------------------------
constexpr int kMaxGrid = 65535;

// Shape and pointers of a cache; 0 or a status code.
int cache_ok(const kcb_kv_cache* c) {
    if (!c || (c->bits != KCB_CACHE_F16 && c->bits != KCB_CACHE_Q4) || c->n_seqs < 0 || c->n_seqs > kMaxGrid || c->kv_heads <= 0 || c->kv_heads > 4096 ||
        c->head_dim <= 0 || c->head_dim % 32 || c->head_dim > 256 || c->capacity <= 0 || c->capacity > (1 << 30) || !c->k || !c->v)
        return KCB_INVALID_VALUE;
    if (misaligned(c->k, 16) || misaligned(c->v, 16) || misaligned(c->n_keys, 4) || misaligned(c->next_pos, 4) || misaligned(c->positions, 4) ||
        misaligned(c->weights, 4))
        return KCB_INVALID_POINTER;
    if (c->bits == KCB_CACHE_F16) {
        const int64_t st[6] = {c->k_row, c->k_head, c->k_seq, c->v_row, c->v_head, c->v_seq};
        for (int64_t x : st) {
            if (x < 0) return KCB_INVALID_VALUE;
            if (x % 8) return KCB_INVALID_POINTER;  // rows are read 16 bytes at a time
        }
    }
    return KCB_SUCCESS;
}
size_t moves_offset(const kcb_kv_cache* c) { return (static_cast<size_t>(c->n_seqs) * c->kv_heads * 4 + 15) / 16 * 16; }
unsigned row_blocks(const kcb_kv_cache* c, int rows) {
    const long long threads = static_cast<long long>(rows) * c->kv_heads * (c->head_dim / 4) * 2;
    return static_cast<unsigned>(std::min<long long>((threads + 255) / 256, 1 << 20));
}

// How an attention call is cut: by rows (single tokens) or by tiles of 64 rows (prompts), and into how many ranges of keys.
struct AttnCut {
    bool tile;
    int row_tiles, nsplit;
    size_t ml_bytes, o_bytes, final_bytes;
};
constexpr int kRowsMax = 16;
AttnCut attn_cut(const kcb_kv_cache* c, const kcb_cache_attn* a) {
    AttnCut r{};
    const long long rows = static_cast<long long>(a->n_tokens) * (a->heads / c->kv_heads);
    r.tile = rows > kRowsMax;
    r.row_tiles = static_cast<int>(r.tile ? (rows + 63) / 64 : (rows + 7) / 8);
    const long long ctas = static_cast<long long>(c->n_seqs) * c->kv_heads * r.row_tiles;
    const long long want = r.tile ? 2 * kSmCount : 4 * kSmCount, least = r.tile ? 512 : 256;
    long long n = std::min<long long>((want + ctas - 1) / std::max<long long>(ctas, 1), (c->capacity + least - 1) / least);
    r.nsplit = static_cast<int>(std::max<long long>(1, n));
    const size_t parts = static_cast<size_t>(c->n_seqs) * c->kv_heads * rows * (r.nsplit > 1 ? r.nsplit : 0);
    r.ml_bytes = (parts * sizeof(float2) + 15) / 16 * 16;
    r.o_bytes = parts * c->head_dim * sizeof(float);
    r.final_bytes = a->accumulate ? (static_cast<size_t>(c->n_seqs) * c->kv_heads * rows * sizeof(float2) + 15) / 16 * 16 : 0;
    return r;
}
int attn_ok(const kcb_kv_cache* c, const kcb_cache_attn* a) {
    if (const int e = cache_ok(c); e != KCB_SUCCESS) return e;
    if (!a || a->n_tokens < 0 || a->heads <= 0 || a->heads % c->kv_heads || !std::isfinite(a->scale) || !(a->softcap >= 0.0f) || !std::isfinite(a->softcap) ||
        !(a->max_bias >= 0.0f) || !std::isfinite(a->max_bias))
        return KCB_INVALID_VALUE;
    const long long rows = static_cast<long long>(a->n_tokens) * (a->heads / c->kv_heads);
    if (rows > (1 << 24)) return KCB_INVALID_VALUE;
    if ((a->q_doc == nullptr) != (a->k_doc == nullptr)) return KCB_INVALID_VALUE;
    if (a->prefix && !a->causal) return KCB_INVALID_VALUE;
    // documents and masks go by slot; a cache with positions keeps different rows in the same slot of different heads
    if (c->positions && (a->k_doc || a->mask)) return KCB_INVALID_VALUE;
    if (a->accumulate && !c->weights) return KCB_INVALID_VALUE;
    const int64_t st[6] = {a->q_token, a->q_head, a->q_seq, a->out_token, a->out_head, a->out_seq};
    for (int64_t x : st) {
        if (x < 0) return KCB_INVALID_VALUE;
        if (x % 4) return KCB_INVALID_POINTER;  // queries and outputs move 16 bytes at a time
    }
    if (a->mask && (a->mask_token < 0 || a->mask_seq < 0)) return KCB_INVALID_VALUE;
    if (misaligned(a->prefix, 4) || misaligned(a->q_pos, 4) || misaligned(a->q_doc, 4) || misaligned(a->k_doc, 4) || misaligned(a->mask, 2)) return KCB_INVALID_POINTER;
    if (c->head_dim == 160 || c->head_dim == 192 || c->head_dim == 224) return KCB_UNSUPPORTED_OPERATION;
    return KCB_SUCCESS;
}

}  // namespace
}  // namespace kcb

using namespace kcb;

extern "C" {

size_t kcb_cache_bytes(int bits, int n_seqs, int kv_heads, int head_dim, int capacity) {
    if (n_seqs < 0 || kv_heads <= 0 || head_dim <= 0 || head_dim % 32 || capacity <= 0) return 0;
    if (bits == KCB_CACHE_F16) return static_cast<size_t>(n_seqs) * kv_heads * capacity * head_dim * 2;
    return bits == KCB_CACHE_Q4 ? static_cast<size_t>(n_seqs) * q4_seq_bytes(kv_heads, head_dim, capacity) : 0;
}

int kcb_cache_append(const kcb_kv_cache* c, const float* k, const float* v, int n_tokens, int64_t token_stride, int64_t seq_stride, void* stream) {
    if (const int e = cache_ok(c); e != KCB_SUCCESS) return e;
    if (!c->n_keys || !k || !v || n_tokens < 0 || token_stride < 0 || seq_stride < 0) return KCB_INVALID_VALUE;
    if (misaligned(k, 16) || misaligned(v, 16) || token_stride % 4 || seq_stride % 4) return KCB_INVALID_POINTER;
    if (n_tokens == 0 || c->n_seqs == 0) return KCB_SUCCESS;
    const auto st = static_cast<cudaStream_t>(stream);
    AppendP A{*c, k, v, token_stride, seq_stride, static_cast<long long>(q4_seq_bytes(c->kv_heads, c->head_dim, c->capacity)),
              static_cast<long long>(q4_param_offset(c->kv_heads, c->head_dim, c->capacity)), n_tokens};
    const dim3 grid(row_blocks(c, n_tokens), c->n_seqs);
    if (c->bits == KCB_CACHE_F16) kv_append_rows_kernel<16><<<grid, 256, 0, st>>>(A);
    else kv_append_rows_kernel<4><<<grid, 256, 0, st>>>(A);
    if (const int e = launch_status(); e != KCB_SUCCESS) return e;
    kv_count_kernel<<<(c->n_seqs + 255) / 256, 256, 0, st>>>(c->n_keys, c->next_pos, c->n_seqs, c->capacity, n_tokens);
    return launch_status();
}

int kcb_cache_read(const kcb_kv_cache* c, int first, int count, float* k_out, float* v_out, void* stream) {
    if (const int e = cache_ok(c); e != KCB_SUCCESS) return e;
    if (!k_out || !v_out || first < 0 || count < 0 || first > c->capacity - count) return KCB_INVALID_VALUE;
    if (misaligned(k_out, 16) || misaligned(v_out, 16)) return KCB_INVALID_POINTER;
    if (count == 0 || c->n_seqs == 0) return KCB_SUCCESS;
    const auto st = static_cast<cudaStream_t>(stream);
    ReadP R{*c, k_out, v_out, static_cast<long long>(q4_seq_bytes(c->kv_heads, c->head_dim, c->capacity)),
            static_cast<long long>(q4_param_offset(c->kv_heads, c->head_dim, c->capacity)), first, count};
    const dim3 grid(row_blocks(c, count), c->n_seqs);
    if (c->bits == KCB_CACHE_F16) kv_read_rows_kernel<16><<<grid, 256, 0, st>>>(R);
    else kv_read_rows_kernel<4><<<grid, 256, 0, st>>>(R);
    return launch_status();
}

size_t kcb_cache_evict_workspace_bytes(const kcb_kv_cache* c, int keep) {
    if (!c || c->n_seqs < 0 || c->kv_heads <= 0 || keep < 0 || keep >= c->capacity) return 0;
    return moves_offset(c) + static_cast<size_t>(c->n_seqs) * c->kv_heads * std::min(keep, c->capacity - keep) * sizeof(int2);
}

int kcb_cache_evict(const kcb_kv_cache* c, int keep, int recent, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int e = cache_ok(c); e != KCB_SUCCESS) return e;
    if (!c->n_keys || !c->next_pos || !c->positions || !c->weights || keep <= 0 || recent < 0 || recent > keep) return KCB_INVALID_VALUE;
    if (keep >= c->capacity || c->n_seqs == 0) return KCB_SUCCESS;  // no sequence can hold more
    if (!workspace || workspace_bytes < kcb_cache_evict_workspace_bytes(c, keep)) return KCB_INVALID_VALUE;
    if (misaligned(workspace, 16)) return KCB_INVALID_POINTER;
    const auto st = static_cast<cudaStream_t>(stream);
    EvictP E{*c, keep, recent, std::min(keep, c->capacity - keep), static_cast<int*>(workspace),
             reinterpret_cast<int2*>(static_cast<uint8_t*>(workspace) + moves_offset(c)), static_cast<long long>(q4_seq_bytes(c->kv_heads, c->head_dim, c->capacity)),
             static_cast<long long>(q4_param_offset(c->kv_heads, c->head_dim, c->capacity))};
    static PerDeviceFlag raised;
    if (!raise_dynamic_smem(kv_select_kernel, kSelKeys * 4, raised)) return KCB_LAUNCH_FAILURE;
    kv_select_kernel<<<dim3(c->kv_heads, c->n_seqs), kSelThreads, std::min(c->capacity, kSelKeys) * 4, st>>>(E);
    if (const int e = launch_status(); e != KCB_SUCCESS) return e;
    const dim3 grid(std::min((E.max_moves + 7) / 8, 1024), c->kv_heads, c->n_seqs);
    if (c->bits == KCB_CACHE_F16) kv_move_kernel<16><<<grid, 256, 0, st>>>(E);
    else kv_move_kernel<4><<<grid, 256, 0, st>>>(E);
    return launch_status();
}

size_t kcb_cache_attention_workspace_bytes(const kcb_kv_cache* c, const kcb_cache_attn* a) {
    if (attn_ok(c, a) != KCB_SUCCESS || a->n_tokens == 0 || c->n_seqs == 0) return 0;
    const AttnCut cut = attn_cut(c, a);
    return cut.ml_bytes + cut.o_bytes + cut.final_bytes;
}

int kcb_cache_attention(const kcb_kv_cache* c, const kcb_cache_attn* a, const float* q, float* out, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int e = attn_ok(c, a); e != KCB_SUCCESS) return e;
    if (!q || !out) return KCB_INVALID_VALUE;
    if (misaligned(q, 16) || misaligned(out, 16)) return KCB_INVALID_POINTER;
    if (a->n_tokens == 0 || c->n_seqs == 0) return KCB_SUCCESS;
    const AttnCut cut = attn_cut(c, a);
    const size_t need = cut.ml_bytes + cut.o_bytes + cut.final_bytes;
    if (need && (!workspace || workspace_bytes < need)) return KCB_INVALID_VALUE;
    if (misaligned(workspace, 16)) return KCB_INVALID_POINTER;
    AttnP P{};
    P.k = static_cast<const uint8_t*>(c->k), P.v = static_cast<const uint8_t*>(c->v);
    P.k_row = c->k_row, P.k_head = c->k_head, P.k_seq = c->k_seq, P.v_row = c->v_row, P.v_head = c->v_head, P.v_seq = c->v_seq;
    P.par_off = static_cast<long long>(q4_param_offset(c->kv_heads, c->head_dim, c->capacity));
    P.seq_bytes = static_cast<long long>(q4_seq_bytes(c->kv_heads, c->head_dim, c->capacity));
    P.q = q, P.out = out;
    P.q_token = a->q_token, P.q_head = a->q_head, P.q_seq = a->q_seq, P.o_token = a->out_token, P.o_head = a->out_head, P.o_seq = a->out_seq;
    P.n_keys = c->n_keys, P.next_pos = c->next_pos, P.positions = c->positions, P.weights = c->weights;
    P.prefix = a->prefix, P.q_pos = a->q_pos, P.q_doc = a->q_doc, P.k_doc = a->k_doc;
    P.mask = static_cast<const unsigned short*>(a->mask), P.mask_token = a->mask_token, P.mask_seq = a->mask_seq;
    P.cap = c->capacity, P.n_seqs = c->n_seqs, P.n_tokens = a->n_tokens, P.heads = a->heads, P.kv_heads = c->kv_heads;
    P.group = a->heads / c->kv_heads, P.rows = a->n_tokens * P.group;
    P.causal = a->causal != 0;
    P.bias_log2_heads = 1;
    while (P.bias_log2_heads * 2 <= a->heads) P.bias_log2_heads *= 2;
    P.bias_step = a->max_bias / static_cast<float>(P.bias_log2_heads);
    P.sc = a->softcap > 0.0f ? a->scale / a->softcap : a->scale * kLog2e;
    P.cap_out = a->softcap * kLog2e;
    P.nsplit = cut.nsplit, P.row_tiles = cut.row_tiles;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    P.part_ml = reinterpret_cast<float2*>(ws), P.part_o = reinterpret_cast<float*>(ws + cut.ml_bytes);
    P.final_ml = a->accumulate ? reinterpret_cast<float2*>(ws + cut.ml_bytes + cut.o_bytes) : nullptr;
    const bool general = a->softcap > 0.0f || a->max_bias > 0.0f || c->positions || a->q_pos || a->q_doc || a->mask || a->prefix;
    const auto st = static_cast<cudaStream_t>(stream);
    return attn_launch_bits(P, c->bits, c->head_dim, general, cut.tile, st);
}

}  // extern "C"

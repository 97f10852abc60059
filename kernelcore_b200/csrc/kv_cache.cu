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
// 512 contiguous bytes and reduces minima and maxima in three shuffle steps.  8 sequences of 4096 tokens, 8 heads of 128: fp16 90 us =
// 4.5 TB/s; 4 bits 135 us = 2.3 TB/s, there bounded by the instructions that round codes.
// The code is rounded from the exact quotient: the fp32 quotient decides unless it lies near a half, where fp64 does.
__device__ __forceinline__ unsigned codes_of(const float (&x)[4], float m, float d, float inv) {
    constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to the nearest integer, to even at ties, into the low bits
    unsigned w = 0;
    float far = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float t = fminf(fmaxf((x[k] - m) * inv, 0.0f), 15.0f), z = t + kMagic;
        far = fmaxf(far, fabsf(t - (z - kMagic)));
        w |= (__float_as_uint(z) & 15u) << (4 * k);
    }
    // t is off by at most 16 * 3 * 2^-24 < 3e-6: nearer than 1e-4 to a half the quotient is taken in 64 bits
    if (far > 0.4999f) {
        w = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const double r = rint((static_cast<double>(x[k]) - static_cast<double>(m)) / static_cast<double>(d));
            w |= static_cast<unsigned>(fmin(fmax(r, 0.0), 15.0)) << (4 * k);
        }
    }
    return w;
}
// x / d by a multiplication: `inv` = ceil(2^32 / d) gives the quotient or one more for every x below 2^31.
__device__ __forceinline__ unsigned divide(unsigned x, unsigned d, unsigned inv) {
    if (d == 1) return x;
    const unsigned q = __umulhi(x, inv);
    return q * d > x ? q - 1 : q;
}
inline unsigned divisor(unsigned d) { return static_cast<unsigned>((0x100000000ull + d - 1) / d); }
// Where a row's four channels 4 jr .. 4 jr + 3 stand in the 4-bit planes: the two bytes of codes, the block's parameters.
struct Q4Place {
    size_t codes, params;
};
__device__ __forceinline__ Q4Place q4_place(const kcb_kv_cache& c, size_t par_off, bool val, int h, long long t, int jr) {
    const int nb = c.head_dim / 32, b = jr >> 3, jj = jr & 7;
    const size_t row = static_cast<size_t>(h) * c.capacity + t;
    const int at = val ? (jj * nb + b) * 2 : ((jj >> 1) * nb + b) * 4 + (jj & 1) * 2;
    return {row * (c.head_dim / 2) + at, par_off + (row * nb + b) * 4};
}
struct AppendP {
    kcb_kv_cache c;
    const float* k;
    const float* v;
    long long tok, seq, seq_bytes, par_off;
    unsigned heads_inv;
    int n_tokens, count;  // count: this launch also moves the counts on (one CTA per sequence)
};
__device__ __forceinline__ float cache_value(float x) {  // what a cache can hold: NaN -> 0, the rest within fp16's range
    return x != x ? 0.0f : fminf(fmaxf(x, -65504.0f), 65504.0f);
}
// D / 4 neighbouring threads to a row, kRowIter rows per thread and step so that as many loads are in flight.
constexpr int kRowThreads = 256, kRowIter = 4;
__device__ __forceinline__ void move_counts(int* n_keys, int* next_pos, int s, int capacity, int n_tokens) {
    const long long n = static_cast<long long>(max(0, n_keys[s])) + n_tokens;
    n_keys[s] = static_cast<int>(n < capacity ? n : capacity);
    if (next_pos) next_pos[s] += n_tokens;
}
template <int BITS>
__global__ void __launch_bounds__(kRowThreads) kv_append_rows_kernel(const __grid_constant__ AppendP A) {
    const kcb_kv_cache& c = A.c;
    const int per_row = c.head_dim / 4, per_cta = kRowThreads / per_row;  // (D = 96 leaves 16 threads idle)
    const int s = blockIdx.y, jr = threadIdx.x % per_row, r0 = threadIdx.x / per_row;
    const unsigned rows = static_cast<unsigned>(A.n_tokens) * c.kv_heads;  // keys, then the same number of values
    const int n0 = max(0, c.n_keys[s]);
    const int first_pos = c.next_pos ? c.next_pos[s] : n0;
    const bool live = r0 < per_cta;
    for (unsigned base = blockIdx.x * (per_cta * kRowIter); base < 2 * rows; base += gridDim.x * (per_cta * kRowIter)) {
        float4 f[kRowIter];
        unsigned hh[kRowIter], tt[kRowIter];
#pragma unroll
        for (int i = 0; i < kRowIter; ++i) {
            const unsigned r = base + i * per_cta + r0, x = r < rows ? r : r - rows;
            tt[i] = divide(x, c.kv_heads, A.heads_inv), hh[i] = x - tt[i] * c.kv_heads;
            f[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (live && r < 2 * rows) f[i] = *reinterpret_cast<const float4*>((r < rows ? A.k : A.v) + s * A.seq + tt[i] * A.tok + static_cast<long long>(hh[i]) * c.head_dim + 4 * jr);
        }
#pragma unroll
        for (int i = 0; i < kRowIter; ++i) {
            const unsigned r = base + i * per_cta + r0;
            const bool val = r >= rows;
            const long long t = static_cast<long long>(n0) + tt[i];
            const int h = static_cast<int>(hh[i]);
            const bool put = live && r < 2 * rows && t < c.capacity;  // rows beyond the capacity are dropped
            if (BITS == 16) {
                if (put) {
                    __half* dst = static_cast<__half*>(val ? c.v : c.k) + (val ? c.v_seq : c.k_seq) * s + (val ? c.v_head : c.k_head) * h + (val ? c.v_row : c.k_row) * t + 4 * jr;
                    *reinterpret_cast<uint2*>(dst) = make_uint2(f32_to_f16_bits(f[i].x) | (f32_to_f16_bits(f[i].y) << 16), f32_to_f16_bits(f[i].z) | (f32_to_f16_bits(f[i].w) << 16));
                }
            } else {
                const float e[4] = {cache_value(f[i].x), cache_value(f[i].y), cache_value(f[i].z), cache_value(f[i].w)};
                float lo = fminf(fminf(e[0], e[1]), fminf(e[2], e[3])), hi = fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3]));
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o)), hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
                const __half mh = __float2half_rn(lo), dh = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
                const float m = __half2float(mh), d = __half2float(dh), inv = d > 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
                const unsigned w = d > 0.0f ? codes_of(e, m, d, inv) : 0u;
                if (put) {
                    uint8_t* plane = static_cast<uint8_t*>(val ? c.v : c.k) + A.seq_bytes * s;
                    const Q4Place at = q4_place(c, A.par_off, val, h, t, jr);
                    *reinterpret_cast<unsigned short*>(plane + at.codes) = static_cast<unsigned short>(w);
                    if ((jr & 7) == 0) *reinterpret_cast<__half2*>(plane + at.params) = __halves2half2(dh, mh);
                }
            }
            if (jr == 0 && !val && put) {
                const size_t at = (static_cast<size_t>(s) * c.kv_heads + h) * c.capacity + t;
                if (c.positions) c.positions[at] = first_pos + static_cast<int>(tt[i]);
                if (c.weights) c.weights[at] = 0.0f;
            }
        }
    }
    if (A.count) {
        __syncthreads();
        if (threadIdx.x == 0) move_counts(c.n_keys, c.next_pos, s, c.capacity, A.n_tokens);
    }
}
// Where several CTAs write a sequence's rows, each of them reads the counts: those move on in a launch of their own.
__global__ void kv_count_kernel(int* n_keys, int* next_pos, int n_seqs, int capacity, int n_tokens) {
    grid_dependency_wait();
    for (int s = blockIdx.x * blockDim.x + threadIdx.x; s < n_seqs; s += gridDim.x * blockDim.x) move_counts(n_keys, next_pos, s, capacity, n_tokens);
}

// ---- rows out ----------------------------------------------------------------------------------------------------------------
// Bounded by memory: 2 or 0.625 bytes read and 4 written per value.  8 sequences of 4096 slots, 8 heads of 128: fp16 71 us = 5.7 TB/s, 4
// bits 69 us = 4.5 TB/s.
struct ReadP {
    kcb_kv_cache c;
    float* k;
    float* v;
    long long seq_bytes, par_off;
    unsigned heads_inv;
    int first, count;
};
template <int BITS>
__global__ void __launch_bounds__(kRowThreads) kv_read_rows_kernel(const __grid_constant__ ReadP R) {
    const kcb_kv_cache& c = R.c;
    const int per_row = c.head_dim / 4, per_cta = kRowThreads / per_row;
    const int s = blockIdx.y, jr = threadIdx.x % per_row, r0 = threadIdx.x / per_row;
    const unsigned rows = static_cast<unsigned>(R.count) * c.kv_heads;
    const int n = c.n_keys ? min(max(0, c.n_keys[s]), c.capacity) : c.capacity;
    if (r0 >= per_cta) return;
    for (unsigned base = blockIdx.x * (per_cta * kRowIter); base < 2 * rows; base += gridDim.x * (per_cta * kRowIter)) {
        uint2 w[kRowIter];  // fp16: four values; 4 bits: codes, {d, m}
#pragma unroll
        for (int i = 0; i < kRowIter; ++i) {
            const unsigned r = base + i * per_cta + r0, x = r < rows ? r : r - rows;
            const bool val = r >= rows;
            const unsigned tok = divide(x, c.kv_heads, R.heads_inv);
            const long long t = static_cast<long long>(R.first) + tok;
            const int h = static_cast<int>(x - tok * c.kv_heads);
            w[i] = make_uint2(0u, 0u);
            if (r >= 2 * rows || t >= n) continue;
            if (BITS == 16) {
                w[i] = *reinterpret_cast<const uint2*>(static_cast<const __half*>(val ? c.v : c.k) + (val ? c.v_seq : c.k_seq) * s + (val ? c.v_head : c.k_head) * h +
                                                       (val ? c.v_row : c.k_row) * t + 4 * jr);
            } else {
                const uint8_t* plane = static_cast<const uint8_t*>(val ? c.v : c.k) + R.seq_bytes * s;
                const Q4Place at = q4_place(c, R.par_off, val, h, t, jr);
                w[i] = make_uint2(*reinterpret_cast<const unsigned short*>(plane + at.codes), *reinterpret_cast<const unsigned*>(plane + at.params));
            }
        }
#pragma unroll
        for (int i = 0; i < kRowIter; ++i) {
            const unsigned r = base + i * per_cta + r0, x = r < rows ? r : r - rows;
            if (r >= 2 * rows) continue;
            float4 f;
            if (BITS == 16) {
                f = make_float4(half_bits_to_float(w[i].x & 0xFFFFu), half_bits_to_float(w[i].x >> 16), half_bits_to_float(w[i].y & 0xFFFFu), half_bits_to_float(w[i].y >> 16));
            } else {
                const float d = half_bits_to_float(w[i].y & 0xFFFFu), m = half_bits_to_float(w[i].y >> 16);
                f = make_float4(fmaf(d, static_cast<float>(w[i].x & 15u), m), fmaf(d, static_cast<float>(w[i].x >> 4 & 15u), m),
                                fmaf(d, static_cast<float>(w[i].x >> 8 & 15u), m), fmaf(d, static_cast<float>(w[i].x >> 12), m));
            }
            reinterpret_cast<float4*>((r < rows ? R.k : R.v) + (static_cast<size_t>(s) * rows + x) * c.head_dim)[jr] = f;
        }
    }
}

// ---- eviction ------------------------------------------------------------------------------------------------------------------
// Which rows stay: one CTA per (sequence, kv head).  A row's key orders first the protected rows (position at or after next_pos -
// recent), then the others by weight; a radix selection over the 32-bit keys finds the keep-th largest, rows that tie with it stay
// from the lowest slot on.  Then the free slots below `keep` and the kept rows at or behind it are listed in ascending order: the
// j-th kept row moves into the j-th free slot, so sources and destinations are disjoint and the rows can move in place, in
// parallel and in any order (the positions beside them say where a row belongs).
// Bounded by the latency of barriers and shared-memory atomics, three passes of them: 64 CTAs of 8192 keys 17 us, 128 of 1025 keys 8 us.
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
// Exclusive prefix over the warps of one value per warp (given in every lane); `total` over all.  slots: 33 ints of shared memory.
__device__ __forceinline__ int warp_prefix(int v, int* slots, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();
    if (lane == 0) slots[warp] = v;
    __syncthreads();
    if (warp == 0) {
        const int t = lane < static_cast<int>(blockDim.x >> 5) ? slots[lane] : 0;
        int y = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int z = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) y += z;
        }
        if (lane < static_cast<int>(blockDim.x >> 5)) slots[lane] = y - t;
        if (lane == 31) slots[32] = y;
    }
    __syncthreads();
    total = slots[32];
    return slots[warp];
}
template <int THREADS>
__global__ void __launch_bounds__(THREADS) kv_select_kernel(const __grid_constant__ EvictP E) {
    extern __shared__ unsigned keys[];
    __shared__ int hist[2048], slots[33], digit, rest;
    const kcb_kv_cache& c = E.c;
    const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const size_t sh = static_cast<size_t>(s) * c.kv_heads + h;
    grid_dependents_may_launch();
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
    // three digits of 11, 11 and 10 bits, from the top: so wide that the weights of a cache, which share few exponents, spread over
    // many counters
    unsigned prefix = 0, mask = 0;
    int need = keep;
#pragma unroll 1
    for (int round = 0; round < 3; ++round) {
        const int shift = round == 0 ? 21 : round == 1 ? 10 : 0, bins = round < 2 ? 2048 : 1024;
#pragma unroll
        for (int i = 0; i < 2048 / THREADS; ++i) hist[i * THREADS + tid] = 0;
        __syncthreads();
#pragma unroll 8
        for (int t = tid; t < n; t += THREADS) {
            unsigned k;
            if (round == 0) {
                k = make_key(t);
                if (held) keys[t] = k;
            } else {
                k = key_of(t);
            }
            if ((k & mask) == prefix) atomicAdd(&hist[k >> shift & (bins - 1)], 1);
        }
        __syncthreads();
        // from the largest digit down, neighbouring ones to a thread: where does the need-th key fall?
        constexpr int kMine = 2048 / THREADS;
        const int a = bins - 1 - kMine * tid;
        int h[kMine], sum = 0;
#pragma unroll
        for (int i = 0; i < kMine; ++i) sum += h[i] = a - i >= 0 ? hist[a - i] : 0;
        int before = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += y;
        }
        int all;
        before += warp_prefix(__shfl_sync(0xffffffffu, before, 31), slots, all) - sum;
        if (before < need && need <= before + sum) {
            int left = need - before;
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                if (left > 0 && left <= h[i]) digit = a - i, rest = left;
                left -= h[i];
            }
        }
        __syncthreads();
        prefix |= static_cast<unsigned>(digit) << shift;
        mask |= static_cast<unsigned>(bins - 1) << shift;
        need = rest;
        __syncthreads();
    }
    // prefix: the keep-th largest key; `need` rows that equal it stay.  Each warp looks after a run of neighbouring slots, 32 at a
    // time, so that ballots give the ascending order.
    constexpr int kWarps = THREADS / 32;
    const int run = ((n + kWarps - 1) / kWarps + 31) / 32 * 32, t0 = min(n, warp * run), t1 = min(n, t0 + run);
    const unsigned below = (1u << lane) - 1u;
    int ties = 0, total;
    for (int t = t0; t < t1; t += 32) ties += __popc(__ballot_sync(0xffffffffu, t + lane < t1 && key_of(t + lane) == prefix));
    const int tie0 = warp_prefix(ties, slots, total);
    // kept(t) of the 32 slots from t on, as a ballot; moves `tie` on
    auto kept_of = [&](int t, int& tie) {
        const unsigned k = t + lane < t1 ? key_of(t + lane) : 0u;
        const bool in = t + lane < t1, eq = in && k == prefix;
        const unsigned eqs = __ballot_sync(0xffffffffu, eq);
        const bool kept = in && (k > prefix || (eq && tie + __popc(eqs & below) < need));
        tie += __popc(eqs);
        return __ballot_sync(0xffffffffu, kept);
    };
    int holes = 0, tails = 0, tie = tie0;
    for (int t = t0; t < t1; t += 32) {
        const unsigned kept = kept_of(t, tie), first = __ballot_sync(0xffffffffu, t + lane < min(keep, t1));
        holes += __popc(first & ~kept), tails += __popc(~first & kept);
    }
    int hole = warp_prefix(holes, slots, total);
    int tail = warp_prefix(tails, slots, total);
    if (tid == 0) E.counts[sh] = total;
    int2* mv = E.moves + sh * E.max_moves;
    tie = tie0;
    for (int t = t0; t < t1; t += 32) {
        const unsigned kept = kept_of(t, tie), first = __ballot_sync(0xffffffffu, t + lane < min(keep, t1));
        const unsigned ho = first & ~kept, ta = ~first & kept;
        if (ho >> lane & 1u) mv[hole + __popc(ho & below)].y = t + lane;
        if (ta >> lane & 1u) mv[tail + __popc(ta & below)].x = t + lane;
        hole += __popc(ho), tail += __popc(ta);
    }
}
// Bounded by memory: every moved row is read and written once (8 sequences of 8 heads, keeping 2048 of 8192 rows of 128: 19 us = 5.3 TB/s).  A warp takes 16 moves at a time, four rows of them in flight.
// Chunk x of a row: 16 bytes of a key or value (fp16; 4 bits: nibbles, then the parameters four bytes at a time).
constexpr int kMoveWarps = 8, kMoveRows = 16;
template <int BITS>
__global__ void __launch_bounds__(32 * kMoveWarps) kv_move_kernel(const __grid_constant__ EvictP E) {
    const kcb_kv_cache& c = E.c;
    const int h = blockIdx.y, s = blockIdx.z, lane = threadIdx.x & 31;
    const size_t sh = static_cast<size_t>(s) * c.kv_heads + h;
    grid_dependency_wait();
    const int count = E.counts[sh];
    if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) c.n_keys[s] = min(max(0, c.n_keys[s]), E.keep);
    const int nb = c.head_dim / 32, chunks = BITS == 16 ? c.head_dim / 8 : 2 * nb;  // per plane
    for (int j0 = (blockIdx.x * kMoveWarps + (threadIdx.x >> 5)) * kMoveRows; j0 < count; j0 += gridDim.x * kMoveWarps * kMoveRows) {
        const int rows = min(kMoveRows, count - j0);
        const int2 mine = E.moves[sh * E.max_moves + j0 + min(lane, rows - 1)];
        if (lane < rows) {
            const size_t at = sh * c.capacity;
            c.positions[at + mine.y] = c.positions[at + mine.x];
            c.weights[at + mine.y] = c.weights[at + mine.x];
        }
        for (int x = lane; x - lane < 2 * chunks; x += 32) {
            const bool on = x < 2 * chunks, val = on && x >= chunks;
            const int y = val ? x - chunks : on ? x : 0;
            const bool wide = BITS == 16 || y < nb;
            uint8_t* base;
            size_t row;
            if (BITS == 16) {
                base = reinterpret_cast<uint8_t*>(static_cast<__half*>(val ? c.v : c.k) + (val ? c.v_seq : c.k_seq) * s + (val ? c.v_head : c.k_head) * h) + 16 * y;
                row = 2 * static_cast<size_t>(val ? c.v_row : c.k_row);
            } else {
                uint8_t* plane = static_cast<uint8_t*>(val ? c.v : c.k) + E.seq_bytes * s;
                row = wide ? 16 * nb : 4 * nb;
                base = plane + (wide ? 0 : E.par_off) + static_cast<size_t>(h) * c.capacity * row + (wide ? 16 * y : 4 * (y - nb));
            }
            for (int j = 0; j < rows; j += 4) {
                uint4 v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const size_t from = static_cast<size_t>(__shfl_sync(0xffffffffu, mine.x, min(j + i, rows - 1)));
                    v[i] = make_uint4(0u, 0u, 0u, 0u);
                    if (!on) continue;
                    if (wide) v[i] = *reinterpret_cast<const uint4*>(base + from * row);
                    else v[i].x = *reinterpret_cast<const unsigned*>(base + from * row);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const size_t to = static_cast<size_t>(__shfl_sync(0xffffffffu, mine.y, min(j + i, rows - 1)));
                    if (!on || j + i >= rows) continue;
                    if (wide) *reinterpret_cast<uint4*>(base + to * row) = v[i];
                    else *reinterpret_cast<unsigned*>(base + to * row) = v[i].x;
                }
            }
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
// Sequences, heads or slots that share their rows (stride 0) can be read, but two of them would write to the same place.
bool rows_apart(const kcb_kv_cache* c) {
    if (c->bits != KCB_CACHE_F16) return true;
    return (c->n_seqs <= 1 || (c->k_seq && c->v_seq)) && (c->kv_heads <= 1 || (c->k_head && c->v_head)) && (c->capacity <= 1 || (c->k_row && c->v_row));
}
size_t moves_offset(const kcb_kv_cache* c) { return (static_cast<size_t>(c->n_seqs) * c->kv_heads * 4 + 15) / 16 * 16; }
// CTAs of the rows-in and rows-out kernels for one sequence.
unsigned row_blocks(const kcb_kv_cache* c, int tokens) {
    const long long rows = 2LL * tokens * c->kv_heads, per_cta = kRowThreads / (c->head_dim / 4) * kRowIter;
    return static_cast<unsigned>(std::min<long long>((rows + per_cta - 1) / per_cta, 1 << 16));
}
constexpr long long kMaxRows = 1LL << 30;  // tokens * kv_heads of one call

// How an attention call is cut: by rows (single tokens) or by tiles of 64 rows (prompts), and into how many ranges of keys.
struct AttnCut {
    AttnKernel which;
    int row_tiles, nsplit;
    size_t ml_bytes, o_bytes, final_bytes, score_bytes;
    size_t bytes() const { return ml_bytes + o_bytes + final_bytes + score_bytes; }
};
// The tcgen05 kernel takes fp16 rows of 32 and 96 channels too, filled up with zeros to 64 and 128 by the tensor copies.
bool tc_takes(const kcb_kv_cache* c) { return c->bits == KCB_CACHE_F16 ? c->head_dim <= 128 : c->head_dim == 64 || c->head_dim == 128; }
// Which kernel (us on a B200, 32 query heads over 8, D = 128 unless said).  The rows kernel reads the cache once per 8 query rows of a
// kv head, straight into registers; the other two once per 64 or 128, through shared memory.
//   fp16, 8 rows: rows 45, tcgen05 47 (32768 slots), 129 and 137 (32 sequences of 4096).  16 rows: the long caches favour tcgen05 (59 and
//   47, 221 and 137), the short ones rows (512 slots: 12 and 18, 4096: 20.5 and 21.7); they meet near 2^17 slots over all heads and
//   sequences (D = 64: 25.8 and 31.6, D = 96: 35.8 and 33.8).  24 rows: 86 and 47.  With weights rows lead up to 16 (16 sequences of
//   4096: 206 and 208), for they keep the scores, where the others compute them anew.
//   4 bits, whose unpacking costs the tile kernels more than reading twice costs rows: 32 rows 67 and 83 (32768 slots), 237 and 305 (32
//   sequences); D = 64: 79 and 123, and 40 rows 95 and 123.
//   Where tcgen05 does not take a shape, rows and tiles: fp16, D = 256, 16 rows 302 and 437, 20 rows 439 and 439; 4 bits, D = 256, 20
//   rows 386 and 427, but 101 and 119 is no more than a fourth group of rows would cost.  The tile kernel never leads tcgen05 by more
//   than a tenth (4 bits, D = 64, up to 64 rows: 38 and 42), and loses by two to three from 96 rows on.
AttnKernel attn_kernel(const kcb_kv_cache* c, const kcb_cache_attn* a, long long rows) {
    const long long slots = static_cast<long long>(c->n_seqs) * c->kv_heads * c->capacity;
    long long few = kRowsMax / 2;
    if (c->bits == KCB_CACHE_Q4 && tc_takes(c)) few = kRowsMax;
    else if (tc_takes(c) && !a->accumulate && slots > 1 << 17) few = 8;
    return rows <= few ? AttnKernel::rows : tc_takes(c) ? AttnKernel::tc : AttnKernel::tile;
}
AttnCut attn_cut(const kcb_kv_cache* c, const kcb_cache_attn* a) {
    AttnCut r{};
    const long long rows = static_cast<long long>(a->n_tokens) * (a->heads / c->kv_heads);
    r.which = attn_kernel(c, a, rows);
    const int per = r.which == AttnKernel::rows ? 8 : r.which == AttnKernel::tile ? 64 : 128;
    r.row_tiles = static_cast<int>((rows + per - 1) / per);
    const long long ctas = static_cast<long long>(c->n_seqs) * c->kv_heads * r.row_tiles;
    // Keys are split until the GPU is full, one CTA per SM (tcgen05; 4 bits, 256 rows of 16384 slots: 86 us, with twice as many 96) or
    // two (rows and tiles; 64 rows of 16384: 47, with one 57), but into no fewer than 128 slots (12 rows of 512 slots: tcgen05 15, with
    // 512 slots a split 20; tiles 17 and 31; 64 slots gain nothing).
    const long long want = (r.which == AttnKernel::tc ? 1 : 2) * kSmCount, least = 128;
    r.nsplit = static_cast<int>(std::max<long long>(1, std::min<long long>(want / std::max<long long>(ctas, 1), (c->capacity + least - 1) / least)));
    // A rows launch adds values up on the tensor cores, whose sums truncate: at most 2048 slots per split are 32 additions per warp
    // (131072 4-bit rows, relative error against 64 bits: 6.4e-6 with 3543 slots a split, 2.7e-6 with 1771, 1.3e-6 with 885, which take
    // 70 us instead of 62).  More splits than the
    // GPU holds CTAs of (two per SM) come in whole rounds of them: 131072 rows of 8 heads 62 us in 74 splits, 67 us in 64.
    if (r.which == AttnKernel::rows && ctas) {
        const long long need = std::max<long long>(r.nsplit, (c->capacity + 2047) / 2048), round = 2 * kSmCount;
        r.nsplit = static_cast<int>(std::max(need, (ctas * need + round - 1) / round * round / ctas));
        if (r.nsplit > need && (c->capacity + r.nsplit - 1) / r.nsplit < least) r.nsplit = static_cast<int>(need);
    }
    // partial sums where keys are split; for weights the rows' final sums (tiles) or every score and the partial sums (rows)
    const size_t all = static_cast<size_t>(c->n_seqs) * c->kv_heads * rows;
    const bool weights = a->accumulate != 0;
    r.ml_bytes = r.nsplit > 1 || (weights && r.which == AttnKernel::rows) ? (all * r.nsplit * sizeof(float2) + 15) / 16 * 16 : 0;
    r.o_bytes = r.nsplit > 1 ? all * r.nsplit * c->head_dim * sizeof(float) : 0;
    r.final_bytes = weights && r.which != AttnKernel::rows ? (all * sizeof(float2) + 15) / 16 * 16 : 0;
    r.score_bytes = weights && r.which == AttnKernel::rows ? all * c->capacity * sizeof(float) : 0;
    return r;
}
int attn_ok(const kcb_kv_cache* c, const kcb_cache_attn* a) {
    if (const int e = cache_ok(c); e != KCB_SUCCESS) return e;
    if (!a || a->n_tokens < 0 || a->heads <= 0 || a->heads % c->kv_heads || !std::isfinite(a->scale) || !(a->softcap >= 0.0f) || !std::isfinite(a->softcap) ||
        !(a->max_bias >= 0.0f) || !std::isfinite(a->max_bias) || !std::isfinite(a->scale * kLog2e))
        return KCB_INVALID_VALUE;
    // scores over their cap, and the cap, stay far inside fp32's range
    if (const float bend = std::fabs(a->scale) / a->softcap; a->softcap > 0.0f && a->scale != 0.0f && !(bend >= 1e-20f && bend <= 1e20f)) return KCB_INVALID_VALUE;
    if (!std::isfinite(a->softcap * kLog2e)) return KCB_INVALID_VALUE;
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
    if (!c->n_keys || !k || !v || n_tokens < 0 || token_stride < 0 || seq_stride < 0 || !rows_apart(c)) return KCB_INVALID_VALUE;
    if (misaligned(k, 16) || misaligned(v, 16) || token_stride % 4 || seq_stride % 4) return KCB_INVALID_POINTER;
    if (static_cast<long long>(n_tokens) * c->kv_heads > kMaxRows) return KCB_INVALID_VALUE;
    if (n_tokens == 0 || c->n_seqs == 0) return KCB_SUCCESS;
    const auto st = static_cast<cudaStream_t>(stream);
    const unsigned blocks = row_blocks(c, n_tokens);
    // a step's few rows: one CTA per sequence, which also moves the counts on (6.2 us, in two launches 8.2; from two CTAs' rows on 10.2
    // and 8.2)
    const bool one = blocks == 1;
    AppendP A{*c, k, v, token_stride, seq_stride, static_cast<long long>(q4_seq_bytes(c->kv_heads, c->head_dim, c->capacity)),
              static_cast<long long>(q4_param_offset(c->kv_heads, c->head_dim, c->capacity)), divisor(c->kv_heads), n_tokens, one};
    const dim3 grid(one ? 1 : blocks, c->n_seqs);
    if (c->bits == KCB_CACHE_F16) kv_append_rows_kernel<16><<<grid, kRowThreads, 0, st>>>(A);
    else kv_append_rows_kernel<4><<<grid, kRowThreads, 0, st>>>(A);
    if (const int e = launch_status(); e != KCB_SUCCESS || one) return e;
    return launch_dependent(kv_count_kernel, dim3((c->n_seqs + 255) / 256), 256, 0, st, c->n_keys, c->next_pos, c->n_seqs, c->capacity, n_tokens);
}

int kcb_cache_read(const kcb_kv_cache* c, int first, int count, float* k_out, float* v_out, void* stream) {
    if (const int e = cache_ok(c); e != KCB_SUCCESS) return e;
    if (!k_out || !v_out || first < 0 || count < 0 || first > c->capacity - count) return KCB_INVALID_VALUE;
    if (misaligned(k_out, 16) || misaligned(v_out, 16)) return KCB_INVALID_POINTER;
    if (static_cast<long long>(count) * c->kv_heads > kMaxRows) return KCB_INVALID_VALUE;
    if (count == 0 || c->n_seqs == 0) return KCB_SUCCESS;
    const auto st = static_cast<cudaStream_t>(stream);
    ReadP R{*c, k_out, v_out, static_cast<long long>(q4_seq_bytes(c->kv_heads, c->head_dim, c->capacity)),
            static_cast<long long>(q4_param_offset(c->kv_heads, c->head_dim, c->capacity)), divisor(c->kv_heads), first, count};
    const dim3 grid(row_blocks(c, count), c->n_seqs);
    if (c->bits == KCB_CACHE_F16) kv_read_rows_kernel<16><<<grid, kRowThreads, 0, st>>>(R);
    else kv_read_rows_kernel<4><<<grid, kRowThreads, 0, st>>>(R);
    return launch_status();
}

size_t kcb_cache_evict_workspace_bytes(const kcb_kv_cache* c, int keep) {
    if (!c || c->n_seqs < 0 || c->kv_heads <= 0 || keep < 0 || keep >= c->capacity) return 0;
    return moves_offset(c) + static_cast<size_t>(c->n_seqs) * c->kv_heads * std::min(keep, c->capacity - keep) * sizeof(int2);
}

int kcb_cache_evict(const kcb_kv_cache* c, int keep, int recent, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int e = cache_ok(c); e != KCB_SUCCESS) return e;
    if (!c->n_keys || !c->next_pos || !c->positions || !c->weights || keep <= 0 || recent < 0 || recent > keep || !rows_apart(c))
        return KCB_INVALID_VALUE;
    if (keep >= c->capacity || c->n_seqs == 0) return KCB_SUCCESS;  // no sequence can hold more
    if (!workspace || workspace_bytes < kcb_cache_evict_workspace_bytes(c, keep)) return KCB_INVALID_VALUE;
    if (misaligned(workspace, 16)) return KCB_INVALID_POINTER;
    const auto st = static_cast<cudaStream_t>(stream);
    EvictP E{*c, keep, recent, std::min(keep, c->capacity - keep), static_cast<int*>(workspace),
             reinterpret_cast<int2*>(static_cast<uint8_t*>(workspace) + moves_offset(c)), static_cast<long long>(q4_seq_bytes(c->kv_heads, c->head_dim, c->capacity)),
             static_cast<long long>(q4_param_offset(c->kv_heads, c->head_dim, c->capacity))};
    static PerDeviceFlag raised;
    if (!raise_dynamic_smem(kv_select_kernel<1024>, kSelKeys * 4, raised)) return KCB_LAUNCH_FAILURE;
    const dim3 heads(c->kv_heads, c->n_seqs);
    const size_t smem = static_cast<size_t>(std::min(c->capacity, kSelKeys)) * 4;
    // Many short caches in small CTAs, of which an SM holds more (64 sequences of 8 heads: 576 slots 23.6 us, with 1024 threads 27.6; 2048
    // slots 69 and 75, 4096 slots 83 and 79); where every CTA has an SM the wider one is as fast or faster (4 sequences of 2048: 21 and 24).
    if (c->capacity <= 2048 && heads.x * heads.y > kSmCount) kv_select_kernel<256><<<heads, 256, smem, st>>>(E);
    else kv_select_kernel<1024><<<heads, 1024, smem, st>>>(E);
    if (const int e = launch_status(); e != KCB_SUCCESS) return e;
    constexpr int per_cta = kMoveWarps * kMoveRows;
    const dim3 grid(std::min((E.max_moves + per_cta - 1) / per_cta, 1024), c->kv_heads, c->n_seqs);
    return c->bits == KCB_CACHE_F16 ? launch_dependent(kv_move_kernel<16>, grid, 32 * kMoveWarps, 0, st, E)
                                    : launch_dependent(kv_move_kernel<4>, grid, 32 * kMoveWarps, 0, st, E);
}

size_t kcb_cache_attention_workspace_bytes(const kcb_kv_cache* c, const kcb_cache_attn* a) {
    if (attn_ok(c, a) != KCB_SUCCESS || a->n_tokens == 0 || c->n_seqs == 0) return 0;
    return attn_cut(c, a).bytes();
}

int kcb_cache_attention(const kcb_kv_cache* c, const kcb_cache_attn* a, const float* q, float* out, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int e = attn_ok(c, a); e != KCB_SUCCESS) return e;
    if (!q || !out) return KCB_INVALID_VALUE;
    if (misaligned(q, 16) || misaligned(out, 16)) return KCB_INVALID_POINTER;
    if (a->n_tokens == 0 || c->n_seqs == 0) return KCB_SUCCESS;
    if ((a->n_tokens > 1 && !a->out_token) || (a->heads > 1 && !a->out_head) || (c->n_seqs > 1 && !a->out_seq)) return KCB_INVALID_VALUE;  // rows on top of each other
    const AttnCut cut = attn_cut(c, a);
    const size_t need = cut.bytes();
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
    P.dim = c->head_dim, P.cap = c->capacity, P.n_seqs = c->n_seqs, P.n_tokens = a->n_tokens, P.heads = a->heads, P.kv_heads = c->kv_heads;
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
    ws += cut.ml_bytes + cut.o_bytes;
    P.final_ml = cut.final_bytes ? reinterpret_cast<float2*>(ws) : nullptr;
    P.scores = cut.score_bytes ? reinterpret_cast<float*>(ws) : nullptr;
    const bool general = a->softcap > 0.0f || a->max_bias > 0.0f || c->positions || a->q_doc || a->mask || ((a->q_pos || a->prefix) && cut.which != AttnKernel::tc);
    const auto st = static_cast<cudaStream_t>(stream);
    return attn_launch_bits(P, c->bits, c->head_dim, general, cut.which, st);
}

}  // extern "C"

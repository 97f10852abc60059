// Prompt attention over a KV cache on the 5th-generation tensor cores (tcgen05, TMEM): 128 query rows per CTA, head dimension 64 or
// 128.  Same mathematics and precision as kv_attention.cuh: queries and probabilities as hi + lo fp16 pairs, both multiplied; an fp16
// cache exact as it is; 4-bit values d code + m (a multiple of 2^-24, as every fp16 number is) as hi + lo pairs too, of whose four
// products with a query or probability the smallest, lo * lo (2^-22), is left out.
//
// Three warpgroups.
//   * Two softmax warpgroups, one query row per thread, take the 64-key tiles in turn; each has its own running maximum, sum and
//     output, joined at the end.  Per tile one thread of the warpgroup issues the score products (queries are the A operand, resident
//     in TMEM; keys from shared memory), every thread turns its row's 64 scores into probabilities and stores them, as hi and lo
//     halves, over the scores in TMEM, and one thread issues the value products.  While one warpgroup computes probabilities the
//     tensor core works for the other.
//   * A tile's output starts from zero in TMEM and is added to the thread's running output in registers, in fp32: no rescaling in
//     TMEM, and the length of the context never meets the truncation of the tensor cores' sums.  The read-back runs under the next
//     score products.
//   * One producer warpgroup brings key and value tiles into a ring of stages in the 128-byte-swizzled layout of the operands
//     (cp.async for fp16 rows, registers for 4-bit rows).  It copies rows in use only (zeros behind them) and looks for values
//     that are not finite, which would reach rows that do not see them as 0 * inf.  That is also why it is not a tensor copy.
// TMEM (512 columns at D = 128): queries hi | lo, 64 columns of scores / probabilities and D columns of output per warpgroup.
// Every wait is bounded: on expiry the CTA raises a flag that all roles poll, waits for its copies and products in flight, counts
// the event, frees its TMEM and returns.
#pragma once

#include "kv_attention.cuh"

namespace kcb {

static __device__ unsigned g_attn_timeouts = 0;

template <int D, int FMT>
struct TcCfg {
    static constexpr int KT = 64, kRows = 128, kThreads = 384;
    static constexpr int kPlane = KT * D * 2;                 // one fp16 tile: D / 64 atoms of 64 keys x 128 bytes
    static constexpr int kV = (FMT == 16 ? 1 : 2) * kPlane;   // keys (hi, lo), then values (hi, lo)
    static constexpr int kStage = 2 * kV;
    static constexpr int kStages = (FMT == 16 ? 6 : 3) * (D == 64 ? 2 : 1) > 8 ? 8 : (FMT == 16 ? 6 : 3) * (D == 64 ? 2 : 1);
    static constexpr int kDepth = FMT == 16 ? 3 : 0;          // tiles whose copies stay in flight behind the one being finished
    static constexpr int kMeta = kStages * kStage;            // per stage: position and document of 64 slots, 64 bits of slots with odd values
    static constexpr int kMetaBytes = 2 * KT * 4 + 16;
    static constexpr int kBars = kMeta + kStages * kMetaBytes;
    static constexpr int kTile0 = kBars + 256;                // bitmap of tiles
    static constexpr int kSmem = kTile0 + kDocBits / 8 + 1024;  // + room to align the base to 1024 bytes
    static constexpr uint32_t kQ = 0, kS = D, kO = D + 2 * KT;  // TMEM columns
    static constexpr int kRegsSoftmax = FMT == 16 ? 224 : 216, kRegsProducer = FMT == 16 ? 56 : 72, kRegsLaunch = 168;
    static_assert(2 * 128 * kRegsSoftmax + 128 * kRegsProducer <= kThreads * kRegsLaunch, "the softmax warpgroups take what the producers give up");
    static_assert(kO + 2 * D <= 512 && 128 * D * 4 + 2048 <= kStages * kStage && kSmem <= kMaxSmem, "TMEM columns; the exchange at the end reuses the ring");
};

__device__ __forceinline__ uint64_t tc_desc(uint32_t addr, uint32_t lbo) {  // 128-byte swizzle, 8-row groups 1024 bytes apart
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(lbo >> 4) << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
           (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
// D (TMEM, fp32) (+)= A (TMEM, fp16) B (shared memory, fp16)
__device__ __forceinline__ void tc_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0), "r"(0), "r"(0), "r"(0)
        : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_ld32(uint32_t addr, float (&v)[32]) {
    unsigned* r = reinterpret_cast<unsigned*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
// The loaded registers hold their data only behind this wait; passing them through it ties every later use to a point after it.
__device__ __forceinline__ void tc_ld_wait(float (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(v[i])::"memory");
}
__device__ __forceinline__ unsigned tc_ld1(uint32_t addr) {
    unsigned r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;" : "=r"(r) : "r"(addr) : "memory");
    return r;
}
__device__ __forceinline__ void tc_st16(uint32_t addr, const unsigned (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tc_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void bar_arrive(uint64_t* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory"); }
__device__ __forceinline__ void named_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ bool tc_wait(uint64_t* bar, uint32_t parity, volatile int* fail) {
    for (int i = 0; i < kMbarSpinLimit; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 255) == 255 && *fail) return false;
    }
    *fail = 1;
    return false;
}

// Capped scores: y = tanh(u) cap, u = y on entry.  The power series below 0.55 (see tanh_acc), elsewhere 1 - 2 / (e^2|u| + 1): there
// the difference costs one bit.  A warp whose scores are all small against the cap, as most are, takes the series alone.
__device__ __forceinline__ void cap_scores(float (&y)[2][32], float cap) {
    float big = 0.0f;
#pragma unroll
    for (int k = 0; k < 64; ++k) big = fmaxf(big, fabsf(y[k >> 5][k & 31]));
    const bool small = __all_sync(0xffffffffu, big < 0.55f);
#pragma unroll
    for (int k = 0; k < 64; ++k) {
        const float u = y[k >> 5][k & 31];
        float r = tanh_series(u);
        if (!small && fabsf(u) >= 0.55f) r = copysignf(1.0f - __fdividef(2.0f, ex2(2.0f * kLog2e * fabsf(u)) + 1.0f), u);
        y[k >> 5][k & 31] = r * cap;
    }
}

template <int D, int FMT, bool GEN>
__global__ void __launch_bounds__(384, 1) attn_tc_kernel(const __grid_constant__ AttnP P) {
    using C = TcCfg<D, FMT>;
    constexpr int KT = C::KT, NB = D / 32, CH = D / 8;
    extern __shared__ uint8_t sm_raw[];
    uint8_t* sm = sm_raw + ((1024u - (smem_u32(sm_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::kBars);  // [stage] tiles written
    uint64_t* empty = full + C::kStages;                          // [stage] tiles read by the products
    uint64_t* sfull = empty + C::kStages;                         // [warpgroup] scores complete
    uint64_t* ofull = sfull + 2;                                  // [warpgroup] outputs complete
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ofull + 2);
    volatile int* fail = reinterpret_cast<volatile int*>(ofull + 3);
    uint32_t* bits = reinterpret_cast<uint32_t*>(sm + C::kTile0);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wg = warp >> 2;
    const int rt = P.row_tiles - 1 - static_cast<int>(blockIdx.x) / P.nsplit, split = blockIdx.x % P.nsplit, kvh = blockIdx.y, s = blockIdx.z;
    const int row0 = rt * C::kRows;
    grid_dependents_may_launch();
    const int n = seq_keys(P, s);
    const int chunk = (n + P.nsplit * 64 - 1) / (P.nsplit * 64) * 64;
    const int begin = min(n, split * chunk);
    int end = min(n, begin + chunk);
    const int tok0 = row0 / P.group, tok1 = (min(P.rows, row0 + C::kRows) - 1) / P.group;
    const int prefix = GEN && P.prefix ? P.prefix[s] : 0;
    if (P.causal && !P.positions && !P.q_pos) end = max(begin, min(end, max(prefix, row_pos(P, s, n, tok1) + 1)));
    const int nt = (end - begin + KT - 1) / KT;
    const bool docs = GEN && P.q_doc != nullptr;

    if (tid == 0) {
        for (int i = 0; i < C::kStages; ++i) mbar_init(&full[i], 128), mbar_init(&empty[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&sfull[i], 1), mbar_init(&ofull[i], 1);
        *fail = 0;
        mbar_init_fence();
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const DocTiles<KT> doc_tiles{bits, nt};
    if (docs) doc_tiles.clear(tid, C::kThreads);
    tc_before_sync();
    __syncthreads();
    tc_after_sync();
    const uint32_t tmem = *tmem_slot;
    if (docs) doc_tiles.find(P, s, tok0, tok1, begin, end, warp, C::kThreads / 32, lane);
    auto next = [&](int i) { return docs ? doc_tiles.next(i) : i + 1; };  // the tile behind tile i that is wanted

    if (wg == 2) {
        // ---- producers ----------------------------------------------------------------------------------------------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsProducer));
        if (docs) __syncthreads();
        __syncthreads();  // (the queries)
        const int ptid = tid - 256;
        const bool hides = GEN || P.causal;
        auto swz = [&](int r, int ch) { return (ch >> 3) * (KT * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4); };
        auto copy = [&](int tile, int stage) {  // fp16: start the copies
            const uint32_t dst = smem_u32(sm) + stage * C::kStage;
            const int t0 = begin + tile * KT;
            const __half* kb = reinterpret_cast<const __half*>(P.k) + static_cast<size_t>(s) * P.k_seq + static_cast<size_t>(kvh) * P.k_head;
            const __half* vb = reinterpret_cast<const __half*>(P.v) + static_cast<size_t>(s) * P.v_seq + static_cast<size_t>(kvh) * P.v_head;
#pragma unroll
            for (int i = 0; i < KT * CH / 128; ++i) {
                const int x = i * 128 + ptid, r = x / CH, ch = x % CH;
                const bool ok = t0 + r < end;
                const size_t t = ok ? t0 + r : 0;
                cp16(dst + swz(r, ch), kb + t * P.k_row + ch * 8, ok);
                cp16(dst + C::kV + swz(r, ch), vb + t * P.v_row + ch * 8, ok);
            }
        };
        auto finish = [&](int tile, int stage) {
            const int t0 = begin + tile * KT;
            uint8_t* st = sm + stage * C::kStage;
            int* meta = reinterpret_cast<int*>(sm + C::kMeta + stage * C::kMetaBytes);
            if (GEN && ptid < KT) {
                const KeyInfo key = key_info(P, s, kvh, t0 + ptid, end);
                meta[ptid] = key.pos, meta[KT + ptid] = key.doc;
            }
            if (FMT == 16) {
                if (hides) {
                    unsigned* odd = reinterpret_cast<unsigned*>(meta + 2 * KT);
                    bool any = false;
#pragma unroll
                    for (int i = 0; i < KT * CH / 128; ++i) {  // the chunks this thread copied itself
                        const int x = i * 128 + ptid;
                        any = any || not_finite(*reinterpret_cast<const uint4*>(st + C::kV + swz(x / CH, x % CH)));
                    }
                    if (any) {
#pragma unroll 1
                        for (int i = 0; i < KT * CH / 128; ++i) {
                            const int x = i * 128 + ptid;
                            uint8_t* at = st + C::kV + swz(x / CH, x % CH);
                            if (!not_finite(*reinterpret_cast<const uint4*>(at))) continue;
                            zero_not_finite(at);
                            atomicOr(&odd[(x / CH) >> 5], 1u << ((x / CH) & 31));
                        }
                    }
                }
            } else {
                // 4 bits: a thread takes a quarter of the key row's and of the value row's groups; two threads to a row
                const uint8_t* kb = P.k + static_cast<size_t>(s) * P.seq_bytes;
                const uint8_t* vb = P.v + static_cast<size_t>(s) * P.seq_bytes;
#pragma unroll
                for (int plane = 0; plane < 2; ++plane) {
                    const int r = ptid >> 1, half = ptid & 1;
                    const bool ok = t0 + r < end;
                    const size_t at = static_cast<size_t>(kvh) * P.cap + (ok ? t0 + r : 0);
                    const uint8_t* rowp = (plane ? vb : kb) + at * (D / 2);
                    const unsigned* par = reinterpret_cast<const unsigned*>((plane ? vb : kb) + P.par_off + at * (4 * NB));
                    uint8_t* hi_t = st + (plane ? C::kV : 0);
                    float d[NB], m[NB];
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        unsigned w = ok ? par[b] : 0u;
                        if ((w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u) w = 0u;  // (a hidden slot's scales may be anything)
                        d[b] = half_bits_to_float(w & 0xFFFFu), m[b] = half_bits_to_float(w >> 16);
                    }
                    // 16-byte pieces of 8 channels: piece 4 b + c of a row; a key row's group c holds the pieces (b, c)
                    // whole, a value row's groups 2 c and 2 c + 1 half of each
#pragma unroll
                    for (int cc = 0; cc < 2; ++cc) {
                        const int c = half * 2 + cc;
                        unsigned v[NB], w[NB];  // the piece's 4 NB bytes, and 8 codes per block
                        if (ok) {
                            if constexpr (NB == 4) {
                                const uint4 t = *reinterpret_cast<const uint4*>(rowp + c * 16);
                                v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
                            } else {
                                const uint2 t = *reinterpret_cast<const uint2*>(rowp + c * 8);
                                v[0] = t.x, v[1] = t.y;
                            }
                        } else {
#pragma unroll
                            for (int b = 0; b < NB; ++b) v[b] = 0u;
                        }
#pragma unroll
                        for (int b = 0; b < NB; ++b) w[b] = plane == 0 ? v[b] : __byte_perm(v[b / 2], v[NB / 2 + b / 2], b & 1 ? 0x7632 : 0x5410);
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            uint4 hi, lo;
                            unsigned* hp = &hi.x;
                            unsigned* lp = &lo.x;
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const float x = fmaf(d[b], static_cast<float>(w[b] >> (8 * k) & 15u), m[b]), y = fmaf(d[b], static_cast<float>(w[b] >> (8 * k + 4) & 15u), m[b]);
                                const __half2 h = __floats2half2_rn(fminf(x, 65504.0f), fminf(y, 65504.0f));  // the rest of a larger value goes to lo
                                const float2 f = __half22float2(h);
                                hp[k] = h2_bits(h), lp[k] = h2_bits(__floats2half2_rn(x - f.x, y - f.y));
                            }
                            const int o = swz(r, 4 * b + c);
                            *reinterpret_cast<uint4*>(hi_t + o) = hi;
                            *reinterpret_cast<uint4*>(hi_t + C::kPlane + o) = lo;
                        }
                    }
                }
            }
            fence_async_shared();
            bar_arrive(&full[stage]);
        };
        // tile number i (in order of use) goes to stage i % kStages
        int put = 0, done = 0, tile = next(-1), ready = tile;
        while (done < put || tile < nt) {
            if (tile < nt && put - done <= C::kDepth) {
                const int stage = put % C::kStages;
                if (put >= C::kStages) tc_wait(&empty[stage], (put / C::kStages - 1) & 1, fail);
                if (ptid < 2) reinterpret_cast<unsigned*>(sm + C::kMeta + stage * C::kMetaBytes + 2 * KT * 4)[ptid] = 0u;
                named_sync(3, 128);  // the odd-value bits are cleared before anybody sets one
                if (FMT == 16) copy(tile, stage);
                cp_commit();
                tile = next(tile), ++put;
                if (put - done <= C::kDepth && tile < nt) continue;
            }
            if (tile < nt) cp_wait<C::kDepth>();
            else cp_wait<0>();
            finish(ready, done % C::kStages);
            ready = next(ready), ++done;
        }
        cp_wait<0>();
    } else {
        // ---- softmax -------------------------------------------------------------------------------------------------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegsSoftmax));
        if (docs) __syncthreads();
        const int r = tid & 127, row = row0 + r;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + C::kS + wg * KT, to = tmem + C::kO + wg * D;
        const bool valid = row < P.rows;
        float ysc;
        {  // the row's query: warpgroup 0 stores the hi halves, warpgroup 1 the lo halves
            const int token = (valid ? row : 0) / P.group, head = kvh * P.group + (valid ? row : 0) % P.group;
            const float4* qp = reinterpret_cast<const float4*>(P.q + static_cast<size_t>(s) * P.q_seq + static_cast<size_t>(token) * P.q_token + static_cast<size_t>(head) * P.q_head);
            float amax = 0.0f;
#pragma unroll 8
            for (int i = 0; i < D / 4; ++i) {
                const float4 f = valid ? qp[i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                amax = fmaxf(fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y))), fmaxf(fabsf(f.z), fabsf(f.w)));
            }
            float up, down;
            row_scale(amax, up, down);
            ysc = P.sc * down;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                unsigned out[16];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float4 f = valid ? qp[i * 8 + k] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    unsigned h0, l0, h1, l1;
                    split2(f.x * up, f.y * up, h0, l0);
                    split2(f.z * up, f.w * up, h1, l1);
                    out[2 * k] = wg ? l0 : h0, out[2 * k + 1] = wg ? l1 : h1;
                }
                tc_st16(tmem + lanes + C::kQ + wg * (D / 2) + i * 16, out);
            }
            tc_st_wait();
        }
        tc_before_sync();
        __syncthreads();
        tc_after_sync();

        const uint32_t base = smem_u32(sm);
        constexpr uint32_t kIdescS = (1u << 4) | (static_cast<uint32_t>(KT >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24);
        constexpr uint32_t kIdescO = (1u << 4) | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24);
        auto issue_scores = [&](int i) {  // tile number i: scores = (hi + lo) keys^T
            const uint32_t st = base + (i % C::kStages) * C::kStage;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                const uint32_t at = st + (k >> 2) * (KT * 128) + (k & 3) * 32;
                const uint32_t qh = tmem + C::kQ + k * 8, ql = qh + D / 2;
                tc_mma(ts, qh, tc_desc(at, 0), kIdescS, k > 0);
                tc_mma(ts, ql, tc_desc(at, 0), kIdescS, 1);
                if (FMT != 16) tc_mma(ts, qh, tc_desc(at + C::kPlane, 0), kIdescS, 1);
            }
            tc_commit(&sfull[wg]);
        };
        auto issue_values = [&](int i) {
            const uint32_t st = base + (i % C::kStages) * C::kStage + C::kV;
#pragma unroll
            for (int k = 0; k < KT / 16; ++k) {
                const uint32_t at = st + k * 2048;
                const uint32_t ph = ts + k * 8, pl = ph + KT / 2;
                tc_mma(to, ph, tc_desc(at, KT * 128), kIdescO, k > 0);
                tc_mma(to, pl, tc_desc(at, KT * 128), kIdescO, 1);
                if (FMT != 16) tc_mma(to, ph, tc_desc(at + C::kPlane, KT * 128), kIdescO, 1);
            }
            tc_commit(&ofull[wg]);
            tc_commit(&empty[i % C::kStages]);
        };
        RowInfo ri;
        int limit = n;
        if (GEN) ri = row_info(P, s, kvh, n, row);
        else if (P.causal) limit = valid ? min(n, row_pos(P, s, n, row / P.group) + 1) : 0;
        limit = min(limit, end);

        float o[D], m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int i = 0; i < D; ++i) o[i] = 0.0f;
        const bool elected = (tid & 127) == 0;
        // tile numbers wg, wg + 2, ...: `tile` is the one of number i
        int tile = next(-1);
        if (wg) tile = next(tile);
        if (tile < nt && elected) {
            if (tc_wait(&full[wg], 0, fail)) issue_scores(wg);
        }
        // (after an expired wait the loops run on, without products, so that every barrier finds its threads)
        uint32_t round = 0;
        for (int i = wg; tile < nt; i += 2, ++round) {
            const int stage = i % C::kStages;
            tc_wait(&sfull[wg], round & 1, fail);
            tc_wait(&full[stage], (i / C::kStages) & 1, fail);  // (long complete: makes what the producers wrote beside the tiles visible)
            __syncwarp();
            tc_after_sync();
            float y[2][32];
            tc_ld32(ts + lanes, y[0]);
            tc_ld32(ts + lanes + 32, y[1]);
            tc_ld_wait(y[0]);
            tc_ld_wait(y[1]);
            const int t0 = begin + tile * KT;
            if (!GEN) {
#pragma unroll
                for (int k = 0; k < KT; ++k) y[k >> 5][k & 31] *= ysc;
                if (!__all_sync(0xffffffffu, t0 + KT <= limit)) {
#pragma unroll
                    for (int k = 0; k < KT; ++k)
                        if (t0 + k >= limit) y[k >> 5][k & 31] = -INFINITY;
                }
            } else {
                const int* meta = reinterpret_cast<const int*>(sm + C::kMeta + stage * C::kMetaBytes);
#pragma unroll
                for (int k = 0; k < KT; ++k) y[k >> 5][k & 31] *= ysc;
                if (P.cap_out != 0.0f) cap_scores(y, P.cap_out);
                if (P.mask) {
                    const unsigned short* mp = ri.mask + t0;
                    const bool wide = ((reinterpret_cast<uintptr_t>(mp) & 15) == 0) && t0 + KT <= end;
#pragma unroll
                    for (int k8 = 0; k8 < KT / 8; ++k8) {
                        unsigned short h[8];
                        if (wide) {
                            *reinterpret_cast<uint4*>(h) = *reinterpret_cast<const uint4*>(mp + 8 * k8);
                        } else {
#pragma unroll
                            for (int k = 0; k < 8; ++k) h[k] = t0 + 8 * k8 + k < end ? mp[8 * k8 + k] : 0xFC00u;
                        }
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            float& v = y[k8 >> 2][(k8 & 3) * 8 + k];
                            v = h[k] == 0xFC00u ? -INFINITY : fmaf(ri.slope, half_bits_to_float(h[k]), v);
                        }
                    }
                } else if (P.bias_step != 0.0f) {
                    const float qp = static_cast<float>(ri.pos);
#pragma unroll
                    for (int k = 0; k < KT; ++k) y[k >> 5][k & 31] -= ri.slope * fabsf(qp - static_cast<float>(meta[k]));
                }
                unsigned see[2] = {valid ? 0xffffffffu : 0u, valid ? 0xffffffffu : 0u};
                if (t0 + KT > end) {
                    const int in = end - t0;  // 1 .. 63
                    see[0] &= in >= 32 ? 0xffffffffu : (1u << in) - 1u;
                    see[1] &= in <= 32 ? 0u : (1u << (in - 32)) - 1u;
                }
                if (P.causal && (P.positions || P.q_pos || !__all_sync(0xffffffffu, t0 + KT - 1 <= ri.pos || t0 + KT <= prefix))) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        unsigned w = 0;
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            const int kp = meta[h * 32 + k];
                            w |= static_cast<unsigned>(kp <= ri.pos || kp < prefix) << k;
                        }
                        see[h] &= w;
                    }
                }
                if (docs) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        unsigned w = 0;
#pragma unroll
                        for (int k = 0; k < 32; ++k) w |= static_cast<unsigned>(meta[KT + h * 32 + k] == ri.doc) << k;
                        see[h] &= w;
                    }
                }
                if (!__all_sync(0xffffffffu, (see[0] & see[1]) == 0xffffffffu)) {
#pragma unroll
                    for (int k = 0; k < KT; ++k)
                        if (!(see[k >> 5] >> (k & 31) & 1u)) y[k >> 5][k & 31] = -INFINITY;
                }
            }
            float mx = m;
#pragma unroll
            for (int k = 0; k < KT; k += 2) mx = fmaxf(mx, fmaxf(y[k >> 5][k & 31], y[k >> 5][(k & 31) + 1]));
            float al = mx > m ? ex2(m - mx) : 1.0f;
            m = mx;
            const float ref = m == -INFINITY ? 0.0f : m - kPShift;
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                unsigned hi[16], lo[16];
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    y[h][k] = ex2(y[h][k] - ref), y[h][k + 1] = ex2(y[h][k + 1] - ref);
                    sum[k & 2] += y[h][k], sum[(k & 2) + 1] += y[h][k + 1];
                    split2(y[h][k], y[h][k + 1], hi[k / 2], lo[k / 2]);
                }
                tc_st16(ts + lanes + h * 16, hi);
                tc_st16(ts + lanes + KT / 2 + h * 16, lo);
            }
            l = fmaf(l, al, (sum[0] + sum[1]) + (sum[2] + sum[3]));
            tc_st_wait();
            if (FMT == 16) {  // rare: values of this tile that are not finite go to the rows that see them one by one
                const unsigned* odd = reinterpret_cast<const unsigned*>(sm + C::kMeta + stage * C::kMetaBytes + 2 * KT * 4);
                const unsigned w0 = odd[0], w1 = odd[1];
                if (w0 | w1) {
                    al = fmaxf(al, 1e-30f);  // an infinity added now stays one when the output is rescaled below
#pragma unroll 1
                    for (int k = 0; k < KT; ++k) {
                        if (!((k < 32 ? w0 >> k : w1 >> (k - 32)) & 1u)) continue;
                        const unsigned* vp = reinterpret_cast<const unsigned*>(reinterpret_cast<const __half*>(P.v) + static_cast<size_t>(s) * P.v_seq +
                                                                               static_cast<size_t>(kvh) * P.v_head + static_cast<size_t>(t0 + k) * P.v_row);
                        const unsigned ph = tc_ld1(ts + lanes + (k >> 1)) >> (16 * (k & 1)), pl = tc_ld1(ts + lanes + KT / 2 + (k >> 1)) >> (16 * (k & 1));
                        const float p = half_bits_to_float(ph & 0xFFFFu) + half_bits_to_float(pl & 0xFFFFu);
                        if (p != 0.0f)
#pragma unroll
                            for (int ch = 0; ch < D / 2; ++ch) add_not_finite(o[2 * ch], o[2 * ch + 1], p, vp[ch]);
                        __syncwarp();
                    }
                }
            }
            tc_before_sync();
            named_sync(1 + wg, 128);
            const int after = next(next(tile));
            if (elected) {
                tc_after_sync();
                if (!*fail) issue_values(i);
                if (after < nt) tc_wait(&full[(i + 2) % C::kStages], ((i + 2) / C::kStages) & 1, fail);
            }
            tc_wait(&ofull[wg], round & 1, fail);
            tc_after_sync();
            if (elected && after < nt && !*fail) issue_scores(i + 2);
            __syncwarp();
#pragma unroll
            for (int h = 0; h < D / 32; ++h) {
                float v[32];
                tc_ld32(to + lanes + h * 32, v);
                tc_ld_wait(v);
#pragma unroll
                for (int k = 0; k < 32; ++k) o[h * 32 + k] = fmaf(o[h * 32 + k], al, v[k]);
            }
            tc_before_sync();  // the next value products overwrite what was read: ordered by the warpgroup's barrier above
            tile = after;
        }
        // ---- the two warpgroups' sums joined: each finishes half of the channels ----------------------------------------------
        named_sync(4, 256);
        float* ex = reinterpret_cast<float*>(sm);                          // [D / 2][128] of either half
        float2* exml = reinterpret_cast<float2*>(sm + 128 * D * 4);        // [2][128]
        exml[wg * 128 + r] = make_float2(m, l);
#pragma unroll
        for (int i = 0; i < D / 2; ++i) ex[((wg ? 0 : D / 2) + i) * 128 + r] = wg ? o[i] : o[D / 2 + i];
        named_sync(4, 256);
        const float2 other = exml[(1 - wg) * 128 + r];
        const float M = fmaxf(m, other.x);
        const float f0 = l != 0.0f ? ex2(m - M) : 0.0f, f1 = other.y != 0.0f ? ex2(other.x - M) : 0.0f;
        const float L = (l != 0.0f ? l * f0 : 0.0f) + (other.y != 0.0f ? other.y * f1 : 0.0f);
        const size_t part = ((static_cast<size_t>(s) * P.kv_heads + kvh) * P.nsplit + split) * P.rows + row;
        if (valid) {
            float* dst;
            float f = 1.0f;
            if (P.nsplit > 1) {
                dst = P.part_o + part * D;
            } else {
                f = L > 0.0f || L != L ? 1.0f / L : 0.0f;
                const int token = row / P.group, head = kvh * P.group + row % P.group;
                dst = P.out + static_cast<size_t>(s) * P.o_seq + static_cast<size_t>(token) * P.o_token + static_cast<size_t>(head) * P.o_head;
            }
            const float a = f0 * f, b = f1 * f;
#pragma unroll
            for (int i = 0; i < D / 2; i += 4) {
                float4 v;
                float* vp = &v.x;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float mine = wg ? o[D / 2 + i + k] : o[i + k];
                    vp[k] = fmaf(mine, a, ex[(wg * (D / 2) + i + k) * 128 + r] * b);
                }
                *reinterpret_cast<float4*>(dst + wg * (D / 2) + i) = v;
            }
            if (wg == 0) {
                if (P.nsplit > 1) P.part_ml[part] = make_float2(M, L);
                else if (P.final_ml) P.final_ml[(static_cast<size_t>(s) * P.kv_heads + kvh) * P.rows + row] = make_float2(M, L);
            }
        }
    }
    // ---- teardown: nothing of this CTA is in flight when its TMEM goes back ---------------------------------------------------
    if (*fail && wg < 2) {  // products still running have a bounded time to end
        for (int i = 0; i < (1 << 16); ++i) __nanosleep(20);
        if (tid == 0) atomicAdd(&g_attn_timeouts, 1u);
    }
    tc_before_sync();
    __syncthreads();
    tc_after_sync();
    if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

template <int D, int FMT>
int attn_launch_tc(const AttnP& P, bool general, cudaStream_t st) {
    if constexpr (D == 64 || D == 128) {
        constexpr int smem = TcCfg<D, FMT>::kSmem;
        static PerDeviceFlag raised[2];
        const dim3 grid(P.row_tiles * P.nsplit, P.kv_heads, P.n_seqs);
        if (general) {
            if (!raise_dynamic_smem(attn_tc_kernel<D, FMT, true>, smem, raised[0])) return KCB_LAUNCH_FAILURE;
            attn_tc_kernel<D, FMT, true><<<grid, 384, smem, st>>>(P);
        } else {
            if (!raise_dynamic_smem(attn_tc_kernel<D, FMT, false>, smem, raised[1])) return KCB_LAUNCH_FAILURE;
            attn_tc_kernel<D, FMT, false><<<grid, 384, smem, st>>>(P);
        }
        return launch_status();
    }
    return KCB_UNSUPPORTED_OPERATION;
}
// Waits of this translation unit's kernels that expired since load; synchronous.
inline unsigned attn_timeouts_here() {
    unsigned v = 0;
    return cudaMemcpyFromSymbol(&v, g_attn_timeouts, sizeof v) == cudaSuccess ? v : 0u;
}

}  // namespace kcb

// Prompt attention over a KV cache on the 5th-generation tensor cores (tcgen05, TMEM): 128 query rows per CTA, head dimension 64 or
// 128 (fp16 also 32 and 96, filled up with zeros).  Same mathematics and precision as kv_attention.cuh: queries and probabilities as hi + lo fp16 pairs, both multiplied; an fp16
// cache exact as it is; 4-bit values d code + m (a multiple of 2^-24, as every fp16 number is) as hi + lo pairs too, of whose four
// products with a query or probability the smallest, lo * lo (2^-22), is left out.
//
// Roles.
//   * Two softmax warpgroups, one query row per thread in each: a tile of keys is cut into halves, and each warpgroup has its half of
//     every tile's scores.  A thread reads its row's scores from TMEM, exchanges their maximum with the thread that has the other half
//     of the row, turns them into probabilities and stores those, as hi and lo halves, to TMEM, the A operand of the value products.
//   * The rest: one warp issues all products -- scores of the next tile as soon as both warpgroups have read this one's, so that they
//     run under the softmax -- and the others bring keys and values into rings of stages in the 128-byte-swizzled layout of the
//     operands: fp16 rows by tensor copies that one thread issues, 4-bit rows unpacked through registers.
//   * A tile's output starts from zero in TMEM and is added to running outputs in registers, in fp32, half of the channels by either
//     warpgroup: no rescaling in TMEM, and the length of the context never meets the tensor cores' sums, which truncate (each product
//     of K = 16 can cost its sum an ulp towards zero).
// TMEM (512 columns at D = 128, fp16): 128 scores, two buffers of 128 probabilities (hi and lo, two to a column), 128 outputs.
// Values that are not finite would reach rows that do not see them as 0 * inf, and so would what lies behind the rows in use, which
// a tensor copy brings along.  Looking for such values costs a third of the kernel's time, so the first pass does not: where an output
// is not finite at its end, the CTA takes a second pass that does, clears them from the tiles, and gives them to the rows that see
// them one by one.  (4-bit rows need none: the unpacking turns scales that are not finite into zeros.)
// Bounded by the issue slots of the softmax warpgroups and, at two products for one, by the tensor pipe.  4096 tokens, 32 heads over 8,
// D = 128: fp16 causal 270 us, all slots 450 us = 610 TFLOP/s (twice that in products), with a cap 416; 4 bits causal 520 us (unpacking
// and three products for one).
// Every wait is bounded: on expiry the CTA raises a flag that all roles poll, runs on without products, waits for its copies and
// products in flight, counts the event, frees its TMEM and returns.
#pragma once

#include "kv_attention.cuh"

#include <cuda.h>  // CUtensorMap and its enums; the encoder itself is looked up through the runtime (no libcuda link)

namespace kcb {

static __device__ unsigned g_attn_timeouts = 0;

template <int D, int FMT>
struct TcCfg {
    static constexpr int HK = FMT == 16 ? 64 : 32;             // keys of a tile per softmax warpgroup
    static constexpr int KT = 2 * HK, kRows = 128;
    // fp16: three producer warps and the products' warp make the third warpgroup; 4 bits: two producer warpgroups, and one that holds
    // the products' warp (and three idle ones)
    static constexpr int kProducers = FMT == 16 ? 96 : 256, kThreads = FMT == 16 ? 384 : 640, kMmaWarp = FMT == 16 ? 11 : 16;
    static constexpr int kPlane = KT * D * 2;                  // one fp16 tile: D / 64 atoms of KT keys x 128 bytes
    static constexpr int kSlot = (FMT == 16 ? 1 : 2) * kPlane; // keys or values of a tile (4 bits: hi, lo)
    static constexpr int kStages = kSlot > 16384 ? 2 : 4;      // of keys, and of values
    static constexpr int kQHalf = kRows * D * 2;               // hi, then lo queries
    static constexpr int kOffK = 2 * kQHalf, kOffV = kOffK + kStages * kSlot;
    static constexpr int kMeta = kOffV + kStages * kSlot;      // per stage: KT positions, KT documents, bits of odd slots
    static constexpr int kMetaBytes = 2 * KT * 4 + 16;
    static constexpr int kMax = kMeta + kStages * kMetaBytes;  // maxima exchanged: [2][warpgroup][row]
    static constexpr int kBars = kMax + 2 * 2 * kRows * 4;
    static constexpr int kTile0 = kBars + 256;                 // bitmap of tiles
    static constexpr int kSmem = kTile0 + kDocBits / 8 + 1024; // + room to align the base to 1024 bytes
    static constexpr uint32_t kS = 0, kP = KT, kO = 3 * KT;    // TMEM columns: scores, two buffers of probabilities, outputs
    // registers per thread: what a launch of kThreads gets (checked when the kernel is first launched: with fewer, the softmax
    // warpgroups would wait for ever for registers that nobody gives up), and after the hand-over
    static constexpr int kRegsLaunch = FMT == 16 ? 168 : 96, kRegsSoftmax = FMT == 16 ? 224 : 152, kRegsProducer = FMT == 16 ? 56 : 64, kRegsMma = 40;
    static_assert(2 * 128 * kRegsSoftmax + (FMT == 16 ? 128 * kRegsProducer : 256 * kRegsProducer + 128 * kRegsMma) <= kThreads * kRegsLaunch,
                  "the softmax warpgroups take what the others give up");
    static_assert(kO + D <= 512 && kMetaBytes % 16 == 0 && kSmem <= kMaxSmem && kSmem > kMaxSmem / 2, "TMEM columns; one CTA per SM");
};

__device__ __forceinline__ uint64_t tc_desc(uint32_t addr, uint32_t lbo) {  // 128-byte swizzle, 8-row groups 1024 bytes apart
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(lbo >> 4) << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
           (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
// D (TMEM, fp32) (+)= A B, fp16: A in shared memory or in TMEM, B in shared memory
// The whole warp comes here, so that addresses and descriptors live in uniform registers; one elected lane issues (a branch to a
// single lane instead made each product take 155 cycles to issue, against 64 to compute).
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tc_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
        : "memory");
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
__device__ __forceinline__ void tc_st16(uint32_t addr, const unsigned* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tc_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void bar_arrive(uint64_t* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory"); }
// Tiled 4-D tensor copy global -> this CTA's shared memory (no multicast); completion counted on `bar`.
__device__ __forceinline__ void tma_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void named_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ bool tc_wait(uint64_t* bar, uint32_t parity, volatile int* fail) {
    for (int i = 0; i < kMbarSpinLimit; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 255) == 255 && *fail) return false;
    }
    *fail = 1;
    return false;
}

// One answer for the whole warp.
__device__ __forceinline__ bool warp_failed(volatile int* fail) { return __any_sync(0xffffffffu, *fail != 0); }
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Capped scores: y = tanh(y c), c positive; the cap itself is multiplied later.  A power series for |u| < 0.3 (to u^9: 5e-8) or
// 0.55 (to u^15, see tanh_series), elsewhere 1 - 2 / (e^2|u| + 1): there the difference costs one bit.  A warp takes the shortest
// that holds for all its scores, most of which are small against the cap.
template <int H>
__device__ __forceinline__ void cap_scores(float (&y)[H][32], float c) {
    float hi = y[0][0], lo = y[0][0];
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int k = 0; k < 32; k += 2) hi = max3(hi, y[h][k], y[h][k + 1]), lo = -max3(-lo, -y[h][k], -y[h][k + 1]);
    const float big = fmaxf(hi, -lo) * c;
    const bool tiny = __all_sync(0xffffffffu, big < 0.3f), small = __all_sync(0xffffffffu, big < 0.55f);
    if (tiny) {
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
                const float2 u = mul2(make_float2(y[h][k], y[h][k + 1]), both(c)), w = mul2(u, u);
                float2 r = fma2(both(2.1869488e-2f), w, both(-5.3968254e-2f));
                r = fma2(r, w, both(1.3333333e-1f));
                r = fma2(r, w, both(-3.3333333e-1f));
                r = fma2(mul2(u, w), r, u);
                y[h][k] = r.x, y[h][k + 1] = r.y;
            }
        return;
    }
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int k = 0; k < 32; ++k) {
            const float u = y[h][k] * c;
            float r = tanh_series(u);
            if (!small && fabsf(u) >= 0.55f) r = copysignf(1.0f - __fdividef(2.0f, ex2(2.0f * kLog2e * fabsf(u)) + 1.0f), u);
            y[h][k] = r;
        }
}

template <int D, int FMT, bool GEN>
__global__ void __launch_bounds__(TcCfg<D, FMT>::kThreads, 1)
    attn_tc_kernel(const __grid_constant__ AttnP P, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
    using C = TcCfg<D, FMT>;
    constexpr int HK = C::HK, KT = C::KT, NB = D / 32, CH = D / 8;
    extern __shared__ uint8_t sm_raw[];
    uint8_t* sm = sm_raw + ((1024u - (smem_u32(sm_raw) & 1023u)) & 1023u);
    uint64_t* kfull = reinterpret_cast<uint64_t*>(sm + C::kBars);  // [stage] keys written
    uint64_t* kempty = kfull + C::kStages;                         // [stage] keys read by the products
    uint64_t* vfull = kempty + C::kStages;                         // [stage] values (and what stands beside them) written
    uint64_t* vempty = vfull + C::kStages;
    uint64_t* varrived = vempty + C::kStages;                      // [stage] fp16: values copied (the second pass waits for vfull, behind the search)
    uint64_t* mfull = varrived + C::kStages;                       // [stage] fp16: positions and documents written
    uint64_t* sfull = mfull + C::kStages;                          // scores of a tile complete
    uint64_t* sread = sfull + 1;                                   // ... and read by both warpgroups
    uint64_t* mxfull = sread + 1;                                  // a tile's maxima written
    uint64_t* pfull = mxfull + 1;                                  // probabilities stored, last output read
    uint64_t* ofull = pfull + 1;                                   // output of a tile complete
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ofull + 1);
    volatile int* fail = reinterpret_cast<volatile int*>(ofull + 2);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wg = warp >> 2;
    const int rt = P.row_tiles - 1 - static_cast<int>(blockIdx.x) / P.nsplit, split = blockIdx.x % P.nsplit, kvh = blockIdx.y, s = blockIdx.z;
    const int row0 = rt * C::kRows;
    grid_dependents_may_launch();
    const int n = seq_keys(P, s);
    const int chunk = (n + P.nsplit * 64 - 1) / (P.nsplit * 64) * 64;
    const int begin = min(n, split * chunk);
    int end = min(n, begin + chunk);
    const int tok0 = row0 / P.group, tok1 = (min(P.rows, row0 + C::kRows) - 1) / P.group;
    const int prefix = P.prefix ? P.prefix[s] : 0;
    if (P.causal && !P.positions && !P.q_pos) end = max(begin, causal_limit(row_pos(P, s, n, tok1), prefix, end));
    const int nt = (end - begin + KT - 1) / KT;
    const bool docs = GEN && P.q_doc != nullptr;

    if (tid == 0) {
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(&kfull[i], FMT == 16 ? 1 : C::kProducers), mbar_init(&kempty[i], 1), mbar_init(&vfull[i], C::kProducers), mbar_init(&vempty[i], 1);
            mbar_init(&varrived[i], 1), mbar_init(&mfull[i], 64);
        }
        mbar_init(sfull, 1), mbar_init(sread, 256), mbar_init(mxfull, 256), mbar_init(pfull, 256), mbar_init(ofull, 1);
        *fail = 0;
        mbar_init_fence();
    }
    if (warp == C::kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const DocTiles<KT> doc_tiles{reinterpret_cast<uint32_t*>(sm + C::kTile0), nt};
    if (docs) {
        doc_tiles.clear(tid, C::kThreads);
        __syncthreads();
        doc_tiles.find(P, s, tok0, tok1, begin, end, warp, C::kThreads / 32, lane);
    }
    auto next = [&](int i) { return docs ? doc_tiles.next(i) : i + 1; };  // the tile behind tile i that is wanted
    auto swz = [&](int rows, int r, int ch) { return (ch >> 3) * (rows * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4); };

    tc_before_sync();
    __syncthreads();
    tc_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    // (after an expired wait every loop below runs on, without products, so that every barrier finds its arrivals)

    if (wg >= 2) {
        if (FMT == 16 || wg < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsProducer));
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsMma));
        if (warp == C::kMmaWarp) {
            // ---- products ----------------------------------------------------------------------------------------------------
            int i = 0;  // tiles so far, over both passes: stages and parities go by it
            for (bool careful = false;; careful = true) {
                const int i0 = i;
                {
                    const uint32_t base = smem_u32(sm);
                    constexpr uint32_t kIdescS = (1u << 4) | (static_cast<uint32_t>(KT >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24);
                    constexpr uint32_t kIdescO = (1u << 4) | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24);
                    uint64_t* vready = FMT == 16 && !careful ? varrived : vfull;
                    auto scores = [&](int j) {  // (hi + lo) keys^T, both halves of the tile
                        const int st = j % C::kStages;
                        tc_wait(&kfull[st], (j / C::kStages) & 1, fail);
                        if (j == 0) named_sync(5, 288);  // the queries are there
                        __syncwarp();
                        tc_after_sync();
                        if (warp_failed(fail)) return;
                        const uint32_t kb = base + C::kOffK + st * C::kSlot;
#pragma unroll
                        for (int k = 0; k < D / 16; ++k) {
                            const uint64_t qh = tc_desc(base + (k >> 2) * (C::kRows * 128) + (k & 3) * 32, 0), ql = qh + (C::kQHalf >> 4);
                            const uint64_t kd = tc_desc(kb + (k >> 2) * (KT * 128) + (k & 3) * 32, 0);
                            tc_mma_ss(tmem + C::kS, qh, kd, kIdescS, k > 0);
                            tc_mma_ss(tmem + C::kS, ql, kd, kIdescS, 1);
                            if (FMT != 16) tc_mma_ss(tmem + C::kS, qh, kd + (C::kPlane >> 4), kIdescS, 1);
                        }
                        tc_commit(sfull);
                        tc_commit(&kempty[st]);
                    };
                    int tile = next(-1);
                    if (tile < nt) scores(i);
                    else if (!careful) named_sync(5, 288);
                    while (tile < nt) {
                        tile = next(tile);
                        tc_wait(sread, i & 1, fail);
                        if (tile < nt) scores(i + 1);
                        const int st = i % C::kStages;
                        const uint32_t vb = base + C::kOffV + st * C::kSlot;
                        tc_wait(&vready[st], ((i - (careful ? i0 : 0)) / C::kStages) & 1, fail);  // (vfull completes in the second pass alone)
                        tc_wait(pfull, i & 1, fail);
                        __syncwarp();
                        tc_after_sync();
                        if (!warp_failed(fail)) {
#pragma unroll
                            for (int k = 0; k < KT / 16; ++k) {
                                const uint32_t ph = tmem + C::kP + (i & 1) * KT + k * 8, pl = ph + KT / 2;
                                const uint64_t vd = tc_desc(vb + k * 2048, KT * 128);
                                tc_mma(tmem + C::kO, ph, vd, kIdescO, k > 0);
                                tc_mma(tmem + C::kO, pl, vd, kIdescO, 1);
                                if (FMT != 16) tc_mma(tmem + C::kO, ph, vd + (C::kPlane >> 4), kIdescO, 1);
                            }
                            tc_commit(ofull);
                            tc_commit(&vempty[st]);
                        }
                        ++i;
                    }
                }
                __syncwarp();
                if (FMT != 16 || !__syncthreads_or(0) || careful) break;
            }
        } else if (warp < C::kMmaWarp) {
            // ---- producers ---------------------------------------------------------------------------------------------------
            const int ptid = tid - 256;
            // 4 bits: a thread has group c of row r of every tile: the pieces (b, c) of 8 channels of every block b (values: groups 2 c
            // and 2 c + 1).  Its bytes are requested while it unpacks something else.
            struct Raw {
                unsigned v[NB], par[NB];
            };
            const int ur = ptid >> 2, uc = ptid & 3;
            auto request = [&](Raw& w, const uint8_t* src, int tile) {
                const int t = begin + tile * KT + ur;
                const bool ok = tile < nt && t < end;  // a row behind those in use is zeros
                const uint8_t* b0 = src + static_cast<size_t>(s) * P.seq_bytes;
                const size_t at = static_cast<size_t>(kvh) * P.cap + (ok ? t : 0);
                const uint8_t* rowp = b0 + at * (D / 2) + uc * (4 * NB);
                const uint8_t* par = b0 + P.par_off + at * (4 * NB);
                if constexpr (NB == 4) {
                    const uint4 x = *reinterpret_cast<const uint4*>(rowp), q = *reinterpret_cast<const uint4*>(par);
                    w.v[0] = x.x, w.v[1] = x.y, w.v[2] = x.z, w.v[3] = x.w;
                    w.par[0] = q.x, w.par[1] = q.y, w.par[2] = q.z, w.par[3] = q.w;
                } else {
                    const uint2 x = *reinterpret_cast<const uint2*>(rowp), q = *reinterpret_cast<const uint2*>(par);
                    w.v[0] = x.x, w.v[1] = x.y;
                    w.par[0] = q.x, w.par[1] = q.y;
                }
                if (!ok)
#pragma unroll
                    for (int b = 0; b < NB; ++b) w.par[b] = 0u;
            };
            auto unpack = [&](const Raw& raw, bool value, uint8_t* dst) {  // values as hi and lo tiles
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const unsigned pw = not_finite2(raw.par[b]) ? 0u : raw.par[b];  // (a hidden slot's scales may be anything)
                    const unsigned w = value ? __byte_perm(raw.v[b / 2], raw.v[NB / 2 + b / 2], b & 1 ? 0x7632 : 0x5410) : raw.v[b];
                    const float d = half_bits_to_float(pw & 0xFFFFu), m = half_bits_to_float(pw >> 16);
                    const float2 mid = both(fmaf(8.0f, d, m));
                    // codes about their middle without an integer conversion: the bits of 2^23 + code, less 2^23 + 8
                    const unsigned even = w & 0x0F0F0F0Fu, odd = (w >> 4) & 0x0F0F0F0Fu;
                    const bool large = fmaf(15.0f, d, fabsf(m)) > 65504.0f;  // the format reaches a little further than fp16
                    unsigned hi[4], lo[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float2 code = add2(make_float2(__uint_as_float(__byte_perm(even, 0x4B000000u, 0x7440 + k)), __uint_as_float(__byte_perm(odd, 0x4B000000u, 0x7440 + k))),
                                                 both(-8388616.0f));
                        const float2 x = fma2(both(d), code, mid);
                        __half2 h = __floats2half2_rn(x.x, x.y);
                        if (large) h = __floats2half2_rn(fminf(x.x, 65504.0f), fminf(x.y, 65504.0f));  // the rest goes to lo
                        const float2 l = fma2(__half22float2(h), both(-1.0f), x);
                        hi[k] = h2_bits(h), lo[k] = h2_bits(__floats2half2_rn(l.x, l.y));
                    }
                    uint8_t* o = dst + swz(KT, ur, 4 * b + uc);
                    *reinterpret_cast<uint4*>(o) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *reinterpret_cast<uint4*>(o + C::kPlane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
            };
            auto beside = [&](int t0, int st, int first, int threads) {  // positions and documents of a tile's slots
                int* meta = reinterpret_cast<int*>(sm + C::kMeta + st * C::kMetaBytes);
                for (int k = first; k < KT; k += threads) {
                    const KeyInfo key = key_info(P, s, kvh, t0 + k, end);
                    meta[k] = key.pos, meta[KT + k] = key.doc;
                }
            };
            const bool beside_wanted = GEN && (P.positions || P.k_doc);
            int i = 0;
            if constexpr (FMT != 16) {
                Raw rk, rv;
                int tile = next(-1);
                request(rk, P.k, tile);
                for (; tile < nt; ++i) {
                    const int st = i % C::kStages, ph = (i / C::kStages - 1) & 1, t0 = begin + tile * KT, after = next(tile);
                    request(rv, P.v, tile);
                    if (i >= C::kStages) tc_wait(&kempty[st], ph, fail);
                    unpack(rk, false, sm + C::kOffK + st * C::kSlot);
                    fence_async_shared();
                    bar_arrive(&kfull[st]);
                    request(rk, P.k, after);
                    if (i >= C::kStages) tc_wait(&vempty[st], ph, fail);
                    unpack(rv, true, sm + C::kOffV + st * C::kSlot);
                    if (beside_wanted) beside(t0, st, ptid, C::kProducers);
                    fence_async_shared();
                    bar_arrive(&vfull[st]);
                    tile = after;
                }
            } else {
                for (bool careful = false;; careful = true) {
                    for (int tile = next(-1); tile < nt; tile = next(tile), ++i) {
                        const int st = i % C::kStages, ph = (i / C::kStages - 1) & 1, t0 = begin + tile * KT;
                        uint8_t* vt = sm + C::kOffV + st * C::kSlot;
                        if (warp == 8 && lane == 0) {
                            if (i >= C::kStages) tc_wait(&kempty[st], ph, fail);
                            mbar_expect_tx(&kfull[st], C::kSlot);
#pragma unroll
                            for (int h = 0; h < D / 64; ++h) tma_4d(smem_u32(sm) + C::kOffK + st * C::kSlot + h * (KT * 128), &map_k, h * 64, kvh, t0, s, &kfull[st]);
                            if (i >= C::kStages) tc_wait(&vempty[st], ph, fail);
                            mbar_expect_tx(&varrived[st], C::kSlot);
#pragma unroll
                            for (int h = 0; h < D / 64; ++h) tma_4d(smem_u32(vt) + h * (KT * 128), &map_v, h * 64, kvh, t0, s, &varrived[st]);
                        }
                        if (warp != 8 && beside_wanted) {
                            if (i >= C::kStages) tc_wait(&vempty[st], ph, fail);
                            beside(t0, st, ptid - 32, 64);
                            bar_arrive(&mfull[st]);
                        }
                        if (careful) {
                            __syncwarp();
                            unsigned* odd = reinterpret_cast<unsigned*>(sm + C::kMeta + st * C::kMetaBytes + 2 * KT * 4);
                            tc_wait(&varrived[st], (i / C::kStages) & 1, fail);
                            if (ptid < KT / 32) odd[ptid] = 0u;
                            named_sync(3, C::kProducers);  // nobody sets a bit before they are cleared
#pragma unroll 1
                            for (int x = ptid; x < KT * CH; x += C::kProducers) {
                                uint8_t* at = vt + swz(KT, x / CH, x % CH);
                                if (!not_finite(*reinterpret_cast<const uint4*>(at))) continue;
                                zero_not_finite(at);
                                atomicOr(&odd[(x / CH) >> 5], 1u << ((x / CH) & 31));
                            }
                            fence_async_shared();
                            bar_arrive(&vfull[st]);
                        }
                    }
                    __syncwarp();
                    if (!__syncthreads_or(0) || careful) break;
                }
            }
        }
    } else {
        // ---- softmax -------------------------------------------------------------------------------------------------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegsSoftmax));
        const int r = tid & 127, row = row0 + r;
        const bool valid = row < P.rows;
        float* maxima = reinterpret_cast<float*>(sm + C::kMax);
        {  // the queries as hi and lo tiles, and each row's factor: eight lanes to a row, so that rows are read in whole lines
            const int l8 = tid & 7;
            constexpr int kPer = CH / 8;  // pieces of 8 channels per lane
            float4 all[C::kRows / 32][kPer][2];
#pragma unroll
            for (int i = 0; i < C::kRows / 32; ++i) {
                const int qrow = row0 + i * 32 + (tid >> 3);
                const bool ok = qrow < P.rows;
                const int token = (ok ? qrow : 0) / P.group, head = kvh * P.group + (ok ? qrow : 0) % P.group;
                const float4* qp = reinterpret_cast<const float4*>(P.q + static_cast<size_t>(s) * P.q_seq + static_cast<size_t>(token) * P.q_token + static_cast<size_t>(head) * P.q_head);
#pragma unroll
                for (int k = 0; k < kPer; ++k)
#pragma unroll
                    for (int e = 0; e < 2; ++e) all[i][k][e] = ok && (k * 8 + l8) * 8 < P.dim ? qp[2 * (k * 8 + l8) + e] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
#pragma unroll
            for (int i = 0; i < C::kRows / 32; ++i) {
                const int q = i * 32 + (tid >> 3);
                const float4(&x)[kPer][2] = all[i];
                float amax = 0.0f;
#pragma unroll
                for (int k = 0; k < kPer; ++k)
#pragma unroll
                    for (int e = 0; e < 2; ++e) amax = fmaxf(fmaxf(amax, fmaxf(fabsf(x[k][e].x), fabsf(x[k][e].y))), fmaxf(fabsf(x[k][e].z), fabsf(x[k][e].w)));
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                float up, down;
                row_scale(amax, up, down);
                // positive, so that the largest product is the largest score; a negative scale goes to the query
                if (l8 == 0) maxima[q] = fmaxf(fabsf(P.sc) * down, 1e-37f);
                if (P.sc < 0.0f) up = -up;
#pragma unroll
                for (int k = 0; k < kPer; ++k) {
                    const float4 a = x[k][0], b = x[k][1];
                    uint4 hi, lo;
                    split2(a.x * up, a.y * up, hi.x, lo.x);
                    split2(a.z * up, a.w * up, hi.y, lo.y);
                    split2(b.x * up, b.y * up, hi.z, lo.z);
                    split2(b.z * up, b.w * up, hi.w, lo.w);
                    const int at = swz(C::kRows, q, k * 8 + l8);
                    *reinterpret_cast<uint4*>(sm + at) = hi;
                    *reinterpret_cast<uint4*>(sm + C::kQHalf + at) = lo;
                }
            }
            fence_async_shared();
        }
        named_sync(5, 288);
        const float ysc = maxima[r];
        named_sync(4, 256);  // the maxima of the first tile go to the same place
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + C::kS + wg * HK + lanes, to = tmem + C::kO + wg * (D / 2) + lanes;
        RowInfo ri{};
        if (GEN) ri = row_info(P, s, kvh, n, row);
        // slots from `limit` on are hidden by the end of the range, or (slot = position) by causality
        int limit = valid ? end : 0;
        if (P.causal && valid && !(GEN && P.positions)) limit = causal_limit(row_pos(P, s, n, row / P.group), prefix, end);

        float2 o[D / 4];  // this warpgroup's half of the channels
        float m, l, al;
        auto drain = [&]() {  // o = o al + the last tile's output
            float v[2][32];  // the next 32 channels are on their way while these are added
            tc_ld32(to, v[0]);
#pragma unroll
            for (int h = 0; h < D / 64; ++h) {
                tc_ld_wait(v[h & 1]);
                if (h + 1 < D / 64) tc_ld32(to + (h + 1) * 32, v[(h + 1) & 1]);
#pragma unroll
                for (int k = 0; k < 16; ++k) o[h * 16 + k] = fma2(o[h * 16 + k], both(al), make_float2(v[h & 1][2 * k], v[h & 1][2 * k + 1]));
            }
        };
        int i = 0;  // tiles so far, over both passes
        for (bool careful = false;; careful = true) {
        const int i0 = i;
        m = -INFINITY, l = 0.0f, al = 1.0f;
#pragma unroll
        for (int k = 0; k < D / 4; ++k) o[k] = make_float2(0.0f, 0.0f);
        for (int tile = next(-1); tile < nt; tile = next(tile), ++i) {
            const int t0 = begin + tile * KT + wg * HK;  // this warpgroup's first slot
            const int st = i % C::kStages;
            const int* meta = reinterpret_cast<const int*>(sm + C::kMeta + st * C::kMetaBytes) + wg * HK;
            tc_wait(sfull, i & 1, fail);
            __syncwarp();
            tc_after_sync();
            float yy[HK / 32][32];
#pragma unroll
            for (int h = 0; h < HK / 32; ++h) tc_ld32(ts + h * 32, yy[h]);
#pragma unroll
            for (int h = 0; h < HK / 32; ++h) tc_ld_wait(yy[h]);
#define Y(k) yy[(k) >> 5][(k) & 31]
            tc_before_sync();
            bar_arrive(sread);
            float fac = ysc;  // what turns y into base-2 scores
            if (GEN) {
                if (P.cap_out != 0.0f) {
                    cap_scores(yy, ysc);
                    fac = P.cap_out;
                }
                if (P.mask || P.bias_step != 0.0f) {
#pragma unroll
                    for (int k = 0; k < HK; k += 2) {
                        const float2 t = mul2(make_float2(Y(k), Y(k + 1)), both(fac));
                        Y(k) = t.x, Y(k + 1) = t.y;
                    }
                    fac = 1.0f;
                }
                if (P.positions || P.k_doc) tc_wait(FMT == 16 ? &mfull[st] : &vfull[st], (i / C::kStages) & 1, fail);
                if (P.mask) {
                    const unsigned short* mp = ri.mask + t0;
                    const bool wide = ((reinterpret_cast<uintptr_t>(mp) & 15) == 0) && t0 + HK <= end;
#pragma unroll
                    for (int k8 = 0; k8 < HK / 8; ++k8) {
                        unsigned w[4];
                        if (wide) {
                            const uint4 t = *reinterpret_cast<const uint4*>(mp + 8 * k8);
                            w[0] = t.x, w[1] = t.y, w[2] = t.z, w[3] = t.w;
                        } else {
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const int t = t0 + 8 * k8 + 2 * k;
                                w[k] = (t < end ? mp[8 * k8 + 2 * k] : 0xFC00u) | (static_cast<unsigned>(t + 1 < end ? mp[8 * k8 + 2 * k + 1] : 0xFC00u) << 16);
                            }
                        }
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            float& v = Y(k8 * 8 + k);
                            const unsigned h = w[k >> 1] >> (16 * (k & 1)) & 0xFFFFu;
                            v = h == 0xFC00u ? -INFINITY : fmaf(ri.slope, half_bits_to_float(h), v);
                        }
                    }
                } else if (P.bias_step != 0.0f) {
                    if (P.positions) {
#pragma unroll
                        for (int k = 0; k < HK; ++k) Y(k) -= ri.slope * fabsf(static_cast<float>(ri.pos - meta[k]));
                    } else {
                        const float far = static_cast<float>(ri.pos - t0);
                        if (__all_sync(0xffffffffu, far >= static_cast<float>(HK - 1))) {  // all of them in front of the query: no absolute value
                            const float nearest = ri.slope * (static_cast<float>(HK - 1) - far);
#pragma unroll
                            for (int k = 0; k < HK; ++k) Y(k) += fmaf(ri.slope, static_cast<float>(k - (HK - 1)), nearest);
                        } else {
#pragma unroll
                            for (int k = 0; k < HK; ++k) Y(k) -= ri.slope * fabsf(far - static_cast<float>(k));
                        }
                    }
                }
                if (P.causal && P.positions) {
#pragma unroll
                    for (int k = 0; k < HK; k += 4) {
                        const int4 kp = *reinterpret_cast<const int4*>(meta + k);
                        if (kp.x > ri.pos && kp.x >= prefix) Y(k) = -INFINITY;
                        if (kp.y > ri.pos && kp.y >= prefix) Y(k + 1) = -INFINITY;
                        if (kp.z > ri.pos && kp.z >= prefix) Y(k + 2) = -INFINITY;
                        if (kp.w > ri.pos && kp.w >= prefix) Y(k + 3) = -INFINITY;
                    }
                }
                if (docs) {
#pragma unroll
                    for (int k = 0; k < HK; k += 4) {
                        const int4 kd = *reinterpret_cast<const int4*>(meta + KT + k);
                        if (kd.x != ri.doc) Y(k) = -INFINITY;
                        if (kd.y != ri.doc) Y(k + 1) = -INFINITY;
                        if (kd.z != ri.doc) Y(k + 2) = -INFINITY;
                        if (kd.w != ri.doc) Y(k + 3) = -INFINITY;
                    }
                }
            }
            if (!__all_sync(0xffffffffu, t0 + HK <= limit)) {
#pragma unroll
                for (int k = 0; k < HK; ++k)
                    if (t0 + k >= limit) Y(k) = -INFINITY;
            }
            float mx = Y(0), mx1 = Y(1);
#pragma unroll
            for (int k = 2; k < HK; k += 4) {
                mx = max3(mx, Y(k), Y(k + 1));
                if (k + 2 < HK) mx1 = max3(mx1, Y(k + 2), Y(k + 3));
            }
            mx = fmaxf(mx, mx1) * fac;
            maxima[((i & 1) * 2 + wg) * C::kRows + r] = mx;
            bar_arrive(mxfull);
            tc_wait(mxfull, i & 1, fail);
            mx = max3(m, mx, maxima[((i & 1) * 2 + 1 - wg) * C::kRows + r]);
            const float al1 = mx > m ? ex2(m - mx) : 1.0f;
            m = mx;
            const float2 ref = both(m == -INFINITY ? 0.0f : kPShift - m);
            float2 sum = make_float2(0.0f, 0.0f), sum1 = sum;
            const uint32_t tp = tmem + C::kP + (i & 1) * KT + wg * (HK / 2) + lanes;
            __syncwarp();
#pragma unroll
            for (int h = 0; h < HK / 32; ++h) {
                unsigned hi[16], lo[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const float2 v = make_float2(yy[h][2 * k], yy[h][2 * k + 1]), e = fma2(v, both(fac), ref);
                    const float2 p = make_float2(ex2(e.x), ex2(e.y));
                    if (k & 1) sum1 = add2(sum1, p);
                    else sum = add2(sum, p);
                    const __half2 hh = __floats2half2_rn(p.x, p.y);
                    const float2 d = fma2(__half22float2(hh), both(-1.0f), p);
                    hi[k] = h2_bits(hh), lo[k] = h2_bits(__floats2half2_rn(d.x, d.y));
                }
                tc_st16(tp + h * 16, hi);
                tc_st16(tp + KT / 2 + h * 16, lo);
            }
#undef Y
            sum = add2(sum, sum1);
            l = fmaf(l, al1, sum.x + sum.y);
            if (i > i0) {
                tc_wait(ofull, (i - 1) & 1, fail);
                __syncwarp();
                tc_after_sync();
                drain();
            }
            al = al1;
            tc_st_wait();
            if (FMT == 16 && careful) {  // values of this tile that are not finite go to the rows that see them one by one
                tc_wait(&vfull[st], ((i - i0) / C::kStages) & 1, fail);
                const unsigned* odd = reinterpret_cast<const unsigned*>(sm + C::kMeta + st * C::kMetaBytes + 2 * KT * 4);
                unsigned any = 0;
#pragma unroll
                for (int h = 0; h < KT / 32; ++h) any |= odd[h];
                tc_before_sync();
                named_sync(4, 256);  // both halves of the probabilities are stored
                tc_after_sync();
                if (any) {
                    al = fmaxf(al, 1e-30f);  // an infinity added now stays one when the output is rescaled
                    const uint32_t pb = tmem + C::kP + (i & 1) * KT + lanes;
                    const int first = begin + tile * KT;
#pragma unroll 1
                    for (int k = 0; k < KT; ++k) {
                        if (!(odd[k >> 5] >> (k & 31) & 1u)) continue;
                        const unsigned* vp = reinterpret_cast<const unsigned*>(reinterpret_cast<const __half*>(P.v) + static_cast<size_t>(s) * P.v_seq +
                                                                               static_cast<size_t>(kvh) * P.v_head + static_cast<size_t>(first + k) * P.v_row + wg * (D / 2));
                        const unsigned ph = tc_ld1(pb + (k >> 1)) >> (16 * (k & 1)), pl = tc_ld1(pb + KT / 2 + (k >> 1)) >> (16 * (k & 1));
                        const float p = half_bits_to_float(ph & 0xFFFFu) + half_bits_to_float(pl & 0xFFFFu);
                        if (p != 0.0f)
#pragma unroll
                            for (int ch = 0; ch < D / 4; ++ch)
                                if (wg * (D / 2) + 2 * ch < P.dim) add_not_finite(o[ch].x, o[ch].y, p, vp[ch]);
                        __syncwarp();
                    }
                }
            }
            tc_before_sync();
            bar_arrive(pfull);
        }
        if (i > i0) {
            tc_wait(ofull, (i - 1) & 1, fail);
            __syncwarp();
            tc_after_sync();
            drain();
        }
        if (FMT != 16) break;
        float2 bad = make_float2(l * 0.0f, 0.0f);  // NaN if anything is not finite
#pragma unroll
        for (int k = 0; k < D / 4; ++k) bad = fma2(o[k], both(0.0f), bad);
        if (!__syncthreads_or(!(bad.x + bad.y == 0.0f)) || careful) break;
        }
        // ---- the row's sum over both halves of its keys; each warpgroup stores its half of the channels ---------------------------
        named_sync(4, 256);
        maxima[wg * C::kRows + r] = l;
        named_sync(4, 256);
        const float L = l + maxima[(1 - wg) * C::kRows + r];
        const float f = P.nsplit > 1 ? 1.0f : L > 0.0f || L != L ? 1.0f / L : 0.0f;
        // through shared memory (the rings are free), so that rows are written in whole lines
        constexpr int kStride = D + 4;
        static_assert(C::kRows * kStride * 4 <= 2 * C::kStages * C::kSlot, "the rings hold the output");
        float* stage_out = reinterpret_cast<float*>(sm + C::kOffK);
#pragma unroll
        for (int k = 0; k < D / 4; k += 2)
            *reinterpret_cast<float4*>(stage_out + r * kStride + wg * (D / 2) + 2 * k) = make_float4(o[k].x * f, o[k].y * f, o[k + 1].x * f, o[k + 1].y * f);
        const size_t part0 = ((static_cast<size_t>(s) * P.kv_heads + kvh) * P.nsplit + split) * P.rows;
        if (wg == 0 && valid) {
            if (P.nsplit > 1) P.part_ml[part0 + row] = make_float2(m, L);
            else if (P.final_ml) P.final_ml[(static_cast<size_t>(s) * P.kv_heads + kvh) * P.rows + row] = make_float2(m, L);
        }
        named_sync(4, 256);
#pragma unroll 8
        for (int x = tid; x < C::kRows * (D / 4); x += 256) {
            const int q = x / (D / 4), ch = x % (D / 4) * 4, qrow = row0 + q;
            if (qrow >= P.rows || ch >= P.dim) continue;
            const int token = qrow / P.group, head = kvh * P.group + qrow % P.group;
            float* dst = P.nsplit > 1 ? P.part_o + (part0 + qrow) * P.dim
                                      : P.out + static_cast<size_t>(s) * P.o_seq + static_cast<size_t>(token) * P.o_token + static_cast<size_t>(head) * P.o_head;
            *reinterpret_cast<float4*>(dst + ch) = *reinterpret_cast<const float4*>(stage_out + q * kStride + ch);
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
    if (warp == C::kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

// Tensor map of an fp16 cache's keys or values: {channel, head, slot, sequence}, boxes of 64 channels x KT slots, 128-byte swizzle.
inline bool cache_map(CUtensorMap* map, const uint8_t* base, const AttnP& P, int head_dim, long long row, long long head, long long seq, int slots) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) p = nullptr;
        return reinterpret_cast<Encode>(p);
    }();
    if (!encode) return false;
    // a dimension of one element is never stepped over: its stride may be anything that is allowed
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(P.kv_heads), static_cast<cuuint64_t>(P.cap), static_cast<cuuint64_t>(P.n_seqs)};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(P.kv_heads > 1 ? head * 2 : 16), static_cast<cuuint64_t>(P.cap > 1 ? row * 2 : 16),
                                   static_cast<cuuint64_t>(P.n_seqs > 1 ? seq * 2 : 16)};
    const cuuint32_t box[4] = {64, 1, static_cast<cuuint32_t>(slots), 1}, one[4] = {1, 1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<uint8_t*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Once per device: room for dynamic shared memory, and whether the kernel was built with the registers that its hand-over counts on.
template <class Kern>
inline bool prepare_kernel(Kern kern, int smem, int regs, PerDeviceFlag& f) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return false;
    if (f.set[dev].load(std::memory_order_acquire)) return true;
    cudaFuncAttributes a;
    if (cudaFuncGetAttributes(&a, kern) != cudaSuccess || a.numRegs < regs) return false;
    return raise_dynamic_smem(kern, smem, f);
}
template <int D, int FMT>
int attn_launch_tc(const AttnP& P, bool general, cudaStream_t st) {
    if constexpr (D == 64 || D == 128) {
        using C = TcCfg<D, FMT>;
        CUtensorMap mk{}, mv{};
        if (FMT == 16 && !(cache_map(&mk, P.k, P, P.dim, P.k_row, P.k_head, P.k_seq, C::KT) && cache_map(&mv, P.v, P, P.dim, P.v_row, P.v_head, P.v_seq, C::KT)))
            return KCB_UNSUPPORTED_OPERATION;
        static PerDeviceFlag raised[2];
        const dim3 grid(P.row_tiles * P.nsplit, P.kv_heads, P.n_seqs);
        if (general) {
            if (!prepare_kernel(attn_tc_kernel<D, FMT, true>, C::kSmem, C::kRegsLaunch, raised[0])) return KCB_LAUNCH_FAILURE;
            attn_tc_kernel<D, FMT, true><<<grid, C::kThreads, C::kSmem, st>>>(P, mk, mv);
        } else {
            if (!prepare_kernel(attn_tc_kernel<D, FMT, false>, C::kSmem, C::kRegsLaunch, raised[1])) return KCB_LAUNCH_FAILURE;
            attn_tc_kernel<D, FMT, false><<<grid, C::kThreads, C::kSmem, st>>>(P, mk, mv);
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

// Causal grouped-query attention over whole prompts, packed back to back:
// sequence b has the queries q_starts[b] .. q_starts[b + 1] - 1 and the
// positions kv_starts[b] .. kv_starts[b + 1] - 1 of k and v; with n_q and n_k
// of them, query i stands at position n_k - n_q + i and attends the
// positions up to its own:
//   out[i, h] = softmax_{p <= n_k - n_q + i}(scale * q[i, h] . k[p, h / g]) . v[p, h / g]
// A query before the first position (n_k < n_q) gets zeros; rows of out that
// belong to no sequence keep their values.
//
// On the tcgen05 tensor cores, head_dim 64 and 128.  A query tile is 128 rows:
// floor(128 / g) tokens of one sequence times the g query heads of one KV
// head (one TMA box of q), so K and V are read once for the group and short
// prompts fill the tile.  A work item is two consecutive query tiles, which
// share every K/V tile of 128 positions; persistent CTAs, one per SM, walk
// the items:
// * warp 8 finds the items, from the largest down (the offsets are read on the
//   device; of up to 256 sequences the pairs of query tiles are ranked by
//   counting, without a sort), hands them on and loads Q and the K and V
//   tiles (TMA, 128-byte swizzle);
// * warp 9 owns tensor memory; one thread issues S_i = Q_i K^T and
//   O_i += P_i V (P_i read from tensor memory, over the first half of S_i).
//   While the softmax of one query tile runs, the products of the other do;
//   at head_dim 64 a third S buffer keeps the next S ready for each;
// * warps 0-3 and 4-7 run the softmax of query tiles 0 and 1, one thread per
//   row: the maximum moves (and O_i is rescaled) only when a score passes it
//   by more than 8 in log2 units.  P is rounded to f16, the operand's type: a
//   second product for its low bits would add half to the tensor work;
// * warps 10 and 11 look through the V tiles that some row sees in part (the
//   last of each item) before they are used: 0 times an infinity or NaN of a
//   masked position would be NaN, so such values are taken out, and the
//   rows that do attend them add them at the end (rare, from global memory).
// Products on S and P of one buffer follow one another in the order in which
// the one issuing lane issues them.
// Bound by the chain softmax -> P V -> S of a query tile (3700 cycles for two
// tiles of 128 x 128 at head_dim 128, where the products take 2048 and the exp2
// unit as many): 8192 tokens, 32/8 heads, head_dim 128: 565 us = 974 TFLOP/s;
// 12 prompts of 60 to 1000 tokens at head_dim 64: 50.5 us.
// Every wait is bounded; an expired wait aborts the CTA, which waits for its
// issued MMAs (bounded) and frees its tensor memory.  No load uses cluster
// multicast.
#include "mote_common.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

namespace mote {
namespace attnv {

using attnp::ex2f;
using attnp::max3f;
using attnp::tma_load_3d;
using attnp::tmem_ld32_nowait;
using attnp::tmem_wait_ld;
using attnp::tmem_wait_st;
using attnp::umma_f16_ss;
using gemm::wait_or_abort;

constexpr int kBM = 128;  // rows of a query tile (TMEM lanes)
constexpr int kBN = 128;  // positions of a K/V tile
constexpr int kProducerWarp = 8;
constexpr int kMmaWarp = 9;
constexpr int kCleanWarps = 2;  // 10 and 11
constexpr int kThreads = 12 * 32;
// Register split (setmaxnreg, per warpgroup): launched at 168 a thread;
// 384 x 168 = 256 x 224 + 128 x 56, and 32 x (224 + 224 + 56) <= 16384.
constexpr int kLaunchRegs = 168;
constexpr int kSoftmaxRegs = 224;
constexpr int kOtherRegs = 56;
static_assert(kThreads * kLaunchRegs == 256 * kSoftmaxRegs + 128 * kOtherRegs, "register split");
static_assert(32 * (2 * kSoftmaxRegs + kOtherRegs) <= 16384, "registers of a sub-partition");
constexpr int kItems = 4;          // items that the producer may be ahead
// P is held as 2^kShift times the probability relative to the reference, which
// the row's maximum passes by 2^8 at most: up to 2^15 in f16, with its 11 bits
// down to 2^-21 of the reference and steps of 2^-31 below (without the shift
// 2^-14 and 2^-24, where a large V of little weight lost its bits).
constexpr float kShift = 7.f;
// score * scale - reference * scale is one fma, whose rounded second product
// leaves up to 2^-24 of it; references beyond this (log2 units) are subtracted
// from the scores instead.  Equal scores meet under different references where a
// row's moves: near 35000 their weights were up to 2^-8 apart (log2), at 1024 it is
// 2^-13.
constexpr float kVast = 1024.f;
// Sequences up to which items are ranked by size: 8 to a lane of the producer
// warp, in registers.  Ranked against in the order of the sequences: 12 prompts
// of 60 to 1000 57 against 62 us, 64 of 50 to 100 over 2000 cached 108 against
// 142, 256 of up to 300 209 against 210 (head_dim 64); 310 against 326 (128).
constexpr std::uint32_t kSorted = 256;
// Items whose "V holds something not finite" flags are kept.  A row's thread
// takes an item from the ring when it is done with the one before, so warps 10
// and 11 are at most kItems items past the one whose flag a row still reads.
constexpr int kFlags = 8;
static_assert(kFlags > kItems, "a flag in use is not written");

// TMEM columns: S buffers of 128, then O_0 and O_1; P over the first 64 of its S.
constexpr std::uint32_t kTmemCols = 512;

struct Params {
    const std::int32_t* q_starts;
    const std::int32_t* kv_starts;
    const __half* v;
    __half* out;
    std::uint32_t tokens, kv_tokens, batch, q_heads, kv_heads, group;
    std::uint32_t tile_tokens;  // floor(128 / group)
    float scale_log2;
};

// Two query tiles of one sequence and KV head.
struct Item {
    std::uint32_t left;    // the sequence's tokens from the first on; 0: no more items
    std::uint32_t kvh;
    std::uint32_t q0;      // packed row of the first token
    std::int32_t pos0;     // its position
    std::uint32_t k0, nk;  // first row and number of the positions
    std::uint32_t n[2];    // K/V tiles that each query tile attends
    std::uint32_t masked;  // the first tile that some row sees in part
    __device__ __forceinline__ std::uint32_t tiles() const { return max(n[0], n[1]); }
};

template <int HD>
struct Smem {
    static constexpr int kHalf = 128 * 128;           // 128 rows of 64 f16
    static constexpr int kTile = HD / 64 * kHalf;     // a Q, K or V tile
    static constexpr int kKV = HD == 64 ? 4 : 2;      // K and V stages
    // S buffers: what tensor memory holds beside the two O
    static constexpr int kS = HD == 64 ? 3 : 2;
    static constexpr std::uint32_t kColO = 128 * kS;  // O_i at kColO + HD i
    static_assert(kColO + 2 * HD <= kTmemCols, "tensor memory");
    static constexpr int kQ = 0;                      // [2] query tiles
    static constexpr int kK = kQ + 2 * kTile;
    static constexpr int kV = kK + kKV * kTile;
    static constexpr int kBar = kV + kKV * kTile;
    // q_full, q_empty, k_full, k_empty, v_full, v_empty, v_clean [kKV],
    // s_full, o_done [2][kS], p_half, p_ready [kS], epi_done[2], drained, item_full, item_empty [kItems]
    static constexpr int kNumBars = 2 + 5 * kKV + 6 * kS + 2 + 1 + 2 * kItems;
    static constexpr int kTmemSlot = kBar + kNumBars * 8;
    static constexpr int kAbort = kTmemSlot + 4;
    static constexpr int kFlag = kAbort + 4;          // [kFlags][kCleanWarps]
    static constexpr int kItem = kFlag + 4 * kFlags * kCleanWarps;  // [kItems]
    static constexpr int kUsed = kItem + kItems * static_cast<int>(sizeof(Item)) + 1008;  // + alignment slack
    // one CTA per SM: its 512 TMEM columns never wait for another's
    static constexpr int kBytes = kUsed > 120 * 1024 ? kUsed : 120 * 1024;
    static_assert(kBytes <= 232448, "shared memory");
};

__device__ __forceinline__ bool sequence_ok(const Params& p, std::int32_t q0, std::int32_t q1,
                                            std::int32_t k0, std::int32_t k1) {
    return q0 >= 0 && q1 >= q0 && static_cast<std::uint32_t>(q1) <= p.tokens && k0 >= 0 &&
           k1 >= k0 && static_cast<std::uint32_t>(k1) <= p.kv_tokens;
}

// Query tile pairs of sequence b, and the level of the first: pair i of a
// sequence is at level i + (positions before its queries) / (tokens of a
// pair), which orders the pairs of all sequences by the tiles they attend.
struct Pairs {
    std::uint32_t count, level;
};
__device__ __forceinline__ Pairs pairs_of(const Params& p, std::uint32_t b) {
    const std::int32_t q0 = __ldg(p.q_starts + b), q1 = __ldg(p.q_starts + b + 1);
    const std::int32_t k0 = __ldg(p.kv_starts + b), k1 = __ldg(p.kv_starts + b + 1);
    if (!sequence_ok(p, q0, q1, k0, k1)) return Pairs{0, 0};
    const std::uint32_t span = 2 * p.tile_tokens, nq = q1 - q0, nk = k1 - k0;
    return Pairs{(nq + span - 1) / span, nk > nq ? (nk - nq) / span : 0};
}

// Pair `i` of sequence b for one KV head.
__device__ __forceinline__ Item make_item(const Params& p, std::uint32_t b, std::uint32_t i,
                                          std::uint32_t kvh) {
    Item it{};
    const std::int32_t q0 = __ldg(p.q_starts + b), q1 = __ldg(p.q_starts + b + 1);
    const std::int32_t k0 = __ldg(p.kv_starts + b), k1 = __ldg(p.kv_starts + b + 1);
    const std::uint64_t t0 = static_cast<std::uint64_t>(i) * (2 * p.tile_tokens);
    if (!sequence_ok(p, q0, q1, k0, k1) || t0 >= static_cast<std::uint32_t>(q1 - q0)) return it;
    it.kvh = kvh;
    it.left = static_cast<std::uint32_t>(q1 - q0) - static_cast<std::uint32_t>(t0);
    it.q0 = static_cast<std::uint32_t>(q0) + static_cast<std::uint32_t>(t0);
    it.k0 = static_cast<std::uint32_t>(k0);
    it.nk = static_cast<std::uint32_t>(k1 - k0);
    it.pos0 = static_cast<std::int32_t>(it.nk) - static_cast<std::int32_t>(it.left);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const std::uint32_t from = m * p.tile_tokens;
        const std::int32_t last = it.pos0 + static_cast<std::int32_t>(min(from + p.tile_tokens, it.left)) - 1;
        it.n[m] = from >= it.left || last < 0 ? 0u : static_cast<std::uint32_t>(last) / kBN + 1;
    }
    it.masked = static_cast<std::uint32_t>(max(it.pos0 + 1, 0)) / kBN;
    return it;
}

// Of up to kSorted sequences, whose pairs the lanes hold (sequence 32 i + lane
// in x[i]): the pair of rank r by falling level.  N(d) pairs are at level d
// or above, so r's level is the largest d with N(d) > r, and it is number
// r - N(d + 1) of the sequences there.  By a whole warp.
constexpr int kHeld = kSorted / 32;
__device__ __forceinline__ Item sorted_item(const Params& p, const Pairs (&x)[kHeld], std::uint32_t r,
                                            std::uint32_t levels, std::uint32_t kvh) {
    const auto at_least = [&](std::uint32_t d) {  // N(d)
        std::uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const std::uint32_t end = x[i].level + x[i].count;
            n += end > d ? min(end - d, x[i].count) : 0u;
        }
        return __reduce_add_sync(0xffffffffu, n);
    };
    std::uint32_t lo = 0, hi = levels;  // N(lo) > r, N(hi) <= r
    while (hi - lo > 1) {
        const std::uint32_t mid = (lo + hi) / 2;
        if (at_least(mid) > r) lo = mid; else hi = mid;
    }
    std::uint32_t e = r - at_least(lo + 1), b = 0, first = 0;
    bool found = false;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const bool here = x[i].level <= lo && lo < x[i].level + x[i].count;
        const unsigned mask = __ballot_sync(0xffffffffu, here);
        const std::uint32_t k = __popc(mask);
        // the lane with e such sequences below it
        const unsigned below = mask & ((1u << (threadIdx.x & 31)) - 1u);
        const unsigned pick = __ballot_sync(0xffffffffu, here && __popc(below) == e);
        if (!found && e < k) {
            const int src = __ffs(pick) - 1;
            found = true, b = 32 * i + src;
            first = __shfl_sync(0xffffffffu, x[i].level, src);
        }
        if (!found) e -= k;
    }
    return make_item(p, b, lo - first, kvh);
}

// Of more, pairs in the order of the sequences: those of sequence b are
// numbered from floor(q_starts[b] / tokens of a pair) + b on, with gaps.
__device__ __forceinline__ Item plain_item(const Params& p, std::uint32_t slot, std::uint32_t kvh) {
    const std::uint32_t span = 2 * p.tile_tokens;
    const auto first = [&](std::uint32_t b) {
        return static_cast<std::uint32_t>(max(__ldg(p.q_starts + b), 0)) / span + b;
    };
    const std::uint32_t b = kvq8::warp_search(p.batch, slot, first);
    const std::uint32_t f = first(b);
    return slot < f ? Item{} : make_item(p, b, slot - f, kvh);
}

// 32 lanes x 16 consecutive columns.
__device__ __forceinline__ void tmem_ld16(std::uint32_t taddr, std::uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(std::uint32_t taddr, const std::uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15])
        : "memory");
}

// One lane of the (converged) warp, always the same.
__device__ __forceinline__ bool elect_one() {
    std::uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ void arrive(std::uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// B operand of P V: V rows (positions) of 64 dimensions; the second 64
// dimensions lie a half tile further (the leading-dimension offset).
template <int HD>
__device__ __forceinline__ std::uint64_t v_desc(std::uint32_t addr) {
    const std::uint64_t d = gemm::smem_desc_sw128(addr);
    return HD == 64 ? d : (d & ~(0x3fffull << 16)) | static_cast<std::uint64_t>(Smem<HD>::kHalf >> 4) << 16;
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
    packed_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const Params p) {
    using L = Smem<HD>;
    constexpr int kKV = L::kKV;
    // kind::f16, f32 accumulators: S: M = 128, N = 128, K-major operands; PV: N = HD, B MN-major
    constexpr std::uint32_t kIdescS = (1u << 4) | ((kBN >> 3) << 17) | ((kBM >> 4) << 24);
    constexpr std::uint32_t kIdescPV = (1u << 4) | (1u << 16) | ((HD >> 3) << 17) | ((kBM >> 4) << 24);
    extern __shared__ std::uint8_t smem_raw[];
    const std::uint32_t raw_base = smem_u32(smem_raw);
    const std::uint32_t base = (raw_base + 1023u) & ~1023u;
    std::uint8_t* smem = smem_raw + (base - raw_base);
    std::uint64_t* bars = reinterpret_cast<std::uint64_t*>(smem + L::kBar);
    std::uint64_t* q_full = bars;
    std::uint64_t* q_empty = bars + 1;
    std::uint64_t* k_full = bars + 2;
    std::uint64_t* k_empty = k_full + kKV;
    std::uint64_t* v_full = k_empty + kKV;
    std::uint64_t* v_empty = v_full + kKV;
    std::uint64_t* v_clean = v_empty + kKV;
    std::uint64_t* s_full = v_clean + kKV;
    std::uint64_t* p_half = s_full + 2 * L::kS;
    std::uint64_t* p_ready = p_half + L::kS;
    std::uint64_t* o_done = p_ready + L::kS;
    std::uint64_t* epi_done = o_done + 2 * L::kS;
    std::uint64_t* drained = epi_done + 2;
    std::uint64_t* item_full = drained + 1;
    std::uint64_t* item_empty = item_full + kItems;
    Item* ring = reinterpret_cast<Item*>(smem + L::kItem);
    volatile std::uint32_t* tmem_slot = reinterpret_cast<volatile std::uint32_t*>(smem + L::kTmemSlot);
    volatile std::uint32_t* abort_flag = reinterpret_cast<volatile std::uint32_t*>(smem + L::kAbort);
    volatile std::uint32_t* not_finite = reinterpret_cast<volatile std::uint32_t*>(smem + L::kFlag);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        for (int s = 0; s < kKV; ++s) {
            mbar_init(&k_full[s], 1);
            mbar_init(&k_empty[s], 1);
            mbar_init(&v_full[s], 1);
            mbar_init(&v_empty[s], 1 + kCleanWarps);  // the last P V, and warps 10 and 11 keep step
            mbar_init(&v_clean[s], kCleanWarps);
        }
        for (int s = 0; s < L::kS; ++s) {
            mbar_init(&s_full[s], 1);
            mbar_init(&s_full[L::kS + s], 1);
            mbar_init(&p_half[s], 4);
            mbar_init(&p_ready[s], 4);
            mbar_init(&o_done[s], 1);
            mbar_init(&o_done[L::kS + s], 1);
        }
        mbar_init(&epi_done[0], 4);
        mbar_init(&epi_done[1], 4);
        for (int s = 0; s < kItems; ++s) {
            mbar_init(&item_full[s], 1);
            mbar_init(&item_empty[s], 11);  // every warp but the producer
        }
        mbar_init(drained, 1);
        *abort_flag = 0u;
        fence_mbarrier_init();
    }
    if (p.tile_tokens * p.group < kBM) {  // rows of a query tile that no box fills stay zero
        for (int i = threadIdx.x; i < 2 * L::kTile / 16; i += kThreads)
            reinterpret_cast<uint4*>(smem + L::kQ)[i] = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
    }
    if (warp == kMmaWarp) gemm::tmem_alloc(base + L::kTmemSlot, kTmemCols);
    gemm::tc_fence_before();
    __syncthreads();
    gemm::tc_fence_after();
    const std::uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();
    pdl_wait();

    // item i of this CTA, as the producer found it (by a whole warp other than
    // the producer's); left == 0 ends the loops, after an abort too
    const auto item_at = [&](std::uint32_t i) {
        Item it{};
        const std::uint32_t s = i % kItems;
        if (__all_sync(0xffffffffu, wait_or_abort(&item_full[s], (i / kItems) & 1u, abort_flag))) it = ring[s];
        __syncwarp();
        if (lane == 0) arrive(&item_empty[s]);
        return it;
    };
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == kProducerWarp) {
            if (blockIdx.x == 0)  // offsets that the items skip are reported
                for (std::uint32_t b = lane; b < p.batch; b += 32)
                    if (!sequence_ok(p, p.q_starts[b], p.q_starts[b + 1], p.kv_starts[b], p.kv_starts[b + 1]))
                        atomicOr(&g_device_status, kDevIndexOutOfRange);
            // Items of falling size to the CTAs in turn, forwards and backwards.
            const std::uint32_t span = 2 * p.tile_tokens;
            const bool sorted = p.batch <= kSorted;
            std::uint32_t pairs = p.tokens / span + p.batch, levels = 0;
            Pairs held[kHeld];
#pragma unroll
            for (int x = 0; x < kHeld; ++x)
                held[x] = sorted && 32u * x + lane < p.batch ? pairs_of(p, 32 * x + lane) : Pairs{0, 0};
            if (sorted) {
                std::uint32_t count = 0;
#pragma unroll
                for (int x = 0; x < kHeld; ++x) {
                    count += held[x].count;
                    levels = max(levels, held[x].level + held[x].count);
                }
                pairs = __reduce_add_sync(0xffffffffu, count);
                levels = __reduce_max_sync(0xffffffffu, levels);
            }
            const std::uint32_t items = pairs * p.kv_heads;
            std::uint32_t c = 0, n = 0, sent = 0;  // K/V tiles, items with any and items so far
            bool ok = true;
            for (std::uint32_t round = 0; ok; ++round) {
                const std::uint64_t at = static_cast<std::uint64_t>(round) * gridDim.x +
                                         (round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
                Item it{};
                if (at < items) {
                    const std::uint32_t r = static_cast<std::uint32_t>(at) / p.kv_heads;
                    const std::uint32_t kvh = static_cast<std::uint32_t>(at) % p.kv_heads;
                    it = sorted ? sorted_item(p, held, r, levels, kvh) : plain_item(p, r, kvh);
                    if (it.left == 0) continue;
                } else if (static_cast<std::uint64_t>(round) * gridDim.x < items) {
                    continue;  // the last round is not full
                }
                if (lane == 0) {
                    const std::uint32_t s = sent % kItems;
                    ok = sent < kItems || wait_or_abort(&item_empty[s], (sent / kItems - 1) & 1u, abort_flag);
                    if (ok) {
                        ring[s] = it;
                        arrive(&item_full[s]);
                    }
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
                ++sent;
                if (it.left == 0) break;
                const std::uint32_t tiles = it.tiles();
                if (tiles == 0 || !ok) continue;
                if (lane == 0) {
                    ok = n == 0 || wait_or_abort(q_empty, (n - 1) & 1u, abort_flag);
                    if (ok) {
                        const std::uint32_t box = p.tile_tokens * p.group * 128;
                        mbar_arrive_expect_tx(q_full, ((it.n[0] > 0) + (it.n[1] > 0)) * (HD / 64) * box);
#pragma unroll
                        for (int m = 0; m < 2; ++m)
                            for (int h = 0; h < HD / 64 && it.n[m] > 0; ++h)
                                tma_load_3d(base + L::kQ + m * L::kTile + h * L::kHalf, &map_q, 64 * h,
                                            static_cast<int>(it.kvh * p.group),
                                            static_cast<int>(it.q0 + m * p.tile_tokens), smem_u32(q_full));
                    }
                    for (std::uint32_t j = 0; ok && j < tiles; ++j) {
                        const std::uint32_t t = c + j, s = t % kKV, ph = (t / kKV - 1) & 1u;
                        const int row = static_cast<int>(it.k0 + j * kBN);
                        if (t >= kKV && !wait_or_abort(&k_empty[s], ph, abort_flag)) ok = false;
                        if (!ok) break;
                        mbar_arrive_expect_tx(&k_full[s], L::kTile);
                        for (int h = 0; h < HD / 64; ++h)
                            tma_load_3d(base + L::kK + s * L::kTile + h * L::kHalf, &map_k, 64 * h,
                                        static_cast<int>(it.kvh), row, smem_u32(&k_full[s]));
                        if (t >= kKV && !wait_or_abort(&v_empty[s], ph, abort_flag)) ok = false;
                        if (!ok) break;
                        mbar_arrive_expect_tx(&v_full[s], L::kTile);
                        for (int h = 0; h < HD / 64; ++h)
                            tma_load_3d(base + L::kV + s * L::kTile + h * L::kHalf, &map_v, 64 * h,
                                        static_cast<int>(it.kvh), row, smem_u32(&v_full[s]));
                    }
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
                c += tiles;
                ++n;
            }
        } else if (warp == kMmaWarp) {
            // The whole warp walks the loops, on values that the compiler knows to
            // be uniform, and one elected lane issues: operands then come from
            // uniform registers (moving each to one cost 100 cycles an MMA).
            const std::uint32_t tm = __reduce_max_sync(0xffffffffu, tmem);
            std::uint32_t c = 0, n = 0, clean = 0;
            // per query tile: items with any tiles, and whether the last one's
            // epilogue has yet to be waited for; and the passes so far
            std::uint32_t outs[2] = {0, 0}, passed = 0;
            bool unread[2] = {false, false};
            const auto wait = [&](std::uint64_t* bar, std::uint32_t parity) {
                return __all_sync(0xffffffffu, wait_or_abort(bar, parity, abort_flag)) != 0;
            };
            bool ok = true;
            for (std::uint32_t i = 0; ok; ++i) {
                const Item it = item_at(i);
                if (it.left == 0) break;
                const std::uint32_t n0 = __reduce_max_sync(0xffffffffu, it.n[0]);
                const std::uint32_t n1 = __reduce_max_sync(0xffffffffu, it.n[1]);
                const std::uint32_t masked = __reduce_max_sync(0xffffffffu, it.masked);
                const std::uint32_t tiles = max(n0, n1);
                if (tiles == 0) continue;
                // The item's passes in order: pass x is tile j of query tile m, tile 0
                // of both, tile 1 of both, and so on (query tile 1 attends as many
                // tiles as 0 or more, or none).  Its S is in buffer (passed + x) % kS.
                const std::uint32_t passes = n0 + n1, both = 2 * min(n0, n1);
                const auto m_of = [&](std::uint32_t x) { return x < both ? static_cast<int>(x & 1) : n1 > n0; };
                const auto j_of = [&](std::uint32_t x) { return x < both ? x / 2 : x - both / 2; };
                const auto wait_k = [&](std::uint32_t j) {
                    const std::uint32_t t = c + j;
                    return wait(&k_full[t % kKV], (t / kKV) & 1u);
                };
                const auto issue_s = [&](std::uint32_t x) {  // then what its last use frees
                    const int m = m_of(x);
                    const std::uint32_t j = j_of(x), s = (c + j) % kKV, buf = (passed + x) % L::kS;
                    const std::uint64_t ad = gemm::smem_desc_sw128(base + L::kQ + m * L::kTile);
                    const std::uint64_t bd = gemm::smem_desc_sw128(base + L::kK + s * L::kTile);
                    const bool last = m == 1 || j >= n1;
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < HD / 16; ++k) {
                            constexpr std::uint32_t kStep = 32 >> 4, kNext = L::kHalf >> 4;
                            const std::uint32_t at = k / 4 * kNext + k % 4 * kStep;
                            umma_f16_ss(tm + 128u * buf, ad + at, bd + at, kIdescS, k != 0 ? 1u : 0u);
                        }
                        gemm::umma_commit(smem_u32(&s_full[m * L::kS + buf]));
                        if (last) gemm::umma_commit(smem_u32(&k_empty[s]));
                        if (x + 1 == passes) gemm::umma_commit(smem_u32(q_empty));
                    }
                    __syncwarp();
                };
                ok = wait(q_full, n & 1u);
                for (std::uint32_t x = 0; ok && x < L::kS && x < passes; ++x) {
                    ok = wait_k(j_of(x));
                    gemm::tc_fence_after();
                    if (ok) issue_s(x);
                }
                for (std::uint32_t x = 0; ok && x < passes; ++x) {
                    const int m = m_of(x);
                    const std::uint32_t j = j_of(x), t = c + j, s = t % kKV;
                    const std::uint32_t buf = (passed + x) % L::kS, phase = ((passed + x) / L::kS) & 1u;
                    if (m == 0 || j >= n0) {
                        // V tile j has landed, and is looked through where rows see it in
                        // part (its barriers go round with the tiles that are)
                        ok = wait(&v_full[s], (t / kKV) & 1u);
                        if (ok && j >= masked) {
                            ok = wait(&v_clean[clean % kKV], (clean / kKV) & 1u);
                            ++clean;
                        }
                    }
                    // the last O is read (of both query tiles, so that neither
                    // softmax group falls behind by more than an item)
                    if (x == 0) {
#pragma unroll
                        for (int y = 0; y < 2; ++y)
                            if (ok && unread[y]) {
                                ok = wait(&epi_done[y], (outs[y] - 1) & 1u);
                                unread[y] = false;
                            }
                    }
                    if (!ok) break;
                    const std::uint64_t vd = v_desc<HD>(base + L::kV + s * L::kTile);
                    const std::uint32_t p_col = tm + 128u * buf, o_col = tm + L::kColO + HD * m;
                    const bool last = m == 1 || j >= n1;
                    // P V in halves, the first while the second half of P is computed
#pragma unroll
                    for (int half = 0; half < 2 && ok; ++half) {
                        ok = wait(half ? &p_ready[buf] : &p_half[buf], phase);
                        gemm::tc_fence_after();
                        if (ok && elect_one()) {
#pragma unroll
                            for (int k = half * kBN / 32; k < (half + 1) * kBN / 32; ++k)
                                gemm::umma_f16_ta(o_col, p_col + k * 8, vd + k * (2048 >> 4), kIdescPV,
                                                  (j | k) != 0 ? 1u : 0u);
                            if (half) {
                                gemm::umma_commit(smem_u32(&o_done[m * L::kS + buf]));
                                if (last) gemm::umma_commit(smem_u32(&v_empty[s]));
                            }
                        }
                        __syncwarp();
                    }
                    if (ok && x + L::kS < passes) {  // into the buffer that this P leaves
                        ok = wait_k(j_of(x + L::kS));
                        gemm::tc_fence_after();
                        if (ok) issue_s(x + L::kS);
                    }
                }
                if (n0 > 0) ++outs[0], unread[0] = true;
                if (n1 > 0) ++outs[1], unread[1] = true;
                passed += passes;
                c += tiles;
                ++n;
            }
            // every issued MMA completes before the tensor memory is freed (commit
            // by the lane that issued)
            if (elect_one()) {
                gemm::umma_commit(smem_u32(drained));
                mbar_wait_bounded(drained, 0, &g_device_status);
            }
            __syncwarp();
        } else {
            std::uint32_t c = 0, n = 0, clean = 0;
            bool ok = true;
            const int me = threadIdx.x - 10 * 32;  // of 64
            for (std::uint32_t i = 0; ok; ++i) {
                const Item it = item_at(i);
                if (it.left == 0) break;
                const std::uint32_t tiles = it.tiles();
                if (tiles == 0) continue;
                volatile std::uint32_t* flag = not_finite + n % kFlags * kCleanWarps + (warp - 10);
                if (lane == 0) *flag = 0u;
                for (std::uint32_t j = 0; ok && j < tiles; ++j) {
                    const std::uint32_t t = c + j, s = t % kKV;
                    ok = __all_sync(0xffffffffu, wait_or_abort(&v_full[s], (t / kKV) & 1u, abort_flag));
                    if (!ok) break;
                    if (j >= it.masked) {
                        uint4* tile = reinterpret_cast<uint4*>(smem + L::kV + s * L::kTile);
                        std::uint32_t bad = 0;  // an exponent of all ones carries into bit 15
#pragma unroll 4
                        for (int x = me; x < L::kTile / 16; x += 32 * kCleanWarps) {
                            const uint4 v = tile[x];
                            bad |= ((v.x & 0x7c007c00u) + 0x04000400u) | ((v.y & 0x7c007c00u) + 0x04000400u) |
                                   ((v.z & 0x7c007c00u) + 0x04000400u) | ((v.w & 0x7c007c00u) + 0x04000400u);
                        }
                        if (__any_sync(0xffffffffu, (bad & 0x80008000u) != 0)) {
                            // 16-byte chunk x belongs to row x / 8 of its half tile
                            const std::uint32_t rows = it.nk - j * kBN;  // of the sequence
                            bool found = false;
                            for (int x = me; x < L::kTile / 16; x += 32 * kCleanWarps) {
                                const uint4 v = tile[x];
                                std::uint32_t w[4] = {v.x, v.y, v.z, v.w};
                                bool any = false;
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    if ((w[e] & 0x7c00u) == 0x7c00u) w[e] &= 0xffff0000u, any = true;
                                    if ((w[e] & 0x7c000000u) == 0x7c000000u) w[e] &= 0x0000ffffu, any = true;
                                }
                                if (any) tile[x] = make_uint4(w[0], w[1], w[2], w[3]);
                                found |= any && static_cast<std::uint32_t>(x / 8 % kBN) < rows;
                            }
                            fence_proxy_async_smem();
                            if (found) *flag = 1u;
                        }
                        __syncwarp();
                        if (lane == 0) arrive(&v_clean[clean % kKV]);
                        ++clean;
                    }
                    if (lane == 0) arrive(&v_empty[s]);
                }
                c += tiles;
                ++n;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        // softmax: warps 4 m .. 4 m + 3 take query tile m, one thread per row
        const int m = warp / 4;
        const int r = 32 * (warp % 4) + lane;
        const std::uint32_t row_tmem = tmem + (static_cast<std::uint32_t>(32 * (warp % 4)) << 16);
        const std::uint32_t o_col = row_tmem + L::kColO + HD * m;
        const std::uint32_t tok = r / p.group, head = r % p.group;
        const float sc = p.scale_log2;
        std::uint32_t passed = 0, n = 0;  // softmax passes (of both query tiles) and items so far
        std::uint32_t seen = 0;           // parity of this query tile's passes on each S buffer
        bool ok = true;
        for (std::uint32_t i = 0;; ++i) {
            const Item it = item_at(i);
            if (it.left == 0) break;
            const std::uint32_t token = m * p.tile_tokens + tok;  // from the item's first
            const bool mine = tok < p.tile_tokens && token < it.left;
            const std::int32_t limit = it.pos0 + static_cast<std::int32_t>(token);  // its position
            // the least position of the warp's rows
            const std::int32_t least = it.pos0 + static_cast<std::int32_t>(
                m * p.tile_tokens + 32u * (warp % 4) / p.group);
            const std::uint32_t tiles = m ? it.n[1] : it.n[0];
            float mx_ref = -INFINITY, l = 0.f;
            float neg = 0.f;    // what the scaled scores get added
            bool vast = false;  // the reference is subtracted from the scores
            // tile j of this query tile is pass number pass_of(j), as the products are
            // issued.  A buffer's S and O barriers are this query tile's own: their
            // phases count its passes there, so a group that lags behind the other,
            // or has no rows for some items, does not lose count.
            const auto pass_of = [&](std::uint32_t j) {
                return passed + min(j, it.n[0]) + min(j, it.n[1]) + (m == 1 && j < it.n[0] ? 1u : 0u);
            };
            const auto wait_own = [&](std::uint64_t* bar, std::uint32_t b, std::uint32_t parity) {
                return __all_sync(0xffffffffu, wait_or_abort(bar + m * L::kS + b, parity, abort_flag)) != 0;
            };
            std::uint32_t last_buf = 0, last_parity = 0;  // the last pass's
            for (std::uint32_t j = 0; j < tiles && ok; ++j) {
                const std::uint32_t x = pass_of(j), buf = x % L::kS, s_col = row_tmem + 128u * buf;
                const std::uint32_t parity = seen >> buf & 1u;
                seen ^= 1u << buf;
                ok = wait_own(s_full, buf, parity);
                if (!ok) break;
                gemm::tc_fence_after();
                std::uint32_t v[4][32];
#pragma unroll
                for (int cc = 0; cc < 4; ++cc) tmem_ld32_nowait(s_col + 32 * cc, v[cc]);
                tmem_wait_ld();
                // causal mask, only in the 32 columns where the warp's rows differ
                // from all or nothing; the scale is positive, so the maximum of the
                // raw scores gives that of the scaled ones
                const std::int32_t kbase = static_cast<std::int32_t>(j * kBN);
                if (kbase + kBN - 1 > least) {
#pragma unroll
                    for (int cc = 0; cc < 4; ++cc) {
                        const std::int32_t cols = limit - (kbase + 32 * cc) + 1;  // attended of these
                        if (least - (kbase + 32 * cc) + 1 >= 32) continue;
                        const std::uint32_t bits = cols >= 32 ? 0xffffffffu : cols <= 0 ? 0u : (1u << cols) - 1u;
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!(bits >> e & 1u)) v[cc][e] = __float_as_uint(-INFINITY);
                    }
                }
                float mx8[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) mx8[e] = -INFINITY;
#pragma unroll
                for (int cc = 0; cc < 4; ++cc)
#pragma unroll
                    for (int e = 0; e < 32; e += 2)
                        mx8[(e / 2) % 8] = max3f(mx8[(e / 2) % 8], __uint_as_float(v[cc][e]),
                                                 __uint_as_float(v[cc][e + 1]));
                const float mx = max3f(max3f(mx8[0], mx8[1], mx8[2]), max3f(mx8[3], mx8[4], mx8[5]),
                                       fmaxf(mx8[6], mx8[7]));
                // the reference moves only when a score passes it by more than 8;
                // -infinity while the row has seen nothing
                const float mnew = fmaxf(mx_ref, mx);
                const bool grow = (mnew - mx_ref) * sc > 8.f;  // false while both are -inf (NaN)
                if (__any_sync(0xffffffffu, grow || vast)) {
                    float alpha = 1.f;
                    if (grow) {
                        alpha = ex2f((mx_ref - mnew) * sc);  // 0 from -infinity
                        mx_ref = mnew;
                        l *= alpha;
                        vast = fabsf(mx_ref) * sc > kVast;
                        neg = vast ? kShift : fmaf(-mx_ref, sc, kShift);
                    }
                    // (a row's own arithmetic, whatever the others of its warp hold)
                    if (__any_sync(0xffffffffu, vast)) {
                        const float from = vast ? mx_ref : 0.f;
#pragma unroll
                        for (int cc = 0; cc < 4; ++cc)
#pragma unroll
                            for (int e = 0; e < 32; ++e) v[cc][e] = __float_as_uint(__uint_as_float(v[cc][e]) - from);
                    }
                    if (j > 0) {
                        // the previous P V is complete before O moves
                        ok = wait_own(o_done, last_buf, last_parity);
                        if (!ok) break;
                        gemm::tc_fence_after();
#pragma unroll
                        for (int cc = 0; cc < HD / 16; ++cc) {
                            std::uint32_t o[16];
                            tmem_ld16(o_col + 16 * cc, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                            tmem_st16(o_col + 16 * cc, o);
                        }
                    }
                }
                const std::uint64_t sc2 = attnp::pack_f32x2(sc, sc), neg2 = attnp::pack_f32x2(neg, neg);
                std::uint64_t acc2[2] = {0, 0};
                // P of 32 columns at a time; the first P V steps start on the first
                // half of P while the second is computed
#pragma unroll
                for (int cc = 0; cc < 4; ++cc) {
                    std::uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        float xa, xb;
                        attnp::unpack_f32x2(attnp::fma_f32x2(attnp::pack_f32x2(__uint_as_float(v[cc][e]),
                                                                               __uint_as_float(v[cc][e + 1])),
                                                             sc2, neg2),
                                            xa, xb);
                        const float a = ex2f(xa), b = ex2f(xb);
                        acc2[e / 2 % 2] = attnp::add_f32x2(acc2[e / 2 % 2], attnp::pack_f32x2(a, b));
                        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(pk[e / 2]) : "f"(b), "f"(a));
                    }
                    if (cc == 2) {  // the stores of the first half have landed meanwhile
                        tmem_wait_st();
                        gemm::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) arrive(&p_half[buf]);
                    }
                    tmem_st16(s_col + 16 * cc, pk);
                }
                tmem_wait_st();
                gemm::tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive(&p_ready[buf]);
                float l0, l1, l2, l3;
                attnp::unpack_f32x2(acc2[0], l0, l1);
                attnp::unpack_f32x2(acc2[1], l2, l3);
                l += (l0 + l1) + (l2 + l3);
                last_buf = buf, last_parity = parity;
            }
            // O / sum; rows before the first position have no sum and get zeros
            if (it.tiles() > 0) ++n;
            if (tiles > 0 && ok) ok = wait_own(o_done, last_buf, last_parity);
            passed += it.n[0] + it.n[1];
            if (ok) {
                gemm::tc_fence_after();
                const bool some = tiles > 0 && limit >= 0;
                const float inv = some ? 1.f / l : 0.f;
                const volatile std::uint32_t* flags = not_finite + (n - 1) % kFlags * kCleanWarps;
                const bool add = some && (flags[0] | flags[1]) != 0u;
                __half* dst = p.out + (static_cast<std::uint64_t>(it.q0 + token) * p.q_heads +
                                       it.kvh * p.group + head) * HD;
#pragma unroll 1
                for (int cc = 0; cc < HD / 32; ++cc) {
                    __syncwarp();
                    std::uint32_t o[32];
                    if (tiles > 0) {
                        tmem_ld32_nowait(o_col + 32 * cc, o);
                        tmem_wait_ld();
                    }
                    if (!mine) continue;
                    if (add) {
                        // what warps 10 and 11 took out of the V tiles that this row attends
                        for (std::uint32_t pos = it.masked * kBN; pos <= static_cast<std::uint32_t>(limit); ++pos) {
                            const __half* src = p.v + (static_cast<std::uint64_t>(it.k0 + pos) * p.kv_heads + it.kvh) * HD + 32 * cc;
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                const float x = __half2float(src[e]);
                                if (!isfinite(x)) o[e] = __float_as_uint(__uint_as_float(o[e]) + x);
                            }
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        std::uint32_t w[4];
#pragma unroll
                        for (int e2 = 0; e2 < 4; ++e2) {
                            const float x0 = some ? __uint_as_float(o[e + 2 * e2]) * inv : 0.f;
                            const float x1 = some ? __uint_as_float(o[e + 2 * e2 + 1]) * inv : 0.f;
                            asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[e2]) : "f"(x1), "f"(x0));
                        }
                        *reinterpret_cast<uint4*>(dst + 32 * cc + e) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                gemm::tc_fence_before();
                __syncwarp();
                if (lane == 0 && tiles > 0) arrive(&epi_done[m]);  // O may be overwritten
            }
        }
    }
    gemm::tc_fence_before();
    __syncthreads();
    gemm::tc_fence_after();
    if (warp == kMmaWarp) gemm::tmem_dealloc(tmem, kTmemCols);
    if (*abort_flag) let_copies_land();
}

// [rows, heads, HD] f16 in boxes of `tokens` rows x `group` heads x 64; rows
// past the last read zeros.
inline int make_map(CUtensorMap* map, const void* ptr, std::uint64_t rows, std::uint64_t heads,
                    std::uint32_t head_dim, std::uint32_t group, std::uint32_t tokens) {
    auto encode = gemm::encode_fn();
    if (encode == nullptr) return static_cast<int>(cudaErrorNotSupported);
    const cuuint64_t dims[3] = {head_dim, heads, rows < 1 ? 1 : rows};
    const cuuint64_t strides[2] = {head_dim * 2ull, heads * head_dim * 2ull};
    const cuuint32_t box[3] = {64, group, tokens};
    const cuuint32_t estr[3] = {1, 1, 1};
    if (encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(ptr), dims, strides, box,
               estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return kInvalidValue;
    return kSuccess;
}

template <int HD>
int launch(const Params& p, const void* q, const void* k, cudaStream_t stream) {
    CUtensorMap map_q{}, map_k{}, map_v{};
    int st = make_map(&map_q, q, p.tokens, p.q_heads, HD, p.group, p.tile_tokens);
    if (st == kSuccess) st = make_map(&map_k, k, p.kv_tokens, p.kv_heads, HD, 1, kBN);
    if (st == kSuccess) st = make_map(&map_v, p.v, p.kv_tokens, p.kv_heads, HD, 1, kBN);
    if (st != kSuccess) return st;
    static std::atomic<std::uint64_t> smem_done{0};
    st = ensure_dynamic_smem(packed_kernel<HD>, Smem<HD>::kBytes, smem_done);
    if (st != kSuccess) return st;
    // The register split is exact for a launch at kLaunchRegs a thread; a build
    // that allocated another count is never launched.
    static std::atomic<int> regs_checked{0};
    if (regs_checked.load(std::memory_order_acquire) == 0) {
        cudaFuncAttributes fa{};
        const cudaError_t ea = cudaFuncGetAttributes(&fa, packed_kernel<HD>);
        if (ea != cudaSuccess) return static_cast<int>(ea);
        if (fa.numRegs != kLaunchRegs) return kInvalidConfiguration;
        regs_checked.store(1, std::memory_order_release);
    }
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return static_cast<int>(e);
    // (at most; how many there are is known on the device)
    const std::uint64_t items = (static_cast<std::uint64_t>(p.tokens) / (2 * p.tile_tokens) + p.batch) * p.kv_heads;
    if (items > 0x7fffffffull) return kInvalidValue;
    const unsigned grid = static_cast<unsigned>(items < static_cast<std::uint64_t>(sms) ? items : sms);
    return launch_pdl_smem(packed_kernel<HD>, dim3(grid), dim3(kThreads), Smem<HD>::kBytes, stream,
                           map_q, map_k, map_v, p);
}

}  // namespace attnv
}  // namespace mote

extern "C" int mote_cuda_gqa_attention_packed_f16(const void* q, const void* k, const void* v,
                                                  const void* q_starts, const void* kv_starts,
                                                  void* out, uint64_t tokens, uint64_t kv_tokens,
                                                  uint64_t batch, uint64_t q_heads,
                                                  uint64_t kv_heads, uint64_t head_dim,
                                                  float scale, void* stream) {
    using namespace mote;
    if (q == nullptr || k == nullptr || v == nullptr || q_starts == nullptr ||
        kv_starts == nullptr || out == nullptr || stream == nullptr)
        return kInvalidValue;
    if ((head_dim != 64 && head_dim != 128) || kv_heads == 0 || q_heads % kv_heads != 0 ||
        q_heads > 65535 || q_heads / kv_heads > 128 || batch > (1u << 20) ||
        tokens > 0x7fffffffull || kv_tokens > 0x7fffffffull || !std::isfinite(scale) ||
        !(scale > 0.f) || !kvq8::aligned16({q, k, v, out}) ||
        !kvq8::aligned4({q_starts, kv_starts}))
        return kInvalidValue;
    if (tokens == 0 || batch == 0 || q_heads == 0) return kSuccess;
    attnv::Params p{};
    p.q_starts = static_cast<const std::int32_t*>(q_starts);
    p.kv_starts = static_cast<const std::int32_t*>(kv_starts);
    p.v = static_cast<const __half*>(v);
    p.out = static_cast<__half*>(out);
    p.tokens = static_cast<std::uint32_t>(tokens);
    p.kv_tokens = static_cast<std::uint32_t>(kv_tokens);
    p.batch = static_cast<std::uint32_t>(batch);
    p.q_heads = static_cast<std::uint32_t>(q_heads);
    p.kv_heads = static_cast<std::uint32_t>(kv_heads);
    p.group = static_cast<std::uint32_t>(q_heads / kv_heads);
    p.tile_tokens = attnv::kBM / p.group;
    p.scale_log2 = scale * 1.4426950408889634f;
    const auto s = static_cast<cudaStream_t>(stream);
    return head_dim == 64 ? attnv::launch<64>(p, q, k, s) : attnv::launch<128>(p, q, k, s);
}

// Attention of new tokens over a paged f16 cache (attention_paged.cu), for the
// sequences with more query rows than the few-row kernel takes: chunks of prompts,
// on the tcgen05 tensor cores.
//
// A query tile is 128 rows: floor(128 / g) tokens of one sequence times the g query
// heads of one KV head (one TMA box of q).  A pair of consecutive query tiles shares
// every K/V tile of 128 positions, which TMA puts together from the pages (boxes of
// the largest power of two of rows that a block holds, 16 to 128 of them; the block
// numbers of the next tile are read while this one's stage is waited for).  Within a
// CTA
// * warp 8 walks the work and loads Q, K and V (TMA, 128-byte swizzle);
// * warps 9 and 10 issue the products, each for its query tile m: S_m = Q_m K^T and
//   O_m += P_m V (P from tensor memory).  One warp for both had to take them in turn,
//   and an MMA costs its warp 30 to 60 cycles to issue: chunk of 2048 over 16384 at
//   head_dim 128 688 us, 633 with two (and turns, below);
// * warps 0-3 and 4-7 run the softmax of the two query tiles, one thread per row: the
//   maximum moves (and O_m is rescaled) only when a score passes it by more than 8 in
//   log2 units.  P is rounded to f16 (11 bits down to 2^-21 of the row's largest);
//   at head_dim 128 it lies over the first half of S, at 64 in columns of its own, so
//   that the next S is computed while P of this one still is;
// * warp 11 takes what is not finite out of V tiles that some row sees in part (later
//   positions, and the rows of a page behind the last position): 0 times an infinity
//   or NaN would be NaN.  The rows that do attend such values add them at the end
//   (rare, from global memory).
// What bounds it: at head_dim 128 the chain S -> maximum -> exponentials -> P V of two
// query tiles, under the power cap in long runs (chunk of 2048 over 16384: 583 GFLOP in 633
// us, 0.57 of the measured tensor rate; 580 on a cooler GPU); at 64 the same chain and the
// exp2 unit (six chunks of 300 to 1024 over up to 2500: 104 us, exp2 49 % of the cycles,
// tensor pipe 24 %).
// Every wait is bounded; an expired wait aborts the CTA, which waits for its issued
// MMAs (bounded) and frees its tensor memory.  No load uses cluster multicast.
//
// The work is a line of positions (attention_paged.cu).  Each CTA takes an
// equal share of it, found on the device from sums of arithmetic series, so one chunk
// over a long cache fills the GPU as well as a batch of prompts does.  A pair that lies in several
// CTAs leaves unnormalised parts, which join_kernel adds up in order.
#include "mote_common.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

namespace mote {
namespace attnpg {
namespace chunk {

using attnp::ex2f;
using attnp::max3f;
using attnp::tma_load_3d;
using attnp::tmem_ld32_nowait;
using attnp::tmem_wait_ld;
using attnp::tmem_wait_st;
using attnv::arrive;
using attnv::elect_one;
using attnv::kBM;
using attnv::kBN;
using attnv::kFlags;
using attnv::kItems;
using attnv::kLaunchRegs;
using attnv::kMmaWarp;
using attnv::kOtherRegs;
using attnv::kProducerWarp;
using attnv::kShift;
using attnv::kSoftmaxRegs;
using attnv::kThreads;
using attnv::kTmemCols;
using attnv::tmem_ld16;
using attnv::tmem_st16;
using attnv::v_desc;
using gemm::wait_or_abort;

constexpr int kMaxCtas = 192;
// The least share, in positions, and the least piece of a pair, in K/V tiles (1024 and 3:
// 8 sequences of 8000 with one token of 32 query heads on one KV head 30.5 us, 22.9 now;
// 16 of 4000 with 5 tokens 73.5 and 71.5).
constexpr std::uint64_t kLeast = 512;
constexpr std::uint32_t kMinTiles = 1;
// score * scale - reference is one fma with the rounded reference, off by up to 2^-24 of
// it; beyond this (log2 units) the reference is subtracted from the scores instead.  Equal
// scores meet under different references, where a row's moves and where its parts are
// joined: near 35000 their weights were up to 2^-8 apart (log2), at 1024 it is 2^-13.
constexpr float kVast = 1024.f;

// One MMA, issued by the lane whose `lead` is set; all lanes of the (converged) warp
// run through it, without a branch.
__device__ __forceinline__ void mma_ss(std::uint32_t lead, std::uint32_t d, std::uint64_t a, std::uint64_t b,
                                       std::uint32_t idesc, std::uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(lead)
        : "memory");
}
// ... with A in tensor memory.
__device__ __forceinline__ void mma_ts(std::uint32_t lead, std::uint32_t d, std::uint32_t a, std::uint64_t b,
                                       std::uint32_t idesc, std::uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(lead)
        : "memory");
}
// An arrival on `bar` when the MMAs that the lane has issued so far are complete.
__device__ __forceinline__ void commit(std::uint32_t lead, std::uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
        "r"(lead)
        : "memory");
}

// Two query tiles of one sequence and KV head, or some of their K/V tiles.
struct Item {
    std::uint32_t left;    // the sequence's tokens from the first on; 0: no more items
    std::uint32_t kvh, b;
    std::uint32_t q0;      // row of the first token in q
    std::int32_t pos0;     // its position
    std::uint32_t nk;      // the sequence's positions
    std::uint32_t t0;      // the first K/V tile
    std::uint32_t n[2];    // K/V tiles from there on that each query tile attends
    std::uint32_t masked;  // the first of them that some row sees in part
    std::int32_t part;     // where the result goes in part; < 0: to out
    __device__ __forceinline__ std::uint32_t tiles() const { return max(n[0], n[1]); }
};

// Parts of a pair that join_kernel adds up: those of `count` CTAs from the one on
// whose number the entry has (0: none).
struct Join {
    std::uint32_t count, left, kvh, q0;
    std::int32_t pos0;
};

template <int HD>
struct Smem {
    static constexpr int kHalf = 128 * 128;           // 128 rows of 64 f16
    static constexpr int kTile = HD / 64 * kHalf;     // a Q, K or V tile
    static constexpr int kKV = HD == 64 ? 4 : 2;      // K and V stages
    // TMEM columns: S_m at 128 m, O_m, and at head_dim 64 P_m; at 128 P_m over S_m
    static constexpr std::uint32_t kColO = 256;
    static constexpr std::uint32_t kColP = HD == 64 ? kColO + 2 * HD : 0;
    static constexpr std::uint32_t kPStep = HD == 64 ? 64 : 128;
    static constexpr int kQ = 0;                      // [2] query tiles
    static constexpr int kK = kQ + 2 * kTile;
    static constexpr int kV = kK + kKV * kTile;
    static constexpr int kBar = kV + kKV * kTile;
    // q_full, q_empty, k_full, k_empty, v_full, v_empty, v_clean [kKV], s_full,
    // s_free, p_half, p_ready, o_done, epi_done, drained [2], item_full, item_empty [kItems]
    static constexpr int kNumBars = 2 + 5 * kKV + 7 * 2 + 2 * kItems;
    static constexpr int kTmemSlot = kBar + kNumBars * 8;
    static constexpr int kAbort = kTmemSlot + 4;
    static constexpr int kFlag = kAbort + 4;          // [kFlags]
    static constexpr int kItem = kFlag + 4 * kFlags;  // [kItems]
    static constexpr int kShare = (kItem + kItems * static_cast<int>(sizeof(Item)) + 7) / 8 * 8;  // first sequence, its begin
    static constexpr int kScan = kShare + 2 * 8;      // [warp][3] sums
    static constexpr int kTurn = kScan + kThreads / 32 * 24;  // [query tile][warp] passes whose exponentials are done
    static constexpr int kUsed = kTurn + 8 * 4 + 1008;  // + alignment slack
    // one CTA per SM: its 512 TMEM columns never wait for another's
    static constexpr int kBytes = kUsed > 120 * 1024 ? kUsed : 120 * 1024;
    static_assert(kBytes <= 232448, "shared memory");
};

struct ChunkParams {
    Params p;
    std::uint32_t box;          // rows of a K or V box
    Join* joins;                // [CTAs]
    float* parts;               // [2 CTAs][HD / 4][256][4], then [256][2]: maxima and sums
};

template <int HD>
constexpr std::uint64_t kPart = 256ull * (HD + 2);

// Of a pair of n K/V tiles, those before position x of it.
__device__ __forceinline__ std::uint32_t cut(std::uint64_t x, std::uint32_t n) {
    const std::uint32_t t = static_cast<std::uint32_t>((x + kBN / 2) / kBN);
    if (t < kMinTiles) return 0;
    return t + kMinTiles > n ? n : t;
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
    chunk_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, const ChunkParams c) {
    const Params& p = c.p;
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
    std::uint64_t* s_free = s_full + 2;
    std::uint64_t* p_half = s_free + 2;
    std::uint64_t* p_ready = p_half + 2;
    std::uint64_t* o_done = p_ready + 2;
    std::uint64_t* epi_done = o_done + 2;
    std::uint64_t* drained = epi_done + 2;
    std::uint64_t* item_full = drained + 2;
    std::uint64_t* item_empty = item_full + kItems;
    Item* ring = reinterpret_cast<Item*>(smem + L::kItem);
    volatile std::uint32_t* tmem_slot = reinterpret_cast<volatile std::uint32_t*>(smem + L::kTmemSlot);
    volatile std::uint32_t* abort_flag = reinterpret_cast<volatile std::uint32_t*>(smem + L::kAbort);
    volatile std::uint32_t* not_finite = reinterpret_cast<volatile std::uint32_t*>(smem + L::kFlag);

    volatile std::uint32_t* turn = reinterpret_cast<volatile std::uint32_t*>(smem + L::kTurn);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        mbar_init(q_empty, 2);
        for (int s = 0; s < kKV; ++s) {
            mbar_init(&k_full[s], 1);
            mbar_init(&k_empty[s], 2);
            mbar_init(&v_full[s], 1);
            mbar_init(&v_empty[s], 3);  // both P V, and warp 11 keeps step
            mbar_init(&v_clean[s], 1);
        }
        for (int m = 0; m < 2; ++m) {
            mbar_init(&s_full[m], 1);
            mbar_init(&s_free[m], 4);
            mbar_init(&p_half[m], 4);
            mbar_init(&p_ready[m], 4);
            mbar_init(&o_done[m], 1);
            mbar_init(&epi_done[m], 4);
            mbar_init(&drained[m], 1);
        }
        for (int s = 0; s < kItems; ++s) {
            mbar_init(&item_full[s], 1);
            mbar_init(&item_empty[s], 11);  // every warp but the producer
        }
        *abort_flag = 0u;
        for (int i = 0; i < 8; ++i) turn[i] = 0u;
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
    // beside the other kernel, which has waited, the wait comes at the end
    if (!p.shares) pdl_wait();

    // ---- the CTA's share of the line ---------------------------------------
    // first sequence (~0: none), length of a share, where the sequence begins; by the
    // producer alone for up to 32 sequences, by all otherwise (8 tokens over 30000 40.2 us,
    // 41.0 by all)
    const std::uint32_t batch = p.c.batch;
    std::uint64_t first_b = ~0ull, per = 0, first_begin = 0;
    const auto scan_up = [&](std::uint64_t x) {  // inclusive, over the warp
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const std::uint64_t y = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += y;
        }
        return x;
    };
    // this kernel's work of sequence b, its cost and the other's work
    const auto work_of = [&](std::uint32_t b, std::uint64_t& cost, std::uint64_t& units) -> std::uint64_t {
        if (b >= batch) return 0;
        const Seq s = sequence(p, b);
        if (p.shares) {
            cost += cost_of(p, s);
            const std::uint32_t n = few::units_of<HD>(few::few_part(p, s));
            units += n == 0 ? 0ull : (static_cast<std::uint64_t>(n) + few::kSplitRowCost) * p.c.kv_heads;
        }
        return Pairs(p, s).all() * p.c.kv_heads;
    };
    // sets `per`; whether the CTA has a share
    const auto divide = [&](std::uint64_t total, std::uint64_t cost, std::uint64_t units) {
        const std::uint32_t ctas = p.shares ? gridDim.x - few_ctas<HD>(gridDim.x, units, cost) : gridDim.x;
        if (blockIdx.x >= ctas) return false;
        per = share_of(total, ctas);
        if (per < kLeast) per = kLeast;
        return true;
    };
    if (__builtin_expect(batch <= 32, 1)) {
        if (warp == kProducerWarp) {
            std::uint64_t cost = 0, units = 0;
            const std::uint64_t mine = work_of(lane, cost, units), incl = scan_up(mine);
            if (p.shares) {
                cost = __shfl_sync(0xffffffffu, scan_up(cost), 31);
                units = __shfl_sync(0xffffffffu, scan_up(units), 31);
            }
            if (divide(__shfl_sync(0xffffffffu, incl, 31), cost, units)) {
                const std::uint64_t at = per * blockIdx.x;
                const unsigned here = __ballot_sync(0xffffffffu, incl - mine <= at && at < incl);
                if (here != 0) {
                    first_b = __ffs(here) - 1;
                    first_begin = __shfl_sync(0xffffffffu, incl - mine, static_cast<int>(first_b));
                }
            }
        }
    } else {
        volatile std::uint64_t* share = reinterpret_cast<volatile std::uint64_t*>(smem + L::kShare);
        volatile std::uint64_t* scan = reinterpret_cast<volatile std::uint64_t*>(smem + L::kScan);
        std::uint64_t sum = 0, cost = 0, units = 0;
        for (std::uint32_t b = threadIdx.x; b < batch; b += kThreads) sum += work_of(b, cost, units);
        sum = scan_up(sum), cost = scan_up(cost), units = scan_up(units);
        if (lane == 31) scan[3 * warp] = sum, scan[3 * warp + 1] = cost, scan[3 * warp + 2] = units;
        if (threadIdx.x == 0) share[0] = ~0ull;
        __syncthreads();
        std::uint64_t total = 0, all_cost = 0, all_units = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) total += scan[3 * w], all_cost += scan[3 * w + 1], all_units += scan[3 * w + 2];
        __syncthreads();
        if (divide(total, all_cost, all_units)) {
            const std::uint64_t at = per * blockIdx.x;
            std::uint64_t before = 0;
            for (std::uint32_t base = 0; base < batch && before <= at; base += kThreads) {
                std::uint64_t cost = 0, units = 0;
                const std::uint64_t mine = work_of(base + threadIdx.x, cost, units), incl = scan_up(mine);
                if (lane == 31) scan[warp] = incl;
                __syncthreads();
                std::uint64_t lower = before;
#pragma unroll
                for (int w = 0; w < kThreads / 32; ++w) {
                    if (w < warp) lower += scan[w];
                    before += scan[w];
                }
                const std::uint64_t begin = lower + incl - mine;
                if (begin <= at && at < lower + incl) {
                    share[0] = base + threadIdx.x;
                    share[1] = begin;
                }
                __syncthreads();
            }
            first_b = share[0], first_begin = share[1];
        }
    }
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
            if (p.reports && blockIdx.x == gridDim.x - 1) report_bad(p, lane, 32);
            const std::uint64_t u0 = per * blockIdx.x, u1 = u0 + per;
            std::uint32_t kv = 0, n = 0, sent = 0;  // K/V tiles, items with any and items so far
            std::uint32_t joined = 0;               // pairs that begin here and end in another CTA
            bool ok = true;
            const auto send = [&](const Item& it) {
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
            };
            // boxes of a K or V tile: the lanes of the lower half load K's, the others V's
            const std::uint32_t half_box = lane % 16, sub = half_box / (HD / 64), dims = half_box % (HD / 64);
            const bool loads = sub < kBN / c.box;
            const auto load = [&](const Item& it) {
                const std::uint32_t tiles = it.tiles();
                // the block of this lane's box of tile j, read a tile ahead, and its row
                // in the cache (what is not there reads as zeros)
                const auto position = [&](std::uint32_t j) { return (it.t0 + j) * kBN + sub * c.box; };
                const auto block_of = [&](std::uint32_t j) {
                    if (!loads || position(j) >= it.nk || j >= tiles) return -1;
                    return fetch(p, p.tables + static_cast<std::uint64_t>(it.b) * p.c.max_blocks + position(j) / p.c.block_tokens);
                };
                const auto row_of = [&](std::uint32_t j, std::int32_t block) {
                    if (!loads || position(j) >= it.nk) return kNowhere;
                    if (block < 0 || static_cast<std::uint64_t>(block) >= p.c.num_blocks) {
                        atomicOr(&g_device_status, kDevIndexOutOfRange);
                        return kNowhere;
                    }
                    return static_cast<int>((static_cast<std::uint32_t>(block) * p.c.kv_heads + it.kvh) * p.c.block_tokens +
                                            position(j) % p.c.block_tokens);
                };
                std::int32_t block = block_of(0);
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
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
                for (std::uint32_t j = 0; ok && j < tiles; ++j) {
                    const std::uint32_t t = kv + j, s = t % kKV, ph = (t / kKV - 1) & 1u;
                    const std::int32_t next = block_of(j + 1);
                    const int row = row_of(j, block);
                    const std::uint32_t at = s * L::kTile + dims * L::kHalf + sub * c.box * 128;
                    if (t >= kKV) ok = __all_sync(0xffffffffu, wait_or_abort(&k_empty[s], ph, abort_flag));
                    if (!ok) break;
                    if (lane == 0) mbar_arrive_expect_tx(&k_full[s], L::kTile);
                    __syncwarp();
                    if (loads && lane < 16) tma_load_3d(base + L::kK + at, &map_k, 0, row, static_cast<int>(dims), smem_u32(&k_full[s]));
                    if (t >= kKV) ok = __all_sync(0xffffffffu, wait_or_abort(&v_empty[s], ph, abort_flag));
                    if (!ok) break;
                    if (lane == 0) mbar_arrive_expect_tx(&v_full[s], L::kTile);
                    __syncwarp();
                    if (loads && lane >= 16) tma_load_3d(base + L::kV + at, &map_v, 0, row, static_cast<int>(dims), smem_u32(&v_full[s]));
                    block = next;
                }
                kv += tiles;
                ++n;
            };
            if (first_b != ~0ull) {
                std::uint32_t b = static_cast<std::uint32_t>(first_b);
                Pairs x(p, sequence(p, b));
                // the pair that u0 lies in
                std::uint64_t begin = first_begin;
                std::uint32_t kvh = 0, i = 0;
                for (const std::uint64_t all = x.all(); begin + all <= u0; begin += all) ++kvh;
                for (std::uint32_t hi = x.count; hi - i > 1;) {
                    const std::uint32_t mid = (i + hi) / 2;
                    if (begin + x.before(mid) <= u0) i = mid; else hi = mid;
                }
                begin += x.before(i);
                while (ok && begin < u1) {
                    const std::uint64_t extent = x.extent(i);
                    const std::uint32_t reach = x.reach(i), tiles = (reach + kBN - 1) / kBN;
                    const std::uint32_t from = begin >= u0 ? 0u : cut(u0 - begin, tiles);
                    const std::uint32_t to = begin + extent <= u1 ? tiles : cut(u1 - begin, tiles);
                    // (a pair without positions, whose rows get zeros, is the CTA's in which it begins)
                    if (from < to || (tiles == 0 && begin >= u0)) {
                        Item it{};
                        it.left = x.s.n - i * x.span;
                        it.kvh = kvh;
                        it.b = b;
                        it.q0 = x.s.q0 + i * x.span;
                        it.nk = x.s.len;
                        it.pos0 = static_cast<std::int32_t>(x.s.len) - static_cast<std::int32_t>(it.left);
                        it.t0 = from;
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            const std::uint32_t first = m * p.tile_tokens;
                            const std::int32_t last = it.pos0 + static_cast<std::int32_t>(min(first + p.tile_tokens, it.left)) - 1;
                            const std::uint32_t whole = first >= it.left || last < 0 ? 0u : static_cast<std::uint32_t>(last) / kBN + 1;
                            it.n[m] = min(whole, to) - min(whole, from);
                        }
                        const std::uint32_t masked = static_cast<std::uint32_t>(max(it.pos0 + 1, 0)) / kBN;
                        it.masked = masked > from ? masked - from : 0u;
                        it.part = from == 0 && to == tiles ? -1 : static_cast<std::int32_t>(2 * blockIdx.x + (from == 0 ? 1 : 0));
                        if (from == 0 && to < tiles) {
                            // the last CTA that has some of it
                            std::uint32_t last = blockIdx.x;
                            while ((last + 1) * per < begin + extent) ++last;
                            if (cut(last * per - begin, tiles) == tiles) --last;
                            joined = last - blockIdx.x + 1;
                            if (lane == 0) c.joins[blockIdx.x] = Join{joined, it.left, kvh, it.q0, it.pos0};
                        }
                        send(it);
                        if (ok && it.tiles() > 0) load(it);
                    }
                    begin += extent;
                    if (++i < x.count) continue;
                    i = 0;
                    if (++kvh < p.c.kv_heads) continue;
                    kvh = 0;
                    // (one sequence after another, 0.33 us each, while the tensor cores wait:
                    // a chunk of 512 behind 400 single tokens 40 us, before them 148)
                    do {
                        if (++b >= p.c.batch) break;
                        x = Pairs(p, sequence(p, b));
                    } while (x.count == 0);
                    if (b >= p.c.batch) break;
                }
            }
            if (joined == 0 && lane == 0) c.joins[blockIdx.x] = Join{};
            if (ok) send(Item{});
        } else if (warp < kMmaWarp + 2) {
            // The whole warp walks the loops, on values that the compiler knows to be
            // uniform, and issues by predicate, without a branch.
            const int m = warp - kMmaWarp;
            const std::uint32_t tm = __reduce_max_sync(0xffffffffu, tmem);
            const std::uint32_t lead = elect_one() ? 1u : 0u;
            const std::uint32_t s_col = tm + 128u * m, o_col = tm + L::kColO + HD * m, p_col = tm + L::kColP + L::kPStep * m;
            const std::uint64_t qd = gemm::smem_desc_sw128(base + L::kQ + m * L::kTile);
            std::uint32_t kv = 0, n = 0, clean = 0, passes = 0, outs = 0;
            bool unread = false, ok = true;  // the last O has yet to be read
            const auto wait = [&](std::uint64_t* bar, std::uint32_t parity) {
                return __all_sync(0xffffffffu, wait_or_abort(bar, parity, abort_flag)) != 0;
            };
            for (std::uint32_t i = 0; ok; ++i) {
                const Item it = item_at(i);
                if (it.left == 0) break;
                const std::uint32_t mine = __reduce_max_sync(0xffffffffu, m ? it.n[1] : it.n[0]);
                const std::uint32_t tiles = __reduce_max_sync(0xffffffffu, it.tiles());
                const std::uint32_t masked = __reduce_max_sync(0xffffffffu, it.masked);
                if (tiles == 0) continue;
                const auto wait_k = [&](std::uint32_t j) {
                    const std::uint32_t t = kv + j;
                    return wait(&k_full[t % kKV], (t / kKV) & 1u);
                };
                const auto issue_s = [&](std::uint32_t j) {  // and then what its last use frees
                    const std::uint32_t s = (kv + j) % kKV;
                    const std::uint64_t kd = gemm::smem_desc_sw128(base + L::kK + s * L::kTile);
                    gemm::tc_fence_after();
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k) {
                        constexpr std::uint32_t kStep = 32 >> 4, kNext = L::kHalf >> 4;
                        const std::uint32_t at = k / 4 * kNext + k % 4 * kStep;
                        mma_ss(lead, s_col, qd + at, kd + at, kIdescS, k != 0 ? 1u : 0u);
                    }
                    commit(lead, &s_full[m]);
                    commit(lead, &k_empty[s]);
                    if (j + 1 == mine) commit(lead, q_empty);
                };
                const auto issue_pv = [&](std::uint64_t vd, std::uint32_t j, int half) {
                    gemm::tc_fence_after();
#pragma unroll
                    for (int k = 0; k < kBN / 32; ++k) {
                        const int step = half * (kBN / 32) + k;
                        mma_ts(lead, o_col, p_col + step * 8, vd + step * (2048 >> 4), kIdescPV, (j | step) != 0 ? 1u : 0u);
                    }
                };
                ok = wait(q_full, n & 1u);
                if (ok && mine == 0 && lane == 0) arrive(q_empty);
                if (ok && mine > 0) {
                    ok = wait_k(0);
                    if (ok) issue_s(0);
                }
                for (std::uint32_t j = 0; ok && j < tiles; ++j) {
                    const std::uint32_t t = kv + j, s = t % kKV;
                    if (j >= mine) {  // the other query tile's alone
                        ok = wait_k(j);
                        if (ok && lane == 0) arrive(&k_empty[s]);
                    }
                    // V tile j has landed, and is looked through where rows see it in part
                    // (its barriers go round with the tiles that are)
                    ok = ok && wait(&v_full[s], (t / kKV) & 1u);
                    if (ok && j >= masked) {
                        ok = wait(&v_clean[clean % kKV], (clean / kKV) & 1u);
                        ++clean;
                    }
                    if (j >= mine) {
                        if (ok && lane == 0) arrive(&v_empty[s]);
                        continue;
                    }
                    if (ok && j == 0 && unread) {
                        ok = wait(&epi_done[m], (outs - 1) & 1u);
                        unread = false;
                    }
                    const std::uint32_t phase = passes++ & 1u;
                    const std::uint64_t vd = v_desc<HD>(base + L::kV + s * L::kTile);
                    // P V in halves, the first while the second half of P is computed
                    if (HD == 64 && ok && j + 1 < mine) {  // S is read, P has columns of its own
                        ok = wait(&s_free[m], phase) && wait_k(j + 1);
                        if (ok) issue_s(j + 1);
                    }
                    ok = ok && wait(&p_half[m], phase);
                    if (ok) issue_pv(vd, j, 0);
                    ok = ok && wait(&p_ready[m], phase);
                    if (ok) {
                        issue_pv(vd, j, 1);
                        commit(lead, &o_done[m]);
                        commit(lead, &v_empty[s]);
                    }
                    if (HD == 128 && ok && j + 1 < mine) {  // into the columns that this P leaves
                        ok = wait_k(j + 1);
                        if (ok) issue_s(j + 1);
                    }
                }
                if (mine > 0) ++outs, unread = true;
                kv += tiles;
                ++n;
            }
            // every issued MMA completes before the tensor memory is freed (commit
            // by the lane that issued)
            commit(lead, &drained[m]);
            if (lead) mbar_wait_bounded(&drained[m], 0, &g_device_status);
            __syncwarp();
        } else {
            std::uint32_t kv = 0, n = 0, clean = 0;
            bool ok = true;
            for (std::uint32_t i = 0; ok; ++i) {
                const Item it = item_at(i);
                if (it.left == 0) break;
                const std::uint32_t tiles = it.tiles();
                if (tiles == 0) continue;
                volatile std::uint32_t* flag = not_finite + n % kFlags;
                if (lane == 0) *flag = 0u;
                for (std::uint32_t j = 0; ok && j < tiles; ++j) {
                    const std::uint32_t t = kv + j, s = t % kKV;
                    ok = __all_sync(0xffffffffu, wait_or_abort(&v_full[s], (t / kKV) & 1u, abort_flag));
                    if (!ok) break;
                    if (j >= it.masked) {
                        uint4* tile = reinterpret_cast<uint4*>(smem + L::kV + s * L::kTile);
                        std::uint32_t bad = 0;  // an exponent of all ones carries into bit 15
#pragma unroll 8
                        for (int x = lane; x < L::kTile / 16; x += 32) {
                            const uint4 v = tile[x];
                            bad |= ((v.x & 0x7c007c00u) + 0x04000400u) | ((v.y & 0x7c007c00u) + 0x04000400u) |
                                   ((v.z & 0x7c007c00u) + 0x04000400u) | ((v.w & 0x7c007c00u) + 0x04000400u);
                        }
                        if (__any_sync(0xffffffffu, (bad & 0x80008000u) != 0)) {
                            // 16-byte chunk x belongs to row x / 8 of its half tile
                            const std::uint32_t rows = it.nk - (it.t0 + j) * kBN;  // of the sequence
                            bool found = false;
                            for (int x = lane; x < L::kTile / 16; x += 32) {
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
                kv += tiles;
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
        const std::uint32_t s_col = row_tmem + 128u * m, p_col = row_tmem + L::kColP + L::kPStep * m;
        std::uint32_t passes = 0, theirs = 0, n = 0;  // of this query tile and of the other, and items with any so far
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
            const auto wait_own = [&](std::uint64_t* bar, std::uint32_t parity) {
                return __all_sync(0xffffffffu, wait_or_abort(bar + m, parity, abort_flag)) != 0;
            };
            for (std::uint32_t j = 0; j < tiles && ok; ++j) {
                const std::uint32_t phase = passes++ & 1u;
                ok = wait_own(s_full, phase);
                if (!ok) break;
                gemm::tc_fence_after();
                std::uint32_t v[4][32];
#pragma unroll
                for (int cc = 0; cc < 4; ++cc) tmem_ld32_nowait(s_col + 32 * cc, v[cc]);
                tmem_wait_ld();
                if (HD == 64) {  // the next S may come
                    gemm::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive(&s_free[m]);
                }
                // causal mask, only in the 32 columns where the warp's rows differ
                // from all or nothing; the scale is positive, so the maximum of the
                // raw scores gives that of the scaled ones
                const std::int32_t kbase = static_cast<std::int32_t>((it.t0 + j) * kBN);
                if (__builtin_expect(kbase + kBN - 1 > least, 0)) {
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
                if (__builtin_expect(__any_sync(0xffffffffu, grow || vast), 0)) {
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
                        ok = wait_own(o_done, phase ^ 1u);
                        if (!ok) break;
                        gemm::tc_fence_after();
#pragma unroll 2
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
                if (HD == 64 && j > 0) {  // the P V before has read P
                    ok = wait_own(o_done, phase ^ 1u);
                    if (!ok) break;
                    gemm::tc_fence_after();
                }
                // The exponentials of the two query tiles take turns, pass after pass: a
                // scheduler's two softmax warps would else share its exp2 unit evenly and
                // come out together, leaving it idle meanwhile.
                {
                    const std::uint32_t other = m ? it.n[0] : it.n[1];
                    const std::uint32_t want = theirs + min(j + (m ? 1u : 0u), other);
                    const volatile std::uint32_t* at = turn + 4 * (1 - m) + warp % 4;
                    if (static_cast<std::int32_t>(*at - want) < 0) {
                        const long long start = clock64();
                        while (static_cast<std::int32_t>(*at - want) < 0 && !*abort_flag)
                            if (clock64() - start > kWaitCycles) {
                                atomicOr(&g_device_status, kDevWaitTimeout);
                                *abort_flag = 1u;
                            }
                    }
                    __syncwarp();
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
                        if (lane == 0) arrive(&p_half[m]);
                    }
                    tmem_st16(p_col + 16 * cc, pk);
                    if (cc == 0) {
                        __syncwarp();
                        if (lane == 0) turn[4 * m + warp % 4] = passes;
                    }
                }
                tmem_wait_st();
                gemm::tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive(&p_ready[m]);
                float l0, l1, l2, l3;
                attnp::unpack_f32x2(acc2[0], l0, l1);
                attnp::unpack_f32x2(acc2[1], l2, l3);
                l += (l0 + l1) + (l2 + l3);
            }
            // O / sum; rows before the first position have no sum and get zeros
            if (it.tiles() > 0) ++n;
            theirs += m ? it.n[0] : it.n[1];
            if (tiles > 0 && ok) ok = wait_own(o_done, (passes - 1) & 1u);
            if (ok) {
                gemm::tc_fence_after();
                const bool some = tiles > 0 && limit >= 0;
                const float inv = some ? 1.f / l : 0.f;
                const volatile std::uint32_t* flags = not_finite + (n - 1) % kFlags;
                const bool add = some && *flags != 0u;
                __half* dst = p.out + (static_cast<std::uint64_t>(it.q0 + token) * p.q_heads +
                                       it.kvh * p.group + head) * HD;
                const std::uint32_t row = m * kBM + r;
                float4* part = reinterpret_cast<float4*>(c.parts + static_cast<std::uint64_t>(max(it.part, 0)) * kPart<HD>) + row;
                if (it.part >= 0)
                    *reinterpret_cast<float2*>(c.parts + static_cast<std::uint64_t>(it.part) * kPart<HD> + 256 * HD + 2 * row) =
                        make_float2(tiles > 0 ? mx_ref : -INFINITY, l);
#pragma unroll 1
                for (int cc = 0; cc < HD / 32; ++cc) {
                    __syncwarp();
                    std::uint32_t o[32];
                    if (tiles > 0) {
                        tmem_ld32_nowait(o_col + 32 * cc, o);
                        tmem_wait_ld();
                    }
                    if (!mine) continue;
                    if (__builtin_expect(add, 0)) {
                        // what warp 11 took out of the V tiles that this row attends
                        const std::uint32_t end = min(static_cast<std::uint32_t>(limit) + 1u, (it.t0 + tiles) * kBN);
                        for (std::uint32_t pos = (it.t0 + it.masked) * kBN; pos < end; ++pos) {
                            const std::int32_t block = fetch(p, p.tables + static_cast<std::uint64_t>(it.b) * p.c.max_blocks + pos / p.c.block_tokens);
                            if (block < 0 || static_cast<std::uint64_t>(block) >= p.c.num_blocks) continue;
                            const __half* src = p.v_cache + ((static_cast<std::uint64_t>(block) * p.c.kv_heads + it.kvh) * p.c.block_tokens +
                                                             pos % p.c.block_tokens) * HD + 32 * cc;
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                const float x = __half2float(__ldcg(src + e));
                                if (!isfinite(x)) o[e] = __float_as_uint(__uint_as_float(o[e]) + x);
                            }
                        }
                    }
                    if (it.part >= 0) {
                        if (tiles > 0)
#pragma unroll
                            for (int e = 0; e < 32; e += 4)
                                part[256 * (8 * cc + e / 4)] = make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]),
                                                                           __uint_as_float(o[e + 2]), __uint_as_float(o[e + 3]));
                        continue;
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
    // this kernel's end is the other's too (a CTA without work that waited would keep
    // its SM from one that has some)
    if (p.shares && blockIdx.x == 0) pdl_wait();
}

// Adds up the parts of the pairs that lie in several CTAs, in order: a CTA takes 32
// rows and 32 dimensions of one pair, or returns where there is none.  One pass, the
// sums moving with the largest maximum so far, so that many parts load at a time.
template <int HD>
__global__ void __launch_bounds__(256) join_kernel(const ChunkParams c) {
    const Params& p = c.p;
    const std::uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, cta = blockIdx.x;
    pdl_launch_dependents();
    pdl_wait();
    const Join j = c.joins[cta];
    const std::uint32_t row = blockIdx.y * 32 + lane, m = row / kBM, tok = row % kBM / p.group, head = row % kBM % p.group;
    const std::uint32_t token = m * p.tile_tokens + tok, d = blockIdx.z * 8 + warp;
    if (j.count == 0 || tok >= p.tile_tokens || token >= j.left) return;
    // the first part is CTA cta's second one, the others the first ones of the CTAs behind
    const float* part = c.parts + static_cast<std::uint64_t>(2 * cta + 1) * kPart<HD>;
    float mt = -INFINITY, lt = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int kAhead = 10;
    for (std::uint32_t k0 = 0; k0 < j.count; k0 += kAhead) {
        float4 y[kAhead];
        float2 a[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const float* at = part + static_cast<std::uint64_t>(k0 + k) * (2 * kPart<HD>) - (k0 + k == 0 ? 0 : kPart<HD>);
            if (k0 + k < j.count) {
                a[k] = __ldcg(reinterpret_cast<const float2*>(at + 256 * HD) + row);
                y[k] = __ldcg(reinterpret_cast<const float4*>(at) + 256 * d + row);
            }
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            // (a part without a position of its own has -infinity and no sums)
            if (k0 + k >= j.count || (a[k].x == -INFINITY && a[k].y == 0.f)) continue;
            const float mn = fmaxf(mt, a[k].x);
            const float f = mt == mn ? 1.f : ex2f((mt - mn) * p.scale_log2);
            const float w = a[k].x == mn || a[k].y != a[k].y ? 1.f : ex2f((a[k].x - mn) * p.scale_log2);
            mt = mn;
            lt = fmaf(a[k].y, w, lt * f);
            o.x = fmaf(y[k].x, w, o.x * f), o.y = fmaf(y[k].y, w, o.y * f);
            o.z = fmaf(y[k].z, w, o.z * f), o.w = fmaf(y[k].w, w, o.w * f);
        }
    }
    const float inv = j.pos0 + static_cast<std::int32_t>(token) < 0 ? 0.f : 1.f / lt;  // nothing attended: zeros
    __half* dst = p.out + (static_cast<std::uint64_t>(j.q0 + token) * p.q_heads + j.kvh * p.group + head) * HD + 4 * d;
    *reinterpret_cast<uint2*>(dst) = make_uint2(attn8::half2_of(o.x * inv, o.y * inv), attn8::half2_of(o.z * inv, o.w * inv));
}

template <int HD>
int launch(const ChunkParams& c, const void* q, const void* k_cache, int ctas, cudaStream_t stream) {
    CUtensorMap map_q{}, map_k{}, map_v{};
    const Params& p = c.p;
    int st = attnv::make_map(&map_q, q, p.tokens, p.q_heads, HD, p.group, p.tile_tokens);
    if (st == kSuccess) st = make_map(&map_k, k_cache, p.c, c.box, 1);
    if (st == kSuccess) st = make_map(&map_v, p.v_cache, p.c, c.box, 1);
    if (st != kSuccess) return st;
    static std::atomic<std::uint64_t> smem_done{0};
    st = ensure_dynamic_smem(chunk_kernel<HD>, Smem<HD>::kBytes, smem_done);
    if (st != kSuccess) return st;
    // The register split is exact for a launch at kLaunchRegs a thread; a build
    // that allocated another count is never launched.
    static std::atomic<int> regs_checked{0};
    if (regs_checked.load(std::memory_order_acquire) == 0) {
        cudaFuncAttributes fa{};
        const cudaError_t ea = cudaFuncGetAttributes(&fa, chunk_kernel<HD>);
        if (ea != cudaSuccess) return static_cast<int>(ea);
        if (fa.numRegs != kLaunchRegs) return kInvalidConfiguration;
        regs_checked.store(1, std::memory_order_release);
    }
    st = launch_pdl_smem(chunk_kernel<HD>, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), Smem<HD>::kBytes,
                         stream, map_q, map_k, map_v, c);
    if (st != kSuccess) return st;
    return launch_pdl(join_kernel<HD>, dim3(static_cast<unsigned>(ctas), 8, HD / 32), dim3(256), stream, c);
}

// Bytes of the workspace: counters and parts of the few-row kernel, then parts and
// joins of this file's.
struct Layout {
    std::uint64_t few_parts, joins, parts, bytes;
};
inline Layout layout(int ctas, std::uint64_t head_dim, std::uint64_t rows) {
    Layout l{};
    l.few_parts = few::kMaxCtas * 4;
    l.joins = l.few_parts + static_cast<std::uint64_t>(ctas) * 2 * few::kCols * (rows <= few::kCols ? 1 : few::kMaxSets) * (head_dim + 2) * 4;
    l.parts = l.bytes = l.joins;
    if (rows > few::kMostRows) {
        l.parts = l.joins + kMaxCtas * sizeof(Join);  // a multiple of 16
        l.bytes = l.parts + static_cast<std::uint64_t>(ctas) * 2 * 256 * (head_dim + 2) * 4;
    }
    return l;
}

}  // namespace chunk
}  // namespace attnpg
}  // namespace mote

extern "C" int mote_cuda_gqa_attention_paged_f16_workspace_bytes(uint64_t q_heads,
                                                                  uint64_t kv_heads,
                                                                  uint64_t head_dim,
                                                                  uint64_t max_new,
                                                                  uint64_t* bytes) {
    using namespace mote;
    if (bytes == nullptr) return kInvalidValue;
    *bytes = 0;
    if (q_heads == 0 || kv_heads == 0 || (head_dim != 64 && head_dim != 128) || max_new > 0x7fffffffull)
        return kSuccess;  // nothing to do, or refused by the call itself
    int n = 0;
    const int st = attnpg::sm_count(n);
    if (st != kSuccess) return st;
    if (n > attnpg::few::kMaxCtas) n = attnpg::few::kMaxCtas;
    *bytes = attnpg::chunk::layout(n, head_dim, max_new * (q_heads / kv_heads)).bytes;
    return kSuccess;
}

extern "C" int mote_cuda_gqa_attention_paged_f16(
    const void* q, const void* k_cache, const void* v_cache, const void* block_tables,
    const void* q_starts, const void* seq_lens, void* out, uint64_t tokens, uint64_t batch,
    uint64_t q_heads, uint64_t kv_heads, uint64_t head_dim, uint64_t num_blocks,
    uint64_t block_tokens, uint64_t max_blocks, uint64_t max_new, float scale, void* workspace,
    uint64_t workspace_bytes, void* stream) {
    using namespace mote;
    using namespace mote::attnpg;
    if (q == nullptr || k_cache == nullptr || v_cache == nullptr || block_tables == nullptr ||
        q_starts == nullptr || seq_lens == nullptr || out == nullptr || stream == nullptr)
        return kInvalidValue;
    if (!kvq8::shape_ok(batch, kv_heads, head_dim, num_blocks, block_tokens, max_blocks) ||
        kv_heads == 0 || q_heads % kv_heads != 0 || q_heads > 65535 || q_heads / kv_heads > 128 ||
        tokens > 0x7fffffffull || max_new > 0x7fffffffull || !(scale > 0.f) ||
        !std::isfinite(scale * 1.4426950408889634f) ||  // (the kernels' factor)
        !kvq8::aligned16({q, k_cache, v_cache, out}) ||
        !kvq8::aligned4({block_tables, q_starts, seq_lens}) ||
        num_blocks * kv_heads * block_tokens > kNowhere)  // below 2^55
        return kInvalidValue;
    if (tokens == 0 || batch == 0 || q_heads == 0) return kSuccess;
    int n = 0;
    int st = sm_count(n);
    if (st != kSuccess) return st;
    if (n > few::kMaxCtas) n = few::kMaxCtas;
    const std::uint64_t group = q_heads / kv_heads;
    const chunk::Layout at = chunk::layout(n, head_dim, max_new * group);
    if (workspace == nullptr || workspace_bytes < at.bytes || !kvq8::aligned16({workspace}))
        return kInvalidValue;
    std::uint8_t* const ws = static_cast<std::uint8_t*>(workspace);
    Params p{};
    p.q = static_cast<const __half*>(q);
    p.v_cache = static_cast<const __half*>(v_cache);
    p.tables = static_cast<const std::int32_t*>(block_tables);
    p.starts = static_cast<const std::int32_t*>(q_starts);
    p.lens = static_cast<const std::int32_t*>(seq_lens);
    p.out = static_cast<__half*>(out);
    p.c = kvq8::make_shape(batch, kv_heads, head_dim, num_blocks, block_tokens, max_blocks);
    p.tokens = static_cast<std::uint32_t>(tokens);
    p.q_heads = static_cast<std::uint32_t>(q_heads);
    p.group = static_cast<std::uint32_t>(group);
    p.max_new = static_cast<std::uint32_t>(max_new);
    p.scale_log2 = scale * 1.4426950408889634f;
    p.counters = reinterpret_cast<unsigned*>(ws);
    p.parts = reinterpret_cast<float*>(ws + at.few_parts);
    p.reports = true;
    const auto s = static_cast<cudaStream_t>(stream);
    // Both kernels where the host cannot tell that one of them has nothing to do: a
    // single sequence, or groups too large for the few-row kernel, are the other's.  No
    // sequence has more tokens than there are (one call alone, one token over 32768 with
    // max_new 64: 33 us, 47 when max_new alone decided; over 117 10.2 and 18.4).
    const std::uint64_t rows = (max_new < tokens ? max_new : tokens) * group;
    const bool chunks = rows > few::kMostRows;
    p.few = chunks && (batch == 1 || group > few::kMostRows) ? 0u : few::kMostRows;
    p.shares = chunks && p.few != 0;
    p.tile_tokens = attnv::kBM / p.group;
    p.sub = head_dim == 64 && block_tokens % 32 != 0 ? 2 : 1;
    if (p.few != 0) {
        const auto run = [&](auto hd) {
            constexpr int HD = decltype(hd)::value;
            return rows <= few::kCols ? few::launch<HD, 1>(p, k_cache, n, s) : few::launch<HD, few::kMaxSets>(p, k_cache, n, s);
        };
        st = head_dim == 64 ? run(std::integral_constant<int, 64>{}) : run(std::integral_constant<int, 128>{});
        if (st != kSuccess || !chunks) return st;
        p.reports = false;
    }
    chunk::ChunkParams c{};
    c.p = p;
    c.box = 16;
    while (c.box < 128 && block_tokens % (2 * c.box) == 0) c.box *= 2;
    c.joins = reinterpret_cast<chunk::Join*>(ws + at.joins);
    c.parts = reinterpret_cast<float*>(ws + at.parts);
    return head_dim == 64 ? chunk::launch<64>(c, q, k_cache, n, s) : chunk::launch<128>(c, q, k_cache, n, s);
}

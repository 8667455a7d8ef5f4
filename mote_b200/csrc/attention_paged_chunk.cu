// Attention of new tokens over a paged f16 cache (attention_paged.cu), for the
// sequences with more query rows than the few-row kernel takes: chunks of prompts,
// on the tcgen05 tensor cores.
//
// A query tile is 128 rows: floor(128 / g) tokens of one sequence times the g query
// heads of one KV head (one TMA box of q).  A pair of consecutive query tiles shares
// every K/V tile of 128 positions, which TMA puts together from the pages (boxes of
// the largest power of two of rows that a block holds, 16 to 128 of them; the block
// numbers of the next tile are read while this one's stage is waited for).  Within a
// CTA the roles are those of attention_packed.cu: warp 8 walks the work and loads,
// warp 9 owns tensor memory and issues S_i = Q_i K^T and O_i += P_i V (P from tensor
// memory), warps 0-3 and 4-7 run the softmax of the two query tiles, one thread per
// row, warps 10 and 11 take what is not finite out of V tiles that some row sees in
// part (later positions, and the rows of a page behind the last position).
//
// The work, all pairs of all sequences and KV heads, is a line of virtual positions:
// a pair is as long as the positions that it attends (times kBoth or kOne, for two
// query tiles or one) and its end (kEnd).  Each CTA takes an equal share of it,
// found on the device from sums of arithmetic series, so one chunk over a long cache
// fills the GPU as well as a batch of prompts does.  A pair that lies in several
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
using attnp::umma_f16_ss;
using attnv::arrive;
using attnv::elect_one;
using attnv::kBM;
using attnv::kBN;
using attnv::kCleanWarps;
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
using attnv::kVast;
using attnv::tmem_ld16;
using attnv::tmem_st16;
using attnv::v_desc;
using gemm::wait_or_abort;

constexpr int kMaxCtas = 192;
// Virtual positions: of a position for a pair of two query tiles and of one, and of a
// pair's end.
constexpr std::uint32_t kBoth = 4, kOne = 3, kEnd = 4 * 256;
// The least share, in virtual positions, and the least piece of a pair, in K/V tiles.
constexpr std::uint64_t kLeast = 4 * 1024;
constexpr std::uint32_t kMinTiles = 3;

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
};

template <int HD>
struct Smem {
    using Base = attnv::Smem<HD>;
    static constexpr int kHalf = Base::kHalf, kTile = Base::kTile, kKV = Base::kKV, kS = Base::kS;
    static constexpr std::uint32_t kColO = Base::kColO;
    static constexpr int kQ = Base::kQ, kK = Base::kK, kV = Base::kV, kBar = Base::kBar;
    static constexpr int kTmemSlot = Base::kTmemSlot, kAbort = Base::kAbort, kFlag = Base::kFlag;
    static constexpr int kItem = (Base::kItem + 15) / 16 * 16;  // [kItems]
    static constexpr int kShare = kItem + kItems * static_cast<int>(sizeof(Item));  // [3] first sequence, share, begin
    static constexpr int kScan = (kShare + 7) / 8 * 8 + 3 * 8;  // [warp] sums
    static constexpr int kUsed = kScan + kThreads / 32 * 8 + 1008;  // + alignment slack
    // one CTA per SM: its 512 TMEM columns never wait for another's
    static constexpr int kBytes = kUsed > 120 * 1024 ? kUsed : 120 * 1024;
    static_assert(kBytes <= 232448, "shared memory");
};

struct ChunkParams {
    Params p;
    std::uint32_t tile_tokens;  // floor(128 / group)
    std::uint32_t box;          // rows of a K or V box
    Join* joins;                // [CTAs]
    float* parts;               // [2 CTAs][HD / 4][256][4], then [256][2]: maxima and sums
};

template <int HD>
constexpr std::uint64_t kPart = 256ull * (HD + 2);

// A sequence's pairs, as the line of virtual positions has them.
struct Pairs {
    Seq s;
    std::uint32_t span, tile;  // tokens of a pair and of a query tile
    std::uint32_t count;       // pairs

    __device__ __forceinline__ Pairs(const ChunkParams& c, std::uint32_t b)
        : s(sequence(c.p, b)), span(2 * c.tile_tokens), tile(c.tile_tokens) {
        if (static_cast<std::uint64_t>(s.n) * c.p.group <= c.p.few) s.n = 0;
        count = (s.n + span - 1) / span;
    }
    // positions that pair i attends
    __device__ __forceinline__ std::uint32_t reach(std::uint32_t i) const {
        const std::int64_t end = static_cast<std::int64_t>(s.len) - s.n + min(static_cast<std::uint64_t>(i + 1) * span, static_cast<std::uint64_t>(s.n));
        return end < 0 ? 0u : static_cast<std::uint32_t>(end);
    }
    __device__ __forceinline__ std::uint64_t extent(std::uint32_t i) const {
        const bool both = s.n - i * span > tile;
        return static_cast<std::uint64_t>(reach(i)) * (both ? kBoth : kOne) + kEnd;
    }
    // extents of the pairs before i (i <= count): a series, but for pairs that
    // attend nothing and the last one
    __device__ __forceinline__ std::uint64_t before(std::uint32_t i) const {
        if (i == 0) return 0;
        const std::uint32_t full = i < count ? i : i - 1;
        const std::int64_t past = static_cast<std::int64_t>(s.len) - s.n;  // negative: some pairs have no positions
        std::uint32_t none = past >= 0 ? 0u : static_cast<std::uint32_t>(-past / span);
        if (none > full) none = full;
        const std::uint64_t m = full - none;
        std::uint64_t x = static_cast<std::uint64_t>(full) * kEnd;
        // reach(k) = past + (k + 1) span for k = none .. full - 1
        x += kBoth * static_cast<std::uint64_t>(static_cast<std::int64_t>(m) * past + static_cast<std::int64_t>(span) * static_cast<std::int64_t>(m * none + m * (m + 1) / 2));
        return i < count ? x : x + extent(count - 1);
    }
    __device__ __forceinline__ std::uint64_t all() const { return before(count); }
};

// Of a pair of n K/V tiles, those before virtual position x of it.
__device__ __forceinline__ std::uint32_t cut(std::uint64_t x, std::uint32_t n, bool both) {
    const std::uint64_t t = (x + 64 * (both ? kBoth : kOne)) / (kBN * (both ? kBoth : kOne));
    if (t < kMinTiles) return 0;
    return t + kMinTiles > n ? n : static_cast<std::uint32_t>(t);
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
    if (c.tile_tokens * p.group < kBM) {  // rows of a query tile that no box fills stay zero
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

    // ---- the CTA's share of the line ---------------------------------------
    volatile std::uint64_t* share = reinterpret_cast<volatile std::uint64_t*>(smem + (L::kShare + 7) / 8 * 8);
    volatile std::uint64_t* scan = reinterpret_cast<volatile std::uint64_t*>(smem + L::kScan);
    {
        const auto scan_up = [&](std::uint64_t x) {  // inclusive, over the warp
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const std::uint64_t y = __shfl_up_sync(0xffffffffu, x, d);
                if (lane >= d) x += y;
            }
            return x;
        };
        const auto line_of = [&](std::uint32_t b) -> std::uint64_t {
            return b < p.c.batch ? Pairs(c, b).all() * p.c.kv_heads : 0;
        };
        std::uint64_t sum = 0;
        for (std::uint32_t b = threadIdx.x; b < p.c.batch; b += kThreads) sum += line_of(b);
        sum = scan_up(sum);
        if (lane == 31) scan[warp] = sum;
        if (threadIdx.x == 0) share[0] = ~0ull;
        __syncthreads();
        std::uint64_t total = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) total += scan[w];
        __syncthreads();
        std::uint64_t per = (total + gridDim.x - 1) / gridDim.x;
        if (per < kLeast) per = kLeast;
        const std::uint64_t at = per * blockIdx.x;
        std::uint64_t before = 0;
        for (std::uint32_t base = 0; base < p.c.batch && before <= at; base += kThreads) {
            const std::uint64_t mine = line_of(base + threadIdx.x), incl = scan_up(mine);
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
                share[2] = begin;
            }
            __syncthreads();
        }
        if (threadIdx.x == 0) share[1] = per;
        __syncthreads();
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
            const std::uint64_t per = share[1], u0 = per * blockIdx.x, u1 = u0 + per;
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
                if (lane == 0) {
                    ok = n == 0 || wait_or_abort(q_empty, (n - 1) & 1u, abort_flag);
                    if (ok) {
                        const std::uint32_t box = c.tile_tokens * p.group * 128;
                        mbar_arrive_expect_tx(q_full, ((it.n[0] > 0) + (it.n[1] > 0)) * (HD / 64) * box);
#pragma unroll
                        for (int m = 0; m < 2; ++m)
                            for (int h = 0; h < HD / 64 && it.n[m] > 0; ++h)
                                tma_load_3d(base + L::kQ + m * L::kTile + h * L::kHalf, &map_q, 64 * h,
                                            static_cast<int>(it.kvh * p.group),
                                            static_cast<int>(it.q0 + m * c.tile_tokens), smem_u32(q_full));
                    }
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
                // the cache row of this lane's box of tile j (what is not there reads as zeros)
                const auto row_of = [&](std::uint32_t j) {
                    const std::uint32_t pos = (it.t0 + j) * kBN + sub * c.box;
                    if (!loads || pos >= it.nk || j >= tiles) return kNowhere;
                    const std::uint32_t i = pos / p.c.block_tokens;
                    const std::int32_t block = __ldg(p.tables + static_cast<std::uint64_t>(it.b) * p.c.max_blocks + i);
                    if (block < 0 || static_cast<std::uint64_t>(block) >= p.c.num_blocks) {
                        atomicOr(&g_device_status, kDevIndexOutOfRange);
                        return kNowhere;
                    }
                    return static_cast<int>((static_cast<std::uint32_t>(block) * p.c.kv_heads + it.kvh) * p.c.block_tokens + pos - i * p.c.block_tokens);
                };
                int row = row_of(0);
                for (std::uint32_t j = 0; ok && j < tiles; ++j) {
                    const std::uint32_t t = kv + j, s = t % kKV, ph = (t / kKV - 1) & 1u;
                    const int next = row_of(j + 1);
                    const std::uint32_t at = s * L::kTile + dims * L::kHalf + sub * c.box * 128;
                    if (t >= kKV) ok = __all_sync(0xffffffffu, wait_or_abort(&k_empty[s], ph, abort_flag));
                    if (!ok) break;
                    if (lane == 0) mbar_arrive_expect_tx(&k_full[s], L::kTile);
                    __syncwarp();
                    if (loads && lane < 16) attn8::tma_load_2d(base + L::kK + at, &map_k, 64 * dims, row, smem_u32(&k_full[s]));
                    if (t >= kKV) ok = __all_sync(0xffffffffu, wait_or_abort(&v_empty[s], ph, abort_flag));
                    if (!ok) break;
                    if (lane == 0) mbar_arrive_expect_tx(&v_full[s], L::kTile);
                    __syncwarp();
                    if (loads && lane >= 16) attn8::tma_load_2d(base + L::kV + at, &map_v, 64 * dims, row, smem_u32(&v_full[s]));
                    row = next;
                }
                kv += tiles;
                ++n;
            };
            if (share[0] != ~0ull) {
                std::uint32_t b = static_cast<std::uint32_t>(share[0]);
                Pairs x(c, b);
                // the pair that u0 lies in
                std::uint64_t begin = share[2];
                std::uint32_t kvh = static_cast<std::uint32_t>((u0 - begin) / x.all()), i = 0;
                begin += kvh * x.all();
                for (std::uint32_t hi = x.count; hi - i > 1;) {
                    const std::uint32_t mid = (i + hi) / 2;
                    if (begin + x.before(mid) <= u0) i = mid; else hi = mid;
                }
                begin += x.before(i);
                while (ok && begin < u1) {
                    const std::uint64_t extent = x.extent(i);
                    const bool both = x.s.n - i * x.span > x.tile;
                    const std::uint32_t reach = x.reach(i), tiles = (reach + kBN - 1) / kBN;
                    const std::uint32_t from = begin >= u0 ? 0u : cut(u0 - begin, tiles, both);
                    const std::uint32_t to = begin + extent <= u1 ? tiles : cut(u1 - begin, tiles, both);
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
                            const std::uint32_t first = m * c.tile_tokens;
                            const std::int32_t last = it.pos0 + static_cast<std::int32_t>(min(first + c.tile_tokens, it.left)) - 1;
                            const std::uint32_t whole = first >= it.left || last < 0 ? 0u : static_cast<std::uint32_t>(last) / kBN + 1;
                            it.n[m] = min(whole, to) - min(whole, from);
                        }
                        const std::uint32_t masked = static_cast<std::uint32_t>(max(it.pos0 + 1, 0)) / kBN;
                        it.masked = masked > from ? masked - from : 0u;
                        it.part = from == 0 && to == tiles ? -1 : static_cast<std::int32_t>(2 * blockIdx.x + (from == 0 ? 1 : 0));
                        if (from == 0 && to < tiles) {
                            // the last CTA that has some of it
                            std::uint64_t last = (begin + extent - 1) / per;
                            if (cut(last * per - begin, tiles, both) == tiles) --last;
                            joined = static_cast<std::uint32_t>(last) - blockIdx.x + 1;
                            if (lane == 0) c.joins[blockIdx.x] = Join{joined, it.left, kvh, it.q0};
                        }
                        send(it);
                        if (ok && it.tiles() > 0) load(it);
                    }
                    begin += extent;
                    if (++i < x.count) continue;
                    i = 0;
                    if (++kvh < p.c.kv_heads) continue;
                    kvh = 0;
                    do {
                        if (++b >= p.c.batch) break;
                        x = Pairs(c, b);
                    } while (x.count == 0);
                    if (b >= p.c.batch) break;
                }
            }
            if (joined == 0 && lane == 0) c.joins[blockIdx.x] = Join{0, 0, 0, 0};
            if (ok) send(Item{});
        } else if (warp == kMmaWarp) {
            // The whole warp walks the loops, on values that the compiler knows to
            // be uniform, and one elected lane issues: operands then come from
            // uniform registers (moving each to one cost 100 cycles an MMA).
            const std::uint32_t tm = __reduce_max_sync(0xffffffffu, tmem);
            std::uint32_t kv = 0, n = 0, clean = 0;
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
                    const std::uint32_t t = kv + j;
                    return wait(&k_full[t % kKV], (t / kKV) & 1u);
                };
                const auto issue_s = [&](std::uint32_t x) {  // then what its last use frees
                    const int m = m_of(x);
                    const std::uint32_t j = j_of(x), s = (kv + j) % kKV, buf = (passed + x) % L::kS;
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
                    const std::uint32_t j = j_of(x), t = kv + j, s = t % kKV;
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
                kv += tiles;
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
            std::uint32_t kv = 0, n = 0, clean = 0;
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
                    const std::uint32_t t = kv + j, s = t % kKV;
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
                            const std::uint32_t rows = it.nk - (it.t0 + j) * kBN;  // of the sequence
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
        std::uint32_t passed = 0, n = 0;  // softmax passes (of both query tiles) and items so far
        std::uint32_t seen = 0;           // parity of this query tile's passes on each S buffer
        bool ok = true;
        for (std::uint32_t i = 0;; ++i) {
            const Item it = item_at(i);
            if (it.left == 0) break;
            const std::uint32_t token = m * c.tile_tokens + tok;  // from the item's first
            const bool mine = tok < c.tile_tokens && token < it.left;
            const std::int32_t limit = it.pos0 + static_cast<std::int32_t>(token);  // its position
            // the least position of the warp's rows
            const std::int32_t least = it.pos0 + static_cast<std::int32_t>(
                m * c.tile_tokens + 32u * (warp % 4) / p.group);
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
                const std::int32_t kbase = static_cast<std::int32_t>((it.t0 + j) * kBN);
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
                    if (add) {
                        // what warps 10 and 11 took out of the V tiles that this row attends
                        const std::uint32_t end = min(static_cast<std::uint32_t>(limit) + 1u, (it.t0 + tiles) * kBN);
                        for (std::uint32_t pos = (it.t0 + it.masked) * kBN; pos < end; ++pos) {
                            const std::int32_t block = __ldg(p.tables + static_cast<std::uint64_t>(it.b) * p.c.max_blocks + pos / p.c.block_tokens);
                            if (block < 0 || static_cast<std::uint64_t>(block) >= p.c.num_blocks) continue;
                            const __half* src = p.v_cache + ((static_cast<std::uint64_t>(block) * p.c.kv_heads + it.kvh) * p.c.block_tokens +
                                                             pos % p.c.block_tokens) * HD + 32 * cc;
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                const float x = __half2float(src[e]);
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
}


// Adds up the parts of the pairs that lie in several CTAs, in order: a CTA takes 32
// rows and 64 dimensions of one pair, or returns where there is none.
template <int HD>
__global__ void __launch_bounds__(256) join_kernel(const ChunkParams c) {
    const Params& p = c.p;
    const std::uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, cta = blockIdx.x;
    pdl_launch_dependents();
    pdl_wait();
    const Join j = c.joins[cta];
    const std::uint32_t row = blockIdx.y * 32 + lane, m = row / kBM, tok = row % kBM / p.group, head = row % kBM % p.group;
    const std::uint32_t token = m * c.tile_tokens + tok, d = blockIdx.z * 16 + warp;
    if (j.count == 0 || tok >= c.tile_tokens || token >= j.left) return;
    const auto part_of = [&](std::uint32_t k) {
        return c.parts + static_cast<std::uint64_t>(2 * (cta + k) + (k == 0 ? 1 : 0)) * kPart<HD>;
    };
    const auto ml_of = [&](std::uint32_t k) {
        return __ldcg(reinterpret_cast<const float2*>(part_of(k) + 256 * HD) + row);
    };
    float mt = -INFINITY, lt = 0.f;
#pragma unroll 8
    for (std::uint32_t k = 0; k < j.count; ++k) mt = fmaxf(mt, ml_of(k).x);
    float4 o[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll 8
    for (std::uint32_t k = 0; k < j.count; ++k) {
        const float4* part = reinterpret_cast<const float4*>(part_of(k)) + row;
        const float4 y0 = __ldcg(part + 256 * d), y1 = __ldcg(part + 256 * (d + 8));
        const float2 a = ml_of(k);
        if (a.x == -INFINITY && a.y == 0.f) continue;  // no position of its own there
        const float w = a.y != a.y || a.x == mt ? 1.f : ex2f((a.x - mt) * p.scale_log2);
        lt = fmaf(a.y, w, lt);
        o[0].x = fmaf(y0.x, w, o[0].x), o[0].y = fmaf(y0.y, w, o[0].y);
        o[0].z = fmaf(y0.z, w, o[0].z), o[0].w = fmaf(y0.w, w, o[0].w);
        o[1].x = fmaf(y1.x, w, o[1].x), o[1].y = fmaf(y1.y, w, o[1].y);
        o[1].z = fmaf(y1.z, w, o[1].z), o[1].w = fmaf(y1.w, w, o[1].w);
    }
    const float inv = lt == 0.f ? 0.f : 1.f / lt;
    __half* dst = p.out + (static_cast<std::uint64_t>(j.q0 + token) * p.q_heads + j.kvh * p.group + head) * HD;
#pragma unroll
    for (int k = 0; k < 2; ++k)
        *reinterpret_cast<uint2*>(dst + 4 * (d + 8 * k)) =
            make_uint2(attn8::half2_of(o[k].x * inv, o[k].y * inv), attn8::half2_of(o[k].z * inv, o[k].w * inv));
}

template <int HD>
int launch(const ChunkParams& c, const void* q, const void* k_cache, int ctas, cudaStream_t stream) {
    CUtensorMap map_q{}, map_k{}, map_v{};
    const Params& p = c.p;
    int st = attnv::make_map(&map_q, q, p.tokens, p.q_heads, HD, p.group, c.tile_tokens);
    if (st == kSuccess) st = make_map(&map_k, k_cache, p.c, c.box);
    if (st == kSuccess) st = make_map(&map_v, p.v_cache, p.c, c.box);
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
    return launch_pdl(join_kernel<HD>, dim3(static_cast<unsigned>(ctas), 8, HD / 64), dim3(256), stream, c);
}

// Bytes of the workspace: counters and parts of the few-row kernel, then parts and
// joins of this file's.
struct Layout {
    std::uint64_t few_parts, joins, parts, bytes;
};
inline Layout layout(int ctas, std::uint64_t head_dim, std::uint64_t rows) {
    Layout l{};
    l.few_parts = few::kMaxCtas * 4;
    l.joins = l.few_parts + static_cast<std::uint64_t>(ctas) * 2 * few::kCols * few::sets_of(rows) * (head_dim + 2) * 4;
    l.parts = l.bytes = l.joins;
    if (rows > few::kCols * few::kMaxSets) {
        l.parts = l.joins + kMaxCtas * sizeof(Join);
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
        tokens > 0x7fffffffull || max_new > 0x7fffffffull || !std::isfinite(scale) ||
        !(scale > 0.f) || !kvq8::aligned16({q, k_cache, v_cache, out}) ||
        !kvq8::aligned4({block_tables, q_starts, seq_lens}) ||
        num_blocks * kv_heads * block_tokens > kNowhere)  // below 2^55
        return kInvalidValue;
    if (tokens == 0 || batch == 0 || q_heads == 0) return kSuccess;
    int n = 0;
    int st = sm_count(n);
    if (st != kSuccess) return st;
    if (n > few::kMaxCtas) n = few::kMaxCtas;
    const std::uint64_t group = q_heads / kv_heads, rows = max_new * group;
    const chunk::Layout at = chunk::layout(n, head_dim, rows);
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
    // single sequence, or groups too large for the few-row kernel, are the other's.
    const std::uint32_t most = few::kCols * few::kMaxSets;
    const bool chunks = rows > most;
    p.few = chunks && (batch == 1 || group > most) ? 0u : most;
    if (p.few != 0) {
        const auto run = [&](auto hd) {
            constexpr int HD = decltype(hd)::value;
            switch (few::sets_of(rows)) {
                case 1: return few::launch<HD, 1>(p, k_cache, n, s);
                case 2: return few::launch<HD, 2>(p, k_cache, n, s);
                default: return few::launch<HD, 4>(p, k_cache, n, s);
            }
        };
        st = head_dim == 64 ? run(std::integral_constant<int, 64>{}) : run(std::integral_constant<int, 128>{});
        if (st != kSuccess || !chunks) return st;
        p.reports = false;
    }
    chunk::ChunkParams c{};
    c.p = p;
    c.tile_tokens = attnv::kBM / p.group;
    c.box = 16;
    while (c.box < 128 && block_tokens % (2 * c.box) == 0) c.box *= 2;
    c.joins = reinterpret_cast<chunk::Join*>(ws + at.joins);
    c.parts = reinterpret_cast<float*>(ws + at.parts);
    return head_dim == 64 ? chunk::launch<64>(c, q, k_cache, n, s) : chunk::launch<128>(c, q, k_cache, n, s);
}

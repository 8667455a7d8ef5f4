// Attention of new tokens over a paged KV cache held in f16: sequence b has the
// queries q_starts[b] .. q_starts[b + 1] - 1, the last of its seq_lens[b]
// cached positions; with n of them, query i attends the positions up to its own:
//   out[i, h] = softmax_{p <= len - n + i}(scale * q[i, h] . K[p, h / g]) . V[p, h / g]
// A query before the first position (len < n) gets zeros; rows that belong to
// no sequence keep their values.
//
// Two kernels, each for its own sequences of a batch (the lengths are on the
// device): this file's for sequences with up to 16 query rows (tokens times grouped
// heads of a KV head), whose cost is the stream of K and V;
// attention_paged_chunk.cu's for more, on the tcgen05 tensor cores.  Where a batch may
// hold both, the kernels run at the same time, on SMs that they divide by the work that
// each has (few_ctas).
//
// Few rows: HBM-bound, K and V of the attended positions are read once.  48 sequences of
// up to 8192 (773 MB, 32 query / 8 KV heads of 128): 122-127 us, 0.93-0.97 of the copy bandwidth;
// one of 32768 (134 MB): 29.8, of which about 10 are the start and the join.
// * The work is cut in units of 8 KB of K and V (16 positions at head_dim 128, 32
//   at 64) of one (sequence, KV head) "row".  One CTA per SM takes an equal share
//   of consecutive units, found from the lengths on the device, so ragged batches
//   balance and the host needs no bound on the lengths.  The 8 warps of a CTA take
//   a row's units in turn, each through a ring of three units that runs ahead
//   across rows; the lane that holds a block's number issues its TMA loads (boxes
//   of 16 positions x 128 bytes, 128-byte swizzle: ldmatrix meets all banks).
// * mma.sync m16n8k16 with the cache as the A operand: S^T = K Q^T with 16
//   positions as rows and 8 (token, head) pairs as columns, then O^T += V^T P^T with
//   16 dimensions as rows, so that 8 columns cost no idle rows; up to two sets of
//   8 columns share the operand.  P^T gets from the accumulator layout to the
//   operand's with movmatrix.
// * The running maximum moves only when a lane's sum of P passes 2^8, so a step
//   costs one vote instead of reductions.  P is rounded to f16 (11 bits), held
//   2^7 up, so that weights down to 2^-21 of the reference keep them.
// * Units that some column sees in part, the last ones of a row, are masked, and
//   what is not finite is taken out of their V: 0 times an infinity or NaN of a
//   masked position would be NaN.  The columns that do attend such a value add it
//   at the end (rare, from global memory).
// * Rows that lie in several CTAs leave unnormalised parts in the workspace; the
//   last CTA to finish joins them in order (a counter per row, left at zero), so
//   results do not depend on timing.
// Every wait is bounded; one that expires is reported in the device status and
// the lane runs on without waiting and without further copies.
#include "mote_common.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

namespace mote {
namespace attnpg {

// A row number that no cache has: TMA fills what lies there with zeros.
constexpr int kNowhere = 0x7fffff00;

struct Params {
    const __half* q;
    const __half* v_cache;
    const std::int32_t* tables;
    const std::int32_t* starts;
    const std::int32_t* lens;
    __half* out;
    kvq8::CacheShape c;
    std::uint32_t tokens, q_heads, group, max_new;
    std::uint32_t few;   // query rows of a KV head up to which a sequence is the first kernel's
    bool reports;        // this kernel tells of sequences that are skipped
    bool shares;         // both kernels run, each on its part of the SMs
    std::uint32_t tile_tokens;  // of a query tile of the chunk kernel: floor(128 / group)
    std::uint32_t sub;   // loads of K in a unit of the few-row kernel
    float scale_log2;
    unsigned* counters;  // [kMaxCtas], zero between calls
    float* parts;
};

// A sequence's first query row, number of new tokens (0: none, or skipped) and length.
struct Seq {
    std::uint32_t q0, n, len;
    bool bad;
};
// Offsets, lengths and block numbers.  A kernel that runs beside the other one does
// not wait for what is before both (that one has), so it reads past its L1.
__device__ __forceinline__ std::int32_t fetch(const Params& p, const std::int32_t* x) {
    return p.shares ? __ldcg(x) : __ldg(x);
}
__device__ __forceinline__ Seq sequence(const Params& p, std::uint32_t b) {
    const std::int32_t s0 = fetch(p, p.starts + b), s1 = fetch(p, p.starts + b + 1), len = fetch(p, p.lens + b);
    Seq s{static_cast<std::uint32_t>(s0), static_cast<std::uint32_t>(s1 - s0), static_cast<std::uint32_t>(len), false};
    s.bad = s0 < 0 || s1 < s0 || static_cast<std::uint32_t>(s1) > p.tokens ||
            (s1 > s0 && (len < 0 || static_cast<std::uint32_t>(len) > p.c.max_blocks * p.c.block_tokens || s.n > p.max_new));
    if (s.bad) s.n = 0;
    return s;
}
__device__ __forceinline__ void report_bad(const Params& p, std::uint32_t first, std::uint32_t step) {
    for (std::uint32_t b = first; b < p.c.batch; b += step)
        if (sequence(p, b).bad) atomicOr(&g_device_status, kDevIndexOutOfRange);
}

// The chunk kernel's work, a line of positions: all pairs of query tiles of all its
// sequences and KV heads, each as long as the positions that it attends and its end
// (kEnd).  A pair whose second tile has no rows counts as much: it streams as much.
constexpr std::uint32_t kEnd = 256;

// A sequence's pairs on that line, for one KV head.
struct Pairs {
    Seq s;
    std::uint32_t tile, span;  // tokens of a query tile and of a pair
    std::uint32_t count;  // pairs

    __device__ __forceinline__ Pairs(const Params& p, const Seq& of) : s(of), tile(p.tile_tokens), span(2 * p.tile_tokens) {
        if (static_cast<std::uint64_t>(s.n) * p.group <= p.few) s.n = 0;
        count = (s.n + span - 1) / span;
    }
    // positions that pair i attends
    __device__ __forceinline__ std::uint32_t reach(std::uint32_t i) const {
        const std::uint32_t end = s.len + min((i + 1) * span, s.n);  // below 2^32
        return end > s.n ? end - s.n : 0u;
    }
    __device__ __forceinline__ std::uint32_t extent(std::uint32_t i) const { return reach(i) + kEnd; }
    // extents of the pairs before i (i <= count): a series, but for pairs that
    // attend nothing and the last one
    __device__ __forceinline__ std::uint64_t before(std::uint32_t i) const {
        const std::uint32_t full = i < count ? i : count == 0 ? 0 : count - 1;
        // reach(k) = len - n + (k + 1) span for k = none .. full - 1
        const std::uint32_t none = s.n > s.len ? min((s.n - s.len) / span, full) : 0u, m = full - none;
        const std::int64_t sum = static_cast<std::int64_t>(m) * (static_cast<std::int64_t>(s.len) - s.n) +
                                 static_cast<std::int64_t>(static_cast<std::uint64_t>(span) * (static_cast<std::uint64_t>(m) * none + static_cast<std::uint64_t>(m) * (m + 1ull) / 2));
        const std::uint64_t x = static_cast<std::uint64_t>(sum) + static_cast<std::uint64_t>(full) * kEnd;
        return i < count || count == 0 ? x : x + extent(count - 1);
    }
    __device__ __forceinline__ std::uint64_t all() const { return before(count); }
    // how long they take, in positions of a pair of two tiles: one tile takes three
    // quarters of it
    __device__ __forceinline__ std::uint64_t cost() const {
        return all() - (count > 0 && s.n - (count - 1) * span <= tile ? extent(count - 1) / 4 : 0u);
    }
};

// The chunk kernel's work of a sequence.
__device__ __forceinline__ std::uint64_t cost_of(const Params& p, const Seq& s) { return Pairs(p, s).cost() * p.c.kv_heads; }
// SMs of `n` that the few-row kernel has where both run, from its work (units, row
// ends counted) and the other's (cost): a unit takes an SM about as long as kUnitCost
// positions of a pair, 160 ns to 20 at head_dim 128 and 16 at 64 (32 tokens over up to
// 4000 beside a chunk of 512 at head_dim 64: 70 us, 88 with half of it and 89 with twice;
// 23 over 3000 at 128: 93, 101 with one more).  On more than 7/8 of the SMs it would wait
// for HBM (38 over 8000 beside two chunks of 100: 239, 287 on 128 SMs and 464 on 137).
// In f32, of which both kernels make the same.
template <int HD>
constexpr float kUnitCost = HD == 128 ? 8.f : 10.f;
template <int HD>
__device__ __forceinline__ std::uint32_t few_ctas(std::uint32_t n, std::uint64_t units, std::uint64_t cost) {
    if (cost == 0) return n;
    if (units == 0) return 0;
    const float mine = __fmul_rn(__ull2float_rn(units), kUnitCost<HD>), all = __fadd_rn(mine, __ull2float_rn(cost));
    const std::uint32_t x = __float2uint_rn(__fmul_rn(__fdiv_rn(mine, all), static_cast<float>(n)));
    return min(max(x, 1u), n - max(n / 8, 1u));
}
// A share of `total` over `ctas`, rounded up (by up to 2^-22 of it).
__device__ __forceinline__ std::uint64_t share_of(std::uint64_t total, std::uint32_t ctas) {
    return __float2ull_ru(__fmul_ru(__ull2float_ru(total), __frcp_ru(static_cast<float>(ctas)))) + 1;
}

namespace few {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kCols = 8;         // columns of a set: (token, query head) pairs
constexpr int kMaxSets = 2;
constexpr int kBox = 2048;       // 16 rows of 128 bytes
constexpr int kStage = 4 * kBox; // K and V of a unit
constexpr int kStages = 3;
constexpr int kMaxCtas = 192;
constexpr int kMinUnits = 2 * kWarps;  // rows of up to this many units are not split
// Sequences up to which every warp finds the CTA's share alone, one to a lane: 16 x 4096
// at head_dim 64 26.2 us, 29.6 with the CTA's warps together (one row of 32768 29.8, 30.7).
constexpr std::uint32_t kFew = 32;
// What a row's end costs a CTA, in units: among shares (with 14: 16 x 4000 with 3 drafted
// tokens 52.2 us, 48.1 now; with none, a row of 32768 31.6, 29.4 now), and between the two kernels (with 20: 23 single tokens over 3000 beside
// a chunk of 512 97.9 us, 93.4 now).
constexpr int kRowCost = 20, kSplitRowCost = 14;

template <int HD>
struct Smem {
    static constexpr int kPitch = HD + 4;  // floats of a column, for the banks
    static constexpr int kRing = 0;        // [warp][stage][2 K boxes, 2 V boxes], 1024-byte aligned
    static constexpr int kFlush = kRing + kWarps * kStages * kStage;  // [warp][column][kPitch] f32
    static constexpr int kState = kWarps * kCols * kPitch * 4;
    static constexpr int kJoin = (kMaxCtas + 1) * kCols * kMaxSets * 4;  // [part][column] weights, 1 / sums
    static constexpr int kMl = kFlush + (kState > kJoin ? kState : kJoin);  // [warp][column][m, l] f32
    static constexpr int kBars = kMl + kWarps * kCols * 8;            // [warp][stage]
    static constexpr int kBad = kBars + kWarps * kStages * 8;         // [warp]
    static constexpr int kLast = kBad + kWarps * 4;
    static constexpr int kBytes = kLast + 16 + 1008;  // + alignment slack (of a 16-byte base)
    static_assert(kBytes <= 232448, "shared memory");
};

__device__ __forceinline__ void ldsm_x4(std::uint32_t addr, std::uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(std::uint32_t addr, std::uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// One warp's state over its units of a row: O^T (dimensions 16 i + lane / 4 and
// 8 more, columns 2 (lane % 4) and + 1 of each set), this lane's part of the sums
// and the reference maxima (log2 units).
template <int HD, int SETS>
struct State {
    float o[HD / 16][SETS][4];
    float m[SETS][2], l[SETS][2];
};

// P is held as 2^kShift times the probability relative to the reference, which a
// lane's sum of them passes by 2^8 at most: up to 2^15 in f16.
constexpr float kShift = 7.f;
constexpr float kMostSum = 32768.f;
// score * scale - reference is one fma with the rounded reference, off by up to
// 2^-24 of it; beyond this (log2 units) the score is rounded alike before it is
// subtracted, so that equal scores of any size weigh the same.
constexpr float kVast = 1024.f;

// One unit more, for SETS of the MOST sets.  `limit` holds how many of the unit's
// positions each of the lane's columns attends, where `masked` (some column does not
// attend all).
template <int HD, int SETS, int MOST>
__device__ __forceinline__ void attend(State<HD, MOST>& s, const std::uint32_t (&qf)[HD / 16][MOST][2],
                                       std::uint32_t stage, std::uint32_t koff,
                                       std::uint32_t voff, float sc, bool masked,
                                       const std::int32_t (&limit)[MOST][2]) {
    constexpr int T = 128 / HD;  // tiles of 16 positions
    const std::uint32_t lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    float x[T][SETS][4];
#pragma unroll
    for (int k = 0; k < T; ++k) {
#pragma unroll
        for (int c = 0; c < SETS; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[k][c][i] = 0.f;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) {
            // head_dim 128: box d / 4 holds dimensions 64 (d / 4) ..; 64: box k positions 16 k ..
            std::uint32_t a[4];
            ldsm_x4(stage + (HD == 128 ? d / 4 : k) * kBox + (koff ^ (d % 4 << 5)), a);
#pragma unroll
            for (int c = 0; c < SETS; ++c)
                attn8::mma_acc(x[k][c], a[0], a[1], a[2], a[3], qf[d][c][0], qf[d][c][1]);
        }
    }
    // positions g, g + 8 of each tile, columns 2 t, 2 t + 1
    const auto mask = [&](float (&y)[T][SETS][4]) {
#pragma unroll
        for (int k = 0; k < T; ++k)
#pragma unroll
            for (int c = 0; c < SETS; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (static_cast<std::int32_t>(16 * k + g + 8 * (i >> 1)) >= limit[c][i & 1]) y[k][c][i] = -INFINITY;
    };
    float p[T][SETS][4], sum[SETS][2];
    const auto weigh = [&] {
#pragma unroll
        for (int c = 0; c < SETS; ++c) {
#pragma unroll
            for (int i = 0; i < 2; ++i) sum[c][i] = 0.f;
#pragma unroll
            for (int k = 0; k < T; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[k][c][i] = attn8::ex2(p[k][c][i]);
                    sum[c][i & 1] += p[k][c][i];
                }
        }
    };
    bool again = false;
#pragma unroll
    for (int c = 0; c < SETS; ++c)
#pragma unroll
        for (int k = 0; k < T; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) p[k][c][i] = fmaf(x[k][c][i], sc, kShift - s.m[c][i & 1]);
    if (masked) mask(p);
    weigh();
#pragma unroll
    for (int c = 0; c < SETS; ++c)
        again |= !(sum[c][0] <= kMostSum && sum[c][1] <= kMostSum) ||
                 (s.m[c][0] != -INFINITY && fabsf(s.m[c][0]) > kVast) || (s.m[c][1] != -INFINITY && fabsf(s.m[c][1]) > kVast);
    if (__any_sync(0xffffffffu, again)) {
#pragma unroll
        for (int k = 0; k < T; ++k)
#pragma unroll
            for (int c = 0; c < SETS; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[k][c][i] *= sc;
        if (masked) mask(x);
#pragma unroll
        for (int c = 0; c < SETS; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float m = -INFINITY;
#pragma unroll
                for (int k = 0; k < T; ++k) m = fmaxf(m, fmaxf(x[k][c][h], x[k][c][2 + h]));
#pragma unroll
                for (int d = 4; d < 32; d *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
                m = fmaxf(m, s.m[c][h]);
                const float f = s.m[c][h] == m ? 1.f : attn8::ex2(s.m[c][h] - m);  // 0 from -infinity
                s.m[c][h] = m;
                s.l[c][h] *= f;
#pragma unroll
                for (int i = 0; i < HD / 16; ++i) s.o[i][c][h] *= f, s.o[i][c][2 + h] *= f;
                // still -infinity where no score is above it: weights of zero
                const float from = m == -INFINITY ? 0.f : m;
#pragma unroll
                for (int k = 0; k < T; ++k) {
                    p[k][c][h] = x[k][c][h] - from + kShift;
                    p[k][c][2 + h] = x[k][c][2 + h] - from + kShift;
                }
            }
        weigh();
    }
    std::uint32_t pt[T][SETS][2];
#pragma unroll
    for (int c = 0; c < SETS; ++c) {
        s.l[c][0] += sum[c][0], s.l[c][1] += sum[c][1];
#pragma unroll
        for (int k = 0; k < T; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                pt[k][c][i] = attn8::transpose8x8(attn8::half2_of(p[k][c][2 * i], p[k][c][2 * i + 1]));
    }
#pragma unroll
    for (int k = 0; k < T; ++k)
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) {
            std::uint32_t a[4];
            ldsm_x4_trans(stage + 2 * kBox + (HD == 128 ? d / 4 : k) * kBox + (voff ^ (d % 4 << 5)), a);
#pragma unroll
            for (int c = 0; c < SETS; ++c)
                attn8::mma_acc(s.o[d][c], a[0], a[1], a[2], a[3], pt[k][c][0], pt[k][c][1]);
        }
}

// Rows of a unit's V behind its first `live` positions become zeros, and values that
// are not finite too; whether there were any among the positions.  By a warp.
template <int HD>
__device__ __forceinline__ bool clean(std::uint8_t* v, std::int32_t live) {
    bool bad = false;

    for (std::uint32_t x = threadIdx.x & 31; x < 2 * kBox / 16; x += 32) {
        // 16-byte chunk x: row x / 8 of the two boxes (head_dim 128: of either)
        const std::int32_t pos = static_cast<std::int32_t>(HD == 128 ? x / 8 % 16 : x / 8);
        const uint4 y = reinterpret_cast<const uint4*>(v)[x];
        std::uint32_t w[4] = {y.x, y.y, y.z, y.w};
        bool any = pos >= live;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (pos >= live) w[e] = 0;
            if ((w[e] & 0x7c00u) == 0x7c00u) w[e] &= 0xffff0000u, any = bad = true;
            if ((w[e] & 0x7c000000u) == 0x7c000000u) w[e] &= 0x0000ffffu, any = bad = true;
        }
        if (any) reinterpret_cast<uint4*>(v)[x] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    fence_proxy_async_smem();  // before the next unit's load into the stage
    __syncwarp();
    return bad;
}

// A sequence where it is this kernel's (n 0 otherwise), and its units.
__device__ __forceinline__ Seq few_part(const Params& p, Seq s) {
    if (static_cast<std::uint64_t>(s.n) * p.group > p.few) s.n = 0;
    return s;
}
template <int HD>
__device__ __forceinline__ std::uint32_t units_of(const Seq& s) {
    constexpr std::uint32_t kUnit = 2048 / HD;
    return s.n == 0 ? 0u : (s.len + kUnit - 1) / kUnit;
}

// A row of the work list: sequence b and KV head r, the units, and the virtual
// unit at which it begins.
struct Row {
    std::uint32_t b, r, n;
    std::uint64_t begin;
    Seq s;
};

template <int HD, int SETS>
__global__ void __launch_bounds__(kThreads, 1)
    few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
               const Params p) {
    using L = Smem<HD>;
    constexpr int kUnit = 2048 / HD;  // positions
    constexpr int kPart = kCols * SETS * (HD + 2);
    extern __shared__ std::uint8_t smem_raw[];
    const std::uint32_t raw = smem_u32(smem_raw);
    const std::uint32_t sbase = (raw + 1023u) & ~1023u;
    std::uint8_t* const smem = smem_raw + (sbase - raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const std::uint32_t ring = sbase + L::kRing + warp * (kStages * kStage);
    std::uint64_t* const full = reinterpret_cast<std::uint64_t*>(smem + L::kBars) + warp * kStages;
    const std::uint32_t bars = smem_u32(full);
    float* const flush = reinterpret_cast<float*>(smem + L::kFlush);
    float* const ml = reinterpret_cast<float*>(smem + L::kMl);
    volatile std::uint32_t* bad_flags = reinterpret_cast<std::uint32_t*>(smem + L::kBad);
    volatile std::uint32_t* last_cta = reinterpret_cast<std::uint32_t*>(smem + L::kLast);
    const std::uint32_t sub = p.sub;  // loads of K in a unit, each of kUnit / sub positions
    if (lane < kStages) {
        mbar_init(&full[lane], sub);
        fence_mbarrier_init();
    }
    if (threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<std::uint64_t>(&map_k)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<std::uint64_t>(&map_v)) : "memory");
    }
    if (!p.shares) pdl_launch_dependents();
    pdl_wait();
    // (the other kernel, which starts then, may rely on what is before this one)
    if (p.shares) pdl_launch_dependents();

    const std::uint32_t batch = p.c.batch, bt = p.c.block_tokens, rows = p.c.kv_heads;
    // sequence b where it is this kernel's (n 0 otherwise)
    const auto mine = [&](std::uint32_t b) { return few_part(p, sequence(p, b)); };
    const auto units = [&](const Seq& s) { return units_of<HD>(s); };
    if (p.reports && blockIdx.x == gridDim.x - 1) report_bad(p, threadIdx.x, kThreads);
    // ---- the CTA's share --------------------------------------------------
    // Equal shares of the units, where a row's end counts as kRowCost units
    // more; or, where the rows are few, equal pieces of each row, one to a
    // CTA, of the smallest size (in small steps) that needs no more CTAs than
    // there are, unless shares are smaller by more than a row's end.
    std::uint32_t longest = 0, filled = 0;  // units, rows with any
    std::uint64_t total = 0, line = 0;      // units, and the other kernel's cost
    std::uint64_t per = 0;  // units of a CTA (past 2^32 where pages are shared without measure)
    std::uint32_t ctas = gridDim.x;
    bool pieces = false;
    const auto least = [&] { return min(longest, static_cast<std::uint32_t>(kMinUnits)); };
    const auto share = [&] {
        return max(share_of(total + static_cast<std::uint64_t>(filled) * kRowCost, ctas), static_cast<std::uint64_t>(least()));
    };
    const auto size = [&](std::uint32_t i, std::uint32_t steps) {  // pieces from the least on
        const std::uint32_t low = max(static_cast<std::uint32_t>(share_of(total, ctas)), least());
        return low + (low * i + steps - 1) / steps;
    };
    const auto extent = [&](std::uint32_t n) -> std::uint32_t {  // a row in virtual units
        const std::uint32_t piece = static_cast<std::uint32_t>(per);  // (of a row: at most 2^28)
        return pieces ? (n + piece - 1) / piece * piece : n == 0 ? 0 : n + kRowCost;
    };
    // sequences without positions
    for (std::uint32_t b = blockIdx.x; b < batch; b += gridDim.x) {
        const Seq s = mine(b);
        if (s.n > 0 && s.len == 0)
            for (std::uint32_t i = threadIdx.x; i < s.n * p.q_heads * (HD / 8); i += kThreads)
                reinterpret_cast<uint4*>(p.out + static_cast<std::uint64_t>(s.q0) * p.q_heads * HD)[i] =
                    make_uint4(0, 0, 0, 0);
    }
    const auto scan_up = [&](std::uint64_t x) {  // inclusive, over the warp
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const std::uint64_t y = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += y;
        }
        return x;
    };
    std::uint64_t u0, at_begin = 0;  // this CTA's first unit, and its sequence's
    std::uint32_t at_b = 0;
    if (batch <= kFew) {
        // every warp for itself, one sequence to a lane
        std::uint32_t n = 0;
        if (static_cast<std::uint32_t>(lane) < batch) {
            const Seq s = sequence(p, lane);
            n = units(few_part(p, s));
            if (p.shares) line = cost_of(p, s);
        }
        if (p.shares) line = __shfl_sync(0xffffffffu, scan_up(line), 31);
        longest = __reduce_max_sync(0xffffffffu, n);
        total = static_cast<std::uint64_t>(__reduce_add_sync(0xffffffffu, n)) * rows;
        filled = __popc(__ballot_sync(0xffffffffu, n > 0)) * rows;
        if (p.shares) ctas = few_ctas<HD>(ctas, total + static_cast<std::uint64_t>(filled) * kSplitRowCost, line);
        if (total == 0 || blockIdx.x >= ctas) return;
        per = share();
        if (filled <= ctas) {
            const std::uint32_t step = size(lane, 32);
            std::uint32_t need = 0;

            for (std::uint32_t b = 0; b < batch; ++b)
                need += (__shfl_sync(0xffffffffu, n, b) + step - 1) / step;
            const unsigned fits = __ballot_sync(0xffffffffu, need * rows <= ctas);
            const std::uint32_t best = __shfl_sync(0xffffffffu, step, fits ? __ffs(fits) - 1 : 0);
            pieces = fits != 0 && best <= per + kRowCost;
            if (pieces) per = best;
        }
        u0 = per * blockIdx.x;
        const std::uint64_t ext = extent(n), incl = scan_up(ext);
        const std::uint64_t begin = (incl - ext) * rows;
        const unsigned here = __ballot_sync(0xffffffffu, n > 0 && begin <= u0 && u0 < incl * rows);
        if (here == 0) return;  // past the last unit
        at_b = __ffs(here) - 1;
        at_begin = __shfl_sync(0xffffffffu, begin, at_b);
    } else {
        // the CTA together (scratch: the flush area)
        volatile std::uint64_t* found = reinterpret_cast<std::uint64_t*>(flush);  // [0..3], sums [4 + warp]
        volatile std::uint32_t* scan = reinterpret_cast<std::uint32_t*>(flush) + 64;  // [warp][2]

        for (std::uint32_t b = threadIdx.x; b < batch; b += kThreads) {
            const Seq s = sequence(p, b);
            const std::uint32_t n = units(few_part(p, s));
            if (p.shares) line += cost_of(p, s);
            total += n;
            filled += n > 0;
            longest = max(longest, n);
        }
        longest = __reduce_max_sync(0xffffffffu, longest);
        filled = __reduce_add_sync(0xffffffffu, filled);
        total = __shfl_sync(0xffffffffu, scan_up(total), 31);
        line = __shfl_sync(0xffffffffu, scan_up(line), 31);
        if (lane == 0) {
            found[4 + warp] = total;
            found[4 + kWarps + warp] = line;
            scan[2 * warp] = longest;
            scan[2 * warp + 1] = filled;
        }
        __syncthreads();
        total = 0, filled = 0, longest = 0, line = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            longest = max(longest, scan[2 * w]);
            total += found[4 + w];
            line += found[4 + kWarps + w];
            filled += scan[2 * w + 1];
        }
        total *= rows;
        filled *= rows;
        __syncthreads();
        if (p.shares) ctas = few_ctas<HD>(ctas, total + static_cast<std::uint64_t>(filled) * kSplitRowCost, line);
        if (total == 0 || blockIdx.x >= ctas) return;
        per = share();
        if (filled <= ctas) {
            const std::uint32_t step = size(warp, kWarps);
            std::uint32_t need = 0;

            for (std::uint32_t b = lane; b < batch; b += 32) need += (units(mine(b)) + step - 1) / step;
            need = __reduce_add_sync(0xffffffffu, need) * rows;
            if (lane == 0) scan[warp] = need <= ctas;
            __syncthreads();
            int w = 0;
            while (w < kWarps && !scan[w]) ++w;
            pieces = w < kWarps && size(w, kWarps) <= per + kRowCost;
            if (pieces) per = size(w, kWarps);
            __syncthreads();
        }
        u0 = per * blockIdx.x;
        std::uint64_t before = 0;  // extents of the sequences before the chunk
        if (threadIdx.x == 0) found[1] = 0;

        for (std::uint32_t base = 0;; base += kThreads) {
            const std::uint32_t b = base + threadIdx.x;
            const std::uint32_t n = b < batch ? units(mine(b)) : 0u;
            const std::uint64_t ext = extent(n), incl = scan_up(ext);
            if (lane == 31) found[4 + warp] = incl;
            __syncthreads();
            std::uint64_t lower = before;
            for (int w = 0; w < kWarps; ++w) {
                if (w < warp) lower += found[4 + w];
                before += found[4 + w];
            }
            const std::uint64_t end = (lower + incl) * rows, begin = (lower + incl - ext) * rows;
            if (n > 0 && begin <= u0 && u0 < end) {
                found[0] = begin;
                found[1] = 1;
                found[2] = b;
            }
            __syncthreads();
            if (found[1] || base + kThreads >= batch) break;
        }
        if (!found[1]) return;  // past the last unit
        at_b = static_cast<std::uint32_t>(found[2]), at_begin = found[0];
        __syncthreads();  // the scratch is read
    }
    const std::uint64_t u1 = u0 + per;
    // the next row with positions, begin ~0 behind the last; one sequence after another
    // (8 tokens over 1000: 14 us, 94 with 248 sequences without tokens behind them)
    const auto next = [&](Row& x) {
        x.begin += extent(x.n);
        if (++x.r < rows) return;
        x.r = 0;
        do {
            if (++x.b >= batch) {
                x.begin = ~0ull;
                return;
            }
            x.s = mine(x.b);
            x.n = units(x.s);
        } while (x.n == 0);
    };
    // this CTA's units [first, last) of a row
    const auto first_of = [&](const Row& x) {
        return x.begin >= u0 ? 0u : static_cast<std::uint32_t>(min(u0 - x.begin, static_cast<std::uint64_t>(x.n)));
    };
    const auto last_of = [&](const Row& x) {
        return static_cast<std::uint32_t>(min(u1 - x.begin, static_cast<std::uint64_t>(x.n)));
    };
    Row row;
    row.b = at_b;
    row.s = mine(row.b);
    row.n = units(row.s);
    row.r = static_cast<std::uint32_t>((u0 - at_begin) / extent(row.n));
    row.begin = at_begin + static_cast<std::uint64_t>(row.r) * extent(row.n);

    // ---- the stream: each warp keeps its ring full, across rows -------------
    // the blocks of 32 / sub units of this warp, from held_unit of sequence held_b
    // on: one lane for each load
    std::uint32_t a_unit = first_of(row) + warp, a_last = last_of(row), a_slot = 0, a_stage = 0;
    Row ahead = row;
    std::int32_t held_block = -1;
    std::uint32_t held_row = 0, held_b = ~0u, held_unit = 0;
    const auto issue = [&]() {

        while (a_unit >= a_last) {
            if (ahead.begin >= u1) return;
            next(ahead);
            if (ahead.begin >= u1) return;
            a_unit = warp, a_last = last_of(ahead), a_slot = 0;
        }
        if (a_slot == 0 && (held_b != ahead.b || held_unit != a_unit)) {
            held_b = ahead.b, held_unit = a_unit;
            const std::uint32_t pos = sub == 1 ? (a_unit + lane * kWarps) * kUnit
                                               : (a_unit + lane / 2 * kWarps) * kUnit + 16 * (lane % 2);
            held_block = -1;
            if (pos < ahead.s.len) {
                const std::uint32_t i = pos / bt;
                held_row = pos - i * bt;
                held_block = fetch(p, p.tables + static_cast<std::uint64_t>(ahead.b) * p.c.max_blocks + i);
                if (held_block < 0 || static_cast<std::uint64_t>(held_block) >= p.c.num_blocks) {
                    held_block = -1;
                    atomicOr(&g_device_status, kDevIndexOutOfRange);
                }
            }
        }
        const std::uint32_t i = lane - a_slot;
        if (i < sub) {
            const std::uint32_t bar = bars + 8 * a_stage;
            const std::uint32_t kt = ring + a_stage * kStage + i * kBox;
            // (what is not there reads as zeros)
            const int y = held_block < 0 ? kNowhere
                                         : static_cast<int>((static_cast<std::uint32_t>(held_block) * p.c.kv_heads + ahead.r) * bt + held_row);
            attn8::mbar_expect(bar, kStage / sub);
            attnp::tma_load_3d(kt, &map_k, 0, y, 0, bar);
            attnp::tma_load_3d(kt + 2 * kBox, &map_v, 0, y, 0, bar);
        }
        a_unit += kWarps;
        a_slot = (a_slot + sub) % 32;
        a_stage = a_stage == kStages - 1 ? 0 : a_stage + 1;
    };
    __syncwarp();

    for (int k = 0; k < kStages - 1; ++k) issue();

    // Q^T as the B operand: dimensions 16 d + 2 t, + 1 and 8 more of column g of each set
    std::uint32_t qf[HD / 16][SETS][2];
    const auto load_q = [&](const Row& x) {
#pragma unroll
        for (int c = 0; c < SETS; ++c) {
            const std::uint32_t col = kCols * c + g, i = col / p.group, h = col - i * p.group;
            const bool in = i < x.s.n;
            const std::uint32_t* src = reinterpret_cast<const std::uint32_t*>(
                p.q + ((static_cast<std::uint64_t>(x.s.q0) + i) * p.q_heads + x.r * p.group + h) * HD);
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) {
                qf[d][c][0] = in ? __ldg(src + 8 * d + t) : 0u;
                qf[d][c][1] = in ? __ldg(src + 8 * d + 4 + t) : 0u;
            }
        }
    };
    if (first_of(row) >= last_of(row)) next(row);  // only that row's end falls to this CTA
    if (row.begin < u1) load_q(row);
    // ldmatrix: matrix lane / 8, its row lane % 8.  K: positions 0-7, 8-15 of
    // dimensions 0-7, then of 8-15; V (transposed): dimensions 0-7, 8-15 of
    // positions 0-7, then of 8-15; a 16-byte chunk's place in its 128-byte line is
    // exchanged by the line's number
    const std::uint32_t mi = lane >> 3, mr = lane & 7;
    const std::uint32_t koff = ((mi & 1) * 8 + mr) * 128 + (((mi >> 1) ^ mr) << 4);
    const std::uint32_t voff = ((mi >> 1) * 8 + mr) * 128 + (((mi & 1) ^ mr) << 4);
    std::uint32_t stage = 0, parity = 0;
    bool waiting = true;
    while (row.begin < u1) {
        const std::uint32_t v0 = first_of(row), v1 = last_of(row);
        const Seq seq = row.s;
        const std::uint32_t cols = seq.n * p.group, sets = (cols + kCols - 1) / kCols;
        State<HD, SETS> s;
        std::int32_t limit[SETS][2];  // positions that each column attends
#pragma unroll
        for (int c = 0; c < SETS; ++c) {
#pragma unroll
            for (int i = 0; i < HD / 16; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) s.o[i][c][k] = 0.f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                s.m[c][h] = -INFINITY, s.l[c][h] = 0.f;
                const std::uint32_t tok = min((kCols * c + 2 * t + h) / p.group, seq.n - 1);
                limit[c][h] = static_cast<std::int32_t>(seq.len - seq.n + tok + 1);
            }
        }
        // positions that every column attends: what follows is looked through
        const std::uint32_t all = static_cast<std::uint32_t>(max(static_cast<std::int32_t>(seq.len - seq.n + 1), 0));
        bool bad = false;
        for (std::uint32_t v = v0 + warp; v < v1; v += kWarps) {
            if (waiting) waiting = mbar_wait_bounded(&full[stage], parity, &g_device_status);
            __syncwarp();  // the unit has landed; the stage before it is read by all lanes
            if (waiting) issue();  // (a stage whose copies are late gets no more)
            const std::int32_t from = static_cast<std::int32_t>(v * kUnit);
            const bool masked = v * kUnit + kUnit > all;  // (up to 2^31)
            std::int32_t here[SETS][2];
#pragma unroll
            for (int c = 0; c < SETS; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h) here[c][h] = limit[c][h] - from;
            if (masked)
                bad |= clean<HD>(smem + L::kRing + (warp * kStages + stage) * kStage + 2 * kBox,
                                 static_cast<std::int32_t>(seq.len) - from);
            if (SETS == 1 || sets == 1)
                attend<HD, 1, SETS>(s, qf, ring + stage * kStage, koff, voff, p.scale_log2, masked, here);
            else
                attend<HD, SETS, SETS>(s, qf, ring + stage * kStage, koff, voff, p.scale_log2, masked, here);
            if (++stage == kStages) stage = 0, parity ^= 1;
        }

        // ---- the warps' states meet, a set of columns at a time -------------
        // (the ring already holds the next row's units, and its queries load)
        const std::uint32_t kvh = row.r, b = row.b;
        const bool whole = v0 == 0 && v1 == row.n;
        const std::uint32_t cta0 = static_cast<std::uint32_t>(row.begin / per);
        const std::uint32_t count = static_cast<std::uint32_t>((row.begin + row.n - 1) / per) - cta0 + 1;
        next(row);
        if (row.begin < u1) load_q(row);
        bad = __any_sync(0xffffffffu, bad);
        if (lane == 0) bad_flags[warp] = bad;
        // what a column's sum of weights divides by; nothing attended: zeros
        const auto inverse = [&](float sum, std::uint32_t col) {
            return seq.len + col / p.group < seq.n ? 0.f : 1.f / sum;
        };
        const auto out_of = [&](std::uint32_t col) {
            const std::uint32_t i = col / p.group, h = col - i * p.group;
            return p.out + ((static_cast<std::uint64_t>(seq.q0) + i) * p.q_heads + kvh * p.group + h) * HD;
        };
        float* part = p.parts + static_cast<std::uint64_t>(2 * blockIdx.x + (v0 == 0 ? 1 : 0)) * kPart;
#pragma unroll
        for (int c = 0; c < SETS; ++c) {
            if (c > 0 && c >= sets) break;
            if (c > 0) __syncthreads();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int d = 4; d < 32; d *= 2) s.l[c][h] += __shfl_xor_sync(0xffffffffu, s.l[c][h], d);
                float* mine_f = flush + (warp * kCols + 2 * t + h) * L::kPitch + g;
#pragma unroll
                for (int i = 0; i < HD / 16; ++i) mine_f[16 * i] = s.o[i][c][h], mine_f[16 * i + 8] = s.o[i][c][2 + h];
                if (g == 0)
                    *reinterpret_cast<float2*>(ml + (warp * kCols + 2 * t + h) * 2) = make_float2(s.m[c][h], s.l[c][h]);
            }
            __syncthreads();
            bool any_bad = false;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) any_bad |= bad_flags[w] != 0;

            for (std::uint32_t x = threadIdx.x; x < kCols * (HD / 2); x += kThreads) {
                const std::uint32_t hq = x / (HD / 2), d = x % (HD / 2) * 2, col = kCols * c + hq;
                if (col >= cols) break;
                float mt = -INFINITY, lt = 0.f;
                float2 o = make_float2(0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) mt = fmaxf(mt, ml[(w * kCols + hq) * 2]);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    // a warp without a position has -infinity and zeros (NaN
                    // scores keep -infinity, and their NaN sums)
                    const float2 a = *reinterpret_cast<const float2*>(ml + (w * kCols + hq) * 2);
                    const float fw = a.y != a.y || a.x == mt ? 1.f : attn8::ex2(a.x - mt);
                    const float2 y = *reinterpret_cast<const float2*>(flush + (w * kCols + hq) * L::kPitch + d);
                    lt = fmaf(a.y, fw, lt);
                    o.x = fmaf(y.x, fw, o.x), o.y = fmaf(y.y, fw, o.y);
                }
                if (any_bad) {
                    // what was taken out of the V that this column attends
                    const std::uint32_t reach = min(static_cast<std::uint32_t>(max(static_cast<std::int32_t>(seq.len - seq.n + col / p.group + 1), 0)), v1 * kUnit);

                    for (std::uint32_t pos = max(all / kUnit, v0) * kUnit; pos < reach; ++pos) {
                        const std::int32_t blk = __ldg(p.tables + static_cast<std::uint64_t>(b) * p.c.max_blocks + pos / bt);
                        if (blk < 0 || static_cast<std::uint64_t>(blk) >= p.c.num_blocks) continue;
                        const __half* src = p.v_cache + ((static_cast<std::uint64_t>(blk) * p.c.kv_heads + kvh) * bt + pos % bt) * HD + d;
                        const float y0 = __half2float(src[0]), y1 = __half2float(src[1]);
                        if (!isfinite(y0)) o.x += y0;
                        if (!isfinite(y1)) o.y += y1;
                    }
                }
                if (whole) {
                    const float inv = inverse(lt, col);
                    *reinterpret_cast<std::uint32_t*>(out_of(col) + d) = attn8::half2_of(o.x * inv, o.y * inv);
                } else {
                    *reinterpret_cast<float2*>(part + col * HD + d) = o;
                    if (d == 0)
                        *reinterpret_cast<float2*>(part + kCols * SETS * HD + 2 * col) = make_float2(mt, lt);
                }
            }
        }
        if (!whole) {
            __syncthreads();
            if (threadIdx.x == 0) {
                __threadfence();  // the CTA's part, which the barrier has gathered
                const unsigned done = atomicAdd(p.counters + cta0, 1u);
                if (done == count - 1) p.counters[cta0] = 0;
                *last_cta = done == count - 1;
                __threadfence();
            }
            __syncthreads();
            if (*last_cta) {
                // the last of the row's CTAs joins the parts: weights, then sums
                // over every `groups`-th part, then over the groups
                const auto part_of = [&](std::uint32_t j) {
                    return p.parts + static_cast<std::uint64_t>(2 * (cta0 + j) + (j == 0 ? 1 : 0)) * kPart;
                };
                float* invs = flush;                    // [columns]
                float* wts = flush + kCols * kMaxSets;  // [count][columns]

                for (std::uint32_t col = warp; col < cols; col += kWarps) {
                    const auto ml_of = [&](std::uint32_t j) {
                        return __ldcg(reinterpret_cast<const float2*>(part_of(j) + kCols * SETS * HD) + col);
                    };
                    constexpr int kHeld = kMaxCtas / 32;
                    float2 held[kHeld];
                    float mt = -INFINITY, lt = 0.f;
#pragma unroll
                    for (int k = 0; k < kHeld; ++k) {
                        held[k] = lane + 32 * k < count ? ml_of(lane + 32 * k) : make_float2(-INFINITY, 0.f);
                        mt = fmaxf(mt, held[k].x);
                    }
                    mt = attn8::warp_max(mt);
#pragma unroll
                    for (int k = 0; k < kHeld; ++k)
                        if (lane + 32 * k < count) {
                            const float w = held[k].y != held[k].y || held[k].x == mt ? 1.f : attn8::ex2(held[k].x - mt);
                            lt += held[k].y * w;
                            wts[(lane + 32 * k) * cols + col] = w;
                        }
#pragma unroll
                    for (int d = 16; d > 0; d /= 2) lt += __shfl_xor_sync(0xffffffffu, lt, d);
                    if (lane == 0) invs[col] = inverse(lt, col);
                }
                __syncthreads();
                const auto sum_of = [&](std::uint32_t cell, std::uint32_t first, std::uint32_t step) {
                    const std::uint32_t col = cell / (HD / 4), d = cell % (HD / 4) * 4;
                    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
                    constexpr int kAhead = SETS == 1 ? 6 : 4;  // loads in flight

                    for (std::uint32_t j0 = first; j0 < count; j0 += kAhead * step) {
                        float4 y[kAhead];
#pragma unroll
                        for (int k = 0; k < kAhead; ++k)
                            if (j0 + k * step < count) y[k] = __ldcg(reinterpret_cast<const float4*>(part_of(j0 + k * step) + col * HD + d));
#pragma unroll
                        for (int k = 0; k < kAhead; ++k) {
                            if (j0 + k * step >= count) break;
                            const float w = wts[(j0 + k * step) * cols + col];
                            o.x = fmaf(y[k].x, w, o.x), o.y = fmaf(y[k].y, w, o.y);
                            o.z = fmaf(y[k].z, w, o.z), o.w = fmaf(y[k].w, w, o.w);
                        }
                    }
                    return o;
                };
                const auto store = [&](std::uint32_t cell, const float4& o) {
                    const std::uint32_t col = cell / (HD / 4), d = cell % (HD / 4) * 4;
                    const float inv = invs[col];
                    *reinterpret_cast<uint2*>(out_of(col) + d) =
                        make_uint2(attn8::half2_of(o.x * inv, o.y * inv), attn8::half2_of(o.z * inv, o.w * inv));
                };
                const std::uint32_t cells = cols * (HD / 4);
                if (cells > kThreads / 2) {

                    for (std::uint32_t x = threadIdx.x; x < cells; x += kThreads) store(x, sum_of(x, 0, 1));
                } else {
                    // groups of threads take every groups-th part, and add up theirs
                    const std::uint32_t groups = kThreads / cells;
                    float4* red = reinterpret_cast<float4*>(wts + ((count * cols + 3) & ~3u));  // [kThreads]
                    if (threadIdx.x < cells * groups)
                        red[threadIdx.x] = sum_of(threadIdx.x % cells, threadIdx.x / cells, groups);
                    __syncthreads();
                    if (threadIdx.x < cells) {
                        float4 o = red[threadIdx.x];

                        for (std::uint32_t k = 1; k < groups; ++k) {
                            const float4 y = red[threadIdx.x + k * cells];
                            o.x += y.x, o.y += y.y, o.z += y.z, o.w += y.w;
                        }
                        store(threadIdx.x, o);
                    }
                }
            }
        }
        __syncthreads();  // the flush area is free again
    }
    if (!waiting) let_copies_land();
}

}  // namespace few

// The cache as rows of a head, 64 dimensions at a time: boxes of `rows` rows and
// `halves` times 64 dimensions, one behind the other.
inline int make_map(CUtensorMap* map, const void* cache, const kvq8::CacheShape& c, std::uint32_t rows,
                    std::uint32_t halves) {
    auto encode = gemm::encode_fn();
    if (encode == nullptr) return static_cast<int>(cudaErrorNotSupported);
    const std::uint64_t all = c.num_blocks * c.kv_heads * c.block_tokens;
    const cuuint32_t box[3] = {64, rows, halves};
    const cuuint64_t dims[3] = {64, all < rows ? rows : all, c.head_dim / 64};  // no blocks: never loaded
    const cuuint64_t strides[2] = {c.head_dim * 2ull, 128};
    const cuuint32_t estr[3] = {1, 1, 1};
    if (encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(cache), dims, strides, box,
               estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return kInvalidValue;
    return kSuccess;
}

inline int sm_count(int& n) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return static_cast<int>(e);
}

namespace few {

// Query rows of a KV head that the kernel takes.  With four sets of columns 16 sequences
// of 4000 with 5 and 8 tokens of 4 grouped heads took 98 and 104 us at head_dim 128
// (registers spill), the chunk kernel takes 72 and 73; at head_dim 64 (32 of 4000, 6
// tokens) 73 against 96, for which alone more code is not kept.
constexpr std::uint32_t kMostRows = kCols * kMaxSets;

template <int HD, int SETS>
int launch(const Params& p, const void* k_cache, int ctas, cudaStream_t stream) {
    CUtensorMap map_k{}, map_v{};
    int st = make_map(&map_k, k_cache, p.c, 2048 / HD / p.sub, HD / 64);
    if (st == kSuccess) st = make_map(&map_v, p.v_cache, p.c, 2048 / HD / p.sub, HD / 64);
    if (st != kSuccess) return st;
    static std::atomic<std::uint64_t> done{0};
    st = ensure_dynamic_smem(few_kernel<HD, SETS>, Smem<HD>::kBytes, done);
    if (st != kSuccess) return st;
    return launch_pdl_smem(few_kernel<HD, SETS>, dim3(static_cast<unsigned>(ctas)), dim3(kThreads),
                           Smem<HD>::kBytes, stream, map_k, map_v, p);
}

}  // namespace few
}  // namespace attnpg
}  // namespace mote

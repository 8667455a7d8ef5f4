// Decode attention over the 8-bit paged cache (kv_cache_q8.cu): one query
// token per sequence,
//   out[b, h] = softmax(scale * q[b, h] . K_b[:len_b, h / g]) . V_b
// with K = qk * sk, V = qv * sv (8-bit integers times the scale of their block
// and head).
//
// HBM-bound: K and V of the attended positions are read once for up to 8 query
// heads of a KV head, which share the read (a larger group reads them once for
// each eight).  Everything else is arranged so that the stream never waits:
// * The work is cut in units of 4096 / head_dim positions of one (sequence, KV
//   head, up to 8 query heads) "row".  One CTA per SM takes an equal share of
//   consecutive units, found from the lengths on the device, so ragged batches
//   balance and the host needs no bound on the lengths.  The 12 warps of a CTA take a row's units in turn, each through a
//   ring of 16 KB that runs ahead across rows; the lane that holds a block's
//   number issues its TMA loads (128-byte swizzle) and its scales.
// * The 8-bit values become f16 exactly (the byte as the low bits of
//   1024 + u, minus 1152) and feed mma.sync.m16n8k16 as the A operand:
//   S^T = K Q^T with 16 positions as rows and 8 heads as columns, then
//   O^T += V^T P^T with 16 dimensions as rows, so no row of the products is
//   idle whatever the grouping.  K's dimensions and V's positions are taken
//   in the order in which a thread's wide shared loads hold them without bank
//   conflicts (the products do not depend on it); P^T gets from the
//   accumulator layout to the operand's with movmatrix.
// * scale * sk multiplies S in f32; sv multiplies P before it is split into f16
//   high and low parts (two products).  For each head, O is held in a unit, a
//   power of two, that keeps the products P * sv at hand within f16's range
//   whatever the sizes of V and of the weights before; it moves both ways.
//   The running maximum and the unit move only when a P passes 2^8 or the
//   products leave the range, so a step costs one vote instead of reductions.
// * Rows that lie in several CTAs leave unnormalised parts in the workspace;
//   the last CTA to finish joins them in order (a counter per row, left at
//   zero), so results do not depend on timing.
// Measured at 32 query / 8 KV heads: one sequence of 32768 (head_dim 128, 67 MB)
// 20.4 us, of which the stream is 11 us (0.94 of the copy bandwidth); 16 x 4096
// at head_dim 64 20.3 us; 48 ragged up to 8192 at head_dim 128 (404 MB) 84 us,
// 0.73 of the copy bandwidth (82 us with one unit for all heads that followed
// V's scales alone, which lost the small V's bits).  head_dim 64 is bound by
// the dependent steps between the 8-bit values and the products at three warps
// a scheduler (0.46 issues a cycle, 1048 instructions a warp for 64 positions;
// stalls on fixed latencies 1.7 an issue, on loads 0.9, on a busy pipe 0.6):
// dequantizing takes 5 instructions for 4 bytes.
// Every wait is bounded; one that expires is reported in the device status
// and the lane runs on without waiting and without further copies.
#include "mote_common.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

namespace mote {
namespace attn8 {

constexpr int kWarps = 12;
constexpr int kThreads = 32 * kWarps;
constexpr int kHeads = 8;     // query heads of a row (columns of the products)
constexpr int kTile = 4096;   // bytes of K (and of V) in a unit: 4096 / head_dim positions
constexpr int kStages = 2;
constexpr int kMaxCtas = 512;
constexpr int kMinUnits = 2 * kWarps;  // rows of up to this many units are not split
// Sequences up to which every warp finds the CTA's share alone, one sequence to
// a lane: 4 sequences of 2000 take 12.0 us against 12.9 by the CTA together, 16
// ragged ones 20.6 against 21.3, 32 36.2 against 37.0.
constexpr std::uint32_t kFew = 32;
// What a row's end costs a CTA, in units: 14 against 8 and 20 measured 52.6
// against 55.3 and 53.7 us (48 ragged sequences up to 8192, head_dim 64), 82.5
// against 89.6 and 79.0 (the same at 128), 43.3 against 48.4 and 44.3 (100 up to
// 2000, 64), 42.8 against 45.7 and 43.5 (128 of 100 to 600, 128).
constexpr int kRowCost = 14;

struct Params {
    const __half* q;
    const float* k_scales;
    const float* v_scales;
    const std::int32_t* tables;
    const std::int32_t* seq_lens;
    __half* out;
    kvq8::CacheShape c;
    std::uint32_t q_heads, group, head_groups;
    float scale_log2;
    unsigned* counters;  // [kMaxCtas], zero between calls
    float* parts;        // [2 * CTAs][kHeads * (HD + 2)]
};

struct Smem {
    static constexpr int kRing = 0;  // [warp][stage][K tile, V tile], 1024-byte aligned
    static constexpr int kFlush = kRing + kWarps * kStages * 2 * kTile;  // [warp][4 heads][HD] f32
    static constexpr int kMl = kFlush + kWarps * 4 * 128 * 4;   // [warp][4 heads][m, l] f32
    static constexpr int kScales = kMl + kWarps * 4 * 8;        // [warp][stage][4 tiles][K, V] f32
    static constexpr int kBars = kScales + kWarps * kStages * 32;  // [warp][stage]
    static constexpr int kLast = kBars + kWarps * kStages * 8;
    static constexpr int kBytes = kLast + 16 + 1008;  // + alignment slack (of a 16-byte base)
};
static_assert(Smem::kBytes <= 232448, "shared memory");
static_assert((kMaxCtas * kHeads + kThreads * 4 + kHeads) * 4 <= Smem::kMl - Smem::kFlush, "the join's scratch");

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
    for (int d = 16; d > 0; d /= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
    return x;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ std::uint32_t transpose8x8(std::uint32_t a) {
    std::uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

__device__ __forceinline__ std::uint32_t half2_of(float a, float b) {
    std::uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
    return d;
}

// Bytes (0, 1) or (2, 3) of w (each 128 + value) as a pair of f16 values.
__device__ __forceinline__ std::uint32_t bytes_to_half2(std::uint32_t w, std::uint32_t sel) {
    return hsub2_u32(prmt(w, 0x64646464u, sel), 0x64806480u);
}

template <int OFF>
__device__ __forceinline__ uint4 lds128i(std::uint32_t base) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4+%5];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(base), "n"(OFF));
    return v;
}
__device__ __forceinline__ uint4 lds128(std::uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr));
    return v;
}

__device__ __forceinline__ void tma_load_2d(std::uint32_t dst, const CUtensorMap* map, int x,
                                            int y, std::uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void cp_async_4(std::uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

__device__ __forceinline__ void mbar_expect(std::uint32_t bar, std::uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// One arrival on `bar` when this thread's copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(std::uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void mbar_arrive(std::uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void mma_acc(float (&d)[4], std::uint32_t a0, std::uint32_t a1,
                                        std::uint32_t a2, std::uint32_t a3, std::uint32_t b0,
                                        std::uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ std::uint64_t mul_f32x2(std::uint64_t a, std::uint64_t b) {
    std::uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Where a tile of 16 positions lies in shared memory (the 128-byte swizzle: a
// 16-byte chunk's place in its 128-byte line is exchanged by the line's number)
// and which positions a thread's rows and columns of the products stand for.
// head_dim 128: position r is line r, row r of S^T is position r; a thread's
// K chunks are 2 t and 2 t + 1.  head_dim 64: two positions to a line, rows
// 2 i and 2 i + 1 of S^T are the positions i % 2 + 4 (i / 2) and that ^ 3.
// Either way a quarter of a warp (half, for 8-byte loads) meets all 32 banks.
template <int HD>
struct Tile {
    static __device__ __forceinline__ std::uint32_t at(std::uint32_t r, std::uint32_t c) {
        return HD == 128 ? r * 128 + ((c ^ (r & 7)) << 4)
                         : (r >> 1) * 128 + ((((r & 1) << 2 | c) ^ ((r >> 1) & 7)) << 4);
    }
    // the position of row 2 i + e, i < 4 (rows 8 + 2 i + e: 8 more)
    static __device__ __forceinline__ std::uint32_t position(std::uint32_t i, std::uint32_t e) {
        return HD == 128 ? 2 * i + e : ((i & 1) + 4 * (i >> 1)) ^ (3 * e);
    }
};

// What a lane reads of a tile of 16 positions, as bytes from its start (the
// rest is immediate: head_dim 128 has the positions 8 further 1024 bytes on).
template <int HD>
struct Offsets {
    std::uint32_t k[2];            // head_dim 128: chunks 2 t, 2 t + 1; 64: positions r, r + 8
    std::uint32_t v[HD == 128 ? 2 : 4];
    __device__ __forceinline__ explicit Offsets(std::uint32_t lane) {
        const std::uint32_t g = lane >> 2, t = lane & 3;
        const std::uint32_t r0 = Tile<HD>::position(g >> 1, g & 1);
        if constexpr (HD == 128) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                k[i] = Tile<HD>::at(r0, 2 * t + i);
                v[i] = Tile<HD>::at(Tile<HD>::position(t, i), g);
            }
        } else {
            k[0] = Tile<HD>::at(r0, t), k[1] = Tile<HD>::at(r0 + 8, t);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] = Tile<HD>::at(Tile<HD>::position(t, i & 1) + 8 * (i >> 1), g >> 1) + 8 * (g & 1);
        }
    }
};

// One warp's state over its units of a row: O^T accumulators (dimension
// HD / 8 * (lane / 4) + 2 i + e of heads 2 (lane % 4), + 1), this lane's part
// of the sums, the reference maxima and the units in which O is held.
template <int HD>
struct State {
    float o[HD / 16][4];
    float m[2], l[2];
    float w[2];  // powers of two: O is held times w
};

// A score less the reference is one fma of the unscaled score, whose rounded
// reference leaves up to 2^-25 of it; beyond this (log2 units) the score is
// rounded alike before it is subtracted, so that equal scores of any size weigh
// the same.
constexpr float kVast = 65536.f;

// P * sv * w is split into f16 high and low parts, off by 2^-25 at most (and by
// 2^-22 of the value above 2^-3).  The largest of a lane's products of a step
// stays in this range, so that is 2^-19 of the step's largest.  Steps of less
// are left in the unit where V is of ordinary size (scales up to kOrdinary, |v|
// up to 127) and a weight of 1 makes a product of kLeastOne or more: weights are
// then off by 2^-27 of the row's largest, and scores that spread widely do not
// move the unit up and down.  A step whose two tiles have scales further apart
// than kApart (a block of large values beside one of small ones) is taken as two.
constexpr float kMostProduct = 32768.f, kLeastProduct = 0x1p-6f, kLeastOne = 4.f;
constexpr float kOrdinary = 1.f, kApart = 64.f;
constexpr int kProductExponent = 6;  // of the largest where a unit is chosen

// 32 positions more, the first `live` of them attended, in two tiles of 16
// whose scores are S times f0 and f1 and whose V scales are sv0 and sv1
// (-infinity: the tile's block is not there).
template <int HD>
__device__ __forceinline__ void attend32(State<HD>& s, const std::uint32_t (&qf)[HD / 8],
                                         const Offsets<HD>& off, std::uint32_t ktile,
                                         std::uint32_t vtile, float f0, float f1, float sv0,
                                         float sv1, std::int32_t live) {
    const std::uint32_t lane = threadIdx.x & 31, g = lane >> 2;
    const std::uint32_t r0 = Tile<HD>::position(g >> 1, g & 1);
    const std::uint32_t ka = ktile + off.k[0], kb = ktile + off.k[1];
    float acc[2][4];
    const auto score = [&](int k, int j, const uint4& a, const uint4& b) {
        const std::uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const std::uint32_t xa = aw[i] ^ 0x80808080u, xb = bw[i] ^ 0x80808080u;
            mma_acc(acc[k], bytes_to_half2(xa, 0x4140u), bytes_to_half2(xb, 0x4140u),
                    bytes_to_half2(xa, 0x4342u), bytes_to_half2(xb, 0x4342u),
                    qf[(4 * j + i) * 2], qf[(4 * j + i) * 2 + 1]);
        }
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[0][i] = acc[1][i] = 0.f;
    if constexpr (HD == 128) {
        const uint4 a0 = lds128i<0>(ka), b0 = lds128i<1024>(ka), a1 = lds128i<2048>(ka), b1 = lds128i<3072>(ka);
        score(0, 0, a0, b0), score(1, 0, a1, b1);
        const uint4 c0 = lds128i<0>(kb), d0 = lds128i<1024>(kb), c1 = lds128i<2048>(kb), d1 = lds128i<3072>(kb);
        score(0, 1, c0, d0), score(1, 1, c1, d1);
    } else {
        const uint4 a0 = lds128i<0>(ka), b0 = lds128i<0>(kb), a1 = lds128i<1024>(ka), b1 = lds128i<1024>(kb);
        score(0, 0, a0, b0), score(1, 0, a1, b1);
    }
    // scores above the reference maxima, +infinity (or NaN) before there is one
    float x[2][4];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[k][i] = fmaf(acc[k][i], k ? f1 : f0, -s.m[i & 1]);
    const bool tail = live < 32 || sv0 == -INFINITY || sv1 == -INFINITY;  // uniform
    const auto mask = [&](float (&y)[2][4]) {
        const std::int32_t n0 = sv0 == -INFINITY ? 0 : live, n1 = sv1 == -INFINITY ? 0 : live - 16;
        const std::int32_t r = static_cast<std::int32_t>(r0);
        if (r >= n0) y[0][0] = y[0][1] = -INFINITY;
        if (r + 8 >= n0) y[0][2] = y[0][3] = -INFINITY;
        if (r >= n1) y[1][0] = y[1][1] = -INFINITY;
        if (r + 8 >= n1) y[1][2] = y[1][3] = -INFINITY;
    };
    if (tail) mask(x);
    // P, its sums, and its products with V's scales (0 where there is no block)
    const float v0 = tail && sv0 == -INFINITY ? 0.f : sv0, v1 = tail && sv1 == -INFINITY ? 0.f : sv1;
    float a[2][4], sum[2];
    const auto weigh = [&] {  // x becomes P (infinity before there is a maximum)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[k][i] = ex2(x[k][i]);
        const auto pair = [&](int k, int i) { return attnp::pack_f32x2(x[k][i], x[k][i + 1]); };
        attnp::unpack_f32x2(attnp::add_f32x2(attnp::add_f32x2(pair(0, 0), pair(0, 2)),
                                             attnp::add_f32x2(pair(1, 0), pair(1, 2))),
                            sum[0], sum[1]);
    };
    const auto scale = [&] {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const float v = k ? v1 : v0;
                const std::uint64_t unit = mul_f32x2(attnp::pack_f32x2(v, v), attnp::pack_f32x2(s.w[0], s.w[1]));
                attnp::unpack_f32x2(mul_f32x2(attnp::pack_f32x2(x[k][i], x[k][i + 1]), unit), a[k][i], a[k][i + 1]);
            }
    };
    weigh();
    scale();
    const float a0 = fmaxf(attnp::max3f(a[0][0], a[0][2], a[1][0]), a[1][2]);
    const float a1 = fmaxf(attnp::max3f(a[0][1], a[0][3], a[1][1]), a[1][3]);
    // ordinary V: fine enough where a weight of 1 is well inside the range
    const float u = fmaxf(v0, v1) <= kOrdinary ? fminf(v0, v1) * (kLeastProduct / kLeastOne) : 0.f;
    const float b0 = fmaxf(a0, s.w[0] * u), b1 = fmaxf(a1, s.w[1] * u);
    if (__any_sync(0xffffffffu, fmaxf(sum[0], sum[1]) > 256.f || fmaxf(a0, a1) > kMostProduct ||
                                    !(fminf(b0, b1) >= kLeastProduct) ||
                                    fmaxf(fabsf(s.m[0]), fabsf(s.m[1])) > kVast)) {
        float y[2][4];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) y[k][i] = acc[k][i] * (k ? f1 : f0);
        if (tail) mask(y);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float m = fmaxf(fmaxf(y[0][h], y[0][2 + h]), fmaxf(y[1][h], y[1][2 + h]));
#pragma unroll
            for (int d = 4; d < 32; d *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
            const float here = m;
            m = fmaxf(m, s.m[h]);
            float f = s.m[h] == m ? 1.f : ex2(s.m[h] - m);  // 0 from -infinity
            s.m[h] = m;
            s.l[h] *= f;
            // another unit where the step's largest product is not near the middle
            // of the range.  Up to 2^64, so that O stays finite (V and P below 2^17
            // and 2^8, 2^31 positions): products that are below the range even
            // then add less than 2^-60 to outputs that end in f16
            const float c = ex2(here - m) * fmaxf(v0, v1);
            const bool fine = (c * s.w[h] >= 1.f || s.w[h] * u >= kLeastProduct) && c * s.w[h] <= 4096.f;
            if (c > 0.f && !fine) {  // (not where NaN)
                const int e = kProductExponent + 127 - (__float_as_int(c) >> 23);
                const float w = __int_as_float((min(max(e, -60), 64) + 127) << 23);
                f *= w / s.w[h];
                s.w[h] = w;
            }
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) s.o[i][h] *= f, s.o[i][2 + h] *= f;
            // a maximum can still be -infinity only where no score is a number
#pragma unroll
            for (int k = 0; k < 2; ++k) x[k][h] = y[k][h] - m, x[k][2 + h] = y[k][2 + h] - m;
        }
        if (tail) mask(x);
        weigh();
        scale();
    }
    s.l[0] += sum[0], s.l[1] += sum[1];
    std::uint32_t hi[2][2], lo[2][2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float b0 = a[k][2 * i], b1 = a[k][2 * i + 1];
            hi[k][i] = half2_of(b0, b1);
            lo[k][i] = half2_of(b0 - half_bits_to_float(hi[k][i] & 0xffffu),
                                b1 - half_bits_to_float(hi[k][i] >> 16));
            hi[k][i] = transpose8x8(hi[k][i]);
            lo[k][i] = transpose8x8(lo[k][i]);
        }
    }
    // O^T += V^T P^T: this thread's four positions of a tile, its HD / 8
    // dimensions from HD / 8 * g on
    constexpr int W = HD / 32;  // 4-byte words of a position
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        std::uint32_t v[4][W];
        if constexpr (HD == 128) {
            const std::uint32_t va = vtile + off.v[0], vb = vtile + off.v[1];
            const uint4 x0 = k ? lds128i<2048>(va) : lds128i<0>(va), x1 = k ? lds128i<2048>(vb) : lds128i<0>(vb);
            const uint4 x2 = k ? lds128i<3072>(va) : lds128i<1024>(va), x3 = k ? lds128i<3072>(vb) : lds128i<1024>(vb);
            const uint4 y[4] = {x0, x1, x2, x3};
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i][0] = y[i].x, v[i][1] = y[i].y, v[i][2] = y[i].z, v[i][3] = y[i].w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint2 y = k ? lds64i<1024>(vtile + off.v[i]) : lds64i<0>(vtile + off.v[i]);
                v[i][0] = y.x, v[i][1] = y.y;
            }
        }
#pragma unroll
        for (int j = 0; j < W; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const std::uint32_t sel = e ? 0x7362u : 0x5140u;  // bytes 2e, 2e + 1 of two positions
                const std::uint32_t ab = prmt(v[0][j], v[1][j], sel) ^ 0x80808080u;
                const std::uint32_t cd = prmt(v[2][j], v[3][j], sel) ^ 0x80808080u;
                const std::uint32_t a0 = bytes_to_half2(ab, 0x4140u), a1 = bytes_to_half2(ab, 0x4342u);
                const std::uint32_t a2 = bytes_to_half2(cd, 0x4140u), a3 = bytes_to_half2(cd, 0x4342u);
                mma_acc(s.o[2 * j + e], a0, a1, a2, a3, hi[k][0], hi[k][1]);
                mma_acc(s.o[2 * j + e], a0, a1, a2, a3, lo[k][0], lo[k][1]);
            }
    }
}

// A row of the work list: sequence b's KV head and head group r, its length
// and units, and the virtual unit at which it begins.
struct Row {
    std::uint32_t b, r, len, n, begin;
};

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
    decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  const Params p) {
    constexpr int kUnit = kTile / HD;  // positions of a unit, in kSub tiles of 16
    constexpr int kSub = kUnit / 16;
    constexpr int kPart = kHeads * (HD + 2);
    extern __shared__ std::uint8_t smem_raw[];
    const std::uint32_t raw = smem_u32(smem_raw);
    const std::uint32_t sbase = (raw + 1023u) & ~1023u;
    std::uint8_t* const smem = smem_raw + (sbase - raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const std::uint32_t ring = sbase + Smem::kRing + warp * (kStages * 2 * kTile);
    const std::uint32_t scl = sbase + Smem::kScales + warp * (kStages * 32);
    std::uint64_t* const full = reinterpret_cast<std::uint64_t*>(smem + Smem::kBars) + warp * kStages;
    const std::uint32_t bars = smem_u32(full);
    float* const flush = reinterpret_cast<float*>(smem + Smem::kFlush);
    float* const ml = reinterpret_cast<float*>(smem + Smem::kMl);
    volatile std::uint32_t* last_cta = reinterpret_cast<std::uint32_t*>(smem + Smem::kLast);
    if (lane < kStages) {
        mbar_init(&full[lane], 2 * kSub);
        fence_mbarrier_init();
    }
    if (threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<std::uint64_t>(&map_k)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<std::uint64_t>(&map_v)) : "memory");
    }
    pdl_launch_dependents();
    pdl_wait();

    const std::uint32_t batch = p.c.batch, bt = p.c.block_tokens;
    const std::uint32_t rows = p.c.kv_heads * p.head_groups;  // of a sequence
    const std::uint32_t cap = p.c.max_blocks * bt;
    const auto length = [&](std::uint32_t b) {
        return min(static_cast<std::uint32_t>(max(__ldg(p.seq_lens + b), 0)), cap);
    };
    const auto units = [&](std::uint32_t len) { return (len + kUnit - 1) / kUnit; };
    // ---- the CTA's share --------------------------------------------------
    // Equal shares of the units, where a row's end counts as kRowCost units
    // more; or, where the rows are few, equal pieces of each row, one to a
    // CTA, of the smallest size (in small steps) that needs no more CTAs than
    // there are, unless shares are smaller by more than a row's end.
    std::uint32_t longest = 0, total = 0, filled = 0;  // units, sequences with any
    std::uint32_t per = 0;                             // units of a CTA
    bool pieces = false;
    const auto least = [&] { return min(longest, static_cast<std::uint32_t>(kMinUnits)); };
    const auto share = [&] { return max((total + filled * kRowCost + gridDim.x - 1) / gridDim.x, least()); };
    const auto size = [&](std::uint32_t i, std::uint32_t steps) {  // pieces from the least on
        const std::uint32_t low = max((total + gridDim.x - 1) / gridDim.x, least());
        return low + (low * i + steps - 1) / steps;
    };
    const auto extent = [&](std::uint32_t n) -> std::uint32_t {  // a row in virtual units
        return pieces ? (n + per - 1) / per * per : n == 0 ? 0 : n + kRowCost;
    };
    const auto clear_empty = [&] {  // sequences without positions
        for (std::uint32_t b = blockIdx.x; b < batch; b += gridDim.x)
            if (length(b) == 0)
                for (std::uint32_t i = threadIdx.x; i < p.q_heads * (HD / 8); i += kThreads)
                    reinterpret_cast<uint4*>(p.out + static_cast<std::uint64_t>(b) * p.q_heads * HD)[i] =
                        make_uint4(0, 0, 0, 0);
    };
    const auto scan_up = [&](std::uint32_t x) {  // inclusive, over the warp
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const std::uint32_t y = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += y;
        }
        return x;
    };
    std::uint32_t u0, at_b = 0, at_begin = 0;  // this CTA's first unit, its sequence and that one's
    if (batch <= kFew) {
        // every warp for itself, one sequence to a lane
        const std::uint32_t n = static_cast<std::uint32_t>(lane) < batch ? units(length(lane)) : 0u;
        longest = __reduce_max_sync(0xffffffffu, n);
        total = __reduce_add_sync(0xffffffffu, n) * rows;
        filled = __popc(__ballot_sync(0xffffffffu, n > 0)) * rows;
        clear_empty();
        if (total == 0) return;
        per = share();
        if (filled <= gridDim.x) {
            const std::uint32_t mine = size(lane, 32);
            std::uint32_t need = 0;
            for (std::uint32_t b = 0; b < batch; ++b)
                need += (__shfl_sync(0xffffffffu, n, b) + mine - 1) / mine;
            const unsigned fits = __ballot_sync(0xffffffffu, need * rows <= gridDim.x);
            const std::uint32_t best = __shfl_sync(0xffffffffu, mine, fits ? __ffs(fits) - 1 : 0);
            pieces = fits != 0 && best <= per + kRowCost;
            if (pieces) per = best;
        }
        u0 = per * blockIdx.x;
        const std::uint32_t mine = extent(n), incl = scan_up(mine);
        const std::uint32_t begin = (incl - mine) * rows;
        const unsigned here = __ballot_sync(0xffffffffu, n > 0 && begin <= u0 && u0 < incl * rows);
        if (here == 0) return;  // past the last unit
        at_b = __ffs(here) - 1;
        at_begin = __shfl_sync(0xffffffffu, begin, at_b);
    } else {
        // the CTA together (scratch: the flush area)
        volatile std::uint32_t* found = reinterpret_cast<std::uint32_t*>(flush);
        volatile std::uint32_t* scan = found + 2 * kWarps + 4;
        for (std::uint32_t b = threadIdx.x; b < batch; b += kThreads) {
            const std::uint32_t n = units(length(b));
            total += n;
            filled += n > 0;
            longest = max(longest, n);
        }
        longest = __reduce_max_sync(0xffffffffu, longest);
        total = __reduce_add_sync(0xffffffffu, total);
        filled = __reduce_add_sync(0xffffffffu, filled);
        if (lane == 0) {
            scan[warp] = longest;
            found[2 * warp] = total;
            found[2 * warp + 1] = filled;
        }
        __syncthreads();
        total = 0, filled = 0, longest = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            longest = max(longest, scan[w]);
            total += found[2 * w];
            filled += found[2 * w + 1];
        }
        total *= rows;
        filled *= rows;
        __syncthreads();
        clear_empty();
        if (total == 0) return;
        per = share();
        if (filled <= gridDim.x) {
            const std::uint32_t mine = size(warp, kWarps);
            std::uint32_t need = 0;
            for (std::uint32_t b = lane; b < batch; b += 32) need += (units(length(b)) + mine - 1) / mine;
            need = __reduce_add_sync(0xffffffffu, need) * rows;
            if (lane == 0) scan[warp] = need <= gridDim.x;
            __syncthreads();
            int w = 0;
            while (w < kWarps && !scan[w]) ++w;
            pieces = w < kWarps && size(w, kWarps) <= per + kRowCost;
            if (pieces) per = size(w, kWarps);
            __syncthreads();
        }
        u0 = per * blockIdx.x;
        std::uint32_t before = 0;  // extents of the sequences before the chunk
        if (threadIdx.x == 0) found[1] = 0;
        for (std::uint32_t base = 0;; base += kThreads) {
            const std::uint32_t b = base + threadIdx.x;
            const std::uint32_t n = b < batch ? units(length(b)) : 0u;
            const std::uint32_t mine = extent(n), incl = scan_up(mine);
            if (lane == 31) found[4 + warp] = incl;
            __syncthreads();
            std::uint32_t lower = before;
            for (int w = 0; w < kWarps; ++w) {
                if (w < warp) lower += found[4 + w];
                before += found[4 + w];
            }
            const std::uint32_t end = (lower + incl) * rows, begin = (lower + incl - mine) * rows;
            if (n > 0 && begin <= u0 && u0 < end) {
                found[0] = begin;
                found[1] = 1;
                found[2] = b;
            }
            __syncthreads();
            if (found[1] || base + kThreads >= batch) break;
        }
        if (!found[1]) return;  // past the last unit
        at_b = found[2], at_begin = found[0];
        __syncthreads();  // the scratch is read
    }
    const std::uint32_t u1 = u0 + per;
    const auto next = [&](Row& x) {  // the next row with positions, begin ~0 behind the last
        x.begin += extent(x.n);
        if (++x.r < rows) return;
        x.r = 0;
        do {
            if (++x.b >= batch) {
                x.begin = ~0u;
                return;
            }
            x.len = length(x.b);
            x.n = units(x.len);
        } while (x.n == 0);
    };
    // this CTA's units [first, last) of a row
    const auto first_of = [&](const Row& x) {
        return x.begin >= u0 ? 0u : min(u0 - x.begin, x.n);
    };
    const auto last_of = [&](const Row& x) {
        return min(u1 - x.begin, x.n);
    };
    Row row;
    row.b = at_b;
    row.len = length(row.b);
    row.n = units(row.len);
    row.r = (u0 - at_begin) / extent(row.n);
    row.begin = at_begin + row.r * extent(row.n);

    // ---- the stream: each warp keeps its ring full, across rows -------------
    // the blocks of 32 / kSub units of this warp, from held_unit of sequence
    // held_b on: one lane for each 16 positions (-1: none)
    std::uint32_t a_unit = first_of(row) + warp, a_last = last_of(row), a_slot = 0, a_stage = 0;
    std::uint32_t a_kvh = row.r / p.head_groups;
    Row ahead = row;
    std::int32_t held_block = -1;
    std::uint32_t held_row = 0, held_b = ~0u, held_unit = 0;
    const auto issue = [&]() {
        while (a_unit >= a_last) {
            if (ahead.begin >= u1) return;
            next(ahead);
            if (ahead.begin >= u1) return;
            a_unit = warp, a_last = last_of(ahead), a_slot = 0, a_kvh = ahead.r / p.head_groups;
        }
        if (a_slot == 0 && (held_b != ahead.b || held_unit != a_unit)) {
            held_b = ahead.b, held_unit = a_unit;
            const std::uint32_t pos = (a_unit + lane / kSub * kWarps) * kUnit + 16 * (lane % kSub);
            held_block = -1;
            if (pos < ahead.len) {
                const std::uint32_t i = pos / bt;
                held_row = pos - i * bt;
                held_block = __ldg(p.tables + static_cast<std::uint64_t>(ahead.b) * p.c.max_blocks + i);
                if (held_block < 0 || static_cast<std::uint64_t>(held_block) >= p.c.num_blocks) {
                    held_block = -1;
                    atomicOr(&g_device_status, kDevIndexOutOfRange);
                }
            }
        }
        const std::uint32_t i = lane - a_slot;
        if (i < kSub) {
            const std::uint32_t bar = bars + 8 * a_stage;
            const std::uint32_t kt = ring + a_stage * 2 * kTile + i * (kTile / kSub);
            const std::uint32_t sc = scl + a_stage * 32 + i * 8;
            if (held_block >= 0) {
                const std::uint64_t tile = static_cast<std::uint64_t>(held_block) * p.c.kv_heads + a_kvh;
                const int y = static_cast<int>((tile * bt + held_row) * HD / 128);
                mbar_expect(bar, 2 * kTile / kSub);
                tma_load_2d(kt, &map_k, 0, y, bar);
                tma_load_2d(kt + kTile, &map_v, 0, y, bar);
                cp_async_4(sc, p.k_scales + tile);
                cp_async_4(sc + 4, p.v_scales + tile);
                cp_async_arrive(bar);
            } else {  // nothing there: a V scale that no block has
                asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(sc), "f"(0.f), "f"(-INFINITY) : "memory");
                mbar_arrive(bar);
                mbar_arrive(bar);
            }
        }
        a_unit += kWarps;
        a_slot = (a_slot + kSub) % 32;
        a_stage = a_stage == kStages - 1 ? 0 : a_stage + 1;
    };
    __syncwarp();
#pragma unroll
    for (int k = 0; k < kStages - 1; ++k) issue();

    // Q^T as the B operand, dimensions in the order of K's loads
    std::uint32_t qf[HD / 8];
    const auto load_q = [&](const Row& x) {
        const std::uint32_t head = (x.r % p.head_groups) * kHeads + g;
        const uint4* src = reinterpret_cast<const uint4*>(
            p.q + (static_cast<std::uint64_t>(x.b) * p.q_heads + x.r / p.head_groups * p.group + head) * HD + HD / 4 * t);
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
            const uint4 a = head < p.group ? __ldg(src + j) : make_uint4(0, 0, 0, 0);
            qf[4 * j] = a.x, qf[4 * j + 1] = a.y, qf[4 * j + 2] = a.z, qf[4 * j + 3] = a.w;
        }
    };
    if (first_of(row) >= last_of(row)) next(row);  // only that row's end falls to this CTA
    if (row.begin < u1) load_q(row);
    const Offsets<HD> off(lane);
    std::uint32_t stage = 0, parity = 0;
    bool waiting = true;
    while (row.begin < u1) {
        const std::uint32_t v0 = first_of(row), v1 = last_of(row);
        State<HD> s;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) s.o[i][k] = 0.f;
        s.m[0] = s.m[1] = -INFINITY;
        s.l[0] = s.l[1] = 0.f;
        s.w[0] = s.w[1] = 1.f;

        for (std::uint32_t v = v0 + warp; v < v1; v += kWarps) {
            if (waiting) waiting = mbar_wait_bounded(&full[stage], parity, &g_device_status);
            __syncwarp();  // the unit has landed; the stage before it is read by all lanes
            if (waiting) issue();  // (a stage whose copies are late gets no more)
            const std::uint32_t kt = ring + stage * 2 * kTile;
            const std::int32_t live = static_cast<std::int32_t>(row.len - v * kUnit);
#pragma unroll
            for (int k = 0; k < kSub / 2; ++k) {
                if (k > 0 && live <= 32 * k) break;
                const uint4 sc = lds128(scl + stage * 32 + k * 16);
                const float sv0 = __uint_as_float(sc.y), sv1 = __uint_as_float(sc.w);
                bool apart = fmaxf(sv0, sv1) > kApart * fminf(sv0, sv1) && fminf(sv0, sv1) >= 0.f;
                bool second = false;
#pragma unroll 1
                for (;;) {
                    attend32<HD>(s, qf, off, kt + k * 32 * HD, kt + kTile + k * 32 * HD,
                                 __uint_as_float(sc.x) * p.scale_log2, __uint_as_float(sc.z) * p.scale_log2,
                                 second ? -INFINITY : sv0, apart ? -INFINITY : sv1, live - 32 * k);
                    if (!apart) break;
                    apart = false, second = true;
                }
            }
            if (++stage == kStages) stage = 0, parity ^= 1;
        }

        // ---- the warps' states meet, four heads at a time -------------------
        // (the ring already holds the next row's units, and its queries load)
        const std::uint32_t head0 = (row.r % p.head_groups) * kHeads;  // in the group
        const std::uint32_t heads = min(p.group - head0, static_cast<std::uint32_t>(kHeads));
        const std::uint64_t q_row = static_cast<std::uint64_t>(row.b) * p.q_heads +
                                    row.r / p.head_groups * p.group + head0;
        const bool whole = v0 == 0 && v1 == row.n;
        const std::uint32_t cta0 = row.begin / per, count = (row.begin + row.n - 1) / per - cta0 + 1;
        next(row);
        if (row.begin < u1) load_q(row);
#pragma unroll
        for (int d = 4; d < 32; d *= 2) {
            s.l[0] += __shfl_xor_sync(0xffffffffu, s.l[0], d);
            s.l[1] += __shfl_xor_sync(0xffffffffu, s.l[1], d);
        }
        const float unit[2] = {1.f / s.w[0], 1.f / s.w[1]};
        float* part = p.parts + static_cast<std::uint64_t>(2 * blockIdx.x + (v0 == 0 ? 1 : 0)) * kPart;
        for (std::uint32_t quad = 0; quad * 4 < heads; ++quad) {
            // [head][pair of dimensions i][g]; the second two heads with i's
            // lowest bit turned, for the banks
            if (static_cast<std::uint32_t>(t >> 1) == quad) {
                float* mine = flush + (warp * 4 + 2 * (t & 1)) * HD + 2 * g;
#pragma unroll
                for (int i = 0; i < HD / 16; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        *reinterpret_cast<float2*>(mine + e * HD + 16 * (i ^ (t & 1))) =
                            make_float2(s.o[i][e] * unit[e], s.o[i][2 + e] * unit[e]);
                if (g == 0)
                    *reinterpret_cast<float4*>(ml + (warp * 4 + 2 * (t & 1)) * 2) =
                        make_float4(s.m[0], s.l[0], s.m[1], s.l[1]);
            }
            __syncthreads();
            const std::uint32_t hq = threadIdx.x / (HD / 2), c = threadIdx.x % (HD / 2);
            const std::uint32_t h = quad * 4 + hq;
            if (hq < 4 && h < heads) {
                float mt = -INFINITY, lt = 0.f;
                float2 o = make_float2(0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) mt = fmaxf(mt, ml[(w * 4 + hq) * 2]);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    // a warp without a position has -infinity and zeros (NaN
                    // scores keep -infinity, and their NaN sums)
                    const float2 a = *reinterpret_cast<const float2*>(ml + (w * 4 + hq) * 2);
                    const float fw = a.y != a.y || a.x == mt ? 1.f : ex2(a.x - mt);
                    const float2 x = *reinterpret_cast<const float2*>(flush + (w * 4 + hq) * HD + 2 * (c ^ (hq >> 1 << 3)));
                    lt = fmaf(a.y, fw, lt);
                    o.x = fmaf(x.x, fw, o.x), o.y = fmaf(x.y, fw, o.y);
                }
                if (whole) {
                    const float inv = lt == 0.f ? 0.f : 1.f / lt;
                    *reinterpret_cast<std::uint32_t*>(p.out + (q_row + h) * HD + HD / 8 * (c & 7) + 2 * (c >> 3)) =
                        half2_of(o.x * inv, o.y * inv);
                } else {
                    *reinterpret_cast<float2*>(part + h * HD + 2 * c) = o;
                    if (c == 0)
                        *reinterpret_cast<float2*>(part + kHeads * HD + 2 * h) = make_float2(mt, lt);
                }
            }
            if (quad * 4 + 4 < heads) __syncthreads();
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
                float* wts = flush;                    // [count][kHeads]
                float* red = wts + kMaxCtas * kHeads;  // [kThreads][4]
                float* invs = red + kThreads * 4;      // [kHeads]
                const std::uint32_t cols = heads * (HD / 4);
                const std::uint32_t groups = kThreads / cols;
                const std::uint32_t col = threadIdx.x % cols, grp = threadIdx.x / cols;
                const std::uint32_t h = col / (HD / 4);
                const auto load = [&](std::uint32_t j) {
                    return __ldcg(reinterpret_cast<const float4*>(part_of(j)) + col);
                };
                constexpr int kFirst = 6;  // loads that run while the weights are found
                float4 x[kFirst];
#pragma unroll
                for (int k = 0; k < kFirst; ++k)
                    if (grp < groups && grp + k * groups < count) x[k] = load(grp + k * groups);
                if (static_cast<std::uint32_t>(warp) < heads) {
                    constexpr int kHeld = 8;  // of up to 256 parts in registers
                    const auto ml_of = [&](std::uint32_t j) {
                        return __ldcg(reinterpret_cast<const float2*>(part_of(j) + kHeads * HD) + warp);
                    };
                    float2 held[kHeld];
                    float mt = -INFINITY, lt = 0.f;
#pragma unroll
                    for (int k = 0; k < kHeld; ++k) {
                        held[k] = lane + 32 * k < count ? ml_of(lane + 32 * k) : make_float2(-INFINITY, 0.f);
                        mt = fmaxf(mt, held[k].x);
                    }
                    for (std::uint32_t j = lane + 32 * kHeld; j < count; j += 32) mt = fmaxf(mt, ml_of(j).x);
                    mt = warp_max(mt);
                    const auto weigh = [&](const float2& a, std::uint32_t j) {
                        const float w = a.y != a.y || a.x == mt ? 1.f : ex2(a.x - mt);
                        lt += a.y * w;
                        wts[j * kHeads + warp] = w;
                    };
#pragma unroll
                    for (int k = 0; k < kHeld; ++k)
                        if (lane + 32 * k < count) weigh(held[k], lane + 32 * k);
                    for (std::uint32_t j = lane + 32 * kHeld; j < count; j += 32) weigh(ml_of(j), j);
#pragma unroll
                    for (int d = 16; d > 0; d /= 2) lt += __shfl_xor_sync(0xffffffffu, lt, d);
                    if (lane == 0) invs[warp] = lt == 0.f ? 0.f : 1.f / lt;
                }
                __syncthreads();
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
                const auto add = [&](const float4& y, std::uint32_t j) {
                    const float w = wts[j * kHeads + h];
                    o.x = fmaf(y.x, w, o.x), o.y = fmaf(y.y, w, o.y);
                    o.z = fmaf(y.z, w, o.z), o.w = fmaf(y.w, w, o.w);
                };
                if (grp < groups) {
#pragma unroll
                    for (int k = 0; k < kFirst; ++k)
                        if (grp + k * groups < count) add(x[k], grp + k * groups);
#pragma unroll 4
                    for (std::uint32_t j = grp + kFirst * groups; j < count; j += groups) add(load(j), j);
                }
                reinterpret_cast<float4*>(red)[threadIdx.x] = o;
                __syncthreads();
                if (threadIdx.x < cols) {
                    for (std::uint32_t k = 1; k < groups; ++k) {
                        const float4 y = reinterpret_cast<const float4*>(red)[threadIdx.x + k * cols];
                        o.x += y.x, o.y += y.y, o.z += y.z, o.w += y.w;
                    }
                    const float inv = invs[h];
                    const std::uint32_t c = threadIdx.x % (HD / 4) * 2;  // pairs c and c + 1
                    __half* dst = p.out + (q_row + h) * HD + HD / 8 * (c & 7) + 2 * (c >> 3);
                    *reinterpret_cast<std::uint32_t*>(dst) = half2_of(o.x * inv, o.y * inv);
                    *reinterpret_cast<std::uint32_t*>(dst + HD / 8) = half2_of(o.z * inv, o.w * inv);
                }
            }
        }
        __syncthreads();  // the flush area is free again
    }
    if (!waiting) let_copies_land();
}

inline int ctas(int& n) {
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    n = sms < kMaxCtas ? sms : kMaxCtas;
    return static_cast<int>(e);
}

inline std::uint64_t workspace_bytes(int n, std::uint64_t head_dim) {
    return kMaxCtas * 4 + static_cast<std::uint64_t>(n) * 2 * kHeads * (head_dim + 2) * 4;
}

// A cache as 128-byte lines, in boxes of 16 positions.
inline int make_map(CUtensorMap* map, const void* cache, const kvq8::CacheShape& c) {
    auto encode = gemm::encode_fn();
    if (encode == nullptr) return static_cast<int>(cudaErrorNotSupported);
    const std::uint64_t lines =
        c.num_blocks * c.kv_heads * c.block_tokens * static_cast<std::uint64_t>(c.head_dim) / 128;
    const cuuint32_t box[2] = {128, c.head_dim / 8};
    const cuuint64_t dims[2] = {128, lines < box[1] ? box[1] : lines};  // no blocks: never loaded
    const cuuint64_t strides[1] = {128};
    const cuuint32_t estr[2] = {1, 1};
    if (lines > 0x7fffffffull ||
        encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(cache), dims, strides, box,
               estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return kInvalidValue;
    return kSuccess;
}

template <int HD>
int launch(const Params& p, const void* k_cache, const void* v_cache, int n, cudaStream_t stream) {
    CUtensorMap map_k{}, map_v{};
    int st = make_map(&map_k, k_cache, p.c);
    if (st == kSuccess) st = make_map(&map_v, v_cache, p.c);
    if (st != kSuccess) return st;
    static std::atomic<std::uint64_t> done{0};
    st = ensure_dynamic_smem(decode_kernel<HD>, Smem::kBytes, done);
    if (st != kSuccess) return st;
    return launch_pdl_smem(decode_kernel<HD>, dim3(static_cast<unsigned>(n)), dim3(kThreads),
                           Smem::kBytes, stream, map_k, map_v, p);
}

}  // namespace attn8
}  // namespace mote

extern "C" int mote_cuda_gqa_attention_decode_q8_workspace_bytes(uint64_t batch, uint64_t q_heads,
                                                                  uint64_t kv_heads,
                                                                  uint64_t head_dim,
                                                                  uint64_t* bytes) {
    using namespace mote;
    if (bytes == nullptr) return kInvalidValue;
    *bytes = 0;
    if (batch == 0 || q_heads == 0 || kv_heads == 0 || (head_dim != 64 && head_dim != 128))
        return kSuccess;  // nothing to do, or refused by the call itself
    int n = 0;
    const int st = attn8::ctas(n);
    if (st == kSuccess) *bytes = attn8::workspace_bytes(n, head_dim);
    return st;
}

extern "C" int mote_cuda_gqa_attention_decode_q8(
    const void* q, const void* k_cache, const void* v_cache, const void* k_scales,
    const void* v_scales, const void* block_tables, const void* seq_lens, void* out,
    uint64_t batch, uint64_t q_heads, uint64_t kv_heads, uint64_t head_dim, uint64_t num_blocks,
    uint64_t block_tokens, uint64_t max_blocks, float scale, void* workspace,
    uint64_t workspace_bytes, void* stream) {
    using namespace mote;
    if (q == nullptr || k_cache == nullptr || v_cache == nullptr || k_scales == nullptr ||
        v_scales == nullptr || block_tables == nullptr || seq_lens == nullptr || out == nullptr ||
        stream == nullptr)
        return kInvalidValue;
    if (!kvq8::shape_ok(batch, kv_heads, head_dim, num_blocks, block_tokens, max_blocks) ||
        kv_heads == 0 || q_heads % kv_heads != 0 || q_heads > 65535 || batch > 65535 ||
        !std::isfinite(scale) || !kvq8::aligned16({q, k_cache, v_cache, out}) ||
        !kvq8::aligned4({k_scales, v_scales, block_tables, seq_lens}))
        return kInvalidValue;
    // units of every row at the tables' full length, with the rows' ends
    const std::uint64_t rows = batch * kv_heads * ((q_heads / kv_heads + attn8::kHeads - 1) / attn8::kHeads);
    const std::uint64_t units = max_blocks * block_tokens * head_dim / attn8::kTile + 1 + attn8::kRowCost;
    if (rows > 0x7fffffffull / units) return kInvalidValue;
    if (batch == 0 || q_heads == 0) return kSuccess;
    int n = 0;
    const int st = attn8::ctas(n);
    if (st != kSuccess) return st;
    if (workspace == nullptr || workspace_bytes < attn8::workspace_bytes(n, head_dim) ||
        !kvq8::aligned16({workspace}))
        return kInvalidValue;
    attn8::Params p{};
    p.q = static_cast<const __half*>(q);
    p.k_scales = static_cast<const float*>(k_scales);
    p.v_scales = static_cast<const float*>(v_scales);
    p.tables = static_cast<const std::int32_t*>(block_tables);
    p.seq_lens = static_cast<const std::int32_t*>(seq_lens);
    p.out = static_cast<__half*>(out);
    p.c = kvq8::make_shape(batch, kv_heads, head_dim, num_blocks, block_tokens, max_blocks);
    p.q_heads = static_cast<std::uint32_t>(q_heads);
    p.group = static_cast<std::uint32_t>(q_heads / kv_heads);
    p.head_groups = (p.group + attn8::kHeads - 1) / attn8::kHeads;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.counters = static_cast<unsigned*>(workspace);
    p.parts = static_cast<float*>(workspace) + attn8::kMaxCtas;
    const auto s = static_cast<cudaStream_t>(stream);
    return head_dim == 64 ? attn8::launch<64>(p, k_cache, v_cache, n, s)
                          : attn8::launch<128>(p, k_cache, v_cache, n, s);
}

// Decode attention over the 8-bit paged cache (kv_cache_q8.cu): one query
// token per sequence,
//   out[b, h] = softmax(scale * q[b, h] . K_b[:len_b, h / g]) . V_b
// with K = qk * sk, V = qv * sv (8-bit integers times the scale of their block
// and head).
//
// HBM-bound: K and V of the attended positions are read once; 8 query heads
// share each read.  Everything else is arranged so that the stream never
// waits:
// * The work is cut in units of 2048 / head_dim positions (2 KB of K and 2 KB
//   of V) of one (sequence, KV head, up to 8 query heads) "row".  Every CTA
//   takes an equal run of consecutive units, found from the lengths on the
//   device, so ragged batches balance and no length bound is needed on the
//   host.  The 8 warps of a CTA take its units in turn, each through a ring of
//   three stages filled with cp.async.
// * The 8-bit values become f16 exactly (the byte as the low bits of
//   1024 + u, minus 1152) and feed mma.sync.m16n8k16 as the A operand:
//   S^T = K Q^T with 16 positions as rows and 8 heads as columns, then
//   O^T += V^T P^T with 16 dimensions as rows, so no row of the products is
//   idle whatever the grouping.  K's dimensions and V's positions are taken
//   in the order in which a thread's 16-byte shared loads hold them (the
//   products do not depend on it); P^T gets from the accumulator layout to the
//   operand's with movmatrix.  Shared rows are swizzled so that these loads
//   have no bank conflicts.
// * scale * sk multiplies S in f32; sv multiplies P, relative to a power of
//   two, before P is split into f16 high and low parts (two products, 22
//   bits).  The running maximum moves only when a score passes it by more
//   than 8 (log2 units), so a unit costs one vote instead of a reduction.
// * Rows that lie in several CTAs leave unnormalised parts in the workspace;
//   the last CTA to finish joins them in order (a counter per row, left at
//   zero), so results do not depend on timing.
#include "mote_common.cuh"

namespace mote {
namespace attn8 {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kHeads = 8;     // query heads of a row (columns of the products)
constexpr int kStages = 3;
constexpr int kTile = 2048;   // bytes of K (and of V) in a unit
constexpr int kCtasPerSm = 2;
constexpr int kMaxCtas = 1024;
constexpr int kMinUnits = 32; // a CTA's share of a row that it splits

struct Params {
    const __half* q;
    const std::int8_t* k_cache;
    const std::int8_t* v_cache;
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
    static constexpr int kRing = 0;  // [warp][stage][K tile, V tile]
    static constexpr int kScales = kRing + kWarps * kStages * 2 * kTile;  // [warp][stage][4] f32
    static constexpr int kMl = kScales + kWarps * kStages * 16;           // [m, l][warp][head] f32
    static constexpr int kScan = kMl + 2 * kWarps * kHeads * 4;           // [16] u32
    static constexpr int kFound = kScan + 64;                             // b, its first unit, last
    static constexpr int kBytes = kFound + 32;
};

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

// Bytes (0, 1) or (2, 3) of w (each 128 + value) as a pair of f16 values.
__device__ __forceinline__ std::uint32_t bytes_to_half2(std::uint32_t w, std::uint32_t sel) {
    return hsub2_u32(prmt(w, 0x64646464u, sel), 0x64806480u);
}

__device__ __forceinline__ uint4 lds128(std::uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr));
    return v;
}

__device__ __forceinline__ float lds_f32(std::uint32_t addr) {
    return __uint_as_float(lds32(addr));
}

__device__ __forceinline__ void cp_async_4(std::uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// Byte offsets of a 16-byte chunk c of row r inside a K or V tile.  A quarter
// of a warp reads K rows i and i + 4, and V rows 0..3 (mod 4) at two chunks.
template <int HD>
__device__ __forceinline__ std::uint32_t k_at(std::uint32_t r, std::uint32_t c) {
    return HD == 128 ? r * 128 + ((c ^ (((r >> 2) & 1) << 2)) << 4)
                     : (r >> 1) * 128 + (((r ^ (r >> 2)) & 1) << 6) + (c << 4);
}
template <int HD>
__device__ __forceinline__ std::uint32_t v_at(std::uint32_t r, std::uint32_t c) {
    return HD == 128 ? r * 128 + ((c ^ ((r & 3) << 1)) << 4)
                     : r * 64 + ((c ^ (r & 2)) << 4);
}

__device__ __forceinline__ void mma_acc(float (&d)[4], std::uint32_t a0, std::uint32_t a1,
                                        std::uint32_t a2, std::uint32_t a3, std::uint32_t b0,
                                        std::uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// One warp's state over its units of a row: O^T accumulators (dimension
// HD / 8 * (lane / 4) + 2 i + e of heads 2 (lane % 4), + 1), this lane's part
// of the sums, the reference maxima and V's reference scale.
template <int HD>
struct State {
    float o[HD / 16][4];
    float m[2], l[2];
    float wref;  // power of two: P is held times sv * wref; 0 until the first V scale
};

template <int HD>
__device__ __forceinline__ void attend16(State<HD>& s, const std::uint32_t (&qf)[HD / 8],
                                         std::uint32_t ktile, std::uint32_t vtile, int row0,
                                         float f, float sv, std::int32_t live) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // S^T: rows are the positions in the order p(r) = r / 2 + 4 (r % 2), + 8
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    const std::uint32_t r0 = row0 + (g >> 1) + 4 * (g & 1);
#pragma unroll
    for (int j = 0; j < HD / 64; ++j) {
        const uint4 a = lds128(ktile + k_at<HD>(r0, t + 4 * j));
        const uint4 b = lds128(ktile + k_at<HD>(r0 + 8, t + 4 * j));
        const std::uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const std::uint32_t xa = aw[i] ^ 0x80808080u, xb = bw[i] ^ 0x80808080u;
            mma_acc(acc, bytes_to_half2(xa, 0x4140u), bytes_to_half2(xb, 0x4140u),
                    bytes_to_half2(xa, 0x4342u), bytes_to_half2(xb, 0x4342u),
                    qf[(4 * j + i) * 2], qf[(4 * j + i) * 2 + 1]);
        }
    }
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = acc[i] * f;
    const std::int32_t p0 = (g >> 1) + 4 * (g & 1);
    if (live < 16) {
        if (p0 >= live) x[0] = x[1] = -INFINITY;
        if (p0 + 8 >= live) x[2] = x[3] = -INFINITY;
    }
    float t0 = fmaxf(x[0], x[2]), t1 = fmaxf(x[1], x[3]);
    if (__any_sync(0xffffffffu, t0 > s.m[0] + 8.f || t1 > s.m[1] + 8.f)) {
#pragma unroll
        for (int d = 4; d < 32; d *= 2) {
            t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, d));
            t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, d));
        }
        t0 = fmaxf(t0, s.m[0]), t1 = fmaxf(t1, s.m[1]);
        const float f0 = s.m[0] == t0 ? 1.f : ex2(s.m[0] - t0);  // 0 from -infinity
        const float f1 = s.m[1] == t1 ? 1.f : ex2(s.m[1] - t1);
        s.m[0] = t0, s.m[1] = t1;
        s.l[0] *= f0, s.l[1] *= f1;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) s.o[i][0] *= f0, s.o[i][2] *= f0, s.o[i][1] *= f1, s.o[i][3] *= f1;
    }
    // V's scale relative to the reference: sv * wref in (2^5, 2^6] where the
    // reference was set, at most 2^7, so P (below 2^8) times it fits f16 and
    // keeps 22 bits down to 2^-14 of the row's largest
    if (!(sv * s.wref <= 128.f) || s.wref == 0.f) {
        const int e = min(max((__float_as_int(fabsf(sv)) >> 23) - 127, -100), 100);
        const float w = __int_as_float((5 - e + 127) << 23);
        const float r = s.wref == 0.f ? 1.f : w / s.wref;
        if (sv != 0.f) {
            s.wref = w;
#pragma unroll
            for (int i = 0; i < HD / 16; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) s.o[i][k] *= r;
        }
    }
    const float m0 = s.m[0] == -INFINITY ? 0.f : s.m[0], m1 = s.m[1] == -INFINITY ? 0.f : s.m[1];
    x[0] = ex2(x[0] - m0), x[2] = ex2(x[2] - m0);
    x[1] = ex2(x[1] - m1), x[3] = ex2(x[3] - m1);
    s.l[0] += x[0] + x[2], s.l[1] += x[1] + x[3];
    const float w = sv * s.wref;
    std::uint32_t hi[2], lo[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float a = x[2 * i] * w, b = x[2 * i + 1] * w;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(hi[i]) : "f"(b), "f"(a));
        const float ra = a - half_bits_to_float(hi[i] & 0xffffu), rb = b - half_bits_to_float(hi[i] >> 16);
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(lo[i]) : "f"(rb), "f"(ra));
        hi[i] = transpose8x8(hi[i]);
        lo[i] = transpose8x8(lo[i]);
    }
    // O^T += V^T P^T: this thread's positions t, t + 4, t + 8, t + 12, its
    // dimensions the HD / 8 from HD / 8 * g on
    constexpr int W = HD / 32;  // 4-byte words of a position
    std::uint32_t v[4][W];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (HD == 128) {
            const uint4 a = lds128(vtile + v_at<HD>(row0 + t + 4 * i, g));
            v[i][0] = a.x, v[i][1] = a.y, v[i][2] = a.z, v[i][3] = a.w;
        } else {
            const uint2 a = lds64(vtile + v_at<HD>(row0 + t + 4 * i, g >> 1) + 8 * (g & 1));
            v[i][0] = a.x, v[i][1] = a.y;
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
            mma_acc(s.o[2 * j + e], a0, a1, a2, a3, hi[0], hi[1]);
            mma_acc(s.o[2 * j + e], a0, a1, a2, a3, lo[0], lo[1]);
        }
}

template <int HD>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) decode_kernel(const Params p) {
    constexpr int U = kTile / HD;  // positions of a unit
    constexpr int SUB = U / 16;
    constexpr int kPart = kHeads * (HD + 2);
    extern __shared__ __align__(128) std::uint8_t smem[];
    const std::uint32_t sbase = smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const std::uint32_t ring = sbase + Smem::kRing + warp * (kStages * 2 * kTile);
    const std::uint32_t scl = sbase + Smem::kScales + warp * (kStages * 16);
    float* sm_m = reinterpret_cast<float*>(smem + Smem::kMl);
    float* sm_l = sm_m + kWarps * kHeads;
    std::uint32_t* scan = reinterpret_cast<std::uint32_t*>(smem + Smem::kScan);
    unsigned long long* found = reinterpret_cast<unsigned long long*>(smem + Smem::kFound);
    pdl_launch_dependents();
    pdl_wait();

    const std::uint32_t batch = p.c.batch, bt = p.c.block_tokens;
    const std::uint32_t rows = p.c.kv_heads * p.head_groups;  // of a sequence
    const std::uint32_t cap = p.c.max_blocks * bt;
    const auto length = [&](std::uint32_t b) {
        return min(static_cast<std::uint32_t>(max(__ldg(p.seq_lens + b), 0)), cap);
    };
    const auto units = [&](std::uint32_t len) { return (len + U - 1) / U; };

    // all units and the longest row's
    std::uint32_t longest = 0;
    unsigned long long total = 0;
    for (std::uint32_t b = threadIdx.x; b < batch; b += kThreads) {
        const std::uint32_t n = units(length(b));
        total += n;
        longest = max(longest, n);
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
#pragma unroll
    for (int d = 16; d > 0; d /= 2) total += __shfl_xor_sync(0xffffffffu, total, d);
    if (lane == 0) {
        scan[warp] = longest;
        reinterpret_cast<unsigned long long*>(sm_m)[warp] = total;
    }
    __syncthreads();
    total = 0, longest = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        longest = max(longest, scan[w]);
        total += reinterpret_cast<unsigned long long*>(sm_m)[w];
    }
    total *= rows;
    // equal shares; rows of up to kMinUnits units stay whole where they can
    const unsigned long long share = (total + gridDim.x - 1) / gridDim.x;
    const unsigned long long per = max(share, static_cast<unsigned long long>(min(longest, static_cast<std::uint32_t>(kMinUnits))));
    const unsigned long long u0 = per * blockIdx.x, u1 = min(total, u0 + per);

    // sequences without positions
    for (std::uint32_t b = blockIdx.x; b < batch; b += gridDim.x)
        if (length(b) == 0)
            for (std::uint32_t i = threadIdx.x; i < p.q_heads * (HD / 8); i += kThreads)
                reinterpret_cast<uint4*>(p.out + static_cast<std::uint64_t>(b) * p.q_heads * HD)[i] =
                    make_uint4(0, 0, 0, 0);
    if (u0 >= u1) return;

    // the sequence of unit u0
    unsigned long long before = 0;  // units of the sequences before the chunk
    for (std::uint32_t base = 0;; base += kThreads) {
        const std::uint32_t b = base + threadIdx.x;
        const std::uint32_t n = b < batch ? units(length(b)) : 0u;
        std::uint32_t incl = n;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const std::uint32_t y = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += y;
        }
        __syncthreads();
        if (lane == 31) scan[warp] = incl;
        if (threadIdx.x == 0) found[1] = 0;
        __syncthreads();
        unsigned long long lower = before;
        for (int w = 0; w < warp; ++w) lower += scan[w];
        const unsigned long long end = (lower + incl) * rows, begin = (lower + incl - n) * rows;
        if (n > 0 && begin <= u0 && u0 < end) {
            found[0] = begin;
            found[1] = 1;
            found[2] = b;
        }
        for (int w = 0; w < kWarps; ++w) before += scan[w];
        __syncthreads();
        if (found[1] || base + kThreads >= batch) break;
    }
    std::uint32_t b = static_cast<std::uint32_t>(found[2]);
    unsigned long long row_begin = found[0];
    std::uint32_t len = length(b), n = units(len);
    std::uint32_t r = static_cast<std::uint32_t>((u0 - row_begin) / n);
    row_begin += static_cast<unsigned long long>(r) * n;

    for (unsigned long long u = u0; u < u1;) {
        // this CTA's units [v0, v1) of row (b, r)
        const std::uint32_t v0 = static_cast<std::uint32_t>(u - row_begin);
        const std::uint32_t v1 = static_cast<std::uint32_t>(min(u1 - row_begin, static_cast<unsigned long long>(n)));
        const std::uint32_t kvh = r / p.head_groups;
        const std::uint32_t head0 = (r % p.head_groups) * kHeads;  // in the group
        const std::uint32_t heads = min(p.group - head0, static_cast<std::uint32_t>(kHeads));
        const std::uint64_t q_row = static_cast<std::uint64_t>(b) * p.q_heads + kvh * p.group + head0;

        // Q^T as the B operand, dimensions in the order of K's loads
        std::uint32_t qf[HD / 8];
#pragma unroll
        for (int j = 0; j < HD / 64; ++j) {
            uint4 a = make_uint4(0, 0, 0, 0), c = a;
            if (static_cast<std::uint32_t>(g) < heads) {
                const uint4* src = reinterpret_cast<const uint4*>(p.q + (q_row + g) * HD + 64 * j + 16 * t);
                a = __ldg(src), c = __ldg(src + 1);
            }
            const std::uint32_t w[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) qf[8 * j + i] = w[i];
        }
        State<HD> s;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) s.o[i][k] = 0.f;
        s.m[0] = s.m[1] = -INFINITY;
        s.l[0] = s.l[1] = 0.f;
        s.wref = 0.f;

        const std::uint32_t mine = v1 - v0 > static_cast<std::uint32_t>(warp)
                                       ? (v1 - v0 - warp + kWarps - 1) / kWarps : 0u;
        // blocks of the next 32 / SUB units, one per lane and 16 positions
        std::int32_t ahead_block = -1;
        std::uint32_t ahead_row = 0;
        std::uint32_t ok_bits = 0;  // of the last units issued, newest lowest
        const auto issue = [&](std::uint32_t k) {
            if (k < mine) {
                constexpr std::uint32_t kAhead = 32 / SUB;
                if (k % kAhead == 0) {
                    const std::uint32_t pos =
                        (v0 + warp + (k + lane / SUB) * kWarps) * U + 16 * (lane % SUB);
                    ahead_block = -1;
                    if (k + lane / SUB < mine && pos < len) {
                        const std::uint32_t i = pos / bt;
                        ahead_row = pos - i * bt;
                        ahead_block = __ldg(p.tables + static_cast<std::uint64_t>(b) * p.c.max_blocks + i);
                        if (ahead_block < 0 || static_cast<std::uint64_t>(ahead_block) >= p.c.num_blocks) {
                            ahead_block = -1;
                            atomicOr(&g_device_status, kDevIndexOutOfRange);
                        }
                    }
                }
                const std::uint32_t st = k % kStages;
                const std::uint32_t kt = ring + st * 2 * kTile, vt = kt + kTile;
#pragma unroll
                for (int i = 0; i < SUB; ++i) {
                    const int from = (k % kAhead) * SUB + i;
                    const std::int32_t block = __shfl_sync(0xffffffffu, ahead_block, from);
                    const std::uint32_t row = __shfl_sync(0xffffffffu, ahead_row, from);
                    ok_bits = ok_bits << 1 | (block >= 0 ? 1u : 0u);
                    if (block >= 0) {
                        const std::uint64_t tile = static_cast<std::uint64_t>(block) * p.c.kv_heads + kvh;
                        const std::uint64_t at = (tile * bt + row) * HD + 16 * lane;
#pragma unroll
                        for (int j = 0; j < HD / 32; ++j) {  // 512 bytes a step
                            const std::uint32_t byte = 512 * j + 16 * lane;
                            const std::uint32_t rr = 16 * i + byte / HD, cc = byte % HD / 16;
                            cp_async_16_default(kt + k_at<HD>(rr, cc), p.k_cache + at + 512 * j);
                            cp_async_16_default(vt + v_at<HD>(rr, cc), p.v_cache + at + 512 * j);
                        }
                        if (lane < 2)
                            cp_async_4(scl + st * 16 + i * 8 + lane * 4,
                                       (lane ? p.v_scales : p.k_scales) + tile);
                    }
                }
            } else {
                ok_bits <<= SUB;
            }
            cp_async_commit();
        };
#pragma unroll
        for (int k = 0; k < kStages - 1; ++k) issue(k);
        for (std::uint32_t k = 0; k < mine; ++k) {
            cp_async_wait<kStages - 2>();
            __syncwarp();  // unit k has landed for all lanes; the stage before it is read
            issue(k + kStages - 1);
            const std::uint32_t st = k % kStages;
            const std::uint32_t kt = ring + st * 2 * kTile;
            const std::uint32_t pos = (v0 + warp + k * kWarps) * U;
#pragma unroll
            for (int i = 0; i < SUB; ++i)
                if (ok_bits >> ((kStages - 1) * SUB + SUB - 1 - i) & 1u) {
                    const float sk = lds_f32(scl + st * 16 + i * 8), sv = lds_f32(scl + st * 16 + i * 8 + 4);
                    attend16<HD>(s, qf, kt, kt + kTile, 16 * i, sk * p.scale_log2, sv,
                                 static_cast<std::int32_t>(len - pos) - 16 * i);
                }
        }
        cp_async_wait<0>();
        __syncwarp();

        // the warps' states meet: each leaves O, its maxima and sums
#pragma unroll
        for (int d = 4; d < 32; d *= 2) {
            s.l[0] += __shfl_xor_sync(0xffffffffu, s.l[0], d);
            s.l[1] += __shfl_xor_sync(0xffffffffu, s.l[1], d);
        }
        const float unref = s.wref == 0.f ? 0.f : 1.f / s.wref;
        float* mine_o = reinterpret_cast<float*>(smem + Smem::kRing + warp * (kStages * 2 * kTile));
#pragma unroll
        for (int i = 0; i < HD / 16; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                *reinterpret_cast<float2*>(mine_o + (2 * t + e) * HD + HD / 8 * g + 2 * i) =
                    make_float2(s.o[i][e] * unref, s.o[i][2 + e] * unref);
        if (g == 0) {
            sm_m[warp * kHeads + 2 * t] = s.m[0], sm_m[warp * kHeads + 2 * t + 1] = s.m[1];
            sm_l[warp * kHeads + 2 * t] = s.l[0], sm_l[warp * kHeads + 2 * t + 1] = s.l[1];
        }
        __syncthreads();
        const bool whole = v0 == 0 && v1 == n;
        const unsigned long long row_end = row_begin + n;
        const std::uint32_t first = static_cast<std::uint32_t>(row_begin / per);
        const std::uint32_t count = static_cast<std::uint32_t>((row_end - 1) / per) - first + 1;
        float* part = p.parts + static_cast<std::uint64_t>(2 * blockIdx.x + (v0 == 0 ? 1 : 0)) * kPart;
        for (std::uint32_t i = threadIdx.x; i < heads * (HD / 4); i += kThreads) {
            const std::uint32_t h = i / (HD / 4), d = i % (HD / 4) * 4;
            float mt = -INFINITY, lt = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) mt = fmaxf(mt, sm_m[w * kHeads + h]);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                // a warp without a position has -infinity and zeros (NaN scores
                // keep -infinity, and their NaN sums)
                const float mw = sm_m[w * kHeads + h];
                const float fw = mw == mt ? 1.f : mw == -INFINITY ? 0.f : ex2(mw - mt);
                const float lw = sm_l[w * kHeads + h];
                if (mw == -INFINITY && lw == 0.f) continue;
                const float4 x = *reinterpret_cast<const float4*>(
                    smem + Smem::kRing + w * (kStages * 2 * kTile) + (h * HD + d) * 4);
                const float gw = lw != lw ? 1.f : fw;
                lt = fmaf(lw, gw, lt);
                o.x = fmaf(x.x, gw, o.x), o.y = fmaf(x.y, gw, o.y);
                o.z = fmaf(x.z, gw, o.z), o.w = fmaf(x.w, gw, o.w);
            }
            if (whole) {
                const float inv = lt == 0.f ? 0.f : 1.f / lt;
                std::uint32_t y0, y1;
                asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y0) : "f"(o.y * inv), "f"(o.x * inv));
                asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y1) : "f"(o.w * inv), "f"(o.z * inv));
                *reinterpret_cast<uint2*>(p.out + (q_row + h) * HD + d) = make_uint2(y0, y1);
            } else {
                *reinterpret_cast<float4*>(part + h * HD + d) = o;
                if (d == 0) {
                    part[kHeads * HD + h] = mt;
                    part[kHeads * HD + kHeads + h] = lt;
                }
            }
        }
        if (!whole) {
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                const unsigned done = atomicAdd(p.counters + first, 1u);
                if (done == count - 1) p.counters[first] = 0;
                scan[0] = done == count - 1;
            }
            __syncthreads();
            if (scan[0]) {
                // join the row's parts: weights, then sums over every kGroups-th part
                __threadfence();
                const auto part_of = [&](std::uint32_t j) {
                    return p.parts + static_cast<std::uint64_t>(2 * (first + j) + (j == 0 ? 1 : 0)) * kPart;
                };
                float* wts = reinterpret_cast<float*>(smem);  // [count][heads]
                float* red = wts + kMaxCtas * kHeads;         // [kThreads][4]
                if (static_cast<std::uint32_t>(warp) < heads) {
                    float mt = -INFINITY, lt = 0.f;
                    for (std::uint32_t j = lane; j < count; j += 32)
                        mt = fmaxf(mt, __ldcg(part_of(j) + kHeads * HD + warp));
#pragma unroll
                    for (int d = 16; d > 0; d /= 2) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, d));
                    for (std::uint32_t j = lane; j < count; j += 32) {
                        const float mj = __ldcg(part_of(j) + kHeads * HD + warp);
                        const float lj = __ldcg(part_of(j) + kHeads * HD + kHeads + warp);
                        const float w = lj != lj ? 1.f : mj == mt ? 1.f : mj == -INFINITY ? 0.f : ex2(mj - mt);
                        lt += lj * w;
                        wts[j * kHeads + warp] = w;
                    }
#pragma unroll
                    for (int d = 16; d > 0; d /= 2) lt += __shfl_xor_sync(0xffffffffu, lt, d);
                    if (lane == 0) sm_l[warp] = lt == 0.f ? 0.f : 1.f / lt;
                }
                __syncthreads();
                const std::uint32_t cols = heads * (HD / 4);
                const std::uint32_t groups = kThreads / cols;
                const std::uint32_t col = threadIdx.x % cols, grp = threadIdx.x / cols;
                const std::uint32_t h = col / (HD / 4), d = col % (HD / 4) * 4;
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
                if (grp < groups)
#pragma unroll 8
                    for (std::uint32_t j = grp; j < count; j += groups) {
                        const float4 x = __ldcg(reinterpret_cast<const float4*>(part_of(j) + h * HD + d));
                        const float w = wts[j * kHeads + h];
                        if (w != 0.f) {
                            o.x = fmaf(x.x, w, o.x), o.y = fmaf(x.y, w, o.y);
                            o.z = fmaf(x.z, w, o.z), o.w = fmaf(x.w, w, o.w);
                        }
                    }
                reinterpret_cast<float4*>(red)[threadIdx.x] = o;
                __syncthreads();
                if (threadIdx.x < cols) {
                    for (std::uint32_t k = 1; k < groups; ++k) {
                        const float4 x = reinterpret_cast<const float4*>(red)[threadIdx.x + k * cols];
                        o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
                    }
                    const float inv = sm_l[h];
                    std::uint32_t y0, y1;
                    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y0) : "f"(o.y * inv), "f"(o.x * inv));
                    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y1) : "f"(o.w * inv), "f"(o.z * inv));
                    *reinterpret_cast<uint2*>(p.out + (q_row + h) * HD + d) = make_uint2(y0, y1);
                }
            }
        }
        __syncthreads();
        // the next row
        u = row_begin + v1;
        if (u >= u1) break;
        row_begin = row_end;
        if (++r == rows) {
            r = 0;
            do {
                len = length(++b);
                n = units(len);
            } while (n == 0);
        }
    }
}

inline int ctas(int& n) {
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    n = sms * kCtasPerSm < kMaxCtas ? sms * kCtasPerSm : kMaxCtas;
    return static_cast<int>(e);
}

inline std::uint64_t workspace_bytes(int n, std::uint64_t head_dim) {
    return kMaxCtas * 4 + static_cast<std::uint64_t>(n) * 2 * kHeads * (head_dim + 2) * 4;
}

template <int HD>
int launch(const Params& p, int n, cudaStream_t stream) {
    static_assert(Smem::kBytes >= (kMaxCtas * kHeads + kThreads * 4) * 4, "the join's scratch");
    static std::atomic<std::uint64_t> done{0};
    const int st = ensure_dynamic_smem(decode_kernel<HD>, Smem::kBytes, done);
    if (st != kSuccess) return st;
    return launch_pdl_smem(decode_kernel<HD>, dim3(static_cast<unsigned>(n)), dim3(kThreads),
                           Smem::kBytes, stream, p);
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
    if (batch == 0 || q_heads == 0) return kSuccess;
    int n = 0;
    const int st = attn8::ctas(n);
    if (st != kSuccess) return st;
    if (workspace == nullptr || workspace_bytes < attn8::workspace_bytes(n, head_dim) ||
        !kvq8::aligned16({workspace}))
        return kInvalidValue;
    attn8::Params p{};
    p.q = static_cast<const __half*>(q);
    p.k_cache = static_cast<const std::int8_t*>(k_cache);
    p.v_cache = static_cast<const std::int8_t*>(v_cache);
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
    return head_dim == 64 ? attn8::launch<64>(p, n, s) : attn8::launch<128>(p, n, s);
}

// KV cache held in 8 bits: append (quantize) and read back (dequantize).
//
// No reference counterpart: the reference names "KV-cache operations" as
// planned primitives (docs/roadmap.md:60) and ships none.
//
// Layout (K and V alike):
//   cache   [num_blocks, kv_heads, block_tokens, head_dim] int8
//   scales  [num_blocks, kv_heads] f32: value = q * scale
//   block_tables [batch, max_blocks] int32: position p of sequence b is row
//           p % block_tokens of block block_tables[b][p / block_tokens]
// One head's rows of a block are contiguous, so attention streams them as
// whole tiles, and one scale serves the tile.
//
// Append, for each block and head that receives rows:
//   s_old = 0 if the block is written from its first row, else its scale
//   s     = max(s_old, fl32(amax / 127)), amax over the new rows
//   inv   = fl32(1 / s)
//   q     = rint(x * inv)                                  (new rows)
//   q'    = rint(q * fl32(s_old * inv))  if the scale grew (rows before them)
// x has 11 bits, q 8 and inv 24, so both products are rounded once, to the
// integer itself: fma(x, inv, 1.5 * 2^23) leaves the integer in the low bits
// of the sum (ties to even).  The result does not depend on the order of
// anything.  A block that is written at once is off by half a step of its scale
// at most, 0.289 rms; rows appended one by one are rounded again whenever the
// scale grows: normal rows end at 0.36 to 0.38 steps rms (0.84 -> 1.05 % of the
// rows' rms with 16 tokens to a block, 0.97 -> 1.29 % with 256), rows that grow
// sevenfold along a block at 0.48 to 0.79.  Rows behind the new ones keep their
// bytes.  A row with an infinity or a NaN makes the block's scale NaN (every row
// of the block then reads as NaN for this head) until the block is written from
// its first row.
#include "mote_common.cuh"

namespace mote {
namespace kvq8 {

struct CacheShape {
    std::uint32_t batch, kv_heads, head_dim;
    std::uint32_t block_tokens, max_blocks;
    std::uint64_t num_blocks;
};

// The largest b in [0, n) with f(b) <= w, for a non-decreasing f with
// f(0) <= w (0 otherwise): a 32-way search by one warp.
template <typename F>
__device__ __forceinline__ std::uint32_t warp_search(std::uint32_t n, std::uint32_t w, F f) {
    const std::uint32_t lane = threadIdx.x & 31u;
    std::uint32_t lo = 0, len = n;
    while (len > 1) {
        const std::uint32_t step = (len + 31) / 32;
        const std::uint32_t i = lane * step;
        const unsigned below = __ballot_sync(0xffffffffu, i < len && f(lo + i) <= w);
        const std::uint32_t run = below == 0xffffffffu ? 32u : __ffs(~below) - 1u;
        if (run == 0) break;
        lo += (run - 1) * step;
        len = min(step, len - (run - 1) * step);
    }
    return lo;
}

// Bad offsets, lengths and blocks are told to the caller's flag, or else to
// the device status.
__device__ __forceinline__ void report(unsigned* error_flag) {
    if (error_flag)
        atomicOr(error_flag, 1u);
    else
        atomicOr(&g_device_status, kDevIndexOutOfRange);
}

// The part of one sequence's rows that lies in one block.
struct Part {
    std::int64_t block;      // < 0: nothing to do
    std::uint32_t row;       // first packed row
    std::uint32_t off;       // its row in the block
    std::uint32_t count;     // rows
};

// Packed row offsets give sequence b the work items [f(b), f(b + 1)) with
// f(b) = starts[b] / block_tokens + 2 b: at least one for each block that
// its rows can touch wherever they begin, found without a prefix sum.
// `end_of(b, n)` is the sequence's length after its n rows.
template <typename EndOf>
__device__ __forceinline__ Part find_part(const CacheShape& c, const std::int32_t* starts,
                                          const std::int32_t* tables, std::uint32_t rows,
                                          std::uint32_t item, unsigned* error_flag, EndOf end_of) {
    Part part{-1, 0, 0, 0};
    const auto slot = [&](std::uint32_t b) {
        return static_cast<std::uint32_t>(max(__ldg(starts + b), 0)) / c.block_tokens + 2 * b;
    };
    const std::uint32_t b = warp_search(c.batch, item, slot);
    const std::int32_t s0 = __ldg(starts + b), s1 = __ldg(starts + b + 1);
    const std::uint32_t first = slot(b);
    if (item < first) return part;
    const auto bad = [&]() {
        if ((threadIdx.x & 31u) == 0 && blockIdx.y == 0 && blockIdx.z == 0) report(error_flag);
        return part;
    };
    if (s0 < 0 || s1 < s0 || static_cast<std::uint32_t>(s1) > rows) return bad();
    const std::uint32_t n = static_cast<std::uint32_t>(s1 - s0);
    if (n == 0) return part;
    const std::int64_t end = end_of(b, n);
    const std::int64_t begin = end - n;
    if (begin < 0) return bad();
    const std::int64_t idx = begin / c.block_tokens + (item - first);
    const std::int64_t p0 = max(begin, idx * c.block_tokens);
    const std::int64_t p1 = min(end, (idx + 1) * c.block_tokens);
    if (p0 >= p1) return part;
    if (idx >= c.max_blocks) return bad();
    const std::int32_t block = __ldg(tables + static_cast<std::uint64_t>(b) * c.max_blocks + idx);
    if (block < 0 || static_cast<std::uint64_t>(block) >= c.num_blocks) return bad();
    part.block = block;
    part.row = static_cast<std::uint32_t>(s0 + (p0 - begin));
    part.off = static_cast<std::uint32_t>(p0 - idx * c.block_tokens);
    part.count = static_cast<std::uint32_t>(p1 - p0);
    return part;
}

// starts not in ascending order can hide sequences from the search: reported.
__device__ __forceinline__ void check_starts(const CacheShape& c, const std::int32_t* starts,
                                             std::uint32_t rows, unsigned* error_flag) {
    bool bad = false;
    for (std::uint32_t b = threadIdx.x; b < c.batch; b += blockDim.x) {
        const std::int32_t s0 = __ldg(starts + b), s1 = __ldg(starts + b + 1);
        bad |= s0 < 0 || s1 < s0 || static_cast<std::uint32_t>(s1) > rows;
    }
    if (bad) report(error_flag);
}

constexpr int kThreads = 128;
constexpr int kHeld = 8;  // 16-byte vectors of a thread

__device__ __forceinline__ std::uint32_t round_to_int8(float x, float m) {
    return static_cast<std::uint32_t>(__float_as_int(__fmaf_rn(x, m, 12582912.f))) & 0xffu;
}

// Byte `sel & 3` of w (128 + value) as f32, exactly: as the low bits of 2^23 + u,
// on the integer and FMA pipes (conversions run at a quarter of their rate).
__device__ __forceinline__ float byte_value(std::uint32_t w, std::uint32_t sel) {
    return __uint_as_float(prmt(w, 0x4b000000u, sel)) - 8388736.f;
}

// One CTA for each (work item, head, K or V).  16 prompts of 40 to 2048 rows
// (17.4 k rows of 8 x 128, 107 MB) take 29 us alone, 0.57 of the copy
// bandwidth: a CTA lives for a chain of dependent loads (offsets, length,
// table, rows) and the reduction, and 28 warps of an SM cover it in part.
// Several heads to a CTA, the next one's rows loading meanwhile, measured
// slower (58 against 44 us with the read back): too few CTAs to balance.
// 32 single rows take 4 us, the chain itself.
__global__ void __launch_bounds__(kThreads)
    append_kernel(const CacheShape c, const __half* k_new, const __half* v_new,
                  std::int8_t* k_cache, std::int8_t* v_cache, float* k_scales, float* v_scales,
                  const std::int32_t* tables, const std::int32_t* starts,
                  const std::int32_t* lens, std::uint32_t rows, unsigned* error_flag) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ std::uint32_t warp_max[kThreads / 32];
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0)
        check_starts(c, starts, rows, error_flag);
    const Part part =
        find_part(c, starts, tables, rows, blockIdx.x, error_flag,
                  [&](std::uint32_t b, std::uint32_t) -> std::int64_t { return __ldg(lens + b); });
    if (part.block < 0) return;
    const std::uint32_t h = blockIdx.y;
    const std::uint32_t vecs = c.head_dim / 8;  // 16-byte vectors of a new row
    const std::uint64_t row_stride = static_cast<std::uint64_t>(c.kv_heads) * c.head_dim;
    const __half* src = (blockIdx.z ? v_new : k_new) + part.row * row_stride + h * c.head_dim;
    const std::uint64_t tile = static_cast<std::uint64_t>(part.block) * c.kv_heads + h;
    std::int8_t* dst = (blockIdx.z ? v_cache : k_cache) + tile * c.block_tokens * c.head_dim;
    float* scale = (blockIdx.z ? v_scales : k_scales) + tile;
    const float s_old = part.off == 0 ? 0.f : *scale;

    // the largest |x|: f16 magnitudes order as their bits, NaN above infinity.
    // The first kHeld vectors of a thread stay in registers (all of them, for
    // blocks of up to 64 tokens), so they are in flight together and read once.
    const std::uint32_t total = part.count * vecs;
    const auto load = [&](std::uint32_t i) {
        return __ldg(reinterpret_cast<const uint4*>(src + (i / vecs) * row_stride) + i % vecs);
    };
    const auto largest = [](const uint4& x) {
        return __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu),
                        __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
    };
    std::uint32_t top = 0;
    uint4 held[kHeld];
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        const std::uint32_t i = threadIdx.x + k * kThreads;
        held[k] = i < total ? load(i) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int k = 0; k < kHeld; ++k) top = __vmaxu2(top, largest(held[k]));
    for (std::uint32_t i = threadIdx.x + kHeld * kThreads; i < total; i += kThreads)
        top = __vmaxu2(top, largest(load(i)));
    top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x / 32] = top;
    __syncthreads();  // every thread has read the old scale
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) top = max(top, warp_max[w]);

    const bool finite = top < 0x7c00u && isfinite(s_old);
    const float s_new = finite ? fmaxf(s_old, __fdiv_rn(half_bits_to_float(top), 127.f))
                               : __int_as_float(0x7fc00000);
    const float inv = s_new > 0.f ? __fdiv_rn(1.f, s_new) : 0.f;
    if (threadIdx.x == 0) *scale = s_new;
    const auto store = [&](const uint4& x, std::uint32_t i) {
        const std::uint32_t w[4] = {x.x, x.y, x.z, x.w};
        std::uint32_t q[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float a = half_bits_to_float(w[e] & 0xffffu), b = half_bits_to_float(w[e] >> 16);
            q[e / 2] |= (round_to_int8(a, inv) | round_to_int8(b, inv) << 8) << (16 * (e & 1));
        }
        if (!finite) q[0] = q[1] = 0;
        reinterpret_cast<uint2*>(dst + part.off * c.head_dim)[i] = make_uint2(q[0], q[1]);
    };
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        const std::uint32_t i = threadIdx.x + k * kThreads;
        if (i < total) store(held[k], i);
    }
    for (std::uint32_t i = threadIdx.x + kHeld * kThreads; i < total; i += kThreads) store(load(i), i);
    if (part.off != 0 && !(s_new == s_old)) {  // rows already there, on the new scale
        const float ratio = finite ? __fmul_rn(s_old, inv) : 0.f;
        uint4* old = reinterpret_cast<uint4*>(dst);
        for (std::uint32_t i = threadIdx.x; i < part.off * c.head_dim / 16; i += kThreads) {
            const uint4 x = old[i];
            const std::uint32_t w[4] = {x.x, x.y, x.z, x.w};
            std::uint32_t q[4] = {0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < 16; ++e)
                q[e / 4] |= round_to_int8(static_cast<float>(static_cast<std::int8_t>(
                                              w[e / 4] >> (8 * (e & 3)))),
                                          ratio)
                            << (8 * (e & 3));
            old[i] = make_uint4(q[0], q[1], q[2], q[3]);
        }
    }
}

// The first n_b = starts[b + 1] - starts[b] cached rows of every sequence in
// f16 (fl32(q * scale), rounded once more), packed at row starts[b].  8-byte
// loads, so that a warp's 16-byte stores are whole lines (16-byte loads and
// pairs of stores: 45 us): 31 k rows of 8 x 128, 193 MB, 35 us = 0.84 of the
// copy bandwidth.
__global__ void __launch_bounds__(kThreads)
    read_kernel(const CacheShape c, const std::int8_t* k_cache, const std::int8_t* v_cache,
                const float* k_scales, const float* v_scales, const std::int32_t* tables,
                const std::int32_t* starts, __half* k_out, __half* v_out, std::uint32_t rows,
                unsigned* error_flag) {
    pdl_launch_dependents();
    pdl_wait();
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0)
        check_starts(c, starts, rows, error_flag);
    const Part part =
        find_part(c, starts, tables, rows, blockIdx.x, error_flag,
                  [&](std::uint32_t, std::uint32_t n) -> std::int64_t { return n; });
    if (part.block < 0) return;
    const std::uint32_t h = blockIdx.y;
    const std::uint32_t vecs = c.head_dim / 8;  // 8 bytes of a cached row, 16 of the result's
    const std::uint64_t row_stride = static_cast<std::uint64_t>(c.kv_heads) * c.head_dim;
    const std::uint64_t tile = static_cast<std::uint64_t>(part.block) * c.kv_heads + h;
    const std::int8_t* src = (blockIdx.z ? v_cache : k_cache) + (tile * c.block_tokens + part.off) * c.head_dim;
    const float scale = (blockIdx.z ? v_scales : k_scales)[tile];
    __half* dst = (blockIdx.z ? v_out : k_out) + part.row * row_stride + h * c.head_dim;
    const std::uint32_t total = part.count * vecs;
    for (std::uint32_t base = threadIdx.x; base < total; base += kHeld * kThreads) {
        uint2 held[kHeld];
#pragma unroll
        for (int k = 0; k < kHeld; ++k)
            if (base + k * kThreads < total) held[k] = __ldg(reinterpret_cast<const uint2*>(src) + base + k * kThreads);
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
            const std::uint32_t i = base + k * kThreads;
            if (i >= total) break;
            std::uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const std::uint32_t w = (e < 2 ? held[k].x : held[k].y) ^ 0x80808080u;
                const float a = byte_value(w, 0x7440u + 2 * (e & 1)) * scale;
                const float b = byte_value(w, 0x7441u + 2 * (e & 1)) * scale;
                asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(o[e]) : "f"(b), "f"(a));
            }
            reinterpret_cast<uint4*>(dst + (i / vecs) * row_stride)[i % vecs] =
                make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
}

// Shapes that the cache operators take: head_dim 64 or 128, blocks of a
// multiple of 16 tokens up to 256, sizes that 32-bit row numbers can hold.
inline bool shape_ok(std::uint64_t batch, std::uint64_t kv_heads, std::uint64_t head_dim,
                     std::uint64_t num_blocks, std::uint64_t block_tokens,
                     std::uint64_t max_blocks) {
    return (head_dim == 64 || head_dim == 128) && kv_heads <= 65535 && block_tokens >= 16 &&
           block_tokens <= 256 && block_tokens % 16 == 0 && batch <= (1u << 20) &&
           num_blocks <= 0x7fffffffull && max_blocks <= 0x7fffffffull / block_tokens;
}

inline CacheShape make_shape(std::uint64_t batch, std::uint64_t kv_heads, std::uint64_t head_dim,
                             std::uint64_t num_blocks, std::uint64_t block_tokens,
                             std::uint64_t max_blocks) {
    return CacheShape{static_cast<std::uint32_t>(batch), static_cast<std::uint32_t>(kv_heads),
                      static_cast<std::uint32_t>(head_dim), static_cast<std::uint32_t>(block_tokens),
                      static_cast<std::uint32_t>(max_blocks), num_blocks};
}

inline bool aligned16(std::initializer_list<const void*> ptrs) {
    for (const void* p : ptrs)
        if (reinterpret_cast<std::uintptr_t>(p) % 16 != 0) return false;
    return true;
}

inline bool aligned4(std::initializer_list<const void*> ptrs) {
    for (const void* p : ptrs)
        if (reinterpret_cast<std::uintptr_t>(p) % 4 != 0) return false;
    return true;
}

}  // namespace kvq8
}  // namespace mote

extern "C" int mote_cuda_kv_cache_append_q8(const void* k_new, const void* v_new, void* k_cache,
                                            void* v_cache, void* k_scales, void* v_scales,
                                            const void* block_tables, const void* seq_starts,
                                            const void* seq_lens, uint64_t tokens, uint64_t batch,
                                            uint64_t kv_heads, uint64_t head_dim,
                                            uint64_t num_blocks, uint64_t block_tokens,
                                            uint64_t max_blocks, void* error_flag, void* stream) {
    using namespace mote;
    using namespace mote::kvq8;
    if (k_new == nullptr || v_new == nullptr || k_cache == nullptr || v_cache == nullptr ||
        k_scales == nullptr || v_scales == nullptr || block_tables == nullptr ||
        seq_starts == nullptr || seq_lens == nullptr || stream == nullptr)
        return kInvalidValue;
    if (!shape_ok(batch, kv_heads, head_dim, num_blocks, block_tokens, max_blocks) ||
        tokens > 0x7fffffffull || !aligned16({k_new, v_new, k_cache, v_cache}) ||
        !aligned4({k_scales, v_scales, block_tables, seq_starts, seq_lens}))
        return kInvalidValue;
    if (tokens == 0 || batch == 0 || kv_heads == 0) return kSuccess;
    const dim3 grid(static_cast<unsigned>(tokens / block_tokens + 2 * batch),
                    static_cast<unsigned>(kv_heads), 2);
    return launch_pdl(append_kernel, grid, dim3(kThreads), static_cast<cudaStream_t>(stream),
                      make_shape(batch, kv_heads, head_dim, num_blocks, block_tokens, max_blocks),
                      static_cast<const __half*>(k_new), static_cast<const __half*>(v_new),
                      static_cast<std::int8_t*>(k_cache), static_cast<std::int8_t*>(v_cache),
                      static_cast<float*>(k_scales), static_cast<float*>(v_scales),
                      static_cast<const std::int32_t*>(block_tables),
                      static_cast<const std::int32_t*>(seq_starts),
                      static_cast<const std::int32_t*>(seq_lens),
                      static_cast<std::uint32_t>(tokens), static_cast<unsigned*>(error_flag));
}

extern "C" int mote_cuda_kv_cache_read_q8(const void* k_cache, const void* v_cache,
                                          const void* k_scales, const void* v_scales,
                                          const void* block_tables, const void* starts,
                                          void* k_out, void* v_out, uint64_t tokens,
                                          uint64_t batch, uint64_t kv_heads, uint64_t head_dim,
                                          uint64_t num_blocks, uint64_t block_tokens,
                                          uint64_t max_blocks, void* error_flag, void* stream) {
    using namespace mote;
    using namespace mote::kvq8;
    if (k_cache == nullptr || v_cache == nullptr || k_scales == nullptr || v_scales == nullptr ||
        block_tables == nullptr || starts == nullptr || k_out == nullptr || v_out == nullptr ||
        stream == nullptr)
        return kInvalidValue;
    if (!shape_ok(batch, kv_heads, head_dim, num_blocks, block_tokens, max_blocks) ||
        tokens > 0x7fffffffull || !aligned16({k_out, v_out, k_cache, v_cache}) ||
        !aligned4({k_scales, v_scales, block_tables, starts}))
        return kInvalidValue;
    if (tokens == 0 || batch == 0 || kv_heads == 0) return kSuccess;
    const dim3 grid(static_cast<unsigned>(tokens / block_tokens + 2 * batch),
                    static_cast<unsigned>(kv_heads), 2);
    return launch_pdl(read_kernel, grid, dim3(kThreads), static_cast<cudaStream_t>(stream),
                      make_shape(batch, kv_heads, head_dim, num_blocks, block_tokens, max_blocks),
                      static_cast<const std::int8_t*>(k_cache),
                      static_cast<const std::int8_t*>(v_cache),
                      static_cast<const float*>(k_scales), static_cast<const float*>(v_scales),
                      static_cast<const std::int32_t*>(block_tables),
                      static_cast<const std::int32_t*>(starts), static_cast<__half*>(k_out),
                      static_cast<__half*>(v_out), static_cast<std::uint32_t>(tokens),
                      static_cast<unsigned*>(error_flag));
}

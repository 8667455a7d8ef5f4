// Rotation on the way into a paged KV cache held in f16.
//
// The fused QKV projection's rows [tokens, q_heads + 2 kv_heads, head_dim] are
// rotated by each token's cos/sin row (q and k; the first 2 pairs dimensions of
// a head, the rest copied) and spread: q to q_out [tokens, q_heads, head_dim],
// k and v to the cache [num_blocks, kv_heads, block_tokens, head_dim], where
// position p of sequence b is row p % block_tokens of block
// block_tables[b][p / block_tokens].  The rows seq_starts[b] .. seq_starts[b + 1]
// - 1 are the last positions of sequence b, whose length with them is seq_lens[b].
//
// No reference counterpart (KV-cache operations are planned primitives,
// docs/roadmap.md:58-60); the rotation is rope_f32's, operation by operation
// (crates/mote-reference/src/lib.rs:170-244), so the values are those of
// mote_cuda_rope_f16 and of a copy, bit for bit.
#include "mote_common.cuh"

namespace mote {
namespace kvpaged {

struct Params {
    const __half* qkv;
    const float* cos;
    const float* sin;
    __half* q_out;
    __half* k_cache;
    __half* v_cache;
    const std::int32_t* tables;
    const std::int32_t* starts;
    const std::int32_t* lens;
    kvq8::CacheShape c;
    std::uint32_t tokens, q_heads, pairs;
    bool interleaved;
    unsigned* error_flag;
};

constexpr int kThreads = 128;

// Where token t's k and v go: rows of the first KV head, a head `head_stride`
// further (k null: nowhere), and whether its row belongs to a sequence at all.
struct Place {
    __half* k;
    __half* v;
    bool any;
};

// By a whole warp.
__device__ __forceinline__ Place place_of(const Params& p, std::uint32_t t) {
    Place x{nullptr, nullptr, false};
    const std::uint32_t lane = threadIdx.x & 31;
    std::uint32_t b;
    std::int32_t s0, s1, length;
    if (p.c.batch <= 32) {  // one sequence to a lane, one round of loads (16 prompts 68.5 us, 69.1 by search)
        const bool here = lane < p.c.batch;
        const std::int32_t a0 = here ? __ldg(p.starts + lane) : 0, a1 = here ? __ldg(p.starts + lane + 1) : 0;
        const std::int32_t al = here ? __ldg(p.lens + lane) : 0;
        const unsigned below = __ballot_sync(0xffffffffu, here && static_cast<std::uint32_t>(max(a0, 0)) <= t);
        const unsigned run = below == 0xffffffffu ? 32u : __ffs(~below) - 1u;  // as warp_search counts
        b = run == 0 ? 0 : run - 1;
        s0 = __shfl_sync(0xffffffffu, a0, b), s1 = __shfl_sync(0xffffffffu, a1, b);
        length = __shfl_sync(0xffffffffu, al, b);
    } else {
        b = kvq8::warp_search(p.c.batch, t, [&](std::uint32_t i) {
            return static_cast<std::uint32_t>(max(__ldg(p.starts + i), 0));
        });
        s0 = __ldg(p.starts + b), s1 = __ldg(p.starts + b + 1), length = __ldg(p.lens + b);
    }
    if (s0 < 0 || s1 < s0 || static_cast<std::uint32_t>(s1) > p.tokens ||
        t < static_cast<std::uint32_t>(s0) || t >= static_cast<std::uint32_t>(s1))
        return x;
    const std::int64_t len = length, pos = len - s1 + t;
    if (len < s1 - s0 || len > static_cast<std::int64_t>(p.c.max_blocks) * p.c.block_tokens) {
        if (lane == 0) kvq8::report(p.error_flag);
        return x;
    }
    x.any = true;
    const std::uint32_t i = static_cast<std::uint32_t>(pos) / p.c.block_tokens;
    const std::int32_t block = __ldg(p.tables + static_cast<std::uint64_t>(b) * p.c.max_blocks + i);
    if (block < 0 || static_cast<std::uint64_t>(block) >= p.c.num_blocks) {
        if (lane == 0) kvq8::report(p.error_flag);
        return x;
    }
    const std::uint64_t row = (static_cast<std::uint64_t>(block) * p.c.kv_heads * p.c.block_tokens +
                               (static_cast<std::uint32_t>(pos) - i * p.c.block_tokens)) * p.c.head_dim;
    x.k = p.k_cache + row;
    x.v = p.v_cache + row;
    return x;
}

// Pairs or head parts that are no whole 16-byte vectors, or tables that are not
// aligned to them: one CTA for each token, element by element.  The same rows with 60 or
// 62 pairs of 64: 316 us in halves, 276 interleaved; 32 single rows 19-21 us on the device,
// 3.2 in vectors.
__global__ void __launch_bounds__(kThreads) append_scalar_kernel(const Params p) {
    pdl_launch_dependents();
    pdl_wait();
    if (blockIdx.x == 0) kvq8::check_starts(p.c, p.starts, p.tokens, p.error_flag);
    const std::uint32_t t = blockIdx.x, hd = p.c.head_dim, kvh = p.c.kv_heads;
    const Place place = place_of(p, t);
    if (!place.any) return;
    const std::uint32_t heads = p.q_heads + 2 * kvh, rotated = p.q_heads + kvh;
    const std::uint64_t stride = static_cast<std::uint64_t>(p.c.block_tokens) * hd;
    const __half* row = p.qkv + static_cast<std::uint64_t>(t) * heads * hd;
    for (std::uint32_t i = threadIdx.x; i < heads * hd; i += kThreads) {
        const std::uint32_t h = i / hd, e = i - h * hd;
        const __half* src = row + h * hd;
        __half* dst = p.q_out + (static_cast<std::uint64_t>(t) * p.q_heads + h) * hd;
        if (h >= p.q_heads) {
            if (place.k == nullptr) continue;
            dst = h < rotated ? place.k + (h - p.q_heads) * stride : place.v + (h - rotated) * stride;
        }
        if (h >= rotated || e >= 2 * p.pairs) {
            dst[e] = src[e];
            continue;
        }
        const std::uint32_t j = p.interleaved ? e / 2 : e % p.pairs;
        const bool second = p.interleaved ? e & 1 : e >= p.pairs;
        const float a = __half2float(src[p.interleaved ? 2 * j : j]);
        const float b = __half2float(src[p.interleaved ? 2 * j + 1 : j + p.pairs]);
        float o1, o2;
        rotate(a, b, p.cos[static_cast<std::uint64_t>(t) * p.pairs + j],
               p.sin[static_cast<std::uint64_t>(t) * p.pairs + j], o1, o2);
        dst[e] = __float2half_rn(second ? o2 : o1);
    }
}

__device__ __forceinline__ float2 halves(std::uint32_t w) {
    __half2 h;
    memcpy(&h, &w, 4);
    return __half22float2(h);
}

// HBM-bound: rows in 16-byte vectors, read and written once (14563 rows of 16 prompts, 32
// query / 8 KV heads of 128, 366 MB: 63.6 us, 0.88 of the copy bandwidth; 67 and 75 with
// half and a quarter of a head rotated in halves; 59 in interleaved pairs).  `per_token` threads
// (32, 64 or 128) take a token.  Each keeps one place within a head (a vector and
// its partner half a rotary width further, or one vector of interleaved pairs) with
// the place's cosines and sines in registers, and goes through the heads; its first
// kHeld of them, and the v heads, load while the token's sequence and page are found.
constexpr int kHeld = 4;
template <bool HALF>
__global__ void __launch_bounds__(kThreads) append_kernel(const Params p, const std::uint32_t per_token) {
    pdl_launch_dependents();
    pdl_wait();
    if (blockIdx.x == 0) kvq8::check_starts(p.c, p.starts, p.tokens, p.error_flag);
    const std::uint32_t t = blockIdx.x * (kThreads / per_token) + threadIdx.x / per_token;
    if (t >= p.tokens) return;  // (whole warps)
    const std::uint32_t me = threadIdx.x % per_token;
    const std::uint32_t hd = p.c.head_dim, kvh = p.c.kv_heads, vecs = hd / 8;
    const std::uint32_t turned = HALF ? p.pairs / 8 : p.pairs / 4;     // places of a head that turn
    const std::uint32_t places = HALF ? vecs - turned : vecs;
    const std::uint32_t step = per_token / places;                     // heads at a time
    const std::uint32_t u = me % places, h0 = me / places < step ? me / places : 0x7fffffffu;
    const bool turns = u < turned;
    const std::uint32_t at = HALF && !turns ? u + turned : u;          // vectors of the place
    const std::uint32_t heads = p.q_heads + 2 * kvh, rotated = p.q_heads + kvh;
    const uint4* row = reinterpret_cast<const uint4*>(p.qkv) + static_cast<std::uint64_t>(t) * heads * vecs;
    uint4 x[kHeld][HALF ? 2 : 1], v = make_uint4(0, 0, 0, 0);
    const auto load = [&](std::uint32_t base) {
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
            const std::uint32_t h = base + k * step;
            if (h >= rotated) break;
            x[k][0] = __ldg(row + h * vecs + at);
            if (HALF && turns) x[k][HALF ? 1 : 0] = __ldg(row + h * vecs + at + turned);
        }
    };
    load(h0);
    if (me < kvh * vecs) v = __ldg(row + rotated * vecs + me);
    constexpr int N = HALF ? 8 : 4;  // pairs of a place
    float c[N], s[N];
    if (turns) {
        const float4* cp = reinterpret_cast<const float4*>(p.cos + static_cast<std::uint64_t>(t) * p.pairs + N * u);
        const float4* sp = reinterpret_cast<const float4*>(p.sin + static_cast<std::uint64_t>(t) * p.pairs + N * u);
#pragma unroll
        for (int k = 0; k < N / 4; ++k) {
            const float4 a = __ldg(cp + k), b = __ldg(sp + k);
            c[4 * k] = a.x, c[4 * k + 1] = a.y, c[4 * k + 2] = a.z, c[4 * k + 3] = a.w;
            s[4 * k] = b.x, s[4 * k + 1] = b.y, s[4 * k + 2] = b.z, s[4 * k + 3] = b.w;
        }
    }
    const Place place = place_of(p, t);
    if (!place.any) return;
    const std::uint64_t stride = static_cast<std::uint64_t>(p.c.block_tokens) * vecs;
    uint4* const q_out = reinterpret_cast<uint4*>(p.q_out) + static_cast<std::uint64_t>(t) * p.q_heads * vecs;
    uint4* const k_out = reinterpret_cast<uint4*>(place.k);
    for (std::uint32_t base = h0; base < rotated; base += kHeld * step) {
        if (base != h0) load(base);
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
            const std::uint32_t h = base + k * step;
            if (h >= rotated) break;
            uint4* const dst = h < p.q_heads ? q_out + h * vecs
                                             : k_out == nullptr ? nullptr : k_out + (h - p.q_heads) * stride;
            if (dst == nullptr) break;  // (the heads behind are k's too)
            if (!turns) {
                dst[at] = x[k][0];
                continue;
            }
            const std::uint32_t a[4] = {x[k][0].x, x[k][0].y, x[k][0].z, x[k][0].w};
            std::uint32_t o[4], o2[4];
            if constexpr (HALF) {
                const std::uint32_t b[4] = {x[k][1].x, x[k][1].y, x[k][1].z, x[k][1].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 y = halves(a[e]), z = halves(b[e]);
                    float r0, r1, w0, w1;
                    rotate(y.x, z.x, c[2 * e], s[2 * e], r0, w0);
                    rotate(y.y, z.y, c[2 * e + 1], s[2 * e + 1], r1, w1);
                    o[e] = attn8::half2_of(r0, r1), o2[e] = attn8::half2_of(w0, w1);
                }
                dst[at + turned] = make_uint4(o2[0], o2[1], o2[2], o2[3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 y = halves(a[e]);
                    float r0, r1;
                    rotate(y.x, y.y, c[e], s[e], r0, r1);
                    o[e] = attn8::half2_of(r0, r1);
                }
            }
            dst[at] = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
    if (place.v == nullptr) return;
    uint4* const v_out = reinterpret_cast<uint4*>(place.v);
    for (std::uint32_t i = me; i < kvh * vecs; i += per_token) {
        if (i != me) v = __ldg(row + rotated * vecs + i);
        v_out[i / vecs * stride + i % vecs] = v;
    }
}

}  // namespace kvpaged
}  // namespace mote

extern "C" int mote_cuda_rope_kv_cache_append_paged_f16(
    const void* qkv, const void* cos, const void* sin, void* q_out, void* k_cache, void* v_cache,
    const void* block_tables, const void* seq_starts, const void* seq_lens, uint64_t tokens,
    uint64_t batch, uint64_t q_heads, uint64_t kv_heads, uint64_t head_dim, uint64_t pairs,
    uint64_t num_blocks, uint64_t block_tokens, uint64_t max_blocks, uint32_t layout,
    void* error_flag, void* stream) {
    using namespace mote;
    if (qkv == nullptr || ((cos == nullptr || sin == nullptr) && pairs != 0) || q_out == nullptr ||
        k_cache == nullptr || v_cache == nullptr || block_tables == nullptr ||
        seq_starts == nullptr || seq_lens == nullptr || stream == nullptr)
        return kInvalidValue;
    if (!kvq8::shape_ok(batch, kv_heads, head_dim, num_blocks, block_tokens, max_blocks) ||
        q_heads > 65535 || 2 * pairs > head_dim || pairs > head_dim || layout > 1 ||
        tokens > 0x7fffffffull || !kvq8::aligned16({qkv, q_out, k_cache, v_cache}) ||
        !kvq8::aligned4({cos, sin, block_tables, seq_starts, seq_lens, error_flag}))
        return kInvalidValue;
    if (tokens == 0 || batch == 0 || (q_heads == 0 && kv_heads == 0)) return kSuccess;
    kvpaged::Params p{};
    p.qkv = static_cast<const __half*>(qkv);
    p.cos = static_cast<const float*>(cos);
    p.sin = static_cast<const float*>(sin);
    p.q_out = static_cast<__half*>(q_out);
    p.k_cache = static_cast<__half*>(k_cache);
    p.v_cache = static_cast<__half*>(v_cache);
    p.tables = static_cast<const std::int32_t*>(block_tables);
    p.starts = static_cast<const std::int32_t*>(seq_starts);
    p.lens = static_cast<const std::int32_t*>(seq_lens);
    p.c = kvq8::make_shape(batch, kv_heads, head_dim, num_blocks, block_tokens, max_blocks);
    p.tokens = static_cast<std::uint32_t>(tokens);
    p.q_heads = static_cast<std::uint32_t>(q_heads);
    p.pairs = static_cast<std::uint32_t>(pairs);
    p.interleaved = layout == 1;
    p.error_flag = static_cast<unsigned*>(error_flag);
    const auto stream_ = static_cast<cudaStream_t>(stream);
    if (p.pairs % (p.interleaved ? 4 : 8) != 0 || !kvq8::aligned16({cos, sin}))
        return launch_pdl(kvpaged::append_scalar_kernel, dim3(p.tokens), dim3(kvpaged::kThreads), stream_, p);
    // threads of a token: one for each place of kHeld heads, or so, but with many tokens at
    // most 64 (32 query / 8 KV heads of 128: 13.1 us with 64 and 12.1 with 128 for 2048
    // tokens, 20.9 and 21.2 for 4096, 62.8 and 65.8 for 16 prompts of up to 2048; 32 threads
    // take 12.9, 22.3 and 61.3, but 45.4 instead of 39 with 32 KV heads)
    const std::uint64_t vecs = head_dim / 8, work = (q_heads + kv_heads) * (p.interleaved ? vecs : vecs - pairs / 8);
    const std::uint32_t per = work <= 32 * kvpaged::kHeld ? 32 : work <= 64 * kvpaged::kHeld || tokens > 2048 ? 64 : 128;
    const std::uint32_t each = kvpaged::kThreads / per;
    return launch_pdl(p.interleaved ? kvpaged::append_kernel<false> : kvpaged::append_kernel<true>,
                      dim3((p.tokens + each - 1) / each), dim3(kvpaged::kThreads), stream_, p, per);
}

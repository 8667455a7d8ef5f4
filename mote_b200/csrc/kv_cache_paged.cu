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

// One CTA for each token.
__global__ void __launch_bounds__(kThreads) append_kernel(const Params p) {
    pdl_launch_dependents();
    pdl_wait();
    if (blockIdx.x == 0) kvq8::check_starts(p.c, p.starts, p.tokens, p.error_flag);
    const std::uint32_t t = blockIdx.x, hd = p.c.head_dim, kvh = p.c.kv_heads;
    const std::uint32_t b = kvq8::warp_search(p.c.batch, t, [&](std::uint32_t i) {
        return static_cast<std::uint32_t>(max(__ldg(p.starts + i), 0));
    });
    const std::int32_t s0 = __ldg(p.starts + b), s1 = __ldg(p.starts + b + 1);
    if (s0 < 0 || s1 < s0 || static_cast<std::uint32_t>(s1) > p.tokens ||
        t < static_cast<std::uint32_t>(s0) || t >= static_cast<std::uint32_t>(s1))
        return;  // a row of no sequence
    const std::int64_t len = __ldg(p.lens + b), pos = len - s1 + t;
    if (len < s1 - s0 || len > static_cast<std::int64_t>(p.c.max_blocks) * p.c.block_tokens) {
        if (threadIdx.x == 0) kvq8::report(p.error_flag);
        return;
    }
    const std::int32_t block = __ldg(p.tables + static_cast<std::uint64_t>(b) * p.c.max_blocks + pos / p.c.block_tokens);
    const bool there = block >= 0 && static_cast<std::uint64_t>(block) < p.c.num_blocks;
    if (!there && threadIdx.x == 0) kvq8::report(p.error_flag);
    const std::uint64_t tile = static_cast<std::uint64_t>(block) * kvh;
    const std::uint32_t off = static_cast<std::uint32_t>(pos % p.c.block_tokens);
    const __half* row = p.qkv + static_cast<std::uint64_t>(t) * (p.q_heads + 2 * kvh) * hd;
    const auto dst_of = [&](std::uint32_t h) -> __half* {
        if (h < p.q_heads) return p.q_out + (static_cast<std::uint64_t>(t) * p.q_heads + h) * hd;
        if (!there) return nullptr;
        const std::uint32_t k = h - p.q_heads;
        return k < kvh ? p.k_cache + ((tile + k) * p.c.block_tokens + off) * hd
                       : p.v_cache + ((tile + k - kvh) * p.c.block_tokens + off) * hd;
    };
    const std::uint32_t heads = p.q_heads + 2 * kvh, rotated = p.q_heads + kvh;
    for (std::uint32_t i = threadIdx.x; i < heads * hd; i += kThreads) {
        const std::uint32_t h = i / hd, e = i - h * hd;
        const __half* src = row + h * hd;
        __half* dst = dst_of(h);
        if (dst == nullptr) continue;
        if (h >= rotated || e >= 2 * p.pairs) {
            dst[e] = src[e];
            continue;
        }
        const std::uint32_t j = p.interleaved ? e / 2 : e % p.pairs;
        const bool second = p.interleaved ? e & 1 : e >= p.pairs;
        const float a = __half2float(src[p.interleaved ? 2 * j : j]);
        const float bb = __half2float(src[p.interleaved ? 2 * j + 1 : j + p.pairs]);
        float o1, o2;
        rotate(a, bb, p.cos[static_cast<std::uint64_t>(t) * p.pairs + j],
               p.sin[static_cast<std::uint64_t>(t) * p.pairs + j], o1, o2);
        dst[e] = __float2half_rn(second ? o2 : o1);
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
    return launch_pdl(kvpaged::append_kernel, dim3(p.tokens), dim3(kvpaged::kThreads),
                      static_cast<cudaStream_t>(stream), p);
}

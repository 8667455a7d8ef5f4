// Attention of new tokens over a paged KV cache held in f16: sequence b has the
// queries q_starts[b] .. q_starts[b + 1] - 1, the last of its seq_lens[b]
// cached positions; with n of them, query i attends the positions up to its own:
//   out[i, h] = softmax_{p <= len - n + i}(scale * q[i, h] . K[p, h / g]) . V[p, h / g]
// A query before the first position (len < n) gets zeros; rows that belong to
// no sequence keep their values.
#include "mote_common.cuh"

namespace mote {
namespace attnpg {

struct Params {
    const __half* q;
    const __half* k_cache;
    const __half* v_cache;
    const std::int32_t* tables;
    const std::int32_t* starts;
    const std::int32_t* lens;
    __half* out;
    kvq8::CacheShape c;
    std::uint32_t tokens, q_heads, group, max_new;
    float scale_log2;
};

// One warp for each query row, one position after another.
template <int HD>
__global__ void __launch_bounds__(128) simple_kernel(const Params p) {
    pdl_launch_dependents();
    pdl_wait();
    const std::uint32_t lane = threadIdx.x & 31;
    const std::uint64_t item = blockIdx.x * 4ull + (threadIdx.x >> 5);
    if (item >= static_cast<std::uint64_t>(p.tokens) * p.q_heads) return;
    const std::uint32_t t = static_cast<std::uint32_t>(item / p.q_heads), h = item % p.q_heads;
    const std::uint32_t b = kvq8::warp_search(p.c.batch, t, [&](std::uint32_t i) {
        return static_cast<std::uint32_t>(max(__ldg(p.starts + i), 0));
    });
    const std::int32_t s0 = __ldg(p.starts + b), s1 = __ldg(p.starts + b + 1);
    if (s0 < 0 || s1 < s0 || static_cast<std::uint32_t>(s1) > p.tokens) {
        if (lane == 0) atomicOr(&g_device_status, kDevIndexOutOfRange);
        return;
    }
    if (t < static_cast<std::uint32_t>(s0) || t >= static_cast<std::uint32_t>(s1)) return;
    const std::int64_t len = __ldg(p.lens + b);
    if (len < 0 || len > static_cast<std::int64_t>(p.c.max_blocks) * p.c.block_tokens ||
        static_cast<std::uint32_t>(s1 - s0) > p.max_new) {
        if (lane == 0) atomicOr(&g_device_status, kDevIndexOutOfRange);
        return;
    }
    const std::int64_t reach = len - s1 + t + 1;
    constexpr int D = HD / 32;
    float q[D], o[D], m = -INFINITY, l = 0.f;
    for (int i = 0; i < D; ++i) q[i] = __half2float(p.q[item * HD + 32 * i + lane]), o[i] = 0.f;
    for (std::int64_t pos = 0; pos < reach; ++pos) {
        const std::int32_t block = __ldg(p.tables + static_cast<std::uint64_t>(b) * p.c.max_blocks + pos / p.c.block_tokens);
        const bool there = block >= 0 && static_cast<std::uint64_t>(block) < p.c.num_blocks;
        if (!there) atomicOr(&g_device_status, kDevIndexOutOfRange);
        const std::uint64_t at = ((static_cast<std::uint64_t>(there ? block : 0) * p.c.kv_heads + h / p.group) * p.c.block_tokens +
                                  pos % p.c.block_tokens) * HD + lane;
        float s = 0.f;
        for (int i = 0; i < D; ++i) s = fmaf(q[i], there ? __half2float(p.k_cache[at + 32 * i]) : 0.f, s);
        for (int d = 16; d > 0; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
        s *= p.scale_log2;
        const float mn = fmaxf(m, s), f = m == mn ? 1.f : exp2f(m - mn), w = exp2f(s - mn);
        m = mn;
        l = l * f + w;
        for (int i = 0; i < D; ++i) o[i] = fmaf(o[i], f, w * (there ? __half2float(p.v_cache[at + 32 * i]) : 0.f));
    }
    for (int i = 0; i < D; ++i) p.out[item * HD + 32 * i + lane] = __float2half_rn(reach > 0 ? o[i] / l : 0.f);
}

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
    (void)q_heads, (void)kv_heads, (void)head_dim, (void)max_new;
    return kSuccess;
}

extern "C" int mote_cuda_gqa_attention_paged_f16(
    const void* q, const void* k_cache, const void* v_cache, const void* block_tables,
    const void* q_starts, const void* seq_lens, void* out, uint64_t tokens, uint64_t batch,
    uint64_t q_heads, uint64_t kv_heads, uint64_t head_dim, uint64_t num_blocks,
    uint64_t block_tokens, uint64_t max_blocks, uint64_t max_new, float scale, void* workspace,
    uint64_t workspace_bytes, void* stream) {
    using namespace mote;
    if (q == nullptr || k_cache == nullptr || v_cache == nullptr || block_tables == nullptr ||
        q_starts == nullptr || seq_lens == nullptr || out == nullptr || stream == nullptr)
        return kInvalidValue;
    if (!kvq8::shape_ok(batch, kv_heads, head_dim, num_blocks, block_tokens, max_blocks) ||
        kv_heads == 0 || q_heads % kv_heads != 0 || q_heads > 65535 || q_heads / kv_heads > 128 ||
        tokens > 0x7fffffffull || max_new > 0x7fffffffull || !std::isfinite(scale) ||
        !(scale > 0.f) || !kvq8::aligned16({q, k_cache, v_cache, out}) ||
        !kvq8::aligned4({block_tables, q_starts, seq_lens}))
        return kInvalidValue;
    if (tokens == 0 || batch == 0 || q_heads == 0) return kSuccess;
    (void)workspace, (void)workspace_bytes;
    attnpg::Params p{};
    p.q = static_cast<const __half*>(q);
    p.k_cache = static_cast<const __half*>(k_cache);
    p.v_cache = static_cast<const __half*>(v_cache);
    p.tables = static_cast<const std::int32_t*>(block_tables);
    p.starts = static_cast<const std::int32_t*>(q_starts);
    p.lens = static_cast<const std::int32_t*>(seq_lens);
    p.out = static_cast<__half*>(out);
    p.c = kvq8::make_shape(batch, kv_heads, head_dim, num_blocks, block_tokens, max_blocks);
    p.tokens = static_cast<std::uint32_t>(tokens);
    p.q_heads = static_cast<std::uint32_t>(q_heads);
    p.group = static_cast<std::uint32_t>(q_heads / kv_heads);
    p.max_new = static_cast<std::uint32_t>(max_new);
    p.scale_log2 = scale * 1.4426950408889634f;
    const std::uint64_t blocks = (tokens * q_heads + 3) / 4;
    if (blocks > 0x7fffffffull) return kInvalidValue;
    return launch_pdl(head_dim == 64 ? attnpg::simple_kernel<64> : attnpg::simple_kernel<128>,
                      dim3(static_cast<unsigned>(blocks)), dim3(128), static_cast<cudaStream_t>(stream), p);
}

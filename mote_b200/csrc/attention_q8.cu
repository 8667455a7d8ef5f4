// Decode attention over the 8-bit paged cache (kv_cache_q8.cu): one query
// token per sequence,
//   out[b, h] = softmax(scale * q[b, h] . K_b[:len_b, h / g]) . V_b
// with K and V = q * (the scale of their block and head).
//
// One CTA per (query head, sequence); each warp takes every eighth
// position, lanes across head_dim, with its own running maximum and sum.
#include "mote_common.cuh"

namespace mote {
namespace attn8 {

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
    std::uint32_t q_heads, group;
    float scale_log2;
};

constexpr int kWarps = 8;

template <int HD>
__global__ void __launch_bounds__(32 * kWarps) decode_kernel(const Params p) {
    constexpr int E = HD / 32;
    __shared__ float sm[kWarps], sl[kWarps], so[kWarps][HD];
    pdl_launch_dependents();
    pdl_wait();
    const std::uint32_t h = blockIdx.x, b = blockIdx.y, kvh = h / p.group;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const std::int64_t cap = static_cast<std::int64_t>(p.c.max_blocks) * p.c.block_tokens;
    const std::int64_t len = min(static_cast<std::int64_t>(max(p.seq_lens[b], 0)), cap);
    const __half* q = p.q + (static_cast<std::uint64_t>(b) * p.q_heads + h) * HD + lane * E;
    float qv[E], o[E];
    for (int e = 0; e < E; ++e) qv[e] = __half2float(q[e]), o[e] = 0.f;
    float m = -INFINITY, l = 0.f;
    for (std::int64_t pos = warp; pos < len; pos += kWarps) {
        const std::int32_t block = p.tables[static_cast<std::uint64_t>(b) * p.c.max_blocks + pos / p.c.block_tokens];
        if (block < 0 || static_cast<std::uint64_t>(block) >= p.c.num_blocks) {
            if (lane == 0) atomicOr(&g_device_status, kDevIndexOutOfRange);
            continue;
        }
        const std::uint64_t tile = static_cast<std::uint64_t>(block) * p.c.kv_heads + kvh;
        const std::uint64_t at = (tile * p.c.block_tokens + pos % p.c.block_tokens) * HD + lane * E;
        float s = 0.f;
        for (int e = 0; e < E; ++e) s += qv[e] * p.k_cache[at + e];
        for (int d = 16; d > 0; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
        s *= p.k_scales[tile] * p.scale_log2;
        const float mn = fmaxf(m, s), f = mn == m ? 1.f : exp2f(m - mn), w = exp2f(s - mn);
        m = mn;
        l = l * f + w;
        const float wv = w * p.v_scales[tile];
        for (int e = 0; e < E; ++e) o[e] = o[e] * f + wv * p.v_cache[at + e];
    }
    if (lane == 0) sm[warp] = m, sl[warp] = l;
    for (int e = 0; e < E; ++e) so[warp][lane * E + e] = o[e];
    __syncthreads();
    if (threadIdx.x < HD) {
        float mt = -INFINITY, lt = 0.f, ot = 0.f;
        bool any = false;
        for (int w = 0; w < kWarps; ++w) {
            any |= sl[w] != 0.f;
            mt = fmaxf(mt, sm[w]);
        }
        for (int w = 0; w < kWarps; ++w) {
            if (sl[w] == 0.f) continue;
            const float f = exp2f(sm[w] - mt);
            lt += sl[w] * f;
            ot += so[w][threadIdx.x] * f;
        }
        p.out[(static_cast<std::uint64_t>(b) * p.q_heads + h) * HD + threadIdx.x] =
            __float2half_rn(any ? ot / lt : 0.f);
    }
}

}  // namespace attn8
}  // namespace mote

extern "C" int mote_cuda_gqa_attention_decode_q8_workspace_bytes(uint64_t batch, uint64_t q_heads,
                                                                  uint64_t kv_heads,
                                                                  uint64_t head_dim,
                                                                  uint64_t* bytes) {
    (void)batch, (void)q_heads, (void)kv_heads, (void)head_dim;
    if (bytes == nullptr) return mote::kInvalidValue;
    *bytes = 0;
    return mote::kSuccess;
}

extern "C" int mote_cuda_gqa_attention_decode_q8(
    const void* q, const void* k_cache, const void* v_cache, const void* k_scales,
    const void* v_scales, const void* block_tables, const void* seq_lens, void* out,
    uint64_t batch, uint64_t q_heads, uint64_t kv_heads, uint64_t head_dim, uint64_t num_blocks,
    uint64_t block_tokens, uint64_t max_blocks, float scale, void* workspace,
    uint64_t workspace_bytes, void* stream) {
    using namespace mote;
    (void)workspace, (void)workspace_bytes;
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
    p.scale_log2 = scale * 1.4426950408889634f;
    const dim3 grid(static_cast<unsigned>(q_heads), static_cast<unsigned>(batch));
    const auto s = static_cast<cudaStream_t>(stream);
    return head_dim == 64
               ? launch_pdl(attn8::decode_kernel<64>, grid, dim3(32 * attn8::kWarps), s, p)
               : launch_pdl(attn8::decode_kernel<128>, grid, dim3(32 * attn8::kWarps), s, p);
}

// Causal grouped-query attention over whole prompts, packed back to back:
// sequence b has the queries q_starts[b] .. q_starts[b + 1] - 1 and the
// positions kv_starts[b] .. kv_starts[b + 1] - 1 of k and v; with n_q and n_k
// of them, query i stands at position n_k - n_q + i and attends the
// positions up to its own:
//   out[i, h] = softmax_{p <= n_k - n_q + i}(scale * q[i, h] . k[p, h / g]) . v[p, h / g]
// A query before the first position (n_k < n_q) gets zeros; rows of out that
// belong to no sequence keep their values.
//
// One warp per (query, head), lanes across head_dim.
#include "mote_common.cuh"

namespace mote {
namespace attnv {

struct Params {
    const __half* q;
    const __half* k;
    const __half* v;
    const std::int32_t* q_starts;
    const std::int32_t* kv_starts;
    __half* out;
    std::uint32_t tokens, kv_tokens, batch, q_heads, kv_heads, group;
    float scale_log2;
};

template <int HD>
__global__ void __launch_bounds__(128) packed_kernel(const Params p) {
    constexpr int E = HD / 32;
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x % 32;
    if (blockIdx.x == 0 && blockIdx.y == 0)
        for (std::uint32_t b = threadIdx.x; b < p.batch; b += blockDim.x) {
            const std::int32_t q0 = p.q_starts[b], q1 = p.q_starts[b + 1];
            const std::int32_t k0 = p.kv_starts[b], k1 = p.kv_starts[b + 1];
            if (q0 < 0 || q1 < q0 || static_cast<std::uint32_t>(q1) > p.tokens || k0 < 0 || k1 < k0 ||
                static_cast<std::uint32_t>(k1) > p.kv_tokens)
                atomicOr(&g_device_status, kDevIndexOutOfRange);
        }
    const std::uint32_t h = blockIdx.y * 4 + threadIdx.x / 32, row = blockIdx.x;
    if (h >= p.q_heads) return;
    const std::uint32_t b = kvq8::warp_search(p.batch, row, [&](std::uint32_t i) {
        return static_cast<std::uint32_t>(max(p.q_starts[i], 0));
    });
    const std::int32_t q0 = p.q_starts[b], q1 = p.q_starts[b + 1];
    const std::int32_t k0 = p.kv_starts[b], k1 = p.kv_starts[b + 1];
    if (q0 < 0 || static_cast<std::int64_t>(row) < q0 || static_cast<std::int64_t>(row) >= q1 ||
        static_cast<std::uint32_t>(q1) > p.tokens || k0 < 0 || k1 < k0 ||
        static_cast<std::uint32_t>(k1) > p.kv_tokens)
        return;
    const std::int64_t last = static_cast<std::int64_t>(k1) - k0 - (q1 - static_cast<std::int64_t>(row));
    const std::uint64_t qa = (static_cast<std::uint64_t>(row) * p.q_heads + h) * HD + lane * E;
    float qv[E], o[E], m = -INFINITY, l = 0.f;
    for (int e = 0; e < E; ++e) qv[e] = __half2float(p.q[qa + e]), o[e] = 0.f;
    for (std::int64_t pos = 0; pos <= last; ++pos) {
        const std::uint64_t at =
            (static_cast<std::uint64_t>(k0 + pos) * p.kv_heads + h / p.group) * HD + lane * E;
        float s = 0.f;
        for (int e = 0; e < E; ++e) s += qv[e] * __half2float(p.k[at + e]);
        for (int d = 16; d > 0; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
        s *= p.scale_log2;
        const float mn = fmaxf(m, s), f = mn == m ? 1.f : exp2f(m - mn), w = exp2f(s - mn);
        m = mn;
        l = l * f + w;
        for (int e = 0; e < E; ++e) o[e] = o[e] * f + w * __half2float(p.v[at + e]);
    }
    for (int e = 0; e < E; ++e) p.out[qa + e] = __float2half_rn(last >= 0 ? o[e] / l : 0.f);
}

}  // namespace attnv
}  // namespace mote

extern "C" int mote_cuda_gqa_attention_packed_f16(const void* q, const void* k, const void* v,
                                                  const void* q_starts, const void* kv_starts,
                                                  void* out, uint64_t tokens, uint64_t kv_tokens,
                                                  uint64_t batch, uint64_t q_heads,
                                                  uint64_t kv_heads, uint64_t head_dim,
                                                  float scale, void* stream) {
    using namespace mote;
    if (q == nullptr || k == nullptr || v == nullptr || q_starts == nullptr ||
        kv_starts == nullptr || out == nullptr || stream == nullptr)
        return kInvalidValue;
    if ((head_dim != 64 && head_dim != 128) || kv_heads == 0 || q_heads % kv_heads != 0 ||
        q_heads > 65535 || q_heads / kv_heads > 128 || batch > (1u << 20) ||
        tokens > 0x7fffffffull || kv_tokens > 0x7fffffffull || !std::isfinite(scale) ||
        !(scale > 0.f) || !kvq8::aligned16({q, k, v, out}) ||
        !kvq8::aligned4({q_starts, kv_starts}))
        return kInvalidValue;
    if (tokens == 0 || batch == 0 || q_heads == 0) return kSuccess;
    attnv::Params p{};
    p.q = static_cast<const __half*>(q);
    p.k = static_cast<const __half*>(k);
    p.v = static_cast<const __half*>(v);
    p.q_starts = static_cast<const std::int32_t*>(q_starts);
    p.kv_starts = static_cast<const std::int32_t*>(kv_starts);
    p.out = static_cast<__half*>(out);
    p.tokens = static_cast<std::uint32_t>(tokens);
    p.kv_tokens = static_cast<std::uint32_t>(kv_tokens);
    p.batch = static_cast<std::uint32_t>(batch);
    p.q_heads = static_cast<std::uint32_t>(q_heads);
    p.kv_heads = static_cast<std::uint32_t>(kv_heads);
    p.group = static_cast<std::uint32_t>(q_heads / kv_heads);
    p.scale_log2 = scale * 1.4426950408889634f;
    const dim3 grid(static_cast<unsigned>(tokens), static_cast<unsigned>((q_heads + 3) / 4));
    const auto s = static_cast<cudaStream_t>(stream);
    return head_dim == 64 ? launch_pdl(attnv::packed_kernel<64>, grid, dim3(128), s, p)
                          : launch_pdl(attnv::packed_kernel<128>, grid, dim3(128), s, p);
}

// cos/sin tables of rotary positions with several axes (time, height, width
// of an image or a video), the f32 [tokens, pairs] tables that every rotation
// of this library takes:
//   angle(t, j) = positions[axis(j)][t] * theta^-e(j),   j < pairs
// order 0, sections: axis a has the next sections[a] pairs, e(j) = j / pairs;
// order 1, interleaved: axis j % axes while j / axes < sections[j % axes], axis
//   0 otherwise, e(j) = j / pairs;
// order 2, own: the pairs of order 0, e = (the pair's number within its axis) /
//   sections[a], so that every axis has a whole series of frequencies.
//
// No reference counterpart (the reference takes such tables as inputs,
// crates/mote-backend-hip/src/rope.rs:66-82).
//
// An angle of a far position needs more than 32 bits before it is reduced to a
// turn.  Frequencies are 64-bit fractions of a turn, so position * frequency modulo 2^64
// is the angle without its whole turns, exactly, in three integer instructions.  A
// frequency f is off by 2^-64 of a turn and, from exp2 and its argument in 64 bits, by up
// to (4 + 3 ln(1 / f)) 2^-53 of itself: the angle by about position * 2^-51 at most, since
// the low frequencies have the large share.  What is left of it to the nearest quarter
// turn goes to f32 for the sine and cosine.  Results are within 2^-23 of the angle's
// own up to positions of 2^26 or so.  65536 positions of 64 pairs: 8.2 us, 0.64 of the
// copy bandwidth (about 28 instructions a pair take half of that; 11.7 us with products
// in f64 and one token at a time).
#include "mote_common.cuh"

#include <cmath>

namespace mote {
namespace ropeaxes {

constexpr std::uint32_t kMaxAxes = 4;
constexpr std::uint32_t kMaxPairs = 128;
constexpr int kThreads = 256;
// Tokens of a thread at a time and CTAs of an SM (tokens, CTAs: 1, 4 took 10.7 us; 2, 4
// 9.2; 4, 4 8.2; 4, 3 8.7 and 2, 6 10.2).
constexpr int kAhead = 4, kPerSm = 4;

struct Params {
    const std::int32_t* positions;  // [axes, tokens]
    float* cos;
    float* sin;
    std::uint64_t tokens;
    std::uint32_t pairs;
    std::uint64_t turns[kMaxPairs];  // of a position, in 2^-64
    std::uint8_t axis[kMaxPairs];
};

__device__ __forceinline__ void angle(std::int32_t position, std::uint64_t turns, float& c, float& s) {
    const std::uint64_t phase = static_cast<std::uint64_t>(static_cast<std::int64_t>(position)) * turns;
    // the nearest quarter turn, and what is left in 2^-32 turns: at most 2^29
    const std::uint32_t u = static_cast<std::uint32_t>(phase >> 32) + (1u << 29), k = u >> 30;
    const std::int32_t r = static_cast<std::int32_t>(u & 0x3fffffffu) - (1 << 29);
    // sine and cosine of x, |x| <= pi / 4, by their Taylor series: what follows x^9
    // and x^10 is below 2^-28
    const float x = static_cast<float>(r) * 1.46291807926715968e-9f;  // 2 pi / 2^32
    const float y = x * x;
    const float sr = fmaf(x * y, fmaf(y, fmaf(y, fmaf(y, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), x);
    const float cr = fmaf(y, fmaf(y, fmaf(y, fmaf(y, fmaf(y, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
    const float a = k & 1 ? sr : cr, b = k & 1 ? cr : sr;
    c = (k + 1) & 2 ? -a : a;
    s = k & 2 ? -b : b;
}

// A thread keeps VEC neighbouring pairs and goes through tokens.
template <int VEC>
__global__ void __launch_bounds__(kThreads, kPerSm) table_kernel(const __grid_constant__ Params p) {
    pdl_launch_dependents();
    const std::uint32_t cols = p.pairs / VEC, rows = blockDim.x / cols;
    const std::uint32_t j = threadIdx.x % cols * VEC, r = threadIdx.x / cols;
    std::uint64_t turns[VEC];
    const std::int32_t* position[VEC];
    // (through shared memory: parameters at an address of each lane's own are read one
    // lane after another)
    __shared__ std::uint64_t all_turns[kMaxPairs];
    __shared__ std::uint32_t all_axes[kMaxPairs];
    for (std::uint32_t i = threadIdx.x; i < p.pairs; i += blockDim.x) all_turns[i] = p.turns[i], all_axes[i] = p.axis[i];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        turns[e] = all_turns[j + e];
        position[e] = p.positions + all_axes[j + e] * p.tokens;
    }
    pdl_wait();
    // kAhead tokens of a thread at a time, whose positions load together
    const std::uint64_t step = static_cast<std::uint64_t>(gridDim.x) * rows;
    for (std::uint64_t t0 = static_cast<std::uint64_t>(blockIdx.x) * rows + r; t0 < p.tokens; t0 += kAhead * step) {
        std::int32_t at[kAhead][VEC];
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (t0 + i * step < p.tokens) at[i][e] = __ldg(position[e] + t0 + i * step);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const std::uint64_t t = t0 + i * step;
            if (t >= p.tokens) break;
            float c[VEC], s[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) angle(at[i][e], turns[e], c[e], s[e]);
            float* const co = p.cos + t * p.pairs + j;
            float* const so = p.sin + t * p.pairs + j;
            if constexpr (VEC == 4) {
                *reinterpret_cast<float4*>(co) = make_float4(c[0], c[1], c[2], c[3]);
                *reinterpret_cast<float4*>(so) = make_float4(s[0], s[1], s[2], s[3]);
            } else {
                *co = c[0];
                *so = s[0];
            }
        }
    }
}

}  // namespace ropeaxes
}  // namespace mote

extern "C" int mote_cuda_rope_cos_sin_axes_f32(const void* positions, void* cos_out, void* sin_out,
                                               uint64_t tokens, uint64_t axes, uint32_t section0,
                                               uint32_t section1, uint32_t section2,
                                               uint32_t section3, uint32_t order, double theta,
                                               void* stream) {
    using namespace mote;
    using namespace mote::ropeaxes;
    if (positions == nullptr || cos_out == nullptr || sin_out == nullptr || stream == nullptr)
        return kInvalidValue;
    if (axes == 0 || axes > kMaxAxes || order > 2 || !std::isfinite(theta) || theta < 1.0 ||
        tokens > 0x7fffffffull || !kvq8::aligned4({positions, cos_out, sin_out}))
        return kInvalidValue;
    const std::uint32_t sections[kMaxAxes] = {section0, section1, section2, section3};
    std::uint64_t pairs = 0;
    for (std::uint32_t a = 0; a < kMaxAxes; ++a) {
        if (a >= axes && sections[a] != 0) return kInvalidValue;
        pairs += sections[a];
    }
    if (pairs > kMaxPairs) return kInvalidValue;
    if (order == 1)  // every axis finds its pairs
        for (std::uint32_t a = 1; a < axes; ++a)
            if (sections[a] != 0 && a + axes * (sections[a] - 1ull) >= pairs) return kInvalidValue;
    if (tokens == 0 || pairs == 0) return kSuccess;
    Params p{};
    p.positions = static_cast<const std::int32_t*>(positions);
    p.cos = static_cast<float*>(cos_out);
    p.sin = static_cast<float*>(sin_out);
    p.tokens = tokens;
    p.pairs = static_cast<std::uint32_t>(pairs);
    const double log2_theta = std::log2(theta);
    std::uint32_t axis = 0, first = 0;
    for (std::uint32_t j = 0; j < pairs; ++j) {
        while (j - first >= sections[axis]) first += sections[axis++];
        double e = static_cast<double>(j) / static_cast<double>(pairs);
        p.axis[j] = static_cast<std::uint8_t>(axis);
        if (order == 1) {
            const std::uint32_t a = j % static_cast<std::uint32_t>(axes);
            p.axis[j] = static_cast<std::uint8_t>(j / axes < sections[a] ? a : 0);
        } else if (order == 2) {
            e = static_cast<double>(j - first) / sections[axis];
        }
        // theta^-e / (2 pi) below 0.16
        p.turns[j] = static_cast<std::uint64_t>(std::ldexp(std::exp2(-e * log2_theta) * 0.15915494309189533577, 64));
    }
    const bool vec = pairs % 4 == 0 && kvq8::aligned16({cos_out, sin_out});
    const std::uint32_t cols = p.pairs / (vec ? 4 : 1), rows = kThreads / cols;
    const std::uint64_t blocks = (tokens + rows - 1) / rows;
    const dim3 grid(static_cast<unsigned>(blocks < 148 * kPerSm ? blocks : 148 * kPerSm));
    return launch_pdl(vec ? table_kernel<4> : table_kernel<1>, grid, dim3(cols * rows),
                      static_cast<cudaStream_t>(stream), p);
}

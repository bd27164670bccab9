// Routing of tokens to experts: scores of every expert, top-k by score and bias among the kept groups, and their weights.
//
//   s = softmax(l) or 1 / (1 + exp(-l));  c = s + bias;  groups of experts in order, by their largest c or the sum of their
//   two largest; the top-k of the kept groups by (c, lowest index); weights s, divided by their sum, times a factor.
//
// The order is what the experts' products depend on, and two scores of a token may be as near as their logits' last bits:
// scores and biased scores are 64-bit numbers, whose ties are ties of the definition.
#include "common.hpp"

#include <cmath>

namespace vt {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kMaxExperts = 1024, kMaxTopK = 16, kMaxGroups = 64;

struct Geometry {
    int tokens, experts, top_k, groups, kept;
    bool sigmoid, pairs, renormalize;
    float scale;
    int score_type;
};

__device__ __forceinline__ void write_score(void* scores, std::int64_t at, int type, float v) {
    if (type == kF16) static_cast<__half*>(scores)[at] = from_f32<__half>(v);
    else if (type == kBF16) static_cast<__hip_bfloat16*>(scores)[at] = from_f32<__hip_bfloat16>(v);
    else static_cast<float*>(scores)[at] = v;
}

template <class V>
__device__ __forceinline__ V wave_sum(V v) {
#pragma unroll
    for (int step = 32; step; step >>= 1) v += __shfl_xor(v, step, 64);
    return v;
}

// A wave per token, experts lane, lane + 64, ..
template <class T, int N>
__global__ __launch_bounds__(kThreads) void route(const T* __restrict__ logits, const float* __restrict__ bias,
                                                  std::int64_t* __restrict__ indices, void* __restrict__ scores, Geometry g) {
    __shared__ double all[kWaves][64 * N];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int token = blockIdx.x * kWaves + wave;
    if (token >= g.tokens) return;
    const T* row = logits + static_cast<std::int64_t>(token) * g.experts;
    const double none = -__builtin_inf();
    double x[N], s[N], c[N], top = none;
    bool broken = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = lane + 64 * i;
        x[i] = e < g.experts ? static_cast<double>(to_f32(row[e])) : none;
        broken |= x[i] != x[i] || (!g.sigmoid && x[i] == -none);
        top = fmax(top, x[i]);
    }
#pragma unroll
    for (int step = 32; step; step >>= 1) top = fmax(top, __shfl_xor(top, step, 64));
    if (g.sigmoid) {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = 1.0 / (1.0 + exp(-x[i]));
    } else {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s[i] = x[i] == none ? 0.0 : exp(x[i] - top);
            sum += s[i];
        }
        sum = wave_sum(sum);
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = sum > 0.0 ? s[i] / sum : 0.0;
    }
    unsigned open = 0;  // the lane's experts that may be chosen
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = lane + 64 * i;
        if (e < g.experts) open |= 1u << i;
        c[i] = e < g.experts && x[i] != none ? (bias ? s[i] + bias[e] : s[i]) : none;
        broken |= c[i] != c[i];
    }
    broken = __any(broken);
    if (g.groups > 1 && !broken) {
        const int size = g.experts / g.groups;
#pragma unroll
        for (int i = 0; i < N; ++i) all[wave][lane + 64 * i] = c[i];
        __builtin_amdgcn_wave_barrier();
        // Lane g ranks group g.
        double first = none, second = none;
        if (lane < g.groups)
            for (int i = 0; i < size; ++i) {
                const double v = all[wave][lane * size + i];
                second = fmax(second, fmin(first, v));
                first = fmax(first, v);
            }
        const double rank = g.pairs && size > 1 ? first + second : first;
        int ahead = 0;
        for (int i = 0; i < g.groups; ++i) {
            const double other = __shfl(rank, i, 64);
            ahead += other > rank || (other == rank && i < lane);
        }
        const unsigned long long kept = __ballot(lane < g.groups && ahead < g.kept);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = lane + 64 * i;
            if (e < g.experts && !(kept >> (e / size) & 1)) open &= ~(1u << i);
        }
    }
    int chosen = -1;
    double weight = 0.0;
    for (int k = 0; k < g.top_k; ++k) {
        double best = none, score = 0.0;
        int at = kMaxExperts;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if ((open >> i & 1) && (at == kMaxExperts || c[i] > best)) best = c[i], score = s[i], at = lane + 64 * i;
#pragma unroll
        for (int step = 32; step; step >>= 1) {
            const double other = __shfl_xor(best, step, 64), other_score = __shfl_xor(score, step, 64);
            const int other_at = __shfl_xor(at, step, 64);
            if (other_at < kMaxExperts && (at == kMaxExperts || other > best || (other == best && other_at < at)))
                best = other, score = other_score, at = other_at;
        }
        if (lane == k) chosen = at, weight = score;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (at == lane + 64 * i) open &= ~(1u << i);
    }
    const double sum = wave_sum(weight);
    if (lane < g.top_k) {
        const std::int64_t at = static_cast<std::int64_t>(token) * g.top_k + lane;
        const double share = !g.renormalize ? weight : sum > 0.0 ? weight / sum : 0.0;
        indices[at] = broken ? -1 : chosen;
        write_score(scores, at, g.score_type, broken ? __builtin_nanf("") : static_cast<float>(share * g.scale));
    }
}

template <class T>
void launch(const void* logits, const float* bias, std::int64_t* indices, void* scores, const Geometry& g, hipStream_t stream) {
    const unsigned grid = static_cast<unsigned>((static_cast<std::int64_t>(g.tokens) + kWaves - 1) / kWaves);
    const auto* x = static_cast<const T*>(logits);
    if (g.experts <= 64) route<T, 1><<<grid, kThreads, 0, stream>>>(x, bias, indices, scores, g);
    else if (g.experts <= 128) route<T, 2><<<grid, kThreads, 0, stream>>>(x, bias, indices, scores, g);
    else if (g.experts <= 256) route<T, 4><<<grid, kThreads, 0, stream>>>(x, bias, indices, scores, g);
    else if (g.experts <= 512) route<T, 8><<<grid, kThreads, 0, stream>>>(x, bias, indices, scores, g);
    else route<T, 16><<<grid, kThreads, 0, stream>>>(x, bias, indices, scores, g);
}

}  // namespace
}  // namespace vt

#define VT_EXPORT extern "C" __attribute__((visibility("default")))

VT_EXPORT int venturi_route_run(const void* logits, const float* bias, std::int64_t* indices, void* scores, int tokens, int experts,
                                int top_k, int groups, int kept_groups, int sigmoid, int pairs, int renormalize, float scale,
                                int dtype, int score_dtype, void* stream) {
    return vt::guarded([&] {
        vt::require(tokens > 0 && experts > 0 && experts <= vt::kMaxExperts, "routing takes 1 to 1024 experts");
        vt::require(groups > 0 && groups <= vt::kMaxGroups && experts % groups == 0 && kept_groups > 0 && kept_groups <= groups,
                    "routing takes up to 64 groups of equal size");
        vt::require(top_k > 0 && top_k <= vt::kMaxTopK && top_k <= experts / groups * kept_groups,
                    "routing takes top_k of at most 16 and of the kept groups' experts");
        vt::require(std::isfinite(scale), "the routing factor must be finite");
        vt::require(logits && indices && scores, "null routing operand");
        vt::require(score_dtype >= vt::kF16 && score_dtype <= vt::kF32, "unsupported score type");
        vt::require(vt::aligned(logits, dtype == vt::kF32 ? 4 : 2) && vt::aligned(bias, 4) && vt::aligned(indices, 8) &&
                        vt::aligned(scores, score_dtype == vt::kF32 ? 4 : 2),
                    "routing operands must be aligned to their elements");
        const vt::Geometry g{tokens, experts, top_k, groups, kept_groups, sigmoid != 0, pairs != 0, renormalize != 0, scale, score_dtype};
        const auto s = static_cast<hipStream_t>(stream);
        if (dtype == vt::kF16)
            vt::launch<__half>(logits, bias, indices, scores, g, s);
        else if (dtype == vt::kBF16)
            vt::launch<__hip_bfloat16>(logits, bias, indices, scores, g, s);
        else if (dtype == vt::kF32)
            vt::launch<float>(logits, bias, indices, scores, g, s);
        else
            throw vt::Invalid("unsupported scalar type");
    });
}

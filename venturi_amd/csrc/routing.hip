// Routing of tokens to experts: scores of every expert, top-k by score and bias among the kept groups, and their weights.
//
//   s = softmax(l) or 1 / (1 + exp(-l));  c = s + bias;  groups of experts in order, by their largest c or the sum of their
//   two largest; the top-k of the kept groups by (c, lowest index); weights s, divided by their sum, times a factor.
//
// The order is what the experts' products depend on, and two scores of a token may be as near as their logits' last bits:
// scores and biased scores are 64-bit numbers. Without a bias (and sums of scores) the order is the logits' own, and 16-bit
// logits need no score but the chosen ones'.
//
// Bound by the vector unit, and for few tokens by the length of its chain: a score's exponential and division are 24 steps of 64
// bits, a choice ten of moves and maxima between the lanes of a token. So a lane sorts its own few experts once (19 exchanges
// of eight), and a choice then is the largest of the lists' heads: 16384 tokens of 128 experts, 16-bit logits 6.0 us (49 with a
// wave per token and one 64-bit maximum over it for each choice), 32-bit ones 7.8; 4099 tokens of 256 in 8 groups, a bias, 8.2
// (22); one token 3.5 to 6.0, of which a launch is 2.3. Memory would take 16384 x 128 of 16 bits 1.1 us.
#include "common.hpp"

#include <cmath>
#include <type_traits>

namespace vt {
namespace {

constexpr int kThreads = 256;
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

template <int CONTROL>
__device__ __forceinline__ std::uint32_t moved(std::uint32_t v) {
    return static_cast<std::uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), CONTROL, 0xf, 0xf, true));
}
template <int CONTROL>
__device__ __forceinline__ double moved(double v) {
    const auto w = __builtin_bit_cast(std::uint64_t, v);
    return __builtin_bit_cast(double, static_cast<std::uint64_t>(moved<CONTROL>(static_cast<std::uint32_t>(w >> 32))) << 32 |
                                          moved<CONTROL>(static_cast<std::uint32_t>(w)));
}
template <int CONTROL>
__device__ __forceinline__ float moved(float v) {
    return __builtin_bit_cast(float, moved<CONTROL>(__builtin_bit_cast(std::uint32_t, v)));
}
template <bool HALVES>
__device__ __forceinline__ std::uint32_t across(std::uint32_t v) {
    // The rows (halves) of the wave exchanged: of a pair both get the other's.
    typedef unsigned uint2v __attribute__((ext_vector_type(2)));
    const bool second = threadIdx.x & (HALVES ? 32 : 16);
    const uint2v pair = HALVES ? __builtin_bit_cast(uint2v, __builtin_amdgcn_permlane32_swap(v, v, false, false))
                               : __builtin_bit_cast(uint2v, __builtin_amdgcn_permlane16_swap(v, v, false, false));
    return second ? pair[0] : pair[1];
}
template <bool HALVES>
__device__ __forceinline__ double across(double v) {
    const auto w = __builtin_bit_cast(std::uint64_t, v);
    return __builtin_bit_cast(double, static_cast<std::uint64_t>(across<HALVES>(static_cast<std::uint32_t>(w >> 32))) << 32 |
                                          across<HALVES>(static_cast<std::uint32_t>(w)));
}
template <bool HALVES>
__device__ __forceinline__ float across(float v) {
    return __builtin_bit_cast(float, across<HALVES>(__builtin_bit_cast(std::uint32_t, v)));
}

// v over the lanes of a token, by moves within rows of 16 lanes and then across them; every lane gets it.
template <int LANES, class V, class F>
__device__ __forceinline__ V join(V v, F&& f) {
    v = f(v, moved<0xb1>(v));   // the neighbour
    v = f(v, moved<0x4e>(v));   // two lanes on
    v = f(v, moved<0x141>(v));  // eight lanes mirrored
    v = f(v, moved<0x140>(v));  // sixteen lanes mirrored
    if constexpr (LANES >= 32) v = f(v, across<false>(v));
    if constexpr (LANES == 64) v = f(v, across<true>(v));
    return v;
}
template <int LANES>
__device__ __forceinline__ double join_sum(double v) {
    return join<LANES>(v, [](double a, double b) { return a + b; });
}

// LDS that a wave's lanes write for each other.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// N neighbouring experts of a lane; those past the last are not touched. VECTOR: rows of 16-byte vectors.
template <class T, int N, bool VECTOR>
__device__ __forceinline__ void load(const T* __restrict__ from, int first, int experts, T (&v)[N]) {
    if constexpr (VECTOR) {
        if (first < experts) {
            constexpr int count = N * sizeof(T) < 16 ? 1 : N * sizeof(T) / 16;
            if constexpr (N * sizeof(T) < 16) {
                const uint2 w = *reinterpret_cast<const uint2*>(from + first);
                __builtin_memcpy(v, &w, sizeof(w));
            } else {
                uint4 w[count];
#pragma unroll
                for (int i = 0; i < count; ++i) w[i] = reinterpret_cast<const uint4*>(from + first)[i];
                __builtin_memcpy(v, w, sizeof(w));
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (first + i < experts) v[i] = from[first + i];
    }
}

// 2^x of B numbers: the Taylor series of e^r for |r| <= ln 2 / 2, whose 13th power is below 2^-53, times 2^n; some units of
// 2^-53 off. Step by step for all of them: one number's steps wait for each other.
template <int B>
__device__ __forceinline__ void power(double (&x)[B]) {
    constexpr double kTerms[] = {1.0 / 479001600.0, 1.0 / 39916800.0, 1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0,
                                 1.0 / 720.0, 1.0 / 120.0, 1.0 / 24.0, 1.0 / 6.0, 0.5, 1.0, 1.0};
    double r[B], p[B];
    int n[B];
#pragma unroll
    for (int i = 0; i < B; ++i) {
        const double whole = rint(x[i]);
        n[i] = static_cast<int>(whole);
        r[i] = (x[i] - whole) * 0.693147180559945309417;
        p[i] = 1.0 / 6227020800.0;
    }
#pragma unroll
    for (int t = 0; t < 13; ++t) {
#pragma unroll
        for (int i = 0; i < B; ++i) p[i] = fma(p[i], r[i], kTerms[t]);
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 0; i < B; ++i) x[i] = ldexp(p[i], n[i]);
}

// 1 / x of normal numbers, by two steps of Newton's from the instruction's first bits.
template <int B>
__device__ __forceinline__ void reciprocal(double (&x)[B]) {
    double r[B];
#pragma unroll
    for (int i = 0; i < B; ++i) r[i] = __builtin_amdgcn_rcp(x[i]);
#pragma unroll
    for (int step = 0; step < 2; ++step) {
        double rest[B];
#pragma unroll
        for (int i = 0; i < B; ++i) rest[i] = fma(-x[i], r[i], 1.0);
#pragma unroll
        for (int i = 0; i < B; ++i) r[i] = fma(r[i], rest[i], r[i]);
    }
#pragma unroll
    for (int i = 0; i < B; ++i) x[i] = r[i];
}

constexpr double kLog2e = 1.44269504088896340736;
constexpr double kLeast = -1.7976931348623157e308;  // of biases of -inf: a masked expert's -inf lies below, whatever its index

// exp(x - top), or 1 / (1 + exp(-x)); below 2^-1000 they are 0, of NaN too.
template <bool SIGMOID, int B>
__device__ __forceinline__ void terms(const float (&x)[B], double top, double (&v)[B]) {
    bool none[B];
#pragma unroll
    for (int i = 0; i < B; ++i) {
        v[i] = SIGMOID ? static_cast<double>(x[i]) * -kLog2e : (static_cast<double>(x[i]) - top) * kLog2e;
        none[i] = SIGMOID ? !(v[i] < 1000.0) : !(v[i] > -1000.0);
        v[i] = fmax(fmin(v[i], 1000.0), -1000.0);
    }
    power(v);
    if constexpr (SIGMOID) {
#pragma unroll
        for (int i = 0; i < B; ++i) v[i] += 1.0;
        reciprocal(v);
    }
#pragma unroll
    for (int i = 0; i < B; ++i) v[i] = none[i] ? 0.0 : v[i];
}
template <bool SIGMOID>
__device__ __forceinline__ double term(float x, double top) {
    const float one[1] = {x};
    double v[1];
    terms<SIGMOID>(one, top, v);
    return v[0];
}
// Of a lane's experts, four at a time.
template <bool SIGMOID, int N>
__device__ __forceinline__ void terms_of(const float (&x)[N], double top, double (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const float four[4] = {x[i], x[i + 1], x[i + 2], x[i + 3]};
        double got[4];
        terms<SIGMOID>(four, top, got);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i + j] = got[j];
    }
}

struct Row {
    double top, inverse;  // of a softmax: the largest logit, and 1 / sum of the exponentials
};

template <bool SIGMOID>
__device__ __forceinline__ double score(float x, const Row& row) {
    return SIGMOID ? term<true>(x, 0.0) : term<false>(x, row.top) * row.inverse;
}

// Writes a token's choices, one a lane, each at its place.
template <int LANES>
__device__ __forceinline__ void write(const Geometry& g, std::int64_t* __restrict__ indices, void* __restrict__ scores, int token,
                                      int place, int expert, double weight, bool broken) {
    if (g.renormalize) {
        const double sum = join_sum<LANES>(place < g.top_k ? weight : 0.0);
        weight = sum > 0.0 ? weight / sum : 0.0;
    }
    if (place >= g.top_k || token >= g.tokens) return;
    const std::int64_t at = static_cast<std::int64_t>(token) * g.top_k + place;
    indices[at] = broken ? -1 : expert;
    write_score(scores, at, g.score_type, broken ? __builtin_nanf("") : static_cast<float>(weight * g.scale));
}

// Descending: odd-even merges of halves, quarters, ..
template <int N>
__device__ __forceinline__ void sort(std::uint32_t (&key)[N]) {
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int k = p; k > 0; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const std::uint32_t a = key[i + j], b = key[i + j + k];
                        key[i + j] = max(a, b);
                        key[i + j + k] = min(a, b);
                    }
}

// The largest keys of a token in order from lists that its lanes have sorted: every choice moves its owner's list up. Lane k
// gets the k-th key and its expert, which `expert` makes of the owner's place and the key; 0 is no key. Goes on after top_k
// keys while `more` of the key at hand and the top_k-th holds for some token of the wave; false if it still does after 16.
template <int LANES, int N, class Expert, class More>
__device__ __forceinline__ bool pick(int top_k, std::uint32_t (&key)[N], int place, std::uint32_t& own, int& chosen, Expert&& expert,
                                    More&& more) {
    sort(key);
    own = 0, chosen = 0;
    std::uint32_t last = 0;
    for (int k = 0; k <= 16; ++k) {
        const std::uint32_t best = join<LANES>(key[0], [](std::uint32_t a, std::uint32_t b) { return max(a, b); });
        if (k >= top_k && !__any(more(best, last))) return true;
        if (k < top_k) last = best;
        const unsigned long long owners = __ballot(key[0] == best) >> ((threadIdx.x & 63) - place);
        const int owner = __ffsll(owners) - 1;  // the first, of this token: some lane has the largest key
        if (place == k && k < 16) own = best, chosen = expert(owner, best);
#pragma unroll
        for (int i = 0; i < N; ++i) key[i] = place == owner ? (i + 1 < N ? key[i + 1] : 0) : key[i];
    }
    return false;
}

// 16-bit logits in their own order (no bias, one group): a logit's rank among all and its expert, from the last on, make one
// 32-bit key, so that the largest key is the choice and its ties are decided.
template <class T, int LANES, int N, bool VECTOR>
__global__ __launch_bounds__(kThreads) void route_logits(const T* __restrict__ logits, std::int64_t* __restrict__ indices,
                                                         void* __restrict__ scores, Geometry g) {
    constexpr std::uint32_t kInf = sizeof(T) == 2 && __is_same(T, __half) ? 0x7c00 : 0x7f80;
    const int place = threadIdx.x % LANES, first = place * N;
    const int token = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
    T x[N];
    load<T, N, VECTOR>(logits + static_cast<std::int64_t>(min(token, g.tokens - 1)) * g.experts, first, g.experts, x);
    std::uint32_t key[N], bad = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        key[i] = 0;
        if (first + i < g.experts) {
            std::uint32_t bits = __builtin_bit_cast(unsigned short, x[i]);
            bad |= (bits & 0x7fff) > kInf || (!g.sigmoid && bits == kInf);
            if (bits == 0x8000) bits = 0;
            key[i] = (bits & 0x8000 ? 0xffff - bits : bits + 0x8000) << 16 | (0xffff - first - i);
        }
    }
    bad = join<LANES>(bad, [](std::uint32_t a, std::uint32_t b) { return a | b; });
    std::uint32_t chosen;
    int expert;
    pick<LANES, N>(g.top_k, key, place, chosen, expert, [](int, std::uint32_t w) { return 0xffff - (w & 0xffff); },
                   [](std::uint32_t, std::uint32_t) { return false; });
    const std::uint32_t top = __shfl(chosen, (threadIdx.x & 63) - place, 64);  // of the token's first lane
    const auto value = [](std::uint32_t w) {
        w >>= 16;
        return to_f32(__builtin_bit_cast(T, static_cast<unsigned short>(w & 0x8000 ? w - 0x8000 : 0xffff - w)));
    };
    Row row = {value(top), 1.0};
    if (!g.sigmoid && !g.renormalize) {
        float logit[N];
        double v[N], sum = 0.0;
#pragma unroll
        for (int i = 0; i < N; ++i) logit[i] = first + i < g.experts ? to_f32(x[i]) : -__builtin_inff();
        terms_of<false>(logit, row.top, v);
#pragma unroll
        for (int i = 0; i < N; ++i) sum += v[i];
        row.inverse = 1.0 / join_sum<LANES>(sum);
    }
    const float logit = value(chosen);
    const double weight = place >= g.top_k || logit == -__builtin_inff() ? 0.0 : g.sigmoid ? score<true>(logit, row) : score<false>(logit, row);
    write<LANES>(g, indices, scores, token, place, expert, weight, bad);
}

// A score's key: its 32-bit number (infinities as the largest there is) in order as a whole number above 0, without the low
// bits that say which of its lane's N experts it is, the first the largest.
template <int N>
__device__ __forceinline__ std::uint32_t key_of(float c, int i) {
    const auto w = __builtin_bit_cast(std::uint32_t, fminf(fmaxf(c, -3.402823466e38f), 3.402823466e38f));
    return ((w & 0x80000000u ? ~w : w | 0x80000000u) & ~(N - 1u)) | (N - 1 - i);
}
// Whether the first of two keys, the larger, may stand for no larger score: the 32-bit rounding and the low bits hide less than
// 2^-18 of either, and of numbers below 2^-126 all. `slack`: 2^-120, or 2^-20 for keys of quick scores.
constexpr float kExactSlack = 0x1p-120f;
__device__ __forceinline__ bool near_keys(std::uint32_t a, std::uint32_t b, float slack) {
    const auto value = [](std::uint32_t k) { return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k); };
    const float most = value(a), difference = most - value(b);
    return b != 0 && !(difference > fmaf(fabsf(most), 0x1p-17f, slack));
}

// 1 / (1 + exp(-x)) to 2^-22: the product's rounding weighs |x| s (1 - s) 2^-24, the exponential's last bit s (1 - s) 2^-23, and
// the sum and its inverse s (2^-24 + 2^-23).
// With a bias of up to 4, whose sum is rounded by 4 x 2^-24 at most, it errs by less than 2^-21: two by less than 2^-20, and
// sums of two with their own rounding by less than 2^-19 each.
constexpr float kQuickBias = 4.0f, kQuickSlack = 0x1p-20f;
__device__ __forceinline__ float quick_sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504f));
}

// The two largest.
template <class V>
struct Best {
    V most, second;
    __device__ __forceinline__ void add(V v, V w) {  // v >= w
        second = max_of(max_of(second, w), min_of(most, v));
        most = max_of(most, v);
    }
    static __device__ __forceinline__ double max_of(double a, double b) { return fmax(a, b); }
    static __device__ __forceinline__ double min_of(double a, double b) { return fmin(a, b); }
    static __device__ __forceinline__ float max_of(float a, float b) { return fmaxf(a, b); }
    static __device__ __forceinline__ float min_of(float a, float b) { return fminf(a, b); }
};

// Takes the experts of groups that are not kept out of `key` (0: not there, or in no kept group). A lane ranks a group, from
// LDS of its own token: from what the lanes of a group have found in their own experts, or where groups end inside a lane's,
// from all scores. False in a lane whose group quick scores neither keep nor drop for sure.
template <class V, int N>
__device__ __forceinline__ bool keep_groups(const Geometry& g, const V (&c)[N], std::uint32_t (&key)[N], V* mine, V* rank_of, int place) {
    constexpr V none = -static_cast<V>(__builtin_inff());
    const int first = place * N, size = g.experts / g.groups;
    Best<V> best = {none, none};
    wave_fence();
    if (size % N == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) best.add(c[i], none);
        mine[2 * place] = best.most, mine[2 * place + 1] = best.second;
        wave_fence();
        best = {none, none};
        const int lanes = size / N;
        if (place < g.groups)
            for (int i = 0; i < lanes; ++i) best.add(mine[2 * (place * lanes + i)], mine[2 * (place * lanes + i) + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) mine[first + i] = c[i];
        wave_fence();
        if (place < g.groups) {
            int at = place % size;  // lanes start apart, so that they read different banks
            for (int i = 0; i < size; ++i) {
                best.add(mine[place * size + at], none);
                at = at + 1 == size ? 0 : at + 1;
            }
        }
    }
    V rank = g.pairs && best.second > none ? best.most + best.second : best.most;
    if constexpr (sizeof(V) == 8) rank = best.most > none ? fmax(rank, kLeast) : none;
    rank_of[place] = rank;
    wave_fence();
    int ahead = 0, may_be_ahead = 0;
#pragma unroll 4
    for (int i = 0; i < g.groups; ++i) {
        const V other = rank_of[i];
        if constexpr (sizeof(V) == 8) {
            ahead += other > rank || (other == rank && i < place);
        } else {
            ahead += other > rank + 4 * kQuickSlack;
            may_be_ahead += other >= rank - 4 * kQuickSlack && i != place;
        }
    }
    const bool keep = place < g.groups && ahead < g.kept;
    const unsigned long long kept = __ballot(keep) >> ((threadIdx.x & 63) - place);
    int group = first / size, in_group = first - group * size;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (!(kept >> min(group, 63) & 1)) key[i] = 0;
        if (++in_group == size) in_group = 0, ++group;
    }
    return sizeof(V) == 8 || !keep || may_be_ahead < g.kept;
}

// The token's choices in order, choice k in lane k, by scores and indices.
template <int LANES, int N>
__device__ __forceinline__ int pick_exactly(int top_k, const double (&c)[N], std::uint32_t open, int place) {
    const double none = -__builtin_inf();
    const int first = place * N;
    int chosen = 0;
    for (int k = 0; k < top_k; ++k) {
        double best = none;
#pragma unroll
        for (int i = 0; i < N; ++i) best = fmax(best, open >> i & 1 ? c[i] : none);
        best = join<LANES>(best, [](double a, double b) { return fmax(a, b); });
        std::uint32_t at = kMaxExperts;
#pragma unroll
        for (int i = N - 1; i >= 0; --i) at = (open >> i & 1) && c[i] == best ? first + i : at;
        at = join<LANES>(at, [](std::uint32_t a, std::uint32_t b) { return min(a, b); });
        if (place == k) chosen = static_cast<int>(at);
        if (static_cast<int>(at) / N == place) open &= ~(1u << (at % N));
    }
    return chosen;
}

// One of 16 neighbouring lanes' (score, expert) against the others': how many are ahead of it.
__device__ __forceinline__ int rank_of_16(double c, std::uint32_t expert) {
    int ahead = 0;
    const auto against = [&](double other, std::uint32_t other_expert) {
        ahead += other > c || (other == c && other_expert < expert);
    };
    against(moved<0x121>(c), moved<0x121>(expert));
    against(moved<0x122>(c), moved<0x122>(expert));
    against(moved<0x123>(c), moved<0x123>(expert));
    against(moved<0x124>(c), moved<0x124>(expert));
    against(moved<0x125>(c), moved<0x125>(expert));
    against(moved<0x126>(c), moved<0x126>(expert));
    against(moved<0x127>(c), moved<0x127>(expert));
    against(moved<0x128>(c), moved<0x128>(expert));
    against(moved<0x129>(c), moved<0x129>(expert));
    against(moved<0x12a>(c), moved<0x12a>(expert));
    against(moved<0x12b>(c), moved<0x12b>(expert));
    against(moved<0x12c>(c), moved<0x12c>(expert));
    against(moved<0x12d>(c), moved<0x12d>(expert));
    against(moved<0x12e>(c), moved<0x12e>(expert));
    against(moved<0x12f>(c), moved<0x12f>(expert));
    return ahead;
}

// Any logits, a bias, groups. Scores have 64 bits; the choice goes by 32-bit keys, past top_k as long as the next key is near
// the last, and where keys that follow each other are near, the scores of the up to 16 candidates, a lane each, decide. More
// candidates than that (many equal scores, or masked experts) are picked score by score. Keys and groups' ranks of sigmoid scores
// are first made of quick 32-bit ones; where those do not decide on the groups, the wave starts again with 64 bits (4099 tokens
// of 256 in 8 groups 9.7 -> 8.2 us, 16384 21.1 -> 17.6). Softmax scores take 64 bits at once (16384 tokens of 128 with a bias 9.7,
// of 256 16.9).
template <class T, int LANES, int N, bool SIGMOID, bool VECTOR>
__global__ __launch_bounds__(kThreads) void route_scores(const T* __restrict__ logits, const float* __restrict__ bias,
                                                         std::int64_t* __restrict__ indices, void* __restrict__ scores, Geometry g) {
    __shared__ double all[kThreads * N], ranks[kThreads];
    const int place = threadIdx.x % LANES, first = place * N, token = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
    const T* from = logits + static_cast<std::int64_t>(min(token, g.tokens - 1)) * g.experts;
    constexpr float kInf = __builtin_inff();
    T raw[N];
    load<T, N, VECTOR>(from, first, g.experts, raw);
    float x[N], b[N], top = -kInf;
    std::uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) b[i] = 0.0f;
    if (bias) load<float, N, VECTOR>(bias, first, g.experts, b);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        x[i] = first + i < g.experts ? to_f32(raw[i]) : -kInf;
        bad |= x[i] != x[i] || (!SIGMOID && x[i] == kInf) || (b[i] != b[i] && x[i] != -kInf);
        top = fmaxf(top, x[i]);
    }
    bad = join<LANES>(bad, [](std::uint32_t a, std::uint32_t b) { return a | b; });
    // Without a bias and sums of scores the logits' own order will do.
    const bool direct = !bias && (g.groups == 1 || !g.pairs);
    Row row = {0.0, 1.0};
    double c[N];
    if constexpr (!SIGMOID) {
        row.top = join<LANES>(top, [](float a, float b) { return fmaxf(a, b); });
        if (!direct || !g.renormalize) {
            double sum = 0.0;
            terms_of<false>(x, row.top, c);
#pragma unroll
            for (int i = 0; i < N; ++i) sum += c[i];
            sum = join_sum<LANES>(sum);
            row.inverse = sum > 0.0 ? 1.0 / sum : 0.0;
        }
    }
    const auto whole = [&](float logit, double s, float offset) {  // a score with its bias
        const double v = direct ? static_cast<double>(logit) : s + static_cast<double>(offset);
        return logit == -kInf ? -__builtin_inf() : fmax(v + 0.0, kLeast);  // one zero, and no NaN
    };
    const auto exactly = [&] {
        if constexpr (SIGMOID) {
            if (!direct) terms_of<true>(x, 0.0, c);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) c[i] = whole(x[i], direct ? 0.0 : c[i] * row.inverse, b[i]);
    };
    std::uint32_t key[N];
    const auto keys_of = [&](auto& v) {
#pragma unroll
        for (int i = 0; i < N; ++i) key[i] = first + i < g.experts ? key_of<N>(static_cast<float>(v[i]), i) : 0;
        using V = std::remove_reference_t<decltype(v[0])>;
        return g.groups == 1 || keep_groups<V, N>(g, v, key, reinterpret_cast<V*>(all + (threadIdx.x - place) * N),
                                                  reinterpret_cast<V*>(ranks + (threadIdx.x - place)), place);
    };
    bool quick = false;
    if constexpr (SIGMOID) {
        if (!direct) {
            float f[N];
            bool far = false;
#pragma unroll
            for (int i = 0; i < N; ++i) far = far || fabsf(b[i]) > kQuickBias;
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = x[i] == -kInf ? -kInf : fmaxf(quick_sigmoid(x[i]) + b[i], -kInf) + 0.0f;
            quick = !__any(far) && __all(keys_of(f) || bad);
        }
    }
    if (!quick) {
        exactly();
        keys_of(c);
    }
    const float slack = quick ? kQuickSlack : kExactSlack;
    std::uint32_t open = 0, own;
#pragma unroll
    for (int i = 0; i < N; ++i) open |= key[i] ? 1u << i : 0;
    int chosen, rank = place;
    const bool whole_list = pick<LANES, N>(g.top_k, key, place, own, chosen,
                                     [](int owner, std::uint32_t w) { return owner * N + N - 1 - static_cast<int>(w & (N - 1)); },
                                     [&](std::uint32_t w, std::uint32_t last) { return near_keys(last, w, slack); });
    const std::uint32_t after = moved<0x101>(own);  // of the next lane; 0 in the last of 16
    bool sure = !__any(place < 15 && own && near_keys(own, after, slack));
    if (!whole_list) {
        if (quick) exactly();
        chosen = pick_exactly<LANES, N>(g.top_k, c, open, place);
        own = 1, sure = true;
    }
    double weight = 0.0, exact = -__builtin_inf();
    const bool candidate = place < (sure ? g.top_k : 16) && own && !bad;
    if (candidate) {
        const float logit = to_f32(from[chosen]);
        if (logit != -kInf) weight = score<SIGMOID>(logit, row);
        if (!sure) exact = whole(logit, weight, bias ? bias[chosen] : 0.0f);
    }
    if (!sure) {
        const int ahead = rank_of_16(exact, candidate ? chosen : kMaxExperts);
        rank = bad ? place : candidate ? ahead : kMaxTopK;
    }
    write<LANES>(g, indices, scores, token, rank, chosen, weight, bad);
}

template <class T, int LANES, int N>
void launch_some(const T* logits, const float* bias, std::int64_t* indices, void* scores, const Geometry& g, hipStream_t stream) {
    constexpr int tokens = kThreads / LANES;
    const auto grid = static_cast<unsigned>((static_cast<std::int64_t>(g.tokens) + tokens - 1) / tokens);
    const bool vector = g.experts % N == 0 && aligned(logits, 16) && aligned(bias, 16);
    if constexpr (sizeof(T) == 2) {
        if (!bias && g.groups == 1) {
            if (vector) route_logits<T, LANES, N, true><<<grid, kThreads, 0, stream>>>(logits, indices, scores, g);
            else route_logits<T, LANES, N, false><<<grid, kThreads, 0, stream>>>(logits, indices, scores, g);
            return;
        }
    }
    const auto run = [&](auto sigmoid) {
        constexpr bool S = decltype(sigmoid)::value;
        if (vector) route_scores<T, LANES, N, S, true><<<grid, kThreads, 0, stream>>>(logits, bias, indices, scores, g);
        else route_scores<T, LANES, N, S, false><<<grid, kThreads, 0, stream>>>(logits, bias, indices, scores, g);
    };
    if (g.sigmoid) run(std::true_type{});
    else run(std::false_type{});
}

// A launch takes 2^24 tokens (its threads are counted in 32 bits).
template <class T, int LANES, int N>
void launch_lanes(const T* logits, const float* bias, std::int64_t* indices, void* scores, const Geometry& g, hipStream_t stream) {
    constexpr int kTokens = 1 << 24;
    const std::int64_t size = g.score_type == kF32 ? 4 : 2;
    for (std::int64_t first = 0; first < g.tokens; first += kTokens) {
        Geometry part = g;
        part.tokens = static_cast<int>(std::min<std::int64_t>(g.tokens - first, kTokens));
        launch_some<T, LANES, N>(logits + first * g.experts, bias, indices + first * g.top_k,
                                 static_cast<char*>(scores) + first * g.top_k * size, part, stream);
        check(hipGetLastError());
    }
}

// A token takes 16, 32 or 64 lanes of eight experts (four where they are few, 16 past 512), as many as groups and choices at
// least. (Us in captured chains, 4 / 8 / 16 experts a lane, sigmoid scores of 256 with a bias: 512 tokens 4.8 / 5.6 / 7.3, 4099 7.1
// / 6.5 / 7.7, 16384 16.7 / 14.2 / 14.4; in 8 groups 6.1 / 6.3 / 8.2, 8.8 / 8.2 / 9.8 and 21.8 / 17.7 / 17.9; 16-bit logits alone
// 3.8 / 3.9 / 4.9, 5.7 / 4.9 / 5.4 and 12.7 / 9.1 / 8.3.)
template <class T>
void launch(const void* logits, const float* bias, std::int64_t* indices, void* scores, const Geometry& g, hipStream_t stream) {
    const auto* x = static_cast<const T*>(logits);
    if (g.groups <= 16 && g.experts <= 64) launch_lanes<T, 16, 4>(x, bias, indices, scores, g, stream);
    else if (g.groups <= 16 && g.experts <= 128) launch_lanes<T, 16, 8>(x, bias, indices, scores, g, stream);
    else if (g.groups <= 32 && g.experts <= 256) launch_lanes<T, 32, 8>(x, bias, indices, scores, g, stream);
    else if (g.experts <= 512) launch_lanes<T, 64, 8>(x, bias, indices, scores, g, stream);
    else launch_lanes<T, 64, 16>(x, bias, indices, scores, g, stream);
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
        const std::uint64_t logit_bytes = (dtype == vt::kF32 ? 4ull : 2ull) * tokens * experts, bias_bytes = 4ull * experts;
        const std::uint64_t index_bytes = 8ull * tokens * top_k, score_bytes = (score_dtype == vt::kF32 ? 4ull : 2ull) * tokens * top_k;
        vt::require(!vt::meet(indices, index_bytes, logits, logit_bytes) && !vt::meet(indices, index_bytes, bias, bias_bytes) &&
                        !vt::meet(scores, score_bytes, logits, logit_bytes) && !vt::meet(scores, score_bytes, bias, bias_bytes) &&
                        !vt::meet(scores, score_bytes, indices, index_bytes),
                    "routing outputs must not overlap other operands");
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

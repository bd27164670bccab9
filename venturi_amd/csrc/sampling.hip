// Sampling one token per row of 16-bit logits from given random numbers.
//
// A 16-bit logit has 65536 values, so a row's order is its histogram: classes of equal logits from the largest down,
// ties by index within a class. The workgroup of a row counts the classes in LDS by their bits (whole numbers: the order
// of the atomics leaves no trace), sums count * exp((v - max) / T) in 64 bits, and finds the borders of top-k, top-p and
// min-p and the place of u in the prefix sums. 64 bits, because a border of a large vocabulary is a token of 1e-6 of the
// mass, and one token more or less there moves every later draw. The token is then the class's rank-th occurrence.
//
// Weights. A lane holds 16 neighbouring classes, which are evenly spaced: their weights are the first one's times powers
// of exp(-spacing / T), two exponentials for 16 classes (at most 16 roundings of 2^-53 apart from the exact ones). A turn
// is a wave's 1024 classes; the 64 turns' sums are one scan, and only turns that a border falls into are opened again.
//
// Counters are 16 bits wide (128 KB of the CU's 160 KB): a row of more than 57344 logits is counted in segments, and
// between two segments every class that has reached 16384 moves to a list (at most one entry per 16384 logits).
//
// The token's place is found in a second pass over the row, of the chunks alone (512 logits) whose largest logit is not below
// the class: noting those costs the count 0.8 us, passing the others by saves the search 5 (256 rows of 151936 logits: 42.2
// -> 40.3 us).
//
// A row takes about 40 us on its CU whatever their number up to 256 (151936 bf16 logits; 256 rows read 78 MB at 1.9 TB/s):
// 21 to clear and count, which the LDS atomics and the vector unit share, 8 to choose, 3 to find the occurrence. Counters in
// memory shared by several workgroups of a row gain nothing (one row 46 us as here, 32 rows 150 us): the atomics and the 256 KB
// that one of them reads at the end cost what the shorter count saves.
//
// Kept distributions are two or three launches: distribution_scan() looks at few long rows, distribution_cut() finds the last token
// that a row keeps and the kept mass, and distribution() writes every token's probability. A row without limits needs no histogram,
// nor does one whose top_k is at most 256 and the number of its chunks of 128 logits (any other top_k, that of the whole row too,
// and top_p or min_p alone do). The write is bound by memory (96 rows of 151936 bf16 logits: 15 us for 88 MB, 5.8 TB/s), the cut by
// its row's one CU (the same rows, all in all: 39 us without limits, 29 with top_k 50, 41 with min_p alone, 52 with top_p alone:
// 20 of those the count, 2 the largest class, 4 the turns' masses, 4 the choice, 7 the search).
#include "common.hpp"

#include <climits>

namespace vt {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kTurns = 64;                 // of 1024 classes, 16 a lane
constexpr int kMaxVocab = 1 << 20;
constexpr int kMaxDistributionRows = 65535;  // a launch's second dimension
constexpr std::uint32_t kHeavy = 16384;
constexpr int kHeavyEntries = 2 * kMaxVocab / kHeavy;
constexpr int kNone = -1;                  // no class
constexpr int kChunks = kMaxVocab / 512;   // of 64 vectors, a wave's turn of a row
// Vectors of 8 logits that a thread counts before the first sweep for heavy classes (57344 logits, beside the up to 14 of the
// row's ragged ends), and between two sweeps (49152, on counters below 16384: 65535 at most).
constexpr int kFirst = 7, kNext = 6;
// Chunks of 16 vectors that a row's largest logits are looked for in, and logits that are then put in order.
constexpr int kListed = 4 * 64, kCandidates = 256;

template <class T> struct Bits;
template <> struct Bits<__half> {
    static constexpr std::uint32_t kInf = 0x7c00;
    static constexpr int kMantissa = 10;
};
template <> struct Bits<__hip_bfloat16> {
    static constexpr std::uint32_t kInf = 0x7f80;
    static constexpr int kMantissa = 7;
};

// Classes by place: 0 .. 32767 are the positive numbers from bits 0x7fff down to 0, the rest the negative ones from 0x8000
// up. -0 belongs to the class of 0; the places of NaN and -inf hold no class.
__device__ __forceinline__ std::uint32_t place_bits(int place) { return place < 32768 ? 32767 - place : place; }

template <class T>
__device__ __forceinline__ bool is_class(int place) {
    const std::uint32_t bits = place_bits(place);
    return (bits & 0x7fff) <= Bits<T>::kInf && bits != (0x8000 | Bits<T>::kInf) && bits != 0x8000;
}

template <class T>
__device__ __forceinline__ double class_value(int place) {
    return static_cast<double>(to_f32(__builtin_bit_cast(T, static_cast<unsigned short>(place_bits(place)))));
}

// The difference of neighbouring classes at a place.
template <class T>
__device__ __forceinline__ double class_step(int place) {
    const std::uint32_t low = place_bits(place) & 0x7fff & ~((1u << Bits<T>::kMantissa) - 1);  // the binade's first
    const auto value = [](std::uint32_t bits) {
        return static_cast<double>(to_f32(__builtin_bit_cast(T, static_cast<unsigned short>(bits))));
    };
    return value(low + 1) - value(low);
}

// A row as `head` elements before its first 16-byte boundary, `vectors` whole vectors of 8, and `tail` elements.
struct Row {
    const unsigned short* start;
    int head, vectors, tail;

    __device__ __forceinline__ Row(const void* logits, int index, int vocab) {
        const std::int64_t first = static_cast<std::int64_t>(index) * vocab;
        start = static_cast<const unsigned short*>(logits) + first;  // the tensor is 16-byte aligned
        head = min(static_cast<int>(-first & 7), vocab);
        vectors = (vocab - head) >> 3;
        tail = vocab - head - 8 * vectors;
    }
    __device__ __forceinline__ const uint4* whole() const { return reinterpret_cast<const uint4*>(start + head); }
    // Element i of the head and tail together, and its index in the row.
    __device__ __forceinline__ int edge(int i) const { return i < head ? i : 8 * vectors + i; }
};

__device__ __forceinline__ std::uint32_t element(const uint4& w, int j) {
    const std::uint32_t u = j < 2 ? w.x : j < 4 ? w.y : j < 6 ? w.z : w.w;
    return (u >> (16 * (j & 1))) & 0xffff;
}

template <int CONTROL, int ROWS>
__device__ __forceinline__ int moved(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CONTROL, ROWS, 0xf, true);
}
template <int CONTROL, int ROWS>
__device__ __forceinline__ double moved(double v) {
    const auto w = __builtin_bit_cast(std::uint64_t, v);
    const std::uint32_t lo = moved<CONTROL, ROWS>(static_cast<int>(w)), hi = moved<CONTROL, ROWS>(static_cast<int>(w >> 32));
    return __builtin_bit_cast(double, static_cast<std::uint64_t>(hi) << 32 | lo);
}
// Sums over lanes 0..lane, by lane moves within rows of 16 and then across rows.
template <class V>
__device__ __forceinline__ V wave_scan(V v) {
    v += moved<0x111, 0xf>(v);
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);
    v += moved<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ int lane_int(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ double lane_double(double v, int lane) {
    const auto w = __builtin_bit_cast(std::uint64_t, v);
    const std::uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(w), lane);
    const std::uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(w >> 32), lane);
    return __builtin_bit_cast(double, static_cast<std::uint64_t>(hi) << 32 | lo);
}
template <class V>
__device__ __forceinline__ V wave_sum(V v) {
    v = wave_scan(v);
    if constexpr (sizeof(V) == 8) return lane_double(v, 63);
    else return lane_int(v, 63);
}

struct Settings {
    float temperature, top_p, min_p, uniform;
    int top_k;
};

struct Shared {
    std::uint32_t histogram[32768];  // of bits 2 i (low half) and 2 i + 1 (high half)
    double turn_mass[kTurns];
    int turn_count[kTurns];
    std::uint32_t heavy_bits[kHeavyEntries], heavy_count[kHeavyEntries];
    short largest[4 * kChunks];      // the largest signed_bits of 16 vectors
    double probability;
    int heavy, top, above_min, place, rank, count;
    bool whole;                      // the chosen class has no occurrence after the chosen one
    // Of distribution rows: chunks of 16 vectors by the upper and then the lower byte of their largest logits, the chunks to
    // look through, and their candidates by order and index.
    std::uint32_t upper[256], bins[256];
    int bin, above;
    unsigned short listed[kListed];
    std::uint64_t candidates[kCandidates], ordered[kCandidates];
    double wave_mass[kWaves];
    float wave_top[kWaves];
};

static_assert(sizeof(Shared) <= 160 * 1024, "a CU's LDS");

// A row's chosen class (kNone: nothing to take), and which of its occurrences.
struct Choice {
    int place, rank;
};

// A barrier of the workgroup's LDS accesses alone: __syncthreads() would also wait for the loads in flight.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ void clear(Shared& s) {
    for (int i = threadIdx.x; i < 32768 / 4; i += kThreads) reinterpret_cast<uint4*>(s.histogram)[i] = make_uint4(0, 0, 0, 0);
    if (threadIdx.x == 0) s.heavy = s.above_min = 0, s.top = 65536;
    lds_barrier();
}

__device__ __forceinline__ void count_element(Shared& s, std::uint32_t bits) {
    atomicAdd(&s.histogram[bits >> 1], 1u << (16 * (bits & 1)));
}

__device__ __forceinline__ void count_vector(Shared& s, const uint4& w) {
    const std::uint32_t u[4] = {w.x, w.y, w.z, w.w};
    auto* bytes = reinterpret_cast<unsigned char*>(s.histogram);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        // A shift takes the low five bits of its amount.
        atomicAdd(reinterpret_cast<std::uint32_t*>(bytes + ((u[j] & 0xfffe) << 1)), 1u << ((u[j] << 4) & 31));
        atomicAdd(reinterpret_cast<std::uint32_t*>(bytes + ((u[j] >> 15) & 0x1fffc)), 1u << ((u[j] >> 12) & 16));
    }
}

// Logits in order as whole numbers: the magnitude's bits with the sign (both zeros are 0).
__device__ __forceinline__ int signed_bits(std::uint32_t bits) {
    const int magnitude = static_cast<int>(bits & 0x7fff);
    return bits & 0x8000 ? -magnitude : magnitude;
}

template <int CONTROL>
__device__ __forceinline__ int larger(int v) {
    return max(v, __builtin_amdgcn_update_dpp(INT_MIN, v, CONTROL, 0xf, 0xf, false));
}

// The largest signed_bits (NaN by its bits) in the vectors of 16 lanes, in the last of them. Where a number has no sign it is
// the largest signed half (and the smallest half less 0x8000 saturates to 0), else the negative of the smallest magnitude.
__device__ __forceinline__ short largest_of_16(const uint4& w) {
    typedef short short2v __attribute__((ext_vector_type(2)));
    typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));
    const std::uint32_t u[4] = {w.x, w.y, w.z, w.w};
    short2v high = __builtin_bit_cast(short2v, u[0]);
    ushort2v low = __builtin_bit_cast(ushort2v, u[0]);
#pragma unroll
    for (int j = 1; j < 4; ++j) {
        high = __builtin_elementwise_max(high, __builtin_bit_cast(short2v, u[j]));
        low = __builtin_elementwise_min(low, __builtin_bit_cast(ushort2v, u[j]));
    }
    const short2v none = {0, 0};
    const ushort2v sign = {0x8000, 0x8000};
    high = __builtin_elementwise_max(high, none) - __builtin_bit_cast(short2v, __builtin_elementwise_sub_sat(low, sign));
    high = __builtin_elementwise_max(high, __builtin_shufflevector(high, high, 1, 0));
    int v = __builtin_bit_cast(int, high);  // ordered by its upper half
    v = larger<0x111>(v);
    v = larger<0x112>(v);
    v = larger<0x114>(v);
    v = larger<0x118>(v);
    return static_cast<short>(v >> 16);
}

// Moves the classes that have reached kHeavy to the list.
__device__ __forceinline__ void sweep(Shared& s) {
    lds_barrier();
    for (int i = threadIdx.x; i < 32768; i += kThreads) {
        std::uint32_t word = s.histogram[i];
        if (!(word & 0xc000c000u)) continue;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const std::uint32_t n = (word >> (16 * half)) & 0xffff;
            if (n >= kHeavy) {
                const int e = atomicAdd(&s.heavy, 1);
                s.heavy_bits[e] = 2 * i + half;
                s.heavy_count[e] = n;
                word -= n << (16 * half);
            }
        }
        s.histogram[i] = word;
    }
    lds_barrier();
}

// 2^x for x <= 0, NaN as 0: the Taylor series of e^r for |r| <= ln 2 / 2, whose 13th power is below 2^-53, times 2^n.
__device__ __forceinline__ double falling_power(double x) {
    const double n = rint(x);
    const double r = (x - n) * 0.693147180559945309417;
    double p = 1.0 / 6227020800.0;
    p = fma(p, r, 1.0 / 479001600.0);
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return x > -1000.0 ? ldexp(p, static_cast<int>(n)) : 0.0;
}

// A lane's 16 classes of a turn: places 1024 turn + 16 lane + i.
template <class T>
struct Lane {
    int n[16];       // occurrences; 0 where there is no class
    int first;       // weights start at class `first` (classes above the row's largest do not occur)
    double start, ratio;

    static __device__ __forceinline__ const uint4* words(const Shared& s, int place) {
        return reinterpret_cast<const uint4*>(s.histogram + (place >= 32768 ? place : 32767 - 15 - place) / 2);
    }

    // Whether any of the turn's classes (or of the places without one) occurs in the counters.
    static __device__ __forceinline__ bool occurs(const Shared& s, int heavy, int turn) {
        const auto* at = words(s, 1024 * turn + 16 * static_cast<int>(threadIdx.x & 63));
        const uint4 a = at[0], b = at[1];
        return heavy > 0 || turn == kTurns / 2 - 1 || ((a.x | a.y | a.z | a.w) | (b.x | b.y | b.z | b.w)) != 0;
    }

    __device__ __forceinline__ bool count(const Shared& s, int heavy, int turn) {
        const int place = 1024 * turn + 16 * static_cast<int>(threadIdx.x & 63);
        const bool negative = turn >= kTurns / 2;
        const auto* at = words(s, place);
        const uint4 a = at[0], b = at[1];
        const std::uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            n[2 * i] = negative ? u[i] & 0xffff : u[7 - i] >> 16;
            n[2 * i + 1] = negative ? u[i] >> 16 : u[7 - i] & 0xffff;
        }
        if (turn == kTurns / 2 - 1 && place == 32767 - 15) n[15] += s.histogram[16384] & 0xffff;  // -0
        for (int e = 0; e < heavy; ++e) {
            const std::uint32_t bits = s.heavy_bits[e] == 0x8000 ? 0 : s.heavy_bits[e];
            const int at = (bits & 0x8000 ? static_cast<int>(bits) : 32767 - static_cast<int>(bits)) - place;
#pragma unroll
            for (int i = 0; i < 16; ++i) n[i] += at == i ? s.heavy_count[e] : 0;
        }
        // Places without a class: NaN and -inf at both halves' ends, and -0.
        if (turn == 0 || turn == kTurns / 2 || turn == kTurns - 1) {
#pragma unroll
            for (int i = 0; i < 16; ++i) n[i] = is_class<T>(place + i) ? n[i] : 0;
        }
        bool some = false;
#pragma unroll
        for (int i = 0; i < 16; ++i) some = some || n[i];
        return some;
    }

    // Every exponent is at most 0: nothing overflows, whatever the temperature.
    __device__ __forceinline__ void weigh(int turn, int top, double max_value, double heat) {
        const int place = 1024 * turn + 16 * static_cast<int>(threadIdx.x & 63);
        first = top > place ? top - place : 0;  // 16 and more: the lane's classes all lie above
        start = falling_power((class_value<T>(first ? top : place) - max_value) * heat);
        if (first || place == top) start = 1.0;  // also where the difference is of two infinities
        ratio = falling_power(-class_step<T>(place) * heat);
    }

    // Visits the lane's classes in order: (index, occurrences, weight).
    template <class Visit>
    __device__ __forceinline__ void each(Visit&& visit) const {
        double w = start;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            visit(i, n[i], n[i] ? w : 0.0);
            if (i >= first) w *= ratio;
        }
    }
};

// log2 e / T, from 4e-39 to 2e45; of a greedy row that of T = 1.
__device__ __forceinline__ double heat_of(float temperature) {
    return 1.44269504088896340736 / (temperature > 0.0f ? static_cast<double>(fminf(temperature, 3.402823466e38f)) : 1.0);
}

// Chooses from the workgroup's complete histogram: the token at the uniform's place, or with LAST the last kept one. The
// probability that it leaves is the token's, or with LAST the kept mass in units of the largest weight.
template <class T, bool LAST>
__device__ __forceinline__ Choice choose(Shared& s, const Settings& set) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, heavy = s.heavy;
    for (int turn = wave; turn < kTurns; turn += kWaves) {
        if (!__any(Lane<T>::occurs(s, heavy, turn))) continue;
        Lane<T> l;
        const unsigned long long occurs = __ballot(l.count(s, heavy, turn));
        if (!occurs) continue;
        if (lane == __ffsll(occurs) - 1) {
            int at = 16;
#pragma unroll
            for (int i = 15; i >= 0; --i) at = l.n[i] ? i : at;
            atomicMin(&s.top, 1024 * turn + 16 * lane + at);
        }
        break;  // this wave's other turns lie below
    }
    __syncthreads();
    const int top = s.top;
    if (top >= 65536) {
        if (t == 0) s.probability = 0.0;
        __syncthreads();
        return {kNone, 0};
    }
    const bool greedy = !(set.temperature > 0.0f);
    const double max_value = class_value<T>(top), least = set.min_p;
    const double heat = heat_of(set.temperature);
    const bool all_above = least <= 0.0;
    int above_min = 0;
    for (int turn = wave; turn < kTurns && !greedy; turn += kWaves) {
        Lane<T> l;
        double mass = 0.0;
        int count = 0;
        if (__any(Lane<T>::occurs(s, heavy, turn)) && __any(l.count(s, heavy, turn))) {
            l.weigh(turn, top, max_value, heat);
            l.each([&](int, int n, double w) {
                mass += n * w;
                count += n;
            });
            if (!all_above) l.each([&](int, int n, double w) { above_min += w >= least ? n : 0; });
            mass = wave_sum(mass);
            count = wave_sum(count);
        }
        if (lane == 0) s.turn_mass[turn] = mass, s.turn_count[turn] = count;
    }
    if (!all_above) {
        above_min = wave_sum(above_min);
        if (lane == 0 && above_min) atomicAdd(&s.above_min, above_min);
    }
    __syncthreads();
    if (wave == 0) {
        Lane<T> l;
        if (greedy) {
            if (lane == 0) s.place = top, s.rank = 0, s.probability = 1.0, s.whole = false;
        } else {
            // What comes before turn `lane` in the whole order.
            const double turn_mass = s.turn_mass[lane], mass_scan = wave_scan(turn_mass), mass_all = lane_double(mass_scan, 63);
            const int turn_count = s.turn_count[lane], count_scan = wave_scan(turn_count), all = lane_int(count_scan, 63);
            const int count_before = count_scan - turn_count;
            const double mass_up = __shfl_up(mass_scan, 1, 64), mass_before = lane ? mass_up : 0.0;
            // The last turn of which a test (true up to some turn) holds; the lane's classes there and what precedes them.
            int turn = -1, before;
            double mass_at;
            const auto open = [&](bool test) {
                const int wanted = max(__popcll(__ballot(test)) - 1, 0);
                if (wanted == turn) return;
                turn = wanted;
                l.count(s, heavy, turn);
                l.weigh(turn, top, max_value, heat);
                int n = 0;
                double mass = 0.0;
                l.each([&](int, int c, double w) { n += c, mass += c * w; });
                before = lane_int(count_before, turn) + wave_scan(n) - n;
                const double up = __shfl_up(wave_scan(mass), 1, 64);
                mass_at = lane_double(mass_before, turn) + (lane ? up : 0.0);
            };
            const auto prefix_mass = [&](int length) {  // of the first `length` tokens
                if (length >= all) return mass_all;
                open(count_before <= length);
                double mass = 0.0;
                int left = length - before;
                l.each([&](int, int n, double w) {
                    mass += min(max(left, 0), n) * w;
                    left -= n;
                });
                return lane_double(mass_before, turn) + wave_sum(mass);
            };
            // Tokens in order up to a border of mass: those that start below it, or those that end at or below it.
            const auto tokens_below = [&](double border, bool ends) {
                open(ends ? mass_before <= border : mass_before < border);
                int in = 0, part = 0;
                double at = mass_at, part_at = 0.0, part_w = 1.0;
                l.each([&](int, int n, double w) {
                    const double last = ends ? at + n * w : at + (n - 1) * w;
                    const bool whole = ends ? last <= border : last < border, some = ends ? at <= border : at < border;
                    if (n && whole) in += n;
                    if (n && !whole && some) part = n, part_at = at, part_w = w;
                    at += n * w;
                });
                if (part) {
                    const double quotient = (border - part_at) / part_w;
                    int count = static_cast<int>(fmin(ends ? floor(quotient) : ceil(quotient), static_cast<double>(part)));
                    if (ends) {
                        if (count > 0 && part_at + count * part_w > border) --count;
                        if (count < part && part_at + (count + 1) * part_w <= border) ++count;
                    } else {
                        if (count > 0 && part_at + (count - 1) * part_w >= border) --count;
                        if (count < part && part_at + count * part_w < border) ++count;
                    }
                    in += count;
                }
                return lane_int(count_before, turn) + wave_sum(in);
            };
            const int limit = set.top_k > 0 ? min(set.top_k, all) : all;
            int length = all_above ? limit : min(limit, s.above_min);
            const double share = set.top_p;
            if (!(share >= 1.0)) {
                const double border = share * (prefix_mass(limit));
                length = min(length, border > 0.0 ? tokens_below(border, false) : 0);
            }
            length = max(length, 1);
            const double kept = prefix_mass(length);
            // A uniform of 1 or more stays below the end of the mass: the last token that adds to it.
            const double target = fmin(static_cast<double>(set.uniform) * kept, kept * (1.0 - 0x1p-52));
            int place;
            if constexpr (LAST) {
                place = length - 1;
            } else {
                place = target >= 0.0 && set.uniform >= 0.0f ? tokens_below(target, true) : 0;
                place = max(min(place, length - 1), 0);
            }
            open(count_before <= place);
            int at = before;
            l.each([&](int i, int n, double w) {
                if (place >= at && place < at + n) {
                    s.place = 1024 * turn + 16 * lane + i;
                    s.rank = place - at;
                    s.probability = LAST ? kept : w / kept;
                    s.whole = place + 1 == at + n;
                }
                at += n;
            });
        }
    }
    __syncthreads();
    return {s.place, s.rank};
}

// A class's bits twice in a word, and the bits to compare (the class of 0 takes either sign).
struct Pattern {
    std::uint32_t bits, mask;
    __device__ __forceinline__ explicit Pattern(int place)
        : bits(place_bits(place) * 0x10001u), mask(bits ? 0xffffffffu : 0x7fff7fffu) {}
};

// Elements of a vector that match: 8 less the halves that differ.
__device__ __forceinline__ int occurrences(const uint4& w, const Pattern& p) {
    typedef unsigned short short2v __attribute__((ext_vector_type(2)));
    const short2v one = {1, 1};
    short2v differ = {0, 0};
    const std::uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) differ += __builtin_elementwise_min(__builtin_bit_cast(short2v, (u[i] ^ p.bits) & p.mask), one);
    return 8 - differ.x - differ.y;
}

// Which of the chunk counts (`count` of them, in order) holds occurrence `rank`; `before` becomes what precedes it there.
// A whole wave; -1 if there are fewer.
__device__ __forceinline__ int find_chunk(const int* counts, int chunks, int rank, int& before) {
    const int lane = threadIdx.x & 63;
    before = 0;
    for (int base = 0; base < chunks; base += 64) {
        const int n = base + lane < chunks ? counts[base + lane] : 0;
        const int end = before + wave_scan(n);
        const unsigned long long hit = __ballot(end > rank);
        if (hit) {
            const int at = __ffsll(hit) - 1;
            before = lane_int(end - n, at);
            return base + at;
        }
        before = lane_int(end, 63);
    }
    return -1;
}

// The element of a vector at which occurrence `rank` of the wave's 64 vectors lies, if it is the lane's; else -1.
__device__ __forceinline__ int find_element(const uint4& w, const Pattern& p, int before, int rank) {
    int at = -1;
    const int n = occurrences(w, p);
    int next = before + wave_scan(n) - n;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (((element(w, j) ^ p.bits) & p.mask & 0xffff) == 0 && next++ == rank) at = j;
    return at;
}

// What a row keeps: classes above `place`, and of its class the tokens up to `index`.
struct Cut {
    double max, heat;    // a token's weight is 2^((logit - max) heat)
    float inverse, rest; // of the kept mass, in two parts
    int place, index;    // place kNone: the row keeps nothing

    __device__ __forceinline__ void set(double top, double heat_, double mass, int place_) {
        const double whole = 1.0 / mass;
        max = top, heat = heat_, place = place_;
        inverse = static_cast<float>(whole);
        rest = static_cast<float>(whole - static_cast<double>(inverse));
    }
};

// A part of a row: its largest logit, and where the row's whole mass counts, the mass in units of that one's weight.
struct Part {
    double mass;
    float top;
    int unused;
};

struct Operands {
    const void* logits;
    const float* uniforms;
    const float* temperature;
    const std::int32_t* top_k;
    const float* top_p;
    const float* min_p;
    std::int64_t* tokens;
    float* probabilities;
    // Of the distribution, in place of tokens and uniforms: a row's cut, its parts, and its chunks' largest logits.
    Cut* cuts;
    Part* parts;
    short* largest;
    int rows, vocab, part_count, chunk_count;

    __device__ __forceinline__ Settings settings(int row) const {
        return {temperature ? temperature[row] : 1.0f, top_p ? top_p[row] : 1.0f, min_p ? min_p[row] : 0.0f, uniforms ? uniforms[row] : 0.0f,
                top_k ? top_k[row] : 0};
    }
};

// Visits the vectors t, t + kThreads, .. below end. The loads run a batch ahead of the visits, unconditional (past the end they
// repeat the last vector): a load under a condition is waited for before the next one is issued. `before` runs once, after the
// first loads are issued; `between`, for the whole workgroup, after every kFirst and then every kNext vectors of a thread.
template <class Before, class Visit, class Between>
__device__ __forceinline__ void each_vector(const uint4* __restrict__ whole, int end, Before&& before, Visit&& visit, Between&& between) {
    if (end <= 0) {
        before();
        return;
    }
    const int at = threadIdx.x;
    const auto load = [&](int i) { return whole[min(at + i * kThreads, end - 1)]; };
    uint4 now[kFirst], next[kNext];
#pragma unroll
    for (int j = 0; j < kFirst; ++j) now[j] = load(j);
    before();
    for (int i = 0, count = kFirst; i * kThreads < end; i += count, count = kNext) {
#pragma unroll
        for (int j = 0; j < kNext; ++j) next[j] = load(i + count + j);
#pragma unroll
        for (int j = 0; j < kFirst; ++j)
            if (j < count && (i + j) * kThreads < end) visit(now[j], i + j, at + (i + j) * kThreads < end);
        if ((i + count) * kThreads < end) between();
#pragma unroll
        for (int j = 0; j < kNext; ++j) now[j] = next[j];
    }
}

// A lane's element of the row's ragged ends (lanes below head + tail of the first wave).
struct Edge {
    std::uint32_t bits;
    bool live;
    __device__ __forceinline__ explicit Edge(const Row& row)
        : live(static_cast<int>(threadIdx.x) < row.head + row.tail) {
        bits = live ? row.start[row.edge(threadIdx.x)] : 0;
    }
    __device__ __forceinline__ bool match(const Pattern& p) const { return live && ((bits ^ p.bits) & p.mask & 0xffff) == 0; }
};

// A row's complete histogram, and its chunks' largest logits.
__device__ __forceinline__ void count_row(Shared& s, const Row& row, const Edge& edge) {
    const int t = threadIdx.x;
    each_vector(
        row.whole(), row.vectors,
        [&] {
            clear(s);
            if (edge.live) count_element(s, edge.bits);
        },
        [&](const uint4& w, int i, bool live) {
            if (live) count_vector(s, w);
            const short largest = largest_of_16(w);  // past the end of the last vector again, which lists no chunk too few
            if ((t & 15) == 15) s.largest[(i * kThreads + t) >> 4] = largest;
        },
        [&] { sweep(s); });
    __syncthreads();
}

// Lists the row's chunks that may hold the class, in order: those whose largest logit is not below it. One wave; their number.
__device__ __forceinline__ int list_chunks(const Shared& s, const Row& row, const Pattern& p, int* list) {
    const int lane = threadIdx.x & 63, chunks = (row.vectors + 63) / 64, least = signed_bits(p.bits & 0xffff);
    int listed = 0;
    for (int base = 0; base < chunks; base += 64) {
        const int chunk = base + lane;
        const short* largest = s.largest + 4 * min(chunk, kChunks - 1);
        const bool may = chunk < chunks && max(max(largest[0], largest[1]), max(largest[2], largest[3])) >= least;
        const unsigned long long all = __ballot(may);
        if (may) list[listed + __popcll(all & ((1ull << lane) - 1))] = chunk;
        listed += __popcll(all);
    }
    return listed;
}

// Occurrences in the listed chunks, batch by batch until more than `rank` are found; every thread gets their number, and
// `counts` holds them by place in the list. `found` is a word of LDS apart from them, 0 at first.
__device__ __forceinline__ int count_matches(const Row& row, const Pattern& p, int rank, const int* list, int listed, int* counts,
                                             int* found) {
    constexpr int kBatch = 6;  // loads of a wave in flight
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int base = 0; base < listed; base += kBatch * kWaves) {
        uint4 w[kBatch];
        int vector[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            vector[j] = list[min(base + j * kWaves + wave, listed - 1)] * 64 + lane;
            w[j] = row.whole()[min(vector[j], row.vectors - 1)];
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int at = base + j * kWaves + wave;
            if (at >= listed) break;
            int n = vector[j] < row.vectors ? occurrences(w[j], p) : 0;
            n = __any(n) ? wave_sum(n) : 0;
            if (lane == 0) {
                counts[at] = n;
                if (n) atomicAdd(found, n);
            }
        }
        __syncthreads();
        const int now = *found;
        __syncthreads();
        if (now > rank) break;
    }
    return *found;
}

// Writes the token of occurrence `rank` of the listed chunks from their counts. One wave.
template <class Index>
__device__ __forceinline__ void write_match(const Row& row, const Pattern& p, int rank, const int* list, int listed, const int* counts,
                                            Index* token) {
    const int lane = threadIdx.x & 63;
    int before;
    const int at = find_chunk(counts, listed, rank, before);
    const int vector = (at < 0 ? 0 : list[at]) * 64 + lane;
    const bool live = at >= 0 && vector < row.vectors;
    const uint4 w = live ? row.whole()[vector] : make_uint4(~p.bits, ~p.bits, ~p.bits, ~p.bits);
    const int element = find_element(w, p, before, rank);
    if (element >= 0) *token = row.head + 8 * vector + element;
}

// Occurrences in the row's head (tail: in its tail); the token, if rank is among them. One wave.
template <class Index>
__device__ __forceinline__ int edge_match(const Row& row, const Edge& edge, const Pattern& p, bool tail, int rank, Index* token) {
    const int lane = threadIdx.x & 63;
    const bool match = edge.match(p) && (lane < row.head) != tail;
    const unsigned long long all = __ballot(match);
    if (match && __popcll(all & ((1ull << lane) - 1)) == rank) *token = row.edge(lane);
    return __popcll(all);
}

// The token of the rank-th occurrence of the class: in the head, in the vectors or in the tail. (choose() has ended with a
// barrier: the histogram's memory is free.)
template <class Index>
__device__ __forceinline__ void find_token(Shared& s, const Row& row, const Edge& edge, const Choice& choice, Index* token) {
    const int t = threadIdx.x, wave = t >> 6;
    const Pattern pattern(choice.place);
    int *counts = reinterpret_cast<int*>(s.histogram), *list = counts + kChunks;
    if (wave == 0) {
        const int n = edge_match(row, edge, pattern, false, choice.rank, token);
        const int listed = list_chunks(s, row, pattern, list);
        if (t == 0) s.heavy = n, s.top = listed, s.count = 0;
    }
    __syncthreads();
    const int first = s.heavy, listed = s.top, rank = choice.rank - first;
    if (rank < 0) return;
    const int found = count_matches(row, pattern, rank, list, listed, counts, &s.count);
    if (wave != 0) return;
    if (found > rank)
        write_match(row, pattern, rank, list, listed, counts, token);
    else
        edge_match(row, edge, pattern, true, rank - found, token);
}

// What of a row decides its distribution.
struct Limits {
    bool open;  // without limits
    int kept;   // at most so many tokens; 0: any number

    __device__ __forceinline__ explicit Limits(const Settings& set) {
        kept = set.temperature > 0.0f ? max(set.top_k, 0) : 1;
        open = kept == 0 && set.top_p >= 1.0f && set.min_p <= 0.0f;
    }
    // Whether the largest logits of chunks of 16 vectors are a bound on what is kept.
    __device__ __forceinline__ bool few(const Row& row) const { return kept > 0 && kept <= min((row.vectors + 15) / 16, kCandidates); }
};

template <class T>
__device__ __forceinline__ float value_of(std::uint32_t bits) {
    return to_f32(__builtin_bit_cast(T, static_cast<unsigned short>(bits)));
}

// Sums of a row's weights 2^((x - top) heat) without a class for each: exponents of 64 bits, whose fraction (half a step of 2^-25)
// goes through an exponential of 32 (a step of 2^-23), added in eights and then in 64 bits. (A difference of logits is no number of
// 32 bits where one is 2^14 times the other: rounded to one, it weighed a whole tail by up to 2^-20 too much. 257 rows of 32003
// 24.2 -> 25.0 us.)
template <class T>
struct Weights {
    double top, heat, least;
    bool infinite;

    __device__ __forceinline__ Weights(float top, double heat)
        : top(top), heat(heat), least(-1000.0 / heat), infinite(top == __builtin_inff()) {}
    __device__ __forceinline__ float of_finite(std::uint32_t bits) const {
        constexpr double kWhole = 0x1.8p52;  // what is added to it is rounded to a whole number, which its low word holds
        const double d = fmax(static_cast<double>(value_of<T>(bits)) - top, least);  // of NaN and -inf too: they weigh nothing
        const double sum = fma(d, heat, kWhole), rest = fma(d, heat, kWhole - sum);
        const int whole = static_cast<int>(__builtin_bit_cast(std::uint64_t, sum));
        return __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f(static_cast<float>(rest)), whole);
    }
    __device__ __forceinline__ float of_infinite(std::uint32_t bits) const { return value_of<T>(bits) == top ? 1.0f : 0.0f; }
    __device__ __forceinline__ float operator()(std::uint32_t bits) const { return infinite ? of_infinite(bits) : of_finite(bits); }
    __device__ __forceinline__ float sum(const uint4& v) const {
        float x[8];
        if (infinite) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = of_infinite(element(v, j));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = of_finite(element(v, j));
        }
        return ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
    }
};

template <class T>
__device__ __forceinline__ float raised(float top, const uint4& w) {
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, value_of<T>(element(w, j)));
    return top;
}
__device__ __forceinline__ float wave_top(float top) {
#pragma unroll
    for (int step = 32; step; step >>= 1) top = fmaxf(top, __shfl_xor(top, step, 64));
    return top;
}

// Few and long rows are first looked at by the whole card: of a row without limits the largest logit and the mass of its parts, of
// one that keeps few logits its chunks' largest ones. (Else a row's one CU sees and sums them. Us in captured chains, with and
// without, for 5 rows of 248320 and 32, 48 and 96 of 151936: no limits 11.0 / 35.5, 18.6 / 30.0, 21.5 / 32.0 and 32.1 / 39.1;
// top_k 50 14.0 / 18.5, 20.5 / 20.5, 23.0 / 22.4 and 30.5 / 29.0. But every batch pays for the launch, rows that use nothing of it
// too: top_p alone 59 / 57, 47 / 45, 49 / 47 and 55 / 52, and of 96 rows with mixed settings, the slowest of which count classes,
// 58 / 51. So it stops at 32 rows, where it gains little for most settings. 16 rows of 32003, which a workgroup's registers hold:
// 10.7 / 10.7 and 14.0 / 13.0.)
constexpr int kScanThreads = 256, kScanWaves = kScanThreads / 64, kScanVectors = 4;  // vectors of a thread
constexpr int kScanPart = kScanThreads * kScanVectors;
constexpr int kScanRows = 32, kScanVocab = 8 * kFirst * kThreads;  // up to so many rows of more logits

template <class T>
__global__ __launch_bounds__(kScanThreads) void distribution_scan(Operands o) {
    __shared__ float tops[kScanWaves];
    __shared__ double masses[kScanWaves];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, index = blockIdx.y, begin = blockIdx.x * kScanPart;
    const Row row(o.logits, index, o.vocab);
    const Settings set = o.settings(index);
    const Limits limits(set);
    if (!limits.open && !limits.few(row)) return;
    const bool edge = blockIdx.x == 0 && t < row.head + row.tail, some = begin < row.vectors;
    const std::uint32_t edge_bits = edge ? row.start[row.edge(t)] : 0;
    uint4 w[kScanVectors];
    if (some) {
#pragma unroll
        for (int j = 0; j < kScanVectors; ++j) w[j] = row.whole()[min(begin + j * kScanThreads + t, row.vectors - 1)];
    }
    if (!limits.open) {
        if (!some) return;
#pragma unroll
        for (int j = 0; j < kScanVectors; ++j) {
            const short largest = largest_of_16(w[j]);  // past the end the last vector again
            const int chunk = (begin + j * kScanThreads + t) >> 4;
            if ((t & 15) == 15 && 16 * chunk < row.vectors) o.largest[static_cast<std::int64_t>(index) * o.chunk_count + chunk] = largest;
        }
        return;
    }
    const float none = -__builtin_inff();
    float top = edge ? fmaxf(value_of<T>(edge_bits), none) : none;
    if (some) {
#pragma unroll
        for (int j = 0; j < kScanVectors; ++j) top = raised<T>(top, w[j]);
    }
    top = wave_top(top);
    if (lane == 0) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kScanWaves; ++i) top = fmaxf(top, tops[i]);
    double mass = 0.0;
    if (top > none) {
        const Weights<T> weight(top, heat_of(set.temperature));
        if (edge) mass = weight(edge_bits);
        if (some) {
#pragma unroll
            for (int j = 0; j < kScanVectors; ++j) {
                const float sum = weight.sum(w[j]);
                if (begin + j * kScanThreads + t < row.vectors) mass += sum;
            }
        }
    }
    mass = wave_sum(mass);
    if (lane == 0) masses[wave] = mass;
    __syncthreads();
    if (t != 0) return;
    mass = 0.0;
    for (int i = 0; i < kScanWaves; ++i) mass += masses[i];
    o.parts[static_cast<std::int64_t>(index) * o.part_count + blockIdx.x] = {mass, top, 0};
}

// A row without limits, down to the lowest number; none at all if its largest logit is no class.
template <class T>
__device__ __forceinline__ Cut cut_of_all(float top, double heat, double mass) {
    Cut cut;
    cut.index = INT_MAX;
    if (top == -__builtin_inff()) cut.set(0.0, heat, 1.0, kNone);
    else cut.set(top, heat, mass, 0x8000 + static_cast<int>(Bits<T>::kInf) - 1);
    return cut;
}

// The same from its parts, two a lane at most. One wave; its first lane's.
template <class T>
__device__ __forceinline__ Cut join_parts(const Part* parts, int count, double heat) {
    const int lane = threadIdx.x & 63;
    const bool there[2] = {lane < count, lane + 64 < count};
    const Part part[2] = {parts[there[0] ? lane : 0], parts[there[1] ? lane + 64 : 0]};
    const float top = wave_top(fmaxf(part[0].top, part[1].top));
    double mass = 0.0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const double keep = part[i].top == top ? 1.0 : falling_power((static_cast<double>(part[i].top) - static_cast<double>(top)) * heat);
        if (there[i]) mass += keep * part[i].mass;
    }
    return cut_of_all<T>(top, heat, wave_sum(mass));
}

// The same by the row's workgroup (257 rows of 32003: 33.5 us through the histogram, 25).
template <class T>
__device__ __forceinline__ Cut keep_all(Shared& s, const Row& row, const Edge& edge, double heat) {
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const float none = -__builtin_inff();
    const auto join_top = [&](float top) {
        top = wave_top(edge.live ? fmaxf(value_of<T>(edge.bits), top) : top);
        if (lane == 0) s.wave_top[wave] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWaves; ++i) top = fmaxf(top, s.wave_top[i]);
        return top;
    };
    float top = none;
    double mass = 0.0;
    if (row.vectors > 0 && row.vectors <= kFirst * kThreads) {  // rows of up to 57344 logits stay in registers
        uint4 all[kFirst];
#pragma unroll
        for (int j = 0; j < kFirst; ++j) all[j] = row.whole()[min(t + j * kThreads, row.vectors - 1)];
#pragma unroll
        for (int j = 0; j < kFirst; ++j) top = raised<T>(top, all[j]);
        top = join_top(top);
        const Weights<T> weight(top, heat);
#pragma unroll
        for (int j = 0; j < kFirst; ++j) {
            if (j * kThreads >= row.vectors) break;
            const float sum = weight.sum(all[j]);
            if (t + j * kThreads < row.vectors) mass += sum;
        }
    } else {
        each_vector(row.whole(), row.vectors, [] {}, [&](const uint4& w, int, bool) { top = raised<T>(top, w); }, [] {});
        top = join_top(top);
        const Weights<T> weight(top, heat);
        each_vector(
            row.whole(), row.vectors, [] {},
            [&](const uint4& w, int, bool live) {
                const float sum = weight.sum(w);
                if (live) mass += sum;
            },
            [] {});
    }
    if (edge.live) mass += Weights<T>(top, heat)(edge.bits);
    mass = wave_sum(mass);
    if (lane == 0) s.wave_mass[wave] = mass;
    __syncthreads();
    mass = 0.0;
    for (int i = 0; i < kWaves; ++i) mass += s.wave_mass[i];
    return cut_of_all<T>(top, heat, mass);
}

// The `kept`-th largest of the chunks' largest logits in order (signed_bits + 32768, a thread's in `own`, 0: none), which
// bounds the row's from below; -1 if there are fewer. Infinities below and NaN count as no chunk. By the upper and then the
// lower byte; the bins are clear at first, and so are 16 counters for each upper byte (most logits share a few) in the
// histogram's place.
template <class T, int OWN>
__device__ __forceinline__ int bound_of(Shared& s, const int (&own)[OWN], int kept) {
    constexpr int kInf = static_cast<int>(Bits<T>::kInf);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int least = 0, left = kept;
#pragma unroll
    for (int level = 0; level < 2; ++level) {
#pragma unroll
        for (int j = 0; j < OWN; ++j)
            if (own[j] > 32768 - kInf && own[j] <= 32768 + kInf && (level == 0 || own[j] >> 8 == least >> 8))
                atomicAdd(level == 0 ? &s.histogram[(own[j] >> 8) * 16 + (lane & 15)] : &s.bins[own[j] & 255], 1u);
        __syncthreads();
        if (level == 0) {
            if (threadIdx.x < 256) {
                std::uint32_t n = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint4 c = reinterpret_cast<const uint4*>(s.histogram)[4 * threadIdx.x + ((i + lane) & 3)];
                    n += (c.x + c.y) + (c.z + c.w);
                }
                s.upper[threadIdx.x] = n;
            }
            __syncthreads();
        }
        const std::uint32_t* bins = level == 0 ? s.upper : s.bins;
        if (wave == 0) {  // bins from the highest down, four a lane
            const int high = 255 - 4 * lane;
            int n[4], four = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) n[i] = bins[high - i], four += n[i];
            int above = wave_scan(four) - four;
            if (lane == 63 && above + four < left) s.bin = -1;  // fewer than wanted
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (above < left && above + n[i] >= left) s.bin = high - i, s.above = above;
                above += n[i];
            }
        }
        __syncthreads();
        const int bin = s.bin;
        if (bin < 0) return -1;
        left -= s.above;
        least |= bin << (level == 0 ? 8 : 0);
        __syncthreads();
    }
    return least;
}

// The last of up to `kept` largest logits that the other limits leave, found without the histogram; false if they are too many
// for that. The logits from `least` on are all in the chunks that reach it, and few. They are put in order by counting who is
// ahead, 16 lanes for each, and the limits go by running sums of 64 bits over them. (5 rows of 248320, top_k 50, top_p 0.95: 43.9
// us through the histogram.)
template <class T, int OWN>
__device__ __forceinline__ bool cut_largest(Shared& s, const Row& row, const Edge& edge, const Settings& set, int kept, const int (&own)[OWN],
                                            int least, Cut& cut) {
    constexpr int kInf = static_cast<int>(Bits<T>::kInf);
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    if (t == 0) s.count = s.rank = 0;
    __syncthreads();
    // List the chunks, and the candidates in them.
#pragma unroll
    for (int j = 0; j < OWN; ++j) {
        const bool may = own[j] >= least;
        if (may) {
            const int at = atomicAdd(&s.count, 1);
            if (at < kListed) s.listed[at] = static_cast<unsigned short>(t + j * kThreads);
        }
    }
    __syncthreads();
    const int listed = s.count;
    if (listed > kListed) return false;
    const auto candidate = [&](std::uint32_t bits, int index) {
        const int order = signed_bits(bits) + 32768;
        if (order < least || order <= 32768 - kInf || order > 32768 + kInf) return;
        const int at = atomicAdd(&s.rank, 1);
        if (at < kCandidates) s.candidates[at] = static_cast<std::uint64_t>(order) << 32 | static_cast<std::uint32_t>(~index);
    };
    uint4 w[kListed / 64];
    int vector[kListed / 64];
#pragma unroll
    for (int j = 0; j < kListed / 64; ++j) {
        vector[j] = s.listed[min(64 * j + (t >> 4), listed - 1)] * 16 + (t & 15);
        w[j] = row.whole()[min(vector[j], row.vectors - 1)];
    }
#pragma unroll
    for (int j = 0; j < kListed / 64; ++j)
        if (64 * j + (t >> 4) < listed && vector[j] < row.vectors)
            for (int i = 0; i < 8; ++i) candidate(element(w[j], i), row.head + 8 * vector[j] + i);
    if (edge.live) candidate(edge.bits, row.edge(t));
    __syncthreads();
    const int found = s.rank;
    if (found > kCandidates) return false;
    for (int base = 0; base < found; base += kThreads / 16) {
        const int at = base + (t >> 4);
        const std::uint64_t mine = s.candidates[min(at, found - 1)];
        int ahead = 0;
        for (int i = t & 15; i < found; i += 16) ahead += s.candidates[i] > mine;
        ahead += moved<0x111, 0xf>(ahead);  // sums over the 16 lanes
        ahead += moved<0x112, 0xf>(ahead);
        ahead += moved<0x114, 0xf>(ahead);
        ahead += moved<0x118, 0xf>(ahead);
        if ((t & 15) == 15 && at < found) s.ordered[ahead] = mine;
    }
    __syncthreads();
    if (wave != 0) return true;
    const auto value = [](std::uint64_t c) {
        const int order = static_cast<int>(c >> 32) - 32768;
        return value_of<T>(order < 0 ? 0x8000 - order : order);
    };
    // Four candidates a lane, in order.
    const float top = value(s.ordered[0]);
    const double heat = heat_of(set.temperature), least_weight = set.min_p, share = set.top_p;
    double w4[4], four = 0.0;
    int above_min = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int at = 4 * lane + i;
        const float v = value(s.ordered[min(at, found - 1)]);
        const double weight = v == top ? 1.0 : falling_power((static_cast<double>(v) - static_cast<double>(top)) * heat);
        w4[i] = at < kept ? weight : 0.0;
        above_min += at < kept && weight >= least_weight;
        four += w4[i];
    }
    const double scan = wave_scan(four), up = __shfl_up(scan, 1, 64), before = lane ? up : 0.0;
    int length = least_weight <= 0.0 ? kept : wave_sum(above_min);
    if (!(share >= 1.0)) {
        const double border = share * lane_double(scan, 63);
        double at = before;
        int in = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            in += 4 * lane + i < kept && at < border;
            at += w4[i];
        }
        length = min(length, wave_sum(in));
    }
    length = max(length, 1);
    double mass = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) mass += 4 * lane + i < length ? w4[i] : 0.0;
    mass = wave_sum(mass);
    if (lane != 0) return true;
    const std::uint64_t last = s.ordered[length - 1];
    const int order = static_cast<int>(last >> 32) - 32768;
    cut.set(top, heat, mass, order < 0 ? 0x8000 - order : 32767 - order);
    cut.index = static_cast<int>(~static_cast<std::uint32_t>(last));
    return true;
}

// What a row keeps: a workgroup per row. Rows without limits are summed; up to 256 largest logits are put in order; else the
// classes are counted and chosen from as sample() does.
template <class T>
__global__ __launch_bounds__(kThreads) void distribution_cut(Operands o) {
    constexpr int kOwn = 4 * kChunks / kThreads;
    extern __shared__ __align__(16) unsigned char memory[];
    Shared& s = *reinterpret_cast<Shared*>(memory);
    const int t = threadIdx.x, wave = t >> 6, index = blockIdx.x;
    const Row row(o.logits, index, o.vocab);
    const int chunks = (row.vectors + 15) / 16;
    const bool scanned = o.part_count > 0;
    if (scanned) {  // used of a row that keeps few, and read beside the settings
        const short* known = o.largest + static_cast<std::int64_t>(index) * o.chunk_count;
        short largest[kOwn];
#pragma unroll
        for (int j = 0; j < kOwn; ++j) largest[j] = j * kThreads < chunks ? known[min(t + j * kThreads, chunks - 1)] : 0;
#pragma unroll
        for (int j = 0; j < kOwn; ++j)
            if (j * kThreads < chunks) s.largest[t + j * kThreads] = largest[j];
    }
    const Settings set = o.settings(index);
    const Limits limits(set);
    const Edge edge(row);
    const double heat = heat_of(set.temperature);
    Cut& cut = o.cuts[index];
    if (limits.open) {
        Cut all;
        if (!scanned) all = keep_all<T>(s, row, edge, heat);
        else if (wave == 0) all = join_parts<T>(o.parts + static_cast<std::int64_t>(index) * o.part_count, o.part_count, heat);
        if (t == 0) cut = all;
        return;
    }
    if (limits.few(row)) {
        reinterpret_cast<uint4*>(s.histogram)[t] = make_uint4(0, 0, 0, 0);
        if (t < 256) s.bins[t] = 0;
        if (!scanned) {
            each_vector(
                row.whole(), row.vectors, [] {},
                [&](const uint4& w, int i, bool) {
                    const short largest = largest_of_16(w);
                    if ((t & 15) == 15) s.largest[(i * kThreads + t) >> 4] = largest;
                },
                [] {});
        }
        __syncthreads();
        int own[kOwn];
#pragma unroll
        for (int j = 0; j < kOwn; ++j) own[j] = t + j * kThreads < chunks ? s.largest[t + j * kThreads] + 32768 : 0;
        const int least = bound_of<T>(s, own, limits.kept);
        if (least >= 0 && cut_largest<T>(s, row, edge, set, limits.kept, own, least, cut)) return;
        __syncthreads();
    }
    count_row(s, row, edge);
    const Choice choice = choose<T, true>(s, set);
    const bool ended = choice.place == kNone || s.whole;
    if (t == 0) {
        if (choice.place == kNone) cut.set(0.0, heat, 1.0, kNone);
        else cut.set(class_value<T>(s.top), heat, s.probability, choice.place);
        if (ended) cut.index = INT_MAX;
    }
    __syncthreads();
    if (!ended) find_token(s, row, edge, choice, &cut.index);
}

// A workgroup per row.
template <class T>
__global__ __launch_bounds__(kThreads) void sample(Operands o) {
    extern __shared__ __align__(16) unsigned char memory[];
    Shared& s = *reinterpret_cast<Shared*>(memory);
    const int t = threadIdx.x, index = blockIdx.x;
    const Row row(o.logits, index, o.vocab);
    const Settings set = o.settings(index);
    const Edge edge(row);
    count_row(s, row, edge);
    const Choice choice = choose<T, false>(s, set);
    if (t == 0 && o.probabilities) o.probabilities[index] = static_cast<float>(s.probability);
    if (choice.place == kNone) {
        if (t == 0) o.tokens[index] = -1;
        return;
    }
    find_token(s, row, edge, choice, o.tokens + index);
}

constexpr int kWriteThreads = 256;

// The probability of a logit that is the row's token `index`.
template <class T>
__device__ __forceinline__ float probability(const Cut& cut, std::uint32_t last, std::uint32_t bits, int index) {
    const float x = to_f32(__builtin_bit_cast(T, static_cast<unsigned short>(bits)));
    // Classes by value; the class of 0 holds both zeros.
    const float border = to_f32(__builtin_bit_cast(T, static_cast<unsigned short>(last)));
    if (!(x > border || (x == border && index <= cut.index))) return 0.0f;  // NaN too
    const double value = x;
    if (value == cut.max) return cut.inverse;
    // The exponent in two 32-bit parts, so that the weight errs by the exponential's own rounding alone.
    const double exponent = (value - cut.max) * cut.heat;
    const float high = static_cast<float>(exponent), low = static_cast<float>(exponent - static_cast<double>(high));
    if (!(high > -150.0f)) return 0.0f;
    // The rests of exponent and inverse together: the exponential's own error and one rounding are left.
    const float w = __builtin_amdgcn_exp2f(high);
    return fmaf(w, cut.inverse, w * fmaf(low * 0.693147181f, cut.inverse, cut.rest));
}

typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));

// Writes a row's probabilities from its cut: a vector of 8 a thread, the row's ragged ends with the first workgroup. (Four
// vectors a thread: 5 rows of 248320 2 us more, 257 of 32003 1 us less.)
template <class T>
__global__ __launch_bounds__(kWriteThreads) void distribution(Operands o) {
    const int index = blockIdx.y;
    const Row row(o.logits, index, o.vocab);
    const Cut cut = o.cuts[index];
    const bool some = cut.place != kNone;
    const std::uint32_t last = place_bits(some ? cut.place : 0);
    float* out = o.probabilities + static_cast<std::int64_t>(index) * o.vocab;
    if (blockIdx.x == 0 && static_cast<int>(threadIdx.x) < row.head + row.tail) {
        const int at = row.edge(threadIdx.x);
        out[at] = some ? probability<T>(cut, last, row.start[at], at) : 0.0f;
    }
    const int i = blockIdx.x * kWriteThreads + threadIdx.x;
    if (i >= row.vectors) return;
    const uint4 w = row.whole()[i];
    const int first = row.head + 8 * i;
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = some ? probability<T>(cut, last, element(w, j), first + j) : 0.0f;
    // Rows of odd vocabularies start at any multiple of 4 bytes.
    *reinterpret_cast<float4u*>(out + first) = float4u{p[0], p[1], p[2], p[3]};
    *reinterpret_cast<float4u*>(out + first + 4) = float4u{p[4], p[5], p[6], p[7]};
}

template <class T>
void launch(const Operands& o, hipStream_t stream) {
    static LdsLimit limit;
    limit.raise(sample<T>, sizeof(Shared));
    sample<T><<<o.rows, kThreads, sizeof(Shared), stream>>>(o);
}

template <class T>
void launch_distribution(const Operands& o, hipStream_t stream) {
    static LdsLimit limit;
    limit.raise(distribution_cut<T>, sizeof(Shared));
    if (o.part_count > 0) {
        distribution_scan<T><<<dim3(o.part_count, o.rows), kScanThreads, 0, stream>>>(o);
        check(hipGetLastError());
    }
    distribution_cut<T><<<o.rows, kThreads, sizeof(Shared), stream>>>(o);
    check(hipGetLastError());
    const unsigned parts = std::max((o.vocab / 8 + kWriteThreads - 1) / kWriteThreads, 1);
    distribution<T><<<dim3(parts, o.rows), kWriteThreads, 0, stream>>>(o);
}

// Of a row that is looked at first; 0: it is not.
int part_count(int rows, int vocab) { return rows <= kScanRows && vocab > kScanVocab ? (vocab / 8 + kScanPart - 1) / kScanPart : 0; }
int chunk_count(int vocab) { return (vocab / 8 + 15) / 16; }
static_assert(kMaxVocab / 8 <= 128 * kScanPart, "two parts a lane");

std::uint64_t distribution_bytes(int rows, int vocab) {
    const int parts = part_count(rows, vocab);
    return (sizeof(Cut) + sizeof(Part) * parts + (parts ? sizeof(short) * chunk_count(vocab) : 0)) * static_cast<std::uint64_t>(rows);
}

void require_geometry(int rows, int vocab) {
    require(rows > 0 && vocab > 0, "sampling needs rows and a vocabulary");
    require(vocab <= kMaxVocab, "sampling takes a vocabulary of at most 1048576");
}

}  // namespace
}  // namespace vt

#define VT_EXPORT extern "C" __attribute__((visibility("default")))

VT_EXPORT int venturi_sample_run(const void* logits, const float* uniforms, const float* temperature, const std::int32_t* top_k,
                                 const float* top_p, const float* min_p, std::int64_t* tokens, float* probabilities,
                                 int rows, int vocab, int dtype, void* stream) {
    return vt::guarded([&] {
        vt::require_geometry(rows, vocab);
        vt::require(logits && uniforms && tokens, "null sampling operand");
        vt::require(vt::aligned(logits, 16), "logits must be 16-byte aligned");
        const auto s = static_cast<hipStream_t>(stream);
        const vt::Operands o{logits, uniforms, temperature, top_k, top_p, min_p, tokens, probabilities, nullptr, nullptr, nullptr, rows, vocab, 0, 0};
        if (dtype == vt::kF16)
            vt::launch<__half>(o, s);
        else if (dtype == vt::kBF16)
            vt::launch<__hip_bfloat16>(o, s);
        else
            throw vt::Invalid("sampling takes fp16 or bf16 logits");
    });
}

VT_EXPORT std::uint64_t venturi_distribution_bytes(int rows, int vocab) {
    std::uint64_t bytes = 0;
    vt::host_guarded([&] {
        vt::require_geometry(rows, vocab);
        vt::require(rows <= vt::kMaxDistributionRows, "a distribution takes at most 65535 rows");
        bytes = vt::distribution_bytes(rows, vocab);
    });
    return bytes;
}

VT_EXPORT int venturi_distribution_run(const void* logits, const float* temperature, const std::int32_t* top_k, const float* top_p,
                                       const float* min_p, float* probabilities, void* workspace, std::uint64_t available,
                                       int rows, int vocab, int dtype, void* stream) {
    return vt::guarded([&] {
        vt::require_geometry(rows, vocab);
        vt::require(rows <= vt::kMaxDistributionRows, "a distribution takes at most 65535 rows");
        vt::require(logits && probabilities, "null distribution operand");
        vt::require(vt::aligned(logits, 16) && vt::aligned(probabilities, 4), "logits must be 16-byte aligned");
        vt::require(workspace && available >= vt::distribution_bytes(rows, vocab) && vt::aligned(workspace, 256),
                    "a distribution needs its workspace, 256-byte aligned");
        const std::uint64_t settings_bytes = 4ull * rows, logit_bytes = 2ull * rows * vocab, needed = vt::distribution_bytes(rows, vocab);
        const auto meets_an_input = [&](const void* out, std::uint64_t bytes) {
            return vt::meet(out, bytes, logits, logit_bytes) || vt::meet(out, bytes, temperature, settings_bytes) ||
                   vt::meet(out, bytes, top_k, settings_bytes) || vt::meet(out, bytes, top_p, settings_bytes) ||
                   vt::meet(out, bytes, min_p, settings_bytes);
        };
        vt::require(!meets_an_input(probabilities, 2 * logit_bytes) && !meets_an_input(workspace, needed) &&
                        !vt::meet(probabilities, 2 * logit_bytes, workspace, needed),
                    "a distribution's outputs must not overlap other operands");
        const auto s = static_cast<hipStream_t>(stream);
        auto* cuts = static_cast<vt::Cut*>(workspace);
        auto* parts = reinterpret_cast<vt::Part*>(cuts + rows);
        const int part_count = vt::part_count(rows, vocab);
        auto* largest = reinterpret_cast<short*>(parts + static_cast<std::int64_t>(rows) * part_count);
        const vt::Operands o{logits, nullptr, temperature, top_k, top_p, min_p, nullptr, probabilities, cuts, parts, largest,
                             rows, vocab, part_count, vt::chunk_count(vocab)};
        if (dtype == vt::kF16)
            vt::launch_distribution<__half>(o, s);
        else if (dtype == vt::kBF16)
            vt::launch_distribution<__hip_bfloat16>(o, s);
        else
            throw vt::Invalid("a distribution takes fp16 or bf16 logits");
    });
}

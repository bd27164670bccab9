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
#include "common.hpp"

#include <climits>

namespace vt {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kTurns = 64;                 // of 1024 classes, 16 a lane
constexpr int kMaxVocab = 1 << 20;
constexpr std::uint32_t kHeavy = 16384;
constexpr int kHeavyEntries = 2 * kMaxVocab / kHeavy;
constexpr int kNone = -1;                  // no class
constexpr int kChunks = kMaxVocab / 512;   // of 64 vectors, a wave's turn of a row
// Vectors of 8 logits that a thread counts before the first sweep for heavy classes (57344 logits, beside the up to 14 of the
// row's ragged ends), and between two sweeps (49152, on counters below 16384: 65535 at most).
constexpr int kFirst = 7, kNext = 6;

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
};

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

// Chooses from the workgroup's complete histogram.
template <class T>
__device__ Choice choose(Shared& s, const Settings& set) {
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
    // log2 e / T, from 4e-39 to 2e45.
    const double max_value = class_value<T>(top), least = set.min_p;
    const double heat = 1.44269504088896340736 / (greedy ? 1.0 : static_cast<double>(fminf(set.temperature, 3.402823466e38f)));
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
            if (lane == 0) s.place = top, s.rank = 0, s.probability = 1.0;
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
                const double border = share * prefix_mass(limit);
                length = min(length, border > 0.0 ? tokens_below(border, false) : 0);
            }
            length = max(length, 1);
            const double kept = prefix_mass(length);
            // A uniform of 1 or more stays below the end of the mass: the last token that adds to it.
            const double target = fmin(static_cast<double>(set.uniform) * kept, kept * (1.0 - 0x1p-52));
            int place = target >= 0.0 && set.uniform >= 0.0f ? tokens_below(target, true) : 0;
            place = max(min(place, length - 1), 0);
            open(count_before <= place);
            int at = before;
            l.each([&](int i, int n, double w) {
                if (place >= at && place < at + n) {
                    s.place = 1024 * turn + 16 * lane + i;
                    s.rank = place - at;
                    s.probability = w / kept;
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

struct Operands {
    const void* logits;
    const float* uniforms;
    const float* temperature;
    const std::int32_t* top_k;
    const float* top_p;
    const float* min_p;
    std::int64_t* tokens;
    float* probabilities;
    int rows, vocab;

    __device__ __forceinline__ Settings settings(int row) const {
        return {temperature ? temperature[row] : 1.0f, top_p ? top_p[row] : 1.0f, min_p ? min_p[row] : 0.0f, uniforms[row],
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
__device__ __forceinline__ void write_match(const Row& row, const Pattern& p, int rank, const int* list, int listed, const int* counts,
                                            std::int64_t* token) {
    const int lane = threadIdx.x & 63;
    int before;
    const int at = find_chunk(counts, listed, rank, before);
    const int vector = (at < 0 ? 0 : list[at]) * 64 + lane;
    const bool live = at >= 0 && vector < row.vectors;
    const uint4 w = live ? row.whole()[vector] : make_uint4(~p.bits, ~p.bits, ~p.bits, ~p.bits);
    const int element = find_element(w, p, before, rank);
    if (element >= 0) *token = row.head + 8ll * vector + element;
}

// Occurrences in the row's head (tail: in its tail); the token, if rank is among them. One wave.
__device__ __forceinline__ int edge_match(const Row& row, const Edge& edge, const Pattern& p, bool tail, int rank, std::int64_t* token) {
    const int lane = threadIdx.x & 63;
    const bool match = edge.match(p) && (lane < row.head) != tail;
    const unsigned long long all = __ballot(match);
    if (match && __popcll(all & ((1ull << lane) - 1)) == rank) *token = row.edge(lane);
    return __popcll(all);
}

// A workgroup per row.
template <class T>
__global__ __launch_bounds__(kThreads) void sample(Operands o) {
    extern __shared__ __align__(16) unsigned char memory[];
    Shared& s = *reinterpret_cast<Shared*>(memory);
    const int t = threadIdx.x, wave = t >> 6, index = blockIdx.x;
    const Row row(o.logits, index, o.vocab);
    const Settings set = o.settings(index);
    const Edge edge(row);
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
    const Choice choice = choose<T>(s, set);
    if (t == 0 && o.probabilities) o.probabilities[index] = static_cast<float>(s.probability);
    if (choice.place == kNone) {
        if (t == 0) o.tokens[index] = -1;
        return;
    }
    // The rank-th occurrence of the class: in the head, in the vectors or in the tail. (choose() has ended with a barrier:
    // the histogram's memory is free.)
    const Pattern pattern(choice.place);
    int *counts = reinterpret_cast<int*>(s.histogram), *list = counts + kChunks;
    if (wave == 0) {
        const int n = edge_match(row, edge, pattern, false, choice.rank, o.tokens + index);
        const int listed = list_chunks(s, row, pattern, list);
        if (t == 0) s.heavy = n, s.top = listed, s.count = 0;
    }
    __syncthreads();
    const int first = s.heavy, listed = s.top, rank = choice.rank - first;
    if (rank < 0) return;
    const int found = count_matches(row, pattern, rank, list, listed, counts, &s.count);
    if (wave != 0) return;
    if (found > rank)
        write_match(row, pattern, rank, list, listed, counts, o.tokens + index);
    else
        edge_match(row, edge, pattern, true, rank - found, o.tokens + index);
}

template <class T>
void launch(const Operands& o, hipStream_t stream) {
    static LdsLimit limit;
    limit.raise(sample<T>, sizeof(Shared));
    sample<T><<<o.rows, kThreads, sizeof(Shared), stream>>>(o);
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
        const vt::Operands o{logits, uniforms, temperature, top_k, top_p, min_p, tokens, probabilities, rows, vocab};
        if (dtype == vt::kF16)
            vt::launch<__half>(o, s);
        else if (dtype == vt::kBF16)
            vt::launch<__hip_bfloat16>(o, s);
        else
            throw vt::Invalid("sampling takes fp16 or bf16 logits");
    });
}

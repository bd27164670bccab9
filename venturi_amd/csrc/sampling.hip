// Sampling one token per row of 16-bit logits from given random numbers.
//
// A 16-bit logit has 65536 values, so a row's order is its histogram: classes of equal logits from the largest down,
// ties by index within a class. The workgroup of a row counts the classes in LDS (whole numbers: the order of the
// atomics leaves no trace), sums count * exp((v - max) / T) over steps of 64 neighbouring classes in 64 bits, and finds
// the borders of top-k, top-p and min-p and the place of u in the prefix sums. 64 bits, because a border of a large
// vocabulary is a token of 1e-6 of the mass, and one token more or less there moves every later draw. Only a class that
// occurs costs an exponential. The token is then the class's rank-th occurrence in the row.
//
// Counters are 16 bits wide (128 KB of the CU's 160 KB): a row of more than 65535 logits is counted in segments, and
// between two segments every class that has reached 16384 moves to a list (at most one entry per 16384 logits).
#include "common.hpp"

namespace vt {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kSteps = 1024;               // of 64 classes
constexpr int kTurns = kSteps / 16;        // of 16 steps
constexpr int kMaxVocab = 1 << 20;
constexpr std::uint32_t kHeavy = 16384;
constexpr int kHeavyEntries = 2 * kMaxVocab / kHeavy;
constexpr std::uint32_t kNone = 0;         // the sort key of logits that are never taken
// Vectors of 8 logits that a thread counts before the first sweep for heavy classes (57344 logits), and between two
// sweeps (49152, on counters below 16384).
constexpr int kFirst = 7, kNext = 6;

// Ascending sort key of a logit's bits: 0 for -inf and NaN, equal for both zeros.
template <class T> struct Bits;
template <> struct Bits<__half> {
    static constexpr std::uint32_t kInf = 0x7c00;
    static constexpr int kMantissa = 10;
};
template <> struct Bits<__hip_bfloat16> {
    static constexpr std::uint32_t kInf = 0x7f80;
    static constexpr int kMantissa = 7;
};

template <class T>
__device__ __forceinline__ std::uint32_t sort_key(std::uint32_t bits) {
    const std::uint32_t size = bits & 0x7fff;
    if (size > Bits<T>::kInf || bits == (0x8000 | Bits<T>::kInf)) return kNone;
    return size == 0 || !(bits & 0x8000) ? size | 0x8000 : bits ^ 0xffff;
}

template <class T>
__device__ __forceinline__ double key_value(std::uint32_t key) {
    const auto bits = static_cast<unsigned short>(key & 0x8000 ? key ^ 0x8000 : key ^ 0xffff);
    return static_cast<double>(to_f32(__builtin_bit_cast(T, bits)));
}

// The step between neighbouring classes at a key.
template <class T>
__device__ __forceinline__ double key_step(std::uint32_t key) {
    const std::uint32_t size = (key & 0x8000 ? key : key ^ 0xffff) & 0x7fff;
    const std::uint32_t low = size & ~((1u << Bits<T>::kMantissa) - 1);  // the binade's first
    return key_value<T>(0x8000 | (low + 1)) - key_value<T>(0x8000 | low);
}

template <class T>
struct Row {
    const unsigned short* logits;  // the tensor, 16-byte aligned
    std::int64_t first, end;       // the row's elements
    std::int64_t vector0;          // the aligned vector of 8 that holds its first
    int vectors;

    __device__ __forceinline__ Row(const void* tensor, int index, int vocab)
        : logits(static_cast<const unsigned short*>(tensor)), first(static_cast<std::int64_t>(index) * vocab), end(first + vocab),
          vector0(first >> 3), vectors(static_cast<int>(((end + 7) >> 3) - vector0)) {}

    // Vector i's logits; NaN bits for elements outside the row.
    __device__ __forceinline__ uint4 load(int i) const {
        const std::int64_t at = (vector0 + i) * 8;
        if (at >= first && at + 8 <= end) return *reinterpret_cast<const uint4*>(logits + at);
        std::uint32_t u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const std::int64_t e = at + 2 * j;
            u[j] = (e >= first && e < end ? logits[e] : 0x7fffu) | (e + 1 >= first && e + 1 < end ? logits[e + 1] : 0x7fffu) << 16;
        }
        return make_uint4(u[0], u[1], u[2], u[3]);
    }
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
    std::uint32_t histogram[32768];  // classes k (low half) and k + 32768 (high half)
    double mass_before[kSteps + 1];
    int count_before[kSteps + 1];
    std::uint32_t heavy_key[kHeavyEntries], heavy_count[kHeavyEntries];
    double wave_mass[kWaves];
    int wave_count[kWaves];
    double probability;
    int heavy, top, above_min, positive, rank, count, last;
    std::uint32_t key;
};

// A row's chosen class: its key (kNone: nothing to take), and which of its `count` occurrences.
struct Choice {
    std::uint32_t key;
    int rank, count;
};

__device__ __forceinline__ void clear(Shared& s) {
    for (int i = threadIdx.x; i < 32768 / 4; i += kThreads) reinterpret_cast<uint4*>(s.histogram)[i] = make_uint4(0, 0, 0, 0);
    if (threadIdx.x == 0) s.heavy = s.top = s.above_min = s.positive = 0;
    __syncthreads();
}

template <class T>
__device__ __forceinline__ void count_vector(Shared& s, const uint4& w, std::uint32_t& top) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const std::uint32_t key = sort_key<T>(element(w, j));
        top = max(top, key);
        if (key != kNone) atomicAdd(&s.histogram[key & 0x7fff], 1u << (16 * (key >> 15)));
    }
}

// Moves the classes that have reached kHeavy to the list.
__device__ __forceinline__ void sweep(Shared& s) {
    __syncthreads();
    for (int i = threadIdx.x; i < 32768; i += kThreads) {
        std::uint32_t word = s.histogram[i];
        if (!(word & 0xc000c000u)) continue;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const std::uint32_t n = (word >> (16 * half)) & 0xffff;
            if (n >= kHeavy) {
                const int e = atomicAdd(&s.heavy, 1);
                s.heavy_key[e] = i + 32768 * half;
                s.heavy_count[e] = n;
                word -= n << (16 * half);
            }
        }
        s.histogram[i] = word;
    }
    __syncthreads();
}

__device__ __forceinline__ int class_count(const Shared& s, std::uint32_t key) {
    std::uint32_t n = (s.histogram[key & 0x7fff] >> (16 * (key >> 15))) & 0xffff;
    for (int e = 0; e < s.heavy; ++e) n += s.heavy_key[e] == key ? s.heavy_count[e] : 0;
    return static_cast<int>(n);
}

// Keys of a step, one a lane, falling; the weight of a class is the step's first occurring class's times
// exp(-distance * spacing / T): neighbouring classes are evenly spaced within a step, so 16 steps of one binade share the
// second factor and compute their first ones side by side. Both exponents are at most 0.
__device__ __forceinline__ std::uint32_t step_key(int step) { return 65535 - (step * 64 + (threadIdx.x & 63)); }

template <class T>
__device__ __forceinline__ double first_weight(std::uint32_t key, std::uint32_t top, double max_value, double heat) {
    return key == top ? 1.0 : exp((key_value<T>(key) - max_value) / heat);
}
template <class T>
__device__ __forceinline__ double distance_weight(std::uint32_t key, double heat) {
    const int lane = threadIdx.x & 63;
    return lane == 0 ? 1.0 : exp(-(lane * key_step<T>(key)) / heat);
}
// distance[lane - first], or 0 below it.
__device__ __forceinline__ double at_distance(double distance, int first) {
    const int lane = threadIdx.x & 63;
    const double w = __shfl(distance, max(lane - first, 0), 64);
    return lane >= first ? w : 0.0;
}

// The largest step that passes a test which holds up to some step; every lane gets it.
template <class Test>
__device__ __forceinline__ int last_step(Test&& test) {
    int passed = 0;
#pragma unroll
    for (int i = 0; i < kSteps; i += 64) passed += __popcll(__ballot(test(i + static_cast<int>(threadIdx.x & 63))));
    return max(passed - 1, 0);
}

// Chooses from the workgroup's complete histogram; s.top has to hold the largest key.
template <class T>
__device__ Choice choose(Shared& s, const Settings& set) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const std::uint32_t top = s.top;
    if (top == kNone) {
        if (t == 0) s.probability = 0.0;
        __syncthreads();
        return {kNone, 0, 0};
    }
    if (!(set.temperature > 0.0f)) {
        if (t == 0) s.probability = 1.0;
        __syncthreads();
        return {top, 0, class_count(s, top)};
    }
    const double max_value = key_value<T>(top), heat = fminf(set.temperature, 3.402823466e38f), least = set.min_p;
    int above_min = 0, positive = 0;
    for (int turn = wave; turn < kTurns; turn += kWaves) {
        int n[16], first = 0, some = 0;  // lane i < 16 keeps step i's first occurring class
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const std::uint32_t key = step_key(turn * 16 + i);
            n[i] = key != kNone ? class_count(s, key) : 0;
            const unsigned long long occurs = __ballot(n[i] != 0);
            some |= occurs ? 1 << i : 0;
            const int at = occurs ? __ffsll(occurs) - 1 : 0;
            first = lane == i ? at : first;
        }
        double mass = 0.0;  // lane i < 16 keeps step i's mass and count
        int count = 0;
        if (some) {
            const std::uint32_t own = 65535 - ((turn * 16 + (lane & 15)) * 64 + first);
            const double start = first_weight<T>(own, top, max_value, heat);
            double distance = 0.0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                constexpr int kShared = (1 << Bits<T>::kMantissa) / 64;  // steps of a binade
                if (i % (kShared < 16 ? kShared : 16) == 0 && (some >> i) & ((1 << (kShared < 16 ? kShared : 16)) - 1))
                    distance = distance_weight<T>(step_key(turn * 16 + i), heat);
                if (!((some >> i) & 1)) continue;
                const double w = lane_double(start, i) * at_distance(distance, lane_int(first, i));
                if (n[i]) {
                    above_min += w >= least ? n[i] : 0;
                    positive += w > 0.0 ? n[i] : 0;
                }
                const double step_mass = wave_sum(n[i] * w);
                const int step_count = wave_sum(n[i]);
                if (lane == i) mass = step_mass, count = step_count;
            }
        }
        if (lane < 16) s.mass_before[turn * 16 + lane] = mass, s.count_before[turn * 16 + lane] = count;
    }
    above_min = wave_sum(above_min);
    positive = wave_sum(positive);
    if (lane == 0) {
        if (above_min) atomicAdd(&s.above_min, above_min);
        if (positive) atomicAdd(&s.positive, positive);
    }
    __syncthreads();
    const double mass_scan = wave_scan(s.mass_before[t]);
    const int count_scan = wave_scan(s.count_before[t]);
    if (lane == 63) s.wave_mass[wave] = mass_scan, s.wave_count[wave] = count_scan;
    __syncthreads();
    double mass_base = 0.0;
    int count_base = 0;
    for (int i = 0; i < wave; ++i) mass_base += s.wave_mass[i], count_base += s.wave_count[i];
    s.mass_before[t + 1] = mass_base + mass_scan;
    s.count_before[t + 1] = count_base + count_scan;
    if (t == 0) s.mass_before[0] = 0.0, s.count_before[0] = 0;
    __syncthreads();
    if (wave == 0) {
        const int all = s.count_before[kSteps];
        // The lane's class of a step: its key, count, weight and what comes before it in the whole order.
        std::uint32_t key;
        int n, before;
        double w, mass_at;
        const auto open = [&](int step) {
            key = step_key(step);
            n = key != kNone ? class_count(s, key) : 0;
            const unsigned long long occurs = __ballot(n != 0);
            const int first = occurs ? __ffsll(occurs) - 1 : 0;
            const double start = first_weight<T>(65535 - (step * 64 + first), top, max_value, heat);
            w = start * at_distance(distance_weight<T>(key, heat), first);  // every lane takes part in the exchange
            if (!n) w = 0.0;
            before = s.count_before[step] + wave_scan(n) - n;
            const double scan = wave_scan(n * w), below = __shfl_up(scan, 1, 64);
            mass_at = s.mass_before[step] + (lane ? below : 0.0);
        };
        const auto prefix_mass = [&](int length) {  // of the first `length` tokens
            if (length >= all) return s.mass_before[kSteps];
            const int step = last_step([&](int i) { return s.count_before[i] <= length; });
            open(step);
            return s.mass_before[step] + wave_sum(min(max(length - before, 0), n) * w);
        };
        const int limit = set.top_k > 0 ? min(set.top_k, all) : all;
        int length = min(limit, s.above_min);
        const double share = set.top_p;
        if (!(share >= 1.0)) {
            const double border = share * prefix_mass(limit);
            int below = 0;  // tokens with less mass than the border before them
            if (border > 0.0) {
                const int step = last_step([&](int i) { return s.mass_before[i] < border; });
                open(step);
                int in = 0;
                if (mass_at < border) {
                    in = n;
                    if (w > 0.0) {
                        in = static_cast<int>(fmin(ceil((border - mass_at) / w), static_cast<double>(n)));
                        if (in > 0 && mass_at + (in - 1) * w >= border) --in;
                        if (in < n && mass_at + in * w < border) ++in;
                    }
                }
                below = s.count_before[step] + wave_sum(in);
            }
            length = min(length, below);
        }
        length = max(length, 1);
        const double kept = prefix_mass(length);
        const double target = static_cast<double>(set.uniform) * kept;
        int place = 0;  // tokens whose share ends at or below the target
        if (target >= 0.0) {
            const int step = last_step([&](int i) { return s.mass_before[i] <= target; });
            open(step);
            int in = 0;
            if (mass_at <= target) {
                in = n;
                if (w > 0.0) {
                    in = static_cast<int>(fmin(floor((target - mass_at) / w), static_cast<double>(n)));
                    if (in > 0 && mass_at + in * w > target) --in;
                    if (in < n && mass_at + (in + 1) * w <= target) ++in;
                }
            }
            place = s.count_before[step] + wave_sum(in);
        }
        place = max(min(place, min(length, s.positive) - 1), 0);
        open(last_step([&](int i) { return s.count_before[i] <= place; }));
        if (place >= before && place < before + n) {
            s.key = key;
            s.rank = place - before;
            s.count = n;
            s.probability = w / kept;
        }
    }
    __syncthreads();
    return {s.key, s.rank, s.count};
}

template <class T>
__device__ __forceinline__ int occurrences(const uint4& w, std::uint32_t key) {
    int n = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) n += sort_key<T>(element(w, j)) == key;
    return n;
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

// The element (of the row) at which occurrence `rank` of 64 vectors lies, if it is the lane's; else -1.
template <class T>
__device__ __forceinline__ int find_element(const Row<T>& row, int vector, int vectors, std::uint32_t key, int before, int rank) {
    int at = -1;
    const uint4 w = vector < vectors ? row.load(vector) : make_uint4(0x7fff7fff, 0x7fff7fff, 0x7fff7fff, 0x7fff7fff);
    const int n = occurrences<T>(w, key);
    int next = before + wave_scan(n) - n;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (sort_key<T>(element(w, j)) == key && next++ == rank) at = static_cast<int>((row.vector0 + vector) * 8 + j - row.first);
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

// Visits a workgroup's vectors begin + t, begin + t + kThreads, .. below end, kAhead loads at a time; `between` runs, for the
// whole workgroup, after every kFirst and then every kNext of them.
constexpr int kAhead = 6;
template <class T, class Visit, class Between>
__device__ __forceinline__ void each_vector(const Row<T>& row, int begin, int end, Visit&& visit, Between&& between) {
    static_assert(kNext == kAhead && kFirst == kAhead + 1, "a sweep between two batches of loads");
    const int at = begin + threadIdx.x;
    const auto batch = [&](int i, int count) {
        uint4 w[kFirst];
#pragma unroll
        for (int j = 0; j < kFirst; ++j)
            w[j] = j < count && at + (i + j) * kThreads < end ? row.load(at + (i + j) * kThreads)
                                                              : make_uint4(0x7fff7fff, 0x7fff7fff, 0x7fff7fff, 0x7fff7fff);
#pragma unroll
        for (int j = 0; j < kFirst; ++j)
            if (j < count && begin + (i + j) * kThreads < end) visit(w[j], i + j);
    };
    batch(0, kFirst);
    for (int i = kFirst; begin + i * kThreads < end; i += kNext) {
        between();
        batch(i, kNext);
    }
}

// A workgroup per row.
template <class T>
__global__ __launch_bounds__(kThreads) void sample(Operands o) {
    extern __shared__ __align__(16) unsigned char memory[];
    Shared& s = *reinterpret_cast<Shared*>(memory);
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, index = blockIdx.x;
    const Row<T> row(o.logits, index, o.vocab);
    const Settings set = o.settings(index);
    clear(s);
    std::uint32_t top = kNone;
    each_vector(row, 0, row.vectors, [&](const uint4& w, int) { count_vector<T>(s, w, top); }, [&] { sweep(s); });
#pragma unroll
    for (int step = 32; step; step >>= 1) top = max(top, static_cast<std::uint32_t>(__shfl_xor(static_cast<int>(top), step, 64)));
    if (lane == 0) atomicMax(&s.top, static_cast<int>(top));
    __syncthreads();
    const Choice choice = choose<T>(s, set);
    if (t == 0 && o.probabilities) o.probabilities[index] = static_cast<float>(s.probability);
    if (choice.key == kNone) {
        if (t == 0) o.tokens[index] = -1;
        return;
    }
    // The rank-th occurrence of the class: occurrences per chunk of 64 vectors, then within the chunk. (choose() has ended
    // with a barrier: the histogram's memory is free.)
    __syncthreads();
    int* counts = reinterpret_cast<int*>(s.histogram);
    const int chunks = (row.vectors + 63) / 64;
    each_vector(
        row, 0, row.vectors,
        [&](const uint4& w, int i) {
            const int n = wave_sum(occurrences<T>(w, choice.key));
            if (lane == 0) counts[i * kWaves + wave] = n;
        },
        [] {});
    __syncthreads();
    if (wave == 0) {
        int before;
        const int chunk = find_chunk(counts, chunks, choice.rank, before);
        if (chunk >= 0) {
            const int at = find_element(row, chunk * 64 + lane, row.vectors, choice.key, before, choice.rank);
            if (at >= 0) o.tokens[index] = at;
        }
    }
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

VT_EXPORT std::uint64_t venturi_sample_bytes(int rows, int vocab) {
    vt::host_guarded([&] { vt::require_geometry(rows, vocab); });
    return 0;
}

VT_EXPORT int venturi_sample_run(const void* logits, const float* uniforms, const float* temperature, const std::int32_t* top_k,
                                 const float* top_p, const float* min_p, std::int64_t* tokens, float* probabilities,
                                 void* workspace, std::uint64_t available, int rows, int vocab, int dtype, void* stream) {
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

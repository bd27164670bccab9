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
constexpr int kFirstSegment = 8191;        // vectors of 8 logits: 65528
constexpr int kNextSegment = 6144;         // 49152, on counters below 16384
constexpr std::uint32_t kHeavy = 16384;
constexpr int kMaxVocab = 1 << 20;         // 64 entries of the list, 2049 chunks of 512 logits
constexpr int kHeavyEntries = kMaxVocab / kHeavy;
constexpr std::uint32_t kNone = 0;         // the sort key of logits that are never taken

// Ascending sort key of a logit's bits: 0 for -inf and NaN, equal for both zeros.
template <class T> struct Bits;
template <> struct Bits<__half> { static constexpr std::uint32_t kInf = 0x7c00; };
template <> struct Bits<__hip_bfloat16> { static constexpr std::uint32_t kInf = 0x7f80; };

template <class T>
__device__ __forceinline__ std::uint32_t sort_key(std::uint32_t bits) {
    if ((bits & 0x7fff) > Bits<T>::kInf || bits == (0x8000 | Bits<T>::kInf)) return kNone;
    if (bits == 0x8000) bits = 0;
    return bits & 0x8000 ? bits ^ 0xffff : bits | 0x8000;
}

template <class T>
__device__ __forceinline__ double key_value(std::uint32_t key) {
    const auto bits = static_cast<unsigned short>(key & 0x8000 ? key ^ 0x8000 : key ^ 0xffff);
    return static_cast<double>(to_f32(__builtin_bit_cast(T, bits)));
}

template <class T>
struct Row {
    const unsigned short* logits;  // the tensor, 16-byte aligned
    std::int64_t first, end;       // the row's elements
    std::int64_t total;            // the tensor's elements
    std::int64_t vector0;          // first aligned vector of 8 that holds one of them
    int vectors;

    // The keys of vector i; elements outside the row get kNone.
    __device__ __forceinline__ void keys(int i, std::uint32_t (&key)[8]) const {
        const std::int64_t at = (vector0 + i) * 8;
        if (at >= first && at + 8 <= end) {
            const uint4 w = *reinterpret_cast<const uint4*>(logits + at);
            const std::uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) key[j] = sort_key<T>((u[j >> 1] >> (16 * (j & 1))) & 0xffff);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) key[j] = at + j >= first && at + j < end ? sort_key<T>(logits[at + j]) : kNone;
        }
    }
};

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int step = 32; step; step >>= 1) v += __shfl_xor(v, step, 64);
    return v;
}
__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
    for (int step = 32; step; step >>= 1) v += __shfl_xor(v, step, 64);
    return v;
}
// Sums over lanes 0..lane.
template <class V>
__device__ __forceinline__ V wave_scan(V v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int step = 1; step < 64; step <<= 1) {
        const V below = __shfl_up(v, step, 64);
        if (lane >= step) v += below;
    }
    return v;
}

struct Shared {
    std::uint32_t histogram[32768];  // classes k (low half) and k + 32768 (high half)
    double mass_before[kSteps + 1];
    int count_before[kSteps + 1];
    std::uint32_t heavy_key[kHeavyEntries], heavy_count[kHeavyEntries];
    double wave_mass[kWaves];
    int wave_count[kWaves];
    int heavy, top, above_min, positive, rank;
    std::uint32_t key;
};

__device__ __forceinline__ int class_count(const Shared& s, std::uint32_t key) {
    std::uint32_t n = (s.histogram[key & 0x7fff] >> (16 * (key >> 15))) & 0xffff;
    for (int e = 0; e < s.heavy; ++e) n += s.heavy_key[e] == key ? s.heavy_count[e] : 0;
    return static_cast<int>(n);
}

// The largest step whose `before` passes the (falling) test; every lane gets it.
template <class Test>
__device__ __forceinline__ int last_step(Test&& test) {
    int passed = 0;
    for (int i = threadIdx.x & 63; i < kSteps; i += 64) passed += test(i);
    return max(wave_sum(passed) - 1, 0);
}

template <class T>
__global__ __launch_bounds__(kThreads) void sample(const void* __restrict__ logits, const float* __restrict__ uniforms,
                                                   const float* __restrict__ temperature, const std::int32_t* __restrict__ top_k,
                                                   const float* __restrict__ top_p, const float* __restrict__ min_p,
                                                   std::int64_t* __restrict__ tokens, float* __restrict__ probabilities, int rows,
                                                   int vocab) {
    extern __shared__ __align__(16) unsigned char memory[];
    Shared& s = *reinterpret_cast<Shared*>(memory);
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, index = blockIdx.x;
    Row<T> row;
    row.logits = static_cast<const unsigned short*>(logits);
    row.first = static_cast<std::int64_t>(index) * vocab;
    row.end = row.first + vocab;
    row.total = static_cast<std::int64_t>(rows) * vocab;
    row.vector0 = row.first >> 3;
    row.vectors = static_cast<int>(((row.end + 7) >> 3) - row.vector0);
    const float heat = temperature ? temperature[index] : 1.0f;

    for (int i = t; i < 32768 / 4; i += kThreads) reinterpret_cast<uint4*>(s.histogram)[i] = make_uint4(0, 0, 0, 0);
    if (t == 0) s.heavy = s.top = s.above_min = s.positive = 0;
    __syncthreads();
    std::uint32_t top = kNone;
    for (int begin = 0, end = min(kFirstSegment, row.vectors);; begin = end, end = min(end + kNextSegment, row.vectors)) {
        for (int i = begin + t; i < end; i += kThreads) {
            std::uint32_t key[8];
            row.keys(i, key);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                top = max(top, key[j]);
                if (key[j] != kNone) atomicAdd(&s.histogram[key[j] & 0x7fff], 1u << (16 * (key[j] >> 15)));
            }
        }
        __syncthreads();
        if (end == row.vectors) break;
        for (int i = t; i < 32768; i += kThreads) {
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
    atomicMax(&s.top, static_cast<int>(top));
    __syncthreads();
    top = s.top;
    if (top == kNone) {
        if (t == 0) {
            tokens[index] = -1;
            if (probabilities) probabilities[index] = 0.0f;
        }
        return;
    }

    double probability = 1.0;
    if (!(heat > 0.0f)) {
        if (t == 0) s.key = top, s.rank = 0;
    } else {
        const double max_value = key_value<T>(top), heat64 = fminf(heat, 3.402823466e38f);
        const double least = min_p ? min_p[index] : 0.0f;
        const auto weight = [&](std::uint32_t key) {
            // An infinite maximum leaves only itself.
            return key == top ? 1.0 : exp((key_value<T>(key) - max_value) / heat64);
        };
        // Classes in falling order: position 0 is key 65535.
        int above_min = 0, positive = 0;
        for (int step = wave; step < kSteps; step += kWaves) {
            const std::uint32_t key = 65535 - (step * 64 + lane);
            const int n = key != kNone ? class_count(s, key) : 0;
            double mass = 0.0;
            if (n) {
                const double w = weight(key);
                mass = n * w;
                above_min += w >= least ? n : 0;
                positive += w > 0.0 ? n : 0;
            }
            mass = wave_sum(mass);
            const int count = wave_sum(n);
            if (lane == 0) s.mass_before[step] = mass, s.count_before[step] = count;
        }
        atomicAdd(&s.above_min, above_min);
        atomicAdd(&s.positive, positive);
        __syncthreads();
        const double mass = s.mass_before[t];
        const int count = s.count_before[t];
        double mass_scan = wave_scan(mass);
        int count_scan = wave_scan(count);
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
                key = 65535 - (step * 64 + lane);
                n = key != kNone ? class_count(s, key) : 0;
                w = n ? weight(key) : 0.0;
                before = s.count_before[step] + wave_scan(n) - n;
                const double scan = wave_scan(n * w), up = __shfl_up(scan, 1, 64);
                mass_at = s.mass_before[step] + (lane ? up : 0.0);
            };
            const auto prefix_mass = [&](int length) {  // of the first `length` tokens
                if (length >= all) return s.mass_before[kSteps];
                const int step = last_step([&](int i) { return s.count_before[i] <= length; });
                open(step);
                return s.mass_before[step] + wave_sum(min(max(length - before, 0), n) * w);
            };
            const int wanted = top_k ? top_k[index] : 0;
            const int limit = wanted > 0 ? min(wanted, all) : all;
            int length = min(limit, s.above_min);
            const double share = top_p ? top_p[index] : 1.0f;
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
            const double target = static_cast<double>(uniforms[index]) * kept;
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
                s.wave_mass[0] = w / kept;
            }
        }
        __syncthreads();
        probability = s.wave_mass[0];
    }
    __syncthreads();

    // The rank-th occurrence of the class: occurrences per chunk of 64 vectors, then within the chunk.
    const std::uint32_t wanted = s.key;
    const int rank = s.rank;
    __syncthreads();  // the histogram's memory is reused below
    int* chunk_count = reinterpret_cast<int*>(s.histogram);
    const int chunks = (row.vectors + 63) / 64;
    for (int c = wave; c < chunks; c += kWaves) {
        int n = 0;
        if (c * 64 + lane < row.vectors) {
            std::uint32_t key[8];
            row.keys(c * 64 + lane, key);
#pragma unroll
            for (int j = 0; j < 8; ++j) n += key[j] == wanted;
        }
        n = wave_sum(n);
        if (lane == 0) chunk_count[c] = n;
    }
    __syncthreads();
    if (wave == 0) {
        int before = 0, chunk = -1;
        for (int base = 0; base < chunks && chunk < 0; base += 64) {
            const int n = base + lane < chunks ? chunk_count[base + lane] : 0;
            const int end = before + wave_scan(n);
            const unsigned long long hit = __ballot(end > rank);
            if (hit) {
                const int at = __ffsll(hit) - 1;
                chunk = base + at;
                before = __shfl(end - n, at, 64);
            } else {
                before = __shfl(end, 63, 64);
            }
        }
        if (chunk >= 0) {
            std::uint32_t key[8];
            int n = 0;
            const int vector = chunk * 64 + lane;
#pragma unroll
            for (int j = 0; j < 8; ++j) key[j] = kNone;
            if (vector < row.vectors) row.keys(vector, key);
#pragma unroll
            for (int j = 0; j < 8; ++j) n += key[j] == wanted;
            int at = before + wave_scan(n) - n;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (key[j] == wanted && at++ == rank) {
                    tokens[index] = (row.vector0 + vector) * 8 + j - row.first;
                    if (probabilities) probabilities[index] = static_cast<float>(probability);
                }
            }
        }
    }
}

template <class T>
void launch(const void* logits, const float* uniforms, const float* temperature, const std::int32_t* top_k, const float* top_p,
            const float* min_p, std::int64_t* tokens, float* probabilities, int rows, int vocab, hipStream_t stream) {
    static LdsLimit limit;
    limit.raise(sample<T>, sizeof(Shared));
    sample<T><<<rows, kThreads, sizeof(Shared), stream>>>(logits, uniforms, temperature, top_k, top_p, min_p, tokens,
                                                          probabilities, rows, vocab);
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
        if (dtype == vt::kF16)
            vt::launch<__half>(logits, uniforms, temperature, top_k, top_p, min_p, tokens, probabilities, rows, vocab, s);
        else if (dtype == vt::kBF16)
            vt::launch<__hip_bfloat16>(logits, uniforms, temperature, top_k, top_p, min_p, tokens, probabilities, rows, vocab, s);
        else
            throw vt::Invalid("sampling takes fp16 or bf16 logits");
    });
}

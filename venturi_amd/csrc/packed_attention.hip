// Causal attention over packed sequences: out = softmax(scale q k^T) v, every query over the keys up to its own.
//
// Bound by the matrix cores (4 rows keys head_dim operations) and, beside them, by the exponentials: at head_dim 128 a
// score costs half a cycle of a SIMD in the matrix unit and as much in the vector unit. A wave takes 32 query rows and
// works through the keys in tiles that its workgroup stages in LDS, double buffered: the next tile is copied there, without
// passing registers, while the present one is computed. 8192 tokens of one sequence, 48 heads on 4 of 128, bf16: 760 to 800
// us, 1030 to 1080 TFLOP/s, matrix cores busy 58% of the time; a large matrix product reaches 1226 on this card.
//
// Rows. The rows of a KV head are its (query, head of the group) pairs, query by query, cut into blocks of 128, so that
// all heads of a group share the staged keys, short sequences fill their tiles, and the diagonal's waste is
// small. S^T = K Q^T leaves a lane 16 keys of one query, which is the operand layout of O^T = V^T P^T with the keys in the
// order (lane half, register): weights, maxima and sums stay in their lane, but for one exchange between the lane halves
// when the reference moves. V^T comes out of row-major V through the transposing LDS reads.
//
// LDS. A row of keys or values takes a power of two of 16-byte units; a unit's place is XORed with the row (values: pairs
// of units, which the transposing read takes together), so that both kinds of reads find their rows on different banks.
//
// Softmax. Weights are 2^(s - m + 8), rounded to the model's type (fp16 2^-11, bf16 2^-8 of each), for a reference m that
// follows the maximum only when a score passes it by more than 4. The sums, in 32 bits, are of the rounded weights, which
// are what multiplies the values: a row's weights add to 1 whatever their rounding, and a dot product takes two at a time.
// The rounding is for the matrix unit's sake: against 64 bits the outputs err 1.2 to 1.4 times as much as by the one rounding
// at the end (11 prompts, fp16: 2.9e-4 of their norm for 2.1e-4; 8192 tokens, bf16: 2.0e-3 for 1.6e-3). A second term of each
// weight takes that away and multiplies every value twice: 190 -> 246 us and 764 -> 1079. fp16 weights reach down to 2^-33 of
// the row's largest.
//
// Split. A workgroup per block of 128 rows and KV head; blocks with the most keys first, as far as a wave can rank the
// sequences (11 prompts of 4096 tokens together: 196 -> 188 us). Few blocks over many keys are cut along the keys and joined
// by a second launch.
#include "kv_cache.hpp"

#include <climits>
#include <cmath>

namespace vt {
namespace {

typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef __bf16 bfloat8v __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef __bf16 bfloat2v __attribute__((ext_vector_type(2)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));

constexpr int kWaves = 4, kThreads = 64 * kWaves, kWaveRows = 32, kRows = kWaves * kWaveRows;
constexpr float kLazy = 4.0f, kShift = 8.0f;
constexpr int kMaxParts = 8;

struct Geometry {
    int tokens, keys, sequences, q_heads, kv_heads, group, head_dim;
    int blocks, parts;  // row blocks of a KV head (at most), and workgroups that share a block's keys
    float scale;
};

template <class T> struct Matrix;
template <> struct Matrix<__half> {
    static constexpr std::uint32_t kExponent = 0x7c00;
    static __device__ __forceinline__ float16v multiply(uint4 a, uint4 b, float16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8v, a), __builtin_bit_cast(half8v, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ std::uint32_t pack(float a, float b) {
        half2v v;
        v[0] = static_cast<_Float16>(a);
        v[1] = static_cast<_Float16>(b);
        return __builtin_bit_cast(std::uint32_t, v);
    }
    // sum + both halves of w.
    static __device__ __forceinline__ float add(std::uint32_t w, float sum) {
        const half2v ones = {static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)};
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, w), ones, sum, false);
    }
};
template <> struct Matrix<__hip_bfloat16> {
    static constexpr std::uint32_t kExponent = 0x7f80;
    static __device__ __forceinline__ float16v multiply(uint4 a, uint4 b, float16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bfloat8v, a), __builtin_bit_cast(bfloat8v, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ std::uint32_t pack(float a, float b) {
        bfloat2v v;
        v[0] = static_cast<__bf16>(a);
        v[1] = static_cast<__bf16>(b);
        return __builtin_bit_cast(std::uint32_t, v);
    }
    static __device__ __forceinline__ float add(std::uint32_t w, float sum) {
        const bfloat2v ones = {static_cast<__bf16>(1.0f), static_cast<__bf16>(1.0f)};
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bfloat2v, w), ones, sum, false);
    }
};

// Geometry of a staged tile of rows of D columns.
template <int D>
struct Tile {
    static constexpr int keys = D <= 128 ? 64 : 32;
    static constexpr int columns = D <= 32 ? 32 : D <= 64 ? 64 : D <= 128 ? 128 : 256;  // of an LDS row
    static constexpr int units = columns / 8;                                            // 16-byte units of an LDS row
    static constexpr int bytes = keys * columns * 2;
    static constexpr int loads = keys * units / kThreads;                                // per wave, of 64 units
    static constexpr int load_rows = kThreads / units;                                   // rows that a load of all waves covers
    // What a unit's place in its row is XORed with. Keys: the same unit of 16 rows lies in 16 places of the 256 bytes that the
    // banks span; in 8 at the largest heads, whose registers do not hold the addresses (882 us against 961 at 8192 tokens and
    // head_dim 256, with twice the LDS cycles). Values: of four rows' windows of four units (a transposing read of half a
    // wave) no two share a place.
    static constexpr int key_turn = units == 32 ? 7 : 15;
    static __device__ __forceinline__ int key_swizzle(int row) {
        if constexpr (units >= 16) return row & key_turn;
        else return (row / (16 / units)) & (units - 1);
    }
    static __device__ __forceinline__ int value_swizzle(int row) {  // even: pairs of units keep their order
        if constexpr (units >= 16) return 4 * (row & 3);
        else return 2 * ((row / (16 / units)) & (units / 2 - 1));
    }
};

// A sequence's part of the packed rows, clamped to the tensors.
struct Span {
    int q_first, queries, k_first, keys;
};

__device__ __forceinline__ Span span_of(const std::int32_t* __restrict__ q_offsets, const std::int32_t* __restrict__ k_offsets,
                                        int sequence, const Geometry& g) {
    Span s;
    s.q_first = min(max(q_offsets[sequence], 0), g.tokens);
    s.queries = min(max(q_offsets[sequence + 1], s.q_first), g.tokens) - s.q_first;
    s.k_first = min(max(k_offsets[sequence], 0), g.keys);
    s.keys = min(max(k_offsets[sequence + 1], s.k_first), g.keys) - s.k_first;
    return s;
}

__device__ __forceinline__ int blocks_of(const std::int32_t* __restrict__ q_offsets, int sequence, const Geometry& g) {
    const int first = min(max(q_offsets[sequence], 0), g.tokens), end = min(max(q_offsets[sequence + 1], first), g.tokens);
    return static_cast<int>((static_cast<std::int64_t>(end - first) * g.group + kRows - 1) / kRows);
}

// The sequence and row block of flat block `flat`. Up to 64 sequences come by falling number of keys, so that the longest
// blocks start first; within a sequence its last block is the longest.
__device__ __forceinline__ bool find_block(const std::int32_t* __restrict__ q_offsets, const std::int32_t* __restrict__ k_offsets,
                                           const Geometry& g, int flat, int& sequence, int& block) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < g.sequences; base += 64) {
        const int s = min(base + lane, g.sequences - 1);
        int n = blocks_of(q_offsets, s, g), own = s;
        if (base + lane >= g.sequences) n = 0;
        if (g.sequences > 1 && g.sequences <= 64) {
            const Span span = span_of(q_offsets, k_offsets, s, g);
            int rank = 0;
            for (int i = 0; i < g.sequences; ++i) {
                const int keys = __builtin_amdgcn_readlane(span.keys, i);
                rank += keys > span.keys || (keys == span.keys && i < lane);
            }
            if (lane >= g.sequences) rank = lane;
            n = __builtin_amdgcn_ds_permute(4 * rank, n);  // to the lane of its rank
            own = __builtin_amdgcn_ds_permute(4 * rank, own);
        }
        int end = n;
#pragma unroll
        for (int step = 1; step < 64; step <<= 1) {
            const int below = __shfl_up(end, step, 64);
            if (lane >= step) end += below;
        }
        end += before;
        const unsigned long long hit = __ballot(end > flat);
        if (hit) {
            const int at = __ffsll(hit) - 1;
            sequence = __builtin_amdgcn_readlane(own, at);
            block = __builtin_amdgcn_readlane(end, at) - 1 - flat;
            return true;
        }
        before = __builtin_amdgcn_readlane(end, 63);
    }
    block = flat - before;  // workgroups past the last block, counted from 0
    return false;
}

typedef int int4v __attribute__((ext_vector_type(4)));

// Copies tiles of rows from memory to LDS without a register: a load of a wave fills 64 consecutive units, so that the
// swizzle is in the address that a lane reads. The buffer's range makes zeros of rows past the sequence; columns past the
// head are sent past it.
template <int D>
struct Copy {
    std::uint32_t key_at[2], value_at;  // bytes from the tile's first row to the lane's unit (of every other load, for keys)
    std::uint32_t row_bytes;

    __device__ __forceinline__ Copy(int stride, int head_dim) : row_bytes(2 * stride) {
        const int row = threadIdx.x / Tile<D>::units, place = threadIdx.x % Tile<D>::units;
        const int value_unit = place ^ Tile<D>::value_swizzle(row);
#pragma unroll
        for (int i = 0; i < 2; ++i) {  // the swizzle repeats every 16 rows, one load or two
            const int key_unit = place ^ Tile<D>::key_swizzle(row + i * Tile<D>::load_rows);
            key_at[i] = 8 * key_unit < head_dim ? row * row_bytes + 16 * key_unit : 0x80000000u;
        }
        value_at = 8 * value_unit < head_dim ? row * row_bytes + 16 * value_unit : 0x80000000u;
    }
    // The tile at `source`, of which `rows` rows exist, to `lds` (a byte address).
    __device__ __forceinline__ void operator()(const void* source, int rows, std::uint32_t even, std::uint32_t odd, std::uint32_t lds) const {
        const auto base = reinterpret_cast<std::uint64_t>(source);
        const int4v buffer = {__builtin_amdgcn_readfirstlane(static_cast<int>(base)),
                              __builtin_amdgcn_readfirstlane(static_cast<int>(base >> 32) & 0xffff),
                              __builtin_amdgcn_readfirstlane(static_cast<int>(min(rows, Tile<D>::keys) * row_bytes)), 0x00020000};
        const std::uint32_t first = __builtin_amdgcn_readfirstlane(lds + (threadIdx.x >> 6) * 1024);
#pragma unroll
        for (int i = 0; i < Tile<D>::loads; ++i)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                         :
                         : "s"(first + i * (kThreads * 16)), "v"((i & 1 ? odd : even) + i * Tile<D>::load_rows * row_bytes), "s"(buffer)
                         : "memory");
    }
};

// Waits for the wave's copies and then for the other waves.
__device__ __forceinline__ void copies_done() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int D>
struct State {
    uint4 query[D / 16];
    float16v out[D / 32];
    float reference, sum;
};

__device__ __forceinline__ std::uint32_t finite_part(std::uint32_t w, std::uint32_t exponent) {
    const std::uint32_t high = exponent << 16;
    return ((w & exponent) == exponent ? 0 : w & 0xffffu) | ((w & high) == high ? 0 : w & 0xffff0000u);
}

// One tile of keys for a wave's 32 rows. MASKED: some row sees only a part of it (`seen` keys of the lane's row, counted
// from the tile's first).
template <class T, int D, bool MASKED>
__device__ __forceinline__ void compute(const unsigned char* __restrict__ keys, const unsigned char* __restrict__ values,
                                        State<D>& a, float factor, int seen) {
    constexpr int kTiles = Tile<D>::keys / 32;
    const int lane = threadIdx.x & 63, m = lane & 31, h = lane >> 5;
    float16v score[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) score[t][r] = 0.0f;
    // The swizzle turns the low bits of a unit; the rest of the address is a constant beside the row's.
    constexpr int kTurn = Tile<D>::units >= 16 ? Tile<D>::key_turn : 15;
    const unsigned char* row = keys + m * (Tile<D>::units * 16);
    const int turn = Tile<D>::key_swizzle(m);
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
        const unsigned char* at = row + ((((2 * s) & kTurn) | h) ^ turn) * 16;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            const uint4 k = *reinterpret_cast<const uint4*>(at + 32 * t * (Tile<D>::units * 16) + ((2 * s) & ~kTurn) * 16);
            score[t] = Matrix<T>::multiply(k, a.query[s], score[t]);
        }
    }
    if constexpr (D <= 128) {
        // The LDS reads run four ahead of the products.
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int i = 0; i < D / 16 * kTiles - 4; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, 4, 0);
    }
    float top = -__builtin_inff();
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            if (MASKED && 32 * t + 8 * (r / 4) + 4 * h + r % 4 >= seen) score[t][r] = -__builtin_inff();
            top = fmaxf(top, score[t][r]);
        }
    top *= factor;
    if (__any(top > a.reference + kLazy)) {
        const float next = fmaxf(a.reference, fmaxf(top, __shfl_xor(top, 32, 64)));
        const float keep = a.reference == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(a.reference - next);
        a.reference = next;
        a.sum *= keep;
#pragma unroll
        for (int d = 0; d < D / 32; ++d) a.out[d] *= keep;
    }
    const float base = a.reference == -__builtin_inff() ? 0.0f : kShift - a.reference;
    uint4 weight[2 * kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
        std::uint32_t w[8];
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
            const float x = __builtin_amdgcn_exp2f(fmaf(score[t][r], factor, base));
            const float y = __builtin_amdgcn_exp2f(fmaf(score[t][r + 1], factor, base));
            w[r / 2] = Matrix<T>::pack(x, y);
            a.sum = Matrix<T>::add(w[r / 2], a.sum);
        }
        weight[2 * t] = make_uint4(w[0], w[1], w[2], w[3]);
        weight[2 * t + 1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
    const int group = lane >> 4, i = lane & 15;
    const int row0 = 4 * h + (i >> 2);  // rows 16 t + 8 p + row0
    bool broken = false;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {
#pragma unroll
        for (int t = 0; t < 2 * kTiles; ++t) {
            uint2 part[2];
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int unit = ((4 * d) & 15) | 2 * (group & 1) | (i & 3) >> 1;
                // From 16 units on the swizzle repeats every 4 rows.
                const int place = unit ^ Tile<D>::value_swizzle(Tile<D>::units >= 16 ? row0 : 16 * t + 8 * p + row0);
                const unsigned char* at = values + row0 * (Tile<D>::units * 16) + place * 16 + 8 * (i & 1) +
                                          ((16 * t + 8 * p) * Tile<D>::units + ((4 * d) & ~15)) * 16;
                typedef __attribute__((address_space(3))) short4v* Lds;
                part[p] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(at)));
            }
            uint4 v = make_uint4(part[0].x, part[0].y, part[1].x, part[1].y);
            if (MASKED) {
                // A weight of 0 would make a NaN of an infinity that its row does not see.
                const uint4 clean = make_uint4(finite_part(v.x, Matrix<T>::kExponent), finite_part(v.y, Matrix<T>::kExponent),
                                               finite_part(v.z, Matrix<T>::kExponent), finite_part(v.w, Matrix<T>::kExponent));
                broken = broken || clean.x != v.x || clean.y != v.y || clean.z != v.z || clean.w != v.w;
                v = clean;
            }
            a.out[d] = Matrix<T>::multiply(v, weight[t], a.out[d]);
        }
    }
    if constexpr (!MASKED && D <= 128) {
        __builtin_amdgcn_sched_group_barrier(0x100, 6, 1);
#pragma unroll
        for (int i = 0; i < D / 32 * 2 * kTiles - 3; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 1);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, 3, 1);
    }
    if (MASKED && __any(broken)) {
        // Rare: infinities and NaN go to the rows that see them, key by key.
        for (int key = 0; key < Tile<D>::keys; ++key) {
            if (!__any(key < seen)) break;
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int column = 32 * d + 8 * (r / 4) + 4 * h + r % 4;
                    const int place = (key * Tile<D>::units + ((column >> 3) ^ Tile<D>::value_swizzle(key))) * 16 + (column & 7) * 2;
                    const std::uint32_t bits = *reinterpret_cast<const unsigned short*>(values + place);
                    if (key < seen && (bits & Matrix<T>::kExponent) == Matrix<T>::kExponent)
                        a.out[d][r] += to_f32(__builtin_bit_cast(T, static_cast<unsigned short>(bits)));
                }
        }
    }
}

// Rows past the last sequence get zeros, from the workgroups that found no block (one a head at least).
template <class T>
__device__ void clear_rest(const std::int32_t* __restrict__ q_offsets, T* __restrict__ out, const Geometry& g, int head, int spare,
                           int spares) {
    int first = 0;
    for (int i = threadIdx.x & 63; i <= g.sequences; i += 64) first = max(first, min(q_offsets[i], g.tokens));
#pragma unroll
    for (int step = 32; step; step >>= 1) first = max(first, __shfl_xor(first, step, 64));
    const int units = g.group * g.head_dim / 8;
    const std::int64_t count = static_cast<std::int64_t>(g.tokens - first) * units;
    for (std::int64_t i = static_cast<std::int64_t>(spare) * kThreads + threadIdx.x; i < count; i += static_cast<std::int64_t>(spares) * kThreads) {
        const std::int64_t token = i / units;
        T* row = out + ((first + token) * g.q_heads + head * g.group) * g.head_dim;
        reinterpret_cast<uint4*>(row)[i - token * units] = make_uint4(0, 0, 0, 0);
    }
}

// Partial results: per workgroup and row D outputs, then the reference and the sum, 16-byte aligned.
template <int D>
constexpr int partial_floats() { return D + 4; }
__host__ __device__ inline std::int64_t partial_row(const Geometry& g, int block_and_head, int part, int row) {
    return (static_cast<std::int64_t>(part) * g.blocks * g.kv_heads + block_and_head) * kRows + row;
}

template <class T, int D>
__global__ __launch_bounds__(kThreads, 2) void packed_attention(
    const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, const std::int32_t* __restrict__ q_offsets,
    const std::int32_t* __restrict__ k_offsets, T* __restrict__ out, float* __restrict__ partial, Geometry g) {
    __shared__ __align__(16) unsigned char memory[4 * Tile<D>::bytes];
    // Neighbouring workgroups go to different XCDs, round robin: with the head as the fast index the workgroups of one head
    // meet in few of the eight L2 caches.
    const int head = blockIdx.x % g.kv_heads, flat = blockIdx.x / g.kv_heads;
    int sequence, block;
    if (!find_block(q_offsets, k_offsets, g, flat, sequence, block)) {
        if (blockIdx.y == 0) clear_rest(q_offsets, out, g, head, block, g.blocks - (flat - block));
        return;
    }
    const Span s = span_of(q_offsets, k_offsets, sequence, g);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 31, h = lane >> 5;
    const int rows = s.queries * g.group;
    const int first_row = block * kRows + wave * kWaveRows, row = first_row + m;
    const bool live = row < rows;
    const int token = live ? row / g.group : 0;
    const std::int64_t place = (static_cast<std::int64_t>(s.q_first + token) * g.q_heads + head * g.group +
                                (live ? row - token * g.group : 0)) * g.head_dim;
    const int hidden = s.queries - s.keys;  // query i sees i + 1 - hidden keys
    const int seen = live ? token + 1 - hidden : INT_MAX;
    // The keys that the wave's first row sees, that its last one sees, and that the workgroup's last one sees.
    const int least = first_row < rows ? first_row / g.group + 1 - hidden : 0;
    const int most = first_row < rows ? min(first_row + kWaveRows - 1, rows - 1) / g.group + 1 - hidden : 0;
    int end = min(block * kRows + kRows - 1, rows - 1) / g.group + 1 - hidden, start = 0;
    if (g.parts > 1) {
        const int share = ((end + Tile<D>::keys - 1) / Tile<D>::keys + g.parts - 1) / g.parts * Tile<D>::keys;
        start = static_cast<int>(blockIdx.y) * share;
        end = min(end, start + share);
    }
    start = __builtin_amdgcn_readfirstlane(start);
    end = __builtin_amdgcn_readfirstlane(end);

    State<D> a;
    // A negative scale turns the queries' signs, so that the largest product is the largest score; 0 empties them.
    const float factor = g.scale == 0.0f ? 1.0f : fabsf(g.scale) * 1.44269504088896340736f;
    const std::uint32_t sign = g.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
        const int column = 16 * i + 8 * h;
        a.query[i] = make_uint4(0, 0, 0, 0);
        if (live && column < g.head_dim && g.scale != 0.0f) {
            const uint4 x = *reinterpret_cast<const uint4*>(q + place + column);
            a.query[i] = make_uint4(x.x ^ sign, x.y ^ sign, x.z ^ sign, x.w ^ sign);
        }
    }
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) a.out[d][r] = 0.0f;
    a.reference = -__builtin_inff();
    a.sum = 0.0f;

    constexpr int kKeys = Tile<D>::keys;
    const std::int64_t stride = static_cast<std::int64_t>(g.kv_heads) * g.head_dim;
    const T* key = k + s.k_first * stride + head * g.head_dim;
    const T* value = v + s.k_first * stride + head * g.head_dim;
    const Copy<D> copy(g.kv_heads * g.head_dim, g.head_dim);
    typedef __attribute__((address_space(3))) unsigned char* Lds;
    const auto lds = static_cast<std::uint32_t>(reinterpret_cast<std::uintptr_t>((Lds)(memory)));
    const auto fetch = [&](int at, int turn) {
        copy(key + at * stride, s.keys - at, copy.key_at[0], copy.key_at[1], lds + turn * (2 * Tile<D>::bytes));
        copy(value + at * stride, s.keys - at, copy.value_at, copy.value_at, lds + turn * (2 * Tile<D>::bytes) + Tile<D>::bytes);
    };
    if (start < end) fetch(start, 0);
    copies_done();
    for (int at = start, turn = 0; at < end; at += kKeys, turn ^= 1) {
        const unsigned char* now = memory + turn * (2 * Tile<D>::bytes);
        if (at + kKeys < end) fetch(at + kKeys, turn ^ 1);
        if (at < most) {
            if (at + kKeys <= least)
                compute<T, D, false>(now, now + Tile<D>::bytes, a, factor, 0);
            else
                compute<T, D, true>(now, now + Tile<D>::bytes, a, factor, seen - at);
        }
        copies_done();
    }
    a.sum += __shfl_xor(a.sum, 32, 64);
    if (!live) return;
    if (g.parts > 1) {
        float* target = partial + partial_row(g, blockIdx.x, blockIdx.y, wave * kWaveRows + m) * partial_floats<D>();
        // A part whose rows see none of its keys leaves no outputs.
        if (a.sum != 0.0f)
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int r = 0; r < 16; r += 4)
                    *reinterpret_cast<float4*>(target + 32 * d + 2 * r + 4 * h) =
                        make_float4(a.out[d][r], a.out[d][r + 1], a.out[d][r + 2], a.out[d][r + 3]);
        if (h == 0) *reinterpret_cast<float2*>(target + D) = make_float2(a.reference, a.sum);
        return;
    }
    const float scale = a.sum != 0.0f ? 1.0f / a.sum : 0.0f;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int column = 32 * d + 2 * r + 4 * h;
            if (column >= g.head_dim) continue;
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = a.sum == 0.0f ? 0.0f : a.out[d][r + j] * scale;
            *reinterpret_cast<uint2*>(out + place + column) = make_uint2(Matrix<T>::pack(x[0], x[1]), Matrix<T>::pack(x[2], x[3]));
        }
}

// Joins the parts of a block's rows: a wave per row, four columns a lane.
template <class T, int D>
__global__ __launch_bounds__(kThreads) void packed_attention_join(const std::int32_t* __restrict__ q_offsets,
                                                                  const std::int32_t* __restrict__ k_offsets, T* __restrict__ out,
                                                                  const float* __restrict__ partial, Geometry g) {
    const int head = blockIdx.x % g.kv_heads;
    int sequence, block;
    if (!find_block(q_offsets, k_offsets, g, blockIdx.x / g.kv_heads, sequence, block)) return;
    const Span s = span_of(q_offsets, k_offsets, sequence, g);
    const int lane = threadIdx.x & 63, in_block = blockIdx.y * kWaves + static_cast<int>(threadIdx.x >> 6);
    const int row = block * kRows + in_block, column = 4 * lane;
    if (row >= s.queries * g.group || column >= g.head_dim) return;
    const std::int64_t stride = partial_row(g, 0, 1, 0) * partial_floats<D>();
    const float* base = partial + partial_row(g, blockIdx.x, 0, in_block) * partial_floats<D>();
    float best = -__builtin_inff(), total = 0.0f, v[4] = {};
    float2 end[kMaxParts];
    float4 x[kMaxParts];
#pragma unroll
    for (int i = 0; i < kMaxParts; ++i) {  // past the last part they repeat it, at no weight
        const float* p = base + min(i, g.parts - 1) * stride;
        end[i] = *reinterpret_cast<const float2*>(p + D);
        x[i] = *reinterpret_cast<const float4*>(p + column);
    }
#pragma unroll
    for (int i = 0; i < kMaxParts; ++i) best = fmaxf(best, end[i].x);
#pragma unroll
    for (int i = 0; i < kMaxParts; ++i) {
        if (i >= g.parts || end[i].y == 0.0f) continue;  // without a weight the outputs were not written
        const float keep = end[i].x == -__builtin_inff() ? __builtin_nanf("") : __builtin_amdgcn_exp2f(end[i].x - best);
        total += end[i].y * keep;
        v[0] += x[i].x * keep, v[1] += x[i].y * keep, v[2] += x[i].z * keep, v[3] += x[i].w * keep;
    }
    const int token = row / g.group;
    const std::int64_t place = (static_cast<std::int64_t>(s.q_first + token) * g.q_heads + head * g.group + row - token * g.group) * g.head_dim;
    const float scale = 1.0f / total;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = total == 0.0f ? 0.0f : v[j] * scale;
    *reinterpret_cast<uint2*>(out + place + column) = make_uint2(Matrix<T>::pack(v[0], v[1]), Matrix<T>::pack(v[2], v[3]));
}

Geometry geometry(int tokens, int keys, int sequences, int q_heads, int kv_heads, int head_dim, float scale) {
    require_head_dim(head_dim);
    require(tokens > 0 && keys > 0 && sequences > 0 && q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0,
            "invalid packed attention geometry");
    const int group = q_heads / kv_heads;
    require(static_cast<std::int64_t>(tokens) * group < (1ll << 31) - kRows, "packed attention rows of a KV head must fit int32");
    // Every sequence leaves at most one block that is not full; one more clears what no sequence covers.
    const std::int64_t blocks = static_cast<std::int64_t>(tokens) * group / kRows + sequences + 1;
    require(blocks * kv_heads < (1ll << 31), "packed attention blocks must fit int32");
    require(static_cast<std::int64_t>(kv_heads) * head_dim < (1 << 23), "packed attention takes key rows of at most 8388607 columns");
    // Few rows over many keys: the blocks' keys are shared by as many workgroups as leave each about four tiles, while the
    // card (two workgroups to a CU) has room. 5 queries over 1505 keys, 48 heads of 128: 32 -> 15 us; 40 over 1540: 36 -> 21;
    // 300 over 1500, 32 heads (80 workgroups): 37 -> 32. Past 96 workgroups the join costs what the split saves (512
    // queries, 196 workgroups: 19 us without, 35 with two parts).
    const std::int64_t busy = (blocks - 1) * kv_heads, tiles = (keys / sequences + 63) / 64;
    const int parts = busy > 96 ? 1 : static_cast<int>(std::max<std::int64_t>(std::min({512 / busy, tiles / 4, std::int64_t{kMaxParts}}), 1));
    return {tokens, keys, sequences, q_heads, kv_heads, group, head_dim, static_cast<int>(blocks), parts, scale};
}

std::uint64_t partial_bytes(const Geometry& g) {
    return g.parts > 1 ? static_cast<std::uint64_t>(partial_row(g, 0, g.parts, 0)) * ((g.head_dim + 31) / 32 * 32 + 4) * sizeof(float) : 0;
}

template <class T, int D>
void launch(const void* q, const void* k, const void* v, const std::int32_t* q_offsets, const std::int32_t* k_offsets, void* out,
            void* workspace, const Geometry& g, hipStream_t stream) {
    const unsigned blocks = static_cast<unsigned>(g.blocks) * g.kv_heads;
    auto* partial = static_cast<float*>(workspace);
    packed_attention<T, D><<<dim3(blocks, g.parts), kThreads, 0, stream>>>(static_cast<const T*>(q), static_cast<const T*>(k),
                                                                          static_cast<const T*>(v), q_offsets, k_offsets,
                                                                          static_cast<T*>(out), partial, g);
    if (g.parts > 1) {
        check(hipGetLastError());
        packed_attention_join<T, D><<<dim3(blocks, kRows / kWaves), kThreads, 0, stream>>>(q_offsets, k_offsets, static_cast<T*>(out),
                                                                                          partial, g);
    }
}

template <class T>
void launch_any(const void* q, const void* k, const void* v, const std::int32_t* q_offsets, const std::int32_t* k_offsets,
                void* out, void* workspace, const Geometry& g, hipStream_t stream) {
    const int padded = (g.head_dim + 31) / 32 * 32;
    switch (padded) {
        case 32: launch<T, 32>(q, k, v, q_offsets, k_offsets, out, workspace, g, stream); break;
        case 64: launch<T, 64>(q, k, v, q_offsets, k_offsets, out, workspace, g, stream); break;
        case 96: launch<T, 96>(q, k, v, q_offsets, k_offsets, out, workspace, g, stream); break;
        case 128: launch<T, 128>(q, k, v, q_offsets, k_offsets, out, workspace, g, stream); break;
        case 160: launch<T, 160>(q, k, v, q_offsets, k_offsets, out, workspace, g, stream); break;
        case 192: launch<T, 192>(q, k, v, q_offsets, k_offsets, out, workspace, g, stream); break;
        case 224: launch<T, 224>(q, k, v, q_offsets, k_offsets, out, workspace, g, stream); break;
        default: launch<T, 256>(q, k, v, q_offsets, k_offsets, out, workspace, g, stream); break;
    }
}

}  // namespace
}  // namespace vt

#define VT_EXPORT extern "C" __attribute__((visibility("default")))

VT_EXPORT std::uint64_t venturi_packed_attention_bytes(int tokens, int keys, int sequences, int q_heads, int kv_heads,
                                                       int head_dim) {
    std::uint64_t bytes = 0;
    vt::host_guarded([&] { bytes = vt::partial_bytes(vt::geometry(tokens, keys, sequences, q_heads, kv_heads, head_dim, 1.0f)); });
    return bytes;
}

VT_EXPORT int venturi_packed_attention_run(const void* q, const void* k, const void* v, const std::int32_t* q_offsets,
                                           const std::int32_t* k_offsets, void* out, void* workspace, std::uint64_t available,
                                           int tokens, int keys, int sequences, int q_heads, int kv_heads, int head_dim,
                                           float scale, int dtype, void* stream) {
    return vt::guarded([&] {
        const auto g = vt::geometry(tokens, keys, sequences, q_heads, kv_heads, head_dim, scale);
        vt::require(q && k && v && q_offsets && k_offsets && out, "null packed attention operand");
        vt::require(std::fabs(scale) <= 0x1p127f, "attention scale must be a number of at most 2^127");
        vt::require(vt::aligned(q, 16) && vt::aligned(k, 16) && vt::aligned(v, 16) && vt::aligned(out, 16),
                    "packed attention rows must be 16-byte aligned");
        const std::uint64_t bytes = vt::partial_bytes(g);
        vt::require(!bytes || (workspace && available >= bytes && vt::aligned(workspace, 256)),
                    "packed attention of few rows needs its workspace, 256-byte aligned");
        const auto s = static_cast<hipStream_t>(stream);
        if (dtype == vt::kF16)
            vt::launch_any<__half>(q, k, v, q_offsets, k_offsets, out, workspace, g, s);
        else if (dtype == vt::kBF16)
            vt::launch_any<__hip_bfloat16>(q, k, v, q_offsets, k_offsets, out, workspace, g, s);
        else
            throw vt::Invalid("packed attention takes fp16 or bf16");
    });
}

// Attention over the paged Q8 cache: out = softmax(scale q k^T) v for the few new tokens of many sequences.
//
// Bound by HBM: every code and scale of K and V is read once (272 bytes a token and head at head_dim 128). A wave takes
// 32 keys at a time out of LDS, into which the next ones' codes and scales are copied beside it without passing registers
// (in registers they left one wave on a SIMD at head_dim 256: 16 x 5 drafted tokens 74 us, now 40), and keeps weights,
// outputs and statistics in registers until the waves of a workgroup join. 4 sequences of 90000 to 131000 keys, 48 heads
// on 4 of 128: 98 us a call, 94 of them this kernel's (503 MB read, 5.3 TB/s), where a large copy reaches 4.9.
//
// Rows. The query rows of one KV head (query_tokens x group) are the columns of 16-wide matrix tiles, so that a KV
// head's codes are read once for all heads that share them: up to 16 rows the four waves of a workgroup take other keys, up
// to 32 rows two waves share a step's codes, above that four. With S^T = K Q^T a lane holds four keys of one query,
// which is the operand layout of O^T = V^T P^T if the 32 keys are taken in the order (tile, lane group, register): the
// weights never leave their lane.
//
// Codes. A code c is stored as the byte u = c + 128, and a byte in the low half of a 16-bit word is the fp16 number
// u 2^-24 (subnormal; the matrix cores keep it), so that one v_perm makes two operands.
//   K: S = sum_groups scale_k * (sum u q - 128 sum q), the second term as the accumulator's start: exact products, fp32.
//   V: a lane holds 8 keys of a few columns, a pair of keys is one v_perm of two keys' bytes, and v = ((u - 128) 2^-9)
//      (scale_v k 2^14), the first factor exact, the product rounded once to fp16 (2^-11). k is a power of two that brings
//      the largest scale so far to at most 1. Scales more than 2^18 below that one (other columns, or keys of any weight)
//      would lose bits at fp16's lower end: steps that hold one multiply those scales apart, brought up by 2^19 or 2^38
//      (32 sequences of 3000 keys, 32 heads on 8 of 128, bf16: 42 us; with such scales in every step 63).
// Queries are scaled by a power of two per row into fp16's range: exact for fp16 and, but for numbers 2^28 below the
// row's largest, for bf16. The weights are rounded to fp16 (2^-11); their sum is of the unrounded ones.
// For bf16 rows, whose own rounding is eight times as coarse, that is that (error against 64 bits 1.01 to 1.02 times that of the
// one rounding at the end; with second terms 16 x 5 drafted tokens 45 -> 54 us). For fp16 rows both factors of O = P V have a
// second term, what the first one's rounding left: the outputs' error against 64 bits at 1021 keys is that of the one
// rounding at the end (2.1e-4 of their norm) where single terms leave 3.3e-4, for 1 to 2% of the time (64 sequences of 1 to
// 8190 keys: 46.4 -> 47.3 us). Weights reach down to 2^-33 of the row's largest (fp16's
// least number beside 2^8): what a key with less weight adds is lost, at most 2^-33 of its value.
//
// Softmax. One pass: weights are 2^(s - m) for a reference m that follows the maximum only when a score passes it by
// more than 4 (a factor of 16 fits fp16's range): the rescaling of the outputs is rare.
//
// Split. The keys of all sequences are cut into chunks of one length, chosen on the device from the sum of the
// lengths, so that the grid is about `kTarget` workgroups whatever the lengths; a workgroup finds its sequence by a scan,
// whole chunks before the sequences' shorter ends.
// Two workgroups to a CU, one round: 512 is faster than 768, 1024 and 2048 (long sequences: 104, 119, 120, 155 us).
// A sequence of one chunk is finished by its workgroup, others leave partial outputs, joined by a second launch.
#include "kv_cache.hpp"

#include <climits>
#include <cmath>
#include <type_traits>

namespace vt {
namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4, kBlock = 32;           // keys of a wave's step
constexpr int kMinChunk = 128;
constexpr int kTarget = 512;                     // workgroups: two to a CU
constexpr float kLazy = 4.0f, kShift = 8.0f;     // weights are 2^(s - m + kShift), at most 2^12
constexpr float kLeastScale = 0x1p-18f;          // of a value scale times k, below which code 1 times it loses bits in fp16

struct Geometry {
    int sequences, query_tokens, q_heads, kv_heads, group, rows;  // rows = query_tokens * group, of one KV head
    int head_dim, row_blocks, max_pages, tiles_per_page;
    std::uint64_t page_magic;                    // ceil(2^36 / tiles_per_page)
    int target;                                  // chunks per KV head and row block
    float scale;
    std::int64_t longest;                        // max_pages * page_tokens
};

// What a workgroup does: chunk `split` of a sequence's `splits`, whose partial results go to `slot`.
struct Work {
    int sequence, split, splits, length, slot;
    std::int64_t chunk;
};

__device__ __forceinline__ std::int64_t wave_sum(std::int64_t v) {
#pragma unroll
    for (int step = 32; step; step >>= 1) v += __shfl_xor(v, step, 64);
    return v;
}

__device__ __forceinline__ int admitted(int length, const Geometry& g) {
    return length < 0 || length > g.longest ? 0 : length;  // a bad length is one chunk, which marks its rows
}

// The lane's share of the lengths: those of sequences base + lane, or 0 past the last.
__device__ __forceinline__ int length_at(const std::int32_t* __restrict__ lengths, const Geometry& g, int base) {
    const int s = base + static_cast<int>(threadIdx.x & 63), length = lengths[min(s, g.sequences - 1)];
    return s < g.sequences ? length : 0;
}

// The chunk's length, from the lengths of the first 64 sequences (in hand) and of the others.
__device__ __forceinline__ std::int64_t chunk_length(const std::int32_t* __restrict__ lengths, const Geometry& g, int first) {
    std::int64_t total = admitted(first, g);
    for (int base = 64; base < g.sequences; base += 64) total += admitted(length_at(lengths, g, base), g);
    total = wave_sum(total);
    // A chunk is no longer than a sequence need be: below 2^31 (uniform, so that the loops over it are).
    const std::int64_t least = (total + g.target - 1) / g.target, blocks = max((least + kMinChunk - 1) / kMinChunk, std::int64_t{1});
    return static_cast<std::int64_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(min(blocks, std::int64_t{INT_MAX / kMinChunk})))) * kMinChunk;
}

// A sequence's whole chunks, and whether a shorter one follows (also where the sequence is empty: it marks or clears its rows).
struct Cut {
    int whole, rest;
    __device__ __forceinline__ Cut(int length, std::int64_t chunk)
        : whole(static_cast<int>(length / chunk)), rest(length == 0 || length != whole * chunk) {}
    __device__ __forceinline__ int chunks() const { return whole + rest; }
};

// Whole chunks of the sequences base + lane, summed over lanes 0..lane.
__device__ __forceinline__ int whole_scan(int length, const Geometry& g, std::int64_t chunk) {
    const int lane = threadIdx.x & 63;
    int end = Cut(admitted(length, g), chunk).whole;
#pragma unroll
    for (int step = 1; step < 64; step <<= 1) {
        const int below = __shfl_up(end, step, 64);
        if (lane >= step) end += below;
    }
    return end;
}

// Workgroups take the whole chunks of all sequences first (at most `target`: one slot each, in order) and then the shorter
// ends (slot target + sequence), which fill what the whole ones leave of the card.
__device__ __forceinline__ bool find_work(const std::int32_t* __restrict__ lengths, const Geometry& g, int flat, Work& w) {
    const int first = length_at(lengths, g, 0);
    w.chunk = chunk_length(lengths, g, first);
    int before = 0;
    for (int base = 0; base < g.sequences; base += 64) {
        const int length = base ? length_at(lengths, g, base) : first;
        const int end = before + whole_scan(length, g, w.chunk);
        const unsigned long long hit = __ballot(end > flat);
        if (hit) {
            const int at = __ffsll(hit) - 1;
            w.sequence = base + at;
            w.length = __builtin_amdgcn_readlane(length, at);
            const Cut cut(w.length, w.chunk);  // whole chunks: an admitted length
            w.splits = cut.chunks();
            w.split = flat - (__builtin_amdgcn_readlane(end, at) - cut.whole);
            w.slot = flat;
            return true;
        }
        before = __builtin_amdgcn_readlane(end, 63);
    }
    w.sequence = flat - before;
    if (w.sequence >= g.sequences) return false;
    w.length = __builtin_amdgcn_readfirstlane(lengths[w.sequence]);
    const Cut cut(admitted(w.length, g), w.chunk);
    w.splits = cut.chunks();
    w.split = cut.whole;
    w.slot = g.target + w.sequence;
    return cut.rest;
}

__device__ __forceinline__ std::uint32_t permute(std::uint32_t high, std::uint32_t low, std::uint32_t selector) {
    return __builtin_amdgcn_perm(high, low, selector);
}

// Bytes b and b + 1 of a word as two fp16 u 2^-24 (selector 0x0c is a zero byte).
template <int B>
__device__ __forceinline__ std::uint32_t spread(std::uint32_t word) {
    return permute(0, word, 0x0c000c00u | B | (B + 1) << 16);
}

__device__ __forceinline__ half8v spread8(std::uint32_t a, std::uint32_t b) {
    const uint4 w = make_uint4(spread<0>(a), spread<2>(a), spread<0>(b), spread<2>(b));
    return __builtin_bit_cast(half8v, w);
}

__device__ __forceinline__ std::uint32_t pack(float a, float b) {
    half2v v;
    v[0] = static_cast<_Float16>(a);
    v[1] = static_cast<_Float16>(b);
    return __builtin_bit_cast(std::uint32_t, v);
}

__device__ __forceinline__ float half_at(const uint2& w, int i) {
    return i & 1 ? half_hi(i < 2 ? w.x : w.y) : half_lo(i < 2 ? w.x : w.y);
}

// The value columns of a lane. A row of D columns is cut into segments of 256, 128, 64 and 32; in a segment of width W
// lane m holds the W / 16 columns from (W / 16) m on.
template <int D>
struct Segments {
    static constexpr int count = (D >= 256 ? 1 : 0) + (D % 256 >= 128 ? 1 : 0) + (D % 128 >= 64 ? 1 : 0) + (D % 64 >= 32 ? 1 : 0);
    static constexpr int width(int i) {
        int left = D;
        for (int w = 256; w >= 32; w >>= 1)
            if (left >= w) {
                if (i-- == 0) return w;
                left -= w;
            }
        return 0;
    }
    static constexpr int offset(int i) {
        int sum = 0;
        for (int j = 0; j < i; ++j) sum += width(j);
        return sum;
    }
    static constexpr int tile(int i) { return offset(i) / 16; }  // first of the segment's matrix tiles
    static constexpr int word(int i) {                           // first of its words in a lane's register copy of a key
        int sum = 0;
        for (int j = 0; j < i; ++j) sum += (width(j) / 16 + 3) / 4;
        return sum;
    }
    static constexpr int words = word(count);
};

// One step of a wave in LDS: 16 keys' codes, twice, for K and for V, then their scales [group][16]. A row's 16-byte units are
// turned by its number, so that the same columns of 16 rows lie on different banks.
template <int D>
struct Step {
    static constexpr int units = D / 16;          // of a row
    static constexpr int tile = 16 * D;           // bytes of a tile's codes
    static constexpr int scales = D;              // bytes of a tile's scales
    static constexpr int bytes = 4 * tile + 4 * scales;
    static constexpr int loads = (D + 63) / 64 + 1;  // of a tile and side
    static __device__ __forceinline__ int swizzle(int row) {
        if constexpr (units == 16) return row & 15;
        else if constexpr (units == 8) return (row >> 1) & 7;
        else if constexpr (units == 4 || units == 12) return (row >> 2) & 3;
        else return 0;  // the rows' own stride spreads them
    }
};

// How a workgroup's waves divide a round: ROWS tiles of 16 rows by KEYS steps of 32 keys, and how many rounds are in flight.
template <int D, int ROWS>
struct Shape {
    static constexpr int keys = kWaves / ROWS;
    static constexpr int round_bytes = keys * Step<D>::bytes;
    static constexpr int ring = 79872 / round_bytes < 2 ? 2 : 79872 / round_bytes > 4 ? 4 : 79872 / round_bytes;
    static constexpr int bytes = ring * round_bytes > 256 * (D + 4) ? ring * round_bytes : 256 * (D + 4);  // or the joined rows
    static constexpr int loads = 4 * Step<D>::loads / ROWS;  // of a wave and round
    static_assert(bytes <= 163840 - 1024, "the ring fits the LDS");
};

typedef const __attribute__((address_space(4))) std::int32_t* Constant;  // read through the scalar cache

struct Pages {
    CachePlanes planes;
    const std::int32_t* table;
    int tiles_per_page, head;
    std::uint64_t magic;
    __device__ __forceinline__ int page_of(int tile) const {
        return static_cast<int>((static_cast<std::uint64_t>(tile) * magic) >> 36);
    }
};

__device__ __forceinline__ void copy16(std::uint32_t lds, const void* base, std::uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(offset), "s"(base) : "memory");
}
__device__ __forceinline__ void copy4(std::uint32_t lds, const void* base, std::uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" : : "s"(lds), "v"(offset), "s"(base) : "memory");
}

// Where the two tiles of a step lie: their pages, and their first keys' places there.
struct Places {
    int page[2], inside[2];
};

__device__ __forceinline__ Places places_of(const Pages& p, int first_tile, int last_tile) {
    Places at;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int tile = min(first_tile + t, last_tile), entry = p.page_of(tile);
        at.inside[t] = (tile - entry * p.tiles_per_page) * 16;
        at.page[t] = reinterpret_cast<Constant>(reinterpret_cast<std::uintptr_t>(p.table))[entry];
    }
    return at;
}

// Starts the copies of a wave's share of a step into LDS: parts (side, tile), every ROWS-th of the four.
template <int D, int ROWS>
__device__ __forceinline__ void fetch(const Pages& p, const Places& at, int share, std::uint32_t lds, bool& bad) {
    const int lane = threadIdx.x & 63;
    const int page_tokens = p.tiles_per_page * 16;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const bool outside = at.page[t] < 0 || at.page[t] >= p.planes.pages;
        bad = bad || outside;
        const std::int64_t base = static_cast<std::int64_t>(outside ? 0 : at.page[t]) * p.planes.kv_heads + p.head;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            if ((2 * side + t) % ROWS != share) continue;
            const std::uint8_t* codes = (side ? p.planes.value_codes : p.planes.key_codes) + (base * page_tokens + at.inside[t]) * D;
            const __half* scales = (side ? p.planes.value_scales : p.planes.key_scales) + base * (D / 32) * page_tokens + at.inside[t];
            const std::uint32_t to = __builtin_amdgcn_readfirstlane(lds + (2 * side + t) * Step<D>::tile);
#pragma unroll
            for (int i = 0; i < Step<D>::loads - 1; ++i) {
                const int unit = 64 * i + lane, row = unit / Step<D>::units, place = unit % Step<D>::units;
                if (64 * i + 64 <= D || unit < D)
                    copy16(to + 1024 * i, codes, row * D + 16 * (place ^ Step<D>::swizzle(row)));
            }
            const std::uint32_t to_scales = __builtin_amdgcn_readfirstlane(lds + 4 * Step<D>::tile + (2 * side + t) * Step<D>::scales);
            if (D == 256 || lane < D / 4) copy4(to_scales, scales, (lane >> 3) * page_tokens * 2 + (lane & 7) * 4);
        }
    }
}

// Where the registers hold it the codes' offset is taken off by the accumulator's start; at large heads by an fma each, which
// leaves two waves on a SIMD.
template <int D>
constexpr bool kOffsetInStart = D <= 128;

// A wave's running state over its 16 query rows.
template <int D>
struct State {
    half8v query[D / 32];
    float4v start[kOffsetInStart<D> ? D / 32 : 1];  // -128 * 2^-24 sum of the group's query numbers
    float factor;                // scale * log2 e * the row's and the codes' powers of two
    int seen;                    // keys that the lane's row sees
    float reference, sum;
    float4v out[D / 16];
    float bring;                 // k: 2^(-ceil(log2 of the largest value scale so far))
};

__device__ __forceinline__ int exponent_above(float v) {  // of the smallest power of two >= v, for v > 0
    int e;
    return frexpf(v, &e) == 0.5f ? e - 1 : e;
}

// The weights of a lane's query for its eight keys; FINE: and what their rounding to fp16 left.
template <bool FINE>
struct Weights {
    half8v near;
    half8v rest;  // of FINE alone
    // Adds the products with the values ((u - 128) 2^-9) steep, the first factor exact, of the codes in byte `byte` of the words.
    __device__ __forceinline__ void multiply(const std::uint32_t (&codes)[8], int byte, const half2v (&steep)[4], float4v& sum) const {
        std::uint32_t v[4], left[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const std::uint32_t pair = permute(codes[2 * j + 1], codes[2 * j], 0x0c000c00u | byte | (4 + byte) << 16);
            const half2v up = static_cast<_Float16>(32768.0f), down = static_cast<_Float16>(-0.25f);
            const half2v code = __builtin_elementwise_fma(__builtin_bit_cast(half2v, pair), up, down);
            const half2v value = code * steep[j];
            v[j] = __builtin_bit_cast(std::uint32_t, value);
            if constexpr (FINE) left[j] = __builtin_bit_cast(std::uint32_t, __builtin_elementwise_fma(code, steep[j], -value));
        }
        const half8v values = __builtin_bit_cast(half8v, make_uint4(v[0], v[1], v[2], v[3]));
        sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(values, near, sum, 0, 0, 0);
        if constexpr (FINE) {
            const half8v lefts = __builtin_bit_cast(half8v, make_uint4(left[0], left[1], left[2], left[3]));
            sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(values, rest, sum, 0, 0, 0);
            sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(lefts, near, sum, 0, 0, 0);
        }
    }
};

// The values of a step whose scales lie far below the largest so far (other columns', or those of keys of any weight), in windows
// of 2^19 from kLeastScale down to 2^-40 (the least: 2^-24 beside 65504). The outputs go up with them and down again. Rare:
// everything is read again, so that the usual step holds nothing for it.
template <int D, bool FINE>
__device__ __forceinline__ void far_below(const unsigned char* __restrict__ step, State<D>& a, const Weights<FINE>& weights, int first_key,
                                          int length) {
#pragma unroll 1
    for (float up = 0x1p19f; up < 0x1p39f; up *= 0x1p19f) {
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane) : : "memory");  // no address of these reads is kept from one window or step to the next
        const int m = lane & 15, g = lane >> 4;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) a.out[d] *= 0x1p19f;
#pragma unroll
        for (int i = 0; i < Segments<D>::count; ++i) {
            const int columns = Segments<D>::width(i) / 16, column = Segments<D>::offset(i) + columns * m;
            half2v steep[4];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint2 scale = *reinterpret_cast<const uint2*>(step + 4 * Step<D>::tile + (2 + t) * Step<D>::scales + 32 * (column >> 5) + 8 * g);
                float x[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[r] = half_at(scale, r) * (a.bring * up);
                    if (!(x[r] >= kLeastScale && x[r] < 2.0f) || first_key + 16 * t + 4 * g + r >= length) x[r] = 0.0f;
                }
                steep[2 * t] = __builtin_bit_cast(half2v, pack(x[0] * 0x1p14f, x[1] * 0x1p14f));
                steep[2 * t + 1] = __builtin_bit_cast(half2v, pack(x[2] * 0x1p14f, x[3] * 0x1p14f));
            }
#pragma unroll
            for (int d = 0; d < columns; d += 4) {
                std::uint32_t codes[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int row = 4 * g + (j & 3);
                    const unsigned char* at = step + (2 + (j >> 2)) * Step<D>::tile + row * D + 16 * ((column >> 4) ^ Step<D>::swizzle(row)) + (column & 15) + d;
                    if (columns == 2) codes[j] = *reinterpret_cast<const unsigned short*>(at);
                    else codes[j] = *reinterpret_cast<const std::uint32_t*>(at);
                }
#pragma unroll
                for (int byte = 0; byte < 4; ++byte)
                    if (d + byte < columns) weights.multiply(codes, byte, steep, a.out[Segments<D>::tile(i) + d + byte]);
            }
        }
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d) a.out[d] *= 0x1p-38f;
}

// One step of 32 keys for the wave's rows, from LDS. FULL: every row sees all of them. FINE: weights and values in two
// fp16 terms. Returns whether values were left out for far_below().
template <int D, bool FULL, bool FINE>
__device__ __forceinline__ bool compute(const unsigned char* __restrict__ step, State<D>& a, int first_key, int length,
                                        Weights<FINE>& weights) {
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const unsigned char* key_rows = step + m * D + 8 * (g & 1);
    const unsigned char* key_scales = step + 4 * Step<D>::tile + 8 * g;
    // A tile's LDS reads before its products, and the values' before the softmax: a read costs its latency once.
    float score[8];
    uint2 codes[2][D / 32], scales[2][D / 32];
    const auto read = [&](int t) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
            codes[t][c] = *reinterpret_cast<const uint2*>(key_rows + t * Step<D>::tile + 16 * ((2 * c + (g >> 1)) ^ Step<D>::swizzle(m)));
            scales[t][c] = *reinterpret_cast<const uint2*>(key_scales + t * Step<D>::scales + 32 * c);
        }
    };
    read(0);
    if constexpr (D <= 128) read(1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        if (D > 128 && t == 1) {  // the registers hold one tile
            read(1);
            __builtin_amdgcn_sched_barrier(0);
        }
        float4v raw[D / 32];
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
            half8v keys = spread8(codes[t][c].x, codes[t][c].y);
            if constexpr (!kOffsetInStart<D>) {
                const half8v up = static_cast<_Float16>(32768.0f), down = static_cast<_Float16>(-0.25f);
                keys = __builtin_elementwise_fma(keys, up, down);  // (u - 128) 2^-9
            }
            float4v start = {0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (kOffsetInStart<D>) start = a.start[c];
            raw[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(keys, a.query[c], start, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            score[4 * t + r] = raw[0][r] * half_at(scales[t][0], r);
#pragma unroll
            for (int c = 1; c < D / 32; ++c) score[4 * t + r] = fmaf(raw[c][r], half_at(scales[t][c], r), score[4 * t + r]);
        }
    }
    std::uint32_t value[8][Segments<D>::words];
#pragma unroll
    for (int i = 0; i < Segments<D>::count; ++i) {
        const int columns = Segments<D>::width(i) / 16, column = Segments<D>::offset(i) + columns * m;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int row = 4 * g + (j & 3);
            const unsigned char* at = step + (2 + (j >> 2)) * Step<D>::tile + row * D + 16 * ((column >> 4) ^ Step<D>::swizzle(row)) + (column & 15);
            std::uint32_t* to = value[j] + Segments<D>::word(i);
            if (columns == 16) {
                const uint4 v = *reinterpret_cast<const uint4*>(at);
                to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
            } else if (columns == 8) {
                const uint2 v = *reinterpret_cast<const uint2*>(at);
                to[0] = v.x, to[1] = v.y;
            } else if (columns == 4) {
                to[0] = *reinterpret_cast<const std::uint32_t*>(at);
            } else {
                to[0] = *reinterpret_cast<const unsigned short*>(at);
            }
        }
    }
    // The largest finite scale and the least positive one, on fp16 bits: infinities and NaN wrap below the finite ones, 0 above
    // all.
    std::uint32_t value_scale[Segments<D>::count][4];
    ushort2v top_bits = {0, 0}, least_bits = {0xffff, 0xffff};
    const ushort2v finite = {0x8400, 0x8400}, one = {1, 1};
#pragma unroll
    for (int i = 0; i < Segments<D>::count; ++i) {
        const int group = (Segments<D>::offset(i) + Segments<D>::width(i) / 16 * m) >> 5;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint2 scale = *reinterpret_cast<const uint2*>(step + 4 * Step<D>::tile + (2 + t) * Step<D>::scales + 32 * group + 8 * g);
            value_scale[i][2 * t] = scale.x, value_scale[i][2 * t + 1] = scale.y;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            std::uint32_t& w = value_scale[i][j];
            // Slots past the length hold anything: their weights are 0, and so has to be what they multiply.
            const int left = length - first_key - (16 * (j >> 1) + 4 * g + 2 * (j & 1));
            if (!FULL && left < 2) w = left < 1 ? 0 : w & 0xffffu;
            const ushort2v bits = __builtin_bit_cast(ushort2v, w);
            top_bits = __builtin_elementwise_max(top_bits, bits + finite);
            least_bits = __builtin_elementwise_min(least_bits, bits - one);
        }
    }
    top_bits = __builtin_elementwise_sub_sat(top_bits, finite);
    float top_scale = half_lo(max(top_bits.x, top_bits.y));
    const float least_scale = half_lo((min(least_bits.x, least_bits.y) + 1) & 0xffff);  // 0: there is none
    bool raise = top_scale * a.bring > 1.99f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        // An infinite scale stands beside codes of 0, whose products with the rounded start may not be: NaN either way.
        score[j] = kOffsetInStart<D> ? fmaf(score[j], 0.0f, score[j] * a.factor) : score[j] * a.factor;
        if (!FULL && first_key + 16 * (j >> 2) + 4 * g + (j & 3) >= a.seen) score[j] = -__builtin_inff();
        raise = raise || score[j] > a.reference + kLazy;
    }
    if (__any(raise)) {
#pragma unroll
        for (int step = 1; step < 64; step <<= 1) top_scale = fmaxf(top_scale, __shfl_xor(top_scale, step, 64));
        float shrink = 1.0f;
        if (top_scale * a.bring > 1.0f) {
            const int e = exponent_above(top_scale);
            shrink = ldexpf(1.0f, -e - exponent_above(a.bring));
            a.bring = ldexpf(1.0f, -e);
        }
        float top = a.reference;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, score[j]);
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float keep = a.reference == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(a.reference - top);
        a.reference = top;
        a.sum *= keep;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) a.out[d] *= keep * shrink;
    }
    const float base = a.reference == -__builtin_inff() ? 0.0f : a.reference - kShift;
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        p[j] = __builtin_amdgcn_exp2f(score[j] - base);
        a.sum += p[j];
    }
    weights.near = __builtin_bit_cast(half8v, make_uint4(pack(p[0], p[1]), pack(p[2], p[3]), pack(p[4], p[5]), pack(p[6], p[7])));
    if constexpr (FINE) {
#pragma unroll
        for (int j = 0; j < 8; ++j) weights.rest[j] = static_cast<_Float16>(p[j] - static_cast<float>(weights.near[j]));
    }
    const bool narrow = __any(least_scale > 0.0f && least_scale * a.bring < kLeastScale);
    const float bring = a.bring * 0x1p14f;
#pragma unroll
    for (int i = 0; i < Segments<D>::count; ++i) {
        half2v steep[4];
        bool broken = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float x[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                x[h] = (h ? half_hi(value_scale[i][j]) : half_lo(value_scale[i][j])) * bring;
                // A row that does not see a key must not see its NaN: while rows differ, such scales are kept out of the
                // product and marked below.
                const bool mark = !FULL && !(x[h] < 0x1p15f);
                broken = broken || mark;
                if (mark || x[h] < 0x1p14f * kLeastScale) x[h] = 0.0f;
            }
            steep[j] = __builtin_bit_cast(half2v, pack(x[0], x[1]));
        }
        const int columns = Segments<D>::width(i) / 16, tile = Segments<D>::tile(i), word = Segments<D>::word(i);
#pragma unroll
        for (int d = 0; d < columns; ++d) {
            std::uint32_t codes[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) codes[j] = value[j][word + d / 4];
            weights.multiply(codes, d & 3, steep, a.out[tile + d]);
        }
        if (!FULL && __any(broken)) {
            half8v marks, sees;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const std::uint32_t w = value_scale[i][j / 2];
                marks[j] = (j & 1 ? half_hi(w) : half_lo(w)) * bring < 0x1p15f ? static_cast<_Float16>(0.0f) : static_cast<_Float16>(1.0f);
                sees[j] = first_key + 16 * (j >> 2) + 4 * g + (j & 3) < a.seen ? static_cast<_Float16>(1.0f) : static_cast<_Float16>(0.0f);
            }
            const float4v none = {0.0f, 0.0f, 0.0f, 0.0f};
            const float4v hits = __builtin_amdgcn_mfma_f32_16x16x32_f16(marks, sees, none, 0, 0, 0);
#pragma unroll
            for (int d = 0; d < columns; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (hits[r] > 0.0f) a.out[tile + d][r] = __builtin_nanf("");
        }
    }
    return narrow;
}

// The wave's 16 query rows from row `first` of the KV head's on: the loads, and what becomes of them.
template <class T, int D>
struct Queries {
    T raw[D / 32][8];
    bool live;

    __device__ __forceinline__ Queries(const T* __restrict__ q, const Geometry& g, const Work& w, int head, int first, State<D>& a) {
        const int lane = threadIdx.x & 63, m = lane & 15, lg = lane >> 4;
        const int row = first + m;
        live = row < g.rows;
        const int token = live ? row / g.group : 0;
        const T* source = q + ((static_cast<std::int64_t>(w.sequence) * g.query_tokens + token) * g.q_heads + head * g.group +
                               (live ? row - token * g.group : 0)) * g.head_dim;
        a.seen = live ? w.length - (g.query_tokens - 1 - token) : 0;
        // Unconditional: a load under a condition is waited for at once.
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
            *reinterpret_cast<uint4*>(raw[c]) = *reinterpret_cast<const uint4*>(source + min(32 * c + 8 * lg, g.head_dim - 8));
    }

    __device__ __forceinline__ void settle(const Geometry& g, State<D>& a) const {
        const int lg = (threadIdx.x & 63) >> 4;
        float x[D / 32][8], top = 0.0f;
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[c][j] = live && 32 * c + 8 * lg < g.head_dim ? to_f32(raw[c][j]) : 0.0f;
                top = fmaxf(top, fabsf(x[c][j]));
            }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        // The largest number comes to [2^14, 2^15).
        const int e = top > 0.0f && top <= 3.402823466e38f ? ilogbf(top) - 14 : 0;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
            float total = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                a.query[c][j] = static_cast<_Float16>(ldexpf(x[c][j], -e));
                total += static_cast<float>(a.query[c][j]);
            }
            if constexpr (kOffsetInStart<D>) {
                total += __shfl_xor(total, 16, 64);
                total += __shfl_xor(total, 32, 64);
                total *= -128.0f * 0x1p-24f;
                a.start[c] = float4v{total, total, total, total};
            }
        }
        // Bounded, so that no score overflows (raw sums times scales are below 2^22, at large heads 2^37). Where the bound
        // holds unequal scores, 2^-72 (2^-57) apart at least, are too far apart to share the weight with either factor.
        constexpr float kMost = kOffsetInStart<D> ? 0x1p100f : 0x1p85f;
        const float factor = ldexpf(g.scale * 1.44269504088896340736f, e + (kOffsetInStart<D> ? 24 : 9));
        a.factor = fminf(fmaxf(factor, -kMost), kMost);
        a.reference = -__builtin_inff();
        a.sum = 0.0f;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) a.out[d] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
        a.bring = 0x1p24f;
    }
};

// Partial results of a chunk: per row D outputs, then the reference and the sum.
template <int D>
constexpr int partial_floats() { return D + 2; }

template <class T, int D, int ROWS>
__global__ __launch_bounds__(kWaves * 64, 2) void kv_attention(const T* __restrict__ q, CachePlanes planes,
                                                            const std::int32_t* __restrict__ page_table,
                                                            const std::int32_t* __restrict__ lengths, T* __restrict__ out,
                                                            float* __restrict__ partial, Geometry g) {
    using S = Shape<D, ROWS>;
    constexpr bool kFine = std::is_same<T, __half>::value;
    extern __shared__ __align__(16) unsigned char memory[];
    __shared__ float references[kWaves][16], sums[kWaves][16];
    __shared__ int broken;
    Work w;
    // The head is the fast index: the same chunk of all heads, then the next.
    const int heads = g.kv_heads * g.row_blocks, flat = blockIdx.x / heads, head_and_block = blockIdx.x - flat * heads;
    if (!find_work(lengths, g, flat, w)) return;
    const int lane = threadIdx.x & 63, m = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row_wave = wave % ROWS, key_wave = wave / ROWS;
    const int head = head_and_block / g.row_blocks, block = head_and_block - head * g.row_blocks;
    if (threadIdx.x == 0) broken = 0;
    const bool bad_length = w.length < 0 || w.length > g.longest;
    const int length = bad_length ? 0 : w.length;
    const int begin = static_cast<int>(w.split * w.chunk), end = static_cast<int>(min<std::int64_t>(begin + w.chunk, length));
    const Pages pages{planes, page_table + static_cast<std::int64_t>(w.sequence) * g.max_pages, g.tiles_per_page, head, g.page_magic};
    const int last_tile = (length + 15) / 16 - 1;
    const int all_see = length - (g.query_tokens - 1);  // keys below are seen by every row
    typedef __attribute__((address_space(3))) unsigned char* Lds;
    const auto lds = static_cast<std::uint32_t>(reinterpret_cast<std::uintptr_t>((Lds)(memory)));
    bool bad = false;
    const int rounds = end > begin ? (end - begin + S::keys * kBlock - 1) / (S::keys * kBlock) : 0;
    const auto key_of = [&](int round) { return begin + (round * S::keys + key_wave) * kBlock; };
    const auto place_of = [&](int round) { return (round % S::ring) * S::round_bytes + key_wave * Step<D>::bytes; };
    const auto places = [&](int round) { return places_of(pages, key_of(round) >> 4, last_tile); };
    const auto start = [&](int round, const Places& at) { fetch<D, ROWS>(pages, at, row_wave, lds + place_of(round), bad); };
    State<D> a;
    const Queries<T, D> queries(q, g, w, head, (block * ROWS + row_wave) * 16, a);
    // The page table is read a round before its pages are (past the last round, of the last tile again).
    Places next = {};
    if (rounds) {
        Places first[S::ring];
#pragma unroll
        for (int i = 0; i < S::ring; ++i) first[i] = places(i);
#pragma unroll
        for (int i = 0; i < S::ring - 1; ++i)
            if (i < rounds) start(i, first[i]);
        next = first[S::ring - 1];
    }
    queries.settle(g, a);
    for (int i = 0; i < rounds; ++i) {
        // The wave's copies of round i are done when those of the ring - 2 rounds after it are all that is in flight.
        if (i + S::ring - 2 < rounds)
            asm volatile("s_waitcnt vmcnt(%0)" : : "i"((S::ring - 2) * S::loads) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
        // Then everybody's are, and everybody has read round i - 1, whose place the next copies take.
        if constexpr (ROWS > 1) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
        if (i + S::ring - 1 < rounds) {
            start(i + S::ring - 1, next);
            next = places(i + S::ring);
        }
        const int key = key_of(i);
        bool narrow = false;
        Weights<kFine> weights;
        if (key + kBlock <= min(all_see, end))
            narrow = compute<D, true, kFine>(memory + place_of(i), a, key, length, weights);
        else if (key < end)
            narrow = compute<D, false, kFine>(memory + place_of(i), a, key, length, weights);
        if (narrow) far_below<D, kFine>(memory + place_of(i), a, weights, key, length);
    }
    __syncthreads();
    if (bad && lane == 0) broken = 1;
    const float nan = __builtin_nanf("");
    // [wave][16][D + 4]: rows on different banks.
    auto* joined = reinterpret_cast<float*>(memory);
    float sum = a.sum;
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (lg == 0) references[wave][m] = a.reference, sums[wave][m] = sum;
    __syncthreads();
    float top = references[row_wave][m];
#pragma unroll
    for (int i = 1; i < S::keys; ++i) top = fmaxf(top, references[row_wave + i * ROWS][m]);
    // 2^-5 / bring undoes the values' power of two.
    const float keep = a.reference == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(a.reference - top);
    const float undo = keep * (0x1p-5f / a.bring);
#pragma unroll
    for (int i = 0; i < Segments<D>::count; ++i) {
        const int columns = Segments<D>::width(i) / 16;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int d = 0; d < columns; ++d)
                joined[(wave * 16 + m) * (D + 4) + Segments<D>::offset(i) + columns * (4 * lg + r) + d] = a.out[Segments<D>::tile(i) + d][r] * undo;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * 16 * D / 4; i += kWaves * 64) {
        const int r = i / (D / 4), column = (i - r * (D / 4)) * 4, row = block * ROWS * 16 + r;
        if (row >= g.rows) continue;
        const int first = r / 16, in = r % 16;
        float best = references[first][in], total = 0.0f;
#pragma unroll
        for (int j = 1; j < S::keys; ++j) best = fmaxf(best, references[first + j * ROWS][in]);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < S::keys; ++j) {
            const int from = first + j * ROWS;
            const float own = references[from][in];
            if (own != -__builtin_inff()) total += sums[from][in] * __builtin_amdgcn_exp2f(own - best);
            else if (sums[from][in] != 0.0f) total = nan;  // scores of NaN alone
            const float4 x = *reinterpret_cast<const float4*>(joined + (from * 16 + in) * (D + 4) + column);
            v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
        }
        if (broken || bad_length) total = nan;
        if (w.splits == 1) {
            const int token = row / g.group;
            T* target = out + ((static_cast<std::int64_t>(w.sequence) * g.query_tokens + token) * g.q_heads + head * g.group +
                               row - token * g.group) * g.head_dim + column;
            const float scale = 1.0f / total;
            const auto bits = [&](float x) {
                return static_cast<std::uint32_t>(__builtin_bit_cast(unsigned short, from_f32<T>(total == 0.0f ? 0.0f : x * scale)));
            };
            if (column < g.head_dim)
                *reinterpret_cast<uint2*>(target) = make_uint2(bits(v.x) | bits(v.y) << 16, bits(v.z) | bits(v.w) << 16);
        } else {
            const std::int64_t slot = static_cast<std::int64_t>(w.slot) * g.kv_heads + head;
            float* target = partial + (slot * g.rows + row) * partial_floats<D>();
            // Rows of D + 2 floats are 8-byte aligned.
            *reinterpret_cast<float2*>(target + column) = make_float2(v.x, v.y);
            *reinterpret_cast<float2*>(target + column + 2) = make_float2(v.z, v.w);
            if (column == 0) *reinterpret_cast<float2*>(target + D) = make_float2(best, total);
        }
    }
}

// Joins the partial results of a sequence of several chunks: a workgroup per query row, whose lanes take four columns each of
// as many chunks side by side as fit.
template <class T, int D>
__global__ __launch_bounds__(256) void kv_attention_join(const std::int32_t* __restrict__ lengths, T* __restrict__ out,
                                                         const float* __restrict__ partial, Geometry g) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int sequence = blockIdx.y;
    const int index = blockIdx.x;  // token * q_heads + head
    __shared__ float sums[4][5][64];
    const int length = length_at(lengths, g, 0);
    const std::int64_t chunk = chunk_length(lengths, g, length);
    const Cut cut(admitted(lengths[sequence], g), chunk);
    const int splits = cut.chunks();
    int first = 0;
    for (int base = 0; base <= sequence; base += 64) {
        const int end = whole_scan(base ? length_at(lengths, g, base) : length, g, chunk);
        first += __builtin_amdgcn_readlane(end, min(sequence - base, 63));
    }
    first -= cut.whole;
    if (splits == 1) return;
    const int token = index / g.q_heads, q_head = index - token * g.q_heads;
    const int head = q_head / g.group, row = token * g.group + q_head - head * g.group;
    const std::int64_t stride = static_cast<std::int64_t>(g.kv_heads) * g.rows * partial_floats<D>();
    const float* base = partial + (static_cast<std::int64_t>(head) * g.rows + row) * partial_floats<D>();
    const auto part = [&](int i) { return base + (i < cut.whole ? first + i : g.target + sequence) * stride; };
    constexpr int kLanes = D / 4, kSide = 64 / kLanes, kSides = 4 * kSide;  // lanes of a row; chunks side by side
    const int in_wave = lane / kLanes, side = wave * kSide + in_wave, column = (lane - in_wave * kLanes) * 4;
    float best = -__builtin_inff();
    for (int i = lane; i < splits; i += 64) best = fmaxf(best, part(i)[D]);
#pragma unroll
    for (int step = 32; step; step >>= 1) best = fmaxf(best, __shfl_xor(best, step, 64));
    float total = 0.0f, v[4] = {};
    // Loads of four chunks a lane at once; past the last chunk they repeat it, at no weight.
    for (int i = side; i < splits; i += 4 * kSides) {
        float2 low[4], high[4], end[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float* p = part(min(i + j * kSides, splits - 1));
            low[j] = *reinterpret_cast<const float2*>(p + column);
            high[j] = *reinterpret_cast<const float2*>(p + column + 2);
            end[j] = *reinterpret_cast<const float2*>(p + D);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (i + j * kSides >= splits || in_wave >= kSide) continue;
            const float keep = end[j].x == -__builtin_inff() ? (end[j].y == 0.0f ? 0.0f : __builtin_nanf(""))
                                                             : __builtin_amdgcn_exp2f(end[j].x - best);
            total += end[j].y * keep;
            v[0] += low[j].x * keep, v[1] += low[j].y * keep, v[2] += high[j].x * keep, v[3] += high[j].y * keep;
        }
    }
    // The sides' sums, in order.
    const float own[5] = {total, v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int k = 0; k < 5; ++k) sums[wave][k][lane] = own[k];
    __syncthreads();
    if (wave) return;
    float sum[5] = {};
#pragma unroll
    for (int i = 0; i < kSides; ++i)
#pragma unroll
        for (int k = 0; k < 5; ++k) sum[k] += sums[i / kSide][k][i % kSide * kLanes + lane % kLanes];
    total = sum[0], v[0] = sum[1], v[1] = sum[2], v[2] = sum[3], v[3] = sum[4];
    if (lane >= kLanes || column >= g.head_dim) return;
    const auto bits = [&](float x) {
        return static_cast<std::uint32_t>(__builtin_bit_cast(unsigned short, from_f32<T>(total == 0.0f ? 0.0f : x / total)));
    };
    T* target = out + ((static_cast<std::int64_t>(sequence) * g.query_tokens + token) * g.q_heads + q_head) * g.head_dim + column;
    *reinterpret_cast<uint2*>(target) = make_uint2(bits(v[0]) | bits(v[1]) << 16, bits(v[2]) | bits(v[3]) << 16);
}

// Row tiles of a workgroup: one wave each, the rest of its four waves take other keys.
int row_tiles(int rows) { return rows > 32 ? 4 : rows > 16 ? 2 : 1; }

// Chunks per KV head and row block that the grid aims at.
int target_chunks(int kv_heads, int row_blocks) { return std::max(1, kTarget / (kv_heads * row_blocks)); }

Geometry geometry(int sequences, int query_tokens, int q_heads, int kv_heads, int head_dim, int max_pages, int page_tokens,
                  float scale) {
    require_head_dim(head_dim);
    require(sequences > 0 && query_tokens > 0 && q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0 && max_pages > 0 &&
                page_tokens > 0 && page_tokens % 16 == 0 && page_tokens <= 4096,
            "invalid cached attention geometry");
    Geometry g;
    g.longest = static_cast<std::int64_t>(max_pages) * page_tokens;
    require(g.longest < (1ll << 31) - 4096, "a sequence's slots must fit int32");
    require(static_cast<std::int64_t>(sequences) * query_tokens * q_heads < (1ll << 31), "cached attention rows must fit int32");
    g.sequences = sequences, g.query_tokens = query_tokens, g.q_heads = q_heads, g.kv_heads = kv_heads;
    g.group = q_heads / kv_heads, g.rows = query_tokens * g.group, g.head_dim = head_dim;
    const int block = 16 * row_tiles(g.rows);
    g.row_blocks = (g.rows + block - 1) / block;
    require(static_cast<std::int64_t>(kv_heads) * g.row_blocks * (sequences + kTarget) < (1ll << 31) && sequences <= 65535,
            "cached attention takes at most 65535 sequences, and workgroups that fit int32");
    g.max_pages = max_pages, g.tiles_per_page = page_tokens / 16;
    g.page_magic = ((std::uint64_t{1} << 36) + g.tiles_per_page - 1) / g.tiles_per_page;
    g.target = target_chunks(kv_heads, g.row_blocks);
    g.scale = scale;
    return g;
}

// Slots for every chunk that could be one of several; none where no sequence can pass one chunk.
std::uint64_t partial_bytes(const Geometry& g) {
    if (g.longest <= kMinChunk) return 0;
    const std::uint64_t chunks = static_cast<std::uint64_t>(g.target) + g.sequences;
    return chunks * g.kv_heads * g.rows * ((g.head_dim + 31) / 32 * 32 + 2) * sizeof(float);
}

template <class T, int D, int ROWS>
void launch_rows(const T* q, const CachePlanes& planes, const std::int32_t* page_table, const std::int32_t* lengths, T* out,
                 float* partial, const Geometry& g, hipStream_t stream) {
    static LdsLimit limit;
    limit.raise(kv_attention<T, D, ROWS>, Shape<D, ROWS>::bytes);
    const unsigned grid = static_cast<unsigned>(g.target + g.sequences) * g.kv_heads * g.row_blocks;
    kv_attention<T, D, ROWS><<<grid, kWaves * 64, Shape<D, ROWS>::bytes, stream>>>(q, planes, page_table, lengths, out, partial, g);
}

template <class T, int D>
void launch(const void* q, const CachePlanes& planes, const std::int32_t* page_table, const std::int32_t* lengths, void* out,
            void* workspace, const Geometry& g, hipStream_t stream) {
    const auto* queries = static_cast<const T*>(q);
    auto* target = static_cast<T*>(out);
    auto* partial = static_cast<float*>(workspace);
    switch (row_tiles(g.rows)) {
        case 1: launch_rows<T, D, 1>(queries, planes, page_table, lengths, target, partial, g, stream); break;
        case 2: launch_rows<T, D, 2>(queries, planes, page_table, lengths, target, partial, g, stream); break;
        default: launch_rows<T, D, 4>(queries, planes, page_table, lengths, target, partial, g, stream); break;
    }
    check(hipGetLastError());
    if (partial_bytes(g)) {
        kv_attention_join<T, D><<<dim3(g.query_tokens * g.q_heads, g.sequences), 256, 0, stream>>>(lengths, target, partial, g);
    }
}

template <class T>
void launch_any(const void* q, const CachePlanes& planes, const std::int32_t* page_table, const std::int32_t* lengths, void* out,
                void* workspace, const Geometry& g, hipStream_t stream) {
    switch (planes.padded) {
        case 32: return launch<T, 32>(q, planes, page_table, lengths, out, workspace, g, stream);
        case 64: return launch<T, 64>(q, planes, page_table, lengths, out, workspace, g, stream);
        case 96: return launch<T, 96>(q, planes, page_table, lengths, out, workspace, g, stream);
        case 128: return launch<T, 128>(q, planes, page_table, lengths, out, workspace, g, stream);
        case 160: return launch<T, 160>(q, planes, page_table, lengths, out, workspace, g, stream);
        case 192: return launch<T, 192>(q, planes, page_table, lengths, out, workspace, g, stream);
        case 224: return launch<T, 224>(q, planes, page_table, lengths, out, workspace, g, stream);
        default: return launch<T, 256>(q, planes, page_table, lengths, out, workspace, g, stream);
    }
}

}  // namespace
}  // namespace vt

#define VT_EXPORT extern "C" __attribute__((visibility("default")))

VT_EXPORT std::uint64_t venturi_kv_attention_bytes(int sequences, int query_tokens, int q_heads, int kv_heads, int head_dim,
                                                   int max_pages, int page_tokens) {
    std::uint64_t bytes = 0;
    vt::host_guarded([&] {
        bytes = vt::partial_bytes(
            vt::geometry(sequences, query_tokens, q_heads, kv_heads, head_dim, max_pages, page_tokens, 1.0f));
    });
    return bytes;
}

VT_EXPORT int venturi_kv_attention_run(const void* q, const void* key_codes, const void* key_scales, const void* value_codes,
                                       const void* value_scales, const std::int32_t* page_table, const std::int32_t* lengths,
                                       void* out, void* workspace, std::uint64_t available, int sequences, int query_tokens,
                                       int q_heads, int kv_heads, int head_dim, int pages, int page_tokens, int max_pages,
                                       float scale, int dtype, void* stream) {
    return vt::guarded([&] {
        const auto planes = vt::cache_planes(key_codes, key_scales, value_codes, value_scales, kv_heads, head_dim, pages,
                                             page_tokens);
        const auto g = vt::geometry(sequences, query_tokens, q_heads, kv_heads, head_dim, max_pages, page_tokens, scale);
        vt::require(q && page_table && lengths && out, "null cached attention operand");
        vt::require(std::fabs(scale) <= 0x1p127f, "attention scale must be a number of at most 2^127");
        vt::require(vt::aligned(q, 16) && vt::aligned(out, 16), "cached attention rows must be 16-byte aligned");
        const std::uint64_t bytes = vt::partial_bytes(g);
        vt::require(!bytes || (workspace && available >= bytes && vt::aligned(workspace, 256)),
                    "cached attention needs its workspace, 256-byte aligned");
        const auto s = static_cast<hipStream_t>(stream);
        if (dtype == vt::kF16)
            vt::launch_any<__half>(q, planes, page_table, lengths, out, workspace, g, s);
        else if (dtype == vt::kBF16)
            vt::launch_any<__hip_bfloat16>(q, planes, page_table, lengths, out, workspace, g, s);
        else
            throw vt::Invalid("cached attention takes fp16 or bf16");
    });
}

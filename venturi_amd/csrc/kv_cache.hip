// Paged Q8 key/value cache: rotary positions with the quantizing write, and the read-back.
//
// Write: one pass over a token's projected row. Eight columns of a head are a unit (one 16-byte load); a rotated unit
// also loads its partner columns, r/2 away (the same lines, from L1). Angles: a position times a pair's rate in turns,
// which is held in two 64-bit words; the product's rounding error and the rest's share are added after the whole turns
// are gone, so that the part of a turn that is rounded to 32 bits is exact to 2^-53 at every position below 2^52. A
// workgroup computes the r/2 cosines and sines once for all heads of its token. K and V units quantize by the q8_g32_fp16 rule:
// four neighbouring lanes hold a group, two lane exchanges give its maximum.
//
// Bound by HBM, and by the launch where tokens are few. 8190 tokens, 32 heads on 8 of 128, fp16: the write 39 us (202
// MB, 5.2 TB/s; a large copy reaches 4.9; 45 us while each column chose its angle by itself), the read-back of K and V 11 us
// (51 MB, 4.6 TB/s); one token 3.4 and 2.4 us.
#include "kv_cache.hpp"

namespace vt {
namespace {

template <class T>
struct WriteArgs {
    const T* qkv;
    const std::int64_t* positions;
    const std::int64_t* slots;
    const double* rates;
    T* q;
    T* k;
    CachePlanes planes;
    int q_heads, kv_heads, head_dim, rotary_dim, interleaved;
    float factor;
};

// position * (rate + rest) less its whole turns, in [-1/2, 1/2]. The product has to be the rounded one in both places.
__device__ __forceinline__ float part_of_turn(double position, double rate, double rest) {
#pragma clang fp contract(off)
    const double turns = position * rate;
    const double part = (turns - rint(turns)) + fma(position, rest, fma(position, rate, -turns));
    return static_cast<float>(part - rint(part));
}

__device__ __forceinline__ void floats8(const float* __restrict__ from, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float4 v = reinterpret_cast<const float4*>(from)[i];
        x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
    }
}

// Eight columns at `column` of a head, rotated. `head` is the head's first column.
template <class T>
__device__ __forceinline__ void rotated(const T* __restrict__ head, int column, int rotary, int interleaved,
                                        const float* __restrict__ cosines, const float* __restrict__ sines, float (&x)[8]) {
    load8(head + column, x);
    if (column >= rotary) return;
    float y[8];
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const bool turns = column + i < rotary;
            const int pair = (column + i) >> 1;
            const float c = turns ? cosines[pair] : 1.0f, s = turns ? sines[pair] : 0.0f;
            y[i] = x[i] * c - x[i + 1] * s;
            y[i + 1] = x[i + 1] * c + x[i] * s;
        }
    } else {
        const int half = rotary >> 1;
        if ((half & 7) == 0) {  // the unit lies on one side: eight pairs in order
            const bool low = column < half;
            const int pair = low ? column : column - half;
            float partner[8], c[8], s[8];
            load8(head + (low ? column + half : pair), partner);
            floats8(cosines + pair, c);
            floats8(sines + pair, s);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = x[i] * c[i] + partner[i] * (low ? -s[i] : s[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = column + i;
                const bool turns = j < rotary, low = j < half;
                const int pair = turns ? (low ? j : j - half) : 0;
                const float partner = turns ? to_f32(head[low ? j + half : j - half]) : 0.0f;
                const float c = turns ? cosines[pair] : 1.0f, s = turns ? sines[pair] : 0.0f;
                y[i] = x[i] * c + (low ? -partner : partner) * s;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = y[i];
}

// Codes and scale of a group held by four neighbouring lanes, eight columns each.
__device__ __forceinline__ uint2 quantized(const float (&x)[8], __half& scale) {
    float top = 0.0f;
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = fabsf(x[i]);
        finite = finite && a <= 3.402823466e38f;
        top = fmaxf(top, a);
    }
    if (!finite) top = __builtin_nanf("");
    // A NaN has to reach the whole group; fmaxf would drop it.
#pragma unroll
    for (int step = 1; step <= 2; step <<= 1) {
        const float other = __shfl_xor(top, step, 64);
        top = top != top || other != other ? __builtin_nanf("") : fmaxf(top, other);
    }
    scale = from_f32<__half>(__fdiv_rn(top, 127.0f));
    const float s = __half2float(scale);
    std::uint32_t words[2] = {0x80808080u, 0x80808080u};
    if (s > 0.0f && s <= 65504.0f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int code = static_cast<int>(fminf(fmaxf(rintf(__fdiv_rn(x[i], s)), -127.0f), 127.0f));
            words[i >> 2] += static_cast<std::uint32_t>(code) << (8 * (i & 3));
        }
    }
    return make_uint2(words[0], words[1]);
}

template <class T>
__global__ __launch_bounds__(256) void kv_write(WriteArgs<T> a) {
    __shared__ __align__(16) float cosines[128], sines[128];
    const std::int64_t token = blockIdx.x;
    if (a.rotary_dim) {
        const int pairs = a.rotary_dim >> 1;
        if (static_cast<int>(threadIdx.x) < pairs) {
            const float part = part_of_turn(static_cast<double>(a.positions[token]), a.rates[threadIdx.x],
                                            a.rates[pairs + threadIdx.x]);
            float s, c;
            sincospif(2.0f * part, &s, &c);
            cosines[threadIdx.x] = a.factor * c;
            sines[threadIdx.x] = a.factor * s;
        }
        __syncthreads();
    }
    const CachePlanes& p = a.planes;
    const int d = a.head_dim, units = d >> 3, padded_units = p.padded >> 3;
    const int q_units = (a.q_heads * units + 3) & ~3, kv_units = a.kv_heads * padded_units;
    const T* row = a.qkv + token * ((a.q_heads + 2 * a.kv_heads) * static_cast<std::int64_t>(d));
    const std::int64_t slot = a.slots[token];
    const bool cached = slot >= 0 && slot < p.slots();
    for (int i = blockIdx.y * 256 + threadIdx.x; i < q_units + 2 * kv_units; i += gridDim.y * 256) {
        float x[8];
        if (i < q_units) {
            const int head = i / units, column = (i - head * units) * 8;
            if (head < a.q_heads) {
                rotated(row + head * d, column, a.rotary_dim, a.interleaved, cosines, sines, x);
                store8(a.q + (token * a.q_heads + head) * d + column, x);
            }
            continue;
        }
        const bool value = i - q_units >= kv_units;
        const int unit = i - q_units - (value ? kv_units : 0);
        const int head = unit / padded_units, column = (unit - head * padded_units) * 8;
        const T* source = row + (a.q_heads + (value ? a.kv_heads : 0) + head) * d;
        const bool inside = column < d;
        if (inside && !value) {
            rotated(source, column, a.rotary_dim, a.interleaved, cosines, sines, x);
            // The cache holds K as rounded to its type, so that a cached and a dense key differ by the quantizer alone.
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = to_f32(from_f32<T>(x[j]));
            if (a.k) store8(a.k + (token * a.kv_heads + head) * d + column, x);
        } else if (inside) {
            load8(source + column, x);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = 0.0f;
        }
        __half scale;
        const uint2 codes = quantized(x, scale);
        if (cached) {
            *reinterpret_cast<uint2*>((value ? p.value_codes : p.key_codes) + p.code_at(slot, head) + column) = codes;
            if ((column & 31) == 0) (value ? p.value_scales : p.key_scales)[p.scale_at(slot, head, column >> 5)] = scale;
        }
    }
}

template <class T>
__global__ __launch_bounds__(256) void kv_read(CachePlanes p, const std::int64_t* __restrict__ slots, T* __restrict__ keys,
                                               T* __restrict__ values, int tokens, int head_dim) {
    const int units = head_dim >> 3;
    const std::int64_t count = static_cast<std::int64_t>(tokens) * p.kv_heads * units;
    for (std::int64_t i = static_cast<std::int64_t>(blockIdx.x) * 256 + threadIdx.x; i < count;
         i += static_cast<std::int64_t>(gridDim.x) * 256) {
        const std::int64_t row = i / units, token = row / p.kv_heads;
        const int column = static_cast<int>(i - row * units) * 8, head = static_cast<int>(row - token * p.kv_heads);
        const std::int64_t slot = slots[token];
        const bool cached = slot >= 0 && slot < p.slots();
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            T* out = side ? values : keys;
            if (!out) continue;
            float x[8];
            if (cached) {
                const uint2 codes =
                    *reinterpret_cast<const uint2*>((side ? p.value_codes : p.key_codes) + p.code_at(slot, head) + column);
                const float s = __half2float((side ? p.value_scales : p.key_scales)[p.scale_at(slot, head, column >> 5)]);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    x[j] = static_cast<float>(static_cast<int>(((j < 4 ? codes.x : codes.y) >> (8 * (j & 3))) & 0xff) - 128) * s;
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = __builtin_nanf("");
            }
            store8(out + row * head_dim + column, x);
        }
    }
}

template <class T>
void launch_write(const void* qkv, const std::int64_t* positions, const std::int64_t* slots, const double* rates, void* q,
                  void* k, const CachePlanes& planes, int tokens, int q_heads, int head_dim, int rotary_dim, int interleaved,
                  float factor, hipStream_t stream) {
    const WriteArgs<T> a{static_cast<const T*>(qkv), positions, slots, rates, static_cast<T*>(q), static_cast<T*>(k), planes,
                         q_heads, planes.kv_heads, head_dim, rotary_dim, interleaved, factor};
    const int units = q_heads * (head_dim / 8) + 2 * planes.kv_heads * (planes.padded / 8);
    // Few tokens: a workgroup per 256 units, so that one token's heads run side by side; many: one workgroup per token.
    const int split = tokens < 256 ? (units + 255) / 256 : 1;
    kv_write<T><<<dim3(tokens, split), 256, 0, stream>>>(a);
}

template <class T>
void launch_read(const CachePlanes& planes, const std::int64_t* slots, void* keys, void* values, int tokens, int head_dim,
                 hipStream_t stream) {
    const std::int64_t count = static_cast<std::int64_t>(tokens) * planes.kv_heads * (head_dim / 8);
    const auto grid = static_cast<unsigned>(std::min<std::int64_t>((count + 255) / 256, 65536));
    kv_read<T><<<grid, 256, 0, stream>>>(planes, slots, static_cast<T*>(keys), static_cast<T*>(values), tokens, head_dim);
}

}  // namespace
}  // namespace vt

#define VT_EXPORT extern "C" __attribute__((visibility("default")))

VT_EXPORT int venturi_kv_write_run(const void* qkv, const std::int64_t* positions, const std::int64_t* slots,
                                   const double* rates, void* q, void* k, void* key_codes, void* key_scales,
                                   void* value_codes, void* value_scales, int tokens, int q_heads, int kv_heads, int head_dim,
                                   int rotary_dim, int interleaved, float factor, int pages, int page_tokens, int dtype,
                                   void* stream) {
    return vt::guarded([&] {
        const auto planes = vt::cache_planes(key_codes, key_scales, value_codes, value_scales, kv_heads, head_dim, pages,
                                             page_tokens);
        vt::require(qkv && slots && tokens > 0 && q_heads >= 0 && (q != nullptr) == (q_heads > 0), "invalid KV write operands");
        vt::require((q_heads + 2ll * kv_heads) * planes.padded < (1ll << 31), "a KV write row must fit int32");
        vt::require(rotary_dim >= 0 && rotary_dim <= head_dim && rotary_dim % 2 == 0 && (!rotary_dim || (positions && rates)),
                    "invalid rotary operands");
        vt::require(vt::aligned(qkv, 16) && vt::aligned(q, 16) && vt::aligned(k, 16), "KV write rows must be 16-byte aligned");
        const auto s = static_cast<hipStream_t>(stream);
        if (dtype == vt::kF16)
            vt::launch_write<__half>(qkv, positions, slots, rates, q, k, planes, tokens, q_heads, head_dim, rotary_dim,
                                     interleaved, factor, s);
        else if (dtype == vt::kBF16)
            vt::launch_write<__hip_bfloat16>(qkv, positions, slots, rates, q, k, planes, tokens, q_heads, head_dim, rotary_dim,
                                             interleaved, factor, s);
        else
            throw vt::Invalid("the KV cache takes fp16 or bf16 rows");
    });
}

VT_EXPORT int venturi_kv_read_run(const void* key_codes, const void* key_scales, const void* value_codes,
                                  const void* value_scales, const std::int64_t* slots, void* keys, void* values, int tokens,
                                  int kv_heads, int head_dim, int pages, int page_tokens, int dtype, void* stream) {
    return vt::guarded([&] {
        const auto planes = vt::cache_planes(key_codes, key_scales, value_codes, value_scales, kv_heads, head_dim, pages,
                                             page_tokens);
        vt::require(slots && (keys || values) && tokens > 0, "invalid KV read operands");
        vt::require(vt::aligned(keys, 16) && vt::aligned(values, 16), "KV read rows must be 16-byte aligned");
        const auto s = static_cast<hipStream_t>(stream);
        if (dtype == vt::kF16)
            vt::launch_read<__half>(planes, slots, keys, values, tokens, head_dim, s);
        else if (dtype == vt::kBF16)
            vt::launch_read<__hip_bfloat16>(planes, slots, keys, values, tokens, head_dim, s);
        else
            throw vt::Invalid("the KV cache takes fp16 or bf16 rows");
    });
}

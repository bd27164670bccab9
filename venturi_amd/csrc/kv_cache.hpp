// The paged Q8 key/value cache's planes, shared by its writer, its reader and the attention over it.
#pragma once

#include "common.hpp"

namespace vt {

// Codes uint8 [pages][kv_heads][page_tokens][padded], code + 128; scales fp16 [pages][kv_heads][padded / 32][page_tokens].
// Offsets are 64-bit: a cache passes 2^32 codes at 8.4M slots of 4 heads of 128.
struct CachePlanes {
    std::uint8_t* key_codes;
    __half* key_scales;
    std::uint8_t* value_codes;
    __half* value_scales;
    int kv_heads, padded, pages, page_tokens;

    __host__ __device__ std::int64_t slots() const { return static_cast<std::int64_t>(pages) * page_tokens; }
    __device__ std::int64_t code_at(std::int64_t slot, int head) const {
        const std::int64_t page = slot / page_tokens;
        return ((page * kv_heads + head) * page_tokens + (slot - page * page_tokens)) * padded;
    }
    __device__ std::int64_t scale_at(std::int64_t slot, int head, int group) const {
        const std::int64_t page = slot / page_tokens;
        return ((page * kv_heads + head) * (padded >> 5) + group) * page_tokens + (slot - page * page_tokens);
    }
};

inline void require_head_dim(int head_dim) {
    require(head_dim > 0 && head_dim % 8 == 0 && head_dim <= 256, "head_dim must be a multiple of 8 of at most 256");
}

inline CachePlanes cache_planes(const void* key_codes, const void* key_scales, const void* value_codes,
                                const void* value_scales, int kv_heads, int head_dim, int pages, int page_tokens) {
    require_head_dim(head_dim);
    require(key_codes && key_scales && value_codes && value_scales && kv_heads > 0 && pages > 0, "invalid KV cache planes");
    require(page_tokens > 0 && page_tokens % 16 == 0 && page_tokens <= 4096,
            "page_tokens must be a multiple of 16 of at most 4096");
    require(aligned(key_codes, 16) && aligned(key_scales, 16) && aligned(value_codes, 16) && aligned(value_scales, 16),
            "KV cache planes must be 16-byte aligned");
    return {static_cast<std::uint8_t*>(const_cast<void*>(key_codes)), static_cast<__half*>(const_cast<void*>(key_scales)),
            static_cast<std::uint8_t*>(const_cast<void*>(value_codes)), static_cast<__half*>(const_cast<void*>(value_scales)),
            kv_heads, (head_dim + 31) / 32 * 32, pages, page_tokens};
}

// Eight consecutive 16-bit values as fp32, and back (one rounding each).
__device__ __forceinline__ void load8(const __half* p, float (&v)[8]) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const std::uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = half_lo(u[i]);
        v[2 * i + 1] = half_hi(u[i]);
    }
}
__device__ __forceinline__ void load8(const __hip_bfloat16* p, float (&v)[8]) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const std::uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = bf16_lo(u[i]);
        v[2 * i + 1] = bf16_hi(u[i]);
    }
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    std::uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        u[i] = static_cast<std::uint32_t>(__builtin_bit_cast(unsigned short, from_f32<T>(v[2 * i]))) |
               static_cast<std::uint32_t>(__builtin_bit_cast(unsigned short, from_f32<T>(v[2 * i + 1]))) << 16;
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}

}  // namespace vt

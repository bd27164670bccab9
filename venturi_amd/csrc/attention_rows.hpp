// Attention of one query row by one wave, online softmax: the plain form of both attention operators.
#pragma once

#include "kv_cache.hpp"

namespace vt {

// Lane l scores key 64c + l (the whole dot product), the wave agrees on the new maximum, and lane l adds
// p_j v_j[l + 64 i] for the 64 keys j. `q` holds the scaled query in fp32 in LDS.
template <class Source>
__device__ __forceinline__ void attend_row(const Source& source, const float* q, int head_dim, std::int64_t seen,
                                           float (&acc)[4], float& total) {
    const int lane = threadIdx.x & 63;
    float top = -__builtin_inff();
    total = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = 0.0f;
    for (std::int64_t c = 0; c < seen; c += 64) {
        float s = -__builtin_inff();
        if (c + lane < seen) {
            s = 0.0f;
            for (int d = 0; d < head_dim; ++d) s = fmaf(q[d], source.key(c + lane, d), s);
        }
        float m = s;
#pragma unroll
        for (int step = 32; step; step >>= 1) m = fmaxf(m, __shfl_xor(m, step, 64));
        const float next = fmaxf(top, m), base = next == -__builtin_inff() ? 0.0f : next;
        const float keep = expf(top - base), p = c + lane < seen ? expf(s - base) : 0.0f;
        top = next;
        float sum = p;
#pragma unroll
        for (int step = 32; step; step >>= 1) sum += __shfl_xor(sum, step, 64);
        total = total * keep + sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] *= keep;
        const int count = static_cast<int>(seen - c < 64 ? seen - c : 64);
        for (int j = 0; j < count; ++j) {
            const float w = __shfl(p, j, 64);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (lane + 64 * i < head_dim) acc[i] = fmaf(w, source.value(c + j, lane + 64 * i), acc[i]);
        }
    }
}

template <class T>
__device__ __forceinline__ void store_row(T* out, const float (&acc)[4], float total, int head_dim) {
    const int lane = threadIdx.x & 63;
    const float scale = total != 0.0f ? 1.0f / total : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < head_dim) out[lane + 64 * i] = from_f32<T>(total == 0.0f ? 0.0f : acc[i] * scale);
}

}  // namespace vt

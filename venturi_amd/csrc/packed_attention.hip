// Causal attention over packed sequences, one wave per query row and head.
#include "attention_rows.hpp"

namespace vt {
namespace {

template <class T>
struct DenseSource {
    const T* k;
    const T* v;
    std::int64_t stride;  // elements between keys
    __device__ float key(std::int64_t j, int d) const { return to_f32(k[j * stride + d]); }
    __device__ float value(std::int64_t j, int d) const { return to_f32(v[j * stride + d]); }
};

template <class T>
__global__ __launch_bounds__(256) void packed_attention(const T* __restrict__ q, const T* __restrict__ k,
                                                        const T* __restrict__ v, const std::int32_t* __restrict__ q_offsets,
                                                        const std::int32_t* __restrict__ k_offsets, T* __restrict__ out,
                                                        int tokens, int keys, int sequences, int q_heads, int kv_heads,
                                                        int head_dim, float scale) {
    __shared__ float query[4][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const std::int64_t row = static_cast<std::int64_t>(blockIdx.x) * 4 + wave;
    if (row >= static_cast<std::int64_t>(tokens) * q_heads) return;
    const int token = static_cast<int>(row / q_heads), head = static_cast<int>(row % q_heads);
    std::int64_t first = 0, seen = 0;
    for (int b = 0; b < sequences; ++b) {
        if (token >= q_offsets[b] && token < q_offsets[b + 1]) {
            first = min(max(k_offsets[b], 0), keys);
            seen = min(max(k_offsets[b + 1], static_cast<int>(first)), keys) - first - (q_offsets[b + 1] - 1 - token);
            break;
        }
    }
    for (int d = lane; d < head_dim; d += 64) query[wave][d] = to_f32(q[row * head_dim + d]) * scale;
    const std::int64_t stride = static_cast<std::int64_t>(kv_heads) * head_dim;
    const std::int64_t offset = first * stride + head / (q_heads / kv_heads) * head_dim;
    float acc[4], total;
    attend_row(DenseSource<T>{k + offset, v + offset, stride}, query[wave], head_dim, seen, acc, total);
    store_row(out + row * head_dim, acc, total, head_dim);
}

template <class T>
void launch(const void* q, const void* k, const void* v, const std::int32_t* q_offsets, const std::int32_t* k_offsets,
            void* out, int tokens, int keys, int sequences, int q_heads, int kv_heads, int head_dim, float scale,
            hipStream_t stream) {
    const std::int64_t rows = static_cast<std::int64_t>(tokens) * q_heads;
    packed_attention<T><<<static_cast<unsigned>((rows + 3) / 4), 256, 0, stream>>>(
        static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v), q_offsets, k_offsets,
        static_cast<T*>(out), tokens, keys, sequences, q_heads, kv_heads, head_dim, scale);
}

void require_geometry(int tokens, int keys, int sequences, int q_heads, int kv_heads, int head_dim) {
    require_head_dim(head_dim);
    require(tokens > 0 && keys > 0 && sequences > 0 && q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0,
            "invalid packed attention geometry");
}

}  // namespace
}  // namespace vt

#define VT_EXPORT extern "C" __attribute__((visibility("default")))

VT_EXPORT std::uint64_t venturi_packed_attention_bytes(int tokens, int keys, int sequences, int q_heads, int kv_heads,
                                                       int head_dim) {
    vt::host_guarded([&] { vt::require_geometry(tokens, keys, sequences, q_heads, kv_heads, head_dim); });
    return 0;
}

VT_EXPORT int venturi_packed_attention_run(const void* q, const void* k, const void* v, const std::int32_t* q_offsets,
                                           const std::int32_t* k_offsets, void* out, void* workspace, std::uint64_t available,
                                           int tokens, int keys, int sequences, int q_heads, int kv_heads, int head_dim,
                                           float scale, int dtype, void* stream) {
    return vt::guarded([&] {
        vt::require_geometry(tokens, keys, sequences, q_heads, kv_heads, head_dim);
        vt::require(q && k && v && q_offsets && k_offsets && out, "null packed attention operand");
        vt::require(vt::aligned(q, 16) && vt::aligned(k, 16) && vt::aligned(v, 16) && vt::aligned(out, 16),
                    "packed attention rows must be 16-byte aligned");
        const auto s = static_cast<hipStream_t>(stream);
        if (dtype == vt::kF16)
            vt::launch<__half>(q, k, v, q_offsets, k_offsets, out, tokens, keys, sequences, q_heads, kv_heads, head_dim, scale, s);
        else if (dtype == vt::kBF16)
            vt::launch<__hip_bfloat16>(q, k, v, q_offsets, k_offsets, out, tokens, keys, sequences, q_heads, kv_heads, head_dim,
                                       scale, s);
        else
            throw vt::Invalid("packed attention takes fp16 or bf16");
    });
}

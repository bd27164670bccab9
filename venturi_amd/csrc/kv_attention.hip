// Attention over the paged Q8 cache, one wave per query row and head.
#include "attention_rows.hpp"

namespace vt {
namespace {

struct CachedSource {
    CachePlanes p;
    const std::int32_t* table;
    int head;
    __device__ std::int64_t slot(std::int64_t j) const {
        const std::int64_t at = j / p.page_tokens;
        return static_cast<std::int64_t>(table[at]) * p.page_tokens + (j - at * p.page_tokens);
    }
    __device__ float key(std::int64_t j, int d) const {
        const std::int64_t s = slot(j);
        return static_cast<float>(p.key_codes[p.code_at(s, head) + d] - 128) * __half2float(p.key_scales[p.scale_at(s, head, d >> 5)]);
    }
    __device__ float value(std::int64_t j, int d) const {
        const std::int64_t s = slot(j);
        return static_cast<float>(p.value_codes[p.code_at(s, head) + d] - 128) *
               __half2float(p.value_scales[p.scale_at(s, head, d >> 5)]);
    }
};

template <class T>
__global__ __launch_bounds__(256) void kv_attention(const T* __restrict__ q, CachePlanes planes,
                                                    const std::int32_t* __restrict__ page_table,
                                                    const std::int32_t* __restrict__ lengths, T* __restrict__ out,
                                                    int sequences, int query_tokens, int q_heads, int head_dim, int max_pages,
                                                    float scale) {
    __shared__ float query[4][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const std::int64_t row = static_cast<std::int64_t>(blockIdx.x) * 4 + wave;
    const std::int64_t token = row / q_heads;
    const int head = static_cast<int>(row - token * q_heads);
    if (token >= static_cast<std::int64_t>(sequences) * query_tokens) return;
    const std::int64_t b = token / query_tokens;
    const int length = lengths[b];
    const std::int32_t* table = page_table + b * max_pages;
    bool bad = length < 0 || length > static_cast<std::int64_t>(max_pages) * planes.page_tokens;
    if (!bad)
        for (int i = lane; i < (length + planes.page_tokens - 1) / planes.page_tokens; i += 64)
            bad |= table[i] < 0 || table[i] >= planes.pages;
    bad = __any(bad);
    for (int d = lane; d < head_dim; d += 64) query[wave][d] = to_f32(q[row * head_dim + d]) * scale;
    float acc[4], total;
    const std::int64_t seen = bad ? 0 : length - (query_tokens - 1 - (token - b * query_tokens));
    attend_row(CachedSource{planes, table, head / (q_heads / planes.kv_heads)}, query[wave], head_dim, seen, acc, total);
    if (bad) total = __builtin_nanf("");
    store_row(out + row * head_dim, acc, total, head_dim);
}

template <class T>
void launch(const void* q, const CachePlanes& planes, const std::int32_t* page_table, const std::int32_t* lengths, void* out,
            int sequences, int query_tokens, int q_heads, int head_dim, int max_pages, float scale, hipStream_t stream) {
    const std::int64_t rows = static_cast<std::int64_t>(sequences) * query_tokens * q_heads;
    kv_attention<T><<<static_cast<unsigned>((rows + 3) / 4), 256, 0, stream>>>(
        static_cast<const T*>(q), planes, page_table, lengths, static_cast<T*>(out), sequences, query_tokens, q_heads, head_dim,
        max_pages, scale);
}

void require_geometry(int sequences, int query_tokens, int q_heads, int kv_heads, int head_dim, int max_pages,
                      int page_tokens) {
    require_head_dim(head_dim);
    require(sequences > 0 && query_tokens > 0 && q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0 && max_pages > 0 &&
                page_tokens > 0 && page_tokens % 16 == 0,
            "invalid cached attention geometry");
    require(static_cast<std::int64_t>(max_pages) * page_tokens < (1ll << 31), "a sequence's slots must fit int32");
    require(static_cast<std::int64_t>(sequences) * query_tokens * q_heads < (1ll << 31), "cached attention rows must fit int32");
}

}  // namespace
}  // namespace vt

#define VT_EXPORT extern "C" __attribute__((visibility("default")))

VT_EXPORT std::uint64_t venturi_kv_attention_bytes(int sequences, int query_tokens, int q_heads, int kv_heads, int head_dim,
                                                   int max_pages, int page_tokens) {
    vt::host_guarded(
        [&] { vt::require_geometry(sequences, query_tokens, q_heads, kv_heads, head_dim, max_pages, page_tokens); });
    return 0;
}

VT_EXPORT int venturi_kv_attention_run(const void* q, const void* key_codes, const void* key_scales, const void* value_codes,
                                       const void* value_scales, const std::int32_t* page_table, const std::int32_t* lengths,
                                       void* out, void* workspace, std::uint64_t available, int sequences, int query_tokens,
                                       int q_heads, int kv_heads, int head_dim, int pages, int page_tokens, int max_pages,
                                       float scale, int dtype, void* stream) {
    return vt::guarded([&] {
        const auto planes = vt::cache_planes(key_codes, key_scales, value_codes, value_scales, kv_heads, head_dim, pages,
                                             page_tokens);
        vt::require_geometry(sequences, query_tokens, q_heads, kv_heads, head_dim, max_pages, page_tokens);
        vt::require(q && page_table && lengths && out, "null cached attention operand");
        vt::require(vt::aligned(q, 16) && vt::aligned(out, 16), "cached attention rows must be 16-byte aligned");
        const auto s = static_cast<hipStream_t>(stream);
        if (dtype == vt::kF16)
            vt::launch<__half>(q, planes, page_table, lengths, out, sequences, query_tokens, q_heads, head_dim, max_pages, scale, s);
        else if (dtype == vt::kBF16)
            vt::launch<__hip_bfloat16>(q, planes, page_table, lengths, out, sequences, query_tokens, q_heads, head_dim, max_pages,
                                       scale, s);
        else
            throw vt::Invalid("cached attention takes fp16 or bf16");
    });
}

// The residual's addition with the RMSNorm after it, and the int8 form of the norm for the A8 projections:
//
//   total = T(x + residual),  out = T((total / rms(total)) * gamma),  workspace = A8(out)  (fp16, one or two passes).
//
// Bytes are those of venturi_add_run, venturi_rms_run and venturi_q8_dp4a_quantize one after another: the statistics are the
// same 256 chains of fused multiply-adds (columns c, c + 256, ..) and the same tree over them, in 32 bits, of the rounded total.
// Bound by memory: two rows read and two written, 8 bytes a column of 16-bit rows, and 9/8 byte of codes and scales a pass.
#include "a8_group.hpp"

#include <cmath>

namespace vt {

std::uint64_t a8_bytes(int tokens, int k, int passes);

namespace {

constexpr int kChains = 256;

// x, residual and total may be the same memory: a thread reads an element before it writes it.
struct Operands {
    const void* x;
    const void* residual;
    const float* gamma;
    void* total;
    void* out;  // null: the codes alone
    std::int8_t* codes;
    float* scales;
    int tokens, k, groups, passes;
    float epsilon;
};

__device__ __forceinline__ float inverse_rms(float sum, int k, float epsilon) {
    return __fdiv_rn(1.0f, sqrt_rn(__fdiv_rn(sum, static_cast<float>(k)) + epsilon));
}

// A workgroup per row, any width and alignment: thread c runs chain c on the elements that it adds and stores, and the norm
// reads them back.
template <class T>
__global__ __launch_bounds__(kChains) void residual_rms_any(Operands o) {
    __shared__ __align__(16) float chains[kChains];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, k = o.k;
    const std::int64_t row = static_cast<std::int64_t>(blockIdx.x) * k;
    const T* x = static_cast<const T*>(o.x) + row;
    const T* residual = static_cast<const T*>(o.residual) + row;
    T* total = static_cast<T*>(o.total) + row;
    float chain = 0.0f;
    for (int col = tid; col < k; col += kChains) {
        const T h = from_f32<T>(__fadd_rn(to_f32(x[col]), to_f32(residual[col])));
        total[col] = h;
        chain = fmaf(to_f32(h), to_f32(h), chain);
    }
    chains[tid] = chain;
    __syncthreads();
    const float4 c = *reinterpret_cast<const float4*>(chains + 4 * lane);
    const float inv = inverse_rms(__shfl(canonical_sum(c.x, c.y, c.z, c.w), 0, 64), k, o.epsilon);
    T* out = o.out ? static_cast<T*>(o.out) + row : nullptr;
    if constexpr (sizeof(T) == 2) {
        if (o.passes) {
            const std::int64_t count = static_cast<std::int64_t>(o.tokens) * o.groups;
            for (int base = 256 * wave; base < 32 * o.groups; base += 1024) {
                const int col = base + 4 * lane, g = col >> 5;
                float r[4];
                bool bad = false;
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    r[v] = 0.0f;
                    if (col + v < k) {
                        const T y = from_f32<T>((to_f32(total[col + v]) * inv) * o.gamma[col + v]);
                        if (out) out[col + v] = y;
                        r[v] = to_f32(y);
                    }
                    bad |= !isfinite(r[v]);
                }
                const std::int64_t index = static_cast<std::int64_t>(blockIdx.x) * o.groups + g;
                if (g < o.groups)  // the 8 lanes of a group share g
                    quantize_group<4, 8>(r, bad, o.passes, o.codes + index * 32 + (col & 31), o.scales + index, count * 32, count,
                                         (lane & 7) == 0);
            }
            return;
        }
    }
    for (int col = tid; col < k; col += kChains) out[col] = from_f32<T>((to_f32(total[col]) * inv) * o.gamma[col]);
}

template <class T>
void launch(const Operands& o, hipStream_t stream) {
    residual_rms_any<T><<<o.tokens, kChains, 0, stream>>>(o);
}

bool meet(const void* a, std::uint64_t a_bytes, const void* b, std::uint64_t b_bytes) {
    const auto first = reinterpret_cast<std::uintptr_t>(a), second = reinterpret_cast<std::uintptr_t>(b);
    return a && b && first < second + b_bytes && second < first + a_bytes;
}

}  // namespace
}  // namespace vt

#define VT_EXPORT extern "C" __attribute__((visibility("default")))

VT_EXPORT int venturi_residual_rms_run(const void* x, const void* residual, const float* gamma, void* total, void* out,
                                       void* workspace, std::uint64_t available, int tokens, int k, int passes, int dtype,
                                       float epsilon, void* stream) {
    return vt::guarded([&] {
        vt::require(tokens > 0 && k > 0, "the residual norm needs tokens and columns");
        vt::require(x && residual && gamma && total, "null residual norm operand");
        vt::require(epsilon > 0.0f && std::isfinite(epsilon), "invalid RMSNorm epsilon");
        vt::require(dtype == vt::kF16 || dtype == vt::kBF16 || dtype == vt::kF32, "unsupported scalar type");
        vt::require(passes >= 0 && passes <= 2 && (passes == 0 || dtype == vt::kF16), "A8 takes fp16 rows in one or two passes");
        vt::require(out || passes, "the residual norm needs an output");
        const std::uint64_t size = dtype == vt::kF32 ? 4 : 2, bytes = size * tokens * static_cast<std::uint64_t>(k);
        const std::uint64_t needed = passes ? vt::a8_bytes(tokens, k, passes) : 0;
        vt::require(vt::aligned(x, size) && vt::aligned(residual, size) && vt::aligned(total, size) && vt::aligned(out, size) &&
                        vt::aligned(gamma, 4),
                    "residual norm operands must be aligned to their elements");
        vt::require(!passes || (workspace && available >= needed && vt::aligned(workspace, 16)),
                    "A8 needs its workspace, 16-byte aligned");
        if (!passes) workspace = nullptr;
        const std::uint64_t weights = 4ull * k;
        vt::require((total == x || !vt::meet(total, bytes, x, bytes)) && (total == residual || !vt::meet(total, bytes, residual, bytes)) &&
                        !vt::meet(total, bytes, gamma, weights) && !vt::meet(out, bytes, x, bytes) &&
                        !vt::meet(out, bytes, residual, bytes) && !vt::meet(out, bytes, total, bytes) &&
                        !vt::meet(out, bytes, gamma, weights) && !vt::meet(workspace, needed, x, bytes) &&
                        !vt::meet(workspace, needed, residual, bytes) && !vt::meet(workspace, needed, total, bytes) &&
                        !vt::meet(workspace, needed, out, bytes) && !vt::meet(workspace, needed, gamma, weights),
                    "residual norm outputs must not overlap other operands");
        const int groups = (k + 31) / 32;
        auto* codes = static_cast<std::int8_t*>(workspace);
        auto* scales = reinterpret_cast<float*>(codes + static_cast<std::int64_t>(tokens) * groups * 32 * passes);
        const vt::Operands o{x, residual, gamma, total, out, codes, scales, tokens, k, groups, passes, epsilon};
        const auto s = static_cast<hipStream_t>(stream);
        if (dtype == vt::kF16)
            vt::launch<__half>(o, s);
        else if (dtype == vt::kBF16)
            vt::launch<__hip_bfloat16>(o, s);
        else
            vt::launch<float>(o, s);
    });
}

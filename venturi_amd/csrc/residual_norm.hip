// The residual's addition with the RMSNorm after it, and the int8 form of the norm for the A8 projections:
//
//   total = T(x + residual),  out = T((total / rms(total)) * gamma),  workspace = A8(out)  (fp16, one or two passes).
//
// Bytes are those of venturi_add_run, venturi_rms_run and venturi_q8_dp4a_quantize one after another: the statistics are the
// same 256 chains of fused multiply-adds (columns c, c + 256, ..) and the same tree over them, in 32 bits, of the rounded total.
// Bound by memory: two rows read and two written, 8 bytes a column of 16-bit rows, and 9/8 byte of codes and scales a pass.
#include "a8_group.hpp"

#include <cmath>
#include <type_traits>

namespace vt {

std::uint64_t a8_bytes(int tokens, int k, int passes);

namespace {

constexpr int kChains = 256;
constexpr int kStaged = 60 * 1024;  // bytes of a row in LDS

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
    int first, count;  // the launch's rows
    float epsilon;
};

__device__ __forceinline__ float inverse_rms(float sum, int k, float epsilon) {
    return __fdiv_rn(1.0f, sqrt_rn(__fdiv_rn(sum, static_cast<float>(k)) + epsilon));
}

// A workgroup per row, any width and alignment: thread c runs chain c on the elements that it adds and stores, and the norm
// reads them back. One element at a time: 8190 rows of 5120 off 16 bytes 111 us where staged ones take 62, 2048 of 16384 fp32
// columns 147 (a copy's rate: 106), 61 of 32768 bf16 columns 68 where the add and the norm apart take 29.
template <class T>
__global__ __launch_bounds__(kChains) void residual_rms_any(Operands o) {
    __shared__ __align__(16) float chains[kChains];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, k = o.k;
    const int token = o.first + blockIdx.x;
    const std::int64_t row = static_cast<std::int64_t>(token) * k;
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
                const std::int64_t index = static_cast<std::int64_t>(token) * o.groups + g;
                if (g < o.groups)  // the 8 lanes of a group share g
                    quantize_group<4, 8>(r, bad, o.passes, o.codes + index * 32 + (col & 31), o.scales + index, count * 32, count,
                                         (lane & 7) == 0);
            }
            return;
        }
    }
    for (int col = tid; col < k; col += kChains) out[col] = from_f32<T>((to_f32(total[col]) * inv) * o.gamma[col]);
}

// Four 16-bit values as f32.
template <class T>
__device__ __forceinline__ void unpack4(const uint2& w, float (&v)[4]) {
    const unsigned short h[4] = {static_cast<unsigned short>(w.x), static_cast<unsigned short>(w.x >> 16),
                                 static_cast<unsigned short>(w.y), static_cast<unsigned short>(w.y >> 16)};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = to_f32(__builtin_bit_cast(T, h[i]));
}
template <class T>
__device__ __forceinline__ uint2 pack4(const T (&v)[4]) {
    uint2 w;
    __builtin_memcpy(&w, v, sizeof(w));
    return w;
}

// A wave per row of 16-bit values that stays in registers: P pieces of 256 columns, four neighbouring ones a lane, which are
// chains 4 lane .. 4 lane + 3, so that no value leaves its lane before the tree.
template <class T, int P>
__global__ __launch_bounds__(256) void residual_rms_wave(Operands o) {
    const int lane = threadIdx.x & 63, k = o.k;
    const int in_launch = blockIdx.x * 4 + (threadIdx.x >> 6), token = o.first + in_launch;
    if (in_launch >= o.count) return;
    const std::int64_t row = static_cast<std::int64_t>(token) * k;
    const T* x = static_cast<const T*>(o.x) + row;
    const T* residual = static_cast<const T*>(o.residual) + row;
    T* total = static_cast<T*>(o.total) + row;
    uint2 h[P], r[P];
#pragma unroll
    for (int j = 0; j < P; ++j) {
        const int col = min(256 * j + 4 * lane, k - 4);
        h[j] = *reinterpret_cast<const uint2*>(x + col);
        r[j] = *reinterpret_cast<const uint2*>(residual + col);
    }
    float chain[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < P; ++j) {
        const int col = 256 * j + 4 * lane;
        float a[4], b[4];
        unpack4<T>(h[j], a);
        unpack4<T>(r[j], b);
        T sum[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) sum[v] = from_f32<T>(__fadd_rn(a[v], b[v]));
        h[j] = pack4(sum);
        if (col >= k) h[j] = make_uint2(0, 0);  // adds nothing to a chain
        else *reinterpret_cast<uint2*>(total + col) = h[j];
        unpack4<T>(h[j], a);
#pragma unroll
        for (int v = 0; v < 4; ++v) chain[v] = fmaf(a[v], a[v], chain[v]);
    }
    const float inv = inverse_rms(__shfl(canonical_sum(chain[0], chain[1], chain[2], chain[3]), 0, 64), k, o.epsilon);
    T* out = o.out ? static_cast<T*>(o.out) + row : nullptr;
    const std::int64_t count = static_cast<std::int64_t>(o.tokens) * o.groups;
#pragma unroll
    for (int j = 0; j < P; ++j) {
        const int col = 256 * j + 4 * lane;
        const float4 g = *reinterpret_cast<const float4*>(o.gamma + min(col, k - 4));
        float a[4];
        unpack4<T>(h[j], a);
        const T y[4] = {from_f32<T>((a[0] * inv) * g.x), from_f32<T>((a[1] * inv) * g.y), from_f32<T>((a[2] * inv) * g.z),
                        from_f32<T>((a[3] * inv) * g.w)};
        if (out && col < k) *reinterpret_cast<uint2*>(out + col) = pack4(y);
        if (o.passes) {
            float q[4];
            bool bad = false;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                q[v] = col < k ? to_f32(y[v]) : 0.0f;
                bad |= !isfinite(q[v]);
            }
            const std::int64_t index = static_cast<std::int64_t>(token) * o.groups + (col >> 5);
            if ((col >> 5) < o.groups)  // the 8 lanes of a group share it
                quantize_group<4, 8>(q, bad, o.passes, o.codes + index * 32 + (col & 31), o.scales + index, count * 32, count,
                                     (lane & 7) == 0);
        }
    }
}

typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));

// A workgroup per row that it stages in LDS: the row comes in one round of loads, and all threads share its columns but for
// the chains. The tensors start at multiples of 16 bytes, and with ROUND so do the rows; else a row's first and last vector
// are partial, and its LDS copy starts as far into a vector as the row does.
template <class T, int THREADS, bool ROUND>
__global__ __launch_bounds__(THREADS) void residual_rms_staged(Operands o) {
    constexpr int V = 16 / sizeof(T);
    extern __shared__ uint4 staged[];
    __shared__ __align__(16) float chains[kChains];
    const int tid = threadIdx.x, lane = tid & 63, k = o.k;
    const int token = o.first + blockIdx.x;
    const std::int64_t row = static_cast<std::int64_t>(token) * k;
    const int shift = ROUND ? 0 : static_cast<int>(row % V), pieces = (k + shift + V - 1) / V;
    auto* held = reinterpret_cast<T*>(staged) + shift;
    const T* x = static_cast<const T*>(o.x) + row;
    const T* residual = static_cast<const T*>(o.residual) + row;
    T* total = static_cast<T*>(o.total) + row;
    for (int p = tid; p < pieces; p += THREADS) {
        const int first = V * p - shift;
        if (ROUND || (first >= 0 && first + V <= k)) {
            const uint4 a = *reinterpret_cast<const uint4*>(x + first), b = *reinterpret_cast<const uint4*>(residual + first);
            T u[V], v[V];
            __builtin_memcpy(u, &a, sizeof(a));
            __builtin_memcpy(v, &b, sizeof(b));
#pragma unroll
            for (int i = 0; i < V; ++i) u[i] = from_f32<T>(__fadd_rn(to_f32(u[i]), to_f32(v[i])));
            uint4 h;
            __builtin_memcpy(&h, u, sizeof(h));
            *reinterpret_cast<uint4*>(total + first) = h;
            staged[p] = h;
        } else {
            for (int col = max(first, 0); col < min(first + V, k); ++col) {
                const T h = from_f32<T>(__fadd_rn(to_f32(x[col]), to_f32(residual[col])));
                total[col] = h;
                held[col] = h;
            }
        }
    }
    __syncthreads();
    if (THREADS == kChains || tid < kChains) {
        float chain = 0.0f;
#pragma unroll 8
        for (int col = tid; col < k; col += kChains) chain = fmaf(to_f32(held[col]), to_f32(held[col]), chain);
        chains[tid] = chain;
    }
    __syncthreads();
    const float4 c = *reinterpret_cast<const float4*>(chains + 4 * lane);
    const float inv = inverse_rms(__shfl(canonical_sum(c.x, c.y, c.z, c.w), 0, 64), k, o.epsilon);
    T* out = o.out ? static_cast<T*>(o.out) + row : nullptr;
    if constexpr (sizeof(T) == 2) {
        if (o.passes) {
            const std::int64_t count = static_cast<std::int64_t>(o.tokens) * o.groups;
            for (int col = 4 * tid; col < 32 * o.groups; col += 4 * THREADS) {
                float q[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                bool bad = false;
                if (ROUND && col < k) {
                    const float4 g = *reinterpret_cast<const float4*>(o.gamma + col);
                    unpack4<T>(*reinterpret_cast<const uint2*>(held + col), q);
                    const T y[4] = {from_f32<T>((q[0] * inv) * g.x), from_f32<T>((q[1] * inv) * g.y), from_f32<T>((q[2] * inv) * g.z),
                                    from_f32<T>((q[3] * inv) * g.w)};
                    if (out) *reinterpret_cast<uint2*>(out + col) = pack4(y);
#pragma unroll
                    for (int v = 0; v < 4; ++v) q[v] = to_f32(y[v]);
                } else if (!ROUND) {
#pragma unroll
                    for (int v = 0; v < 4; ++v)
                        if (col + v < k) {
                            const T y = from_f32<T>((to_f32(held[col + v]) * inv) * o.gamma[col + v]);
                            if (out) out[col + v] = y;
                            q[v] = to_f32(y);
                        }
                }
#pragma unroll
                for (int v = 0; v < 4; ++v) bad |= !isfinite(q[v]);
                const std::int64_t index = static_cast<std::int64_t>(token) * o.groups + (col >> 5);
                quantize_group<4, 8>(q, bad, o.passes, o.codes + index * 32 + (col & 31), o.scales + index, count * 32, count,
                                     (lane & 7) == 0);  // the 8 lanes of a group share it
            }
            return;
        }
    }
    for (int p = tid; p < pieces; p += THREADS) {
        const int first = V * p - shift;
        if (ROUND || (first >= 0 && first + V <= k)) {
            const uint4 h = staged[p];
            T u[V];
            __builtin_memcpy(u, &h, sizeof(h));
#pragma unroll
            for (int i = 0; i < V; i += 4) {
                const float4u g = *reinterpret_cast<const float4u*>(o.gamma + first + i);
                u[i] = from_f32<T>((to_f32(u[i]) * inv) * g[0]);
                u[i + 1] = from_f32<T>((to_f32(u[i + 1]) * inv) * g[1]);
                u[i + 2] = from_f32<T>((to_f32(u[i + 2]) * inv) * g[2]);
                u[i + 3] = from_f32<T>((to_f32(u[i + 3]) * inv) * g[3]);
            }
            uint4 y;
            __builtin_memcpy(&y, u, sizeof(y));
            *reinterpret_cast<uint4*>(out + first) = y;
        } else {
            for (int col = max(first, 0); col < min(first + V, k); ++col) out[col] = from_f32<T>((to_f32(held[col]) * inv) * o.gamma[col]);
        }
    }
}

template <class T>
void launch(const Operands& o, hipStream_t stream) {
    if constexpr (sizeof(T) == 2) {
        // Short rows leave most of a workgroup idle (us, wave against workgroup, fp16 without codes / with two passes: 512
        // tokens of 256 2.6 / 3.5 against 2.9 / 3.6; 2048 of 1024 5.5 / 9.5 against 6.2 / 9.3; 60000 of 1024 88 / 123 against
        // 96 / 142, of 512 46 / 66 against 67 / 93; but 512 of 1024 3.6 / 6.8 against 3.4 / 4.3).
        const bool wave = o.k <= 256 || (o.k <= 1024 && o.tokens >= 2048);
        if (wave && o.k % 4 == 0 && aligned(o.x, 8) && aligned(o.residual, 8) && aligned(o.total, 8) && aligned(o.out, 8) &&
            aligned(o.gamma, 16)) {
            const auto grid = static_cast<unsigned>((o.count + 3) / 4);
            if (o.k <= 256) residual_rms_wave<T, 1><<<grid, 256, 0, stream>>>(o);
            else if (o.k <= 512) residual_rms_wave<T, 2><<<grid, 256, 0, stream>>>(o);
            else residual_rms_wave<T, 4><<<grid, 256, 0, stream>>>(o);
            return;
        }
    }
    // Few rows are as fast as a row's threads are many; many rows as the CU is full (us, 1024 / 512 / 256 threads, fp16 without
    // codes: 61 tokens of 5120 3.9 / 4.1 / 4.8; 600 9.0 / 8.1 / 7.8; 2048 17.3 / 15.9 / 15.2; 8190 66 / 63 / 65; with two
    // passes 61: 5.2 / 6.3 / 8.5; 600: 12.6 / 12.6 / 13.1; 8190: 101 / 90 / 91).
    const std::int64_t bytes = static_cast<std::int64_t>(o.k) * sizeof(T);
    if (bytes > kStaged || !(aligned(o.x, 16) && aligned(o.residual, 16) && aligned(o.total, 16) && aligned(o.out, 16) && aligned(o.gamma, 16))) {
        residual_rms_any<T><<<o.count, kChains, 0, stream>>>(o);
        return;
    }
    const auto staged = [&](auto round) {
        constexpr bool R = decltype(round)::value;
        const auto lds = static_cast<std::size_t>(bytes + 31) / 16 * 16;  // and what comes before the row in its first vector
        if (o.k > 2048 && o.tokens <= 256) residual_rms_staged<T, 1024, R><<<o.count, 1024, lds, stream>>>(o);
        else if (o.k > 2048) residual_rms_staged<T, 512, R><<<o.count, 512, lds, stream>>>(o);
        else residual_rms_staged<T, kChains, R><<<o.count, kChains, lds, stream>>>(o);
    };
    if (bytes % 16 == 0) staged(std::true_type{});
    else staged(std::false_type{});
}

}  // namespace
}  // namespace vt

#define VT_EXPORT extern "C" __attribute__((visibility("default")))

VT_EXPORT int venturi_residual_rms_run(const void* x, const void* residual, const float* gamma, void* total, void* out,
                                       void* workspace, std::uint64_t available, int tokens, int k, int passes, int dtype,
                                       float epsilon, void* stream) {
    return vt::guarded([&] {
        vt::require(tokens > 0 && k > 0, "the residual norm needs tokens and columns");
        vt::require(k <= INT32_MAX - 1024, "the residual norm counts columns, a workgroup's step past the last, in 32 bits");
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
        const auto s = static_cast<hipStream_t>(stream);
        // A launch takes 2^21 rows: its threads are counted in 32 bits.
        for (std::int64_t first = 0; first < tokens; first += 1 << 21) {
            const int count = static_cast<int>(std::min<std::int64_t>(tokens - first, 1 << 21));
            const vt::Operands o{x, residual, gamma, total, out, codes, scales, tokens, k, groups, passes, static_cast<int>(first), count, epsilon};
            if (dtype == vt::kF16)
                vt::launch<__half>(o, s);
            else if (dtype == vt::kBF16)
                vt::launch<__hip_bfloat16>(o, s);
            else
                vt::launch<float>(o, s);
            vt::check(hipGetLastError());
        }
    });
}

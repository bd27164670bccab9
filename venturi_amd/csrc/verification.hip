// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Draft i of a sequence stands while u_i q_i(d_i) < p_i(d_i) (q = 1 for certain drafts): both sides are products of 32-bit
// numbers, exact in 64 bits. After the first refusal the next token comes from max(p - q, 0) of that row (of certain drafts:
// p without the draft), where that has a mass, else from p; after the last draft from p of the row behind it. It is the first
// token, by index, at which the running sum passes u times the whole one; sums in 64 bits, in a fixed order.
//
// Bound by memory: one or two rows of 4-byte probabilities a sequence. A row is cut into parts that workgroups sum; one
// workgroup of a second launch finds the part and goes through it again.
#include "common.hpp"

#include <climits>

namespace vt {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxDrafts = 64, kMaxParts = 64, kMaxVocab = 1 << 20, kMaxSequences = 65535;

struct Operands {
    const float* target;          // [sequences][drafts + 1][vocab]
    const float* proposal;        // [sequences][drafts][vocab], or null: certain drafts
    const std::int64_t* drafted;  // [sequences][drafts]
    const std::int32_t* counts;   // [sequences], or null: all drafts
    const float* uniforms;        // [sequences][drafts + 1]
    std::int64_t* tokens;         // [sequences][drafts + 1]
    std::int32_t* accepted;       // [sequences]
    double2* sums;                // [sequences][parts]: of the remainder, and of the target's row
    int drafts, vocab, parts, slice;
};

// The row that a sequence's last token comes from.
struct Draw {
    const float* p;
    const float* q;  // null: nothing is taken off
    int without;     // a refused certain draft, or -1
    int accepted;
};

// What is no positive finite number is 0.
__device__ __forceinline__ double positive(float p) { return p > 0.0f && p <= 3.402823466e38f ? static_cast<double>(p) : 0.0; }

// For a whole wave.
__device__ __forceinline__ Draw draw_of(const Operands& o, int sequence) {
    const int lane = threadIdx.x & 63;
    const int count = o.counts ? min(max(o.counts[sequence], 0), o.drafts) : o.drafts;
    const std::int64_t first = static_cast<std::int64_t>(sequence) * o.drafts;  // of the sequence's drafts
    bool refused = false;
    int token = -1;
    if (lane < count) {
        const std::int64_t id = o.drafted[first + lane];
        refused = true;
        if (id >= 0 && id < o.vocab) {
            token = static_cast<int>(id);
            const double p = positive(o.target[(first + sequence + lane) * o.vocab + id]);
            const double q = o.proposal ? o.proposal[(first + lane) * o.vocab + id] : 1.0;
            refused = !(o.uniforms[first + sequence + lane] * q < p);
        }
    }
    const unsigned long long bad = __ballot(refused);
    Draw d;
    d.accepted = bad ? __ffsll(bad) - 1 : count;
    d.p = o.target + (first + sequence + d.accepted) * o.vocab;
    d.q = bad && o.proposal ? o.proposal + (first + d.accepted) * o.vocab : nullptr;
    d.without = bad && !o.proposal ? __shfl(token, d.accepted, 64) : -1;
    return d;
}

// A token's share of the remainder and of the target's row.
__device__ __forceinline__ double2 share(const Draw& d, int index) {
    double2 s;
    s.y = positive(d.p[index]);
    s.x = index == d.without ? 0.0 : s.y;
    if (d.q) {
        const double left = s.y - static_cast<double>(d.q[index]);
        s.x = left > 0.0 ? left : 0.0;
    }
    return s;
}

__device__ __forceinline__ double wave_scan(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int step = 1; step < 64; step <<= 1) {
        const double below = __shfl_up(v, step, 64);
        if (lane >= step) v += below;
    }
    return v;
}

// Inclusive scan over the workgroup's threads, in order. `waves` is LDS of kWaves doubles.
__device__ __forceinline__ double block_scan(double v, double* waves) {
    const int wave = threadIdx.x >> 6;
    v = wave_scan(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) waves[wave] = v;
    __syncthreads();
    double before = 0.0;
    for (int i = 0; i < wave; ++i) before += waves[i];
    return v + before;
}

// Sums of a part.
__global__ __launch_bounds__(kThreads) void verify_sum(Operands o) {
    __shared__ double waves[kWaves];
    const int sequence = blockIdx.y, part = blockIdx.x;
    const Draw d = draw_of(o, sequence);
    const int begin = part * o.slice, end = min(begin + o.slice, o.vocab);
    double2 sum = {0.0, 0.0};
    for (int i = begin + threadIdx.x; i < end; i += kThreads) {
        const double2 s = share(d, i);
        sum.x += s.x, sum.y += s.y;
    }
    sum.x = block_scan(sum.x, waves);
    sum.y = block_scan(sum.y, waves);
    if (threadIdx.x == kThreads - 1) o.sums[static_cast<std::int64_t>(sequence) * o.parts + part] = sum;
}

// The sequence's tokens. A workgroup per sequence; with one part it sums the row itself.
__global__ __launch_bounds__(kThreads) void verify_take(Operands o) {
    __shared__ double waves[kWaves];
    __shared__ int found, last;
    const int sequence = blockIdx.x, lane = threadIdx.x & 63;
    const Draw d = draw_of(o, sequence);
    const std::int64_t row = static_cast<std::int64_t>(sequence) * (o.drafts + 1);
    for (int i = threadIdx.x; i <= o.drafts; i += kThreads)
        if (i != d.accepted) o.tokens[row + i] = i < d.accepted ? o.drafted[row - sequence + i] : -1;
    if (threadIdx.x == 0) o.accepted[sequence] = d.accepted, found = INT_MAX, last = -1;
    const double u = o.uniforms[row + o.drafts];
    int begin = 0, end = o.vocab;
    double before = 0.0, target = 0.0;
    bool rest = true;  // draw from the remainder
    if (o.parts > 1) {
        // Every wave looks for the part on its own.
        const double2 none = {0.0, 0.0};
        const double2 own = lane < o.parts ? o.sums[static_cast<std::int64_t>(sequence) * o.parts + lane] : none;
        const double2 scan = {wave_scan(own.x), wave_scan(own.y)};
        rest = __shfl(scan.x, 63, 64) > 0.0;
        const double mine = rest ? own.x : own.y, sum = rest ? scan.x : scan.y;
        target = u * __shfl(sum, 63, 64);
        const unsigned long long some = __ballot(mine > 0.0), past = __ballot(mine > 0.0 && sum > target);
        const int part = past ? __ffsll(past) - 1 : some ? 63 - __clzll(some) : 0;
        const double up = __shfl_up(sum, 1, 64);
        before = __shfl(lane ? up : 0.0, part, 64);
        begin = part * o.slice;
        end = min(begin + o.slice, o.vocab);
    }
    // A thread's run of tokens.
    const int run = (end - begin + kThreads - 1) / kThreads;
    const int first = begin + static_cast<int>(threadIdx.x) * run, stop = min(first + run, end);
    double2 sum = {0.0, 0.0};
    for (int i = first; i < stop; ++i) {
        const double2 s = share(d, i);
        sum.x += s.x, sum.y += s.y;
    }
    const double scan_x = block_scan(sum.x, waves);
    double all = 0.0;
    for (int i = 0; i < kWaves; ++i) all += waves[i];
    const double scan_y = block_scan(sum.y, waves);
    if (o.parts == 1) {
        double whole = 0.0;
        for (int i = 0; i < kWaves; ++i) whole += waves[i];
        rest = all > 0.0;
        target = u * (rest ? all : whole);
    }
    double at = before + (rest ? scan_x - sum.x : scan_y - sum.y);
    for (int i = first; i < stop; ++i) {
        const double2 s = share(d, i);
        const double w = rest ? s.x : s.y;
        at += w;
        if (w > 0.0) {
            atomicMax(&last, i);
            if (at > target) {
                atomicMin(&found, i);
                break;
            }
        }
    }
    __syncthreads();
    // Where no sum passes the target (a uniform of 1, or a last rounding) it is the last token with a share.
    if (threadIdx.x == 0) o.tokens[row + d.accepted] = found != INT_MAX ? found : last;
}

Operands geometry(int sequences, int drafts, int vocab) {
    require(sequences > 0 && sequences <= kMaxSequences, "verification takes 1 to 65535 sequences");
    require(drafts > 0 && drafts <= kMaxDrafts, "verification takes 1 to 64 drafts of a sequence");
    require(vocab > 0 && vocab <= kMaxVocab, "verification takes a vocabulary of at most 1048576");
    // Parts of 2048 tokens and more, about 2048 workgroups in all.
    const int parts = std::max(std::min({kMaxParts, 2048 / sequences, vocab / 2048}), 1);
    Operands o{};
    o.drafts = drafts, o.vocab = vocab, o.parts = parts, o.slice = (vocab + parts - 1) / parts;
    return o;
}

std::uint64_t sum_bytes(const Operands& o, int sequences) {
    return o.parts > 1 ? sizeof(double2) * static_cast<std::uint64_t>(o.parts) * sequences : 0;
}

}  // namespace
}  // namespace vt

#define VT_EXPORT extern "C" __attribute__((visibility("default")))

VT_EXPORT std::uint64_t venturi_verify_bytes(int sequences, int drafts, int vocab) {
    std::uint64_t bytes = 0;
    vt::host_guarded([&] { bytes = vt::sum_bytes(vt::geometry(sequences, drafts, vocab), sequences); });
    return bytes;
}

VT_EXPORT int venturi_verify_run(const float* target, const float* proposal, const std::int64_t* drafted, const std::int32_t* counts,
                                 const float* uniforms, std::int64_t* tokens, std::int32_t* accepted, void* workspace,
                                 std::uint64_t available, int sequences, int drafts, int vocab, void* stream) {
    return vt::guarded([&] {
        auto o = vt::geometry(sequences, drafts, vocab);
        vt::require(target && drafted && uniforms && tokens && accepted, "null verification operand");
        vt::require(vt::aligned(target, 4) && vt::aligned(proposal, 4) && vt::aligned(drafted, 8) && vt::aligned(counts, 4) &&
                        vt::aligned(uniforms, 4) && vt::aligned(tokens, 8) && vt::aligned(accepted, 4),
                    "verification operands must be aligned to their elements");
        const std::uint64_t bytes = vt::sum_bytes(o, sequences);
        vt::require(!bytes || (workspace && available >= bytes && vt::aligned(workspace, 256)),
                    "verification needs its workspace, 256-byte aligned");
        o.target = target, o.proposal = proposal, o.drafted = drafted, o.counts = counts, o.uniforms = uniforms;
        o.tokens = tokens, o.accepted = accepted, o.sums = static_cast<double2*>(workspace);
        const auto s = static_cast<hipStream_t>(stream);
        if (o.parts > 1) {
            vt::verify_sum<<<dim3(o.parts, sequences), vt::kThreads, 0, s>>>(o);
            vt::check(hipGetLastError());
        }
        vt::verify_take<<<sequences, vt::kThreads, 0, s>>>(o);
    });
}

// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Draft i of a sequence stands while u_i q_i(d_i) < p_i(d_i) (q = 1 for certain drafts): both sides are products of 32-bit
// numbers, exact in 64 bits. After the first refusal the next token comes from max(p - q, 0) of that row (of certain drafts:
// p without the draft), where that has a mass, else from p; after the last draft from p of the row behind it. It is the first
// token, by index, at which the running sum passes u times the whole one; sums in 64 bits, in a fixed order.
//
// Bound by memory where sequences are many: one or two rows of 4-byte probabilities each (128 of 151936 tokens with a drafter's
// rows 33.4 us, 4.7 TB/s), else by two launches and their chains of loads: the drafts, their probabilities, the row, and
// in the second launch the sums, the part, and the run of it again (one sequence of 248320 tokens 8.6, 61 of 32003 11.4). A row
// is cut into parts that workgroups sum; one workgroup of the second launch finds the part and the token in it. (The chosen
// part token by token, a run a thread: 82.6, 20.2 and 16.6.)
#include "common.hpp"

namespace vt {
namespace {

constexpr int kMaxDrafts = 64, kMaxParts = 64, kMaxVocab = 1 << 20, kMaxSequences = 65535;

// What a sequence's drafts came to.
struct Verdict {
    int accepted;
    int refused;  // the next token comes from what is left of the target's row
    int without;  // a refused certain draft, or -1
    int unused;
};

struct Operands {
    const float* target;          // [sequences][drafts + 1][vocab]
    const float* proposal;        // [sequences][drafts][vocab], or null: certain drafts
    const std::int64_t* drafted;  // [sequences][drafts]
    const std::int32_t* counts;   // [sequences], or null: all drafts
    const float* uniforms;        // [sequences][drafts + 1]
    std::int64_t* tokens;         // [sequences][drafts + 1]
    std::int32_t* accepted;       // [sequences]
    Verdict* verdicts;            // [sequences], where rows are summed in parts
    double2* sums;                // [sequences][parts]: of the remainder, and of the target's row
    int drafts, vocab, parts, slice;
};

// What is no positive finite number is 0.
__device__ __forceinline__ float positive(float p) { return p > 0.0f && p <= 3.402823466e38f ? p : 0.0f; }

// For a whole wave. What the drafts are looked up by comes in one round of loads, their probabilities in a second.
__device__ __forceinline__ Verdict verdict_of(const Operands& o, int sequence) {
    const int lane = threadIdx.x & 63, draft = min(lane, o.drafts - 1);
    const std::int64_t first = static_cast<std::int64_t>(sequence) * o.drafts;  // of the sequence's drafts
    const std::int32_t* counts = o.counts ? o.counts + sequence : nullptr;
    const std::int64_t id = o.drafted[first + draft];
    const double u = o.uniforms[first + sequence + draft];
    const int count = counts ? min(max(*counts, 0), o.drafts) : o.drafts;
    const bool there = id >= 0 && id < o.vocab;
    const int token = there ? static_cast<int>(id) : -1;
    const std::int64_t at = there ? id : 0;
    const double p = positive(o.target[(first + sequence + draft) * o.vocab + at]);
    const double q = o.proposal ? o.proposal[(first + draft) * o.vocab + at] : 1.0;
    const unsigned long long bad = __ballot(lane < count && !(there && u * q < p));
    const int accepted = bad ? __ffsll(bad) - 1 : count;
    return {accepted, bad != 0, bad && !o.proposal ? __shfl(token, accepted, 64) : -1, 0};
}

// Rows start at any multiple of 4 bytes.
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));

// The row that a sequence's last token comes from.
struct Draw {
    const float* p;
    const float* q;  // null: nothing is taken off
    int without, vocab;

    __device__ __forceinline__ Draw(const Operands& o, const Verdict& v, int sequence) : without(v.without), vocab(o.vocab) {
        const std::int64_t first = static_cast<std::int64_t>(sequence) * o.drafts;
        p = o.target + (first + sequence + v.accepted) * o.vocab;
        q = v.refused && o.proposal ? o.proposal + (first + v.accepted) * o.vocab : nullptr;
    }
    // Where four tokens from `at` on are loaded from: the last four of the row may come in their place.
    __device__ __forceinline__ int place(int at) const { return max(min(at, vocab - 4), 0); }
    __device__ __forceinline__ float4u load(const float* row, int at) const {
        if (vocab >= 4) return *reinterpret_cast<const float4u*>(row + at);
        return float4u{row[0], row[min(1, vocab - 1)], row[min(2, vocab - 1)], 0.0f};
    }
    // Shares of the loaded tokens in the remainder (x) and in the target's row (y), of those from `at` up to `end`.
    __device__ __forceinline__ double2 share(const float4u& pv, const float4u& qv, int j, int at, int end) const {
        const int index = place(at) + j;
        double2 s;
        s.y = index >= at && index < end ? static_cast<double>(positive(pv[j])) : 0.0;
        s.x = q ? fmax(s.y - static_cast<double>(qv[j]), 0.0) : index == without ? 0.0 : s.y;
        if (!(s.y > 0.0)) s.x = 0.0;  // of a proposal below 0, too
        return s;
    }
};

template <int CONTROL, int ROWS>
__device__ __forceinline__ double moved(double v) {
    const auto w = __builtin_bit_cast(std::uint64_t, v);
    const auto lo = static_cast<std::uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(w), CONTROL, ROWS, 0xf, true));
    const auto hi = static_cast<std::uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(w >> 32), CONTROL, ROWS, 0xf, true));
    return __builtin_bit_cast(double, static_cast<std::uint64_t>(hi) << 32 | lo);
}
// Sums over lanes 0..lane, by lane moves within rows of 16 and then across rows.
__device__ __forceinline__ double wave_scan(double v) {
    v += moved<0x111, 0xf>(v);
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);
    v += moved<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ double lane_value(double v, int lane) {
    const auto w = __builtin_bit_cast(std::uint64_t, v);
    const std::uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(w), lane);
    const std::uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(w >> 32), lane);
    return __builtin_bit_cast(double, static_cast<std::uint64_t>(hi) << 32 | lo);
}

// A thread's sum of the tokens begin + 4 thread .. + 3, and every 4 THREADS on, below end, two loads of each row at once.
template <int THREADS>
__device__ __forceinline__ double2 sum_of(const Draw& d, int thread, int begin, int end) {
    constexpr int kAhead = 2;  // 4 or 8 load past the end of most runs: 128 sequences of 151936 tokens 33.4, 34.3, 46.9 us
    double2 sum = {0.0, 0.0};
    for (int first = begin + 4 * thread; first < end; first += 4 * THREADS * kAhead) {
        float4u p[kAhead], q[kAhead] = {};
#pragma unroll
        for (int u = 0; u < kAhead; ++u) p[u] = d.load(d.p, d.place(first + u * 4 * THREADS));
        if (d.q) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) q[u] = d.load(d.q, d.place(first + u * 4 * THREADS));
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const double2 s = d.share(p[u], q[u], j, first + u * 4 * THREADS, end);
                sum.x += s.x, sum.y += s.y;
            }
    }
    return sum;
}

// Sums of a part, and with the first one the verdict.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void verify_sum(Operands o) {
    __shared__ double2 waves[THREADS / 64];
    const int sequence = blockIdx.y, part = blockIdx.x;
    const Verdict v = verdict_of(o, sequence);
    const Draw d(o, v, sequence);
    const int begin = part * o.slice, end = min(begin + o.slice, o.vocab);
    double2 sum = sum_of<THREADS>(d, threadIdx.x, begin, end);
    sum = {wave_scan(sum.x), wave_scan(sum.y)};
    if ((threadIdx.x & 63) == 63) waves[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < THREADS / 64; ++i) waves[0].x += waves[i].x, waves[0].y += waves[i].y;
        o.sums[static_cast<std::int64_t>(sequence) * o.parts + part] = waves[0];
        if (part == 0) o.verdicts[sequence] = v;
    }
}

// Which of up to 64 shares in order (a lane each) the target falls into: the first whose running sum passes it, or the last one
// there is. `before` becomes what precedes it. For a whole wave.
__device__ __forceinline__ int find(double share, double target, double& before) {
    const double scan = before + wave_scan(share);
    const unsigned long long some = __ballot(share > 0.0), past = __ballot(share > 0.0 && scan > target);
    const int at = past ? __ffsll(past) - 1 : some ? 63 - __clzll(some) : 0;
    if (at) before = lane_value(scan, at - 1);
    return at;
}

// The sequence's tokens. A workgroup per sequence; with one part it sums the row itself. A wave takes a run of the part.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void verify_take(Operands o) {
    constexpr int kWaves = THREADS / 64;
    __shared__ double2 waves[kWaves];
    const int sequence = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Verdict v = o.parts > 1 ? o.verdicts[sequence] : verdict_of(o, sequence);
    const Draw d(o, v, sequence);
    const std::int64_t row = static_cast<std::int64_t>(sequence) * (o.drafts + 1);
    if (static_cast<int>(threadIdx.x) <= o.drafts && static_cast<int>(threadIdx.x) != v.accepted)
        o.tokens[row + threadIdx.x] = static_cast<int>(threadIdx.x) < v.accepted ? o.drafted[row - sequence + threadIdx.x] : -1;
    if (threadIdx.x == 0) o.accepted[sequence] = v.accepted;
    const double u = o.uniforms[row + o.drafts];
    int begin = 0, end = o.vocab;
    double before = 0.0, target = 0.0;
    bool rest = true;  // draw from the remainder
    if (o.parts > 1) {
        const double2 none = {0.0, 0.0};
        const double2 own = lane < o.parts ? o.sums[static_cast<std::int64_t>(sequence) * o.parts + lane] : none;
        const double all = lane_value(wave_scan(own.x), 63);
        rest = all > 0.0;
        target = u * (rest ? all : lane_value(wave_scan(own.y), 63));
        begin = find(rest ? own.x : own.y, target, before) * o.slice;
        end = min(begin + o.slice, o.vocab);
    }
    const int run = ((end - begin + kWaves - 1) / kWaves + 3) / 4 * 4;
    begin += wave * run;
    end = min(begin + run, end);
    double2 sum = sum_of<64>(d, lane, begin, end);
    sum = {wave_scan(sum.x), wave_scan(sum.y)};
    if (lane == 63) waves[wave] = sum;
    __syncthreads();
    const double2 own = lane < kWaves ? waves[lane] : double2{0.0, 0.0};
    if (o.parts == 1) {
        const double all = lane_value(wave_scan(own.x), 63);
        rest = all > 0.0;
        target = u * (rest ? all : lane_value(wave_scan(own.y), 63));
    }
    if (find(rest ? own.x : own.y, target, before) != wave) return;
    // The wave that the token lies in goes through its run again.
    int token = -1;
    for (int first = begin; first < end; first += 256) {
        const int at = first + 4 * lane;
        const float4u p = d.load(d.p, d.place(at)), q = d.q ? d.load(d.q, d.place(at)) : float4u{};
        double w[4], four = 0.0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const double2 s = d.share(p, q, j, at, end);
            w[j] = rest ? s.x : s.y;
            four += w[j];
        }
        const double scan = before + wave_scan(four);
        const unsigned long long some = __ballot(four > 0.0), past = __ballot(four > 0.0 && scan > target);
        if (some) {
            const int mine = past ? __ffsll(past) - 1 : 63 - __clzll(some);
            // Of the lane's four the first that passes, or else the last with a share.
            double running = mine ? lane_value(scan, mine - 1) : before;
            int found = -1;
            bool passed = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                running += lane_value(w[j], mine);
                if (lane_value(w[j], mine) > 0.0 && !passed) {
                    found = d.place(first + 4 * mine) + j;
                    passed = running > target;
                }
            }
            token = found;
        }
        if (past) break;
        before = lane_value(scan, 63);
    }
    if (lane == 0) o.tokens[row + v.accepted] = token;
}

Operands geometry(int sequences, int drafts, int vocab) {
    require(sequences > 0 && sequences <= kMaxSequences, "verification takes 1 to 65535 sequences");
    require(drafts > 0 && drafts <= kMaxDrafts, "verification takes 1 to 64 drafts of a sequence");
    require(vocab > 0 && vocab <= kMaxVocab, "verification takes a vocabulary of at most 1048576");
    // Parts of 2048 tokens and more, about 2048 workgroups in all.
    const int parts = std::max(std::min({kMaxParts, 2048 / sequences, vocab / 2048}), 1);
    Operands o{};
    o.drafts = drafts, o.vocab = vocab, o.parts = parts, o.slice = ((vocab + parts - 1) / parts + 3) / 4 * 4;
    return o;
}

template <int THREADS>
void launch_sum(const Operands& o, int sequences, hipStream_t stream) {
    verify_sum<THREADS><<<dim3(o.parts, sequences), THREADS, 0, stream>>>(o);
}
template <int THREADS>
void launch_take(const Operands& o, int sequences, hipStream_t stream) {
    verify_take<THREADS><<<sequences, THREADS, 0, stream>>>(o);
}

// Where the card is full, small workgroups, which repeat the verdict's loads in fewer waves (us, 128 threads against 256: 128
// sequences of 151936 tokens 34.3 / 36.9, 64 19.8 / 22.1; one of 248320 11.5 / 9.3).
void launch_sum(const Operands& o, int sequences, hipStream_t stream) {
    if (o.parts * sequences > 256) launch_sum<128>(o, sequences, stream);
    else launch_sum<256>(o, sequences, stream);
}

// As many threads as have a run of some length, fewer where sequences are many (they start sooner). Us, 256 / 512 / 1024
// threads: one sequence of 1000 tokens 4.9 / 5.4 / 6.5, of 248320 (3880 in a part) 9.5 / 9.3 / 10.1; 128 of 151936 (9496) 42 /
// 39 / 37; 512 of 32003 (8004) 31 / 28 / 31; 2100 of 9001 (one part) 34 / 42 / 49.
void launch_take(const Operands& o, int sequences, hipStream_t stream) {
    if (o.slice <= 1024 || sequences > 1024) launch_take<256>(o, sequences, stream);
    else if (o.slice <= 6144 || sequences > 256) launch_take<512>(o, sequences, stream);
    else launch_take<1024>(o, sequences, stream);
}

std::uint64_t sum_bytes(const Operands& o, int sequences) {
    return o.parts > 1 ? (sizeof(Verdict) + sizeof(double2) * o.parts) * static_cast<std::uint64_t>(sequences) : 0;
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
        o.tokens = tokens, o.accepted = accepted, o.verdicts = static_cast<vt::Verdict*>(workspace);
        o.sums = reinterpret_cast<double2*>(o.verdicts + sequences);
        const auto s = static_cast<hipStream_t>(stream);
        if (o.parts > 1) {
            vt::launch_sum(o, sequences, s);
            vt::check(hipGetLastError());
        }
        vt::launch_take(o, sequences, s);
    });
}

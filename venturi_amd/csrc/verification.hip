// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Draft i of a sequence stands while u_i q_i(d_i) < p_i(d_i) and p_i(d_i) > 0 (q = 1 for certain drafts): both sides are products
// of 32-bit numbers, exact in 64 bits. After the first refusal the next token comes from max(p - q, 0) of that row (of certain drafts:
// p without the draft), where that has a mass, else from p; after the last draft from p of the row behind it. It is the first
// token, by index, at which the running sum passes u times the whole one; sums in 64 bits, in a fixed order.
//
// Bound by memory where sequences are many: one or two rows of 4-byte probabilities each (128 of 151936 tokens with a drafter's
// rows 30.2 us, 5.1 TB/s), else by launches and their chains of loads: the drafts, their probabilities, the row. A long row is cut
// into parts that workgroups sum, and in a second launch one workgroup finds the part and the token in it (one sequence of 248320
// tokens 8.2 us); a short one is summed and searched in one launch from registers (61 of 32003 10.1). Times are a call's in a
// captured chain; a call from the host takes 8 with one launch and 11 with two.
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
    double* sums;                 // [sequences][parts]
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
    const unsigned long long bad = __ballot(lane < count && !(there && p > 0.0 && u * q < p));
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
    // Shares of the tokens at .. at + 3 that lie below `end`, loaded from their place, where the wave's first is `first`. A step
    // of a wave that ends before `end` and does not hold the refused draft needs no look at indices: 4 operations a token, 8
    // with a proposal.
    __device__ __forceinline__ void shares(const float4u& pv, const float4u& qv, int first, int at, int end, double (&w)[4]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = share(pv[j], qv[j]);
        if (first + 256 > end || (without >= first && without < first + 256)) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int index = place(at) + j;
                w[j] = index >= at && index < end && index != without ? w[j] : 0.0;
            }
        }
    }

private:
    __device__ __forceinline__ double share(float pj, float qj) const {
        constexpr int kPositive = 0x180;  // normal and subnormal numbers above 0
        const bool some = __builtin_amdgcn_classf(pj, kPositive);
        if (!q) return static_cast<double>(some ? pj : 0.0f);
        const double rest = fmax(static_cast<double>(pj) - static_cast<double>(qj), 0.0);
        return some ? rest : 0.0;
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
__device__ __forceinline__ double sum_of(const Draw& d, int thread, int begin, int end) {
    constexpr int kAhead = 2;  // 1 and 4: 300 sequences of 151936 tokens 74 us, 87, 80
    const int lane = thread & 63;
    double sum = 0.0;
    for (int first = begin + 4 * (thread - lane); first < end; first += 4 * THREADS * kAhead) {
        float4u p[kAhead], q[kAhead] = {};
#pragma unroll
        for (int u = 0; u < kAhead; ++u) p[u] = d.load(d.p, d.place(first + 4 * lane + u * 4 * THREADS));
        if (d.q) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) q[u] = d.load(d.q, d.place(first + 4 * lane + u * 4 * THREADS));
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            double w[4];
            d.shares(p[u], q[u], first + u * 4 * THREADS, first + 4 * lane + u * 4 * THREADS, end, w);
            sum += (w[0] + w[1]) + (w[2] + w[3]);
        }
    }
    return sum;
}

// Tokens of a wave's run, where `waves` of them share a part: whole vectors.
__host__ __device__ constexpr int run_of(int tokens, int waves) { return ((tokens + waves - 1) / waves + 3) / 4 * 4; }

// Sums of a part, and with the first one the verdict.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void verify_sum(Operands o) {
    __shared__ double waves[THREADS / 64];
    const int sequence = blockIdx.y, part = blockIdx.x;
    const Verdict v = verdict_of(o, sequence);
    const Draw d(o, v, sequence);
    const int begin = part * o.slice, end = min(begin + o.slice, o.vocab);
    const double sum = wave_scan(sum_of<THREADS>(d, threadIdx.x, begin, end));
    if ((threadIdx.x & 63) == 63) waves[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        double all = waves[0];
        for (int i = 1; i < THREADS / 64; ++i) all += waves[i];
        o.sums[static_cast<std::int64_t>(sequence) * o.parts + part] = all;
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

// Goes through a run of the row from `before` on: the first token at which the running sum passes the target, or the last one
// with a share; -1 if there is none. For a whole wave, 256 tokens at a step.
struct Search {
    double before, target;
    int token;
    bool past;

    __device__ __forceinline__ void step(const Draw& d, const float4u& p, const float4u& q, int first, int end) {
        double w[4];
        d.shares(p, q, first, first + 4 * static_cast<int>(threadIdx.x & 63), end, w);
        const double four = (w[0] + w[1]) + (w[2] + w[3]), scan = before + wave_scan(four);
        const unsigned long long some = __ballot(four > 0.0), beyond = __ballot(four > 0.0 && scan > target);
        if (some) {
            const int mine = beyond ? __ffsll(beyond) - 1 : 63 - __clzll(some);
            // Of the lane's four the first that passes, or else the last with a share.
            double running = mine ? lane_value(scan, mine - 1) : before;
            bool passed = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                running += lane_value(w[j], mine);
                if (lane_value(w[j], mine) > 0.0 && !passed) {
                    token = d.place(first + 4 * mine) + j;
                    passed = running > target;
                }
            }
        }
        past = beyond != 0;
        before = lane_value(scan, 63);
    }
};

// The sequence's tokens. A workgroup per sequence; with one part it sums the row itself. A wave takes a run of the part: one of
// up to 256 HELD tokens stays in its registers, else the wave that the token lies in reads its run again. Where nothing is left
// of the target's row without the proposal, the workgroup starts again with the whole of it.
template <int THREADS, int HELD>
__global__ __launch_bounds__(THREADS) void verify_take(Operands o) {
    constexpr int kWaves = THREADS / 64;
    __shared__ double waves[kWaves];
    const int sequence = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Verdict v = o.parts > 1 ? o.verdicts[sequence] : verdict_of(o, sequence);
    Draw d(o, v, sequence);
    const std::int64_t row = static_cast<std::int64_t>(sequence) * (o.drafts + 1);
    if (static_cast<int>(threadIdx.x) <= o.drafts && static_cast<int>(threadIdx.x) != v.accepted)
        o.tokens[row + threadIdx.x] = static_cast<int>(threadIdx.x) < v.accepted ? o.drafted[row - sequence + threadIdx.x] : -1;
    if (threadIdx.x == 0) o.accepted[sequence] = v.accepted;
    const double u = o.uniforms[row + o.drafts];
    int begin = 0, end = o.vocab;
    double before = 0.0, target = 0.0, own = 0.0;
    bool narrow = o.parts == 1;  // to one part
    if (o.parts > 1) {
        const double share = lane < o.parts ? o.sums[static_cast<std::int64_t>(sequence) * o.parts + lane] : 0.0;
        const double all = lane_value(wave_scan(share), 63);
        narrow = all > 0.0;
        target = u * all;
        if (narrow) begin = find(share, target, before) * o.slice, end = min(begin + o.slice, o.vocab);
    }
    float4u p[HELD ? HELD : 1], q[HELD ? HELD : 1];
    const auto split = [&] {  // the wave's run
        const int run = run_of(end - begin, kWaves);
        begin += wave * run;
        end = min(begin + run, end);
    };
    const auto join = [&](double sum) {
        sum = wave_scan(sum);
        if (lane == 63) waves[wave] = sum;
        __syncthreads();
        own = lane < kWaves ? waves[lane] : 0.0;
    };
    if (narrow) {
        split();
        double sum = 0.0;
        if constexpr (HELD) {
#pragma unroll
            for (int i = 0; i < HELD; ++i) p[i] = d.load(d.p, d.place(begin + 256 * i + 4 * lane));
            if (d.q) {
#pragma unroll
                for (int i = 0; i < HELD; ++i) q[i] = d.load(d.q, d.place(begin + 256 * i + 4 * lane));
            }
#pragma unroll
            for (int i = 0; i < HELD; ++i) {
                if (begin + 256 * i >= end) break;
                double w[4];
                d.shares(p[i], q[i], begin + 256 * i, begin + 256 * i + 4 * lane, end, w);
                sum += (w[0] + w[1]) + (w[2] + w[3]);
            }
        } else {
            sum = sum_of<64>(d, lane, begin, end);
        }
        join(sum);
        if (o.parts == 1) {
            const double all = lane_value(wave_scan(own), 63);
            narrow = all > 0.0;
            target = u * all;
        }
    }
    const bool held = HELD && narrow;
    if (!narrow) {
        d.q = nullptr, d.without = -1;
        begin = 0, end = o.vocab;
        split();
        __syncthreads();
        join(sum_of<64>(d, lane, begin, end));
        target = u * lane_value(wave_scan(own), 63);
    }
    if (find(own, target, before) != wave) return;
    Search search{before, target, -1, false};
    if (held) {
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            if (!search.past && begin + 256 * i < end) search.step(d, p[i], q[i], begin + 256 * i, end);
    } else {
        for (int first = begin; first < end && !search.past; first += 256) {
            const int at = d.place(first + 4 * lane);
            search.step(d, d.load(d.p, at), d.q ? d.load(d.q, at) : float4u{}, first, end);
        }
    }
    if (lane == 0) o.tokens[row + v.accepted] = search.token;
}

Operands geometry(int sequences, int drafts, int vocab) {
    require(sequences > 0 && sequences <= kMaxSequences, "verification takes 1 to 65535 sequences");
    require(drafts > 0 && drafts <= kMaxDrafts, "verification takes 1 to 64 drafts of a sequence");
    require(vocab > 0 && vocab <= kMaxVocab, "verification takes a vocabulary of at most 1048576");
    // Parts of 2048 tokens and more, about 2048 workgroups in all; one part, and one launch, where a workgroup's registers hold
    // the row and each has a CU, where the row is short, or where two parts would be all. (Us in a chain of calls, parts against
    // one: one sequence of 32003 tokens 11.9 / 9.1, 61 11.8 / 11.3, 256 14.6 / 14.0, 257 15.8 / 19.7; 300 of 16001 13.1 / 12.7, of
    // 32003 19.4 / 23.7; 512 of 151936 98 / 125, 700 170 / 157. A call with one launch takes the host 8, with two 11.)
    int parts = std::max(std::min({kMaxParts, 2048 / sequences, vocab / 2048}), 1);
    if (parts < 3 || vocab <= (sequences <= 256 ? 32768 : 16384)) parts = 1;
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
    const int run = run_of(std::min(o.slice, o.vocab), THREADS / 64);
    if (run <= 1024) verify_take<THREADS, 4><<<sequences, THREADS, 0, stream>>>(o);
    else if (run <= 2048) verify_take<THREADS, 8><<<sequences, THREADS, 0, stream>>>(o);
    else verify_take<THREADS, 0><<<sequences, THREADS, 0, stream>>>(o);
}

// Where the card is full, small workgroups, which repeat the verdict's loads in fewer waves (us, 128 threads against 256: 128
// sequences of 151936 tokens 28.0 / 28.5, 64 17.1 / 18.5; one of 248320 9.0 / 8.2).
void launch_sum(const Operands& o, int sequences, hipStream_t stream) {
    if (o.parts * sequences > 256) launch_sum<128>(o, sequences, stream);
    else launch_sum<256>(o, sequences, stream);
}

// As many threads as have a run of some length, fewer where sequences are many (they start sooner). Us, 256 / 512 / 1024
// threads: 300 sequences of 1000 tokens 4.5 / 5.2 / 7.7, of 9001 12.5 / 9.1 / 10.3; one of 5001 5.6 / 4.4 / 4.6, of 16001 9.9 /
// 6.5 / 6.0, of 248320 (3880 in a part) 7.7 / 7.5 / 8.0; 128 of 151936 (9496) 29.5 / 25.6 / 24.7; 2100 of 9001 28 / 31 / 40.
void launch_take(const Operands& o, int sequences, hipStream_t stream) {
    if (o.slice <= 1024 || sequences > 1024) launch_take<256>(o, sequences, stream);
    else if (o.slice <= 6144 || sequences > 256) launch_take<512>(o, sequences, stream);
    else launch_take<1024>(o, sequences, stream);
}

std::uint64_t sum_bytes(const Operands& o, int sequences) {
    return o.parts > 1 ? (sizeof(Verdict) + sizeof(double) * o.parts) * static_cast<std::uint64_t>(sequences) : 0;
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
        const std::uint64_t n = sequences, d = drafts, token_bytes = 8 * n * (d + 1), accepted_bytes = 4 * n;
        const auto meets_an_input = [&](const void* out, std::uint64_t size) {
            return vt::meet(out, size, target, 4 * n * (d + 1) * vocab) || vt::meet(out, size, proposal, 4 * n * d * vocab) ||
                   vt::meet(out, size, drafted, 8 * n * d) || vt::meet(out, size, counts, 4 * n) ||
                   vt::meet(out, size, uniforms, 4 * n * (d + 1));
        };
        vt::require(!meets_an_input(tokens, token_bytes) && !meets_an_input(accepted, accepted_bytes) &&
                        !meets_an_input(workspace, bytes) && !vt::meet(tokens, token_bytes, accepted, accepted_bytes) &&
                        !vt::meet(workspace, bytes, tokens, token_bytes) && !vt::meet(workspace, bytes, accepted, accepted_bytes),
                    "verification outputs must not overlap other operands");
        o.target = target, o.proposal = proposal, o.drafted = drafted, o.counts = counts, o.uniforms = uniforms;
        o.tokens = tokens, o.accepted = accepted, o.verdicts = static_cast<vt::Verdict*>(workspace);
        o.sums = reinterpret_cast<double*>(o.verdicts + sequences);
        const auto s = static_cast<hipStream_t>(stream);
        if (o.parts > 1) {
            vt::launch_sum(o, sequences, s);
            vt::check(hipGetLastError());
        }
        vt::launch_take(o, sequences, s);
    });
}

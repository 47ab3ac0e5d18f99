// Drafted tokens against the target's probabilities, from given random numbers.
//
// A sequence has the rows starts[b] .. starts[b + 1] - 1 of a step: its last token and behind it the drafted ones.  Row i of the target
// holds the probabilities p of the token behind it, row i of the draft those, q, that the next row's token x was drawn from.  In order,
// x is accepted if u[i] q(x) < p(x) (with probability min(1, p / q)); behind the last accepted one comes a token drawn from
// max(p - q, 0) of the row that refused, or from p where none did, so that all tokens are distributed as the target's.
//
// Drawing by the running sum of the weights against w times their sum: a border between two tokens may lie anywhere, so the sums are
// in float64, where p - q is exact or nearly so and the order of the additions moves a border by some 1e-15.  Half-precision
// sums would move one in a thousand draws.
//
// A block has a run of the vocabulary of one sequence; every block checks the drafts itself (two numbers each), so that it knows the row
// to read, and asks for 8192 of its probabilities at once, or 16 384.  Sums go to the last block that arrives, which finds the run, in it the piece of
// 512 that a wavefront reads with one instruction, the lane and the token.  Each probability is read once, the run of the token twice.  Bound by
// a chain of eight trips to memory, in the large by the conversions and float64 sums too, which follow a block's loads and do not overlap them: 128 rows of
// 131 072 float16 24 us, 1.6 TB/s, vector instructions 42 %.
#include <type_traits>

#include "common.hpp"

using namespace lq;

namespace {

constexpr unsigned kThreads = 256, kWaves = kThreads / 64, kVec = 8, kRound = kThreads * kVec;  // tokens
constexpr unsigned kNone = 0xffffffffu;

struct Args {
    const void *target, *draft;  // [rows, vocab]; draft NULL: q is 1 at the drafted token
    const int *tokens, *starts;
    const float *uniforms, *last;
    int *new_tokens, *counts;
    unsigned rows, vocab, run;  // run: tokens of a block, a multiple of 8
    double* sums;               // [batch][runs][2]
    int* arrived;               // [batch], zero between launches
};

// what counts of a probability: a positive finite number
__device__ __forceinline__ float counted(float p) { return p < __builtin_inff() ? fmaxf(p, 0.f) : 0.f; }  // (fmaxf of a NaN is 0)

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}
// the sum over the lanes up to this one
__device__ __forceinline__ double wave_scan(double v, unsigned lane) {
#pragma unroll
    for (unsigned d = 1; d < 64; d <<= 1) {
        const double up = __shfl_up(v, d, 64);
        if (lane >= d) v += up;
    }
    return v;
}

// Eight values of a row as they lie in memory.
template <class T>
struct Raw {
    T v[kVec];
};

// The row that a sequence's next token is drawn from: p alone, without token x (kNone: with all), or p - q.  A lane's eight tokens from v on: of
// those that reach past `end` the last eight before it are loaded, and what is before v does not count, so that no load has a branch (code
// that a block runs once comes from memory: one row of 540 float32 by value with branches 10.2 us, so
// 8.9; 128 rows of 131 072 33.5 and 34.7).  TINY: rows of fewer than eight, by value.
template <class T, bool DRAFT, bool TINY>
struct Row {
    const T *p, *q;  // q NULL: p alone
    unsigned x;
    struct Eight {
        Raw<T> p, q[DRAFT ? 1 : 0];
    };
    static __device__ __forceinline__ unsigned place(unsigned v, unsigned end) { return !TINY && v + kVec > end ? end - kVec : v; }
    static __device__ __forceinline__ Raw<T> load8(const T* row, unsigned v, unsigned end) {
        Raw<T> raw;
        if constexpr (TINY) {
#pragma unroll
            for (unsigned e = 0; e < kVec; ++e) raw.v[e] = row[v + e < end ? v + e : 0];
        } else {
            __builtin_memcpy(&raw, row + place(v, end), sizeof raw);  // (rows of odd length are not 16-byte aligned)
        }
        return raw;
    }
    __device__ __forceinline__ Eight load(unsigned v, unsigned end) const {
        Eight r;
        r.p = load8(p, v, end);
        if constexpr (DRAFT)
            if (q) r.q[0] = load8(q, v, end);
        return r;
    }
    // the weights of tokens place(v, end) + e; all: those of p where q is there
    __device__ __forceinline__ void weights(const Eight& r, unsigned v, unsigned end, double (&w)[kVec], double& all) const {
        all = 0.0;
        const unsigned at = place(v, end);
#pragma unroll
        for (unsigned e = 0; e < kVec; ++e) {
            const bool own = TINY ? v + e < end : at + e >= v;
            w[e] = own ? double(counted(float(r.p.v[e]))) : 0.0;
        }
        if constexpr (DRAFT) {
            if (q) {
#pragma unroll
                for (unsigned e = 0; e < kVec; ++e) {
                    all += w[e];
                    w[e] = fmax(w[e] - double(counted(float(r.q[0].v[e]))), 0.0);
                }
            }
        } else if (x - at < kVec) {
#pragma unroll
            for (unsigned e = 0; e < kVec; ++e)
                if (at + e == x) w[e] = 0.0;
        }
    }
};

// The lane that the running sum passes `goal` in, of `v` with `before` in front, and what is in front of it: the lowest with something in it that does,
// else the last with something in it; -1 without any.  The same for all lanes.
__device__ __forceinline__ int passing(double v, double goal, unsigned lane, double& before) {
    const double upto = before + wave_scan(v, lane);
    const uint64_t some = __builtin_amdgcn_ballot_w64(v > 0.0), over = __builtin_amdgcn_ballot_w64(v > 0.0 && upto > goal);
    if (!some) return -1;
    const int at = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
    if (at) before = __shfl(upto, at - 1, 64);
    return at;
}

constexpr int kBlocks = 4;  // of a CU: what their registers leave room for
template <class T, bool DRAFT>
constexpr unsigned kAhead = sizeof(T) == 2 && !DRAFT ? 8 : 4;  // times eight probabilities that a thread asks for at once

template <class T, bool DRAFT, bool TINY>
__global__ __launch_bounds__(256, kBlocks) void verify_drafts_kernel(Args a) {
    constexpr unsigned kAtOnce = TINY ? 1 : kAhead<T, DRAFT>;
    __shared__ double s_sum[2][kWaves], s_piece[kAtOnce * kWaves];
    __shared__ unsigned s_first;
    __shared__ int s_is_last, s_next;
    const unsigned b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, runs = gridDim.x;
    const long lo = a.starts[b], hi = a.starts[b + 1];
    const unsigned from = unsigned(lo < 0 ? 0 : lo > long(a.rows) ? long(a.rows) : lo), to = unsigned(hi < lo ? from : hi > long(a.rows) ? long(a.rows) : hi < 0 ? 0 : hi);
    const unsigned n = to > from ? to - from : 0;
    if (n == 0) {  // (the same for all blocks of a sequence)
        if (blockIdx.x == 0 && tid == 0) a.counts[b] = 0;
        return;
    }
    const T* const target = static_cast<const T*>(a.target);
    const T* const draft = static_cast<const T*>(a.draft);
    // the first draft that is refused, or n - 1
    unsigned accepted = n - 1;
    for (unsigned i0 = 0; i0 + 1 < n; i0 += kThreads) {
        if (tid == 0) s_first = n - 1;
        __syncthreads();
        const unsigned i = i0 + tid;
        if (i + 1 < n) {
            const unsigned x = unsigned(a.tokens[from + i + 1]);
            const float u = a.uniforms[from + i];
            bool ok = false;
            if (x < a.vocab) {
                const double p = double(float(target[size_t(from + i) * a.vocab + x]));
                const double q = DRAFT ? double(float(draft[size_t(from + i) * a.vocab + x])) : 1.0;
                ok = double(u) * q < p;
            }
            if (!ok) atomicMin(&s_first, i);
        }
        __syncthreads();
        accepted = s_first;
        if (accepted < n - 1) break;  // uniform
        __syncthreads();
    }
    const bool refused = accepted < n - 1;
    Row<T, DRAFT, TINY> row{target + size_t(from + accepted) * a.vocab, refused && DRAFT ? draft + size_t(from + accepted) * a.vocab : nullptr,
               refused && !DRAFT ? unsigned(a.tokens[from + accepted + 1]) : kNone};

    // sums of this run
    const unsigned begin = blockIdx.x * a.run, end = begin + a.run < a.vocab ? begin + a.run : a.vocab;
    double all = 0.0, rest = 0.0;
    for (unsigned v0 = begin; v0 < end; v0 += kAtOnce * kRound) {
        typename Row<T, DRAFT, TINY>::Eight r[kAtOnce];
#pragma unroll
        for (unsigned u = 0; u < kAtOnce; ++u)
            if (v0 + u * kRound < end) r[u] = row.load(v0 + u * kRound + tid * kVec, end);
#pragma unroll
        for (unsigned u = 0; u < kAtOnce; ++u) {
            if (v0 + u * kRound >= end) continue;  // uniform
            double w[kVec], some;
            row.weights(r[u], v0 + u * kRound + tid * kVec, end, w, some);
            all += some;
            rest += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
        }
    }
    rest = wave_sum(rest);
    if (row.q) all = wave_sum(all);
    if (lane == 0) s_sum[0][wave] = rest, s_sum[1][wave] = all;
    __syncthreads();
    rest = (s_sum[0][0] + s_sum[0][1]) + (s_sum[0][2] + s_sum[0][3]), all = (s_sum[1][0] + s_sum[1][1]) + (s_sum[1][2] + s_sum[1][3]);
    double run_sum = lane == 0 ? rest : 0.0, run_all = lane == 0 ? all : 0.0;  // a lane has the sums of one run
    if (runs > 1) {
        if (tid == 0) {
            double* const out = a.sums + (size_t(b) * runs + blockIdx.x) * 2;
            // (through to where every block sees it)
            __hip_atomic_store(out, rest, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(out + 1, all, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            // (both go past the caches, and the last block reads them so: that they have arrived is order enough, no cache need be written back)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            s_is_last = __hip_atomic_fetch_add(&a.arrived[b], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == int(runs) - 1;
        }
        __syncthreads();
        if (!s_is_last) return;
        // the last block of the sequence
        const double* const sums = a.sums + (size_t(b) * runs + lane) * 2;
        run_sum = lane < runs ? __hip_atomic_load(sums, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
        run_all = lane < runs ? __hip_atomic_load(sums + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
    }
    double total = wave_sum(run_sum), before = 0.0;
    if (tid == 0) s_next = -1;
    if (refused && !(total > 0.0)) {
        // nothing is left of p: from p itself (without a draft that is x alone)
        if (row.q) {
            row.q = nullptr, run_sum = run_all, total = wave_sum(run_all);
        } else if (row.x < a.vocab && counted(float(row.p[row.x])) > 0.f) {
            __syncthreads();
            if (tid == 0) s_next = int(row.x);
        }
    }
    const double goal = double(a.last[b]) * total;
    const int run = passing(run_sum, goal, lane, before);
    if (run >= 0) {
        const unsigned first = unsigned(run) * a.run, stop = first + a.run < a.vocab ? first + a.run : a.vocab;
        for (unsigned v0 = first; v0 < stop; v0 += kAtOnce * kRound) {
            double sum[kAtOnce];
            typename Row<T, DRAFT, TINY>::Eight r[kAtOnce];
#pragma unroll
            for (unsigned u = 0; u < kAtOnce; ++u) r[u] = row.load(v0 + u * kRound + tid * kVec, stop);
            __syncthreads();  // (the pieces' sums before have been read)
#pragma unroll
            for (unsigned u = 0; u < kAtOnce; ++u) {
                double w[kVec], some;
                row.weights(r[u], v0 + u * kRound + tid * kVec, stop, w, some);
                sum[u] = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
                const double piece = wave_sum(sum[u]);
                if (lane == 0) s_piece[u * kWaves + wave] = piece;
            }
            __syncthreads();
            const double piece_sum = lane < kAtOnce * kWaves ? s_piece[lane] : 0.0, here = wave_sum(piece_sum);
            // (the last of a run's rounds with something in it decides if none passes)
            double at_piece = before;
            const int piece = passing(piece_sum, goal, lane, at_piece);
            if (piece >= 0 && unsigned(piece) % kWaves == wave) {
                const unsigned u = unsigned(piece) / kWaves;
                double mine = sum[0];
#pragma unroll
                for (unsigned k = 1; k < kAtOnce; ++k) mine = u == k ? sum[k] : mine;
                const int at_lane = passing(mine, goal, lane, at_piece);
                if (at_lane == int(lane)) {
                    const unsigned v = v0 + u * kRound + tid * kVec;
                    double w[kVec], some;
                    row.weights(row.load(v, stop), v, stop, w, some);
                    int next = -1;
                    bool passed = false;
#pragma unroll
                    for (unsigned e = 0; e < kVec; ++e)
                        if (w[e] > 0.0 && !passed) at_piece += w[e], next = int(row.place(v, stop) + e), passed = at_piece > goal;
                    s_next = next;
                }
            }
            before += here;
            if (before > goal) break;  // uniform
        }
    }
    __syncthreads();
    if (runs > 1 && tid == 0) a.arrived[b] = 0;
    const int next = s_next;
    for (unsigned i = tid; i < n; i += kThreads) a.new_tokens[from + i] = i < accepted ? a.tokens[from + i + 1] : i == accepted ? next : -1;
    if (tid == 0) a.counts[b] = int(accepted) + 1;
}

}  // namespace

extern "C" int lq_verify_drafts(const void* target, const void* draft, int dtype, int rows, int vocab, const int32_t* tokens, const int32_t* starts,
                                int batch, const float* uniforms, const float* last, int32_t* new_tokens, int32_t* counts, lq_stream stream) {
    LQ_REQUIRE(dtype == LQ_F32 || dtype == LQ_F16, LQ_ERR_DTYPE, "verify_drafts: probabilities are float32 or float16");
    LQ_REQUIRE(rows >= 0 && batch >= 0 && batch <= 65535, LQ_ERR_SHAPE, "verify_drafts: %d rows of %d sequences (65535 at most)", rows, batch);
    LQ_REQUIRE(vocab >= 1 && vocab <= 1 << 24, LQ_ERR_SHAPE, "verify_drafts: a vocabulary of %d tokens; 1 to 2^24", vocab);
    if (batch == 0) return LQ_OK;
    LQ_REQUIRE(starts && last && counts, LQ_ERR_VALUE, "verify_drafts: starts, last or counts is NULL");
    LQ_REQUIRE(rows == 0 || (target && tokens && uniforms && new_tokens), LQ_ERR_VALUE, "verify_drafts: a NULL pointer");
    // a sequence's last block writes while other sequences' blocks still read
    const size_t n = size_t(rows), seqs = size_t(batch), probabilities = n * size_t(vocab) * (dtype == LQ_F16 ? 2 : 4);
    const Span results[2] = {{new_tokens, n * 4}, {counts, seqs * 4}};
    bool sound = apart(results[0], results[1]);
    for (const Span& to : results)
        for (const Span& from : {Span{target, probabilities}, Span{draft, probabilities}, Span{tokens, n * 4}, Span{starts, (seqs + 1) * 4}, Span{uniforms, n * 4},
                                 Span{last, seqs * 4}})
            sound = sound && apart(to, from);
    LQ_REQUIRE(sound, LQ_ERR_VALUE, "verify_drafts: a result lies on what is read, or on the other result");
    // As many blocks as are resident, 8192 tokens at least each: what a block asks for at once, where one that is alone need not wait for others; 64 of
    // a sequence at most.  (16 x 131 072 float32 22 us of 2048 tokens, 13.2 of 8192; 16 x 32 000 12.5 and 11.1.  128 rows of 131 072
    // float16: 8 blocks a sequence that ask for all of their run at once 23.5 us, 12 and 16 of smaller runs 26 and 24.5, in rounds of 8192 tokens 29.)
    unsigned runs = 256u * unsigned(kBlocks) / unsigned(batch);
    const unsigned most = (unsigned(vocab) + 4 * kRound - 1) / (4 * kRound);
    runs = runs < 1 ? 1 : runs > 64 ? 64 : runs;
    if (runs > most) runs = most;
    const unsigned run = ((unsigned(vocab) + runs - 1) / runs + kVec - 1) / kVec * kVec;
    runs = (unsigned(vocab) + run - 1) / run;
    const hipStream_t st = as_stream(stream);
    const auto lock = scratch_lock(st);
    SkScratch scratch;
    if (const int rc = sk_scratch(size_t(batch), size_t(batch) * runs * 2 * sizeof(double), st, &scratch)) return rc;
    const Args a{target, draft, tokens, starts, uniforms, last, new_tokens, counts, unsigned(rows), unsigned(vocab), run,
                 reinterpret_cast<double*>(scratch.slabs), scratch.counters};
    const dim3 grid(runs, unsigned(batch));
    const auto of = [&](auto value, auto tiny) {
        using T = decltype(value);
        return draft ? verify_drafts_kernel<T, true, decltype(tiny)::value> : verify_drafts_kernel<T, false, decltype(tiny)::value>;
    };
    const bool tiny = unsigned(vocab) < kVec;
    const auto kernel = dtype == LQ_F32 ? (tiny ? of(0.f, std::true_type{}) : of(0.f, std::false_type{}))
                                        : (tiny ? of(_Float16(0.f), std::true_type{}) : of(_Float16(0.f), std::false_type{}));
    kernel<<<grid, kThreads, 0, st>>>(a);
    LQ_CHECK_LAUNCH("verify_drafts");
    return LQ_OK;
}

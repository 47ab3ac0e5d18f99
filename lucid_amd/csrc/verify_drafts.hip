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
// A block has a run of the vocabulary of one sequence; every block judges the drafts itself (two numbers each), so that it knows the row
// to read.  Sums go to the last block that arrives, which finds the run and in it the token.  Each probability is read once, the run of
// the token twice.  Bound by memory.
#include <type_traits>

#include "common.hpp"

using namespace lq;

namespace {

constexpr unsigned kThreads = 256, kVec = 8;

struct Args {
    const void *target, *draft;  // [rows, vocab]; draft NULL: q is 1 at the drafted token
    const int *tokens, *starts;
    const float *uniforms, *last;
    int *new_tokens, *counts;
    unsigned rows, vocab, run;  // run: tokens of a block, a multiple of 8
    double* sums;               // [batch][runs][2]
    int* arrived;               // [batch], zero between launches
};

// what counts of a weight: a positive finite number
__device__ __forceinline__ double positive(double d) { return d > 0.0 && d < __builtin_inf() ? d : 0.0; }

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

// eight values from v on, zeros from `end` on
template <class T>
__device__ __forceinline__ void load8(const T* row, unsigned v, unsigned end, float (&p)[kVec]) {
    if (v + kVec <= end) {
        T raw[kVec];
        __builtin_memcpy(raw, row + v, sizeof raw);  // (rows of odd length are not 16-byte aligned)
#pragma unroll
        for (unsigned e = 0; e < kVec; ++e) p[e] = float(raw[e]);
    } else {
#pragma unroll
        for (unsigned e = 0; e < kVec; ++e) p[e] = v + e < end ? float(row[v + e]) : 0.f;
    }
}

// The weights of eight tokens: those of the row's distribution, and of what a refused draft leaves of it.
template <class T>
__device__ __forceinline__ void weights8(const T* p_row, const T* q_row, bool refused, unsigned x, unsigned v, unsigned end, double (&all)[kVec],
                                         double (&rest)[kVec]) {
    float p[kVec], q[kVec];
    load8(p_row, v, end, p);
    if (refused && q_row) load8(q_row, v, end, q);
#pragma unroll
    for (unsigned e = 0; e < kVec; ++e) {
        all[e] = positive(double(p[e]));
        rest[e] = !refused ? 0.0 : q_row ? positive(double(p[e]) - positive(double(q[e]))) : v + e == x ? 0.0 : all[e];
    }
}

template <class T>
__global__ __launch_bounds__(256) void verify_drafts_kernel(Args a) {
    __shared__ double s_sum[2][kThreads / 64], s_scan[kThreads / 64];
    __shared__ unsigned s_first, s_found, s_last;
    __shared__ int s_is_last;
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
            bool ok = false;
            if (x < a.vocab) {
                const double p = double(float(target[size_t(from + i) * a.vocab + x]));
                const double q = draft ? double(float(draft[size_t(from + i) * a.vocab + x])) : 1.0;
                ok = double(a.uniforms[from + i]) * q < p;
            }
            if (!ok) atomicMin(&s_first, i);
        }
        __syncthreads();
        accepted = s_first;
        if (accepted < n - 1) break;  // uniform
        __syncthreads();
    }
    const bool refused = accepted < n - 1;
    const unsigned x = refused ? unsigned(a.tokens[from + accepted + 1]) : 0;
    const T* const p_row = target + size_t(from + accepted) * a.vocab;
    const T* const q_row = draft ? draft + size_t(from + accepted) * a.vocab : nullptr;

    // sums of this run
    const unsigned begin = blockIdx.x * a.run, end = begin + a.run < a.vocab ? begin + a.run : a.vocab;
    double all = 0.0, rest = 0.0;
    for (unsigned v = begin + tid * kVec; v < end; v += kThreads * kVec) {
        double wa[kVec], wr[kVec];
        weights8(p_row, q_row, refused, x, v, end, wa, wr);
#pragma unroll
        for (unsigned e = 0; e < kVec; ++e) all += wa[e], rest += wr[e];
    }
    all = wave_sum(all), rest = wave_sum(rest);
    if (lane == 0) s_sum[0][wave] = all, s_sum[1][wave] = rest;
    __syncthreads();
    if (tid == 0) {
        all = (s_sum[0][0] + s_sum[0][1]) + (s_sum[0][2] + s_sum[0][3]), rest = (s_sum[1][0] + s_sum[1][1]) + (s_sum[1][2] + s_sum[1][3]);
        double* const out = a.sums + (size_t(b) * runs + blockIdx.x) * 2;
        // (through to where every block sees it)
        __hip_atomic_store(out, all, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(out + 1, rest, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_is_last = __hip_atomic_fetch_add(&a.arrived[b], 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == int(runs) - 1;
    }
    __syncthreads();
    if (!s_is_last) return;

    // the last block of the sequence: which weights, which run (a lane has the sums of one), which token
    const double* const sums = a.sums + (size_t(b) * runs + lane) * 2;
    const double run_all = lane < runs ? __hip_atomic_load(sums, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
    const double run_rest = lane < runs ? __hip_atomic_load(sums + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
    const bool of_rest = refused && wave_sum(run_rest) > 0.0;
    const double run_sum = of_rest ? run_rest : run_all;
    const double upto = wave_scan(run_sum, lane), goal = double(a.last[b]) * __shfl(upto, 63, 64);
    const uint64_t some = __builtin_amdgcn_ballot_w64(run_sum > 0.0), over = __builtin_amdgcn_ballot_w64(run_sum > 0.0 && upto > goal);
    // (none is over with numbers of 1 and more, and NaN: the last token then)
    const int run = over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : 0;
    const double before = run ? __shfl(upto, run - 1, 64) : 0.0;
    // a thread has consecutive tokens of the run
    const unsigned first = unsigned(run) * a.run, stop = first + a.run < a.vocab ? first + a.run : a.vocab;
    const unsigned each = (a.run + kThreads * kVec - 1) / (kThreads * kVec) * kVec, mine = first + tid * each;
    auto over_mine = [&](auto&& f) {
        for (unsigned v = mine; v < mine + each && v < stop; v += kVec) {
            double wa[kVec], wr[kVec];
            weights8(p_row, q_row, refused, x, v, stop, wa, wr);
#pragma unroll
            for (unsigned e = 0; e < kVec; ++e) f(v + e, of_rest ? wr[e] : wa[e]);
        }
    };
    double sum = 0.0;
    over_mine([&](unsigned, double w) { sum += w; });
    // what the threads before it have
    const double scan = wave_scan(sum, lane);
    if (lane == 63) s_scan[wave] = scan;
    if (tid == 0) s_found = 0xffffffffu, s_last = 0;
    __syncthreads();
    double at = before + (scan - sum);
    for (unsigned i = 0; i < wave; ++i) at += s_scan[i];
    unsigned found = 0xffffffffu, last = 0;
    if (sum > 0.0)
        over_mine([&](unsigned v, double w) {
            if (w > 0.0) {
                at += w, last = v + 1;
                if (at > goal && found == 0xffffffffu) found = v;
            }
        });
    if (found != 0xffffffffu) atomicMin(&s_found, found);
    if (last) atomicMax(&s_last, last);
    __syncthreads();
    if (tid == 0) a.arrived[b] = 0;
    const int next = s_found != 0xffffffffu ? int(s_found) : int(s_last) - 1;  // (-1: no weight at all)
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
    LQ_REQUIRE(new_tokens != tokens || !tokens, LQ_ERR_VALUE, "verify_drafts: the new tokens cannot take the drafted ones' place");
    LQ_REQUIRE(rows == 0 || (target && tokens && uniforms && new_tokens), LQ_ERR_VALUE, "verify_drafts: a NULL pointer");
    // Runs of 8192 tokens, shorter ones of few sequences, so that some 512 blocks share the work, and 64 of a sequence at most.
    unsigned runs = unsigned(vocab + 8191) / 8192;
    const unsigned fill = 512 / unsigned(batch), most = unsigned(vocab + 2047) / 2048;
    if (runs < fill) runs = fill < most ? fill : most;
    if (runs > 64) runs = 64;
    const unsigned run = ((unsigned(vocab) + runs - 1) / runs + kVec - 1) / kVec * kVec;
    runs = (unsigned(vocab) + run - 1) / run;
    const hipStream_t st = as_stream(stream);
    const auto lock = scratch_lock(st);
    SkScratch scratch;
    if (const int rc = sk_scratch(size_t(batch), size_t(batch) * runs * 2 * sizeof(double), st, &scratch)) return rc;
    const Args a{target, draft, tokens, starts, uniforms, last, new_tokens, counts, unsigned(rows), unsigned(vocab), run,
                 reinterpret_cast<double*>(scratch.slabs), scratch.counters};
    const dim3 grid(runs, unsigned(batch));
    if (dtype == LQ_F32) verify_drafts_kernel<float><<<grid, kThreads, 0, st>>>(a);
    else verify_drafts_kernel<_Float16><<<grid, kThreads, 0, st>>>(a);
    LQ_CHECK_LAUNCH("verify_drafts");
    return LQ_OK;
}

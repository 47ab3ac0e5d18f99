// Gated projections of few rows (wq_gated.hpp has the mathematics): bound by reading the weights.
//
// A wavefront has 16 columns of both weights and steps of 128 or 64 k; the wavefronts of a block that have the same columns and other steps add
// their sums in LDS at the end.  What a step needs goes from memory straight into LDS, into a ring of steps, with neighbouring lanes on
// neighbouring bytes: a load whose lanes are an operand's (row = lane % 16) costs the address unit a cycle a lane, whatever it carries (1 x 11008 x
// 4096 of 4 bits took 24 us that way, with half or all of the vector work and whatever was under way).  Scales and biases come likewise, runs of 16 or 32
// groups of a row at a time (two tables take turns): the few of each step asked for with its codes, 4 bytes a row, took as long as the
// codes (16 x 11008 x 4096, 8 bits: 18 us for the codes alone, 37 with them).  In LDS the 16-byte chunks of a row
// change places with its number, so that the 16 rows of an operand lie in different banks.  The sums of x of a group are a product with ones.
//
// x as it enters the matrix instructions: float16 as it is; a float32 row times the power of two that brings its largest value below 2^15,
// as two float16, hi = x rounded, lo = x - hi rounded: 22 bits, or 2^-39 of the largest value.
//
// gated_few_kernel, up to 4 rows that leave room for two blocks a CU: a block has 16 columns, its four wavefronts every fourth step each.  It brings x
// into LDS itself, while its first weights are under way, and beside that shares the tables alone, so that a barrier comes once a table.  A row of x
// lies on every fourth row of the instruction: a lane then has one element of each result.
//
// gated_rows_kernel: a block of eight wavefronts has CG times 16 columns, a wavefront 16 of them and every SG-th step (CG SG = 8), so that CG share
// an x (16 rows of float32 are as many bytes as the codes of 16 columns of both weights in 8 bits, and come from the L2 for every block again:
// 16 x 11008 x 4096, 16 columns a block and no x shared, 41 us).  What a block takes is a chain of steps, so with few columns steps are dealt
// to more wavefronts as far as the blocks are one a CU: 16 x 2048 x 4096, 4 bits, float16, 16 us with CG = 4, 10.6 with 2, 8.0 with 1.  float32 rows
// are split by a launch of their own.
#pragma once
#include <algorithm>
#include <type_traits>

#include "wq_gated.hpp"

namespace lq {
namespace gated {
namespace {

// (The compiler waits for every load under way into LDS before it reads there through a type that aliases all others, as the vector types of HIP's
// headers are copied: these are types of the language.)
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kFewWaves = 4, kFewStep = 128;  // k of a step

struct RowsX {
    const _Float16* part[2];  // [M, K]; float16 x: the first
    const float* unscale;     // [M], of float32 x
};

// A wavefront's part of a step of STEP k in LDS: the codes of 16 rows of both weights.
template <int BITS, int STEP>
struct Codes {
    static constexpr int ROW = STEP * BITS / 8, CHUNKS = ROW / 16;
    static constexpr int LOADS = ROW / 32, BYTES = LOADS * 1024;  // instructions that move 1 KiB
    static __device__ __forceinline__ int swizzle(int r) { return CHUNKS == 2 ? (r >> 3) & 1 : CHUNKS == 4 ? (r >> 2) & 3 : (r >> 1) & 7; }
};

// The scales and biases of 16 rows of both weights for a run of GROUPS groups: [weight][scales, biases][row][group].
template <int GROUPS>
struct Numbers {
    static constexpr int CHUNKS = GROUPS / 4, ARRAY = 16 * GROUPS * 4, BYTES = 4 * ARRAY, LOADS = ARRAY / 1024;  // of an array
    static __device__ __forceinline__ int swizzle(int r) { return CHUNKS == 4 ? (r >> 2) & 3 : (r >> 1) & 7; }
    static __device__ __forceinline__ int at(int array, int r, int g) { return array * ARRAY + r * (GROUPS * 4) + (((g >> 2) ^ swizzle(r)) * 4 + (g & 3)) * 4; }
};

typedef __attribute__((address_space(1))) void* gptr;
typedef __attribute__((address_space(3))) void* lptr;

// What a wavefront keeps to load codes (rows past N: the last one's bytes; their results go nowhere).
template <int BITS, int STEP>
struct CodesFrom {
    using C = Codes<BITS, STEP>;
    const char* codes[C::LOADS];
    unsigned row_bytes;
    int last, lane;
    __device__ __forceinline__ CodesFrom(const Args& a, int n0, int lane_) {
        n0 = n0 < a.N ? n0 : a.N - 1;  // (a wavefront past N)
        lane = lane_, last = a.N - 1 - n0, row_bytes = unsigned(a.K) * BITS / 8;
#pragma unroll
        for (int u = 0; u < C::LOADS; ++u)  // (one instruction has both weights, half its lanes each, or several one)
            codes[u] = reinterpret_cast<const char*>((u * 64 + lane) / (16 * C::CHUNKS) ? a.w[1].packed : a.w[0].packed) + size_t(n0) * row_bytes;
    }
    __device__ __forceinline__ void load(int s, char* to) const {
#pragma unroll
        for (int u = 0; u < C::LOADS; ++u) {
            const int i = u * 64 + lane, r = i / C::CHUNKS % 16, chunk = (i % C::CHUNKS) ^ C::swizzle(r);
            const unsigned at = unsigned(s) * C::ROW + unsigned(chunk) * 16;  // (past K: the row's first bytes, which meet zeros of x)
            __builtin_amdgcn_global_load_lds((gptr)(codes[u] + (unsigned(r < last ? r : last) * row_bytes + (at < row_bytes ? at : 0))),
                                             (lptr)(to + u * 1024), 16, 0, 0);
        }
    }
};

// Array `array` of a run of GROUPS groups from group g0 on.  16 bytes a lane where all rows are aligned, else 4; past the last group: others.
template <int GROUPS>
__device__ __forceinline__ void load_numbers(const Args& a, int array, int n0, int g0, char* table, int lane, bool aligned) {
    using B = Numbers<GROUPS>;
    n0 = n0 < a.N ? n0 : a.N - 1;
    const int last = a.N - 1 - n0, groups = a.K >> a.gs_shift;
    const Weight& w = array & 2 ? a.w[1] : a.w[0];
    const float* from = (array & 1 ? w.biases : w.scales) + size_t(n0) * groups;
    char* const to = table + array * B::ARRAY;
    if (aligned) {
#pragma unroll
        for (int u = 0; u < B::LOADS; ++u) {
            const int i = u * 64 + lane, r = i / B::CHUNKS, g = g0 + ((i % B::CHUNKS) ^ B::swizzle(r)) * 4;
            __builtin_amdgcn_global_load_lds((gptr)(from + (r < last ? r : last) * groups + (g < groups ? g : groups - 4)), (lptr)(to + u * 1024), 16, 0, 0);
        }
    } else {
#pragma unroll 1
        for (int u = 0; u < B::LOADS * 4; ++u) {
            const int i = u * 64 + lane, r = i / GROUPS, g = g0 + ((i % GROUPS / 4) ^ B::swizzle(r)) * 4 + i % 4;
            __builtin_amdgcn_global_load_lds((gptr)(from + (r < last ? r : last) * groups + (g < groups ? g : groups - 1)), (lptr)(to + u * 256), 4, 0, 0);
        }
    }
}

__device__ __forceinline__ bool numbers_aligned(const Args& a) {
    return (a.K >> a.gs_shift) % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.w[0].scales) | reinterpret_cast<uintptr_t>(a.w[0].biases) |
                                             reinterpret_cast<uintptr_t>(a.w[1].scales) | reinterpret_cast<uintptr_t>(a.w[1].biases)) & 15) == 0;
}

// y += the products of a step whose groups begin with g of the table; x_at(k, part, tile) is eight x from k on, in the codes' slots.
template <int PARTS, int BITS, int GS, int STEP, int TABLE, int MT, int RU, class F>
__device__ __forceinline__ void multiply(const char* at, const char* table, int g, int lane, float (&y)[2][MT][RU], F&& x_at) {
    using C = Codes<BITS, STEP>;
    using B = Numbers<TABLE>;
    constexpr int SEGS = GS < STEP ? STEP / GS : 1, IPS = STEP / 32 / SEGS, BYTES = IPS * BITS;  // instructions (32 k) of a group; a lane's bytes of one, consecutive
    const int ln = lane & 15, q = lane >> 4;
    const _Float16 o = _Float16(1.f);
    const v8h one{o, o, o, o, o, o, o, o};
#pragma unroll
    for (int e = 0; e < SEGS; ++e) {
        uint32_t wd[2][8];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int b = 0; b < (BYTES + 15) / 16; ++b) {
                const int byte = e * (C::ROW / SEGS) + q * BYTES + b * 16;
                const char* from = at + i * (16 * C::ROW) + ln * C::ROW + ((byte >> 4) ^ C::swizzle(ln)) * 16 + (byte & 15);
                if constexpr (BYTES >= 16) {
                    const u32x4 t = *reinterpret_cast<const u32x4*>(from);
#pragma unroll
                    for (int d = 0; d < 4; ++d) wd[i][b * 4 + d] = t[d];
                } else if constexpr (BYTES == 8) {
                    const u32x2 t = *reinterpret_cast<const u32x2*>(from);
                    wd[i][0] = t[0], wd[i][1] = t[1];
                } else {
                    wd[i][0] = *reinterpret_cast<const uint32_t*>(from);
                }
            }
        v4f acc[2][MT], sum[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[0][t] = acc[1][t] = sum[t] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ii = 0; ii < IPS; ++ii) {
            constexpr int W = BITS / 4;  // words of eight codes
            const uint32_t wg[4] = {wd[0][ii * W], wd[0][ii * W + W - 1], 0u, 0u}, wu[4] = {wd[1][ii * W], wd[1][ii * W + W - 1], 0u, 0u};
            const v8h cg = codes_f16<BITS>(wg, 0), cu = codes_f16<BITS>(wu, 0);
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    const v8h f = x_at(e * (STEP / SEGS) + q * (IPS * 8) + ii * 8, p, t);
                    acc[0][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, cg, acc[0][t], 0, 0, 0);
                    acc[1][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, cu, acc[1][t], 0, 0, 0);
                    sum[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, one, sum[t], 0, 0, 0);
                }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float sc = *reinterpret_cast<const float*>(table + B::at(2 * i, ln, g + e));
            const float b = __builtin_fmaf(-float(kWqCentre<BITS>), sc, *reinterpret_cast<const float*>(table + B::at(2 * i + 1, ln, g + e)));
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int r = 0; r < RU; ++r) y[i][t][r] = __builtin_fmaf(sc, acc[i][t][r], __builtin_fmaf(b, sum[t][r], y[i][t][r]));
        }
    }
}

// s_waitcnt immediates: vmcnt <= n alone, and with every LDS read done; every LDS read done
constexpr int vmcnt_only(int n) { return (n & 0xF) | ((n >> 4) << 14) | (0x7 << 4) | (0xF << 8); }
constexpr int vmcnt_and_lds(int n) { return (n & 0xF) | ((n >> 4) << 14) | (0x7 << 4); }
constexpr int kLdsDone = 0xF | (0x3 << 14) | (0x7 << 4);

__device__ __forceinline__ void pin() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// ---------------------------------------------------------------- up to four rows
constexpr int kFewTable = 32;
// (as many steps as three blocks a CU have room for)
template <int BITS>
constexpr int kFewRing = BITS == 4 ? 3 : 2;
template <int BITS>
constexpr int kFewFixed = kFewWaves * kFewRing<BITS> * Codes<BITS, kFewStep>::BYTES + 2 * Numbers<kFewTable>::BYTES;  // bytes of LDS without x
// For x where a CU has two blocks.  (One: 2 x 11008 x 4096, float32 and 8 bits, 37.3 us, by the other kernel 25.7; two: 4 bits, 26.4 and 27.7.)
template <int BITS>
constexpr int kFewRoom = 77 * 1024 - kFewFixed<BITS>;

template <class T, int PARTS, int BITS, int GS>
__global__ __launch_bounds__(64 * kFewWaves) void gated_few_kernel(Args a) {
    using C = Codes<BITS, kFewStep>;
    constexpr int RING = kFewRing<BITS>, LOADS = C::LOADS;
    constexpr int TURN = kFewTable * GS / (kFewStep * kFewWaves);  // steps of a wavefront for a table
    extern __shared__ __attribute__((aligned(1024))) char smem[];  // the wavefronts' rings, the tables, then x: [part][row][K rounded up to steps, and 8]
    __shared__ float s_y[kFewWaves][2][64];
    __shared__ float s_unscale[4], s_top[kFewWaves];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * 16, steps = (a.K + kFewStep - 1) / kFewStep;
    char* const ring = smem + wave * (RING * C::BYTES);
    char* const tables = smem + kFewWaves * RING * C::BYTES;
    char* const s_x = smem + kFewFixed<BITS>;
    const unsigned stride = unsigned(steps) * (kFewStep * 2) + 16, x_part = unsigned(a.M) * stride;  // bytes of a row, of a part
    const CodesFrom<BITS, kFewStep> from(a, n0, lane);
    const bool aligned = numbers_aligned(a);
    auto load = [&](int s, char* to) { from.load(s < steps ? s : steps - 1, to); };  // (past the end: any step, to keep the count)
    constexpr int QUADS = PARTS == 1 ? 1 : 2;
    const unsigned octets = unsigned(steps) * (kFewStep / 8), total = unsigned(a.M) * octets;
    auto fetch = [&](unsigned u, uint4 (&raw)[QUADS]) {
        u = u < total ? u : 0;
        const unsigned m = u / octets, k = (u - m * octets) * 8;
        __builtin_memcpy(raw, static_cast<const T*>(a.x) + size_t(m) * a.K + (k < unsigned(a.K) ? k : 0), 16 * QUADS);
    };
    auto place = [&](unsigned u, uint4 (&raw)[QUADS]) {
        if (u >= total) return;
        const unsigned m = u / octets, o = u - m * octets, at = m * stride + o * 16;
        if (o * 8 >= unsigned(a.K))
#pragma unroll
            for (int h = 0; h < QUADS; ++h) raw[h] = uint4{0u, 0u, 0u, 0u};
        if constexpr (PARTS == 1) {
            *reinterpret_cast<v8h*>(s_x + at) = slots_f16<BITS>(raw[0]);
        } else {
            float f[8];
            __builtin_memcpy(f, raw, 32);
            uint4 part[2];
            split_f16(f, 1.0f / s_unscale[m], part);
#pragma unroll
            for (int p = 0; p < 2; ++p) *reinterpret_cast<v8h*>(s_x + p * x_part + at) = slots_f16<BITS>(part[p]);
        }
    };
    if constexpr (PARTS == 2) {
        for (int m = 0; m < a.M; ++m) {
            float top = 0.f;
            for (unsigned c = threadIdx.x; c < unsigned(a.K) / 8; c += 64 * kFewWaves) {
                float f[8];
                __builtin_memcpy(f, static_cast<const float*>(a.x) + size_t(m) * a.K + c * 8, 32);
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(f[e]));
            }
#pragma unroll
            for (int d = 32; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
            __syncthreads();  // (the row before has been read)
            if (lane == 0) s_top[wave] = top;
            __syncthreads();
            if (threadIdx.x == 0) s_unscale[m] = row_unscale(fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3])));
        }
        __syncthreads();
    }
    load_numbers<kFewTable>(a, wave, n0, 0, tables, lane, aligned);  // (four arrays, four wavefronts)
    pin();
    // the first octets of a thread are under way before the weights
    uint4 first[2][QUADS];
    fetch(threadIdx.x, first[0]);
    fetch(threadIdx.x + 64 * kFewWaves, first[1]);
    pin();
#pragma unroll
    for (int d = 0; d < RING; ++d) load(wave + d * kFewWaves, ring + d * C::BYTES);
    pin();
    place(threadIdx.x, first[0]);
    place(threadIdx.x + 64 * kFewWaves, first[1]);
    for (unsigned u = threadIdx.x + 2 * 64 * kFewWaves; u < total; u += 64 * kFewWaves) {
        fetch(u, first[0]);
        place(u, first[0]);
    }
    const char* const x_row = s_x + unsigned(((lane & 15) >> 2) < a.M ? (lane & 15) >> 2 : 0) * stride;
    float y[2][1][1] = {};
    int slot = 0;
    for (int i = 0; i * kFewWaves < steps; ++i) {
        const char* const table = tables + (i / TURN & 1) * Numbers<kFewTable>::BYTES;
        if (i % TURN == 0) {
            // this wavefront's part of the table has landed (at least so many loads came after it); with everybody's, nobody reads the other
            pin();
            __builtin_amdgcn_s_waitcnt(vmcnt_and_lds(LOADS * (TURN < RING ? TURN : RING)));
            __builtin_amdgcn_s_barrier();
            pin();
            if ((i + TURN) * kFewWaves < steps)
                load_numbers<kFewTable>(a, wave, n0, (i / TURN + 1) * kFewTable, tables + ((i / TURN + 1) & 1) * Numbers<kFewTable>::BYTES, lane, aligned);
        }
        char* const at = ring + slot * C::BYTES;
        slot = slot + 1 == RING ? 0 : slot + 1;
        const int s = i * kFewWaves + wave;
        pin();
        __builtin_amdgcn_s_waitcnt(vmcnt_only(LOADS * (RING - 1)));
        pin();
        if (s < steps)
            multiply<PARTS, BITS, GS, kFewStep, kFewTable, 1, 1>(at, table, s * kFewStep / GS % kFewTable, lane, y, [&](int k, int p, int) {
                return *reinterpret_cast<const v8h*>(x_row + p * x_part + unsigned(s * kFewStep + k) * 2);
            });
        pin();
        __builtin_amdgcn_s_waitcnt(kLdsDone);  // the step has been read
        pin();
        load(s + RING * kFewWaves, at);
    }
    s_y[wave][0][lane] = y[0][0][0], s_y[wave][1][lane] = y[1][0][0];
    __builtin_amdgcn_s_waitcnt(vmcnt_and_lds(0));  // the loads past the end have landed before the LDS is given up
    __syncthreads();
    // a thread has a column and row q that lane column + 16 q holds
    const int n = n0 + (threadIdx.x & 15), m = threadIdx.x >> 4;
    if (n >= a.N || m >= a.M) return;
    float g = 0.f, u = 0.f;
#pragma unroll
    for (int p = 0; p < kFewWaves; ++p) g += s_y[p][0][threadIdx.x], u += s_y[p][1][threadIdx.x];
    if constexpr (PARTS == 2) g *= s_unscale[m & 3], u *= s_unscale[m & 3];
    if (a.w[0].bias) g += a.w[0].bias[n];
    if (a.w[1].bias) u += a.w[1].bias[n];
    static_cast<T*>(a.out)[size_t(m) * a.N + n] = T(activate(a.act, g) * u);
}

// ---------------------------------------------------------------- more rows
// A step is 128 k where LDS has room for two of them beside the tables, else 64 (16 x 11008 x 4096, 8 bits, float32, without the launch that
// splits x: 25.2 us, 28.9 with steps of 64 and a ring of four).
template <int PARTS, int BITS, int MT, int CG, int SG, int STEP>
constexpr int kRowsBytes = CG * SG * Codes<BITS, STEP>::BYTES + SG * PARTS * MT * STEP * 32;
template <int PARTS, int BITS, int GS, int MT, int CG, int SG>
struct RowsStep {
    static constexpr int WAVES = CG * SG, GROUPS = SG == 8 ? 32 : 16;  // of a table
    static constexpr int TABLE = CG * Numbers<GROUPS>::BYTES, ROOM = 158 * 1024 - 2 * TABLE;  // a table of the block's columns
    static constexpr int STEP = 2 * kRowsBytes<PARTS, BITS, MT, CG, SG, 128> <= ROOM ? 128 : 64, BYTES = kRowsBytes<PARTS, BITS, MT, CG, SG, STEP>;
    using C = Codes<BITS, STEP>;
    // x of each group of steps: [part][tile][16 rows of 2 STEP bytes], 1 KiB has 512 / STEP rows
    static constexpr int OCTETS = STEP / 8, ROWS = 512 / STEP, PIECES = PARTS * MT * 16 / ROWS;
    static constexpr int PER_WAVE = (PIECES + CG - 1) / CG;
    static constexpr int LOADS = C::LOADS + PER_WAVE;
    static constexpr int TURN = GROUPS * GS / (STEP * SG);  // iterations for a table: it has landed when RING - 2 are under way
    static constexpr int FIT = ROOM / BYTES, MOST = TURN < 2 ? TURN + 2 : 4, RING = FIT > MOST ? MOST : FIT;
    static_assert(RING >= 2 && LOADS * (RING - 2) <= 63 && TURN >= RING - 2, "");
    static __device__ __forceinline__ int swizzle(int r) { return STEP == 128 ? r : r >> 1; }
};

__device__ const uint4 kZeros = {0u, 0u, 0u, 0u};  // what a step past K has for x

template <class T, int PARTS, int BITS, int GS, int MT, int CG, int SG>
__global__ __launch_bounds__(64 * CG * SG) void gated_rows_kernel(Args a, RowsX rx) {
    using S = RowsStep<PARTS, BITS, GS, MT, CG, SG>;
    using C = typename S::C;
    extern __shared__ __attribute__((aligned(1024))) char smem[];  // the tables, the ring of steps; at the end the sums
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ln = lane & 15;
    const int cg = wave % CG, sg = wave / CG;
    const int n0 = (blockIdx.x * CG + cg) * 16, m0 = blockIdx.y * (16 * MT), steps = (a.K + S::STEP - 1) / S::STEP;
    const CodesFrom<BITS, S::STEP> from(a, n0, lane);
    const bool aligned = numbers_aligned(a);
    // this wavefront's pieces of x (rows past M: the last one's bytes; one that there is not: another's again)
    const _Float16* x_from[S::PER_WAVE];
    int x_piece[S::PER_WAVE], x_k[S::PER_WAVE];
#pragma unroll
    for (int u = 0; u < S::PER_WAVE; ++u) {
        x_piece[u] = (u * CG + cg) % S::PIECES;
        const int tile = x_piece[u] * S::ROWS / 16, r = x_piece[u] * S::ROWS % 16 + lane / S::OCTETS, m = m0 + tile % MT * 16 + r;
        x_from[u] = (tile / MT ? rx.part[PARTS - 1] : rx.part[0]) + size_t(m < a.M ? m : a.M - 1) * a.K;
        x_k[u] = ((lane % S::OCTETS) ^ (S::swizzle(r) % S::OCTETS)) * 8;
    }
    auto load = [&](int i, int slot) {
        const int want = i * SG + sg, s = want < steps ? want : steps - 1;  // past the end: any step, to keep the count
        char* const to = smem + 2 * S::TABLE + slot * S::BYTES;
        from.load(s, to + wave * C::BYTES);
#pragma unroll
        for (int u = 0; u < S::PER_WAVE; ++u) {
            const int k = s * S::STEP + x_k[u];
            __builtin_amdgcn_global_load_lds((gptr)(k < a.K ? reinterpret_cast<const char*>(x_from[u] + k) : reinterpret_cast<const char*>(&kZeros)),
                                             (lptr)(to + S::WAVES * C::BYTES + (sg * S::PIECES + x_piece[u]) * 1024), 16, 0, 0);
        }
    };
    float y[2][MT][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) y[i][t][r] = 0.f;
    // two arrays of its columns' tables are each wavefront's to load
    auto load_table = [&](int j) {
        char* const table = smem + (j & 1) * S::TABLE + cg * Numbers<S::GROUPS>::BYTES;
#pragma unroll
        for (int u = 0; u < (SG > 4 ? 1 : 4 / SG); ++u)
            load_numbers<S::GROUPS>(a, SG > 4 ? sg % 4 : sg * (4 / SG) + u, n0, j * S::GROUPS, table, lane, aligned);
    };
    load_table(0);
#pragma unroll
    for (int d = 0; d < S::RING - 1; ++d) load(d, d);
    int slot = 0;
    for (int i = 0; i * SG < steps; ++i) {
        pin();
        __builtin_amdgcn_s_waitcnt(vmcnt_and_lds(S::LOADS * (S::RING - 2)));
        __builtin_amdgcn_s_barrier();
        pin();
        if (i % S::TURN == 0 && (i + S::TURN) * SG < steps) load_table(i / S::TURN + 1);
        load(i + S::RING - 1, slot == 0 ? S::RING - 1 : slot - 1);  // (the slot that everybody has just left)
        const char* const at = smem + 2 * S::TABLE + slot * S::BYTES;
        slot = slot + 1 == S::RING ? 0 : slot + 1;
        const int s = i * SG + sg;
        if (s >= steps) continue;  // uniform: the other group's last step
        const char* const x = at + S::WAVES * C::BYTES + sg * (S::PIECES * 1024) + ln * (2 * S::STEP);
        const char* const table = smem + (i / S::TURN & 1) * S::TABLE + cg * Numbers<S::GROUPS>::BYTES;
        multiply<PARTS, BITS, GS, S::STEP, S::GROUPS, MT, 4>(at + wave * C::BYTES, table, s * S::STEP / GS % S::GROUPS, lane, y, [&](int k, int p, int t) {
            const u32x4 raw = *reinterpret_cast<const u32x4*>(x + (p * MT + t) * (32 * S::STEP) + ((k >> 3) ^ (S::swizzle(ln) % S::OCTETS)) * 16);
            return slots_f16<BITS>(uint4{raw[0], raw[1], raw[2], raw[3]});
        });
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_and_lds(0));  // the loads past the end have landed
    __syncthreads();
    float(*const s_y)[2][MT][4][64] = reinterpret_cast<float(*)[2][MT][4][64]>(smem);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) s_y[wave][i][t][r][lane] = y[i][t][r];
    __syncthreads();
    // a thread has a column and rows ROWS apart: element row % 4 of lane column + 16 (row / 4)
    constexpr int COLS = CG * 16, ROWS = 4 * SG;
    const int col = threadIdx.x % COLS, n = blockIdx.x * COLS + col;
    if (n >= a.N) return;
    const float bg = a.w[0].bias ? a.w[0].bias[n] : 0.f, bu = a.w[1].bias ? a.w[1].bias[n] : 0.f;
#pragma unroll 1  // (one copy of the activations: a block's first instructions come from memory)
    for (int j = 0; j < (16 * MT + ROWS - 1) / ROWS; ++j) {
        const int row = j * ROWS + threadIdx.x / COLS, m = m0 + row, t = row >> 4, from_lane = (col & 15) + 16 * ((row >> 2) & 3);
        if ((16 * MT % ROWS && row >= 16 * MT) || m >= a.M) return;
        float g = 0.f, u = 0.f;
#pragma unroll
        for (int p = 0; p < SG; ++p) {
            g += s_y[p * CG + (col >> 4)][0][t][row & 3][from_lane];
            u += s_y[p * CG + (col >> 4)][1][t][row & 3][from_lane];
        }
        if constexpr (PARTS == 2) g *= rx.unscale[m], u *= rx.unscale[m];
        static_cast<T*>(a.out)[size_t(m) * a.N + n] = T(activate(a.act, g + bg) * (u + bu));
    }
}

// A float32 row as two float16, and what undoes its factor: a block a row, up to 16384 of it in registers.
__global__ __launch_bounds__(512) void gated_split_kernel(const float* __restrict__ x, int K, _Float16* __restrict__ hi, _Float16* __restrict__ lo,
                                                          float* __restrict__ unscale) {
    constexpr int HELD = 4;
    __shared__ float s_top[8];
    const size_t base = size_t(blockIdx.x) * K;
    const unsigned octets = unsigned(K) / 8;
    float f[HELD][8], top = 0.f;
#pragma unroll
    for (int u = 0; u < HELD; ++u) {
        const unsigned c = u * 512 + threadIdx.x;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[u][e] = 0.f;
        if (c < octets) __builtin_memcpy(f[u], x + base + c * 8, 32);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(f[u][e]));
    }
    float g[8];
    for (unsigned c = HELD * 512 + threadIdx.x; c < octets; c += 512) {
        __builtin_memcpy(g, x + base + c * 8, 32);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(g[e]));
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    if ((threadIdx.x & 63) == 0) s_top[threadIdx.x >> 6] = top;
    __syncthreads();
    top = s_top[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) top = fmaxf(top, s_top[w]);
    const float u = row_unscale(top), factor = 1.0f / u;
    if (threadIdx.x == 0) unscale[blockIdx.x] = u;
    auto put = [&](unsigned c, const float(&v)[8]) {
        uint4 part[2];
        split_f16(v, factor, part);
        *reinterpret_cast<uint4*>(hi + base + c * 8) = part[0], *reinterpret_cast<uint4*>(lo + base + c * 8) = part[1];
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (i * 512 + threadIdx.x < octets) put(i * 512 + threadIdx.x, f[i]);
    for (unsigned c = HELD * 512 + threadIdx.x; c < octets; c += 512) {
        __builtin_memcpy(g, x + base + c * 8, 32);
        put(c, g);
    }
}

// f(BITS, GS) as constants
template <class F>
int by_group(int bits, int gs, F&& f) {
    using std::integral_constant;
    auto of_bits = [&](auto b) {
        if (gs == 32) return f(b, integral_constant<int, 32>{});
        if (gs == 64) return f(b, integral_constant<int, 64>{});
        return f(b, integral_constant<int, 128>{});
    };
    return bits == 4 ? of_bits(integral_constant<int, 4>{}) : of_bits(integral_constant<int, 8>{});
}

// f(MT, CG, SG) of a tile of kRowsTiles: eight wavefronts
template <int PARTS, int AT = 0, class F>
int by_tile(int tile, F&& f) {
    if constexpr (AT < kRowsTiles<PARTS>.size()) {
        using std::integral_constant;
        constexpr RowsTile t = kRowsTiles<PARTS>[AT];
        if (tile == AT) return f(integral_constant<int, t.mt>{}, integral_constant<int, t.cg>{}, integral_constant<int, 8 / t.cg>{});
        return by_tile<PARTS, AT + 1>(tile, f);
    }
    return fail(LQ_ERR_VALUE, "quantized_gated_matmul: no tile");
}

template <class T, int PARTS>
int launch_rows_chunk(const Args& a, int bits, int tile, hipStream_t st) {
    const auto lock = scratch_lock(st);
    RowsX rx{{static_cast<const _Float16*>(a.x), nullptr}, nullptr};
    if constexpr (PARTS == 2) {
        void* ws = nullptr;
        const size_t part = size_t(a.M) * a.K;
        if (const int rc = call_buffer(11, part * 4 + size_t(a.M) * 4, st, &ws)) return rc;
        _Float16* const hi = static_cast<_Float16*>(ws);
        float* const unscale = reinterpret_cast<float*>(hi + 2 * part);
        gated_split_kernel<<<unsigned(a.M), 512, 0, st>>>(static_cast<const float*>(a.x), a.K, hi, hi + part, unscale);
        LQ_CHECK_LAUNCH("quantized_gated_matmul");
        rx = RowsX{{hi, hi + part}, unscale};
    }
    return by_group(bits, 1 << a.gs_shift, [&](auto bits_c, auto gs_c) -> int {
        constexpr int BITS = decltype(bits_c)::value, GS = decltype(gs_c)::value;
        return by_tile<PARTS>(tile, [&](auto mt, auto cg, auto sg) -> int {
            constexpr int MT = decltype(mt)::value, CG = decltype(cg)::value, SG = decltype(sg)::value;
            using S = RowsStep<PARTS, BITS, GS, MT, CG, SG>;
            const dim3 grid((unsigned(a.N) + CG * 16 - 1) / (CG * 16), (unsigned(a.M) + 16 * MT - 1) / (16 * MT));
            const auto kernel = gated_rows_kernel<T, PARTS, BITS, GS, MT, CG, SG>;
            constexpr int need = 2 * S::TABLE + S::RING * S::BYTES, sums = S::WAVES * MT * 2048, lds = need > sums ? need : sums;
            static DeviceOnce once;
            if (const int rc = allow_dynamic_lds(once, reinterpret_cast<const void*>(kernel), lds)) return rc;
            kernel<<<grid, 64 * S::WAVES, lds, st>>>(a, rx);
            LQ_CHECK_LAUNCH("quantized_gated_matmul");
            return LQ_OK;
        });
    });
}

template <class T>
int launch_rows(Args a, int bits, int tile, hipStream_t st) {
    constexpr int PARTS = std::is_same_v<T, float> ? 2 : 1;
    LQ_REQUIRE(a.K < 1 << 26, LQ_ERR_SHAPE, "quantized_gated_matmul: K = %d", a.K);  // (offsets of 16 rows are 32-bit)
    const size_t few = size_t(PARTS) * a.M * ((a.K + kFewStep - 1) / kFewStep * (kFewStep * 2) + 16);
    if (a.M <= 4 && few <= size_t(bits == 4 ? kFewRoom<4> : kFewRoom<8>))
        return by_group(bits, 1 << a.gs_shift, [&](auto bits_c, auto gs_c) -> int {
            constexpr int BITS = decltype(bits_c)::value, GS = decltype(gs_c)::value;
            const auto kernel = gated_few_kernel<T, PARTS, BITS, GS>;
            static DeviceOnce once;
            if (const int rc = allow_dynamic_lds(once, reinterpret_cast<const void*>(kernel), kFewFixed<BITS> + kFewRoom<BITS>)) return rc;
            kernel<<<(unsigned(a.N) + 15) / 16, 64 * kFewWaves, kFewFixed<BITS> + few, st>>>(a);
            LQ_CHECK_LAUNCH("quantized_gated_matmul");
            return LQ_OK;
        });
    // rows in chunks of whole tiles whose parts stay below 2^30 bytes
    const int M = a.M, most = int(std::clamp<size_t>((size_t(1) << 28) / a.K / 64 * 64, 64, 65535 * 16));
    for (int m0 = 0; m0 < M; m0 += a.M) {
        a.M = std::min(most, M - m0);
        if (const int rc = launch_rows_chunk<T, PARTS>(a, bits, tile, st)) return rc;
        a.x = static_cast<const T*>(a.x) + size_t(a.M) * a.K, a.out = static_cast<T*>(a.out) + size_t(a.M) * a.N;
    }
    return LQ_OK;
}

}  // namespace
}  // namespace gated
}  // namespace lq

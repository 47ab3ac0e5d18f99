// Gated projections of many rows (wq_gated.hpp has the mathematics): bound by the matrix cores and the vector work beside them.
//
// gated_prepare_kernel lays out, once a call, what every block would otherwise make again: x in operand order (a fragment = 16 rows x 32 k
// of one part = 1 KiB, the lanes' 16 bytes in lane order), its sums over the groups and the groups' b + 2^(bits-1) s as operands of bfloat16
// parts, and the scales group after group.  float16 x enters as it is; a float32 row is multiplied by the power of two that brings its
// largest value below 2^15 and enters as two float16, hi = x rounded, lo = x - hi rounded: 22 bits, or 2^-39 of the largest value.
//
// gated_gemm_kernel: a block of four wavefronts takes 16 MT rows x 64 CT columns of both weights, a wavefront all rows x 16 CT columns of each, so
// that no code is turned into float16 twice in a block.  What a stage of 64 k needs comes from memory straight into LDS in pieces of
// 1 KiB per wavefront and instruction, in a ring of stages: every wavefront issues as many loads per stage, so that "stage s has arrived"
// is a count of outstanding loads.  The products of a group (at most 64 k) go to accumulators of their own, and from there with their scale to
// the sums.  The terms of b come last, as a product over the groups of three bfloat16 parts of each side, which leaves 2^-24 of them: whatever
// x's type, as they cancel against the codes' products wherever a group's middle is far from zero (two parts, 2^-16, left results of float16 off by ten
// steps and more behind a weight of one among small ones).
#pragma once
#include <algorithm>
#include <type_traits>

#include "wq_gated.hpp"

namespace lq {
namespace gated {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));  // (see wq_gated_rows.hpp on types in LDS)

constexpr int kPiece = 1024;  // bytes one wavefront moves into LDS with one instruction

constexpr int kSumParts = 3;

struct Prepared {
    char* x;          // [stage][row tile][2][part] pieces
    char* sums;       // [row tile][group step][sum part] pieces: groups as k
    char* biases;     // [weight][column tile of 16][group step][sum part] pieces
    float* scales;    // [group][block of columns][weight][64 CT]
    float* unscale;   // [row] of float32 x: what its row was multiplied by, inverse
    int mtiles, stages, group_steps, tiles_n;
};

// The power of two of each row: one wavefront a row.
__global__ __launch_bounds__(256) void gated_row_scale_kernel(const float* __restrict__ x, int M, int K, float* __restrict__ unscale) {
    const int m = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (m >= M) return;
    const float* row = x + size_t(m) * K;
    float top = 0.f;
    for (int k = lane * 4; k < K; k += 256) {  // K is a multiple of 32
        float4 v;
        __builtin_memcpy(&v, row + k, 16);
        top = fmaxf(fmaxf(fmaxf(top, fabsf(v.x)), fmaxf(fabsf(v.y), fabsf(v.z))), fabsf(v.w));
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    if (lane == 0) unscale[m] = row_unscale(top);
}

// Two kinds of blocks.  The first `x_blocks`: 16 rows x 128 k, a thread has eight k.  The others: 64 columns of a weight, a wavefront eight groups.
template <class T, int PARTS, int BITS, int CT>
__global__ __launch_bounds__(256) void gated_prepare_kernel(Args a, Prepared p, unsigned x_blocks) {
    constexpr int SP = kSumParts, kCols = 64 * CT;
    const int gs = 1 << a.gs_shift;
    if (blockIdx.x >= x_blocks) {
        const unsigned i = blockIdx.x - x_blocks, across = unsigned(p.tiles_n) * (kCols / 64), which = (i / across) & 1, lane = threadIdx.x & 63;
        const int octet = int(i / across / 2) * 4 + int(threadIdx.x >> 6), n = int(i % across) * 64 + int(lane), groups = a.K >> a.gs_shift;
        if (octet >= p.group_steps * 4) return;
        const Weight& w = a.w[which];
        float s[8], b[8];
        const size_t row = size_t(n < a.N ? n : a.N - 1) * groups;
        if (groups % 8 == 0 && aligned16(w.scales) && aligned16(w.biases)) {  // (a lane has a row: as few requests as can be)
            const size_t from = row + (octet * 8 < groups ? octet * 8 : 0);
            __builtin_memcpy(s, __builtin_assume_aligned(w.scales + from, 16), 32);
            __builtin_memcpy(b, __builtin_assume_aligned(w.biases + from, 16), 32);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const size_t from = row + (octet * 8 + e < groups ? octet * 8 + e : 0);
                s[e] = w.scales[from], b[e] = w.biases[from];
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int g = octet * 8 + e;
            const bool there = n < a.N && g < groups;
            s[e] = there ? s[e] : 0.f, b[e] = there ? b[e] - float(kWqCentre<BITS>) * s[e] : 0.f;
            // (what a stage past K asks for lies within group_steps * 32 groups)
            p.scales[(size_t(g) * p.tiles_n + n / kCols) * (2 * kCols) + which * kCols + n % kCols] = s[e];
        }
        uint32_t d[3][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) wq_split3x2(b[2 * j], b[2 * j + 1], d[0][j], d[1][j], d[2][j]);
        const size_t tile = size_t(which) * p.tiles_n * (kCols / 16) + n / 16;
#pragma unroll
        for (int part = 0; part < SP; ++part)
            reinterpret_cast<uint4*>(p.biases)[((tile * p.group_steps + octet / 4) * SP + part) * 64 + n % 16 + 16 * (octet % 4)] =
                uint4{d[part][0], d[part][1], d[part][2], d[part][3]};
        return;
    }
    const int mt = int(blockIdx.x % unsigned(p.mtiles)), pair = int(blockIdx.x / unsigned(p.mtiles));
    const int oct = threadIdx.x & 15, row = threadIdx.x >> 4, m = mt * 16 + row, k = pair * 128 + oct * 8, stage = pair * 2 + (oct >> 3);
    const bool there = m < a.M && k < a.K;  // K is a multiple of 32
    float v[8];
    uint4 piece[PARTS];
    if constexpr (PARTS == 1) {
        uint4 raw{0u, 0u, 0u, 0u};
        if (there) __builtin_memcpy(&raw, static_cast<const _Float16*>(a.x) + size_t(m) * a.K + k, 16);
        const v8h h = __builtin_bit_cast(v8h, raw);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = float(h[e]);
        piece[0] = __builtin_bit_cast(uint4, slots_f16<BITS>(raw));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
        float f = 1.0f;
        if (there) {
            __builtin_memcpy(v, static_cast<const float*>(a.x) + size_t(m) * a.K + k, 32);
            f = 1.0f / p.unscale[m];  // (powers of two)
        }
        uint4 part[2];
        split_f16(v, f, part);
#pragma unroll
        for (int i = 0; i < 2; ++i) piece[i] = __builtin_bit_cast(uint4, slots_f16<BITS>(part[i]));
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= f;
    }
    if (stage < p.stages) {
#pragma unroll
        for (int part = 0; part < PARTS; ++part)
            reinterpret_cast<uint4*>(p.x)[(((size_t(stage) * p.mtiles + mt) * 2 + ((oct >> 2) & 1)) * PARTS + part) * 64 + row + 16 * (oct & 3)] = piece[part];
    }
    float sum = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    sum += __shfl_xor(sum, 1, 64);
    sum += __shfl_xor(sum, 2, 64);
    if (gs >= 64) sum += __shfl_xor(sum, 4, 64);
    if (gs == 128) sum += __shfl_xor(sum, 8, 64);
    const int g = k >> a.gs_shift;
    if ((oct & (gs / 8 - 1)) == 0 && g < p.group_steps * 32) {
        uint32_t d[3];
        wq_split3x2(sum, 0.f, d[0], d[1], d[2]);
#pragma unroll
        for (int part = 0; part < SP; ++part)
            reinterpret_cast<uint16_t*>(p.sums)[(((size_t(mt) * p.group_steps + g / 32) * SP + part) * 64 + row + 16 * (g % 32 / 8)) * 8 + g % 8] = uint16_t(d[part]);
    }
}

// What a stage of one block is made of, in pieces.
template <int PARTS, int BITS, int GS, int MT, int CT>
struct Stage {
    static constexpr int SEGS = GS == 32 ? 2 : 1;     // groups of a stage
    static constexpr int X = 2 * MT * PARTS;          // fragments
    static constexpr int S = SEGS * CT / 2;           // 64 CT scales of both weights
    static constexpr int W = CT * BITS;               // 64 CT rows of 8 BITS bytes, of both
    static constexpr int PIECES = X + S + W;
    static constexpr int PER_WAVE = (PIECES + 3) / 4;
    static constexpr int FIT = 80 / PIECES;  // two blocks a CU
    static constexpr int RING = FIT > 4 ? 4 : FIT;
    static_assert(RING >= 2 && PER_WAVE * (RING - 2) <= 63, "");
};

// Row tiles of sums that a block has in LDS at once: all, or a half or a third, so that two blocks fit a CU.
__host__ __device__ constexpr int epilogue_rows(int mt, int ct) { return mt * ct <= 8 ? mt : mt % 2 == 0 ? mt / 2 : mt / 3; }

// s_waitcnt immediate for vmcnt <= n and every LDS read done
constexpr int vmcnt_lds(int n) { return (n & 0xF) | ((n >> 4) << 14) | (0x7 << 4); }

template <class T, int PARTS, int BITS, int GS, int MT, int CT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void gated_gemm_kernel(Args a, Prepared p, int tiles_m) {
    using S = Stage<PARTS, BITS, GS, MT, CT>;
    constexpr int SP = kSumParts, kCols = 64 * CT, JT = 2 * CT;  // column tiles of a wavefront: the gate's, then the other's
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ln = lane & 15, q = lane >> 4;
    // every XCD gets a contiguous range of tiles, row tiles first: its L2 then reads a weight row once
    const int nblk = gridDim.x, xcd = blockIdx.x & 7, quot = nblk >> 3, rem = nblk & 7;
    const int lid = xcd * quot + (xcd < rem ? xcd : rem) + (int(blockIdx.x) >> 3);
    const int tn = lid / tiles_m, tm = lid - tn * tiles_m;

    // ---- the loads of a stage: piece u * 4 + wave (the last round repeats pieces: the counts stay equal)
    constexpr int ROW = 8 * BITS, CH = ROW / 16;  // bytes of codes per row and stage; 16-byte chunks
    const unsigned row_bytes = unsigned(a.K) * BITS / 8;
    // A piece's address is a scalar, which goes on by `step` from stage to stage, and a lane's offset: no branch, next to no vector work.
    const char* src[S::PER_WAVE];
    size_t step[S::PER_WAVE];
    unsigned off[S::PER_WAVE], back[S::PER_WAVE];
    bool twice[S::PER_WAVE];  // (scales of groups of 128: every second stage)
#pragma unroll
    for (int u = 0; u < S::PER_WAVE; ++u) {
        int at = u * 4 + wave;
        at = at < S::PIECES ? at : at - 4;
        off[u] = unsigned(lane) * 16, back[u] = 0, twice[u] = false;
        if (at < S::X) {
            src[u] = p.x + size_t(tm) * (S::X * kPiece) + at * kPiece;
            step[u] = size_t(p.mtiles) * (2 * PARTS * kPiece);
        } else if (at < S::X + S::S) {
            const int i = at - S::X;  // CT / 2 pieces a group
            src[u] = reinterpret_cast<const char*>(p.scales) + (size_t(i / (CT / 2)) * p.tiles_n + tn) * (CT / 2 * kPiece) + i % (CT / 2) * kPiece;
            step[u] = size_t(S::SEGS) * p.tiles_n * (CT / 2 * kPiece), twice[u] = GS == 128;
        } else {
            // the chunks of a row change places with its number, so that the 16 rows of an operand lie in different banks
            const int i = at - (S::X + S::S), which = i / (S::W / 2), r = i % (S::W / 2) * (64 / CH) + lane / CH;
            const int n = tn * kCols + r < a.N ? tn * kCols + r : a.N - 1, chunk = (lane % CH) ^ ((r / (16 / CH)) % CH);
            src[u] = reinterpret_cast<const char*>(which ? a.w[1].packed : a.w[0].packed);
            step[u] = ROW;
            off[u] = unsigned(n) * row_bytes + unsigned(chunk) * 16;
            // the second half of a stage that ends half-way is past the row: the first half again (its x is zero)
            back[u] = GS == 32 && chunk >= CH / 2 && a.K % 64 ? ROW / 2 : 0;
        }
    }
    int loaded = 0;  // the stage that src is at
    auto load_stage = [&](int slot) {
        const bool last = loaded >= p.stages - 1;
#pragma unroll
        for (int u = 0; u < S::PER_WAVE; ++u) {
            int at = u * 4 + wave;
            at = at < S::PIECES ? at : at - 4;
            unsigned o = off[u];
            if constexpr (GS == 32) o -= last ? back[u] : 0;  // (K is a multiple of 64 otherwise)
            __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)(src[u] + o),
                                             (__attribute__((address_space(3))) void*)(smem + (slot * S::PIECES + at) * kPiece), 16, 0, 0);
            // past the end: the last stage again, to keep the count
            src[u] += last || (GS == 128 && twice[u] && loaded % 2 == 0) ? 0 : step[u];
        }
        ++loaded;
    };

    v4f y[JT][MT];
#pragma unroll
    for (int j = 0; j < JT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) y[j][i] = v4f{0.f, 0.f, 0.f, 0.f};
    v4f acc[2][S::SEGS][MT];
    float f_last[S::SEGS];
#pragma unroll
    for (int e = 0; e < S::SEGS; ++e) {
        f_last[e] = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[1][e][i] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    auto scale_sums = [&](int j, const float(&f)[S::SEGS], const v4f(&sums)[S::SEGS][MT]) {
#pragma unroll
        for (int e = 0; e < S::SEGS; ++e)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) y[j][i][r] = __builtin_fmaf(f[e], sums[e][i][r], y[j][i][r]);
    };
#pragma unroll
    for (int s = 0; s < S::RING - 1; ++s) load_stage(s);
    int slot = 0;
    for (int s = 0; s < p.stages; ++s) {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(vmcnt_lds(S::PER_WAVE * (S::RING - 2)));
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        load_stage(slot == 0 ? S::RING - 1 : slot - 1);  // (the slot that everybody has just left)
        const char* base = smem + slot * (S::PIECES * kPiece);
        slot = slot + 1 == S::RING ? 0 : slot + 1;
        const char* codes = base + (S::X + S::S) * kPiece;
        v8h x[2][MT][PARTS];
#pragma unroll
        for (int ii = 0; ii < 2; ++ii)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int part = 0; part < PARTS; ++part)
                    x[ii][i][part] = *reinterpret_cast<const v8h*>(base + ((i * 2 + ii) * PARTS + part) * kPiece + lane * 16);
        // Column tile j is multiplied while the sums of the one before it are scaled (of the last: in the next stage) and the codes of the one
        // behind it are decoded.
        uint32_t raw[JT][2][BITS / 4];
#pragma unroll
        for (int j = 0; j < JT; ++j) {
            const int r = (wave * CT + j % CT) * 16 + ln;
            const char* row = codes + j / CT * (S::W / 2 * kPiece) + r * ROW;
#pragma unroll
            for (int ii = 0; ii < 2; ++ii) {
                if constexpr (BITS == 4) {
                    raw[j][ii][0] = *reinterpret_cast<const uint32_t*>(row + (ii ^ ((r >> 3) & 1)) * 16 + q * 4);
                } else {
                    const u32x2 t = *reinterpret_cast<const u32x2*>(row + ((ii * 2 + (q >> 1)) ^ ((r >> 2) & 3)) * 16 + (q & 1) * 8);
                    raw[j][ii][0] = t[0], raw[j][ii][BITS / 4 - 1] = t[1];
                }
            }
        }
        auto decode = [&](int j, v8h(&c)[2]) {
#pragma unroll
            for (int ii = 0; ii < 2; ++ii) {
                const uint32_t wd[4] = {raw[j][ii][0], raw[j][ii][BITS / 4 - 1], 0u, 0u};
                c[ii] = codes_f16<BITS>(wd, 0);
            }
        };
        float f[JT][S::SEGS];
#pragma unroll
        for (int j = 0; j < JT; ++j)
#pragma unroll
            for (int e = 0; e < S::SEGS; ++e)
                f[j][e] = *reinterpret_cast<const float*>(base + (S::X + e * (CT / 2)) * kPiece + (j / CT * kCols + (wave * CT + j % CT) * 16 + ln) * 4);
        v8h c[2][2];
        decode(0, c[0]);
#pragma unroll
        for (int j = 0; j < JT; ++j) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int ii = 0; ii < 2; ++ii)
#pragma unroll
                for (int part = 0; part < PARTS; ++part)
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        const int e = S::SEGS == 2 ? ii : 0;
                        const bool first = part == 0 && (S::SEGS == 2 || ii == 0);
                        acc[j & 1][e][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[ii][i][part], c[j & 1][ii], first ? v4f{0.f, 0.f, 0.f, 0.f} : acc[j & 1][e][i], 0, 0, 0);
                    }
            scale_sums(j == 0 ? JT - 1 : j - 1, j == 0 ? f_last : f[j - 1], acc[(j & 1) ^ 1]);
            if (j < JT - 1) decode(j + 1, c[(j & 1) ^ 1]);
            constexpr int MFMAS = 2 * PARTS * MT, VALU = (4 * MT * S::SEGS + 2 * (BITS == 4 ? 9 : 8)) / MFMAS + 1;
#pragma unroll
            for (int k = 0; k < MFMAS; ++k) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < S::SEGS; ++e) f_last[e] = f[JT - 1][e];
    }
    scale_sums(JT - 1, f_last, acc[1]);
    // the terms of b, the small ones first: those of 2^-16 of hi hi, of 2^-8, itself
#pragma unroll 1
    for (int g = 0; g < p.group_steps; ++g) {
        v8bf sums[MT][SP];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int part = 0; part < SP; ++part)
                sums[i][part] = __builtin_bit_cast(v8bf, reinterpret_cast<const uint4*>(p.sums)[((size_t(tm * MT + i) * p.group_steps + g) * SP + part) * 64 + lane]);
#pragma unroll
        for (int j = 0; j < JT; ++j) {
            const size_t tile = size_t(j / CT) * p.tiles_n * (kCols / 16) + tn * (kCols / 16) + wave * CT + j % CT;
            v8bf b[SP];
#pragma unroll
            for (int part = 0; part < SP; ++part)
                b[part] = __builtin_bit_cast(v8bf, reinterpret_cast<const uint4*>(p.biases)[((tile * p.group_steps + g) * SP + part) * 64 + lane]);
#pragma unroll
            for (int order = SP - 1; order >= 0; --order)
#pragma unroll
                for (int part = 0; part <= order; ++part)
#pragma unroll
                    for (int i = 0; i < MT; ++i) y[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(sums[i][part], b[order - part], y[j][i], 0, 0, 0);
        }
    }
    // A wavefront's sums go through LDS, ROWS tiles at a time, so that a lane has four columns of a row and the activations stand in the code once: a block's
    // first instructions come from memory (sigmoid of each accumulator by itself: 2048 x 11008 x 4096 float16 465 us, so 453; 2896 x 3864 x 128 51 and 44).
    constexpr int ROWS = epilogue_rows(MT, CT), STRIDE = 16 * CT + 4, QUADS = 4 * CT;
    __builtin_amdgcn_s_waitcnt(vmcnt_lds(0));  // the loads past the end have landed
    __syncthreads();                           // and everybody has left the ring
    float(*const s_y)[16 * ROWS][STRIDE] = reinterpret_cast<float(*)[16 * ROWS][STRIDE]>(smem) + 2 * wave;
    const int col = lane % QUADS * 4, n = tn * kCols + wave * (16 * CT) + col;
    float bias[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) bias[i][e] = a.w[i].bias ? a.w[i].bias[n + e < a.N ? n + e : a.N - 1] : 0.f;
#pragma unroll
    for (int i0 = 0; i0 < MT; i0 += ROWS) {
        // accumulator element r of a lane: row 4 * quarter + r, column lane % 16
#pragma unroll
        for (int j = 0; j < JT; ++j)
#pragma unroll
            for (int i = 0; i < ROWS; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) s_y[j / CT][i * 16 + q * 4 + r][j % CT * 16 + ln] = y[j][i0 + i][r];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (of this wavefront alone)
#pragma unroll 1
        for (int row = lane / QUADS; row < 16 * ROWS; row += 64 / QUADS) {
            const int m = (tm * MT + i0) * 16 + row;
            if (m >= a.M) break;
            const v4f g4 = *reinterpret_cast<const v4f*>(&s_y[0][row][col]), u4 = *reinterpret_cast<const v4f*>(&s_y[1][row][col]);
            const float f = PARTS == 1 ? 1.0f : p.unscale[m];
            T h[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = T(activate(a.act, g4[e] * f + bias[0][e]) * (u4[e] * f + bias[1][e]));
            T* const to = static_cast<T*>(a.out) + size_t(m) * a.N + n;
            if (n + 4 <= a.N) {
                __builtin_memcpy(to, h, sizeof h);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n + e < a.N) to[e] = h[e];
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

template <class T, int PARTS, int BITS, int GS, int MT, int CT>
int launch_gemm_tile(const Args& a, hipStream_t st) {
    using S = Stage<PARTS, BITS, GS, MT, CT>;
    constexpr int SP = kSumParts, kCols = 64 * CT;
    Prepared p;
    const int tiles_m = (a.M + 16 * MT - 1) / (16 * MT);
    p.mtiles = tiles_m * MT, p.stages = (a.K + 63) / 64, p.group_steps = (a.K / GS + 31) / 32, p.tiles_n = (a.N + kCols - 1) / kCols;
    const size_t x_bytes = size_t(p.stages) * p.mtiles * (2 * PARTS * kPiece), sum_bytes = size_t(p.mtiles) * p.group_steps * (SP * kPiece);
    const size_t bias_bytes = size_t(2) * p.tiles_n * (kCols / 16) * p.group_steps * (SP * kPiece);
    const size_t scale_bytes = size_t(p.group_steps) * 32 * p.tiles_n * (CT / 2 * kPiece), unscale_bytes = PARTS == 1 ? 0 : size_t(a.M) * 4;
    const auto lock = scratch_lock(st);
    void* ws = nullptr;
    if (const int rc = call_buffer(11, x_bytes + sum_bytes + bias_bytes + scale_bytes + unscale_bytes, st, &ws)) return rc;
    p.x = static_cast<char*>(ws), p.sums = p.x + x_bytes, p.biases = p.sums + sum_bytes;
    p.scales = reinterpret_cast<float*>(p.biases + bias_bytes), p.unscale = reinterpret_cast<float*>(p.biases + bias_bytes + scale_bytes);
    if constexpr (PARTS == 2) {
        gated_row_scale_kernel<<<unsigned((a.M + 3) / 4), 256, 0, st>>>(static_cast<const float*>(a.x), a.M, a.K, p.unscale);
        LQ_CHECK_LAUNCH("quantized_gated_matmul");
    }
    // 128 k a block, all that the sums' steps of 32 groups reach over
    const unsigned x_blocks = unsigned(p.mtiles) * unsigned(p.group_steps * 32 * GS / 128);
    const unsigned w_blocks = unsigned(p.tiles_n) * (kCols / 64) * 2 * unsigned(p.group_steps);
    gated_prepare_kernel<T, PARTS, BITS, CT><<<x_blocks + w_blocks, 256, 0, st>>>(a, p, x_blocks);
    LQ_CHECK_LAUNCH("quantized_gated_matmul");
    static DeviceOnce once;
    constexpr int ring = S::RING * S::PIECES * kPiece, sums = 4 * 2 * 16 * epilogue_rows(MT, CT) * (16 * CT + 4) * 4, lds = ring > sums ? ring : sums;
    const auto kernel = gated_gemm_kernel<T, PARTS, BITS, GS, MT, CT>;
    if (const int rc = allow_dynamic_lds(once, reinterpret_cast<const void*>(kernel), lds)) return rc;
    kernel<<<unsigned(tiles_m) * unsigned(p.tiles_n), 256, lds, st>>>(a, p, tiles_m);
    LQ_CHECK_LAUNCH("quantized_gated_matmul");
    return LQ_OK;
}

// Rows in chunks whose prepared x stays below 2^30 bytes; whole tiles, so that the bits do not depend on them.
template <class T, int PARTS, int BITS, int GS, int MT, int CT>
int launch_gemm_chunks(Args a, hipStream_t st) {
    const size_t tile = size_t((a.K + 63) / 64) * (2 * PARTS * MT) * kPiece, tiles = tile < size_t(1) << 30 ? (size_t(1) << 30) / tile : 1;
    const int M = a.M, rows = int(std::min<size_t>(tiles * 16 * MT, size_t(M)));
    for (int m0 = 0; m0 < M; m0 += a.M) {
        a.M = std::min(rows, M - m0);
        if (const int rc = launch_gemm_tile<T, PARTS, BITS, GS, MT, CT>(a, st)) return rc;
        a.x = static_cast<const T*>(a.x) + size_t(a.M) * a.K, a.out = static_cast<T*>(a.out) + size_t(a.M) * a.N;
    }
    return LQ_OK;
}

// f(MT, CT) of a tile of kGemmTiles
template <int PARTS, int BITS, int AT = 0, class F>
int by_gemm_tile(int tile, F&& f) {
    if constexpr (AT < kGemmTiles<PARTS, BITS>.size()) {
        constexpr GemmTile t = kGemmTiles<PARTS, BITS>[AT];
        if (tile == AT) return f(std::integral_constant<int, t.mt>{}, std::integral_constant<int, t.ct>{});
        return by_gemm_tile<PARTS, BITS, AT + 1>(tile, f);
    }
    return fail(LQ_ERR_VALUE, "quantized_gated_matmul: no tile");
}

template <class T, int PARTS, int BITS>
int launch_gemm(const Args& a, int tile, hipStream_t st) {
    auto of_group = [&](auto gs_c) -> int {
        constexpr int GS = decltype(gs_c)::value;
        return by_gemm_tile<PARTS, BITS>(tile, [&](auto mt, auto ct) -> int {
            return launch_gemm_chunks<T, PARTS, BITS, GS, decltype(mt)::value, decltype(ct)::value>(a, st);
        });
    };
    const int gs = 1 << a.gs_shift;
    if (gs == 32) return of_group(std::integral_constant<int, 32>{});
    if (gs == 64) return of_group(std::integral_constant<int, 64>{});
    return of_group(std::integral_constant<int, 128>{});
}

}  // namespace
}  // namespace gated
}  // namespace lq

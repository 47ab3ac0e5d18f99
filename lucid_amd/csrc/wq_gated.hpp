// Both projections of a gated feed-forward block on group-wise int4 / int8 weights, with the activation and the product:
//
//   h[m, n] = act(g[m, n] + bg[n]) * (u[m, n] + bu[n])
//   g, u [m, n] = sum over groups of  s[n, group] * (sum_{k in group} c[n, k] x[m, k])  +  b[n, group] * (sum_{k in group} x[m, k])
//
// for the weights of the gate and of the way up.  Codes enter the matrix instructions as the whole numbers c - 2^(bits-1) that they are
// (the rest of the code goes to b, and b + 2^(bits-1) s is rounded to float32), so that nothing else of a weight is rounded: scales follow in float32, on
// the sums of a group.  float16 x enters as it is; a float32 row times a power of two as two float16 of 22 bits together.
#pragma once
#include <array>

#include "wq_pack.hpp"

namespace lq {
namespace gated {

enum Act { kSilu = 0, kGelu = 1, kRelu = 2, kSigmoid = 3 };

struct Weight {
    const uint32_t* packed;      // [N, K * bits / 32]
    const float *scales, *biases;  // [N, K / group]
    const float* bias;           // [N] or NULL
};

struct Args {
    const void* x;
    void* out;
    Weight w[2];  // gate, up
    int M, N, K, gs_shift, act;
};

namespace {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float activate(int act, float g) {
    if (act == kSilu) return g / (1.0f + expf(-g));
    if (act == kGelu) return 0.5f * g * erfcf(g * -0.70710678118654752440f);  // (erfc: nothing cancels below zero)
    if (act == kRelu) return g < 0.0f ? 0.0f : g;
    return 1.0f / (1.0f + expf(-g));
}

// The codes of instruction i of a window (see wq_codes) as float16: c - 2^(bits-1), exactly.  A 4-bit code under the upper bits of 1024
// is 1024 + c; four bits further up 1024 + 16 c, a sixteenth of which is 64 + c.  Slots as wq_codes has them.
template <int BITS>
__device__ __forceinline__ v8h codes_f16(const uint32_t (&wd)[4], int i) {
    union { v2h h[4]; v8h all; } f;
    auto half2 = [](uint32_t u) { return __builtin_bit_cast(v2h, u); };
    if constexpr (BITS == 4) {
        uint32_t low = 0x000f000fu, high = 0x00f000f0u, one = 0x64006400u;
        asm("" : "+s"(low));  // in registers: an AND-OR takes one literal at most
        asm("" : "+s"(high));
        asm("" : "+v"(one));
        const uint32_t c = wd[i], d = c >> 8;
        const v2h off{_Float16(-1032.f), _Float16(-1032.f)}, unit{_Float16(0.0625f), _Float16(0.0625f)}, off16{_Float16(-72.f), _Float16(-72.f)};
        f.h[0] = half2((c & low) | one) + off;
        f.h[1] = __builtin_elementwise_fma(half2((c & high) | one), unit, off16);
        f.h[2] = half2((d & low) | one) + off;
        f.h[3] = __builtin_elementwise_fma(half2((d & high) | one), unit, off16);
    } else {
        const v2h off{_Float16(-1152.f), _Float16(-1152.f)};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t c = wd[(2 * i + j) & 3];
            f.h[2 * j] = half2(__builtin_amdgcn_perm(0x64646464u, c, 0x04010400u)) + off;
            f.h[2 * j + 1] = half2(__builtin_amdgcn_perm(0x64646464u, c, 0x04030402u)) + off;
        }
    }
    return f.all;
}

// Eight consecutive x in the slots of the codes: of 4 bits element d beside d + 4.
template <int BITS>
__device__ __forceinline__ v8h slots_f16(uint4 x) {
    if constexpr (BITS == 8) return __builtin_bit_cast(v8h, x);
    auto low = [](uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); };
    auto high = [](uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); };
    return __builtin_bit_cast(v8h, uint4{low(x.x, x.z), high(x.x, x.z), low(x.y, x.w), high(x.y, x.w)});
}

// What undoes the factor of a float32 row whose largest value is `top` = 2^e t, t in [0.5, 1): 2^(e - 15), within what a float32 and its
// inverse can say.  (A row that is not finite keeps its values, and gives no number.)
__device__ __forceinline__ float row_unscale(float top) {
    int e = 15;
    if (top > 0.f && top < __builtin_inff()) frexpf(top, &e);
    return ldexpf(1.0f, (e < -111 ? -111 : e) - 15);
}
// Eight values times f as two float16 each
__device__ __forceinline__ void split_f16(const float (&v)[8], float f, uint4 (&part)[2]) {
    v8h hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) hi[e] = _Float16(v[e] * f), lo[e] = _Float16(v[e] * f - float(hi[e]));
    part[0] = __builtin_bit_cast(uint4, hi), part[1] = __builtin_bit_cast(uint4, lo);
}

}  // namespace

// Few rows or columns (wq_gated_rows.hpp): 16 mt rows x 16 cg columns a block, and what 64 k of it take (us), on average of 4 and 8 bits: measured with
// 6 to 256 rows and 512 to 11008 columns at K = 4096 and 14336.  bits 4 or 8, groups of 32, 64 or 128; `tile` of these.
struct RowsTile {
    int mt, cg;
    float us;
};
template <int PARTS>  // (of a float32 x there is no room for more)
constexpr std::array<RowsTile, 6> kRowsTiles = {{{4, 4, 0.80f}, {2, 4, 0.47f}, {2, 2, 0.28f}, {1, 4, 0.30f}, {1, 2, 0.175f}, {1, 1, 0.112f}}};
template <>
inline constexpr std::array<RowsTile, 7> kRowsTiles<1> = {
    {{4, 4, 0.45f}, {2, 4, 0.27f}, {2, 2, 0.152f}, {2, 1, 0.109f}, {1, 4, 0.21f}, {1, 2, 0.115f}, {1, 1, 0.0625f}}};
int launch_rows_f16(const Args& a, int bits, int tile, hipStream_t st);
int launch_rows_f32(const Args& a, int bits, int tile, hipStream_t st);

// Many rows (wq_gated_gemm.hpp): 16 mt rows x 64 ct columns a block, and what a stage of 64 k takes (us) when a CU has one block, or two: measured
// with 4-bit codes in groups of 128 at K = 4096, N = 11008 and 64 to 2048 rows, without what a round takes besides.  (8-bit codes of wide blocks leave no room for a ring of stages.)
struct GemmTile {
    int mt, ct;
    float one, two;
};
template <int PARTS, int BITS>
constexpr std::array<GemmTile, 3> kGemmTiles = {{{4, 2, 0.89f, 1.11f}, {6, 2, 1.09f, 1.58f}, {3, 4, 1.26f, 1.81f}}};
template <>
inline constexpr std::array<GemmTile, 2> kGemmTiles<1, 8> = {{{4, 2, 0.89f, 1.11f}, {6, 2, 1.09f, 1.58f}}};
template <>
inline constexpr std::array<GemmTile, 4> kGemmTiles<2, 4> = {{{2, 2, 0.85f, 1.08f}, {4, 2, 1.25f, 1.76f}, {2, 4, 1.30f, 2.13f}, {3, 4, 1.60f, 2.73f}}};
template <>
inline constexpr std::array<GemmTile, 3> kGemmTiles<2, 8> = {{{2, 2, 0.85f, 1.08f}, {3, 2, 1.10f, 1.36f}, {4, 2, 1.25f, 1.76f}}};
// By type and bits, `tile` of these; weights below 2 GiB.
int launch_gemm_f16_4(const Args& a, int tile, hipStream_t st);
int launch_gemm_f16_8(const Args& a, int tile, hipStream_t st);
int launch_gemm_f32_4(const Args& a, int tile, hipStream_t st);
int launch_gemm_f32_8(const Args& a, int tile, hipStream_t st);

}  // namespace gated
}  // namespace lq

// Gated projections on group-wise weights: the entry point, and which kernel takes a call (wq_gated.hpp).
#include "wq_gated.hpp"

using namespace lq;

namespace {

struct Choice {
    int tile;  // of the kernel of many rows; -1: the one of few
    float us;
};

// The kernel, and of the one of many rows the tile, that takes the least time as rounds of blocks: for few rows one block a CU, for many two, or one
// where a last round has no more than 256.  Few rows take 0.3 to 0.53 us for 64 k (float32, two parts of x: 0.4 to 1), and 5 us before for splitting
// float32; many rows 6 or 12 us before for laying out their operands.  us, few / many, 4 bits in groups of 128, K = 4096: 64 x 11008 float16 34 / 52, 65
// 64 / 60, 128 66 / 69, 128 x 4096 (8 bits) 36 / 57; 64 x 11008 float32 70 / 72, 65 125 / 77.
Choice choose(const gated::Args& a, bool half, int bits) {
    const gated::GemmTile* const tiles = half ? (bits == 4 ? gated::kGemmTile<1, 4> : gated::kGemmTile<1, 8>) : (bits == 4 ? gated::kGemmTile<2, 4> : gated::kGemmTile<2, 8>);
    const int few_tiles = a.M <= 16 ? 1 : a.M <= 32 ? 2 : 4;
    const int64_t few_blocks = (int64_t(a.N) + 63) / 64 * ((int64_t(a.M) + 16 * few_tiles - 1) / (16 * few_tiles)), stages = (a.K + 63) / 64;
    const float per_stage = half ? (few_tiles == 1 ? 0.30f : few_tiles == 2 ? 0.36f : 0.53f) : (few_tiles == 1 ? 0.40f : few_tiles == 2 ? 0.50f : 1.0f);
    Choice best{-1, (half ? 0.f : 5.f) + float((few_blocks + 255) / 256) * float(stages) * per_stage};
    if (size_t(a.N) * a.K * bits / 8 >= 0x7fffffffull) return best;  // (offsets of codes are 32-bit in the kernel of many rows)
    for (int t = 0; t < gated::kGemmTiles && tiles[t].mt; ++t) {
        const gated::GemmTile& tile = tiles[t];
        const int64_t blocks = (int64_t(a.M) + 16 * tile.mt - 1) / (16 * tile.mt) * ((int64_t(a.N) + 64 * tile.ct - 1) / (64 * tile.ct)), rest = blocks % 512;
        const float us = (half ? 6.f : 12.f) + float(stages) * (float(blocks / 512) * tile.two + (rest == 0 ? 0.f : rest <= 256 ? tile.one : tile.two));
        if (us < best.us) best = Choice{t, us};
    }
    return best;
}

}  // namespace

extern "C" int lq_wq_gated_matmul(const lq_wq_gated_args* g, lq_stream stream) {
    LQ_REQUIRE(g, LQ_ERR_VALUE, "quantized_gated_matmul: args is NULL");
    LQ_REQUIRE(g->bits == 4 || g->bits == 8, LQ_ERR_VALUE, "quantized_gated_matmul: bits must be 4 or 8 (got %d)", g->bits);
    LQ_REQUIRE(g->group_size == 32 || g->group_size == 64 || g->group_size == 128, LQ_ERR_VALUE,
               "quantized_gated_matmul: group_size must be 32, 64 or 128 (got %d)", g->group_size);
    LQ_REQUIRE(g->dtype == LQ_F32 || g->dtype == LQ_F16, LQ_ERR_DTYPE, "quantized_gated_matmul: float32 and float16 are taken");
    LQ_REQUIRE(g->act >= 0 && g->act <= 3, LQ_ERR_VALUE, "quantized_gated_matmul: activation %d", g->act);
    LQ_REQUIRE(g->M >= 0 && g->N >= 0, LQ_ERR_SHAPE, "quantized_gated_matmul: negative extent");
    LQ_REQUIRE(g->K > 0 && g->K % g->group_size == 0, LQ_ERR_SHAPE, "quantized_gated_matmul: the quantized axis (%d) must be a multiple of group_size %d",
               g->K, g->group_size);
    LQ_REQUIRE(g->K < 1 << 30, LQ_ERR_SHAPE, "quantized_gated_matmul: K = %d", g->K);
    if (g->M == 0 || g->N == 0) return LQ_OK;
    gated::Args a;
    a.x = g->x, a.out = g->out, a.M = g->M, a.N = g->N, a.K = g->K, a.gs_shift = 31 - __builtin_clz(unsigned(g->group_size)), a.act = g->act;
    for (int i = 0; i < 2; ++i) {
        a.w[i] = gated::Weight{g->packed[i], g->scales[i], g->biases[i], g->bias[i]};
        LQ_REQUIRE(a.w[i].packed && a.w[i].scales && a.w[i].biases, LQ_ERR_VALUE, "quantized_gated_matmul: NULL pointer");
        LQ_REQUIRE(aligned16(a.w[i].packed), LQ_ERR_VALUE, "quantized_gated_matmul: packed weights must be 16-byte aligned");
        LQ_REQUIRE((reinterpret_cast<uintptr_t>(a.w[i].scales) | reinterpret_cast<uintptr_t>(a.w[i].biases)) % 4 == 0, LQ_ERR_VALUE,
                   "quantized_gated_matmul: scales must be aligned");
    }
    LQ_REQUIRE(a.x && a.out, LQ_ERR_VALUE, "quantized_gated_matmul: NULL pointer");
    LQ_REQUIRE(aligned16(a.x), LQ_ERR_VALUE, "quantized_gated_matmul: x must be 16-byte aligned");
    const size_t item = g->dtype == LQ_F16 ? 2 : 4;
    const uintptr_t x0 = reinterpret_cast<uintptr_t>(a.x), out0 = reinterpret_cast<uintptr_t>(a.out);
    LQ_REQUIRE(x0 + size_t(a.M) * a.K * item <= out0 || out0 + size_t(a.M) * a.N * item <= x0, LQ_ERR_VALUE,
               "quantized_gated_matmul: the result cannot take x's place");
    const hipStream_t st = as_stream(stream);
    const bool half = g->dtype == LQ_F16;
    const Choice c = choose(a, half, g->bits);
    if (c.tile < 0) return half ? gated::launch_rows_f16(a, g->bits, st) : gated::launch_rows_f32(a, g->bits, st);
    if (half) return g->bits == 4 ? gated::launch_gemm_f16_4(a, c.tile, st) : gated::launch_gemm_f16_8(a, c.tile, st);
    return g->bits == 4 ? gated::launch_gemm_f32_4(a, c.tile, st) : gated::launch_gemm_f32_8(a, c.tile, st);
}

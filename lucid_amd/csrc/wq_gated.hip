// Gated projections on group-wise weights: the entry point, and which kernel takes a call (wq_gated.hpp).
#include "wq_gated.hpp"

using namespace lq;

namespace {

struct Choice {
    bool rows;  // the kernel of few rows
    int tile;
    float us;
};

// The kernel and the tile that take the least time as rounds of blocks.  Of few rows a CU has one block, which takes 4 us (6: float32) beside its
// stages of 64 k; many small blocks end sooner as long as they are one round (16 x 4096 x 4096, 4 bits, float16: 64, 32, 16 columns a block 16.7, 11.3,
// 8.8 us; 16 x 11008 x 4096 18.1, 21.6, 20.5).  Of many rows a CU has two blocks, which take 9 us (14) beside their stages, or one (4, 7) where a last round
// has no more than 256; the launch before them and what is once 12 us.  us, few / many, 4 bits, float16: 128 x 11008 x 4096 64 / 66, 200 96 / 89, 512
// 190 / 137, 1024 x 2816 x 1024 33 / 37, 4056 x 1088 x 256 32 / 34, 435 x 9023 x 256 26 / 23, 1024 x 1024 x 14336 107 / 186; float32: 65 x 11008 x 4096
// 82 / 82, 128 94 / 88, 512 x 4096 x 4096 127 / 98, 435 x 9023 x 320 46 / 33.
template <int PARTS, int BITS>
Choice choose(const gated::Args& a) {
    constexpr bool half = PARTS == 1;
    const float stages = float((int64_t(a.K) + 63) / 64);
    const auto blocks_of = [&](int rows, int cols) { return (int64_t(a.M) + rows - 1) / rows * ((int64_t(a.N) + cols - 1) / cols); };
    Choice best{true, 0, 3.4e38f};
    for (size_t t = 0; t < gated::kRowsTiles<PARTS>.size(); ++t) {
        const gated::RowsTile& tile = gated::kRowsTiles<PARTS>[t];
        const float us = (half ? -0.5f : 1.f) + float((blocks_of(16 * tile.mt, 16 * tile.cg) + 255) / 256) * ((half ? 4.f : 6.f) + stages * tile.us);
        if (us < best.us) best = Choice{true, int(t), us};
    }
    if (size_t(a.N) * a.K * BITS / 8 >= 0x7fffffffull) return best;  // (offsets of codes are 32-bit in the kernel of many rows)
    for (size_t t = 0; t < gated::kGemmTiles<PARTS, BITS>.size(); ++t) {
        const gated::GemmTile& tile = gated::kGemmTiles<PARTS, BITS>[t];
        const int64_t blocks = blocks_of(16 * tile.mt, 64 * tile.ct), rest = blocks % 512;
        const float one = (half ? 4.f : 7.f) + stages * tile.one, two = (half ? 9.f : 14.f) + stages * tile.two;
        const float us = 12.f + float(blocks / 512) * two + (rest == 0 ? 0.f : rest <= 256 ? one : two);
        if (us < best.us) best = Choice{false, int(t), us};
    }
    return best;
}

Choice choose(const gated::Args& a, bool half, int bits) {
    return half ? (bits == 4 ? choose<1, 4>(a) : choose<1, 8>(a)) : (bits == 4 ? choose<2, 4>(a) : choose<2, 8>(a));
}

}  // namespace

extern "C" {

int lq_wq_gated_tile(int M, int N, int K, int bits, int dtype, int* many, int* rows, int* columns) {
    LQ_REQUIRE(many && rows && columns, LQ_ERR_VALUE, "wq_gated_tile: NULL pointer");
    LQ_REQUIRE(bits == 4 || bits == 8, LQ_ERR_VALUE, "wq_gated_tile: bits must be 4 or 8 (got %d)", bits);
    LQ_REQUIRE(dtype == LQ_F32 || dtype == LQ_F16, LQ_ERR_DTYPE, "wq_gated_tile: float32 and float16 are taken");
    LQ_REQUIRE(M > 0 && N > 0 && K > 0, LQ_ERR_SHAPE, "wq_gated_tile: %d x %d x %d", M, N, K);
    gated::Args a{};
    a.M = M, a.N = N, a.K = K;
    const bool half = dtype == LQ_F16;
    const Choice c = choose(a, half, bits);
    const auto of_rows = [&](const gated::RowsTile& t) { *rows = 16 * t.mt, *columns = 16 * t.cg; };
    const auto of_many = [&](const gated::GemmTile& t) { *rows = 16 * t.mt, *columns = 64 * t.ct; };
    *many = c.rows ? 0 : 1;
    if (c.rows && half) of_rows(gated::kRowsTiles<1>[c.tile]);
    else if (c.rows) of_rows(gated::kRowsTiles<2>[c.tile]);
    else if (half && bits == 4) of_many(gated::kGemmTiles<1, 4>[c.tile]);
    else if (half) of_many(gated::kGemmTiles<1, 8>[c.tile]);
    else if (bits == 4) of_many(gated::kGemmTiles<2, 4>[c.tile]);
    else of_many(gated::kGemmTiles<2, 8>[c.tile]);
    return LQ_OK;
}

int lq_wq_gated_matmul(const lq_wq_gated_args* g, lq_stream stream) {
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
    // (blocks write while others still read)
    const size_t item = g->dtype == LQ_F16 ? 2 : 4, codes = size_t(a.N) * a.K * g->bits / 8, numbers = size_t(a.N) * (a.K / g->group_size) * 4;
    const Span out{a.out, size_t(a.M) * a.N * item};
    bool sound = apart(out, Span{a.x, size_t(a.M) * a.K * item});
    for (const gated::Weight& w : a.w)
        sound = sound && apart(out, Span{w.packed, codes}) && apart(out, Span{w.scales, numbers}) && apart(out, Span{w.biases, numbers}) &&
                apart(out, Span{w.bias, size_t(a.N) * 4});
    LQ_REQUIRE(sound, LQ_ERR_VALUE, "quantized_gated_matmul: the result cannot lie on x, a weight or a bias");
    const hipStream_t st = as_stream(stream);
    const bool half = g->dtype == LQ_F16;
    const Choice c = choose(a, half, g->bits);
    if (c.rows) return half ? gated::launch_rows_f16(a, g->bits, c.tile, st) : gated::launch_rows_f32(a, g->bits, c.tile, st);
    if (half) return g->bits == 4 ? gated::launch_gemm_f16_4(a, c.tile, st) : gated::launch_gemm_f16_8(a, c.tile, st);
    return g->bits == 4 ? gated::launch_gemm_f32_4(a, c.tile, st) : gated::launch_gemm_f32_8(a, c.tile, st);
}

}  // extern "C"

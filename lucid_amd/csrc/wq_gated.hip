// Gated projections on group-wise weights: the entry point, and which kernel takes a call (wq_gated.hpp).
#include "wq_gated.hpp"

using namespace lq;

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
    LQ_REQUIRE(a.x != a.out, LQ_ERR_VALUE, "quantized_gated_matmul: the result cannot take x's place");
    const hipStream_t st = as_stream(stream);
    // (offsets of codes are 32-bit in the kernel of many rows)
    if (a.M > 64 && size_t(a.N) * a.K * g->bits / 8 < 0x7fffffffull) {
        if (g->dtype == LQ_F16) return g->bits == 4 ? gated::launch_gemm_f16_4(a, st) : gated::launch_gemm_f16_8(a, st);
        return g->bits == 4 ? gated::launch_gemm_f32_4(a, st) : gated::launch_gemm_f32_8(a, st);
    }
    return g->dtype == LQ_F16 ? gated::launch_rows_f16(a, g->bits, st) : gated::launch_rows_f32(a, g->bits, st);
}

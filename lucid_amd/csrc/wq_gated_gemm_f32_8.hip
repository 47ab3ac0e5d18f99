#include "wq_gated_gemm.hpp"

int lq::gated::launch_gemm_f32_8(const Args& a, int tile, hipStream_t st) { return launch_gemm<float, 2, 8>(a, tile, st); }

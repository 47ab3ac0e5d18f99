#include "wq_gated_gemm.hpp"

int lq::gated::launch_gemm_f32_4(const Args& a, int tile, hipStream_t st) { return launch_gemm<float, 2, 4>(a, tile, st); }

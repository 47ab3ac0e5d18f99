#include "wq_gated_gemm.hpp"

int lq::gated::launch_gemm_f16_4(const Args& a, int tile, hipStream_t st) { return launch_gemm<_Float16, 1, 4>(a, tile, st); }

#include "wq_gated_gemm.hpp"

int lq::gated::launch_gemm_f16_8(const Args& a, int tile, hipStream_t st) { return launch_gemm<_Float16, 1, 8>(a, tile, st); }

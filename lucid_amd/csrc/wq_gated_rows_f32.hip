#include "wq_gated_rows.hpp"

int lq::gated::launch_rows_f32(const Args& a, int bits, int tile, hipStream_t st) { return launch_rows<float>(a, bits, tile, st); }

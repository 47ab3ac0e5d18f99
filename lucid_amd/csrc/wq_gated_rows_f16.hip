#include "wq_gated_rows.hpp"

int lq::gated::launch_rows_f16(const Args& a, int bits, int tile, hipStream_t st) { return launch_rows<_Float16>(a, bits, tile, st); }

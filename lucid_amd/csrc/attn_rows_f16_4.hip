#include "attn_rows.hpp"

namespace lq::attn {
template void launch_rows_of<_Float16, 4>(const AttnArgs&, const _Float16*, _Float16*, int, int, bool, hipStream_t);
}

#include "attn_rows.hpp"

namespace lq::attn {
template void launch_rows_of<float, 4>(const AttnArgs&, const float*, float*, int, int, bool, hipStream_t);
}

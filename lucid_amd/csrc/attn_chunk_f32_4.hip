#include "attn_chunk.hpp"

namespace lq::attn {
template int launch_chunk_of<float, 4>(const AttnArgs&, const float*, float*, bool, int, bool, hipStream_t);
}

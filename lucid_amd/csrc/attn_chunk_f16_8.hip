#include "attn_chunk.hpp"

namespace lq::attn {
template int launch_chunk_of<_Float16, 8>(const AttnArgs&, const _Float16*, _Float16*, bool, int, bool, hipStream_t);
}

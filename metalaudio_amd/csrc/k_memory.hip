// Attention of a decoder's tokens to an encoder's states.
#include "rows_attention.hpp"

namespace mnn {
namespace k {

int64_t memory_part_floats(const LaunchCtx& c, const MemoryArgs& a) { return memory_rows_part_floats(c, a); }
void memory_attention(const LaunchCtx& c, const MemoryArgs& a, float* part) { memory_rows(c, a, part); }

}  // namespace k
}  // namespace mnn

// Attention of a few rows (tokens x the query heads of one key/value head) of each sequence to many keys: a decoder's
// next tokens on an encoder's states, or on a rolling cache in 8 bits.
#pragma once

#include "token_ops.hpp"

namespace mnn {
namespace k {

JoinSize memory_rows_join(const LaunchCtx& c, const MemoryArgs& a);
void memory_rows(const LaunchCtx& c, const MemoryArgs& a, const Join& join);

}  // namespace k
}  // namespace mnn

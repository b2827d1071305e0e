// Attention over blocks of 4-bit slots for few query rows.
#include "attend_span_few.hpp"

namespace vq {
int launch_blocks_few4(const SpanCall &c, const BlockLists &bl) { return launch_blocks_few_as<4>(c, bl); }
}  // namespace vq

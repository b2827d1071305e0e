// Attention over blocks of 2-bit slots for few query rows.
#include "attend_span_few.hpp"

namespace vq {
int launch_blocks_few2(const SpanCall &c, const BlockLists &bl) { return launch_blocks_few_as<2>(c, bl); }
}  // namespace vq

#include "attend_span_few.hpp"

namespace vq {
int launch_span_both4(const SpanCall &c) { return c.a.D == 64 ? launch_span_both_as<4, 64>(c) : launch_span_both_as<4, 128>(c); }
}  // namespace vq

#include "attend_span_few.hpp"

namespace vq {
int launch_span_both2(const SpanCall &c) { return c.a.D == 64 ? launch_span_both_as<2, 64>(c) : launch_span_both_as<2, 128>(c); }
}  // namespace vq

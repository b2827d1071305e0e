#include "attend_span.hpp"

namespace vq {

bool span_mfma_supported(const vq_store_attend_args &) { return false; }
void span_mfma_plan(SpanCall &, int) {}
int launch_span_mfma(const SpanCall &, int) { return VQ_ERR_UNSUPPORTED; }

}  // namespace vq

#include "attend_span_mfma.hpp"

VQ_SPAN_LAUNCHER(launch_span_rows_bf16, 0, bf16_t)

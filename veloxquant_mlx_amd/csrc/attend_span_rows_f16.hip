#include "attend_span_mfma.hpp"

VQ_SPAN_LAUNCHER(launch_span_rows_f16, 0, f16)

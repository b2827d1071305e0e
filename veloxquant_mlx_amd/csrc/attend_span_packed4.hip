#include "attend_span_mfma.hpp"

VQ_SPAN_LAUNCHER(launch_span_packed4, 4, f16)

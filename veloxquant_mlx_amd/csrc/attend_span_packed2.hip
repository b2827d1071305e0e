#include "attend_span_mfma.hpp"

VQ_SPAN_LAUNCHER(launch_span_packed2, 2, f16)

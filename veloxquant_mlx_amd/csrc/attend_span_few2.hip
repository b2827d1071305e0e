#include "attend_span_few.hpp"

VQ_SPAN_FEW_LAUNCHER(launch_span_few2, 2)

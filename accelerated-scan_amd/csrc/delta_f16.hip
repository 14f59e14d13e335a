// Gated delta rule kernels and their dispatch for one element type (ElemF16).
#include "delta_dispatch.h"

ASCAN_DEFINE_DELTA(f16, ElemF16, 2, 3)

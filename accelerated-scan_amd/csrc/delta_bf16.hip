// Gated delta rule kernels and their dispatch for one element type (ElemBF16).
#include "delta_dispatch.h"

ASCAN_DEFINE_DELTA(bf16, ElemBF16, 1, 3)

// Gated delta rule kernels and their dispatch for one element type (ElemF32).
#include "delta_dispatch.h"

ASCAN_DEFINE_DELTA(f32, ElemF32, 0, 0)

// kd_xent_f16.hip -- surface_cross_entropy of fp16 data (kd_xent.hpp).
#include "kd_xent.hpp"

KD_XENT(f16, kd::half_t)

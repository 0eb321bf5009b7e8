// kd_xent_bf16.hip -- surface_cross_entropy of bf16 data (kd_xent.hpp).
#include "kd_xent.hpp"

KD_XENT(bf16, kd::bfloat_t)

// kd_xent_f32.hip -- surface_cross_entropy of fp32 data (kd_xent.hpp).
#include "kd_xent.hpp"

KD_XENT(f32, float)

extern "C" {

// bytes for any of the types: 2 or 4 bytes an element
size_t kd_surface_xent_state_size(int64_t n, int64_t rows, int channels, int element_size,
                                  int need_features, int need_embeddings) {
  if (kd::xent::check(n, rows, channels, 1.0, 0) != KD_OK ||
      (element_size != 2 && element_size != 4))
    return 0;
  const int np = element_size == 4 ? 3 : 1;
  kd::xent::Args a = kd::xent::shape(n, rows, channels, np, 1.0, 0);
  return kd::xent::lay_state(a, np, need_features, need_embeddings, nullptr);
}

size_t kd_surface_xent_scratch_size(int64_t n, int64_t rows, int channels, int element_size,
                                    int need_features, int need_embeddings, int backward) {
  if (kd::xent::check(n, rows, channels, 1.0, 0) != KD_OK ||
      (element_size != 2 && element_size != 4))
    return 0;
  const int np = element_size == 4 ? 3 : 1;
  kd::xent::Args a = kd::xent::shape(n, rows, channels, np, 1.0, 0);
  return backward ? kd::xent::lay_backward(a, np, need_embeddings, nullptr)
                  : kd::xent::lay_forward(a, np, need_features, need_embeddings, nullptr);
}

}  // extern "C"

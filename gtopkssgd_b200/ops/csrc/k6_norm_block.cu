// K6 backward inside a feed-forward block, where x may be codes and more is taken and given: apart, to be compiled beside
// the rest.
#include "k6_norm.cuh"

namespace gtk {

template <typename T>
int norm_backward_block(bool codes, const void* dy, const void* x, const float* mean, const float* rstd, const void* w, const void* add, void* dx, void* dw,
                        void* db, float* partial, NormShape s, NormMore<T> more, cudaStream_t stream) {
  return codes ? norm_backward<T, signed char, true>(dy, x, mean, rstd, w, add, dx, dw, db, partial, s, more, stream)
               : norm_backward<T, T, true>(dy, x, mean, rstd, w, add, dx, dw, db, partial, s, more, stream);
}

#define GTK_BLOCK(T) \
  template int norm_backward_block<T>(bool, const void*, const void*, const float*, const float*, const void*, const void*, void*, void*, void*, float*, NormShape, NormMore<T>, cudaStream_t);
GTK_BLOCK(float)
GTK_BLOCK(__half)
GTK_BLOCK(__nv_bfloat16)

}  // namespace gtk

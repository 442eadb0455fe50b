// Backward pass of the residual update z_new = z + dropout(y), ln = LN(z_new):
//   dz = dz_new + (the LayerNorm's gradient of dln at z_new);  dy = dropout(dz) with the forward pass's draws.
// z's gradient is dz as it is. One pass over z_new, dz_new and dln; it writes dz and dy.
#include "bzpf_rowgrad.h"

namespace bzpf {

hipError_t launch_dropout_add_ln_bwd(const float* dz_new, const void* dln, int ln_dt, const float* z_new,
                                     const float* w, float eps, const Drop& drop, float* dz, void* dy, int y_dt,
                                     float* dw, float* db, float* ws, int64_t rows, int D, hipStream_t st) {
  return with_types(y_dt, ln_dt, [&](auto ty, auto tg) {
    typedef std::remove_cv_t<std::remove_pointer_t<decltype(ty)>> TY;
    typedef std::remove_cv_t<std::remove_pointer_t<decltype(tg)>> TG;
    const RowGrad<float, TG, TY> a{z_new, static_cast<const TG*>(dln), dz_new, w, eps, dz, static_cast<TY*>(dy), drop,
                                   ws, dw, db, rows, D};
    return launch_row_grad<true>(a, st);
  });
}

}  // namespace bzpf

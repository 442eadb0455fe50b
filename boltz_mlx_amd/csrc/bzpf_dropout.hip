// Dropout, and the residual update z + dropout(y) with the LayerNorm that follows it (the training form of add_ln).
// The draws are formed where they are used (bzpf_dropout.h) and no mask is read or written, so both are bound by their
// tensors' bytes.
#include <type_traits>

#include "bzpf_dropout.h"

namespace bzpf {

// One chunk of eight columns a thread; rows of any width. A chunk that passes the row's end takes its elements one by
// one (rows may be shorter than a chunk here).
template <typename TX, typename TY>
__global__ __launch_bounds__(256) void dropout_k(const TX* __restrict__ x, Drop drop, TY* __restrict__ y, int64_t rows,
                                                 int64_t D) {
  const int64_t chunks = (D + 7) / 8, n = rows * chunks, per = (D + 3) / 4;
  Key key{};
  if (drop.mode != DROP_OFF) key = drop_key(drop);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / chunks, at = 8 * (i - r * chunks);
    const TX* const xp = x + r * D + at;
    TY* const yp = y + r * D + at;
    const int m = D - at < 8 ? (int)(D - at) : 8;
    f8 v{};
    if (m == 8) {
      v = load8(xp);
    } else {
#pragma unroll
      for (int e = 0; e < 7; e++)
        if (e < m) v[e] = (float)xp[e];
    }
    if (drop.mode == DROP_ELEMENT) v = drop_elements(drop, key, (uint64_t)r * per + (at >> 2), 0, v);
    if (drop.mode >= DROP_ROW) v = draw_shared(drop, key, r) <= drop.last ? f8{} : v * drop.scale;
    if (m == 8) {
      store8(yp, v);
    } else {
#pragma unroll
      for (int e = 0; e < 7; e++)
        if (e < m) yp[e] = (TY)v[e];
    }
  }
}

hipError_t launch_dropout(const void* x, int x_dt, const Drop& drop, void* y, int y_dt, int64_t rows, int64_t D,
                          hipStream_t st) {
  return with_types(x_dt, y_dt, [&](auto tx, auto ty) {
    typedef std::remove_cv_t<std::remove_pointer_t<decltype(tx)>> TX;
    typedef std::remove_cv_t<std::remove_pointer_t<decltype(ty)>> TY;
    dropout_k<TX, TY><<<row_blocks(rows * ((D + 7) / 8), 256, 1 << 16), 256, 0, st>>>(
        static_cast<const TX*>(x), drop, static_cast<TY*>(y), rows, D);
    return hipGetLastError();
  });
}

template <typename TY, typename TO, int L, int NV>
__global__ __launch_bounds__(256) void dropout_add_ln_k(const float* __restrict__ z, const TY* __restrict__ y,
                                                        Drop drop, const float* __restrict__ w,
                                                        const float* __restrict__ b, float eps,
                                                        float* __restrict__ z_new, TO* __restrict__ ln, int64_t rows,
                                                        int D) {
  __shared__ float red[8];
  const RowSpan<L, NV> sp(threadIdx.x % L, D);
  const int64_t per = (D + 3) / 4;
  constexpr int R = 256 / L;
  Key key{};
  if (drop.mode != DROP_OFF) key = drop_key(drop);
  for (int64_t r = (int64_t)blockIdx.x * R + threadIdx.x / L; r < rows; r += (int64_t)gridDim.x * R) {
    f8 v[NV];
    bool dropped = false;
    if (drop.mode >= DROP_ROW) dropped = draw_shared(drop, key, r) <= drop.last;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      v[k] = load8(z + r * D + sp.at[k]);
      f8 t = load8(y + r * D + sp.at[k]);
      if (drop.mode == DROP_ELEMENT)
        t = drop_elements(drop, key, (uint64_t)r * per + (sp.at[k] >> 2), sp.at[k] & 3, t);
      if (drop.mode >= DROP_ROW) t = dropped ? f8{} : t * drop.scale;
      v[k] += t;
      sp.store(k, z_new + r * D, v[k]);
    }
    const float rstd = centre_row<L, NV>(v, sp, D, eps, red);
#pragma unroll
    for (int k = 0; k < NV; k++) {
      f8 o = v[k] * rstd;
      if (w) o *= load8(w + sp.at[k]);
      if (b) o += load8(b + sp.at[k]);
      sp.store(k, ln + r * D, o);
    }
  }
}

hipError_t launch_dropout_add_ln(const float* z, const void* y, int y_dt, const Drop& drop, const float* w,
                                 const float* b, float eps, float* z_new, void* ln, int ln_dt, int64_t rows, int D,
                                 hipStream_t st) {
  return with_types(y_dt, ln_dt, [&](auto ty, auto to) {
    return with_row_layout(D, [&](auto lay) {
      typedef decltype(lay) Lay;
      typedef std::remove_cv_t<std::remove_pointer_t<decltype(ty)>> TY;
      typedef std::remove_cv_t<std::remove_pointer_t<decltype(to)>> TO;
      dropout_add_ln_k<TY, TO, Lay::L, Lay::NV><<<row_blocks(rows, 256 / Lay::L, 1 << 20), 256, 0, st>>>(
          z, static_cast<const TY*>(y), drop, w, b, eps, z_new, static_cast<TO*>(ln), rows, D);
      return hipGetLastError();
    });
  });
}

}  // namespace bzpf

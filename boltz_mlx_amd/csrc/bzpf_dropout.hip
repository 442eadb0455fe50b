// Dropout, and the residual update z + dropout(y) with the LayerNorm that follows it (the training form of add_ln).
// The draws are formed where they are used (bzpf_dropout.h) and no mask is read or written, so both are bound by their
// tensors' bytes.
#include <type_traits>

#include "bzpf_dropout.h"

namespace bzpf {

// One chunk of VE columns a thread (two or four, their loads together, measured the same or slower). FLAT: D is a multiple
// of VE, so chunk i is element VE i, block VE i / 4, and only a shared draw needs its row. Otherwise a chunk that would
// pass the row's end is moved back to D - VE: its first elements are the neighbour's too, who writes the same values there
// (each is one product, of the same factors). Rows shorter than a chunk (D < VE) are taken element by element.
// Bound by memory; the draws of 128 M fp16 elements (ten rounds of two 32-bit products and two three-way XORs for four of
// them) fit under its 83 us (6.2 TB/s; 82 without draws, 81 with one a row). 100,000 rows of 77: 12 us (2.5 TB/s).
template <typename TX, typename TY, int MODE, bool FLAT>
__global__ __launch_bounds__(256) void dropout_k(const TX* __restrict__ x, Drop drop, TY* __restrict__ y, int64_t rows,
                                                 int64_t D) {
  constexpr int VE = chunk_of<TX, TY>();
  const int64_t chunks = (D + VE - 1) / VE, n = rows * chunks, per = (D + 3) / 4;
  const bool small = n >> 32 == 0;
  Key key{};
  if (MODE != DROP_OFF) key = drop_key(drop);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    // the 32-bit division is a third as long
    const int64_t r = FLAT && MODE < DROP_ROW ? 0 : small ? (int64_t)((uint32_t)i / (uint32_t)chunks) : i / chunks;
    int64_t col = 0, at = VE * i;  // the chunk's column and its first element
    if (!FLAT) {
      col = VE * (i - r * chunks);
      col = col + VE <= D ? col : D < VE ? 0 : D - VE;
      at = r * D + col;
    }
    fv<VE> v{};
    if (FLAT || D >= VE) {
      v = load_chunk<VE>(x + at);
    } else {
#pragma unroll
      for (int e = 0; e < VE - 1; e++)
        if (e < D) v[e] = (float)x[at + e];
    }
    if (MODE == DROP_ELEMENT) {
      const uint64_t block = FLAT ? (uint64_t)at >> 2 : (uint64_t)(r * per + (col >> 2));
      v = keep<VE>(drop, kept<VE>(drop, key, block, (int)(col & 3)), 0, v);
    }
    if (MODE >= DROP_ROW) v = drops_row(drop, key, r) ? fv<VE>{} : v * drop.scale;
    if (FLAT || D >= VE) {
      store_chunk<VE>(y + at, v);
    } else {
#pragma unroll
      for (int e = 0; e < VE - 1; e++)
        if (e < D) y[at + e] = (TY)v[e];
    }
  }
}

template <typename TX, typename TY, bool FLAT>
static auto dropout_kernel(int mode) {
  return mode == DROP_OFF       ? dropout_k<TX, TY, DROP_OFF, FLAT>
         : mode == DROP_ELEMENT ? dropout_k<TX, TY, DROP_ELEMENT, FLAT>
                                : dropout_k<TX, TY, DROP_ROW, FLAT>;  // column draws too
}

hipError_t launch_dropout(const void* x, int x_dt, const Drop& drop, void* y, int y_dt, int64_t rows, int64_t D,
                          hipStream_t st) {
  return with_types(x_dt, y_dt, [&](auto tx, auto ty) {
    typedef std::remove_cv_t<std::remove_pointer_t<decltype(tx)>> TX;
    typedef std::remove_cv_t<std::remove_pointer_t<decltype(ty)>> TY;
    constexpr int VE = chunk_of<TX, TY>();
    const auto kernel =
        D % VE == 0 ? dropout_kernel<TX, TY, true>(drop.mode) : dropout_kernel<TX, TY, false>(drop.mode);
    kernel<<<row_blocks(rows * ((D + VE - 1) / VE), 256, 1 << 16), 256, 0, st>>>(
        static_cast<const TX*>(x), drop, static_cast<TY*>(y), rows, D);
    return hipGetLastError();
  });
}

// The update and the LayerNorm of it in one pass: z and y are read once, z_new and ln written once, the statistics are of
// the values that z_new gets. 1 M rows of 128, fp16 y and ln: 246 us (6.2 TB/s); 160,000: 36 us; 20,667 of 77, fp32 y and
// bf16 ln, a draw for each element: 8.1 us (2.8 TB/s).
template <typename TY, typename TO, int L, int E, bool LINES>
__global__ __launch_bounds__(row_threads(L)) void dropout_add_ln_k(
    const float* __restrict__ z, const TY* __restrict__ y, Drop drop, const float* __restrict__ w,
    const float* __restrict__ b, float eps, float* __restrict__ z_new, TO* __restrict__ ln, int64_t rows, int D) {
  __shared__ float red[2 * row_red(L)];
  constexpr int R = row_threads(L) / L, VE = 4, NV = E / VE;
  const RowSpan<L, NV, VE, LINES> sp(threadIdx.x % L, D);
  const int64_t per = (D + 3) / 4;
  Key key{};
  if (drop.mode != DROP_OFF) key = drop_key(drop);
  fv<VE> pw[NV], pb[NV];
  row_param(pw, sp, w, 1.f);
  row_param(pb, sp, b, 0.f);
  for (int64_t r = (int64_t)blockIdx.x * R + threadIdx.x / L; r < rows; r += (int64_t)gridDim.x * R) {
    fv<VE> v[NV];
    const bool dropped = drop.mode >= DROP_ROW && drops_row(drop, key, r);
#pragma unroll
    for (int k = 0; k < NV; k++) {
      v[k] = load_chunk<VE>(z + r * D + sp.at[k]);
      fv<VE> t = load_chunk<VE>(y + r * D + sp.at[k]);
      if (drop.mode == DROP_ELEMENT)
        t = keep<VE>(drop, kept<VE>(drop, key, (uint64_t)r * per + (sp.at[k] >> 2), sp.at[k] & 3), 0, t);
      if (drop.mode >= DROP_ROW) t = dropped ? fv<VE>{} : t * drop.scale;
      v[k] += t;
      sp.store(k, z_new + r * D, v[k]);
    }
    const float rstd = centre_row(v, sp, D, eps, red);
#pragma unroll
    for (int k = 0; k < NV; k++) sp.store(k, ln + r * D, v[k] * rstd * pw[k] + pb[k]);
  }
}

hipError_t launch_dropout_add_ln(const float* z, const void* y, int y_dt, const Drop& drop, const float* w,
                                 const float* b, float eps, float* z_new, void* ln, int ln_dt, int64_t rows, int D,
                                 hipStream_t st) {
  return with_types(y_dt, ln_dt, [&](auto ty, auto to) {
    return with_row_layout<true>(D, [&](auto lay) {
      typedef decltype(lay) Lay;
      typedef std::remove_cv_t<std::remove_pointer_t<decltype(ty)>> TY;
      typedef std::remove_cv_t<std::remove_pointer_t<decltype(to)>> TO;
      constexpr int T = row_threads(Lay::L);
      dropout_add_ln_k<TY, TO, Lay::L, Lay::E, Lay::LINES><<<row_blocks(rows, T / Lay::L, 1 << 20), T, 0, st>>>(
          z, static_cast<const TY*>(y), drop, w, b, eps, z_new, static_cast<TO*>(ln), rows, D);
      return hipGetLastError();
    });
  });
}

}  // namespace bzpf

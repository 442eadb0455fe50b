// LayerNorm at any width and type, and its backward pass with the weight's and bias's gradients.
//   y = xh w + b, xh = (x - mean) rstd;   g = dy w;   dx = rstd (g - mean(g) - xh mean(g xh));
//   dw = sum over rows of dy xh;   db = sum over rows of dy.
// The backward pass reads x and dy and writes dx; the row's statistics are formed again from x, which is in registers
// anyway, so the forward pass saves nothing but its input. Both are bound by memory.
// dw and db: each thread sums its own columns over its workgroup's rows, a workgroup's sums meet in LDS, and a second
// kernel adds the workgroups' partial sums in their order: no atomics, so that equal inputs give equal bits.
#include "bzpf_rowgrad.h"

namespace bzpf {

template <typename TX, typename TY, int L, int NV>
__global__ __launch_bounds__(256) void ln_rows_k(const TX* __restrict__ x, const float* __restrict__ w,
                                                 const float* __restrict__ b, float eps, TY* __restrict__ y,
                                                 int64_t rows, int D) {
  __shared__ float red[8];
  const RowSpan<L, NV> sp(threadIdx.x % L, D);
  constexpr int R = 256 / L;
  for (int64_t r = (int64_t)blockIdx.x * R + threadIdx.x / L; r < rows; r += (int64_t)gridDim.x * R) {
    f8 v[NV];
#pragma unroll
    for (int k = 0; k < NV; k++) v[k] = load8(x + r * D + sp.at[k]);
    const float rstd = centre_row<L, NV>(v, sp, D, eps, red);
#pragma unroll
    for (int k = 0; k < NV; k++) {
      f8 o = v[k] * rstd;
      if (w) o *= load8(w + sp.at[k]);
      if (b) o += load8(b + sp.at[k]);
      sp.store(k, y + r * D, o);
    }
  }
}

hipError_t launch_layernorm_rows(const void* x, int x_dt, const float* w, const float* b, float eps, void* y, int y_dt,
                                 int64_t rows, int D, hipStream_t st) {
  return with_types(x_dt, y_dt, [&](auto tx, auto ty) {
    return with_row_layout(D, [&](auto lay) {
      typedef decltype(lay) Lay;
      typedef std::remove_cv_t<std::remove_pointer_t<decltype(tx)>> TX;
      typedef std::remove_cv_t<std::remove_pointer_t<decltype(ty)>> TY;
      ln_rows_k<TX, TY, Lay::L, Lay::NV><<<row_blocks(rows, 256 / Lay::L, 1 << 20), 256, 0, st>>>(
          static_cast<const TX*>(x), w, b, eps, static_cast<TY*>(y), rows, D);
      return hipGetLastError();
    });
  });
}

hipError_t launch_layernorm_bwd(const void* dy, int dy_dt, const void* x, int x_dt, const float* w, float eps, void* dx,
                                float* dw, float* db, float* ws, int64_t rows, int D, hipStream_t st) {
  return with_types(x_dt, dy_dt, [&](auto tx, auto tg) {
    typedef std::remove_cv_t<std::remove_pointer_t<decltype(tx)>> TX;
    typedef std::remove_cv_t<std::remove_pointer_t<decltype(tg)>> TG;
    const RowGrad<TX, TG, float> a{static_cast<const TX*>(x), static_cast<const TG*>(dy), nullptr, w, eps,
                                   static_cast<TX*>(dx), nullptr, Drop{}, ws, dw, db, rows, D};
    return launch_row_grad<false>(a, st);
  });
}

// Sums of the workgroups' partial [2][D] (dw, then db) over `blocks` workgroups: 16 threads for each of 16 columns, each
// adding every sixteenth partial sum, then the 16 in order.
__global__ __launch_bounds__(256) void row_grad_sum_k(const float* __restrict__ ws, int64_t blocks, int D,
                                                      float* __restrict__ dw, float* __restrict__ db) {
  __shared__ float part[16][17];
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
  const int64_t col = (int64_t)blockIdx.x * 16 + c;
  float s = 0.f;
  if (col < 2 * D)
    for (int64_t i = g; i < blocks; i += 16) s += ws[i * 2 * D + col];
  part[g][c] = s;
  __syncthreads();
  if (g == 0 && col < 2 * D) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) s += part[i][c];
    float* out = col < D ? dw : db;
    if (out) out[col < D ? col : col - D] = s;
  }
}

hipError_t launch_row_grad_sum(const float* ws, int64_t blocks, int D, float* dw, float* db, hipStream_t st) {
  row_grad_sum_k<<<(unsigned)((2 * D + 15) / 16), 256, 0, st>>>(ws, blocks, D, dw, db);
  return hipGetLastError();
}

int64_t row_grad_ws_bytes(int64_t rows, int D) {
  const int64_t blocks = row_grad_blocks(rows, D);
  return blocks > 1 ? blocks * 2 * D * (int64_t)sizeof(float) : 0;
}

}  // namespace bzpf

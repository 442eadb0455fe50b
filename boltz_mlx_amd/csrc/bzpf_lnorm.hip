// LayerNorm at any width and type, and its backward pass with the weight's and bias's gradients.
//   y = xh w + b, xh = (x - mean) rstd;   g = dy w;   dx = rstd (g - mean(g) - xh mean(g xh));
//   dw = sum over rows of dy xh;   db = sum over rows of dy.
// The backward pass reads x and dy and writes dx; the row's statistics are formed again from x, which is in registers
// anyway, so the forward pass saves nothing but its input. Both are bound by memory.
// dw and db: each thread sums its own columns over its workgroup's rows, a workgroup's sums meet in LDS, and a second
// kernel adds the workgroups' partial sums in their order: no atomics, so that equal inputs give equal bits.
#include "bzpf_rowgrad.h"

namespace bzpf {

// Bound by memory: one read of x, one write of y, a row a group of L lanes; enough workgroups in flight hide the two sums
// of a row. 1 M rows of 128, fp32 to bf16: 124 us (6.2 TB/s); 4099 of 1021 fp32: 6.3 us (5.3 TB/s); 2050 of 8192 bf16:
// 13.3 us (5.1 TB/s).
template <typename TX, typename TY, int L, int E, bool LINES>
__global__ __launch_bounds__(row_threads(L)) void ln_rows_k(const TX* __restrict__ x, const float* __restrict__ w,
                                                            const float* __restrict__ b, float eps,
                                                            TY* __restrict__ y, int64_t rows, int D) {
  __shared__ float red[2 * row_red(L)];
  constexpr int R = row_threads(L) / L, VE = chunk_of<TX, TY>(), NV = E / VE;
  const RowSpan<L, NV, VE, LINES> sp(threadIdx.x % L, D);
  fv<VE> pw[NV], pb[NV];
  row_param(pw, sp, w, 1.f);
  row_param(pb, sp, b, 0.f);
  for (int64_t r = (int64_t)blockIdx.x * R + threadIdx.x / L; r < rows; r += (int64_t)gridDim.x * R) {
    fv<VE> v[NV];
#pragma unroll
    for (int k = 0; k < NV; k++) v[k] = load_chunk<VE>(x + r * D + sp.at[k]);
    const float rstd = centre_row(v, sp, D, eps, red);
#pragma unroll
    for (int k = 0; k < NV; k++) sp.store(k, y + r * D, v[k] * rstd * pw[k] + pb[k]);
  }
}

hipError_t launch_layernorm_rows(const void* x, int x_dt, const float* w, const float* b, float eps, void* y, int y_dt,
                                 int64_t rows, int D, hipStream_t st) {
  return with_types(x_dt, y_dt, [&](auto tx, auto ty) {
    return with_row_layout<false>(D, [&](auto lay) {
      typedef decltype(lay) Lay;
      typedef std::remove_cv_t<std::remove_pointer_t<decltype(tx)>> TX;
      typedef std::remove_cv_t<std::remove_pointer_t<decltype(ty)>> TY;
      constexpr int T = row_threads(Lay::L);
      ln_rows_k<TX, TY, Lay::L, Lay::E, Lay::LINES><<<row_blocks(rows, T / Lay::L, 1 << 20), T, 0, st>>>(
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

// Sums of the workgroups' partial [2][D] (dw, then db) over `blocks` <= ROW_GRAD_BLOCKS workgroups. A workgroup takes 32 columns (whole
// lines of the partial sums; 16 took 8.3 us instead of 5.1 at 256 x 16384 columns): 32 threads a column each add every
// 32nd partial sum, all loads in flight at once, then the 32 meet in a fixed order.
__global__ __launch_bounds__(1024) void row_grad_sum_k(const float* __restrict__ ws, int blocks, int D,
                                                       float* __restrict__ dw, float* __restrict__ db) {
  __shared__ float part[32][33];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int col = min((int)blockIdx.x * 32 + c, 2 * D - 1);
  constexpr int V = ROW_GRAD_BLOCKS / 32;
  float v[V];
#pragma unroll
  for (int i = 0; i < V; i++) v[i] = g + 32 * i < blocks ? ws[(int64_t)(g + 32 * i) * 2 * D + col] : 0.f;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < V; i++) s += v[i];
  part[g][c] = s;
  __syncthreads();
  if (threadIdx.x < 32 && blockIdx.x * 32 + c < 2 * D) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; i += 4) s += (part[i][c] + part[i + 1][c]) + (part[i + 2][c] + part[i + 3][c]);
    float* out = col < D ? dw : db;
    if (out) out[col < D ? col : col - D] = s;
  }
}

hipError_t launch_row_grad_sum(const float* ws, int64_t blocks, int D, float* dw, float* db, hipStream_t st) {
  if (blocks > ROW_GRAD_BLOCKS) return hipErrorInvalidValue;
  row_grad_sum_k<<<(unsigned)((2 * D + 31) / 32), 1024, 0, st>>>(ws, (int)blocks, D, dw, db);
  return hipGetLastError();
}

int64_t row_grad_ws_bytes(int64_t rows, int D) {
  const int64_t a = row_grad_blocks<false>(rows, D), b = row_grad_blocks<true>(rows, D), blocks = a > b ? a : b;
  return blocks > 1 ? blocks * 2 * D * (int64_t)sizeof(float) : 0;
}

}  // namespace bzpf

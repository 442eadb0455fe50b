// The backward pass of a LayerNorm over rows, alone (bzpf_lnorm.hip) and after a residual update with dropout
// (bzpf_dropout_bwd.hip).
#pragma once

#include <type_traits>

#include "bzpf_dropout.h"

namespace bzpf {

// RES = false: x -> dx (TX). RES = true: x is the updated stream (fp32), dx = its own gradient dz_new (null: zero) plus
// the LayerNorm's, and dy = dropout(dx).
template <typename TX, typename TG, typename TY>
struct RowGrad {
  const TX* x;
  const TG* g;
  const float* dz_new;
  const float* w;
  float eps;
  TX* dx;
  TY* dy;
  Drop drop;
  float* ws;  // partial sums [workgroups][2][D]; null: no parameter gradient is wanted
  float* dw;
  float* db;
  int64_t rows;
  int D;
};

// Workgroups of the backward pass: one for every four rows of each of its row places, up to 1024 (four for each
// compute unit), so that the partial sums stay few.
static inline int64_t row_grad_blocks(int64_t rows, int D) {
  const int per = D <= 64 ? 32 : D <= 128 ? 16 : D <= 256 ? 8 : D <= 2048 ? 4 : 1;  // rows that it holds at once
  return row_blocks(rows, 4 * per, 1024);
}

// The sum of v over the 64 / L lanes of a wave that hold the same columns of different rows.
template <int L>
__device__ __forceinline__ float column_sum(float v) {
  if constexpr (L <= 8) v = dpp_add<0x128>(v);  // row_ror by 8: the other half of the DPP row
  if constexpr (L <= 16) {
    const unsigned u = __float_as_uint(v);
    const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
  if constexpr (L <= 32) {
    const unsigned u = __float_as_uint(v);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
  return v;
}

// The workgroup's sums over its rows of s (chunks as in sp) into out [D].
template <int L, int NV>
__device__ __forceinline__ void meet_columns(f8 (&s)[NV], const RowSpan<L, NV>& sp, int D, float* meet, float* out) {
  if constexpr (L == 256) {
#pragma unroll
    for (int k = 0; k < NV; k++) sp.store(k, out, s[k]);
  } else {
    __syncthreads();  // meet's last reader is done
#pragma unroll
    for (int k = 0; k < NV; k++) {
#pragma unroll
      for (int e = 0; e < 8; e++) s[k][e] = column_sum<L>(s[k][e]);
      if ((threadIdx.x & 63) < L) sp.store(k, meet + (threadIdx.x >> 6) * D, s[k]);
    }
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += 256) out[c] = (meet[c] + meet[D + c]) + (meet[2 * D + c] + meet[3 * D + c]);
  }
}

template <bool RES, typename TX, typename TG, typename TY, int L, int NV>
__global__ __launch_bounds__(256) void row_grad_k(RowGrad<TX, TG, TY> a) {
  constexpr int R = 256 / L;
  __shared__ float red[16];
  __shared__ float meet[L < 256 ? 4 * 8 * L * NV : 1];
  const int D = a.D;
  const RowSpan<L, NV> sp(threadIdx.x % L, D);
  const int64_t per = (D + 3) / 4;
  const float inv = 1.0f / D;
  Key key{};
  if (RES && a.drop.mode != DROP_OFF) key = drop_key(a.drop);
  f8 sw[NV], sb[NV];
#pragma unroll
  for (int k = 0; k < NV; k++) sw[k] = sb[k] = f8{};
  for (int64_t r = (int64_t)blockIdx.x * R + threadIdx.x / L; r < a.rows; r += (int64_t)gridDim.x * R) {
    f8 v[NV], g[NV];
#pragma unroll
    for (int k = 0; k < NV; k++) {
      v[k] = load8(a.x + r * D + sp.at[k]);
      g[k] = load8(a.g + r * D + sp.at[k]);
    }
    const float rstd = centre_row<L, NV>(v, sp, D, a.eps, red);
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      v[k] *= rstd;
      sw[k] += g[k] * v[k];
      sb[k] += g[k];
      if (a.w) g[k] *= load8(a.w + sp.at[k]);
      c1 += sum8(sp.own(k, g[k]));
      c2 += sum8(sp.own(k, g[k] * v[k]));
    }
    c1 = row_sum<L>(c1, red + 8) * inv;
    c2 = row_sum<L>(c2, red + 12) * inv;
    bool dropped = false;
    if (RES && a.drop.mode >= DROP_ROW) dropped = draw_shared(a.drop, key, r) <= a.drop.last;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      f8 o = (g[k] - c1 - v[k] * c2) * rstd;
      if (RES && a.dz_new) o += load8(a.dz_new + r * D + sp.at[k]);
      sp.store(k, a.dx + r * D, o);
      if constexpr (RES) {
        if (a.drop.mode == DROP_ELEMENT)
          o = drop_elements(a.drop, key, (uint64_t)r * per + (sp.at[k] >> 2), sp.at[k] & 3, o);
        if (a.drop.mode >= DROP_ROW) o = dropped ? f8{} : o * a.drop.scale;
        sp.store(k, a.dy + r * D, o);
      }
    }
  }
  if (!a.dw && !a.db) return;
  float* const ow = gridDim.x > 1 ? a.ws + (int64_t)blockIdx.x * 2 * D : a.dw;
  float* const ob = gridDim.x > 1 ? a.ws + (int64_t)blockIdx.x * 2 * D + D : a.db;
  if (ow) meet_columns<L, NV>(sw, sp, D, meet, ow);
  if (ob) meet_columns<L, NV>(sb, sp, D, meet, ob);
}

template <bool RES, typename TX, typename TG, typename TY>
static hipError_t launch_row_grad(const RowGrad<TX, TG, TY>& a, hipStream_t st) {
  const unsigned blocks = (unsigned)row_grad_blocks(a.rows, a.D);
  const hipError_t e = with_row_layout(a.D, [&](auto lay) {
    typedef decltype(lay) Lay;
    row_grad_k<RES, TX, TG, TY, Lay::L, Lay::NV><<<blocks, 256, 0, st>>>(a);
    return hipGetLastError();
  });
  if (e != hipSuccess || blocks == 1 || (!a.dw && !a.db)) return e;
  return launch_row_grad_sum(a.ws, blocks, a.D, a.dw, a.db, st);
}

}  // namespace bzpf

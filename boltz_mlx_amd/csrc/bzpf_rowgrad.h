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

// Workgroups of the backward pass: enough for four rows in each of their row places, but not fewer than one for each
// compute unit while rows last (two up to D = 128, whose partial sums are small), nor more than two (one past D = 2048):
// each writes its partial sums, which the second kernel reads. Measured with 256 / 512 / 768 workgroups in bf16 (fp32):
// 1 M rows of 128 195 / 140 / 133 us (270 / 288 / 287), 16000 of 1024 26 / 26 / 26 (41 / 41 / 43), 6000 of 2048
// 33 / 27 / 24 (33 / 33 / 34); 4096 of 4096 with 256 / 512 30 / 30 (44 / 47), 2048 of 8192 31 / 43 (47 / 56). At the lower
// end, 256 / 512: 20667 rows of 80 9.8 / 9.4 (with a residual update 13.7 / 12.8), 2000 of 768 9.6 / 10.0 (12.5 / 15.8).
// One rule serves every type, a compromise where rows are many and narrow: 768 would give bf16 5% there, 256 fp32 6%.
template <bool RES>
static inline int64_t row_grad_blocks(int64_t rows, int D) {
  const int per = row_places<RES>(D);
  const int64_t least = row_blocks(rows, per, D <= 128 ? ROW_GRAD_BLOCKS : ROW_GRAD_BLOCKS / 2);
  const int64_t four = row_blocks(rows, 4 * per, D <= 2048 ? ROW_GRAD_BLOCKS : ROW_GRAD_BLOCKS / 2);
  return least > four ? least : four;
}

// The sum of v over the 64 / L lanes of a wave that hold the same columns of different rows.
template <int L>
__device__ __forceinline__ float column_sum(float v) {
  if constexpr (L <= 2) v = dpp_add<0x122>(v);  // row_ror by 2, 4 and 8: the other lanes of the DPP row
  if constexpr (L <= 4) v = dpp_add<0x124>(v);
  if constexpr (L <= 8) v = dpp_add<0x128>(v);
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

// The sums of a lane's own columns in chunk k, in fp32 (their chunk takes two accesses where it has eight channels).
template <int L, int NV, int VE, bool LINES>
__device__ __forceinline__ void store_param(const RowSpan<L, NV, VE, LINES>& sp, int k, float* row, fv<VE> v) {
  if (sp.whole(k) || sp.skip[k] == 0) {
#pragma unroll
    for (int j = 0; j < VE; j += 4) store_chunk<4>(row + sp.at[k] + j, fv<4>{v[j], v[j + 1], v[j + 2], v[j + 3]});
  } else {
#pragma unroll
    for (int e = 1; e < VE; e++)
      if (e >= sp.skip[k]) row[sp.at[k] + e] = v[e];
  }
}

// The workgroup's sums over its rows of s (chunks as in sp) into out [D].
template <int L, int NV, int VE, bool LINES>
__device__ __forceinline__ void meet_columns(fv<VE> (&s)[NV], const RowSpan<L, NV, VE, LINES>& sp, int D, float* meet,
                                             float* out) {
  if constexpr (L > 64) {
#pragma unroll
    for (int k = 0; k < NV; k++) store_param(sp, k, out, s[k]);
  } else {
    __syncthreads();  // meet's last reader is done
#pragma unroll
    for (int k = 0; k < NV; k++) {
#pragma unroll
      for (int e = 0; e < VE; e++) s[k][e] = column_sum<L>(s[k][e]);
      if ((threadIdx.x & 63) < L) store_param(sp, k, meet + (threadIdx.x >> 6) * D, s[k]);
    }
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += 256) out[c] = (meet[c] + meet[D + c]) + (meet[2 * D + c] + meet[3 * D + c]);
  }
}

// One pass over x and the gradient (and dz_new), the next row's loads in flight while a row's three sums are formed.
// Bound by memory where rows are many: 1 M rows of 128 fp32 with an fp16 gradient 213 us (6.0 TB/s), the residual update's
// 357 us (5.7 TB/s), 2050 of 8192 bf16 20.5 us (5.7 TB/s with the partial sums). Where each lane has few rows the chain of
// the sums shows: 2000 of 768 bf16 6.2 us.
// Four waves a SIMD (128 registers) with 8 channels a lane, two with 16 or 24: what the sums, the row and the next row's loads
// need without spilling.
template <bool RES, typename TX, typename TG, typename TY, int L, int E, bool LINES>
__global__ __launch_bounds__(row_threads(L), E == 8 ? 4 : 2) void row_grad_k(RowGrad<TX, TG, TY> a) {
  constexpr int R = row_threads(L) / L, VE = RES ? 4 : chunk_of<TX, TG>(), NV = E / VE;
  __shared__ float red[4 * row_red(L)];
  __shared__ float meet[L <= 64 ? 4 * L * E : 1];
  const int D = a.D;
  const RowSpan<L, NV, VE, LINES> sp(threadIdx.x % L, D);
  const int64_t per = (D + 3) / 4;
  const float inv = 1.0f / D;
  Key key{};
  if (RES && a.drop.mode != DROP_OFF) key = drop_key(a.drop);
  fv<VE> sw[NV], sb[NV], w[NV];
  row_param(w, sp, a.w, 1.f);
#pragma unroll
  for (int k = 0; k < NV; k++) sw[k] = sb[k] = fv<VE>{};
  // the next row's loads are in flight while this one's sums are formed
  Raw<TX, VE> rx[NV];
  Raw<TG, VE> rg[NV];
  const auto fetch = [&](int64_t r) {
#pragma unroll
    for (int k = 0; k < NV; k++) {
      rx[k].load(a.x + r * D + sp.at[k]);
      rg[k].load(a.g + r * D + sp.at[k]);
    }
  };
  int64_t r = (int64_t)blockIdx.x * R + threadIdx.x / L;
  const int64_t step = (int64_t)gridDim.x * R;
  if (r < a.rows) fetch(r);
  for (; r < a.rows; r += step) {
    fv<VE> v[NV], g[NV];
    Raw<float, 4> z[NV];
#pragma unroll
    for (int k = 0; k < NV; k++) {
      if (RES && a.dz_new) z[k].load(a.dz_new + r * D + sp.at[k]);  // used last: it may be on its way meanwhile
      v[k] = rx[k].get();
      g[k] = rg[k].get();
    }
    if (r + step < a.rows) fetch(r + step);
    uint32_t bits = 0;  // of the lane's E elements, those that are kept
    if constexpr (RES) {
      if (a.drop.mode == DROP_ELEMENT) {
#pragma unroll
        for (int k = 0; k < NV; k++)
          bits |= (kept<VE>(a.drop, key, (uint64_t)r * per + (sp.at[k] >> 2), sp.at[k] & 3) & ((1u << VE) - 1)) << (k * VE);
      } else {
        bits = a.drop.mode >= DROP_ROW && drops_row(a.drop, key, r) ? 0u : ~0u;
      }
    }
    const float rstd = centre_row(v, sp, D, a.eps, red);
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      v[k] *= rstd;
      sw[k] += g[k] * v[k];
      sb[k] += g[k];
      g[k] *= w[k];
      c1 += sp.sum(k, g[k]);
      c2 += sp.sum(k, g[k] * v[k]);
    }
    c1 = row_sum<L>(c1, red + 2 * row_red(L)) * inv;
    c2 = row_sum<L>(c2, red + 3 * row_red(L)) * inv;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      fv<VE> o = (g[k] - c1 - v[k] * c2) * rstd;
      if constexpr (RES) {
        if (a.dz_new) o += z[k].get();
      }
      sp.store(k, a.dx + r * D, o);
      if constexpr (RES) {
        if (a.drop.mode != DROP_OFF) o = keep<VE>(a.drop, bits, k * VE, o);
        sp.store(k, a.dy + r * D, o);
      }
    }
  }
  if (!a.dw && !a.db) return;
  float* const ow = gridDim.x > 1 ? a.ws + (int64_t)blockIdx.x * 2 * D : a.dw;
  float* const ob = gridDim.x > 1 ? a.ws + (int64_t)blockIdx.x * 2 * D + D : a.db;
  if (ow) meet_columns(sw, sp, D, meet, ow);
  if (ob) meet_columns(sb, sp, D, meet, ob);
}

template <bool RES, typename TX, typename TG, typename TY>
static hipError_t launch_row_grad(const RowGrad<TX, TG, TY>& a, hipStream_t st) {
  const unsigned blocks = (unsigned)row_grad_blocks<RES>(a.rows, a.D);
  const hipError_t e = with_row_layout<RES>(a.D, [&](auto lay) {
    typedef decltype(lay) Lay;
    row_grad_k<RES, TX, TG, TY, Lay::L, Lay::E, Lay::LINES><<<blocks, row_threads(Lay::L), 0, st>>>(a);
    return hipGetLastError();
  });
  if (e != hipSuccess || blocks == 1 || (!a.dw && !a.db)) return e;
  return launch_row_grad_sum(a.ws, blocks, a.D, a.dw, a.db, st);
}

}  // namespace bzpf

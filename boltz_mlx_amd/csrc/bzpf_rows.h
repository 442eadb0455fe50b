// Rows of any width 8 <= D <= 8192 for the training kernels (LayerNorm, dropout, residual update): a row lies in the
// registers of L lanes, lane q holding the 8-channel chunks q, q + L, .. (NV of them), so that every pass over the row
// after the first is free of memory traffic.
#pragma once

#include "bzpf_common.h"
#include "bzpf_kernels.h"

typedef __bf16 bf16_t;
typedef float f8 __attribute__((ext_vector_type(8)));

namespace bzpf {

// Eight consecutive elements at element alignment (rows of odd widths, views at odd offsets): gfx950 loads and stores
// 16 bytes at any element alignment in one instruction, and at a 16-byte boundary as fast as an aligned type.
typedef float f4e __attribute__((ext_vector_type(4), aligned(4)));
typedef half_t h8e __attribute__((ext_vector_type(8), aligned(2)));
typedef bf16_t b8e __attribute__((ext_vector_type(8), aligned(2)));
typedef bf16_t b8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f8 load8(const float* p) {
  const f4e a = *reinterpret_cast<const f4e*>(p), b = *reinterpret_cast<const f4e*>(p + 4);
  return f8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
__device__ __forceinline__ f8 load8(const half_t* p) {
  return __builtin_convertvector(static_cast<half8>(*reinterpret_cast<const h8e*>(p)), f8);
}
__device__ __forceinline__ f8 load8(const bf16_t* p) {
  return __builtin_convertvector(static_cast<b8>(*reinterpret_cast<const b8e*>(p)), f8);
}
__device__ __forceinline__ void store8(float* p, f8 v) {
  *reinterpret_cast<f4e*>(p) = f4e{v[0], v[1], v[2], v[3]};
  *reinterpret_cast<f4e*>(p + 4) = f4e{v[4], v[5], v[6], v[7]};
}
__device__ __forceinline__ void store8(half_t* p, f8 v) {
  *reinterpret_cast<h8e*>(p) = __builtin_convertvector(v, half8);
}
__device__ __forceinline__ void store8(bf16_t* p, f8 v) { *reinterpret_cast<b8e*>(p) = __builtin_convertvector(v, b8); }

// Where a lane's chunks lie: chunk k covers the columns at[k] .. at[k] + 7. A chunk that would pass the row's end is
// moved back to D - 8, and its first skip[k] elements belong to its neighbour (8 or more: the chunk lies wholly past
// the end). Loads then need no branch; sums and stores leave the skipped elements out.
template <int L, int NV>
struct RowSpan {
  int at[NV], skip[NV];
  __device__ __forceinline__ RowSpan(int q, int D) {
#pragma unroll
    for (int k = 0; k < NV; k++) {
      const int c = 8 * (q + L * k);
      at[k] = min(c, D - 8);
      skip[k] = c - at[k];
    }
  }
  // v[k] without the skipped elements (zeros in their place)
  __device__ __forceinline__ f8 own(int k, f8 v) const {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = e >= skip[k] ? v[e] : 0.f;
    return v;
  }
  template <typename T>
  __device__ __forceinline__ void store(int k, T* row, f8 v) const {
    if (skip[k] == 0) {
      store8(row + at[k], v);
    } else if (skip[k] < 8) {
#pragma unroll
      for (int e = 1; e < 8; e++)
        if (e >= skip[k]) row[at[k] + e] = (T)v[e];
    }
  }
};

__device__ __forceinline__ float sum8(f8 v) { return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7])); }

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  const int u = __builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true);
  return v + __int_as_float(u);
}

// The sum of v over the L lanes of a row, in every one of them, in a fixed order. Steps of 1 and 2 lanes are quad
// permutations, 4 and 8 the mirrors of half a DPP row and of a whole one (the lanes that they pair hold equal sums by
// then), 16 and 32 the row and half-wave swaps. L = 256: the four waves' sums meet in `red` (four floats; a kernel that
// calls it several times in a loop gives each call its own four, at least two of them, so that the next call's barrier
// stands between a slot's reads and its next write).
template <int L>
__device__ __forceinline__ float row_sum(float v, float* red) {
  static_assert(L == 8 || L == 16 || L == 32 || L == 64 || L == 256, "lanes per row");
  v = dpp_add<0xB1>(v);   // quad_perm [1, 0, 3, 2]
  v = dpp_add<0x4E>(v);   // quad_perm [2, 3, 0, 1]
  v = dpp_add<0x141>(v);  // row_half_mirror
  if constexpr (L >= 16) v = dpp_add<0x140>(v);  // row_mirror
  if constexpr (L >= 32) {
    const unsigned u = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  if constexpr (L >= 64) {
    const unsigned u = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  if constexpr (L == 256) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
  }
  return v;
}

// Centres the row in v and returns 1 / sqrt(var + eps), by two passes over the registers (mean, then the squared
// deviations): both sums in fp32. Skipped elements are centred too and left out of the sums.
template <int L, int NV>
__device__ __forceinline__ float centre_row(f8 (&v)[NV], const RowSpan<L, NV>& sp, int D, float eps, float* red) {
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < NV; k++) s += sum8(sp.own(k, v[k]));
  const float inv = 1.0f / D;
  const float mean = row_sum<L>(s, red) * inv;
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < NV; k++) {
    v[k] -= mean;
    ss += sum8(sp.own(k, v[k] * v[k]));
  }
  return 1.0f / sqrtf(row_sum<L>(ss, red + 4) * inv + eps);
}

template <int L_, int NV_>
struct RowLayout {
  static constexpr int L = L_, NV = NV_;
};

// Calls fn with the row layout of width D: the fewest lanes that hold the row in one chunk each, then whole waves of 2
// and 4 chunks a lane, then whole workgroups.
template <typename Fn>
static inline hipError_t with_row_layout(int D, Fn&& fn) {
  if (D <= 64) return fn(RowLayout<8, 1>());
  if (D <= 128) return fn(RowLayout<16, 1>());
  if (D <= 256) return fn(RowLayout<32, 1>());
  if (D <= 512) return fn(RowLayout<64, 1>());
  if (D <= 1024) return fn(RowLayout<64, 2>());
  if (D <= 2048) return fn(RowLayout<64, 4>());
  if (D <= 4096) return fn(RowLayout<256, 2>());
  return fn(RowLayout<256, 4>());
}

// Calls fn(a, b) with a null pointer of each of the two storage types: fp32, fp16, bf16, but not fp16 with bf16.
template <typename Fn>
static inline hipError_t with_types(int a, int b, Fn&& fn) {
  typedef const float* F;
  typedef const half_t* H;
  typedef const bf16_t* B;
  if (a == DT_F32 && b == DT_F32) return fn(F(), F());
  if (a == DT_F32 && b == DT_F16) return fn(F(), H());
  if (a == DT_F32 && b == DT_BF16) return fn(F(), B());
  if (a == DT_F16 && b == DT_F16) return fn(H(), H());
  if (a == DT_F16 && b == DT_F32) return fn(H(), F());
  if (a == DT_BF16 && b == DT_BF16) return fn(B(), B());
  if (a == DT_BF16 && b == DT_F32) return fn(B(), F());
  return hipErrorInvalidValue;
}

// Workgroups for `rows` rows where one of 256 threads holds `per` rows at once: all of them up to `most`, the rest by
// a loop with the grid's stride.
static inline unsigned row_blocks(int64_t rows, int per, int64_t most) {
  const int64_t n = (rows + per - 1) / per;
  return (unsigned)(n < most ? n : most);
}

}  // namespace bzpf

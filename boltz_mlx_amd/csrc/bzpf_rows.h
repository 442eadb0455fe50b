// Rows of any width 8 <= D <= 8192 for the training kernels (LayerNorm, dropout, residual update): a row lies in the
// registers of L lanes, lane q holding the chunks q, q + L, .. (NV of them) of VE channels, so that every pass over the
// row after the first is free of memory traffic.
#pragma once

#include "bzpf_common.h"
#include "bzpf_kernels.h"

typedef __bf16 bf16_t;

namespace bzpf {

// Chunks are 16 bytes of the widest type of a call: 4 channels where one of its tensors is fp32, else 8. Then every load
// and store of a wave covers whole lines: chunks of 8 fp32 channels take two instructions of alternate 16-byte pieces,
// whose halves of a line reach memory apart.
template <typename... T> constexpr int chunk_of() { return (... || (sizeof(T) == 4)) ? 4 : 8; }

template <int VE> struct Chunk;
template <> struct Chunk<4> { typedef float f __attribute__((ext_vector_type(4))); };
template <> struct Chunk<8> { typedef float f __attribute__((ext_vector_type(8))); };
template <int VE> using fv = typename Chunk<VE>::f;

// VE consecutive elements of T at element alignment (rows of odd widths, views at odd offsets): gfx950 loads and stores 8
// or 16 bytes at any element alignment in one instruction, and at a whole boundary as fast as an aligned type. A Raw is a
// chunk as it is in memory, so that a load in flight holds the registers of its own type only.
template <typename T, int VE> struct Raw {
  typedef T V __attribute__((ext_vector_type(VE)));
  typedef T U __attribute__((ext_vector_type(VE), aligned(sizeof(T))));
  static_assert(VE * sizeof(T) <= 16, "one access");
  V v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const U*>(p); }
  __device__ __forceinline__ fv<VE> get() const { return __builtin_convertvector(v, fv<VE>); }
};

template <int VE, typename T>
__device__ __forceinline__ fv<VE> load_chunk(const T* p) {
  Raw<T, VE> r;
  r.load(p);
  return r.get();
}
// Outputs go out as non-temporal stores of whole lines: nothing of them waits in L2 for the write-back at the kernel's end.
// Residual update of 20 M elements 42 us instead of 45 (5 M: 11.7, 14.2), LayerNorm backward 39 instead of 42 (13.6, 15.6),
// dropout in fp16 22 instead of 24; at 128 M elements the gain is 2 to 4%. NT = false: ordinary stores (RowSpan::store).
template <int VE, bool NT = true, typename T>
__device__ __forceinline__ void store_chunk(T* p, fv<VE> v) {
  typedef typename Raw<T, VE>::V V;
  typedef typename Raw<T, VE>::U U;
  const U u = __builtin_convertvector(v, V);
  if constexpr (NT) __builtin_nontemporal_store(u, reinterpret_cast<U*>(p));
  else *reinterpret_cast<U*>(p) = u;
}

__device__ __forceinline__ float sum_of(fv<4> v) { return (v[0] + v[1]) + (v[2] + v[3]); }
__device__ __forceinline__ float sum_of(fv<8> v) {
  return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
}

// Where a lane's chunks lie: chunk k covers the columns at[k] .. at[k] + VE - 1. A chunk that would pass the row's end is
// moved back to D - VE, and its first skip[k] elements belong to its neighbour (VE or more: the chunk lies wholly past
// the end). Loads then need no branch; sums leave the skipped elements out. The first half of a lane's chunks is never
// moved (a layout serves widths past half of its own), none is where D fills the layout.
template <int L, int NV, int VE, bool LINES>
struct RowSpan {
  int at[NV], skip[NV];
  bool full, first;
  __device__ __forceinline__ RowSpan(int q, int D) {
#pragma unroll
    for (int k = 0; k < NV; k++) {
      const int c = VE * (q + L * k);
      at[k] = min(c, D - VE);
      skip[k] = c - at[k];
    }
    full = D == L * NV * VE;
    first = q == 0;
  }
  static constexpr bool whole(int k) { return k < NV / 2; }
  // the sum of chunk k's own elements
  __device__ __forceinline__ float sum(int k, fv<VE> v) const {
    if (!whole(k) && !full) {
#pragma unroll
      for (int e = 0; e < VE; e++) v[e] = e >= skip[k] ? v[e] : 0.f;
    }
    return sum_of(v);
  }
  // Chunk k of a row to memory. A chunk that was moved back writes its skipped elements too: the neighbour, who forms them in
  // the same chunk by the same instructions from the same values, writes the same bits (bf16 LayerNorm of 64 M elements at
  // D = 77 2.6 -> 3.3 TB/s, 100 3.5 -> 4.9); a row's first lane has its neighbour's in another chunk and writes its own one
  // by one.
  // Not LINES: several rows lie in a wave and end inside a 64-byte line in fp32, which ordinary stores leave to L2 to join:
  // residual update of 64 M elements at D = 77 3.5 -> 4.6 TB/s, 100 4.4 -> 5.2, 150 4.1 -> 5.0; from D = 257 on they lose
  // (300: 5.1 -> 4.9), and so do chunks of 8 half channels (LayerNorm of 16 M, D = 77: 3.1, 2.4).
  template <typename T>
  __device__ __forceinline__ void store(int k, T* row, fv<VE> v) const {
    if (whole(k) || skip[k] == 0 || (skip[k] < VE && !first)) {
      store_chunk<VE, LINES || VE == 8>(row + at[k], v);
    } else if (skip[k] < VE) {
#pragma unroll
      for (int e = 1; e < VE; e++)
        if (e >= skip[k]) row[at[k] + e] = (T)v[e];
    }
  }
};

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  const int u = __builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true);
  return v + __int_as_float(u);
}

// Threads of a workgroup whose rows take L lanes each: 256, or the L of one wide row.
constexpr int row_threads(int L) { return L > 256 ? L : 256; }

// The sum of v over the L lanes of a row, in every one of them, in a fixed order. Steps of 1 and 2 lanes are quad
// permutations, 4 and 8 the mirrors of half a DPP row and of a whole one (the lanes that they pair hold equal sums by
// then), 16 and 32 the row and half-wave swaps. L > 64 (the workgroup holds one row): the waves' sums meet in `red` (one
// float a wave; a kernel that calls it several times in a loop gives each call floats of its own, at least two such
// sets, so that the next call's barrier stands between a set's reads and its next write).
template <int L>
__device__ __forceinline__ float row_sum(float v, float* red) {
  static_assert(L >= 2 && L <= 1024 && (L & (L - 1)) == 0, "lanes per row");
  v = dpp_add<0xB1>(v);                          // quad_perm [1, 0, 3, 2]
  if constexpr (L >= 4) v = dpp_add<0x4E>(v);    // quad_perm [2, 3, 0, 1]
  if constexpr (L >= 8) v = dpp_add<0x141>(v);   // row_half_mirror
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
  if constexpr (L > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < L / 64; i += 2) v += red[i] + red[i + 1];
  }
  return v;
}
constexpr int row_red(int L) { return L > 64 ? L / 64 : 1; }  // floats that one call of row_sum needs

// A LayerNorm parameter at a lane's columns, or `none` where there is none: loaded before the rows, so that no load stands
// between a row's sums and its use (the wait for it would also wait for the next row's loads, which were issued before).
template <int L, int NV, int VE, bool LINES>
__device__ __forceinline__ void row_param(fv<VE> (&v)[NV], const RowSpan<L, NV, VE, LINES>& sp, const float* p, float none) {
#pragma unroll
  for (int k = 0; k < NV; k++) {
    if (p) {
#pragma unroll
      for (int j = 0; j < VE; j += 4) {
        const fv<4> t = load_chunk<4>(p + sp.at[k] + j);
        v[k][j] = t[0], v[k][j + 1] = t[1], v[k][j + 2] = t[2], v[k][j + 3] = t[3];
      }
    } else {
      v[k] = fv<VE>{} + none;
    }
  }
}

// Centres the row in v and returns 1 / sqrt(var + eps), by two passes over the registers (mean, then the squared
// deviations): both sums in fp32. Skipped elements are centred too and left out of the sums.
template <int L, int NV, int VE, bool LINES>
__device__ __forceinline__ float centre_row(fv<VE> (&v)[NV], const RowSpan<L, NV, VE, LINES>& sp, int D, float eps,
                                            float* red) {
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < NV; k++) s += sp.sum(k, v[k]);
  const float inv = 1.0f / D;
  const float mean = row_sum<L>(s, red) * inv;
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < NV; k++) {
    v[k] -= mean;
    ss += sp.sum(k, v[k] * v[k]);
  }
  const float var = row_sum<L>(ss, red + row_red(L)) * inv + eps;
  const bool tiny = var < 0x1p-100f;  // v_rsq_f32 (1 ulp) takes a denormal for 0
  return __builtin_amdgcn_rsqf(tiny ? var * 0x1p100f : var) * (tiny ? 0x1p50f : 1.f);
}

// L lanes a row, E channels a lane (E / VE chunks), LINES as in RowSpan::store.
template <int L_, int E_, bool LINES_ = true>
struct RowLayout {
  static constexpr int L = L_, E = E_;
  static constexpr bool LINES = LINES_;
};

// Calls fn with the row layout of width D. One wave or less a row while its registers hold it (no barrier then): 16 channels
// a lane, 24 without a residual update, whose backward pass spills there (1030 channels of 64 M elements: LayerNorm backward
// in bf16 2.0 -> 4.6 TB/s, with an update 3.6 -> 2.5). Whole workgroups beyond. Measured on the backward pass of 16 M
// elements in bf16 (fp32): D = 1024 as 64 x 16 26 us (43), as 256 x 8 39 (45); D = 2048 as 256 x 8 33 (42), as 64 x 32 (over
// 256 registers) 43 (57); D = 4096 as 256 x 16 30 (43), as 512 x 8 32 (43); D = 8192 as 512 x 16 31 (48), as 1024 x 8
// 34 (51).
template <bool RES, typename Fn>
static inline auto with_row_layout(int D, Fn&& fn) {
  if (D <= 256 && D % 16) {
    if (D <= 16) return fn(RowLayout<2, 8, false>());
    if (D <= 32) return fn(RowLayout<4, 8, false>());
    if (D <= 64) return fn(RowLayout<8, 8, false>());
    if (D <= 128) return fn(RowLayout<16, 8, false>());
    return fn(RowLayout<32, 8, false>());
  }
  if (D <= 16) return fn(RowLayout<2, 8>());
  if (D <= 32) return fn(RowLayout<4, 8>());
  if (D <= 64) return fn(RowLayout<8, 8>());
  if (D <= 128) return fn(RowLayout<16, 8>());
  if (D <= 256) return fn(RowLayout<32, 8>());
  if (D <= 512) return fn(RowLayout<64, 8>());
  if (D <= 1024) return fn(RowLayout<64, 16>());
  if constexpr (!RES) {
    if (D <= 1536) return fn(RowLayout<64, 24>());
  }
  if (D <= 2048) return fn(RowLayout<256, 8>());
  if (D <= 4096) return fn(RowLayout<256, 16>());
  return fn(RowLayout<512, 16>());
}

// Rows that a workgroup holds at once at width D.
template <bool RES>
static inline int row_places(int D) {
  return with_row_layout<RES>(D, [](auto lay) { return row_threads(decltype(lay)::L) / decltype(lay)::L; });
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

// Workgroups for `rows` rows where one holds `per` rows at once: all of them up to `most`, the rest by
// a loop with the grid's stride.
static inline unsigned row_blocks(int64_t rows, int per, int64_t most) {
  const int64_t n = (rows + per - 1) / per;
  return (unsigned)(n < most ? n : most);
}

}  // namespace bzpf

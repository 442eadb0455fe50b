// Pieces of the sequence attention's training form (bzpf_attn_fwd.hip, bzpf_attn_bwd.hip), in fp32, fp16 and bf16:
//   x = q.k / sqrt(C) + bias, without the keys that the mask leaves out;  p = softmax(x);  out = sigmoid(g) (p v).
// Products run in 32 x 32 MFMA tiles over steps of 16: a lane's fragment is 8 elements of one row, k = 8 (lane / 32) ..
// + 7 of the step; an fp32 step is eight v_mfma_f32_32x32x2 (fragment element j at instruction j: both operands take their
// k in the same order, so that the sum over the step is the same). An accumulator holds D[8 (i / 4) + 4 (lane / 32) + i % 4]
// [lane % 32], i = 0..15, which is the fragment layout of the next product's second operand with its k in the order
// 16 s + {4 hl .. 4 hl + 3, 8 + 4 hl .. 8 + 4 hl + 3}: probabilities never leave their lanes.
#pragma once

#include <type_traits>

#include "bzpf_common.h"
#include "bzpf_kernels.h"
#include "bzpf_rows.h"

namespace bzpf {

constexpr float LOG2E = 1.4426950408889634f;

template <typename T> struct Frag { typedef T V __attribute__((ext_vector_type(8))); };
template <typename T> using frag = typename Frag<T>::V;

__device__ __forceinline__ f16x mma(frag<half_t> a, frag<half_t> b, f16x c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f16x mma(frag<bf16_t> a, frag<bf16_t> b, f16x c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f16x mma(frag<float> a, frag<float> b, f16x c) {
#pragma unroll
  for (int j = 0; j < 8; j++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// Accumulator rows 16 s .. 16 s + 15 as a second operand (rounded to T: for half types a probability or its gradient is
// off by half a step of its own size, as the outputs are).
template <typename T>
__device__ __forceinline__ frag<T> as_frag(const f16x& c, int s) {
  frag<T> f;
#pragma unroll
  for (int j = 0; j < 8; j++) f[j] = (T)c[8 * s + j];
  return f;
}

// Tiles in LDS: rows of 32 NT channels, padded so that 16-byte reads of consecutive rows fall on different banks.
template <typename T, int KS> constexpr int TILE_LD = 32 * ((KS + 1) / 2) + 16 / (int)sizeof(T);

// Fragment of a product over channels: row `row`, channels 16 m + 8 hl ..
template <typename T, int KS>
__device__ __forceinline__ frag<T> row_frag(const T* tile, int row, int m) {
  const int hl = (threadIdx.x & 63) >> 5;
  return *reinterpret_cast<const frag<T>*>(tile + row * TILE_LD<T, KS> + 16 * m + 8 * hl);
}

// Fragment of a product over the tile's rows: channel 32 tt + lane % 32, rows row0 + {4 hl .., 8 + 4 hl ..}. Half types take
// it with the transposing LDS reads: 16 lanes read four rows of 16 channels and get four rows of one channel each.
template <typename T, int KS>
__device__ __forceinline__ frag<T> col_frag(const T* tile, int row0, int tt) {
  const int l = threadIdx.x & 63, hl = l >> 5;
  frag<T> f;
  if constexpr (sizeof(T) == 4) {
    const T* p = tile + (row0 + 4 * hl) * TILE_LD<T, KS> + 32 * tt + (l & 31);
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] = p[(j < 4 ? j : j + 4) * TILE_LD<T, KS>];
  } else {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4* lds4;
    const T* p = tile + (row0 + 4 * hl + ((l & 15) >> 2)) * TILE_LD<T, KS> + 32 * tt + 16 * ((l >> 4) & 1) + 4 * (l & 3);
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p);
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 8 * TILE_LD<T, KS>));
    f = __builtin_bit_cast(frag<T>, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  return f;
}

// 8 elements of a row in memory, at element alignment.
template <typename T>
__device__ __forceinline__ frag<T> load8(const T* p) {
  typedef T U __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  return *reinterpret_cast<const U*>(p);
}

// BR rows of a [rows][C] operand on their way from memory to a tile: loads are issued by load() and end in store(), a block
// of work later. Rows past the end are read at the last one and stored as zeros, as are those that `keep` leaves out
// (bit r: row r), so that nothing of theirs, infinite or NaN, meets a zero probability; so are the channels past C.
template <typename T, int KS, int BR, int NTH>
struct Stage {
  static constexpr int TOTAL = BR * 2 * KS, NV = (TOTAL + NTH - 1) / NTH;
  frag<T> r[NV];
  __device__ __forceinline__ void load(const T* base, int64_t ld, int64_t row0, int64_t rows, int C) {
#pragma unroll
    for (int n = 0; n < NV; n++) {
      const int e = threadIdx.x + NTH * n, c = 8 * (e % (2 * KS));
      const int64_t row = min(row0 + min(e / (2 * KS), BR - 1), rows - 1);
      r[n] = load8(base + row * ld + (c < C ? c : 0));
    }
  }
  __device__ __forceinline__ void store(T* tile, uint64_t keep, int C) const {
#pragma unroll
    for (int n = 0; n < NV; n++) {
      const int e = threadIdx.x + NTH * n, row = e / (2 * KS), c = 8 * (e % (2 * KS));
      if (TOTAL % NTH && e >= TOTAL) break;
      const bool on = c < C && (keep >> row & 1);
      *reinterpret_cast<frag<T>*>(tile + row * TILE_LD<T, KS> + c) = on ? r[n] : frag<T>{};
    }
  }
};

// Four consecutive bias elements of a row, of which n (4 and more: all) exist.
template <typename BT>
struct Bias4 {
  typedef BT V __attribute__((ext_vector_type(4)));
  V v;
  __device__ __forceinline__ void load(const BT* p) {
    typedef BT U __attribute__((ext_vector_type(4), aligned(sizeof(BT))));
    v = *reinterpret_cast<const U*>(p);
  }
  __device__ __forceinline__ void load(const BT* p, int64_t n) {
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = e < n ? p[e] : (BT)0.f;
  }
};

__device__ __forceinline__ float both_max(float v) {
  const unsigned u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float both_sum(float v) {
  const unsigned u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Whether the mask leaves the sample a key: one without keys runs without its mask.
template <int NTH>
__device__ __forceinline__ bool any_key(const float* mask, int64_t M) {
  if (!mask) return true;
  for (int64_t k = 0; k < M; k += NTH) {
    const int64_t at = k + threadIdx.x;
    if (__syncthreads_or(at < M && mask[at] != 0.0f)) return true;
  }
  return false;
}

// A workgroup's unit of work (block of rows fastest, then the sample, then the head), dealt to the 8 XCDs in contiguous
// ranges: workgroup b runs on XCD b % 8, so that an XCD's L2 holds a few heads' keys and biases. False: none.
struct Unit {
  int64_t block;
  int smp, h;
};
__device__ __forceinline__ bool unit_of(const Attn& a, int64_t blocks, int64_t per_xcd, Unit* u) {
  const int64_t n = (int64_t)(blockIdx.x % 8) * per_xcd + blockIdx.x / 8;
  if (n >= blocks * a.S * a.H) return false;
  u->block = n % blocks;
  u->smp = (int)(n / blocks % a.S);
  u->h = (int)(n / blocks / a.S);
  return true;
}

constexpr uint64_t all_rows(int n) { return n >= 64 ? ~0ull : (1ull << n) - 1; }

// Calls fn(T, BT, KS) with the types of q and of the bias and the number of 16-channel steps.
template <typename Fn>
static inline hipError_t with_attn(const Attn& a, Fn&& fn) {
  const auto steps = [&](auto t, auto b) {
    if (a.C <= 16) return fn(t, b, std::integral_constant<int, 1>());
    if (a.C <= 32) return fn(t, b, std::integral_constant<int, 2>());
    if (a.C <= 48) return fn(t, b, std::integral_constant<int, 3>());
    if (a.C <= 64) return fn(t, b, std::integral_constant<int, 4>());
    if (a.C <= 96) return fn(t, b, std::integral_constant<int, 6>());
    return fn(t, b, std::integral_constant<int, 8>());
  };
  if (a.dt == DT_F16) return steps(half_t(), half_t());
  if (a.dt == DT_BF16) return steps(bf16_t(), bf16_t());
  if (a.bias_dt == DT_F16) return steps(float(), half_t());
  if (a.bias_dt == DT_BF16) return steps(float(), bf16_t());
  return steps(float(), float());
}

}  // namespace bzpf

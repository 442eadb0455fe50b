// Pieces of the sequence attention's training form (bzpf_attn_fwd.hip, bzpf_attn_bwd.hip), in fp32, fp16 and bf16:
//   x = q.k / sqrt(C) + bias, without the keys that the mask leaves out;  p = softmax(x);  out = sigmoid(g) (p v).
// Products run in 32 x 32 MFMA tiles over steps of 16: a lane's fragment is 8 elements of one row, k = 8 (lane / 32) ..
// + 7 of the step; an fp32 step is eight v_mfma_f32_32x32x2 (fragment element j at instruction j: both operands take their
// k in the same order, so that the sum over the step is the same). An accumulator holds D[8 (i / 4) + 4 (lane / 32) + i % 4]
// [lane % 32], i = 0..15, which is the fragment layout of the next product's second operand with its k in the order
// 16 s + {4 hl .. 4 hl + 3, 8 + 4 hl .. 8 + 4 hl + 3}: probabilities never leave their lanes.
// Where the keys are an accumulator's rows (forward, dq), a tile's LDS rows hold them in the order that gives a lane's i-th
// element key 16 hl + i: a lane's 16 biases are then neighbours in memory.
#pragma once

#include <type_traits>

#include "bzpf_common.h"
#include "bzpf_kernels.h"
#include "bzpf_rows.h"

namespace bzpf {

constexpr float LOG2E = 1.4426950408889634f;

// A row's exponentials are 2^(x log2 e - at) for at = top log2 e rounded: one instruction before the exponential. What the
// rounding of at is worth, 2^off, is put right once for a row. Past 2^20 that would be too much for a half type's
// probabilities (and from 2^30 on for any): such a row (`big`) has 2^((x - top) log2 e), two instructions, with by = 1 and
// at = top; so a row whose logits are all the type's lowest value, or all one bar of any size, is a softmax over equals. A row
// without logits (top = -inf) has at = 0 and exponentials of 0.
struct Exponent {
  float top, by, at;
  __device__ __forceinline__ Exponent() {}
  __device__ __forceinline__ explicit Exponent(float t) : top(t) {
    by = __builtin_fabsf(t) > 0x1p20f && t != -INFINITY ? 1.0f : LOG2E;
    at = t == -INFINITY ? 0.f : t * by;
  }
  __device__ __forceinline__ bool big() const { return by == 1.0f; }
  __device__ __forceinline__ float of(float x) const {
    const float z = fmaf(x, by, -at);
    return __builtin_amdgcn_exp2f(big() ? z * LOG2E : z);
  }
  __device__ __forceinline__ float off() const { return top == -INFINITY ? 0.f : fmaf(top, by, -at); }
  // What sums of an earlier maximum are worth at this one, which is no smaller (of a row without logits so far: nothing).
  __device__ __forceinline__ float since(const Exponent& old) const {
    return old.top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(fmaf(old.top - top, LOG2E, off() - old.off()));
  }
};

// 16 logits' exponentials for a row a lane, where waves without big rows have one instruction each; `less`: powers of two off
// those of big rows.
__device__ __forceinline__ void exponentials(f16x& x, const Exponent& ex, bool some_big, float less = 0.f) {
  if (some_big) {
#pragma unroll
    for (int i = 0; i < 16; i++) x[i] = ex.big() ? fmaf(x[i] - ex.at, LOG2E, -less) : x[i];
  }
  const float at = ex.big() ? 0.f : ex.at;
#pragma unroll
  for (int i = 0; i < 16; i++) x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], ex.by, -at));
}

// How a launch's waves work (attn_split chooses): in the wide form the four waves of a workgroup hold 32 rows each and share
// tiles of the other side's rows, in two buffers; in the split form they hold the same 32 rows, each with every fourth block
// of the other side and tiles of its own (no barrier: a wave's LDS accesses keep their order), and meet at the end.
template <typename T, bool SPLIT>
struct Form {
  static constexpr int NW = SPLIT ? 1 : 4, GROUPS = SPLIT ? 4 : 1, NTH = 64 * NW, ROWS = 32 * NW;
  static constexpr int BR = SPLIT || sizeof(T) == 4 ? 32 : 64, BUFS = SPLIT ? 1 : 2;
  // Between a tile's writes and its reads. Two buffers: the other one's readers passed the barrier before, this one's next
  // writer passes the next one.
  static __device__ __forceinline__ void sync() {
    if constexpr (SPLIT) order();
    else __syncthreads();
  }
  // Between a tile's reads and its next writes.
  static __device__ __forceinline__ void again() {
    if constexpr (SPLIT) order();
  }
  static __device__ __forceinline__ void order() {  // of a wave's own LDS accesses: the compiler is to keep it
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
};

// Split where 128-row workgroups would be fewer than 300 (half types; 512 in fp32). dk/dv in us, wide and split, with bias and
// gate, of S H = 16, 48, 64, 72, 80, 128 heads of 400 x 400, which are 64, 192, 256, 288, 320, 512 such workgroups:
//   48 channels fp16: 29, 14; 30, 29; 31, 33; 38, 34; 39, 42; 42, 57.   24 channels fp32: 44, 18; 45, 39; 47, 49; 72, 49; 72, 59; 74, 80.
//   64 channels fp16: 29, 17; 30, 35; 31, 39; 39, 41; 40, 52; 44, 74.   64 channels fp32: 69, 29; 71, 82; 74, 109; 122, 110; 121, 135; 126, 190.
// The forward pass and dq turn at about the same places. One limit for all loses where the wide form fills the chip once, at 192 to 256
// workgroups of 64 and more channels (96 channels fp16 at 256: 42, 76), in fp32 of 64 channels at 320 and more too, and where a head's
// last workgroup is nearly empty. Heads past 96 channels have the wide form alone (their split form needs more registers than
// there are; the gated split form of 64 channels spills 5 to 14 of them in fp16).
constexpr int SPLIT_STEPS = 6;
static inline bool attn_split(int64_t rows, const Attn& a) {
  return a.C <= 16 * SPLIT_STEPS && (rows + 127) / 128 * a.S * a.H < (a.dt == DT_F32 ? 512 : 300);
}
// Calls fn(true_type) or fn(false_type) for it.
template <int KS, typename Fn>
static inline hipError_t with_split(int64_t rows, const Attn& a, Fn&& fn) {
  if constexpr (KS <= SPLIT_STEPS) {
    if (attn_split(rows, a)) return fn(std::true_type());
  }
  return fn(std::false_type());
}

// The sum over the four waves of a split workgroup of what each has in acc[NT] (a 32 x 32 tile each), for the accumulator rows
// 8 w .. 8 w + 7 of wave w: its part of the result, 4 elements for each of the tiles. `scale`: each wave's factor for its own.
template <int NT>
__device__ __forceinline__ void meet4(const f16x (&acc)[NT], f4* lds, int wave, int l, float scale, f4 (&out)[NT]) {
  __syncthreads();  // the area's last readers are done
#pragma unroll
  for (int tt = 0; tt < NT; tt++)
#pragma unroll
    for (int qq = 0; qq < 4; qq++) {
      f4 v;
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = acc[tt][4 * qq + e] * scale;
      lds[((wave * NT + tt) * 4 + qq) * 64 + l] = v;
    }
  __syncthreads();
#pragma unroll
  for (int tt = 0; tt < NT; tt++) {
    const f4* const p = lds + (tt * 4 + wave) * 64 + l;
    out[tt] = (p[0] + p[NT * 256]) + (p[2 * NT * 256] + p[3 * NT * 256]);
  }
}

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

constexpr __host__ __device__ uint64_t all_rows(int n) { return n >= 64 ? ~0ull : (1ull << n) - 1; }

// p and a 32-bit byte offset: with a wave-uniform p both are operands of the load itself.
template <typename T>
__device__ __forceinline__ T* at_byte(T* p, uint32_t bytes) {
  typedef std::conditional_t<std::is_const_v<T>, const char, char> B;
  return reinterpret_cast<T*>(reinterpret_cast<B*>(p) + bytes);
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
// Addresses are a wave's own base and a lane's 32-bit byte offset (one instruction's own operands): row pitches are below 2^23.
// KEYS: rows in the order of an accumulator's rows, as above.
template <typename T, int KS, int BR, int NTH, bool KEYS>
struct Stage {
  static constexpr int TOTAL = BR * 2 * KS, NV = (TOTAL + NTH - 1) / NTH;
  frag<T> r[NV];
  // base: the first row; left: rows from it on (at least one); t: the thread's number among NTH
  __device__ __forceinline__ void load(const T* base, uint32_t ld, int64_t left, int C, int t) {
    const int last = left < BR ? (int)left - 1 : BR - 1;
#pragma unroll
    for (int n = 0; n < NV; n++) {
      const int e = t + NTH * n, c = 8 * (e % (2 * KS));
      r[n] = load8(at_byte(base, ((uint32_t)min(e / (2 * KS), last) * ld + (c < C ? c : 0)) * (uint32_t)sizeof(T)));
    }
  }
  __device__ __forceinline__ void store(T* tile, uint64_t keep, int C, int t) const {
#pragma unroll
    for (int n = 0; n < NV; n++) {
      const int e = t + NTH * n, row = e / (2 * KS), c = 8 * (e % (2 * KS));
      if (TOTAL % NTH && e >= TOTAL) break;
      const bool on = c < C && (keep == all_rows(BR) || (keep >> row & 1));
      const int at = KEYS ? (row & ~31) + 8 * (row >> 2 & 3) + 4 * (row >> 4 & 1) + (row & 3) : row;
      *reinterpret_cast<frag<T>*>(tile + at * TILE_LD<T, KS> + c) = on ? r[n] : frag<T>{};
    }
  }
};

typedef unsigned int u4 __attribute__((ext_vector_type(4)));

// 16 bytes of elements without the first s of them (0 <= s < 16 / sizeof(BT); zeros come in behind).
template <typename BT>
__device__ __forceinline__ u4 without(u4 v, int s) {
  if constexpr (sizeof(BT) == 2) {
    if (s & 1) v = u4{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
    s >>= 1;
  }
  if (s & 1) v = u4{v[1], v[2], v[3], 0u};
  if (s & 2) v = u4{v[2], v[3], 0u, 0u};
  return v;
}
template <typename BT>
__device__ __forceinline__ u4 load_all(const BT* p) {
  typedef BT U __attribute__((ext_vector_type(16 / sizeof(BT)), aligned(sizeof(BT))));
  return __builtin_bit_cast(u4, *reinterpret_cast<const U*>(p));
}

// The biases of a wave's 32 rows against BK keys, on their way through LDS: from memory in whole rows (a lane for each row
// would take 32 lines an instruction: forward pass of 4096 x 4096, 16 heads bf16 227 us instead of 171), to the lanes that own
// the rows. 16-byte pieces lie at places that keep the lanes' reads of one column on different banks.
template <typename BT, int BK>
struct BiasRows {
  static constexpr int CPR = BK * (int)sizeof(BT) / 16, NV = 32 * CPR / 64, E = 16 / (int)sizeof(BT), BYTES = 32 * CPR * 16;
  u4 r[NV];
  static __device__ __forceinline__ int place(int row, int c) {
    return row * CPR + (CPR == 8 ? c ^ (row & 7) : c ^ (row >> 1 & 3));
  }
  // base: the wave's first row; rows: those of the 32 that exist (at least one); from key k0 on. A piece that the row's end cuts
  // is read where it ends with the row, and put right in store() (an element at a time took 1.2 to 1.5 times as long for the
  // whole kernel at 400 and 2000 keys).
  __device__ __forceinline__ void load(const BT* base, int rows, int M, int k0) {
    const int l = threadIdx.x & 63, last = M - k0 - E;
    if (M < E) {
      load_short(base, rows, M);
      return;
    }
#pragma unroll
    for (int n = 0; n < NV; n++) {
      const int id = l + 64 * n;
      r[n] = load_all(at_byte(base, (uint32_t)(min(id / CPR, rows - 1) * M + k0 + min(id % CPR * E, last)) * (uint32_t)sizeof(BT)));
    }
  }
  // Rows of fewer elements than a piece has: one by one, from the first on.
  __device__ __forceinline__ void load_short(const BT* base, int rows, int M) {
    typedef BT V __attribute__((ext_vector_type(E)));
    const int l = threadIdx.x & 63;
    V v[NV] = {};
#pragma unroll 1
    for (int e = M - 1; e >= 0; e--) {
#pragma unroll
      for (int n = 0; n < NV; n++) {
        const BT x = base[min((l + 64 * n) / CPR, rows - 1) * M + e];
        V w;
        w[0] = x;
#pragma unroll
        for (int i = 1; i < E; i++) w[i] = v[n][i - 1];
        v[n] = w;
      }
    }
#pragma unroll
    for (int n = 0; n < NV; n++) r[n] = __builtin_bit_cast(u4, v[n]);
  }
  __device__ __forceinline__ void store(u4* lds, int M, int k0) const {
    const int l = threadIdx.x & 63, last = M - k0 - E;
#pragma unroll
    for (int n = 0; n < NV; n++) {
      const int c = (l + 64 * n) % CPR;
      u4 v = r[n];
      if (last < BK - E && M >= E) v = without<BT>(v, max(c * E - last, 0) & (E - 1));  // a piece past the end: no matter what
      lds[place((l + 64 * n) / CPR, c)] = v;
    }
  }
  // The lane's 16 of tile kt.
  static __device__ __forceinline__ f16x get(const u4* lds, int kt) {
    typedef BT V __attribute__((ext_vector_type(E)));
    const int l = threadIdx.x & 63;
    f16x x;
#pragma unroll
    for (int p = 0; p < 16 / E; p++) {
      const V v = __builtin_bit_cast(V, lds[place(l & 31, (32 * kt + 16 * (l >> 5)) / E + p)]);
#pragma unroll
      for (int e = 0; e < E; e++) x[p * E + e] = (float)v[e];
    }
    return x;
  }
};

// Rows of a matrix tile whose columns are a wave's lanes, a row an instruction: the tile is a buffer, the row's offset the
// instruction's scalar one, so that an access costs no address arithmetic. Past the buffer's end loads give 0 and stores drop.
template <typename BT>
struct Columns {
  __amdgpu_buffer_rsrc_t rsrc;
  uint32_t pitch;  // bytes
  // base: the tile's first row; rows: those of it that exist
  __device__ __forceinline__ Columns(const BT* base, int rows, int64_t M)
      : rsrc(__builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)(rows * M * (int64_t)sizeof(BT)), 0x00020000)),
        pitch((uint32_t)M * (uint32_t)sizeof(BT)) {}
  // lane: byte offset of the lane's first row and column; r: the row from there; whole: every row of the tile exists (else the
  // row has to be in the lane's offset, which the range check covers: 16 of them, not to be kept over a loop)
  __device__ __forceinline__ BT get(uint32_t lane, int r, bool whole) const {
    if (!whole) asm volatile("" : "+v"(lane));
    const int v = whole ? (int)lane : (int)(lane + r * pitch), s = whole ? (int)(r * pitch) : 0;
    if constexpr (sizeof(BT) == 2)
      return __builtin_bit_cast(BT, (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rsrc, v, s, 0));
    else
      return __builtin_bit_cast(BT, (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rsrc, v, s, 0));
  }
  // 16 values on their way to memory: those of half types in pairs, as conversions make them; zeros where not `on`.
  struct Packed {
    static constexpr int E = 4 / (int)sizeof(BT);
    uint32_t w[16 / E];
    __device__ __forceinline__ Packed(const f16x& x, bool on) {
      typedef BT V __attribute__((ext_vector_type(E)));
#pragma unroll
      for (int i = 0; i < 16; i += E) {
        V v;
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = (BT)x[i + e];
        w[i / E] = on ? __builtin_bit_cast(uint32_t, v) : 0u;
      }
    }
    __device__ __forceinline__ uint32_t operator[](int i) const { return w[i / E] >> (32 / E * (i % E) & 31); }
  };
  __device__ __forceinline__ void put(uint32_t lane, int r, bool whole, uint32_t x) const {
    if (!whole) asm volatile("" : "+v"(lane));
    const int v = whole ? (int)lane : (int)(lane + r * pitch), s = whole ? (int)(r * pitch) : 0;
    if constexpr (sizeof(BT) == 2)
      __builtin_amdgcn_raw_buffer_store_b16((uint16_t)x, rsrc, v, s, 0);
    else
      __builtin_amdgcn_raw_buffer_store_b32(x, rsrc, v, s, 0);
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

// Whether the mask leaves the sample a key (all 256 threads of the workgroup): one without keys runs without its mask.
__device__ __forceinline__ bool any_key(const float* mask, int64_t M) {
  for (int64_t k = 0; k < M; k += 256) {
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
__device__ __forceinline__ bool unit_of(const Attn& a, int64_t blocks, int64_t per_xcd, Unit* u) {  // all below 2^31
  const uint32_t n = blockIdx.x % 8 * (uint32_t)per_xcd + blockIdx.x / 8, per_head = (uint32_t)blocks * (uint32_t)a.S;
  u->h = (int)(n / per_head);
  if (u->h >= a.H) return false;
  const uint32_t rest = n - (uint32_t)u->h * per_head;
  u->smp = (int)(rest / (uint32_t)blocks);
  u->block = rest - (uint32_t)u->smp * (uint32_t)blocks;
  return true;
}

// Calls fn(T, BT, KS) with the types of q and of the bias and the number of 16-channel steps.
template <typename Fn>
static inline hipError_t with_attn(const Attn& a, Fn&& fn) {
  const auto steps = [&](auto t, auto b) {
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

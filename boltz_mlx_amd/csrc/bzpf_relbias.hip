// A learned relative position bias by buckets, and its table's gradient:
//   bias[b][h][i][j] = table[bucket(pos_q[b][i] - pos_k[b][j])][h] (+ add[b][h][i][j])
//   dtable[k][h] = sum over (b, i, j) whose pair lies in bucket k of dbias[b][h][i][j].
// bucket(d) = lut[clamp(d - lo, 0, span - 1)], not falling with d; pairs of different groups (chains) take the last one.
//
// Both are bound by memory: the bias is written once (the pair bias read once), its gradient read once. A thread owns a
// chunk of 16 bytes of a row. As buckets do not fall with the distance, the ends of a chunk's positions say whether it lies
// beyond the first or the last edge (most do, or are of another chain): then one number serves the whole chunk.
#include <type_traits>

#include "bzpf_common.h"
#include "bzpf_kernels.h"
#include "bzpf_rows.h"

namespace bzpf {

namespace {

// A position or group number, 32 or 64 bits wide. Both are two loads of 32 bits, the second of the same ones where there are
// no others: a branch would end in a wait for each number, one after the other (table's gradient of 16 x 2000 x 2000 in
// bfloat16 with one row in flight 58 us so, 96 us with a branch).
template <typename P>
__device__ __forceinline__ int64_t number(P p, bool wide, int64_t i) {
  const int64_t at = i << wide;
  const uint32_t lo = p[at], hi = p[at + wide];
  return (int64_t)((uint64_t)(wide ? hi : (uint32_t)((int32_t)lo >> 31)) << 32 | lo);
}
__device__ __forceinline__ int64_t whole(const void* p, bool wide, int64_t i) {
  return number(static_cast<const uint32_t*>(p), wide, i);
}
// At a place that is the same in every lane: scalar loads.
__device__ __forceinline__ int64_t scalar(const void* p, bool wide, int64_t i) {
  return number((const __attribute__((address_space(4))) uint32_t*)p, wide, i);
}

// V of them from place i on, of which there are at least n (the last one stands in for the rest). In vectors, the branch around
// all of them: two loads a number, each lane's a line of its own, took 22 us instead of 12 for the bias of 400 x 400.
template <int V>
__device__ __forceinline__ void numbers(const void* p, bool wide, int64_t i, int64_t n, int64_t (&to)[V]) {
  typedef int64_t W __attribute__((ext_vector_type(2), aligned(8)));
  typedef int32_t D __attribute__((ext_vector_type(4), aligned(4)));
  if (n < V) {
#pragma unroll 1
    for (int e = 0; e < V; e++) {
      const int64_t x = whole(p, wide, i + (e < n ? e : n - 1));
#pragma unroll
      for (int k = 0; k < V; k++) to[k] = k == e ? x : to[k];
    }
  } else if (wide) {
    const W* const q = reinterpret_cast<const W*>(static_cast<const int64_t*>(p) + i);
#pragma unroll
    for (int e = 0; e < V; e++) to[e] = q[e / 2][e % 2];
  } else {
    const D* const q = reinterpret_cast<const D*>(static_cast<const int32_t*>(p) + i);
#pragma unroll
    for (int e = 0; e < V; e++) to[e] = q[e / 4][e % 4];
  }
}

// The distance d from the lowest one, lo, held to `most` either way (past it all are alike: edges are at most 2^14 apart). Numbers
// are below 2^62 in size, so that d takes 63 bits and d - lo may take 64.
__device__ __forceinline__ int from_lowest(int64_t d, int64_t lo, int64_t most) {
  return (int)(d < lo - most ? -most : d > lo + most ? most : d - lo);
}

// Where a chunk of keys lies for a query: in one bucket (the first, the last, other groups') or in several.
enum { FIRST, LAST, OTHER, MIXED };

// A chunk of V keys: their positions from the first one's on in 32 bits, and their groups, one up to `cut` and another from
// there on. `rare`: positions that do not fit, or more groups; such a chunk's keys are looked at one by one in memory.
template <int V>
struct Keys {
  int rel[V], least, most, cut;
  int64_t base, group0, group1;
  bool rare;
  __device__ __forceinline__ void load(const RelBias& a, int64_t at, int n) {
    rare = false, cut = V, least = most = 0;
    int64_t pos[V], group[V];
    numbers(a.pos_k, a.wide, at, n, pos);
    if (a.group_k) numbers(a.group_k, a.wide, at, n, group);
    base = pos[0];
    if (a.group_k) group0 = group[0], group1 = group[V - 1];
#pragma unroll
    for (int e = 0; e < V; e++) {
      const int64_t d = pos[e] - base;
      rare |= d >= FAR || d <= -FAR;
      rel[e] = (int)d;
      least = min(least, rel[e]);
      most = max(most, rel[e]);
      if (a.group_k) {
        if (cut == V && group[e] != group0) cut = e;
        rare |= e >= cut && group[e] != group1;
      }
    }
  }
  static constexpr int64_t FAR = 1 << 29;
};

// A query against a chunk.
template <int V>
struct Query {
  int from, kind;  // distance - lo of the chunk's first key, at most 2^30 either way
  bool same0, same1;
  __device__ __forceinline__ Query(const RelBias& a, const Keys<V>& k, int64_t pos, int64_t group) {
    from = from_lowest(pos - k.base, a.lo, 2 * Keys<V>::FAR);
    same0 = !a.group_k || group == k.group0;
    same1 = k.cut == V ? same0 : group == k.group1;
    kind = !same0 && !same1 ? OTHER : !same0 || !same1 ? MIXED : from - k.least <= 0 ? FIRST : from - k.most >= a.span - 1 ? LAST : MIXED;
    if (k.rare) kind = MIXED;
  }
  // The keys' buckets, of a chunk that is not rare.
  __device__ __forceinline__ void buckets(const RelBias& a, const uint8_t* lut, const Keys<V>& k, int (&at)[V]) const {
#pragma unroll
    for (int e = 0; e < V; e++) at[e] = lut[min(max(from - k.rel[e], 0), a.span - 1)];
    if (a.group_k) {
      const unsigned first = (1u << k.cut) - 1, same = (same0 ? first : 0u) | (same1 ? ~first : 0u);
#pragma unroll
      for (int e = 0; e < V; e++) at[e] = same >> e & 1 ? at[e] : a.count - 1;
    }
  }
  // The bucket of a chunk that lies in one.
  __device__ __forceinline__ int one(const RelBias& a, const uint8_t* lut) const {
    return kind == OTHER ? a.count - 1 : lut[kind == FIRST ? 0 : a.span - 1];
  }
};

// The bucket of query i and key j from memory.
__device__ __forceinline__ int bucket_of(const RelBias& a, const uint8_t* lut, int64_t i, int64_t j) {
  if (a.group_q && whole(a.group_q, a.wide, i) != whole(a.group_k, a.wide, j)) return a.count - 1;
  const int d = from_lowest(whole(a.pos_q, a.wide, i) - whole(a.pos_k, a.wide, j), a.lo, a.span);
  return lut[min(max(d, 0), a.span - 1)];
}

// The batch element's own positions and groups.
__device__ __forceinline__ RelBias of_batch(RelBias a, int64_t b) {
  const int64_t w = a.wide ? 8 : 4;
  const auto step = [&](const void* p, int64_t n) { return p ? static_cast<const char*>(p) + b * n * w : nullptr; };
  a.pos_q = step(a.pos_q, a.batch_q), a.group_q = step(a.group_q, a.batch_q);
  a.pos_k = step(a.pos_k, a.batch_k), a.group_k = step(a.group_k, a.batch_k);
  return a;
}

template <typename T>
constexpr int CHUNK = 16 / (int)sizeof(T);

// Threads of a row (a power of two) in a workgroup of `threads`: enough for its chunks.
__host__ __device__ __forceinline__ int row_lanes(int64_t chunks, int threads) {
  int n = 1;
  while (n < threads && n < chunks) n *= 2;
  return n;
}

// grid (row blocks, head groups of `heads`, batch); LDS: the group's part of the table, then the look-up table. A thread keeps
// its keys over its rows and heads. Bound by the writes: 16 x 2000 x 2000 fp32 44 us (5.8 TB/s), bf16 28 us (4.5), bf16 with a
// pair bias 53 us (4.8); 2 x 16 x 400 x 400 fp16 with one 9.9 us, latency.
template <typename T>
__global__ __launch_bounds__(256) void rel_bias_k(RelBias a, const T* __restrict__ add, T* __restrict__ out, int heads,
                                                  int rows_per) {
  constexpr int V = CHUNK<T>;
  extern __shared__ float tab[];
  const int h0 = blockIdx.y * heads, nh = min(heads, a.H - h0), t = threadIdx.x;
  uint8_t* const lut = reinterpret_cast<uint8_t*>(tab + heads * a.count);
  for (int h = t >> 6; h < nh; h += 4)
    for (int k = t & 63; k < a.count; k += 64) tab[h * a.count + k] = a.table[(int64_t)k * a.H + h0 + h];
  for (int e = t; e < a.span; e += 256) lut[e] = a.lut[e];
  __syncthreads();
  const int64_t b = blockIdx.z;
  a = of_batch(a, b);
  const int64_t chunks = (a.M + V - 1) / V, r1 = min(a.N, ((int64_t)blockIdx.x + 1) * rows_per);
  const int L = row_lanes(chunks, 256), n = a.M < V ? (int)a.M : V;
  for (int64_t c = t % L; c < chunks; c += L) {
    const int64_t j0 = min(c * V, a.M - n);  // the last chunk is moved back: its neighbour's keys get the same values
    Keys<V> keys;
    keys.load(a, j0, n);
    const int64_t plane = a.N * a.M;
    int64_t i = (int64_t)blockIdx.x * rows_per + t / L;
    const auto pos_of = [&](int64_t i) { return whole(a.pos_q, a.wide, min(i, a.N - 1)); };
    const auto group_of = [&](int64_t i) { return a.group_q ? whole(a.group_q, a.wide, min(i, a.N - 1)) : 0; };
    int64_t pos = pos_of(i), group = group_of(i);
    for (; i < r1; i += 256 / L) {
      const Query<V> q(a, keys, pos, group);
      pos = pos_of(i + 256 / L), group = group_of(i + 256 / L);  // the next row's, on their way
      const int64_t base = ((b * a.H + h0) * a.N + i) * a.M + j0;
      if (keys.rare || n < V) {
#pragma unroll 1
        for (int e = 0; e < n; e++) {
          const int k = bucket_of(a, lut, i, j0 + e);
#pragma unroll 1
          for (int h = 0; h < nh; h++) {
            const int64_t to = base + h * plane + e;
            out[to] = (T)(add ? tab[h * a.count + k] + (float)add[to] : tab[h * a.count + k]);
          }
        }
        continue;
      }
      int at[V];
      if (q.kind == MIXED) {
        q.buckets(a, lut, keys, at);
      } else {
        const int one = q.one(a, lut);
#pragma unroll
        for (int e = 0; e < V; e++) at[e] = one;
      }
      const bool all_one = __all(q.kind != MIXED);
#pragma unroll 1
      for (int h = 0; h < nh; h += 4) {  // four heads' pair biases on their way at once
        Raw<T, V> r[4];
        if (add) {
#pragma unroll
          for (int u = 0; u < 4; u++) r[u].load(add + base + min(h + u, nh - 1) * plane);
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
          if (h + u >= nh) break;
          const float* const row = tab + (h + u) * a.count;
          fv<V> v;
          if (all_one) {
            v = fv<V>{} + row[at[0]];
          } else {
#pragma unroll
            for (int e = 0; e < V; e++) v[e] = row[at[e]];
          }
          if (add) v += r[u].get();
          store_chunk<V, false>(out + base + (h + u) * plane, v);
        }
      }
    }
  }
}

// The gradient as products with one-hot rows on the matrix cores: a wave takes 32 keys of a row at a time for 16 heads, the
// heads' 32 values as a 32 x 16 operand and, for every 16 buckets that the pairs reach, a 16 x 32 one whose rows say which
// pairs lie in a bucket: 16 x 16 sums in fp32. Adding into LDS, a column a thread, took 104 us for 16 x 2000 x 2000 bf16 (an LDS
// addition of a wave's 64 lanes costs about 100 cycles there). Half types are their own operand, fp32 goes as three bf16
// parts, which hold its 24 bits. Rows whose 32 pairs lie in one bucket (beyond the first or last edge, in another chain: most)
// are added up without a product, and a product is left out where none of its 16 buckets is reached. A value that is not
// finite spoils its head's sums. 16 x 2000 x 2000 bf16, logarithmic buckets to 512: 37 us (3.4 TB/s); 2 x 16 x 400 x 400 fp16, three
// chains: 14 us, which is the latency of eight rows behind the keys' and the look-up table's.
template <typename T> struct OneHot;
template <> struct OneHot<half_t> {
  typedef half_t P;
  static constexpr uint32_t ONE = 0x3C00u;
  static constexpr int PARTS = 1;
};
template <> struct OneHot<bf16_t> {
  typedef bf16_t P;
  static constexpr uint32_t ONE = 0x3F80u;
  static constexpr int PARTS = 1;
};
template <> struct OneHot<float> {
  typedef bf16_t P;
  static constexpr uint32_t ONE = 0x3F80u;
  static constexpr int PARTS = 3;
};
typedef half_t h8 __attribute__((ext_vector_type(8)));
typedef bf16_t b8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ f4 mma16(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 mma16(b8 a, b8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

constexpr int64_t BOUND = (int64_t)1 << 30;  // of distances from the lowest one

constexpr int GK = 8;  // keys of a lane: a product's k = 8 (lane / 16) .. + 7

// A wave's 32 keys, each lane's 8 neighbours: their distances from the first key and their groups, in 32 bits. Past the end a
// lane's keys are moved back to the last 8, and the first `skip` of them are its neighbours' (there are at least 8).
struct KeyTile {
  int rel[GK], group[GK];
  int64_t base;
  int least, most, first_group;
  bool one_group, rare;  // rare: positions or groups that 32 bits do not hold
  int64_t j;             // the lane's first key
  int skip;
  __device__ __forceinline__ void load(const RelBias& a, int64_t j0) {
    const int64_t want = j0 + GK * ((threadIdx.x & 63) >> 4);
    j = min(want, max(a.M - GK, (int64_t)0));
    skip = (int)min(want - j, (int64_t)GK);
    base = scalar(a.pos_k, a.wide, j0);
    int64_t pos[GK], groups[GK] = {};
    numbers(a.pos_k, a.wide, j, a.M, pos);
    if (a.group_k) numbers(a.group_k, a.wide, j, a.M, groups);
    bool far = false, other = false;
    int lo = 0, hi = 0;
    first_group = __builtin_amdgcn_readfirstlane((int)groups[0]);
#pragma unroll
    for (int e = 0; e < GK; e++) {
      const int64_t d = pos[e] - base;
      rel[e] = (int)d;
      group[e] = (int)groups[e];
      far |= d < -BOUND / 2 || d > BOUND / 2 || group[e] != groups[e];
      lo = min(lo, rel[e]);
      hi = max(hi, rel[e]);
      other |= group[e] != first_group;
    }
    for (int o = 16; o < 64; o *= 2) lo = min(lo, __shfl_xor(lo, o)), hi = max(hi, __shfl_xor(hi, o));
    least = __builtin_amdgcn_readfirstlane(lo);
    most = __builtin_amdgcn_readfirstlane(hi);
    one_group = !__any(other);
    rare = __any(far);
  }
};

// Eight neighbouring values on their way. ODD: 16-bit ones that may begin inside a dword, where a load of 16 bytes takes twice
// as long: it begins at the dword then, with the value before them, and the last one comes by itself.
template <typename T, bool ODD>
struct EightOf {
  typedef T V __attribute__((ext_vector_type(GK)));
  typedef T U __attribute__((ext_vector_type(GK), aligned(sizeof(T))));
  V v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const U*>(p); }
  __device__ __forceinline__ V get() const { return v; }
};
template <typename T>
struct EightOf<T, true> {
  typedef T V __attribute__((ext_vector_type(GK)));
  typedef uint32_t D __attribute__((ext_vector_type(4), aligned(4)));
  D x;
  uint16_t last;
  uint32_t shift;
  __device__ __forceinline__ void load(const T* p) {
    const int odd = (int)(reinterpret_cast<uintptr_t>(p) >> 1 & 1);
    x = *reinterpret_cast<const D*>(p - odd);
    last = __builtin_bit_cast(uint16_t, p[GK - 1]);
    shift = 16u * odd;
  }
  __device__ __forceinline__ V get() const {
    D y;
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = __builtin_amdgcn_alignbit(e < 3 ? x[e + 1] : (uint32_t)last, x[e], shift);
    return __builtin_bit_cast(V, y);
  }
};

// grid (blocks of 128 keys, row blocks, batch times groups of 16 heads); partial sums [row block, key block, batch][H][count].
// BT: groups of 16 buckets.
template <typename T, int BT>
__global__ __launch_bounds__(256) void rel_bias_bwd_k(RelBias a, const T* __restrict__ dy, float* __restrict__ part, int rows_per) {
  typedef OneHot<T> OH;
  typedef typename OH::P P;
  typedef P P8 __attribute__((ext_vector_type(8)));
  typedef T TV __attribute__((ext_vector_type(GK)));
  typedef T TU __attribute__((ext_vector_type(GK), aligned(sizeof(T))));
  __shared__ float meet[16][16 * BT + 1];
  const int l = threadIdx.x & 63, c = l & 15, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hg = (a.H + 15) / 16;
  const int64_t b = blockIdx.z / hg;
  const int h0 = 16 * (int)(blockIdx.z % hg), h = min(h0 + c, a.H - 1);
  a = of_batch(a, b);
  for (int e = threadIdx.x; e < 16 * (16 * BT + 1); e += 256) (&meet[0][0])[e] = 0.f;
  // The lane's buckets, 16 t + c: distances (from lo) `from` .. from + width - 1. The look-up table does not fall: bucket k's
  // distances start where its entries reach k.
  __shared__ int start[257];
  for (int i = 1 + threadIdx.x; i < a.span; i += 256)
    for (int k = a.lut[i - 1] + 1; k <= a.lut[i]; k++) start[k] = i;
  __syncthreads();
  int from[BT];
  uint32_t width[BT];
  const int first = a.lut[0], last = a.lut[a.span - 1];
  // The distance of a pair of different groups: none that a pair has, or one of the last bucket where that is theirs too.
  const int others = last == a.count - 1 ? (int)BOUND : INT32_MIN;
#pragma unroll
  for (int t = 0; t < BT; t++) {
    const int k = 16 * t + c;
    const bool in = k >= first && k <= last;
    const int64_t at = in && k > first ? start[k] : -BOUND * 2 + 1, end = in && k < last ? start[k + 1] : BOUND * 2;
    from[t] = in ? (int)at : 0;
    width[t] = in ? (uint32_t)(end - at) : 0u;
    if (a.group_k && k == a.count - 1 && k != last) from[t] = others, width[t] = 1;
  }
  f4 acc[BT];
#pragma unroll
  for (int t = 0; t < BT; t++) acc[t] = f4{};
  float run[3] = {0.f, 0.f, 0.f};  // the lane's head, of rows in one bucket
  const int64_t r0 = (int64_t)blockIdx.y * rows_per, r1 = min(a.N, r0 + rows_per);
  const int64_t j0 = (int64_t)blockIdx.x * 16 * GK + 4 * GK * wave;
  if (j0 < a.M) {
    KeyTile keys;
    keys.load(a, j0);
    // lanes past the last head have its values too, in sums of their own that go nowhere
    const T* const col = dy + ((b * a.H + h) * a.N) * a.M + keys.j;
    // 32 pairs of a row in several buckets, at distances d: a product for each 16 buckets of `reached`.
    const auto products = [&](const TV& v, const int (&d)[GK], uint32_t reached) {
      P8 x[OH::PARTS];
#pragma unroll
      for (int e = 0; e < GK; e++) {
        if constexpr (OH::PARTS == 1) {
          x[0][e] = v[e];
        } else {
          // cut off, not rounded: the largest numbers would round to infinity
          const auto cut = [](float x) { return __uint_as_float(__float_as_uint(x) & 0xFFFF0000u); };
          const float hi = cut(v[e]), mid = cut(v[e] - hi);
          x[0][e] = (P)hi;
          x[1][e] = (P)mid;
          x[2][e] = (P)(v[e] - hi - mid);
        }
      }
#pragma unroll
      for (int t = 0; t < BT; t++) {
        if (BT > 2 && !(reached >> t & 1)) continue;
        typedef uint32_t W4 __attribute__((ext_vector_type(4)));
        W4 w;
#pragma unroll
        for (int e = 0; e < GK; e += 2) {
          const bool p = (uint32_t)d[e] - (uint32_t)from[t] < width[t], q = (uint32_t)d[e + 1] - (uint32_t)from[t] < width[t];
          w[e / 2] = (p ? OH::ONE : 0u) | (q ? OH::ONE << 16 : 0u);
        }
#pragma unroll
        for (int p = 0; p < OH::PARTS; p++) acc[t] = mma16(__builtin_bit_cast(P8, w), x[p], acc[t]);
      }
    };
    const auto sum_up = [&](const TV& v, int k) {  // 32 pairs in one bucket
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < GK; e += 2) s += (float)v[e] + (float)v[e + 1];
      if (k == FIRST) run[FIRST] += s;
      else if (k == LAST) run[LAST] += s;
      else run[OTHER] += s;
    };
    // 64 rows' distances, kinds and reached buckets at once, a lane a row; then row by row, some rows' values on their way.
    const auto all_rows = [&](auto odd_rows) {
      constexpr bool ODD = decltype(odd_rows)::value;
      constexpr int U = BT > 5 ? 2 : 4;
      const bool whole_tile = j0 + 4 * GK <= a.M;
      const auto fetch = [&](int64_t i) {
        EightOf<T, ODD> f;
        f.load(col + min(i, r1 - 1) * a.M);
        return f;
      };
      EightOf<T, ODD> f[U];
#pragma unroll
      for (int u = 0; u < U; u++) f[u] = fetch(r0 + u);
      for (int64_t c0 = r0; c0 < r1; c0 += 64) {
        const int64_t r = min(c0 + l, r1 - 1);
        const int at = from_lowest(whole(a.pos_q, a.wide, r) - keys.base, a.lo, BOUND), n = (int)min(r1 - c0, (int64_t)64);
        const int64_t group = a.group_q ? whole(a.group_q, a.wide, r) : 0;
        const bool alien = group != (int)group, same = group == keys.first_group;  // alien: no key's group
        const bool low = same && at - keys.least <= 0, high = same && !low && at - keys.most >= a.span - 1;
        uint32_t reached = 0;
        if constexpr (BT > 2) {
#pragma unroll
          for (int t = 0; t < BT; t++) {
            const int k0 = 16 * t, k1 = 16 * t + 16;
            const bool from = k0 <= last && (k0 <= first || at - keys.least >= start[k0]);
            reached |= (uint32_t)(from && k1 > first && (k1 > last || at - keys.most < start[k1])) << t;
          }
        }
        if (!keys.one_group) reached |= 1u << (a.count - 1) / 16;
        const uint64_t firsts = __ballot(low), lasts = __ballot(high), aliens = __ballot(alien);
        const uint64_t ones = keys.one_group ? firsts | lasts | __ballot(!same) : aliens;
        for (int i0 = 0; i0 < n; i0 += U) {
#pragma unroll
          for (int u = 0; u < U; u++) {
            TV v = f[u].get();
            f[u] = fetch(c0 + i0 + u + U);
            const int i = i0 + u;
            if (i >= n) continue;
            if (!whole_tile) {
#pragma unroll
              for (int e = 0; e < GK; e++) v[e] = e >= keys.skip ? v[e] : (T)0.f;
            }
            if (ones >> i & 1) {
              sum_up(v, keys.one_group && firsts >> i & 1 ? FIRST : keys.one_group && lasts >> i & 1 ? LAST : OTHER);
            } else {
              const int row = __builtin_amdgcn_readlane(at, i);
              int d[GK];
#pragma unroll
              for (int e = 0; e < GK; e++) d[e] = row - keys.rel[e];
              if (!keys.one_group) {
                const int g = __builtin_amdgcn_readlane((int)group, i);
#pragma unroll
                for (int e = 0; e < GK; e++) d[e] = keys.group[e] == g ? d[e] : others;
              }
              products(v, d, __builtin_amdgcn_readlane(reached, i));
            }
          }
        }
      }
    };
    if (a.M >= GK && !keys.rare) {
      // Rows of an odd number of 16-bit values begin inside a dword every other time (16 x 4001 x 4001 bf16 158 us, 213 with
      // loads that begin there). The tensor has to begin at one: the value before it is not read.
      if constexpr (sizeof(T) == 2) {
        if (a.M % 2 && (reinterpret_cast<uintptr_t>(dy) & 3) == 0) all_rows(std::true_type());
        else all_rows(std::false_type());
      } else {
        all_rows(std::false_type());
      }
    } else {
      // Fewer than 8 keys, or such as 32 bits do not hold: one row after the other, all buckets.
#pragma unroll 1
      for (int64_t i = r0; i < r1; i++) {
        const int64_t pos = scalar(a.pos_q, a.wide, i), group = a.group_q ? scalar(a.group_q, a.wide, i) : 0;
        const T* const p = col + i * a.M;
        TV v = TV{};
        if (a.M >= GK) {
          v = *reinterpret_cast<const TU*>(p);
        } else {
#pragma unroll
          for (int e = 0; e < GK - 1; e++)
            if (e < a.M) v[e] = p[e];
        }
#pragma unroll
        for (int e = 0; e < GK; e++) v[e] = e >= keys.skip ? v[e] : (T)0.f;
        int d[GK];
#pragma unroll
        for (int e = 0; e < GK; e++) {
          const int64_t j = min(keys.j + e, a.M - 1);
          const bool other = a.group_k && whole(a.group_k, a.wide, j) != group;
          d[e] = other ? others : from_lowest(pos - whole(a.pos_k, a.wide, j), a.lo, BOUND);
        }
        products(v, d, ~0u);
      }
    }
  }
  // The workgroup's sums: a wave at a time, in their order. acc[t][i] is bucket 16 t + 4 (lane / 16) + i of head h0 + c.
#pragma unroll
  for (int k = 0; k < 3; k++) run[k] = xgroups_sum(run[k]);
  for (int w = 0; w < 4; w++) {
    if (w == wave) {
#pragma unroll
      for (int t = 0; t < BT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) meet[c][16 * t + 4 * (l >> 4) + i] += acc[t][i];
      if (l < 16) {
        meet[c][first] += run[FIRST];
        meet[c][last] += run[LAST];
        meet[c][a.count - 1] += run[OTHER];
      }
    }
    __syncthreads();
  }
  float* const to = part + (((b * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x) * a.H + h0) * a.count;
  const int heads = min(16, a.H - h0);
  for (int e = threadIdx.x; e < heads * a.count; e += 256) to[e] = meet[e / a.count][e % a.count];
}

// dtable[k][h] from the partial sums [blocks][H][count], in a fixed order: 16 waves a workgroup each add every 16th, a lane
// a bucket. 768 sums of 16 heads 5 us: latency.
__global__ __launch_bounds__(1024) void rel_bias_sum_k(const float* __restrict__ part, int64_t blocks, int H, int count,
                                                       float* __restrict__ dtable) {
  __shared__ float meet[16][64];
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, h = blockIdx.y, k = min((int)blockIdx.x * 64 + l, count - 1);
  float s = 0.f;
#pragma unroll 8
  for (int64_t p = w; p < blocks; p += 16) s += part[(p * H + h) * count + k];
  meet[w][l] = s;
  __syncthreads();
  if (w || (int)blockIdx.x * 64 + l >= count) return;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i += 4) s += (meet[i][l] + meet[i + 1][l]) + (meet[i + 2][l] + meet[i + 3][l]);
  dtable[(int64_t)k * H + h] = s;
}

// Row blocks of the gradient: about three workgroups a compute unit over key blocks, heads and batch, and at least 8 rows each.
int64_t grad_blocks(int64_t B, int H, int64_t N, int64_t M) {
  const int64_t others = B * ((H + 15) / 16) * ((M + 16 * GK - 1) / (16 * GK)), want = (768 + others - 1) / others, most = (N + 7) / 8;
  return want < most ? want : most;
}

template <typename Fn>
hipError_t with_type(int dt, Fn&& fn) {
  if (dt == DT_F32) return fn(float());
  if (dt == DT_F16) return fn(half_t());
  if (dt == DT_BF16) return fn(bf16_t());
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_rel_bias(const RelBias& a, const void* add, void* out, int dt, int64_t B, hipStream_t st) {
  return with_type(dt, [&](auto t) {
    typedef decltype(t) T;
    constexpr int V = CHUNK<T>;
    const int64_t chunks = (a.M + V - 1) / V;
    const int L = row_lanes(chunks, 256);
    // Heads of a workgroup: all that 32 KB hold, fewer where the grid would leave compute units without one.
    int heads = a.H < 32768 / 4 / a.count ? a.H : 32768 / 4 / a.count;
    const auto blocks = [&](int per) { return (a.N + per - 1) / per; };
    int per = 4 * 256 / L;
    while (per > 256 / L && blocks(per) * B * ((a.H + heads - 1) / heads) < 1024) per /= 2;
    while (heads > 1 && blocks(per) * B * ((a.H + heads - 1) / heads) < 512) heads = (heads + 1) / 2;
    const size_t lds = (size_t)heads * a.count * 4 + (size_t)(a.span + 3) / 4 * 4;
    const dim3 grid((unsigned)blocks(per), (unsigned)((a.H + heads - 1) / heads), (unsigned)B);
    rel_bias_k<T><<<grid, 256, lds, st>>>(a, static_cast<const T*>(add), static_cast<T*>(out), heads, per);
    return hipGetLastError();
  });
}

int64_t rel_bias_bwd_ws_bytes(int64_t B, int H, int64_t N, int64_t M, int count) {
  return B * grad_blocks(B, H, N, M) * ((M + 16 * GK - 1) / (16 * GK)) * H * count * (int64_t)sizeof(float);
}

hipError_t launch_rel_bias_bwd(const RelBias& a, const void* dy, int dt, float* dtable, float* ws, int64_t B,
                               hipStream_t st) {
  const int64_t nb = grad_blocks(B, a.H, a.N, a.M), per = (a.N + nb - 1) / nb, kb = (a.M + 16 * GK - 1) / (16 * GK), bh = B * ((a.H + 15) / 16);
  if (nb > 65535 || bh > 65535) return hipErrorInvalidValue;
  const hipError_t e = with_type(dt, [&](auto t) {
    typedef decltype(t) T;
    const auto go = [&](auto bt) {
      rel_bias_bwd_k<T, decltype(bt)::value><<<dim3((unsigned)kb, (unsigned)nb, (unsigned)bh), 256, 0, st>>>(
          a, static_cast<const T*>(dy), ws, (int)per);
      return hipGetLastError();
    };
    if (a.count <= 32) return go(std::integral_constant<int, 2>());
    if (a.count <= 80) return go(std::integral_constant<int, 5>());
    return go(std::integral_constant<int, 16>());
  });
  if (e != hipSuccess) return e;
  rel_bias_sum_k<<<dim3((unsigned)((a.count + 63) / 64), (unsigned)a.H), 1024, 0, st>>>(ws, B * nb * kb, a.H, a.count, dtable);
  return hipGetLastError();
}

}  // namespace bzpf

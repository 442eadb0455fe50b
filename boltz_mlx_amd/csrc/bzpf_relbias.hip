// A learned relative position bias by buckets, and its table's gradient:
//   bias[b][h][i][j] = table[bucket(pos_q[b][i] - pos_k[b][j])][h] (+ add[b][h][i][j])
//   dtable[k][h] = sum over (b, i, j) whose pair lies in bucket k of dbias[b][h][i][j].
// bucket(d) = lut[clamp(d - lo, 0, span - 1)], not falling with d; pairs of different groups (chains) take the last one.
//
// Both are bound by memory: the bias is written once (the pair bias read once), its gradient read once. A thread owns a
// chunk of 16 bytes of a row. As buckets do not fall with the distance, the two ends of a chunk's positions say whether the
// whole chunk lies in one bucket (most do: those beyond the reach, or in another chain); then one look-up serves it.
#include "bzpf_common.h"
#include "bzpf_kernels.h"
#include "bzpf_rows.h"

namespace bzpf {

namespace {

// A position or group number, 32 or 64 bits wide.
__device__ __forceinline__ int64_t whole(const void* p, bool wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}

// A chunk of V keys: their positions, the ends of these, and the keys' group where they share one.
template <int V>
struct Keys {
  int64_t pos[V], least, most, group;
  bool one_group;
  __device__ __forceinline__ void load(const RelBias& a, int64_t at, int n) {
    one_group = true;
    group = a.group_k ? whole(a.group_k, a.wide, at) : 0;
#pragma unroll
    for (int e = 0; e < V; e++) {
      const int64_t j = at + (e < n ? e : 0);
      pos[e] = whole(a.pos_k, a.wide, j);
      least = e == 0 || pos[e] < least ? pos[e] : least;
      most = e == 0 || pos[e] > most ? pos[e] : most;
      if (a.group_k) one_group &= whole(a.group_k, a.wide, j) == group;
    }
  }
};

__device__ __forceinline__ int bucket_of(const RelBias& a, const uint8_t* lut, int64_t d) {
  d -= a.lo;
  return lut[d < 0 ? 0 : d >= a.span ? a.span - 1 : (int)d];
}

// The buckets of a query at `pos` of `group` against the chunk: in at[], or in at[0] alone where they are one (returned).
template <int V>
__device__ __forceinline__ bool buckets(const RelBias& a, const uint8_t* lut, const Keys<V>& k, int64_t pos, int64_t group,
                                        int64_t key0, int n, int (&at)[V]) {
  if (k.one_group) {
    at[0] = bucket_of(a, lut, pos - k.most);
    const bool one = at[0] == bucket_of(a, lut, pos - k.least);
    if (a.group_q && group != k.group) {
      at[0] = a.count - 1;
      return true;
    }
    if (one) return true;
  }
#pragma unroll
  for (int e = 0; e < V; e++) {
    at[e] = bucket_of(a, lut, pos - k.pos[e]);
    if (!k.one_group && whole(a.group_k, a.wide, key0 + (e < n ? e : 0)) != group) at[e] = a.count - 1;
  }
  return false;
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

// grid (row blocks, head groups of `heads`, batch); LDS: the group's part of the table, then the look-up table.
template <typename T>
__global__ __launch_bounds__(256) void rel_bias_k(RelBias a, const T* __restrict__ add, T* __restrict__ out, int heads,
                                                  int rows_per) {
  constexpr int V = CHUNK<T>;
  extern __shared__ float tab[];
  const int h0 = blockIdx.y * heads, nh = min(heads, a.H - h0), t = threadIdx.x;
  uint8_t* const lut = reinterpret_cast<uint8_t*>(tab + heads * a.count);
  for (int e = t; e < nh * a.count; e += 256) tab[e] = a.table[(int64_t)(e % a.count) * a.H + h0 + e / a.count];
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
    for (int64_t i = (int64_t)blockIdx.x * rows_per + t / L; i < r1; i += 256 / L) {
      int at[V];
      const bool one = buckets(a, lut, keys, whole(a.pos_q, a.wide, i), a.group_q ? whole(a.group_q, a.wide, i) : 0, j0, n, at);
      const int64_t plane = a.N * a.M, base = ((b * a.H + h0) * a.N + i) * a.M + j0;
      if (n < V) {
        for (int h = 0; h < nh; h++)
#pragma unroll
          for (int e = 0; e < V - 1; e++)
            if (e < n) {
              const float v = tab[h * a.count + (one ? at[0] : at[e])];
              out[base + h * plane + e] = (T)(add ? v + (float)add[base + h * plane + e] : v);
            }
        continue;
      }
      if (!one) {
        for (int h = 0; h < nh; h++) {
          fv<V> v;
#pragma unroll
          for (int e = 0; e < V; e++) v[e] = tab[h * a.count + at[e]];
          if (add) v += load_chunk<V>(add + base + h * plane);
          store_chunk<V, false>(out + base + h * plane, v);
        }
      } else {
        for (int h = 0; h < nh; h++) {
          fv<V> v = fv<V>{} + tab[h * a.count + at[0]];
          if (add) v += load_chunk<V>(add + base + h * plane);
          store_chunk<V, false>(out + base + h * plane, v);
        }
      }
    }
  }
}

constexpr int GT = 128;  // threads of a gradient workgroup, each with a column of sums of its own in LDS

// A thread adds its elements into its own column [bucket][thread] of LDS (ds_add_f32 without contention, so that the order
// of a column's additions is the program's: equal inputs give equal bits), and keeps the sum of the bucket it is in a
// register while successive chunks stay in one. grid (row blocks, heads, batch).
template <typename T>
__global__ __launch_bounds__(GT) void rel_bias_bwd_k(RelBias a, const T* __restrict__ dy, float* __restrict__ part,
                                                     int64_t step, int rows_per) {
  constexpr int V = CHUNK<T>, U = 4;
  extern __shared__ float sums[];
  const int t = threadIdx.x;
  uint8_t* const lut = reinterpret_cast<uint8_t*>(sums + a.count * GT);
  for (int k = 0; k < a.count; k++) sums[k * GT + t] = 0.f;
  for (int e = t; e < a.span; e += GT) lut[e] = a.lut[e];
  __syncthreads();
  const int64_t b = blockIdx.z;
  const int h = blockIdx.y;
  a = of_batch(a, b);
  const int64_t chunks = (a.M + V - 1) / V, r1 = min(a.N, ((int64_t)blockIdx.x + 1) * rows_per);
  const int L = row_lanes(chunks, GT), n = a.M < V ? (int)a.M : V;
  float* const mine = sums + t;
  float run = 0.f;
  int cur = 0;
  for (int64_t c = t % L; c < chunks; c += L) {
    const int64_t j0 = min(c * V, a.M - n);
    const int skip = (int)(c * V - j0);  // elements that the neighbour has
    Keys<V> keys;
    keys.load(a, j0, n);
    const T* const col = dy + ((b * a.H + h) * a.N) * a.M + j0;
    const int stride = GT / L;
    for (int64_t i = (int64_t)blockIdx.x * rows_per + t / L; i < r1; i += (int64_t)U * stride) {
      Raw<T, V> raw[U];
      int64_t pos[U], group[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int64_t r = min(i + (int64_t)u * stride, r1 - 1);
        if (n == V) raw[u].load(col + r * a.M);
        else
#pragma unroll
          for (int e = 0; e < V; e++) raw[u].v[e] = e < n ? col[r * a.M + e] : (T)0.f;
        pos[u] = whole(a.pos_q, a.wide, r);
        group[u] = a.group_q ? whole(a.group_q, a.wide, r) : 0;
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (i + (int64_t)u * stride >= r1) break;
        fv<V> v = raw[u].get();
#pragma unroll
        for (int e = 0; e < V; e++) v[e] = e >= skip ? v[e] : 0.f;
        int at[V];
        if (buckets(a, lut, keys, pos[u], group[u], j0, n, at)) {
          if (at[0] != cur) {
            atomicAdd(mine + cur * GT, run);
            run = 0.f;
            cur = at[0];
          }
          run += sum_of(v);
        } else {
#pragma unroll
          for (int e = 0; e < V; e++)
            if (e >= skip && e < n) atomicAdd(mine + at[e] * GT, v[e]);
        }
      }
    }
  }
  atomicAdd(mine + cur * GT, run);
  __syncthreads();
  float* const to = part + ((b * gridDim.x + blockIdx.x) * a.H + h) * step;
  for (int k = t >> 6; k < a.count; k += GT / 64) {
    const float s = row_sum<64>(sums[k * GT + (t & 63)] + sums[k * GT + 64 + (t & 63)], nullptr);
    if ((t & 63) == 0) to[k] = s;
  }
}

// dtable[k][h] from the partial sums [blocks][H][count], in a fixed order: 16 waves a workgroup each add every 16th, a lane
// a bucket.
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

// Row blocks of a (batch element, head)'s gradient: about eight workgroups a compute unit over all of them, and at least
// four chunks for each thread.
int64_t grad_blocks(int64_t B, int H, int64_t N, int64_t M) {
  const int64_t want = (2048 + B * H - 1) / (B * H), most = (N * ((M + 7) / 8) + 4 * GT - 1) / (4 * GT);
  int64_t n = want < most ? want : most;
  if (n > N) n = N;
  return n < 1 ? 1 : n;
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
  return B * grad_blocks(B, H, N, M) * H * count * (int64_t)sizeof(float);
}

hipError_t launch_rel_bias_bwd(const RelBias& a, const void* dy, int dt, float* dtable, float* ws, int64_t B,
                               hipStream_t st) {
  const int64_t nb = grad_blocks(B, a.H, a.N, a.M), per = (a.N + nb - 1) / nb;
  const hipError_t e = with_type(dt, [&](auto t) {
    typedef decltype(t) T;
    const size_t lds = (size_t)a.count * GT * 4 + (size_t)(a.span + 3) / 4 * 4;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&rel_bias_bwd_k<T>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != hipSuccess) return e;
    rel_bias_bwd_k<T><<<dim3((unsigned)nb, (unsigned)a.H, (unsigned)B), GT, lds, st>>>(a, static_cast<const T*>(dy), ws,
                                                                                    a.count, (int)per);
    return hipGetLastError();
  });
  if (e != hipSuccess) return e;
  rel_bias_sum_k<<<dim3((unsigned)((a.count + 63) / 64), (unsigned)a.H), 1024, 0, st>>>(ws, B * nb, a.H, a.count, dtable);
  return hipGetLastError();
}

}  // namespace bzpf

// Norms of queries and keys for each head with the position rotation in the same pass, and their backward pass:
//   xh = x / sqrt(mean(x^2) + eps),  y = R(pos) (w xh)            over the C channels of each head
//   g = R(-pos) dy,  dw = sum over rows and heads of g xh,  dx = (w g - xh mean(w g xh)) / sqrt(mean(x^2) + eps).
// R turns the pair p of the first `rot` channels by pos base^(-2p/rot); pairs are (p, p + rot/2), or (2p, 2p + 1) where
// interleaved. The channels past `rot` pass by, as pairs without an angle.
//
// Bound by memory: one read of q and k (and of their outputs' gradients), one write. A head lies in the registers of L
// lanes, V pairs each, so that a pair never crosses lanes. A token's angles are formed once by a lane for all of the heads
// that it works on: turns = pos base^(-2p/rot) / 2 pi in 64 bits, whole turns dropped there, so that positions of millions
// keep their angles to 2^-24 of a turn.
#include "bzpf_rowgrad.h"

namespace bzpf {

namespace {

// V elements of T (one where V is 1).
template <typename T, int V>
__device__ __forceinline__ void get(const T* p, float (&e)[2 * V], int at) {
  typedef T U __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  if constexpr (V == 1) {
    e[at] = (float)*p;
  } else {
    const U u = *reinterpret_cast<const U*>(p);
#pragma unroll
    for (int i = 0; i < V; i++) e[at + i] = (float)u[i];
  }
}
template <typename T, int V>
__device__ __forceinline__ void put(T* p, const float (&e)[2 * V], int at) {
  typedef T U __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  if constexpr (V == 1) {
    *p = (T)e[at];
  } else {
    U u;
#pragma unroll
    for (int i = 0; i < V; i++) u[i] = (T)e[at + i];
    *reinterpret_cast<U*>(p) = u;
  }
}

// The sum over L (a power of two) neighbouring lanes, in each of them.
__device__ __forceinline__ float lanes_sum(float v, int L) {
  if (L >= 2) v = dpp_add<0xB1>(v);
  if (L >= 4) v = dpp_add<0x4E>(v);
  if (L >= 8) v = dpp_add<0x141>(v);
  if (L >= 16) v = dpp_add<0x140>(v);
  if (L >= 32) v += __shfl_xor(v, 16);
  if (L >= 64) v += __shfl_xor(v, 32);
  return v;
}

// A lane's chunks of V pairs, K of them: where their first and second V elements lie in a head.
template <int V, int K, bool INTER>
struct Pairs {
  static constexpr int A = INTER ? 2 : 1, B = INTER ? 1 : V;  // pair i is elements A i and A i + B of a chunk
  int first[K], second[K], pair[K];
  bool mine[K];
  __device__ __forceinline__ Pairs(int li, int L, const QKNorm& a) {
    const int half = a.rot / 2, tail = (a.C - a.rot) / 2;
#pragma unroll
    for (int k = 0; k < K; k++) {
      const int p = (li + L * k) * V;
      mine[k] = p < a.C / 2;
      pair[k] = p;
      const int c = mine[k] ? p : 0;
      if constexpr (INTER) {
        first[k] = 2 * c;
        second[k] = 2 * c + V;
      } else {
        first[k] = c < half ? c : a.rot + c - half;
        second[k] = first[k] + (c < half ? half : tail);
      }
    }
  }
};

// 1 / sqrt(v); v_rsq_f32 (1 ulp) takes a denormal for 0.
__device__ __forceinline__ float rsqrt_of(float v) {
  const bool tiny = v < 0x1p-100f;
  return __builtin_amdgcn_rsqf(tiny ? v * 0x1p100f : v) * (tiny ? 0x1p50f : 1.f);
}

// grid.y = 2: a workgroup takes the queries or the keys alone (few rows). Waves: lanes are (token, head, part of a head),
// tokens' heads in turns of `hp`, split over `sub` waves where tokens are few. Backward pass of 32,008 tokens of 16 + 4 heads of
// 128 bf16 120 us (4.1 TB/s; with the next turn's values on their way the same); 400 tokens of 16 + 16 heads of 24 fp32 5.2 us
// forward, 10 us backward, one token 4.0 us: latency.
template <bool BWD, typename TX, typename TY, int V, int K, bool INTER>
__global__ __launch_bounds__(256) void qk_norm_k(QKNorm a) {
  typedef Pairs<V, K, INTER> PR;
  constexpr int A = PR::A, B = PR::B;
  const int l = threadIdx.x & 63, L = a.L, hp = a.hp, tp = 64 / (L * hp);
  const int li = l % L, hs = l / L % hp, ts = l / (L * hp);
  const PR pr(li, L, a);
  double freq[K * V];
#pragma unroll
  for (int k = 0; k < K; k++)
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int p = pr.pair[k] + i;
      freq[k * V + i] = a.pos && 2 * p < a.rot ? exp2(a.log2_base * (-2.0 * p / a.rot)) * 0.15915494309189535 : 0.0;
    }
  const float inv = 1.0f / a.C;
  float sw[2][K][2 * V], w[2][K][2 * V];
#pragma unroll
  for (int s = 0; s < 2; s++)
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
      for (int e = 0; e < 2 * V; e++) {
        sw[s][k][e] = 0.f;
        w[s][k][e] = a.w[s] ? a.w[s][e < V ? pr.first[k] + e : pr.second[k] + e - V] : 1.f;
      }
  const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), waves = (int64_t)gridDim.x * 4;
  const int sub = (int)(wave % a.sub);
  for (int64_t r = wave / a.sub * tp + ts; r < a.rows; r += waves / a.sub * tp) {
    float cs[K * V], sn[K * V];
#pragma unroll
    for (int k = 0; k < K * V; k++) cs[k] = 1.f, sn[k] = 0.f;
    if (a.pos) {
      const int64_t at = r < a.pos_rows ? r : a.rows <= UINT32_MAX ? (uint32_t)r % (uint32_t)a.pos_rows : r % a.pos_rows;
      const double pos = a.wide ? (double)static_cast<const int64_t*>(a.pos)[at] : (double)static_cast<const int32_t*>(a.pos)[at];
#pragma unroll
      for (int k = 0; k < K * V; k++) {
        const double t = pos * freq[k];
        sincospif((float)(2.0 * (t - rint(t))), &sn[k], &cs[k]);
      }
    }
#pragma unroll
    for (int s = 0; s < 2; s++) {
      if (gridDim.y == 2 && (int)blockIdx.y != s) continue;
      const int H = a.H[s];
      const TX* const x = static_cast<const TX*>(a.x[s]) + r * a.ld[s];
      for (int h0 = sub * hp; h0 < H; h0 += a.sub * hp) {
        const int h = h0 + hs;
        const bool on = h < H;
        const int64_t at = (int64_t)(on ? h : 0) * a.C;
        float e[K][2 * V], g[K][2 * V], ss = 0.f;
#pragma unroll
        for (int k = 0; k < K; k++) {
          get<TX, V>(x + at + pr.first[k], e[k], 0);
          get<TX, V>(x + at + pr.second[k], e[k], V);
          if constexpr (BWD) {
            const TY* const dy = static_cast<const TY*>(a.y[s]) + r * H * a.C + at;
            get<TY, V>(dy + pr.first[k], g[k], 0);
            get<TY, V>(dy + pr.second[k], g[k], V);
          }
        }
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
          for (int i = 0; i < 2 * V; i++) ss += pr.mine[k] ? e[k][i] * e[k][i] : 0.f;
        const float rs = rsqrt_of(lanes_sum(ss, L) * inv + a.eps);
        if constexpr (!BWD) {
          TY* const y = static_cast<TY*>(a.y[s]) + r * H * a.C + at;
#pragma unroll
          for (int k = 0; k < K; k++) {
#pragma unroll
            for (int i = 0; i < V; i++) {
              const float u = e[k][A * i] * rs * w[s][k][A * i], v = e[k][A * i + B] * rs * w[s][k][A * i + B];
              e[k][A * i] = u * cs[k * V + i] - v * sn[k * V + i];
              e[k][A * i + B] = u * sn[k * V + i] + v * cs[k * V + i];
            }
            if (on && pr.mine[k]) {
              put<TY, V>(y + pr.first[k], e[k], 0);
              put<TY, V>(y + pr.second[k], e[k], V);
            }
          }
        } else {
          float m = 0.f;
#pragma unroll
          for (int k = 0; k < K; k++)
#pragma unroll
            for (int i = 0; i < V; i++) {
              const float u = g[k][A * i], v = g[k][A * i + B];
              g[k][A * i] = u * cs[k * V + i] + v * sn[k * V + i];
              g[k][A * i + B] = v * cs[k * V + i] - u * sn[k * V + i];
#pragma unroll
              for (int j = A * i; j <= A * i + B; j += B) {
                e[k][j] *= rs;
                if (on && pr.mine[k]) sw[s][k][j] += g[k][j] * e[k][j];
                g[k][j] *= w[s][k][j];
                m += pr.mine[k] ? g[k][j] * e[k][j] : 0.f;
              }
            }
          m = lanes_sum(m, L) * inv;
          TX* const dx = static_cast<TX*>(a.dx[s]) + r * H * a.C + at;
#pragma unroll
          for (int k = 0; k < K; k++) {
#pragma unroll
            for (int i = 0; i < 2 * V; i++) g[k][i] = (g[k][i] - e[k][i] * m) * rs;
            if (on && pr.mine[k]) {
              put<TX, V>(dx + pr.first[k], g[k], 0);
              put<TX, V>(dx + pr.second[k], g[k], V);
            }
          }
        }
      }
    }
  }
  if constexpr (BWD) {
    if (!a.ws) return;
    // The workgroup's sums: the lanes that hold the same channels, then its four waves; [workgroups][2][C] in all.
    __shared__ float meet[4][2][QK_MAX_C];
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
      for (int k = 0; k < K; k++)
#pragma unroll
        for (int i = 0; i < 2 * V; i++) {
          float v = sw[s][k][i];
          for (int o = L; o < 64; o *= 2) v += __shfl_xor(v, o);
          if (l < L && pr.mine[k]) meet[threadIdx.x >> 6][s][i < V ? pr.first[k] + i : pr.second[k] + i - V] = v;
        }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * a.C; c += 256) {
      const int s = c / a.C, j = c % a.C;
      if (gridDim.y == 2 && (int)blockIdx.y != s) continue;
      a.ws[(int64_t)blockIdx.x * 2 * a.C + c] = (meet[0][s][j] + meet[1][s][j]) + (meet[2][s][j] + meet[3][s][j]);
    }
  }
}

int pow2_from(int n) {
  int p = 1;
  while (p < n) p *= 2;
  return p;
}

// Pairs of a chunk: as many as 16 bytes of the widest type hold (`most`), fewer where the head's two parts are no multiples.
int pairs_of(int C, int rot, int most) {
  int v = most;
  while (rot / 2 % v || (C - rot) / 2 % v) v /= 2;
  return v;
}

int64_t blocks_of(int64_t rows, int C, int rot, int Hq, int Hk, int most, bool bwd, QKNorm* a, unsigned* y) {
  const int v = pairs_of(C, rot, most), L = pow2_from((C / 2 + v - 1) / v);
  a->L = L < 64 ? L : 64;
  const int H = Hq > Hk ? Hq : Hk, hp = pow2_from(H);
  a->hp = hp < 64 / a->L ? hp : 64 / a->L;
  const int tp = 64 / (a->L * a->hp), turns = (H + a->hp - 1) / a->hp;
  const int64_t waves = (rows + tp - 1) / tp;
  // Few rows: queries and keys, and the turns over a token's heads, are work of different waves.
  *y = waves < 2048 ? 2 : 1;
  a->sub = 1;
  while (a->sub < turns && waves * a->sub < 2048) a->sub *= 2;
  const int64_t n = (waves * a->sub + 3) / 4, cap = bwd ? ROW_GRAD_BLOCKS : 1 << 16;
  // `sub` divides the waves of the grid
  int64_t blocks = n < cap ? n : cap;
  if (a->sub > 4) blocks = (blocks + a->sub / 4 - 1) / (a->sub / 4) * (a->sub / 4);
  return blocks;
}

template <bool BWD, typename TX, typename TY>
hipError_t launch(QKNorm a, float* dwq, float* dwk, hipStream_t st) {
  constexpr int most = sizeof(TX) == 4 || sizeof(TY) == 4 ? 4 : 8;
  unsigned y;
  const int64_t blocks = blocks_of(a.rows, a.C, a.rot, a.H[0], a.H[1], most, BWD, &a, &y);
  const dim3 grid((unsigned)blocks, y);
  const int v = pairs_of(a.C, a.rot, most);
#define BZ_QK(VV, KK)                                                                   \
  if (a.inter)                                                                          \
    qk_norm_k<BWD, TX, TY, VV, KK, true><<<grid, 256, 0, st>>>(a);                      \
  else                                                                                  \
    qk_norm_k<BWD, TX, TY, VV, KK, false><<<grid, 256, 0, st>>>(a)
  if (v == 8) {
    if constexpr (most == 8) {
      BZ_QK(8, 1);
    }
  } else if (v == 4) {
    BZ_QK(4, 1);
  } else if (v == 2) {
    BZ_QK(2, 1);
  } else if (a.C <= 128) {
    BZ_QK(1, 1);
  } else {
    BZ_QK(1, 2);
  }
#undef BZ_QK
  const hipError_t e = hipGetLastError();
  if (!BWD || e != hipSuccess || !a.ws) return e;
  return launch_row_grad_sum(a.ws, blocks, a.C, dwq, dwk, st);
}

template <bool BWD>
hipError_t with(const QKNorm& a, int x_dt, int y_dt, float* dwq, float* dwk, hipStream_t st) {
  return with_types(x_dt, y_dt, [&](auto tx, auto ty) {
    typedef std::remove_cv_t<std::remove_pointer_t<decltype(tx)>> TX;
    typedef std::remove_cv_t<std::remove_pointer_t<decltype(ty)>> TY;
    return launch<BWD, TX, TY>(a, dwq, dwk, st);
  });
}

}  // namespace

hipError_t launch_qk_norm(const QKNorm& a, int x_dt, int y_dt, hipStream_t st) {
  return with<false>(a, x_dt, y_dt, nullptr, nullptr, st);
}

int64_t qk_norm_ws_bytes(int C) { return (int64_t)ROW_GRAD_BLOCKS * 2 * C * (int64_t)sizeof(float); }

hipError_t launch_qk_norm_bwd(const QKNorm& a, int x_dt, int dy_dt, float* dwq, float* dwk, hipStream_t st) {
  return with<true>(a, x_dt, dy_dt, dwq, dwk, st);
}

}  // namespace bzpf

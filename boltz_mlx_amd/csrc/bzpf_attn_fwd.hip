// The sequence attention's forward pass with the statistics that its backward pass needs (bzpf_attn.h has the formulas).
// One pass over the keys with the running maximum and sum of each row's softmax; a wave holds 32 queries as the columns of
// S^T = K Q^T, so that a row's statistics are a lane's own (and its other half's). Logits stay in natural units until their
// maximum is subtracted. 4096 x 4096, 16 heads of 64 channels bf16 with a bias 163 us (420 TFLOP/s, 3.5 TB/s), bound by
// issue: vector instructions take 1,372 cycles of a wave's 64 keys, products 512, two waves to a SIMD. 5 x 16 x 400 x 400 in 48
// channels fp16 22 us, 16 x 400 x 400 in 24 channels fp32 14 us: latency of each block's chain.
#include "bzpf_attn.h"

namespace bzpf {

namespace {

template <typename T, typename BT, int KS, bool SPLIT>
__global__ __launch_bounds__(256, sizeof(T) == 2 && KS <= 4 ? 2 : 1) void attn_fwd_k(Attn a, int64_t per_xcd) {
  typedef Form<T, SPLIT> F;
  constexpr int BK = F::BR, KT = BK / 32, NT = (KS + 1) / 2, TILE = BK * TILE_LD<T, KS>;
  constexpr int TILES = F::GROUPS * F::BUFS * 2 * TILE * (int)sizeof(T), MEET = SPLIT ? 4 * NT * 4096 + 4 * 64 * 8 : 0;
  __shared__ LDS_ALIGN char lds[TILES > MEET ? TILES : MEET];
  __shared__ LDS_ALIGN char bias_lds[4 * BiasRows<BT, BK>::BYTES];
  const int64_t qblocks = (a.N + F::ROWS - 1) / F::ROWS;
  Unit un;
  if (!unit_of(a, qblocks, per_xcd, &un)) return;  // whole workgroup
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63, hl = l >> 5;
  const int t = SPLIT ? l : threadIdx.x, group = SPLIT ? wave : 0;
  T* const Kt = reinterpret_cast<T*>(lds) + group * F::BUFS * 2 * TILE;
  T* const Vt = Kt + F::BUFS * TILE;
  const int64_t j0 = un.block * F::ROWS, j = j0 + (SPLIT ? 0 : 32 * wave) + (l & 31), jc = min(j, a.N - 1);
  const int hc = un.h * a.C;
  const T* const q = static_cast<const T*>(a.q) + un.smp * a.sq + jc * a.ldq + hc;
  const T* const k = static_cast<const T*>(a.k) + un.smp * a.sk + hc;
  const T* const v = static_cast<const T*>(a.v) + un.smp * a.sv + hc;
  const int64_t b0 = min(j0 + (SPLIT ? 0 : 32 * wave), a.N - 1);  // the wave's first row
  const BT* const bias = a.bias ? static_cast<const BT*>(a.bias) + (((int64_t)(un.smp / a.mult) * a.H + un.h) * a.N + b0) * a.M : nullptr;
  const int brows = (int)min(a.N - b0, (int64_t)32);
  u4* const Bt = reinterpret_cast<u4*>(bias_lds + wave * BiasRows<BT, BK>::BYTES);
  const float* mask = a.mask ? a.mask + un.smp * a.M : nullptr;

  frag<T> qf[KS];
#pragma unroll
  for (int m = 0; m < KS; m++) qf[m] = 16 * m + 8 * hl < a.C ? load8(q + 16 * m + 8 * hl) : frag<T>{};
  f16x o[NT];
#pragma unroll
  for (int tt = 0; tt < NT; tt++) o[tt] = f16x{};
  float top = -INFINITY, sum = 0.f;
  Exponent ex(top);

  Stage<T, KS, BK, F::NTH, true> ks, vs;
  BiasRows<BT, BK> bs;
  float mk = 1.f;
  const auto fetch = [&](int64_t k0) {
    ks.load(k + k0 * a.ldk, (uint32_t)a.ldk, a.M - k0, a.C, t);
    vs.load(v + k0 * a.ldv, (uint32_t)a.ldv, a.M - k0, a.C, t);
    if (mask) mk = mask[min(k0 + l, a.M - 1)];
  };
  const auto fetch_bias = [&](int64_t k0) {
    if (bias) bs.load(bias, brows, (int)a.M, (int)k0);
  };
  constexpr int STEP = F::GROUPS * BK;
  int64_t k0 = group * BK;
  if (k0 < a.M) {
    fetch(k0);
    fetch_bias(k0);
  }
  const bool masked = mask && any_key(mask, a.M);  // the first loads are on their way
  for (int buf = 0; k0 < a.M; k0 += STEP, buf = (buf + 1) % F::BUFS) {
    const uint64_t keep = __ballot(k0 + l < a.M && l < BK && (!masked || mk != 0.f));
    T* const Kb = Kt + buf * TILE;
    T* const Vb = Vt + buf * TILE;
    ks.store(Kb, keep, a.C, t);
    vs.store(Vb, keep, a.C, t);
    if (bias) bs.store(Bt, (int)a.M, (int)k0);
    F::sync();
    const bool more = k0 + STEP < a.M;
    if (more) {
      fetch(k0 + STEP);
      fetch_bias(k0 + STEP);
    }
    f16x x[KT];
    float most = top;
#pragma unroll
    for (int kt = 0; kt < KT; kt++) {
      f16x s = f16x{};
#pragma unroll
      for (int m = 0; m < KS; m++) s = mma(row_frag<T, KS>(Kb, 32 * kt + (l & 31), m), qf[m], s);
      f16x b = f16x{};
      if (bias) b = BiasRows<BT, BK>::get(Bt, kt);
#pragma unroll
      for (int i = 0; i < 16; i++) s[i] = fmaf(s[i], a.scale, b[i]);
      if (keep != all_rows(BK)) {
        const uint32_t w = (uint32_t)(keep >> (32 * kt)) >> (16 * hl);
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = w >> i & 1 ? s[i] : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 16; i += 2) most = fmaxf(fmaxf(most, s[i]), s[i + 1]);
      x[kt] = s;
    }
    most = both_max(most);
    // Without a branch: around the accumulators the compiler copies them all (4096 x 4096, 16 heads of 64 channels bf16 163 us
    // so, 186 us with one; a base that follows the maximum only where that is e^4 past it gains nothing).
    const Exponent now(most);
    const float by = now.since(ex);
#pragma unroll
    for (int tt = 0; tt < NT; tt++) o[tt] *= by;
    sum *= by;
    top = most;
    ex = now;
    const bool some_big = __any(ex.big());
#pragma unroll
    for (int kt = 0; kt < KT; kt++) {
      exponentials(x[kt], ex, some_big);
#pragma unroll
      for (int i = 0; i < 16; i++) sum += x[kt][i];
#pragma unroll
      for (int s = 0; s < 2; s++) {
        const frag<T> p = as_frag<T>(x[kt], s);
#pragma unroll
        for (int tt = 0; tt < NT; tt++) o[tt] = mma(col_frag<T, KS>(Vb, 32 * kt + 16 * s, tt), p, o[tt]);
      }
    }
    F::again();
    if constexpr (!SPLIT) F::order();  // the biases are the wave's own
  }
  sum = both_sum(sum);
  const T* const g = a.g ? static_cast<const T*>(a.g) + un.smp * a.sg + jc * a.ldg + hc : nullptr;
  T* const out = static_cast<T*>(a.out) + (un.smp * a.N + jc) * a.H * a.C + hc;
  const auto put = [&](int tt, int qq, f4 r, float inv) {
    const int c = 32 * tt + 8 * qq + 4 * hl;
    if (c >= a.C) return;
    r *= inv;
    if (g) {
      const fv<4> gv = load_chunk<4>(g + c);
#pragma unroll
      for (int e = 0; e < 4; e++) r[e] *= sigmoidf_(gv[e]);
    }
    store_chunk<4, false>(out + c, fv<4>{r[0], r[1], r[2], r[3]});
  };
  const auto stats = [&] {  // of the first wave's lanes, a row each
    float* const st = a.stats + (((int64_t)un.smp * a.H + un.h) * a.N + j) * 2;
    st[0] = top;
    st[1] = sum * __builtin_amdgcn_exp2f(-ex.off());
  };
  if constexpr (SPLIT) {
    // the waves' maxima and sums, then their outputs to the common maximum
    float2* const st = reinterpret_cast<float2*>(lds + 4 * NT * 4096);
    __syncthreads();
    st[wave * 64 + l] = float2{top, sum};
    __syncthreads();
    float most = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; w++) most = fmaxf(most, st[w * 64 + l].x);
    const Exponent all(most);
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) total += st[w * 64 + l].y * all.since(Exponent(st[w * 64 + l].x));
    f4 r[NT];
    meet4<NT>(o, reinterpret_cast<f4*>(lds), wave, l, all.since(ex), r);
    top = most, sum = total, ex = all;
    if (j >= a.N) return;
    if (threadIdx.x < 32) stats();
#pragma unroll
    for (int tt = 0; tt < NT; tt++) put(tt, wave, r[tt], sum == 0.f ? 0.f : 1.0f / sum);
  } else {
    if (j >= a.N) return;
    if (hl == 0) stats();
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
    for (int tt = 0; tt < NT; tt++)
#pragma unroll
      for (int qq = 0; qq < 4; qq++) put(tt, qq, f4{o[tt][4 * qq], o[tt][4 * qq + 1], o[tt][4 * qq + 2], o[tt][4 * qq + 3]}, inv);
  }
}

// Few queries (a token against a long axis): no matrix product fills its rows, and what counts is latency. L lanes a key, 8
// channels each, so that loads are whole rows; every group of lanes has a running maximum, sum and output of its own over
// its keys, which meet at the end, in the wave by lane swaps, then in LDS. A long axis is split over workgroups whose parts
// another kernel joins. One row of 400 keys in 24 channels, 16 heads, fp32: 6.4 us (11.7 us in 32 x 32 tiles).
constexpr int FEW_KEYS = 4;  // keys of a group of lanes on their way at once

template <int L>
struct Part {
  float top, sum, acc[8];
  __device__ __forceinline__ void clear() {
    top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) acc[e] = 0.f;
  }
  __device__ __forceinline__ void join(const Part& o) {
    const Exponent old(top), other(o.top), now(fmaxf(top, o.top));
    const float x = now.since(old), y = now.since(other);
    top = fmaxf(top, o.top);
    sum = sum * x + o.sum * y;
#pragma unroll
    for (int e = 0; e < 8; e++) acc[e] = acc[e] * x + o.acc[e] * y;
  }
  // The groups of a wave: in lanes 0 .. L - 1.
  __device__ __forceinline__ void join_wave() {
#pragma unroll
    for (int s = L; s < 64; s *= 2) {
      Part o;
      o.top = __shfl_xor(top, s), o.sum = __shfl_xor(sum, s);
#pragma unroll
      for (int e = 0; e < 8; e++) o.acc[e] = __shfl_xor(acc[e], s);
      join(o);
    }
  }
  // The groups of the workgroup: true in lanes 0 .. L - 1 of its first wave, which have the result.
  __device__ __forceinline__ bool join_all(Part (&meet)[4][L]) {
    const int l = threadIdx.x % L;
    join_wave();
    if ((threadIdx.x & 63) < L) meet[threadIdx.x >> 6][l] = *this;
    __syncthreads();
    if (threadIdx.x >= L) return false;
    *this = meet[0][l];
#pragma unroll
    for (int w = 1; w < 4; w++) join(meet[w][l]);
    return true;
  }
  // The row's output and statistics, by L lanes.
  template <typename T>
  __device__ __forceinline__ void finish(const Attn& a, int64_t row, int l) const {
    const int64_t n = row % a.N, sh = row / a.N, smp = sh / a.H, h = sh % a.H;
    const Exponent ex(top);
    if (l == 0) {
      a.stats[2 * row] = top;
      a.stats[2 * row + 1] = sum * __builtin_amdgcn_exp2f(-ex.off());
    }
    const int c = 8 * l;
    if (c >= a.C) return;
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; e++) y[e] = acc[e] * inv;
    if (a.g) {
      const frag<T> g = load8(static_cast<const T*>(a.g) + smp * a.sg + n * a.ldg + h * a.C + c);
#pragma unroll
      for (int e = 0; e < 8; e++) y[e] *= sigmoidf_((float)g[e]);
    }
    T* const out = static_cast<T*>(a.out) + ((smp * a.N + n) * a.H + h) * a.C + c;
#pragma unroll
    for (int e = 0; e < 8; e += 4) store_chunk<4, false>(out + e, fv<4>{y[e], y[e + 1], y[e + 2], y[e + 3]});
  }
};

// Workgroup: a row ([S][H][N]) and `per` keys. parts (or null: all the row's keys are here): [row][split][L].
template <typename T, typename BT, int L>
__global__ __launch_bounds__(256) void attn_few_k(Attn a, uint32_t splits, int64_t per, Part<L>* parts) {
  constexpr int G = 256 / L, U = FEW_KEYS;
  __shared__ Part<L> meet[4][L];
  const int l = threadIdx.x % L, group = threadIdx.x / L, c = 8 * l < a.C ? 8 * l : 0;
  const int64_t row = blockIdx.x / splits, n = row % a.N, sh = row / a.N, smp = sh / a.H, h = sh % a.H;
  const int64_t first = blockIdx.x % splits * per, end = min(first + per, a.M);
  const T* const k = static_cast<const T*>(a.k) + smp * a.sk + h * a.C + c;
  const T* const v = static_cast<const T*>(a.v) + smp * a.sv + h * a.C + c;
  const BT* const bias = a.bias ? static_cast<const BT*>(a.bias) + ((smp / a.mult * a.H + h) * a.N + n) * a.M : nullptr;
  const float* const mask = a.mask ? a.mask + smp * a.M : nullptr;
  const frag<T> raw = load8(static_cast<const T*>(a.q) + smp * a.sq + n * a.ldq + h * a.C + c);
  struct Keys {
    frag<T> k[U], v[U];
    BT b[U];
    float mk[U];
  };
  const auto fetch = [&](int64_t k0) {
    Keys f;
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int64_t at = min(k0 + group + G * u, end - 1);
      f.k[u] = load8(k + at * a.ldk);
      f.v[u] = load8(v + at * a.ldv);
      f.b[u] = bias ? bias[at] : (BT)0.f;
      f.mk[u] = mask ? mask[at] : 1.f;
    }
    return f;
  };
  Keys f = fetch(first);
  const bool masked = mask && any_key(mask, a.M);  // the first keys are on their way
  float q[8];
#pragma unroll
  for (int e = 0; e < 8; e++) q[e] = 8 * l < a.C ? (float)raw[e] : 0.f;
  Part<L> p;
  p.clear();
  Exponent ex(p.top);
  for (int64_t k0 = first; k0 < end; k0 += G * U) {
    const Keys now = f;
    f = fetch(k0 + G * U);
    float x[U], most = p.top;
    bool on[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; e++) s = fmaf(q[e], (float)now.k[u][e], s);
      s = row_sum<L>(s, nullptr);
      on[u] = k0 + group + G * u < end && (!masked || now.mk[u] != 0.f);
      x[u] = on[u] ? fmaf(s, a.scale, (float)now.b[u]) : -INFINITY;
      most = fmaxf(most, x[u]);
    }
    const Exponent to(most);
    const float by = to.since(ex);
    p.sum *= by;
#pragma unroll
    for (int e = 0; e < 8; e++) p.acc[e] *= by;
#pragma unroll
    for (int u = 0; u < U; u++) {
      const float w = to.of(x[u]);
      p.sum += w;
#pragma unroll
      for (int e = 0; e < 8; e++) p.acc[e] = fmaf(w, on[u] ? (float)now.v[u][e] : 0.f, p.acc[e]);
    }
    p.top = most;
    ex = to;
  }
  if (!p.join_all(meet)) return;
  if (parts) parts[(int64_t)blockIdx.x * L + l] = p;
  else p.template finish<T>(a, row, l);
}

// A workgroup a row: its groups of lanes each take every (256 / L)th part.
template <typename T, int L>
__global__ __launch_bounds__(256) void attn_join_k(Attn a, uint32_t splits, const Part<L>* parts) {
  __shared__ Part<L> meet[4][L];
  const int l = threadIdx.x % L;
  const int64_t row = blockIdx.x;
  Part<L> p;
  p.clear();
#pragma unroll 4
  for (uint32_t s = threadIdx.x / L; s < splits; s += 256 / L) p.join(parts[(row * splits + s) * L + l]);
  if (p.join_all(meet)) p.template finish<T>(a, row, l);
}

// Lanes of a key: 4, 8 or 16.
int few_lanes(int C) { return C <= 32 ? 4 : C <= 64 ? 8 : 16; }

// Whether a call takes the kernels for few queries: one query a head, or so few rows in all that 32 x 32 tiles, whose
// workgroups then take M / 128 steps of 1.2 to 3 us, wait longer than the rows' share of the keys takes here. 16 heads of 64
// channels, 4096 keys bf16: 1, 4, 8 queries 12, 14, 19 us (38 in tiles); 2 heads, 131072 keys: 1 query 30 us (1069); 16 heads,
// fp32: 1, 4, 8 queries 199, 350, 589 us (3060). 64 x 16 heads, 2000 keys fp16: 1, 2, 4 queries 102, 167, 316 us (151 to 163).
struct Few {
  bool use;
  int64_t rows, per, splits;
  explicit Few(const Attn& a) {
    const int step = 256 / few_lanes(a.C);
    rows = (int64_t)a.S * a.H * a.N;
    use = a.N == 1 || rows <= 192;
    const int64_t want = rows < 1024 ? (1024 + rows - 1) / rows : 1, share = (a.M + want - 1) / want, least = 16 * step;
    const int64_t unit = step * FEW_KEYS;
    per = ((share > least ? share : least) + unit - 1) / unit * unit;
    splits = (a.M + per - 1) / per;
  }
  int64_t bytes(int C) const { return use && splits > 1 ? rows * splits * few_lanes(C) * (int64_t)sizeof(Part<4>) : 0; }
};

}  // namespace

int64_t attention_ws_bytes(const Attn& a) { return Few(a).bytes(a.C); }

hipError_t launch_attention(const Attn& a, void* ws, hipStream_t st) {
  const Few few(a);
  if (few.use) {
    const int64_t wgs = few.rows * few.splits;
    if (wgs > INT32_MAX) return hipErrorInvalidValue;
    return with_attn(a, [&](auto t, auto b, auto ks) {
      typedef decltype(t) T;
      typedef decltype(b) BT;
      constexpr int L = decltype(ks)::value <= 2 ? 4 : decltype(ks)::value <= 4 ? 8 : 16;
      Part<L>* const parts = few.splits > 1 ? static_cast<Part<L>*>(ws) : nullptr;
      attn_few_k<T, BT, L><<<(unsigned)wgs, 256, 0, st>>>(a, (uint32_t)few.splits, few.per, parts);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess || !parts) return e;
      attn_join_k<T, L><<<(unsigned)few.rows, 256, 0, st>>>(a, (uint32_t)few.splits, parts);
      return hipGetLastError();
    });
  }
  return with_attn(a, [&](auto t, auto b, auto ks) {
    typedef decltype(t) T;
    typedef decltype(b) BT;
    constexpr int KS = decltype(ks)::value;
    const auto go = [&](auto split) {
      constexpr bool SPLIT = decltype(split)::value;
      const int64_t per = ((a.N + Form<T, SPLIT>::ROWS - 1) / Form<T, SPLIT>::ROWS * a.S * a.H + 7) / 8;
      if (8 * per > INT32_MAX) return hipErrorInvalidValue;
      attn_fwd_k<T, BT, KS, SPLIT><<<(unsigned)(8 * per), 256, 0, st>>>(a, per);
      return hipGetLastError();
    };
    return with_split<KS>(a.N, a, go);
  });
}

}  // namespace bzpf

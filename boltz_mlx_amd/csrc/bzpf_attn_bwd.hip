// The sequence attention's backward pass (bzpf_attn.h has the forward one). With dO = sigmoid(g) dout and the row sums
// delta = sum over c of dout out (= sum over c of dO (p v)):
//   dg = dout out (1 - sigmoid(g));  dp = dO v^T;  ds = p (dp - delta);
//   dv = p^T dO;  dq = ds k / sqrt(C);  dk = ds^T q / sqrt(C);  dbias = ds, summed over the samples that share a bias.
// Probabilities are formed again from the row's maximum and sum. Four kernels, no atomics (equal inputs give equal bits): the
// row sums; dq, by blocks of queries over all keys; dk and dv, by blocks of keys over all queries (and dbias, where each
// sample has its own); dbias of a shared bias, by tiles of it over its samples.
//
// Half types round p and ds once, as operands of their products. What else they would lose is kept:
// - delta comes from the rounded output. The sum over a row of ds is 0 but for that error, so that dq's kernel, which has the
//   sum in fp32, hands the mended delta on; from dq it takes (sum of the rounded ds) (sum of p k), one more product, which
//   leaves of each rounding what its key differs from the row's mean key by.
// - dO is not a value of the type: it goes as two of them, the rounded one and the rest, in the products of dp and dv.
// Without these the gradients were 1.7 to 2.3 times as far from the exact ones as their own rounding puts them, now 1.0
// (dbias), 1.3 (dq), 1.4 (dk, dv) and 1.5 times (dg, from the output as it was rounded). Where ds is below fp16's 2^-14, dq and
// dk err by about one of the type's smallest steps; where it is past its largest number, Scale. p below 2^-14 (tens of thousands of
// keys) costs dv some sqrt(N) 2^-25 of dO.
#include "bzpf_attn.h"

namespace bzpf {

namespace {

// What the other kernels need of a row (p = Exponent(by, at).of(x) inv), [S][H][N], and with a gate dO (two parts in half
// types) and dg. L lanes a head, 8 channels each. Bound by memory: 2 x 16 x 2000 rows of 64 channels bf16 with a gate 13.6 us (4.1 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void attn_rows_k(Attn a, int L) {
  const int l = threadIdx.x % L, heads = 256 / L;
  const int64_t n = (int64_t)blockIdx.x * heads + threadIdx.x / L, total = (int64_t)a.S * a.N * a.H;
  const int64_t r = min(n, total - 1), row = r / a.H, smp = row / a.N;
  const int h = (int)(r % a.H), c = 8 * l;
  const int64_t at = r * a.C + c;
  const bool on = n < total && c < a.C;
  float d = 0.f;
  if (on) {
    const frag<T> dout = load8(static_cast<const T*>(a.dout) + at), o = load8(static_cast<const T*>(a.out) + at);
    frag<T> gv{}, dg, dO, lo;
    if (a.g) gv = load8(static_cast<const T*>(a.g) + smp * a.sg + (row - smp * a.N) * a.ldg + h * a.C + c);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float y = (float)dout[e] * (float)o[e];
      d += y;
      if (a.g) {
        const float s = sigmoidf_((float)gv[e]);
        const float full = (float)dout[e] * s;
        dO[e] = (T)full;
        lo[e] = (T)(full - (float)dO[e]);
        dg[e] = (T)(y * (1.f - s));
      }
    }
    if (a.g) {
      typedef T U __attribute__((ext_vector_type(8), aligned(sizeof(T))));
      *reinterpret_cast<U*>(static_cast<T*>(a.dO) + at) = dO;
      if constexpr (sizeof(T) == 2) *reinterpret_cast<U*>(static_cast<T*>(a.dO_lo) + at) = lo;
      *reinterpret_cast<U*>(static_cast<T*>(a.dg) + at) = dg;
    }
  }
  for (int o = 1; o < L; o *= 2) d += __shfl_xor(d, o);
  if (on && l == 0) {
    const int64_t to = (smp * a.H + h) * a.N + row - smp * a.N;
    const float top = a.stats[2 * to], sum = a.stats[2 * to + 1];
    const Exponent ex(top);
    static_cast<f4*>(a.rows)[to] = f4{ex.at, sum == 0.f ? 0.f : __builtin_amdgcn_exp2f(-ex.off()) / sum, d, ex.by};
  }
}

// A row as attn_rows_k left it.
struct RowStat {
  Exponent ex;
  float inv, delta;
  __device__ __forceinline__ explicit RowStat(f4 v) { ex.at = v[0], ex.by = v[3], inv = v[1], delta = v[2]; }
  // Exponentials of a row smaller by 2^n, at most the root of the sum and of C; what is then left of its reciprocal; n.
  __device__ __forceinline__ float root(int C) {
    const float n = inv == 0.f ? 0.f : (float)(max((127 - (int)(__float_as_uint(inv) >> 23)) / 2, 0) + (31 - __builtin_clz(C)) / 2);
    const float at = ex.big() ? ex.at : ex.at + n;
    inv *= __builtin_amdgcn_exp2f(ex.big() ? n : at - ex.at);
    ex.at = at;
    return n;
  }
};

// ds on its way into a product, for a lane's key (dk) or row (dq). In fp16 it may pass the type's largest number where the product
// does not: a ds of 10^6 meets a query of 0.01 under 1 / sqrt(C). The accumulators are infinite or NaN then, and the lanes
// that have such go over the other axis again with ds times 2^-12, and so on to 2^-23 (finite operands give |ds| below 2^38). The
// largest scaled ds is 2^4 or more then, so that what others lose below 2^-14 is 2^-29 of it. Operands that are not finite take
// two or three rounds more too (2 x 16 x 2000 x 2000 in 64 channels without a gate 632 us instead of 207). The other types' ds have fp32's
// range. The multiplication and the check cost the backward pass 4% at that size (with a gate and a bias 320 -> 331 us), 11%
// where the registers of the split form were full (16 x 400 x 400, 64 channels with both 30.2 -> 33.7 us).
template <typename T>
struct Scale {
  static constexpr bool ON = std::is_same<T, half_t>::value;
  float by;
  // n terms of a size in C channels: their product is some sqrt(n / C) of them where that is more than they are, and so small ones
  // are lost where the product is.
  __device__ __forceinline__ Scale(int64_t n, int C)
      : by(ON && n > C ? (float)(1 << (31 - __builtin_clz((uint32_t)(n / C))) / 2) : 1.f) {}
  // Accumulator rows 16 s .. 16 s + 15 as the products take them.
  __device__ __forceinline__ frag<T> as_frag(const f16x& c, int s) const {
    if constexpr (!ON) return bzpf::as_frag<T>(c, s);
    frag<T> f;
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] = (T)(c[8 * s + j] * by);
    return f;
  }
  __device__ __forceinline__ float back() const { return ON ? 1.f / by : 1.f; }
  // Where a round begins, unknown to the compiler: addresses of a second round's first loads, formed before the first round and
  // kept over it, took 15 registers and spilled.
  static __device__ __forceinline__ int first(int at) {
    if constexpr (ON) asm volatile("" : "+s"(at));
    return at;
  }
  // Whether the workgroup has to go over the axis again (the same in all of its threads). Channels past C hold what lay in LDS
  // and do not count, nor does a lane's column unless it is `mine`.
  template <int NT>
  __device__ __forceinline__ bool again(const f16x (&acc)[NT], int C, bool mine) {
    if constexpr (!ON) return false;
    f4 bad = f4{};  // stays 0 over finite numbers
#pragma unroll
    for (int tt = 0; tt < NT; tt++)
#pragma unroll
      for (int qq = 0; qq < 4; qq++) {
        if (32 * tt + 8 * qq >= C) break;
#pragma unroll
        for (int e = 0; e < 4; e++) bad[e] = fmaf(acc[tt][4 * qq + e], 0.f, bad[e]);
      }
    const bool more = !(both_sum((bad[0] + bad[1]) + (bad[2] + bad[3])) == 0.f) && mine && by > 0x1p-23f;
    by = more ? by * 0x1p-12f : by;
    return __syncthreads_or(more);
  }
};

// dq: a wave holds 32 queries as the columns of S^T, as the forward pass does. The sum's reciprocal is a row's own, so that it
// (in fp16: what root() leaves of it) scales dq at the end and ds is rounded before it. TWO: dO has a second part.
// 2 x 16 x 2000 x 2000 in 64 channels bf16 with a gate 133 to 146 us (matrix cores 38% busy, some pipe issuing 77% of the
// time), without 123; 16 x 400 x 400 in 24 channels fp32 15 us, latency.
template <typename T, typename BT, int KS, bool SPLIT, bool TWO>
__global__ __launch_bounds__(256, sizeof(T) == 2 && KS <= 4 ? 2 : 1) void attn_dq_k(Attn a, int64_t per_xcd) {
  typedef Form<T, SPLIT> F;
  constexpr int BK = F::BR, KT = BK / 32, NT = (KS + 1) / 2, TILE = BK * TILE_LD<T, KS>;
  constexpr int TILES = F::GROUPS * F::BUFS * 2 * TILE * (int)sizeof(T), MEET = SPLIT ? 4 * NT * 4096 : 0;
  constexpr bool MEND = sizeof(T) == 2;
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
  const int64_t orow = (un.smp * a.N + jc) * a.H * a.C + hc;
  const T* const dO = static_cast<const T*>(a.dO) + orow;
  const T* const dO_lo = TWO ? static_cast<const T*>(a.dO_lo) + orow : nullptr;
  const int64_t b0 = min(j0 + (SPLIT ? 0 : 32 * wave), a.N - 1);  // the wave's first row
  const BT* const bias = a.bias ? static_cast<const BT*>(a.bias) + (((int64_t)(un.smp / a.mult) * a.H + un.h) * a.N + b0) * a.M : nullptr;
  const int brows = (int)min(a.N - b0, (int64_t)32);
  u4* const Bt = reinterpret_cast<u4*>(bias_lds + wave * BiasRows<BT, BK>::BYTES);
  const float* mask = a.mask ? a.mask + un.smp * a.M : nullptr;
  const int64_t srow = ((int64_t)un.smp * a.H + un.h) * a.N + jc;
  RowStat rs(static_cast<const f4*>(a.rows)[srow]);
  // A sum of K terms of a size is some sqrt(K) of it: with p at sqrt(K / C) times its size, ds leaves fp16's range where dq of
  // keys of size one does.
  float less = 0.f;
  if constexpr (std::is_same<T, half_t>::value) less = rs.root(a.C);
  const bool some_big = __any(rs.ex.big());

  // dO's second part waits in LDS in the wide form (in registers 64 channels spill: dq of 2 x 16 x 2000 x
  // 2000 bf16 146 us so, 184 us there).
  constexpr bool ASIDE = TWO && !SPLIT;
  __shared__ frag<T> aside[ASIDE ? 4 * KS * 64 : 1];
  frag<T> qf[KS], df[KS], dl[TWO && !ASIDE ? KS : 1];
#pragma unroll
  for (int m = 0; m < KS; m++) {
    const bool in = 16 * m + 8 * hl < a.C;
    qf[m] = in ? load8(q + 16 * m + 8 * hl) : frag<T>{};
    df[m] = in ? load8(dO + 16 * m + 8 * hl) : frag<T>{};
    if constexpr (TWO) {
      const frag<T> f = in ? load8(dO_lo + 16 * m + 8 * hl) : frag<T>{};
      if constexpr (ASIDE) aside[(wave * KS + m) * 64 + l] = f;  // read by the lane that wrote it
      else dl[m] = f;
    }
  }
  f16x dq[NT], pk[MEND ? NT : 1];
  float off, taken;  // the row's sums of ds and of what its products take for it
  Scale<T> scale(0, a.C);  // root() is what dq needs

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
  int64_t k0;
  const auto start = [&] {
    off = taken = 0.f;
#pragma unroll
    for (int tt = 0; tt < NT; tt++) {
      dq[tt] = f16x{};
      if constexpr (MEND) pk[tt] = f16x{};
    }
    k0 = Scale<T>::first(group * BK);
    if (k0 < a.M) {
      fetch(k0);
      fetch_bias(k0);
    }
  };
  start();
  const bool masked = mask && any_key(mask, a.M);  // the first loads are on their way
  bool more;
  do {
    for (int buf = 0; k0 < a.M; k0 += STEP, buf = (buf + 1) % F::BUFS) {
      const uint64_t keep = __ballot(k0 + l < a.M && l < BK && (!masked || mk != 0.f));
      T* const Kb = Kt + buf * TILE;
      T* const Vb = Vt + buf * TILE;
      ks.store(Kb, keep, a.C, t);
      vs.store(Vb, keep, a.C, t);
      if (bias) bs.store(Bt, (int)a.M, (int)k0);
      F::sync();
      if (k0 + STEP < a.M) {
        fetch(k0 + STEP);
        fetch_bias(k0 + STEP);
      }
#pragma unroll
      for (int kt = 0; kt < KT; kt++) {
        f16x x = f16x{}, dp = f16x{};
#pragma unroll
        for (int m = 0; m < KS; m++) {
          x = mma(row_frag<T, KS>(Kb, 32 * kt + (l & 31), m), qf[m], x);
          const frag<T> vm = row_frag<T, KS>(Vb, 32 * kt + (l & 31), m);
          dp = mma(vm, df[m], dp);
          if constexpr (ASIDE) dp = mma(vm, aside[(wave * KS + m) * 64 + l], dp);
          else if constexpr (TWO) dp = mma(vm, dl[m], dp);
        }
        f16x b = f16x{};
        if (bias) b = BiasRows<BT, BK>::get(Bt, kt);
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = fmaf(x[i], a.scale, b[i]);
        exponentials(x, rs.ex, some_big, less);
#pragma unroll
        for (int i = 0; i < 16; i++) dp[i] = x[i] * (dp[i] - rs.delta);
        if (keep != all_rows(BK)) {
          const uint32_t w = (uint32_t)(keep >> (32 * kt)) >> (16 * hl);
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const bool on = w >> i & 1;
            x[i] = on ? x[i] : 0.f;
            dp[i] = on ? dp[i] : 0.f;
          }
        }
#pragma unroll
        for (int s = 0; s < 2; s++) {
          const frag<T> d = scale.as_frag(dp, s), p = as_frag<T>(x, s);
          if constexpr (MEND) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
              off += dp[8 * s + e];
              taken += (float)d[e];
            }
          }
#pragma unroll
          for (int tt = 0; tt < NT; tt++) {
            const frag<T> kf = col_frag<T, KS>(Kb, 32 * kt + 16 * s, tt);
            dq[tt] = mma(kf, d, dq[tt]);
            if constexpr (MEND) pk[tt] = mma(kf, p, pk[tt]);
          }
        }
      }
      F::again();
      if constexpr (!SPLIT) F::order();  // the biases are the wave's own
    }
    more = scale.again(dq, a.C, true);
    if (more) start();
  } while (more);
  if constexpr (MEND) {
    off = both_sum(off), taken = both_sum(taken) * scale.back();
    if constexpr (SPLIT) {
      float* const sums = reinterpret_cast<float*>(lds);
      __syncthreads();
      sums[threadIdx.x] = off;
      sums[256 + threadIdx.x] = taken;
      __syncthreads();
      off = (sums[l] + sums[64 + l]) + (sums[128 + l] + sums[192 + l]);
      taken = (sums[256 + l] + sums[320 + l]) + (sums[384 + l] + sums[448 + l]);
    }
    off *= rs.inv, taken *= rs.inv;
#pragma unroll
    for (int tt = 0; tt < NT; tt++) dq[tt] = dq[tt] * scale.back() - taken * pk[tt];
    // no other workgroup reads this row's, and this one's waves have what they need
    if (j < a.N && hl == 0 && (!SPLIT || wave == 0)) static_cast<float*>(a.rows)[4 * srow + 2] = rs.delta + off;
  }
  T* const out = static_cast<T*>(a.dq) + orow;
  const auto put = [&](int tt, int qq, f4 r) {
    const int c = 32 * tt + 8 * qq + 4 * hl;
    if (c >= a.C) return;
    r *= rs.inv * a.scale;
    store_chunk<4, false>(out + c, fv<4>{r[0], r[1], r[2], r[3]});
  };
  if constexpr (SPLIT) {
    f4 r[NT];
    meet4<NT>(dq, reinterpret_cast<f4*>(lds), wave, l, 1.f, r);
    if (j >= a.N) return;
#pragma unroll
    for (int tt = 0; tt < NT; tt++) put(tt, wave, r[tt]);
  } else {
    if (j >= a.N) return;
#pragma unroll
    for (int tt = 0; tt < NT; tt++)
#pragma unroll
      for (int qq = 0; qq < 4; qq++) put(tt, qq, f4{dq[tt][4 * qq], dq[tt][4 * qq + 1], dq[tt][4 * qq + 2], dq[tt][4 * qq + 3]});
  }
}

// dk and dv (and dbias): a wave holds 32 keys as the columns of S = Q K^T, so that dk^T = q^T ds and dv^T = dO^T p take p and
// ds from their lanes; the queries' statistics come from LDS, four rows a read. 2 x 16 x 2000 x 2000 in 64 channels bf16 with a
// gate 189 to 201 us with dbias, 179 without, 139 without a bias; matrix cores 29% busy, LDS 32%, some pipe issuing 76% of the
// time: two waves a SIMD take turns. 16 x 400 x 400 in 24 channels fp32 20 us, latency.
template <typename T, typename BT, int KS, bool SPLIT, bool TWO>
__global__ __launch_bounds__(256, sizeof(T) == 2 && KS <= 4 ? 2 : 1) void attn_dkv_k(Attn a, int64_t per_xcd) {
  typedef Form<T, SPLIT> F;
  constexpr int BQ = F::BR, QT = BQ / 32, NT = (KS + 1) / 2, TILE = BQ * TILE_LD<T, KS>, PARTS = TWO ? 3 : 2;
  constexpr int TILES = F::GROUPS * F::BUFS * PARTS * TILE * (int)sizeof(T), MEET = SPLIT ? 4 * NT * 4096 : 0;
  __shared__ LDS_ALIGN char lds[TILES > MEET ? TILES : MEET];
  __shared__ LDS_ALIGN float St[F::GROUPS][F::BUFS][4][BQ];
  __shared__ int Big[F::GROUPS][F::BUFS];
  static_assert(BQ <= F::NTH, "a thread a row of statistics");
  const int64_t kblocks = (a.M + F::ROWS - 1) / F::ROWS;
  Unit un;
  if (!unit_of(a, kblocks, per_xcd, &un)) return;  // whole workgroup
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63, hl = l >> 5;
  const int t = SPLIT ? l : threadIdx.x, group = SPLIT ? wave : 0;
  T* const Qt = reinterpret_cast<T*>(lds) + group * F::BUFS * PARTS * TILE;
  T* const Dt = Qt + F::BUFS * TILE;
  T* const Lt = Dt + F::BUFS * TILE;
  const int64_t key = un.block * F::ROWS + (SPLIT ? 0 : 32 * wave) + (l & 31), kc = min(key, a.M - 1);
  const int hc = un.h * a.C;
  const int64_t pitch = (int64_t)a.H * a.C, osmp = un.smp * a.N * pitch + hc;
  const T* const q = static_cast<const T*>(a.q) + un.smp * a.sq + hc;
  const T* const dO = static_cast<const T*>(a.dO) + osmp;
  const T* const dO_lo = TWO ? static_cast<const T*>(a.dO_lo) + osmp : nullptr;
  const T* const k = static_cast<const T*>(a.k) + un.smp * a.sk + kc * a.ldk + hc;
  const T* const v = static_cast<const T*>(a.v) + un.smp * a.sv + kc * a.ldv + hc;
  const int64_t plane = ((int64_t)(un.smp / a.mult) * a.H + un.h) * a.N * a.M;
  const BT* const bias = a.bias ? static_cast<const BT*>(a.bias) + plane : nullptr;
  BT* const db = a.dbias && a.mult == 1 ? static_cast<BT*>(a.dbias) + plane : nullptr;
  const uint32_t boff = (4 * hl * (uint32_t)a.M + (uint32_t)kc) * (uint32_t)sizeof(BT);  // a lane's first row of a tile, its key
  const int64_t srow = ((int64_t)un.smp * a.H + un.h) * a.N;
  const float* mask = a.mask ? a.mask + un.smp * a.M : nullptr;
  frag<T> kf[KS], vf[KS];
#pragma unroll
  for (int m = 0; m < KS; m++) {
    const int c = 16 * m + 8 * hl < a.C ? 16 * m + 8 * hl : 0;
    kf[m] = load8(k + c);
    vf[m] = load8(v + c);
  }
  const float mk = mask ? mask[kc] : 1.f;
  f16x dk[NT], dv[NT];
  Scale<T> scale(a.N, a.C);

  Stage<T, KS, BQ, F::NTH, false> qs, ds, ls;
  BT bs[16] = {};  // the next tile's biases, a row's 32 keys a half wave and instruction; zero where there are none
  f4 st;
  // The loop's loads depend on no condition (past the end they repeat the last block): the waits after a branch that leaves
  // some out would be for all loads in flight, the next block's among them.
  const auto fetch = [&](int64_t q0) {
    q0 = min(q0, (a.N - 1) / BQ * BQ);
    qs.load(q + q0 * a.ldq, (uint32_t)a.ldq, a.N - q0, a.C, t);
    ds.load(dO + q0 * pitch, (uint32_t)pitch, a.N - q0, a.C, t);
    if constexpr (TWO) ls.load(dO_lo + q0 * pitch, (uint32_t)pitch, a.N - q0, a.C, t);
    st = static_cast<const f4*>(a.rows)[srow + min(q0 + t % BQ, a.N - 1)];
  };
  const auto fetch_bias = [&](int64_t r0) {
    r0 = min(r0, (a.N - 1) / 32 * 32);
    const int n = (int)min(a.N - r0, (int64_t)32);
    const Columns<BT> at(bias ? bias + r0 * a.M : nullptr, bias ? n : 0, a.M);
    if (n == 32) {
#pragma unroll
      for (int i = 0; i < 16; i++) bs[i] = at.get(boff, 8 * (i >> 2) + (i & 3), true);
    } else {
#pragma unroll
      for (int i = 0; i < 16; i++) bs[i] = at.get(boff, 8 * (i >> 2) + (i & 3), false);
    }
  };
  constexpr int STEP = F::GROUPS * BQ;
  int64_t q0;
  const auto start = [&] {
#pragma unroll
    for (int tt = 0; tt < NT; tt++) dk[tt] = dv[tt] = f16x{};
    q0 = Scale<T>::first(group * BQ);
    fetch(q0);
    fetch_bias(q0);
  };
  start();
  const bool masked = mask && any_key(mask, a.M);  // of the whole workgroup; the first loads are on their way
  const bool on = key < a.M && (!masked || mk != 0.f);
#pragma unroll
  for (int m = 0; m < KS; m++) {
    const bool in = on && 16 * m + 8 * hl < a.C;
    kf[m] = in ? kf[m] : frag<T>{};
    vf[m] = in ? vf[m] : frag<T>{};
  }
  // A key that takes no part has zeros; lanes without a key write past every buffer's end.
  const uint32_t to = key < a.M ? boff : 0x80000000u;
  const auto put_bias = [&](int64_t r0, const f16x& x) {
    const int n = (int)min(a.N - r0, (int64_t)32);
    const Columns<BT> at(db + r0 * a.M, n, a.M);
    const typename Columns<BT>::Packed v(x, on);
    if (n == 32) {
#pragma unroll
      for (int i = 0; i < 16; i++) at.put(to, 8 * (i >> 2) + (i & 3), true, v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 16; i++) at.put(to, 8 * (i >> 2) + (i & 3), false, v[i]);
    }
  };
  bool more;
  do {
    for (int buf = 0; q0 < a.N; q0 += STEP, buf = (buf + 1) % F::BUFS) {
      const uint64_t rows = all_rows((int)min(a.N - q0, (int64_t)BQ));
      T* const Qb = Qt + buf * TILE;
      T* const Db = Dt + buf * TILE;
      T* const Lb = Lt + buf * TILE;
      float(*const Sb)[BQ] = St[group][buf];
      qs.store(Qb, rows, a.C, t);
      ds.store(Db, rows, a.C, t);
      if constexpr (TWO) ls.store(Lb, rows, a.C, t);
      if (t < BQ) {
        if (q0 + t >= a.N) st = f4{INFINITY, 0.f, 0.f, LOG2E};  // past the end: 2^(y by - inf) = 0
#pragma unroll
        for (int i = 0; i < 4; i++) Sb[i][t] = st[i];
        Big[group][buf] = __any(st[3] != LOG2E);
      }
      F::sync();
      const bool big = __builtin_amdgcn_readfirstlane(Big[group][buf]);  // a big row (Exponent)
      fetch(q0 + STEP);
#pragma unroll
      for (int qt = 0; qt < QT; qt++) {
        const int64_t r0 = q0 + 32 * qt;
        if (r0 >= a.N) break;
        const int64_t next = qt + 1 < QT ? r0 + 32 : q0 + STEP;
        f16x x = f16x{}, dp = f16x{};
#pragma unroll
        for (int m = 0; m < KS; m++) {
          x = mma(row_frag<T, KS>(Qb, 32 * qt + (l & 31), m), kf[m], x);
          dp = mma(row_frag<T, KS>(Db, 32 * qt + (l & 31), m), vf[m], dp);
          if constexpr (TWO) dp = mma(row_frag<T, KS>(Lb, 32 * qt + (l & 31), m), vf[m], dp);
        }
        // A key that takes no part has what it has in its own column alone, which ends as zeros.
        const auto probs = [&](auto any) {
#pragma unroll
          for (int qq = 0; qq < 4; qq++) {
            const int r = 32 * qt + 8 * qq + 4 * hl;
            const f4 at = *reinterpret_cast<const f4*>(&Sb[0][r]);
            const f4 inv = *reinterpret_cast<const f4*>(&Sb[1][r]);
            const f4 delta = *reinterpret_cast<const f4*>(&Sb[2][r]);
            f4 by = f4{LOG2E, LOG2E, LOG2E, LOG2E};
            if constexpr (any()) by = *reinterpret_cast<const f4*>(&Sb[3][r]);
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int i = 4 * qq + e;
              float z = fmaf(fmaf(x[i], a.scale, (float)bs[i]), by[e], -at[e]);
              if constexpr (any()) z = by[e] == 1.0f ? z * LOG2E : z;
              x[i] = __builtin_amdgcn_exp2f(z) * inv[e];
              dp[i] = x[i] * (dp[i] - delta[e]);
            }
            __builtin_amdgcn_sched_barrier(0);  // sixteen rows' statistics at once would not fit in the registers
          }
        };
        if (big) probs(std::true_type());
        else probs(std::false_type());
        fetch_bias(next);
        if (db) put_bias(r0, dp);
#pragma unroll
        for (int s = 0; s < 2; s++) {
          const frag<T> p = as_frag<T>(x, s), d = scale.as_frag(dp, s);
#pragma unroll
          for (int tt = 0; tt < NT; tt++) {
            dv[tt] = mma(col_frag<T, KS>(Db, 32 * qt + 16 * s, tt), p, dv[tt]);
            if constexpr (TWO) dv[tt] = mma(col_frag<T, KS>(Lb, 32 * qt + 16 * s, tt), p, dv[tt]);
            dk[tt] = mma(col_frag<T, KS>(Qb, 32 * qt + 16 * s, tt), d, dk[tt]);
          }
        }
      }
      F::again();
    }
    more = scale.again(dk, a.C, on);
    if (more) start();
  } while (more);
  const int64_t at = (un.smp * a.M + kc) * pitch + hc;
  const auto put = [&](void* to, int tt, int qq, f4 r, float by) {
    const int c = 32 * tt + 8 * qq + 4 * hl;
    if (!on) r = f4{};
    if (key < a.M && c < a.C) store_chunk<4, false>(static_cast<T*>(to) + at + c, fv<4>{r[0] * by, r[1] * by, r[2] * by, r[3] * by});
  };
  if constexpr (SPLIT) {
    f4 r[NT];
    meet4<NT>(dk, reinterpret_cast<f4*>(lds), wave, l, scale.back(), r);
#pragma unroll
    for (int tt = 0; tt < NT; tt++) put(a.dk, tt, wave, r[tt], a.scale);
    meet4<NT>(dv, reinterpret_cast<f4*>(lds), wave, l, 1.f, r);
#pragma unroll
    for (int tt = 0; tt < NT; tt++) put(a.dv, tt, wave, r[tt], 1.f);
  } else {
#pragma unroll
    for (int tt = 0; tt < NT; tt++)
#pragma unroll
      for (int qq = 0; qq < 4; qq++) {
        put(a.dk, tt, qq, f4{dk[tt][4 * qq], dk[tt][4 * qq + 1], dk[tt][4 * qq + 2], dk[tt][4 * qq + 3]}, a.scale * scale.back());
        put(a.dv, tt, qq, f4{dv[tt][4 * qq], dv[tt][4 * qq + 1], dv[tt][4 * qq + 2], dv[tt][4 * qq + 3]}, 1.f);
      }
  }
}

// dbias of a bias that `mult` samples share: a wave sums ds of one 32 x 32 tile over them in registers, the workgroup's four a
// 64 x 64 one whose rows of q, dO, k and v go through LDS, the next sample's on their way meanwhile (5 x 16 x 400 x 400 in 48 channels
// fp16 28 us; operands from L2 to each wave 41 us). Bound by latency, two barriers a sample.
template <typename T, typename BT, int KS, bool TWO>
__global__ __launch_bounds__(256, 1) void attn_dbias_k(Attn a, uint32_t tiles_k, uint32_t tiles_q) {
  constexpr int TILE = 64 * TILE_LD<T, KS>;
  __shared__ LDS_ALIGN T tiles[(TWO ? 5 : 4) * TILE];
  static_assert(sizeof(tiles) >= 4 * BiasRows<BT, 32>::BYTES, "the biases go through them first");
  T* const Qt = tiles;
  T* const Dt = Qt + TILE;
  T* const Kt = Dt + TILE;
  T* const Vt = Kt + TILE;
  T* const Lt = Vt + TILE;
  const int t = threadIdx.x, l = t & 63, hl = l >> 5, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const uint32_t per_head = tiles_k * tiles_q, bh = blockIdx.x / per_head, rest = blockIdx.x - bh * per_head;
  const int64_t q0 = 64 * (int64_t)(rest / tiles_k), k0 = 64 * (int64_t)(rest % tiles_k);
  const int h = (int)(bh % (uint32_t)a.H), b = (int)(bh / (uint32_t)a.H), hc = h * a.C;
  const int qw = 32 * (wave & 1), kw = 32 * (wave >> 1);  // the wave's tile
  const int64_t j = q0 + qw + (l & 31), jc = min(j, a.N - 1), first = k0 + kw + 16 * hl;  // the lane's query and first key
  const int64_t pitch = (int64_t)a.H * a.C;
  Stage<T, KS, 64, 256, false> qs, ds, ls;
  Stage<T, KS, 64, 256, true> ks, vs;
  float mk = 1.f;
  f4 rows;
  const auto fetch = [&](int64_t smp) {
    const int64_t out = (smp * a.N + q0) * pitch + hc;
    qs.load(static_cast<const T*>(a.q) + smp * a.sq + q0 * a.ldq + hc, (uint32_t)a.ldq, a.N - q0, a.C, t);
    ds.load(static_cast<const T*>(a.dO) + out, (uint32_t)pitch, a.N - q0, a.C, t);
    if constexpr (TWO) ls.load(static_cast<const T*>(a.dO_lo) + out, (uint32_t)pitch, a.N - q0, a.C, t);
    ks.load(static_cast<const T*>(a.k) + smp * a.sk + k0 * a.ldk + hc, (uint32_t)a.ldk, a.M - k0, a.C, t);
    vs.load(static_cast<const T*>(a.v) + smp * a.sv + k0 * a.ldv + hc, (uint32_t)a.ldv, a.M - k0, a.C, t);
    rows = static_cast<const f4*>(a.rows)[(smp * a.H + h) * a.N + jc];
    if (a.mask) mk = a.mask[smp * a.M + min(k0 + l, a.M - 1)];
  };
  const int64_t s0 = (int64_t)b * a.mult, s1 = s0 + a.mult;
  fetch(s0);
  f16x bias, sum = f16x{};
  {
    const int64_t r0 = min(q0 + qw, a.N - 1), c0 = min(k0 + kw, a.M - 1);
    BiasRows<BT, 32> bs;
    u4* const Bt = reinterpret_cast<u4*>(reinterpret_cast<char*>(tiles) + wave * BiasRows<BT, 32>::BYTES);
    bs.load(static_cast<const BT*>(a.bias) + ((int64_t)bh * a.N + r0) * a.M, (int)min(a.N - r0, (int64_t)32), (int)a.M, (int)c0);
    bs.store(Bt, (int)a.M, (int)c0);
    Form<T, true>::order();
    bias = BiasRows<BT, 32>::get(Bt, 0);
  }
  for (int64_t smp = s0; smp < s1; smp++) {
    uint64_t keep = __ballot(k0 + l < a.M && mk != 0.f);
    if (!keep) {  // none of these keys: does the sample have one at all?
      bool found = false;
      for (int64_t i = l; i < a.M && !__any(found); i += 64) found = a.mask[smp * a.M + i] != 0.f;
      if (!__any(found)) keep = __ballot(k0 + l < a.M);
    }
    const uint64_t live = all_rows((int)min(a.N - q0, (int64_t)64));
    __syncthreads();  // the tiles' readers are done
    qs.store(Qt, live, a.C, t);
    ds.store(Dt, live, a.C, t);
    if constexpr (TWO) ls.store(Lt, live, a.C, t);
    ks.store(Kt, keep, a.C, t);
    vs.store(Vt, keep, a.C, t);
    RowStat rs(rows);
    __syncthreads();
    if (smp + 1 < s1) fetch(smp + 1);
    if (!keep) continue;  // the same in every wave
    f16x x = f16x{}, dp = f16x{};
#pragma unroll
    for (int m = 0; m < KS; m++) {
      x = mma(row_frag<T, KS>(Kt, kw + (l & 31), m), row_frag<T, KS>(Qt, qw + (l & 31), m), x);
      const frag<T> vm = row_frag<T, KS>(Vt, kw + (l & 31), m);
      dp = mma(vm, row_frag<T, KS>(Dt, qw + (l & 31), m), dp);
      if constexpr (TWO) dp = mma(vm, row_frag<T, KS>(Lt, qw + (l & 31), m), dp);
    }
#pragma unroll
    for (int i = 0; i < 16; i++) x[i] = fmaf(x[i], a.scale, bias[i]);
    exponentials(x, rs.ex, __any(rs.ex.big()));
    const uint32_t on = (uint32_t)(keep >> kw) >> (16 * hl);
#pragma unroll
    for (int i = 0; i < 16; i++) dp[i] = x[i] * rs.inv * (dp[i] - rs.delta);
    if (keep != all_rows(64)) {
#pragma unroll
      for (int i = 0; i < 16; i++) dp[i] = on >> i & 1 ? dp[i] : 0.f;
    }
    sum += dp;
  }
  if (j >= a.N || first >= a.M) return;
  BT* const out = static_cast<BT*>(a.dbias) + ((int64_t)bh * a.N + j) * a.M + first;
  constexpr int V = 16 / (int)sizeof(BT);
#pragma unroll
  for (int c = 0; c < 16; c += V) {
    if (first + c + V <= a.M) {
      fv<V> y;
#pragma unroll
      for (int e = 0; e < V; e++) y[e] = sum[c + e];
      store_chunk<V, false>(out + c, y);
    } else {
#pragma unroll
      for (int e = 0; e < V; e++)
        if (first + c + e < a.M) out[c + e] = (BT)sum[c + e];
    }
  }
}

}  // namespace

// The workspace: what each row needs, then dO (in half types its second part after it) where there is a gate.
static int64_t stat_bytes(int64_t rows) { return rows * 16; }
static int64_t part_bytes(int dt, int64_t rows, int C) { return rows * C * (dt == DT_F32 ? 4 : 2); }

int64_t attention_bwd_ws_bytes(int dt, int64_t S, int64_t N, int H, int C, bool gate) {
  const int64_t rows = S * N * H;
  return stat_bytes(rows) + (gate ? part_bytes(dt, rows, C) * (dt == DT_F32 ? 1 : 2) : 0);
}

hipError_t launch_attention_bwd(Attn a, void* ws, hipStream_t st) {
  const int64_t rows = (int64_t)a.S * a.N * a.H;
  a.rows = ws;
  char* const parts = static_cast<char*>(ws) + stat_bytes(rows);
  a.dO = a.g ? parts : const_cast<void*>(a.dout);
  a.dO_lo = parts + part_bytes(a.dt, rows, a.C);
  return with_attn(a, [&](auto t, auto b, auto ks) {
    typedef decltype(t) T;
    typedef decltype(b) BT;
    constexpr int KS = decltype(ks)::value;
    int L = 1;
    while (8 * L < a.C) L *= 2;
    const int64_t wgs = (rows + 256 / L - 1) / (256 / L);
    if (wgs > INT32_MAX) return hipErrorInvalidValue;
    attn_rows_k<T><<<(unsigned)wgs, 256, 0, st>>>(a, L);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const auto blocks = [&](int64_t n, int rows) { return ((n + rows - 1) / rows * a.S * a.H + 7) / 8; };  // for each XCD
    const auto go = [&](auto two) {
      constexpr bool TWO = decltype(two)::value;
      const auto dq = [&](auto split) {
        const int64_t per = blocks(a.N, Form<T, decltype(split)::value>::ROWS);
        if (8 * per > INT32_MAX) return hipErrorInvalidValue;
        attn_dq_k<T, BT, KS, decltype(split)::value, TWO><<<(unsigned)(8 * per), 256, 0, st>>>(a, per);
        return hipGetLastError();
      };
      const auto dkv = [&](auto split) {
        const int64_t per = blocks(a.M, Form<T, decltype(split)::value>::ROWS);
        if (8 * per > INT32_MAX) return hipErrorInvalidValue;
        attn_dkv_k<T, BT, KS, decltype(split)::value, TWO><<<(unsigned)(8 * per), 256, 0, st>>>(a, per);
        return hipGetLastError();
      };
      hipError_t e = with_split<KS>(a.N, a, dq);
      if (e == hipSuccess) e = with_split<KS>(a.M, a, dkv);
      if (e != hipSuccess || !a.dbias || a.mult == 1) return e;
      const int64_t tk = (a.M + 63) / 64, tq = (a.N + 63) / 64, tiles = tk * tq * a.H * (a.S / a.mult);
      if (tiles > INT32_MAX) return hipErrorInvalidValue;
      attn_dbias_k<T, BT, KS, TWO><<<(unsigned)tiles, 256, 0, st>>>(a, (uint32_t)tk, (uint32_t)tq);
      return hipGetLastError();
    };
    if constexpr (sizeof(T) == 2) {
      if (a.g) return go(std::true_type());
    }
    return go(std::false_type());
  });
}

}  // namespace bzpf

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
//   sum in fp32, takes it off again (with one more product, p k) and hands the mended delta on.
// - dO is not a value of the type: it goes as two of them, the rounded one and the rest, in the products of dp and dv.
// Without these the gradients were 1.7 to 2.3 times as far from the exact ones as their own rounding puts them, now 1.0 to 1.4.
#include "bzpf_attn.h"

namespace bzpf {

namespace {

// delta [S][H][N], and with a gate dO (two parts in half types) and dg. L lanes a head, 8 channels each.
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
  if (on && l == 0) a.delta[(smp * a.H + h) * a.N + row - smp * a.N] = d;
}

// A row's maximum (0 for a row without logits, whose probabilities are exp(-inf)) and the sum's reciprocal (0 for it).
struct RowStat {
  float top, inv, delta;
  __device__ __forceinline__ RowStat(const Attn& a, int64_t row) {
    const float m = a.stats[2 * row], s = a.stats[2 * row + 1];
    top = m == -INFINITY ? 0.f : m;
    inv = s == 0.f ? 0.f : 1.0f / s;
    delta = a.delta[row];
  }
};

// dq: a wave holds 32 queries as the columns of S^T, as the forward pass does. The sum's reciprocal is a row's own, so that it
// scales dq at the end and ds is rounded before it. TWO: dO has a second part.
template <typename T, typename BT, int KS, int NW, bool TWO>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 2 && KS <= 4 ? 2 : 1) void attn_dq_k(Attn a, int64_t per_xcd) {
  constexpr int BK = sizeof(T) == 2 ? 64 : 32, KT = BK / 32, NT = (KS + 1) / 2, NTH = 64 * NW, WQ = 32 * NW;
  __shared__ LDS_ALIGN T Kt[2][BK * TILE_LD<T, KS>];
  __shared__ LDS_ALIGN T Vt[2][BK * TILE_LD<T, KS>];
  const int64_t qblocks = (a.N + WQ - 1) / WQ;
  Unit un;
  if (!unit_of(a, qblocks, per_xcd, &un)) return;  // whole workgroup
  const int t = threadIdx.x, l = t & 63, hl = l >> 5;
  const int64_t j = un.block * WQ + 32 * (t >> 6) + (l & 31), jc = min(j, a.N - 1);
  const int hc = un.h * a.C;
  const T* const q = static_cast<const T*>(a.q) + un.smp * a.sq + jc * a.ldq + hc;
  const T* const k = static_cast<const T*>(a.k) + un.smp * a.sk + hc;
  const T* const v = static_cast<const T*>(a.v) + un.smp * a.sv + hc;
  const T* const dO = static_cast<const T*>(a.dO) + (un.smp * a.N + jc) * a.H * a.C + hc;
  const BT* const bias = a.bias ? static_cast<const BT*>(a.bias) + (((int64_t)(un.smp / a.mult) * a.H + un.h) * a.N + jc) * a.M : nullptr;
  const float* mask = a.mask ? a.mask + un.smp * a.M : nullptr;
  if (!any_key<NTH>(mask, a.M)) mask = nullptr;
  const T* const dO_lo = TWO ? static_cast<const T*>(a.dO_lo) + (un.smp * a.N + jc) * a.H * a.C + hc : nullptr;
  const int64_t srow = ((int64_t)un.smp * a.H + un.h) * a.N + jc;
  const RowStat rs(a, srow);
  constexpr bool MEND = sizeof(T) == 2;

  frag<T> qf[KS], df[KS], dl[TWO ? KS : 1];
#pragma unroll
  for (int m = 0; m < KS; m++) {
    const bool in = 16 * m + 8 * hl < a.C;
    qf[m] = in ? load8(q + 16 * m + 8 * hl) : frag<T>{};
    df[m] = in ? load8(dO + 16 * m + 8 * hl) : frag<T>{};
    if constexpr (TWO) dl[m] = in ? load8(dO_lo + 16 * m + 8 * hl) : frag<T>{};
  }
  f16x dq[NT], pk[MEND ? NT : 1];
  float off = 0.f;  // the row's sum of ds
#pragma unroll
  for (int tt = 0; tt < NT; tt++) {
    dq[tt] = f16x{};
    if constexpr (MEND) pk[tt] = f16x{};
  }

  Stage<T, KS, BK, NTH> ks, vs;
  Bias4<BT> bs[KT][4];
  float mk = 1.f;
  const auto fetch = [&](int64_t k0) {
    ks.load(k, a.ldk, k0, a.M, a.C);
    vs.load(v, a.ldv, k0, a.M, a.C);
    if (mask) mk = mask[min(k0 + l, a.M - 1)];
  };
  const auto fetch_bias = [&](int64_t k0) {
    if (!bias) return;
#pragma unroll
    for (int kt = 0; kt < KT; kt++)
#pragma unroll
      for (int qq = 0; qq < 4; qq++) {
        const int64_t at = k0 + 32 * kt + 8 * qq + 4 * hl;
        if (k0 + BK <= a.M) bs[kt][qq].load(bias + at);
        else bs[kt][qq].load(bias + at, a.M - at);
      }
  };
  fetch(0);
  fetch_bias(0);
  for (int64_t k0 = 0; k0 < a.M; k0 += BK) {
    const int buf = (int)(k0 / BK & 1);
    const uint64_t keep = __ballot(k0 + l < a.M && l < BK && mk != 0.f);
    ks.store(Kt[buf], keep, a.C);
    vs.store(Vt[buf], keep, a.C);
    __syncthreads();  // as in the forward pass
    const bool more = k0 + BK < a.M;
    if (more) fetch(k0 + BK);
#pragma unroll
    for (int kt = 0; kt < KT; kt++) {
      f16x x = f16x{}, dp = f16x{};
#pragma unroll
      for (int m = 0; m < KS; m++) {
        x = mma(row_frag<T, KS>(Kt[buf], 32 * kt + (l & 31), m), qf[m], x);
        const frag<T> vm = row_frag<T, KS>(Vt[buf], 32 * kt + (l & 31), m);
        dp = mma(vm, df[m], dp);
        if constexpr (TWO) dp = mma(vm, dl[m], dp);
      }
      if (bias) {
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = fmaf(x[i], a.scale, (float)bs[kt][i >> 2].v[i & 3]);
      } else {
        x *= a.scale;
      }
      const uint32_t w = (uint32_t)(keep >> (32 * kt)) >> (4 * hl);
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const bool on = keep == all_rows(BK) || (w >> (8 * (i >> 2) + (i & 3)) & 1);
        x[i] = on ? __builtin_amdgcn_exp2f((x[i] - rs.top) * LOG2E) : 0.f;
        dp[i] = on ? x[i] * (dp[i] - rs.delta) : 0.f;
        if constexpr (MEND) off += dp[i];
      }
#pragma unroll
      for (int s = 0; s < 2; s++) {
        const frag<T> d = as_frag<T>(dp, s), p = as_frag<T>(x, s);
#pragma unroll
        for (int tt = 0; tt < NT; tt++) {
          const frag<T> kf = col_frag<T, KS>(Kt[buf], 32 * kt + 16 * s, tt);
          dq[tt] = mma(kf, d, dq[tt]);
          if constexpr (MEND) pk[tt] = mma(kf, p, pk[tt]);
        }
      }
    }
    if (more) fetch_bias(k0 + BK);
  }
  if constexpr (MEND) {
    off = both_sum(off) * rs.inv;
#pragma unroll
    for (int tt = 0; tt < NT; tt++) dq[tt] -= off * pk[tt];
    if (j < a.N && hl == 0) a.delta[srow] = rs.delta + off;  // this lane's row alone: no other reads it in this kernel
  }
  if (j >= a.N) return;
  const float by = rs.inv * a.scale;
  T* const out = static_cast<T*>(a.dq) + (un.smp * a.N + j) * a.H * a.C + hc;
#pragma unroll
  for (int tt = 0; tt < NT; tt++)
#pragma unroll
    for (int qq = 0; qq < 4; qq++) {
      const int c = 32 * tt + 8 * qq + 4 * hl;
      if (c >= a.C) continue;
      fv<4> r;
#pragma unroll
      for (int e = 0; e < 4; e++) r[e] = dq[tt][4 * qq + e] * by;
      store_chunk<4, false>(out + c, r);
    }
}

// dk and dv (and dbias): a wave holds 32 keys as the columns of S = Q K^T, so that dk^T = q^T ds and dv^T = dO^T p take p and
// ds from their lanes; the queries' statistics come from LDS, four rows a read.
template <typename T, typename BT, int KS, int NW, bool TWO>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 2 && KS <= 4 ? 2 : 1) void attn_dkv_k(Attn a, int64_t per_xcd) {
  constexpr int BQ = sizeof(T) == 2 ? 64 : 32, QT = BQ / 32, NT = (KS + 1) / 2, NTH = 64 * NW, WK = 32 * NW;
  static_assert(BQ <= NTH, "a thread a row of statistics");
  __shared__ LDS_ALIGN T Qt[2][BQ * TILE_LD<T, KS>];
  __shared__ LDS_ALIGN T Dt[2][BQ * TILE_LD<T, KS>];
  __shared__ LDS_ALIGN T Lt[TWO ? 2 : 1][TWO ? BQ * TILE_LD<T, KS> : 8];
  __shared__ LDS_ALIGN float St[2][3][BQ];
  const int64_t kblocks = (a.M + WK - 1) / WK;
  Unit un;
  if (!unit_of(a, kblocks, per_xcd, &un)) return;  // whole workgroup
  const int t = threadIdx.x, l = t & 63, hl = l >> 5;
  const int64_t key = un.block * WK + 32 * (t >> 6) + (l & 31), kc = min(key, a.M - 1);
  const int hc = un.h * a.C;
  const T* const q = static_cast<const T*>(a.q) + un.smp * a.sq + hc;
  const T* const dO = static_cast<const T*>(a.dO) + un.smp * a.N * a.H * a.C + hc;
  const T* const dO_lo = TWO ? static_cast<const T*>(a.dO_lo) + un.smp * a.N * a.H * a.C + hc : nullptr;
  const T* const k = static_cast<const T*>(a.k) + un.smp * a.sk + kc * a.ldk + hc;
  const T* const v = static_cast<const T*>(a.v) + un.smp * a.sv + kc * a.ldv + hc;
  const int64_t plane = ((int64_t)(un.smp / a.mult) * a.H + un.h) * a.N * a.M;
  const BT* const bias = a.bias ? static_cast<const BT*>(a.bias) + plane + kc : nullptr;
  BT* const db = a.dbias && a.mult == 1 ? static_cast<BT*>(a.dbias) + plane + kc : nullptr;
  const int64_t srow = ((int64_t)un.smp * a.H + un.h) * a.N;
  const float* mask = a.mask ? a.mask + un.smp * a.M : nullptr;
  if (!any_key<NTH>(mask, a.M)) mask = nullptr;
  const bool on = key < a.M && (!mask || mask[kc] != 0.f);

  frag<T> kf[KS], vf[KS];
#pragma unroll
  for (int m = 0; m < KS; m++) {
    const bool in = on && 16 * m + 8 * hl < a.C;
    kf[m] = in ? load8(k + 16 * m + 8 * hl) : frag<T>{};
    vf[m] = in ? load8(v + 16 * m + 8 * hl) : frag<T>{};
  }
  f16x dk[NT], dv[NT];
#pragma unroll
  for (int tt = 0; tt < NT; tt++) dk[tt] = dv[tt] = f16x{};

  Stage<T, KS, BQ, NTH> qs, ds, ls;
  BT bs[QT][16];
  float st[3];
  const auto fetch = [&](int64_t q0) {
    qs.load(q, a.ldq, q0, a.N, a.C);
    ds.load(dO, (int64_t)a.H * a.C, q0, a.N, a.C);
    if constexpr (TWO) ls.load(dO_lo, (int64_t)a.H * a.C, q0, a.N, a.C);
    if (t < BQ) {
      const RowStat r(a, srow + min(q0 + t, a.N - 1));
      const bool in = q0 + t < a.N;  // past the end: exp(y - inf) = 0
      st[0] = in ? r.top : INFINITY;
      st[1] = in ? r.inv : 0.f;
      st[2] = in ? r.delta : 0.f;
    }
  };
  const auto fetch_bias = [&](int64_t q0) {
    if (!bias) return;
#pragma unroll
    for (int qt = 0; qt < QT; qt++)
#pragma unroll
      for (int i = 0; i < 16; i++) bs[qt][i] = bias[min(q0 + 32 * qt + 8 * (i >> 2) + 4 * hl + (i & 3), a.N - 1) * a.M];
  };
  fetch(0);
  fetch_bias(0);
  for (int64_t q0 = 0; q0 < a.N; q0 += BQ) {
    const int buf = (int)(q0 / BQ & 1);
    const uint64_t rows = all_rows((int)min(a.N - q0, (int64_t)BQ));
    qs.store(Qt[buf], rows, a.C);
    ds.store(Dt[buf], rows, a.C);
    if constexpr (TWO) ls.store(Lt[buf], rows, a.C);
    if (t < BQ)
#pragma unroll
      for (int i = 0; i < 3; i++) St[buf][i][t] = st[i];
    __syncthreads();  // as in the forward pass
    const bool more = q0 + BQ < a.N;
    if (more) fetch(q0 + BQ);
#pragma unroll
    for (int qt = 0; qt < QT; qt++) {
      f16x x = f16x{}, dp = f16x{};
#pragma unroll
      for (int m = 0; m < KS; m++) {
        x = mma(row_frag<T, KS>(Qt[buf], 32 * qt + (l & 31), m), kf[m], x);
        dp = mma(row_frag<T, KS>(Dt[buf], 32 * qt + (l & 31), m), vf[m], dp);
        if constexpr (TWO) dp = mma(row_frag<T, KS>(Lt[buf], 32 * qt + (l & 31), m), vf[m], dp);
      }
#pragma unroll
      for (int qq = 0; qq < 4; qq++) {
        const int r = 32 * qt + 8 * qq + 4 * hl;
        const f4 top = *reinterpret_cast<const f4*>(&St[buf][0][r]);
        const f4 inv = *reinterpret_cast<const f4*>(&St[buf][1][r]);
        const f4 delta = *reinterpret_cast<const f4*>(&St[buf][2][r]);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int i = 4 * qq + e;
          const float y = bias ? fmaf(x[i], a.scale, (float)bs[qt][i]) : x[i] * a.scale;
          const float p = on ? __builtin_amdgcn_exp2f((y - top[e]) * LOG2E) * inv[e] : 0.f;
          x[i] = p;
          dp[i] = on ? p * (dp[i] - delta[e]) : 0.f;
        }
      }
      if (db && key < a.M) {
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int64_t r = q0 + 32 * qt + 8 * (i >> 2) + 4 * hl + (i & 3);
          if (r < a.N) db[r * a.M] = (BT)dp[i];
        }
      }
#pragma unroll
      for (int s = 0; s < 2; s++) {
        const frag<T> p = as_frag<T>(x, s), d = as_frag<T>(dp, s);
#pragma unroll
        for (int tt = 0; tt < NT; tt++) {
          dv[tt] = mma(col_frag<T, KS>(Dt[buf], 32 * qt + 16 * s, tt), p, dv[tt]);
          if constexpr (TWO) dv[tt] = mma(col_frag<T, KS>(Lt[buf], 32 * qt + 16 * s, tt), p, dv[tt]);
          dk[tt] = mma(col_frag<T, KS>(Qt[buf], 32 * qt + 16 * s, tt), d, dk[tt]);
        }
      }
    }
    if (more) fetch_bias(q0 + BQ);
  }
  if (key >= a.M) return;
  const int64_t at = (un.smp * a.M + key) * a.H * a.C + hc;
#pragma unroll
  for (int tt = 0; tt < NT; tt++)
#pragma unroll
    for (int qq = 0; qq < 4; qq++) {
      const int c = 32 * tt + 8 * qq + 4 * hl;
      if (c >= a.C) continue;
      fv<4> rk, rv;
#pragma unroll
      for (int e = 0; e < 4; e++) rk[e] = dk[tt][4 * qq + e] * a.scale, rv[e] = dv[tt][4 * qq + e];
      store_chunk<4, false>(static_cast<T*>(a.dk) + at + c, rk);
      store_chunk<4, false>(static_cast<T*>(a.dv) + at + c, rv);
    }
}

// dbias of a bias that `mult` samples share: a wave sums ds of one 32 x 32 tile over them in registers. Operands come
// from L2, where the samples' rows lie.
template <typename T, typename BT, int KS, bool TWO>
__global__ __launch_bounds__(256, 1) void attn_dbias_k(Attn a, int64_t tiles_k, int64_t tiles) {
  const int l = threadIdx.x & 63, hl = l >> 5;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= tiles) return;  // whole wave; no barriers
  const int64_t kt = w % tiles_k, tiles_q = (a.N + 31) / 32, qt = w / tiles_k % tiles_q, bh = w / tiles_k / tiles_q;
  const int h = (int)(bh % a.H), hc = h * a.C;
  const int64_t b = bh / a.H, j = 32 * qt + (l & 31), jc = min(j, a.N - 1), kc = min(32 * kt + (l & 31), a.M - 1);
  const int64_t k4 = 32 * kt + 4 * hl, row = (bh * a.N + jc) * a.M;
  Bias4<BT> bs[4];
#pragma unroll
  for (int qq = 0; qq < 4; qq++) bs[qq].load(static_cast<const BT*>(a.bias) + row + k4 + 8 * qq, a.M - k4 - 8 * qq);
  f16x sum = f16x{};
  for (int64_t smp = b * a.mult; smp < (b + 1) * a.mult; smp++) {
    const T* const q = static_cast<const T*>(a.q) + smp * a.sq + jc * a.ldq + hc;
    const T* const dO = static_cast<const T*>(a.dO) + (smp * a.N + jc) * a.H * a.C + hc;
    const T* const dO_lo = TWO ? static_cast<const T*>(a.dO_lo) + (smp * a.N + jc) * a.H * a.C + hc : nullptr;
    const T* const k = static_cast<const T*>(a.k) + smp * a.sk + kc * a.ldk + hc;
    const T* const v = static_cast<const T*>(a.v) + smp * a.sv + kc * a.ldv + hc;
    bool on = true;
    if (a.mask) {
      const float* const mask = a.mask + smp * a.M;
      on = mask[kc] != 0.f;
      if (!__any(on)) {  // none of this tile's keys: does the sample have one at all?
        bool found = false;
        for (int64_t i = l; i < a.M && !found; i += 64) found = mask[i] != 0.f;
        on = !__any(found);
        if (!on) continue;
      }
    }
    const uint32_t keep = (uint32_t)__ballot(on) >> (4 * hl);
    const RowStat rs(a, (smp * a.H + h) * a.N + jc);
    f16x x = f16x{}, dp = f16x{};
#pragma unroll
    for (int m = 0; m < KS; m++) {
      const int c = 16 * m + 8 * hl;
      const bool in = c < a.C;
      const frag<T> z{};
      x = mma(in && on ? load8(k + c) : z, in ? load8(q + c) : z, x);
      const frag<T> vm = in && on ? load8(v + c) : z;
      dp = mma(vm, in ? load8(dO + c) : z, dp);
      if constexpr (TWO) dp = mma(vm, in ? load8(dO_lo + c) : z, dp);
    }
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const float y = fmaf(x[i], a.scale, (float)bs[i >> 2].v[i & 3]);
      const float d = __builtin_amdgcn_exp2f((y - rs.top) * LOG2E) * rs.inv * (dp[i] - rs.delta);
      sum[i] += keep >> (8 * (i >> 2) + (i & 3)) & 1 ? d : 0.f;
    }
  }
  if (j >= a.N) return;
  BT* const out = static_cast<BT*>(a.dbias) + row;
#pragma unroll
  for (int qq = 0; qq < 4; qq++) {
    const int64_t at = k4 + 8 * qq;
    if (at + 4 <= a.M) {
      store_chunk<4, false>(out + at, fv<4>{sum[4 * qq], sum[4 * qq + 1], sum[4 * qq + 2], sum[4 * qq + 3]});
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (at + e < a.M) out[at + e] = (BT)sum[4 * qq + e];
    }
  }
}

}  // namespace

// The workspace: delta, then dO (in half types its second part after it) where there is a gate.
static int64_t delta_bytes(int64_t rows) { return (rows * 4 + 15) / 16 * 16; }
static int64_t part_bytes(int dt, int64_t rows, int C) { return rows * C * (dt == DT_F32 ? 4 : 2); }

int64_t attention_bwd_ws_bytes(int dt, int64_t S, int64_t N, int H, int C, bool gate) {
  const int64_t rows = S * N * H;
  return delta_bytes(rows) + (gate ? part_bytes(dt, rows, C) * (dt == DT_F32 ? 1 : 2) : 0);
}

hipError_t launch_attention_bwd(Attn a, void* ws, hipStream_t st) {
  const int64_t rows = (int64_t)a.S * a.N * a.H;
  a.delta = static_cast<float*>(ws);
  char* const parts = static_cast<char*>(ws) + delta_bytes(rows);
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
    const auto go = [&](auto nw, auto two) {
      constexpr int NW = decltype(nw)::value;
      constexpr bool TWO = decltype(two)::value;
      const int64_t uq = (a.N + 32 * NW - 1) / (32 * NW) * a.S * a.H, pq = (uq + 7) / 8;
      const int64_t uk = (a.M + 32 * NW - 1) / (32 * NW) * a.S * a.H, pk = (uk + 7) / 8;
      const int64_t tk = (a.M + 31) / 32, tiles = tk * ((a.N + 31) / 32) * a.H * (a.S / a.mult);
      if (8 * pq > INT32_MAX || 8 * pk > INT32_MAX || (tiles + 3) / 4 > INT32_MAX) return hipErrorInvalidValue;
      attn_dq_k<T, BT, KS, NW, TWO><<<(unsigned)(8 * pq), 64 * NW, 0, st>>>(a, pq);
      hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
      attn_dkv_k<T, BT, KS, NW, TWO><<<(unsigned)(8 * pk), 64 * NW, 0, st>>>(a, pk);
      e = hipGetLastError();
      if (e != hipSuccess || !a.dbias || a.mult == 1) return e;
      attn_dbias_k<T, BT, KS, TWO><<<(unsigned)((tiles + 3) / 4), 256, 0, st>>>(a, tk, tiles);
      return hipGetLastError();
    };
    const int64_t n = a.N < a.M ? a.N : a.M;
    const bool few = (n + 127) / 128 * a.S * a.H < 512;
    typedef std::integral_constant<int, 2> Two;
    typedef std::integral_constant<int, 4> Four;
    if constexpr (sizeof(T) == 2) {
      if (a.g) return few ? go(Two(), std::true_type()) : go(Four(), std::true_type());
    }
    return few ? go(Two(), std::false_type()) : go(Four(), std::false_type());
  });
}

}  // namespace bzpf

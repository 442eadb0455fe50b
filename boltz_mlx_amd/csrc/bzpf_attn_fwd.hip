// The sequence attention's forward pass with the statistics that its backward pass needs (bzpf_attn.h has the formulas).
// One pass over the keys with the running maximum and sum of each row's softmax; a wave holds 32 queries as the columns of
// S^T = K Q^T, so that a row's statistics are a lane's own (and its other half's). Logits stay in natural units until their
// maximum is subtracted.
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
    const Exponent now(most);
    const float by = __builtin_amdgcn_exp2f(fminf(ex.at - now.at, 0.f));  // a row without logits so far: 0 times anything
#pragma unroll
    for (int tt = 0; tt < NT; tt++) o[tt] *= by;
    sum *= by;
    top = most;
    ex = now;
#pragma unroll
    for (int kt = 0; kt < KT; kt++) {
#pragma unroll
      for (int i = 0; i < 16; i++) {
        x[kt][i] = ex.of(x[kt][i]);
        sum += x[kt][i];
      }
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
    st[1] = sum * __builtin_amdgcn_exp2f(-ex.off(top));
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
    const auto by = [&](float at) { return __builtin_amdgcn_exp2f(fminf(at - all.at, 0.f)); };
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) total += st[w * 64 + l].y * by(Exponent(st[w * 64 + l].x).at);
    f4 r[NT];
    meet4<NT>(o, reinterpret_cast<f4*>(lds), wave, l, by(ex.at), r);
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

}  // namespace

hipError_t launch_attention(const Attn& a, hipStream_t st) {
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

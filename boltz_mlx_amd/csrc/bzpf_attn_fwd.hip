// The sequence attention's forward pass with the statistics that its backward pass needs (bzpf_attn.h has the formulas).
// One pass over the keys with the running maximum and sum of each row's softmax; every workgroup holds 32 NW queries, a wave
// 32 as the columns of S^T = K Q^T, so that a row's statistics are a lane's own. Logits stay in natural units until their
// maximum is subtracted: a row whose logits are all at the type's lowest value is a softmax over equals like any other.
#include "bzpf_attn.h"

namespace bzpf {

namespace {

template <typename T, typename BT, int KS, int NW>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 2 && KS <= 4 ? 2 : 1) void attn_fwd_k(Attn a, int64_t per_xcd) {
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
  const BT* const bias = a.bias ? static_cast<const BT*>(a.bias) + (((int64_t)(un.smp / a.mult) * a.H + un.h) * a.N + jc) * a.M : nullptr;
  const float* mask = a.mask ? a.mask + un.smp * a.M : nullptr;
  if (!any_key<NTH>(mask, a.M)) mask = nullptr;

  frag<T> qf[KS];
#pragma unroll
  for (int m = 0; m < KS; m++) qf[m] = 16 * m + 8 * hl < a.C ? load8(q + 16 * m + 8 * hl) : frag<T>{};
  f16x o[NT];
#pragma unroll
  for (int tt = 0; tt < NT; tt++) o[tt] = f16x{};
  float top = -INFINITY, sum = 0.f;

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
    __syncthreads();  // the other buffer's readers passed the barrier before; this one's next writer passes the next
    const bool more = k0 + BK < a.M;
    if (more) fetch(k0 + BK);
    f16x x[KT];
    float most = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < KT; kt++) {
      f16x s = f16x{};
#pragma unroll
      for (int m = 0; m < KS; m++) s = mma(row_frag<T, KS>(Kt[buf], 32 * kt + (l & 31), m), qf[m], s);
      if (bias) {
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = fmaf(s[i], a.scale, (float)bs[kt][i >> 2].v[i & 3]);
      } else {
        s *= a.scale;
      }
      if (keep != all_rows(BK)) {
        const uint32_t w = (uint32_t)(keep >> (32 * kt)) >> (4 * hl);
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = w >> (8 * (i >> 2) + (i & 3)) & 1 ? s[i] : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 16; i += 2) most = fmaxf(fmaxf(most, s[i]), s[i + 1]);
      x[kt] = s;
    }
    if (more) fetch_bias(k0 + BK);
    most = fmaxf(top, both_max(most));
    if (__any(most > top)) {
      const float by = most > top ? __builtin_amdgcn_exp2f((top - most) * LOG2E) : 1.f;
#pragma unroll
      for (int tt = 0; tt < NT; tt++) o[tt] *= by;
      sum *= by;
      top = most;
    }
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int kt = 0; kt < KT; kt++) {
#pragma unroll
      for (int i = 0; i < 16; i++) {
        x[kt][i] = __builtin_amdgcn_exp2f((x[kt][i] - ref) * LOG2E);
        sum += x[kt][i];
      }
#pragma unroll
      for (int s = 0; s < 2; s++) {
        const frag<T> p = as_frag<T>(x[kt], s);
#pragma unroll
        for (int tt = 0; tt < NT; tt++) o[tt] = mma(col_frag<T, KS>(Vt[buf], 32 * kt + 16 * s, tt), p, o[tt]);
      }
    }
  }
  sum = both_sum(sum);
  if (j >= a.N) return;
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  if (hl == 0) {
    float* const st = a.stats + (((int64_t)un.smp * a.H + un.h) * a.N + j) * 2;
    st[0] = top;
    st[1] = sum;
  }
  T* const out = static_cast<T*>(a.out) + (un.smp * a.N + j) * a.H * a.C + hc;
  const T* const g = a.g ? static_cast<const T*>(a.g) + un.smp * a.sg + j * a.ldg + hc : nullptr;
#pragma unroll
  for (int tt = 0; tt < NT; tt++)
#pragma unroll
    for (int qq = 0; qq < 4; qq++) {
      const int c = 32 * tt + 8 * qq + 4 * hl;
      if (c >= a.C) continue;
      fv<4> r;
#pragma unroll
      for (int e = 0; e < 4; e++) r[e] = o[tt][4 * qq + e] * inv;
      if (g) {
        const fv<4> gv = load_chunk<4>(g + c);
#pragma unroll
        for (int e = 0; e < 4; e++) r[e] *= sigmoidf_(gv[e]);
      }
      store_chunk<4, false>(out + c, r);
    }
}

}  // namespace

hipError_t launch_attention(const Attn& a, hipStream_t st) {
  return with_attn(a, [&](auto t, auto b, auto ks) {
    typedef decltype(t) T;
    typedef decltype(b) BT;
    constexpr int KS = decltype(ks)::value;
    const auto go = [&](auto nw) {
      constexpr int NW = decltype(nw)::value;
      const int64_t units = (a.N + 32 * NW - 1) / (32 * NW) * a.S * a.H, per = (units + 7) / 8;
      if (8 * per > INT32_MAX) return hipErrorInvalidValue;
      attn_fwd_k<T, BT, KS, NW><<<(unsigned)(8 * per), 64 * NW, 0, st>>>(a, per);
      return hipGetLastError();
    };
    if ((a.N + 127) / 128 * a.S * a.H < 512) return go(std::integral_constant<int, 2>());
    return go(std::integral_constant<int, 4>());
  });
}

}  // namespace bzpf

// C-ABI entry points of the sequence attention's training form (declared in include/bzpf.h): argument validation, dispatch.
#include <cmath>

#include "bzpf.h"
#include "bzpf_api.h"
#include "bzpf_kernels.h"

namespace {

using namespace bzpf_api;

int64_t size_of(int dt) { return dt == BZPF_F32 ? 4 : 2; }
// a * b * c * d where it is below 2^62, else -1 (all >= 0).
int64_t product(int64_t a, int64_t b, int64_t c, int64_t d) {
  unsigned __int128 n = 1;
  for (int64_t x : {a, b, c, d}) {
    n *= (unsigned __int128)x;
    if (n >> 62) return -1;
  }
  return (int64_t)n;
}

struct Range {
  const void* p;
  int64_t bytes;
};
bool apart_from(const Range& a, const Range& b) {
  const auto at = [](const Range& r) { return reinterpret_cast<uintptr_t>(r.p); };
  return !a.p || !b.p || a.bytes == 0 || b.bytes == 0 || at(a) + (unsigned __int128)a.bytes <= at(b) ||
         at(b) + (unsigned __int128)b.bytes <= at(a);
}
// Whether the outputs share no byte with an input or with each other.
template <size_t NO, size_t NI>
bool all_apart(const Range (&outs)[NO], const Range (&ins)[NI]) {
  for (size_t i = 0; i < NO; i++) {
    for (const Range& in : ins)
      if (!apart_from(outs[i], in)) return false;
    for (size_t j = 0; j < i; j++)
      if (!apart_from(outs[i], outs[j])) return false;
  }
  return true;
}

// The arguments that the bias and its gradient share, checked into *a.
int make_rel(const char* who, const void* t, int dt, const unsigned char* lut, int64_t lo, int span, int count,
             const void* pos_q, const void* pos_k, const void* group_q, const void* group_k, int wide, int64_t batch_q,
             int64_t batch_k, int64_t B, int H, int64_t N, int64_t M, bzpf::RelBias* a) {
  REQUIRE(dt3_ok(dt), "%s: bad dtype %d", who, dt);
  REQUIRE(count >= 1 && count <= 256 && span >= 1 && span <= 16384, "%s: need 1 <= count <= 256 and 1 <= span <= 16384 (%d, %d)",
          who, count, span);
  REQUIRE(lo > -((int64_t)1 << 62) && lo < ((int64_t)1 << 62), "%s: lo out of range", who);
  REQUIRE(B >= 0 && B <= 65535 && H >= 1 && H <= 65535 && N >= 0 && M >= 0 && N <= INT32_MAX && M <= INT32_MAX &&
              product(B, H, N, M) >= 0,
          "%s: bad sizes (B=%lld H=%d N=%lld M=%lld)", who, (long long)B, H, (long long)N, (long long)M);
  if (product(B, H, N, M) == 0) return BZPF_OK;
  REQUIRE(t && aligned_el(t, dt), "%s: a tensor is null or misaligned", who);
  const uintptr_t whole = wide ? 7 : 3;
  for (const void* p : {pos_q, pos_k, group_q, group_k})
    REQUIRE((reinterpret_cast<uintptr_t>(p) & whole) == 0, "%s: positions or groups misaligned", who);
  REQUIRE(lut && pos_q && pos_k && !group_q == !group_k, "%s: lut, pos_q and pos_k must be given, and both groups or none", who);
  REQUIRE((batch_q == 0 || batch_q >= N) && (batch_k == 0 || batch_k >= M) && product(B, batch_q, 8, 1) >= 0 &&
              product(B, batch_k, 8, 1) >= 0,
          "%s: batch strides below the lengths or too large", who);
  *a = bzpf::RelBias{nullptr, lut, lo, span, count, H, pos_q, pos_k, group_q, group_k, wide != 0, batch_q, batch_k, N, M};
  return BZPF_OK;
}

}  // namespace

extern "C" {

int bzpf_rel_bias(const float* table, const unsigned char* lut, int64_t lo, int span, int count, const void* pos_q,
                  const void* pos_k, const void* group_q, const void* group_k, int wide, int64_t batch_q, int64_t batch_k,
                  const void* add, void* out, int dt, int64_t B, int H, int64_t N, int64_t M, void* stream) {
  bzpf::RelBias a;
  const int rc = make_rel("bzpf_rel_bias", out, dt, lut, lo, span, count, pos_q, pos_k, group_q, group_k, wide, batch_q,
                          batch_k, B, H, N, M, &a);
  const int64_t n = rc == BZPF_OK ? product(B, H, N, M) : 0;
  if (n == 0) return rc;
  REQUIRE_EL(table, BZPF_F32);
  REQUIRE(aligned_el(add, dt), "bzpf_rel_bias: add misaligned");
  const Range outs[] = {{out, n * size_of(dt)}};
  const int64_t w = wide ? 8 : 4, nq = ((B - 1) * batch_q + N) * w, nk = ((B - 1) * batch_k + M) * w;
  const Range ins[] = {{add, n * size_of(dt)}, {table, (int64_t)count * H * 4}, {lut, span}, {pos_q, nq}, {group_q, nq},
                       {pos_k, nk}, {group_k, nk}};
  REQUIRE(all_apart(outs, ins), "bzpf_rel_bias: out overlaps another tensor");
  a.table = table;
  return done(bzpf::launch_rel_bias(a, add, out, dt, B, S(stream)), "bzpf_rel_bias");
}

int64_t bzpf_rel_bias_bwd_ws(int64_t B, int H, int64_t N, int64_t M, int count) {
  if (B < 1 || B > 65535 || H < 1 || H > 65535 || N < 1 || M < 1 || N > INT32_MAX || M > INT32_MAX || count < 1 || count > 256 ||
      product(B, H, N, M) < 0 || B * ((H + 15) / 16) > 65535)
    return -1;
  return bzpf::rel_bias_bwd_ws_bytes(B, H, N, M, count);
}

int bzpf_rel_bias_bwd(const void* dout, int dt, const unsigned char* lut, int64_t lo, int span, int count, const void* pos_q,
                      const void* pos_k, const void* group_q, const void* group_k, int wide, int64_t batch_q,
                      int64_t batch_k, float* dtable, float* ws, int64_t ws_bytes, int64_t B, int H, int64_t N, int64_t M,
                      void* stream) {
  bzpf::RelBias a;
  REQUIRE(B >= 1 && N >= 1 && M >= 1, "bzpf_rel_bias_bwd: no pairs (B=%lld N=%lld M=%lld)", (long long)B, (long long)N,
          (long long)M);
  const int rc = make_rel("bzpf_rel_bias_bwd", dout, dt, lut, lo, span, count, pos_q, pos_k, group_q, group_k, wide, batch_q,
                          batch_k, B, H, N, M, &a);
  if (rc != BZPF_OK) return rc;
  REQUIRE(B * ((H + 15) / 16) <= 65535, "bzpf_rel_bias_bwd: at most 65535 groups of 16 heads over the batch (B=%lld H=%d)", (long long)B, H);
  REQUIRE_EL(dtable, BZPF_F32);
  REQUIRE_EL(ws, BZPF_F32);
  const int64_t need = bzpf::rel_bias_bwd_ws_bytes(B, H, N, M, count);
  REQUIRE(ws_bytes >= need, "bzpf_rel_bias_bwd: ws holds %lld bytes of %lld", (long long)ws_bytes, (long long)need);
  const Range outs[] = {{dtable, (int64_t)count * H * 4}, {ws, need}};
  const int64_t w = wide ? 8 : 4, nq = ((B - 1) * batch_q + N) * w, nk = ((B - 1) * batch_k + M) * w;
  const Range ins[] = {{dout, product(B, H, N, M) * size_of(dt)}, {lut, span}, {pos_q, nq}, {group_q, nq}, {pos_k, nk},
                       {group_k, nk}};
  REQUIRE(all_apart(outs, ins), "bzpf_rel_bias_bwd: dtable or ws overlaps another tensor");
  return done(bzpf::launch_rel_bias_bwd(a, dout, dt, dtable, ws, B, S(stream)), "bzpf_rel_bias_bwd");
}

}  // extern "C"

namespace {

int make_qk(const char* who, const void* q, int64_t ldq, const void* k, int64_t ldk, int x_dt, const float* w_q,
            const float* w_k, float eps, const void* pos, int wide, int64_t pos_rows, double base, int rotary, int interleaved,
            const void* yq, const void* yk, int y_dt, int64_t rows, int H, int Hk, int C, bzpf::QKNorm* a) {
  REQUIRE(pair_ok(x_dt, y_dt), "%s: bad dtype %d/%d", who, x_dt, y_dt);
  REQUIRE(C >= 2 && C <= bzpf::QK_MAX_C && C % 2 == 0, "%s: heads of an even 2 to 256 channels (C=%d)", who, C);
  REQUIRE(rotary >= 0 && rotary <= C && rotary % 2 == 0, "%s: rotary must be even, 0 to C (%d)", who, rotary);
  REQUIRE(H >= 1 && H <= 1024 && Hk >= 1 && Hk <= 1024, "%s: 1 to 1024 heads (%d, %d)", who, H, Hk);
  REQUIRE(rows >= 0 && product(rows, H > Hk ? H : Hk, C, 4) >= 0, "%s: bad row count", who);
  if (rows == 0) return BZPF_OK;
  REQUIRE(q && k && yq && yk, "%s: NULL pointer", who);
  REQUIRE(aligned_el(q, x_dt) && aligned_el(k, x_dt) && aligned_el(yq, y_dt) && aligned_el(yk, y_dt) &&
              aligned_el(w_q, BZPF_F32) && aligned_el(w_k, BZPF_F32),
          "%s: a tensor is misaligned", who);
  REQUIRE(rows == 1 || (ldq >= (int64_t)H * C && ldk >= (int64_t)Hk * C), "%s: row pitches below a row's width", who);
  REQUIRE(product(rows, ldq > ldk ? ldq : ldk, 4, 1) >= 0, "%s: bad row pitches", who);
  REQUIRE(!pos || (pos_rows >= 1 && (reinterpret_cast<uintptr_t>(pos) & (wide ? 7 : 3)) == 0),
          "%s: pos misaligned or without rows", who);
  REQUIRE(!pos || (base > 0 && std::isfinite(base)), "%s: base must be positive", who);
  *a = bzpf::QKNorm{};
  a->x[0] = q, a->x[1] = k;
  a->ld[0] = ldq, a->ld[1] = ldk;
  a->w[0] = w_q, a->w[1] = w_k;
  a->y[0] = const_cast<void*>(yq), a->y[1] = const_cast<void*>(yk);
  a->H[0] = H, a->H[1] = Hk;
  a->C = C, a->rot = rotary;
  a->inter = interleaved != 0, a->wide = wide != 0;
  a->pos = rotary ? pos : nullptr, a->pos_rows = pos_rows, a->rows = rows;
  a->log2_base = pos ? std::log2(base) : 0.0;
  a->eps = eps;
  return BZPF_OK;
}

// The bytes from a view's first element to its last, of rows of `width` elements.
int64_t extent(int64_t S, int64_t s, int64_t rows, int64_t ld, int64_t width, int dt) {
  return ((S - 1) * s + (rows - 1) * ld + width) * size_of(dt);
}

}  // namespace

extern "C" {

int bzpf_qk_norm_rope(const void* q, int64_t ldq, const void* k, int64_t ldk, int x_dt, const float* w_q, const float* w_k,
                      float eps, const void* pos, int wide, int64_t pos_rows, double base, int rotary, int interleaved,
                      void* qn, void* kn, int y_dt, int64_t rows, int H, int Hk, int C, void* stream) {
  bzpf::QKNorm a;
  const int rc = make_qk("bzpf_qk_norm_rope", q, ldq, k, ldk, x_dt, w_q, w_k, eps, pos, wide, pos_rows, base, rotary,
                         interleaved, qn, kn, y_dt, rows, H, Hk, C, &a);
  if (rc != BZPF_OK || rows == 0) return rc;
  const int64_t wq = (int64_t)H * C, wk = (int64_t)Hk * C;
  const Range outs[] = {{qn, rows * wq * size_of(y_dt)}, {kn, rows * wk * size_of(y_dt)}};
  const Range ins[] = {{q, extent(1, 0, rows, ldq, wq, x_dt)}, {k, extent(1, 0, rows, ldk, wk, x_dt)}, {w_q, 4 * C},
                       {w_k, 4 * C}, {pos, pos ? pos_rows * (wide ? 8 : 4) : 0}};
  REQUIRE(all_apart(outs, ins), "bzpf_qk_norm_rope: qn or kn overlaps another tensor");
  return done(bzpf::launch_qk_norm(a, x_dt, y_dt, S(stream)), "bzpf_qk_norm_rope");
}

int64_t bzpf_qk_norm_rope_bwd_ws(int C) {
  return C >= 2 && C <= bzpf::QK_MAX_C && C % 2 == 0 ? bzpf::qk_norm_ws_bytes(C) : -1;
}

int bzpf_qk_norm_rope_bwd(const void* dqn, const void* dkn, int y_dt, const void* q, int64_t ldq, const void* k, int64_t ldk,
                          int x_dt, const float* w_q, const float* w_k, float eps, const void* pos, int wide,
                          int64_t pos_rows, double base, int rotary, int interleaved, void* dq, void* dk, float* dw_q,
                          float* dw_k, float* ws, int64_t ws_bytes, int64_t rows, int H, int Hk, int C, void* stream) {
  bzpf::QKNorm a;
  REQUIRE(rows >= 1, "bzpf_qk_norm_rope_bwd: rows < 1");
  const int rc = make_qk("bzpf_qk_norm_rope_bwd", q, ldq, k, ldk, x_dt, w_q, w_k, eps, pos, wide, pos_rows, base, rotary,
                         interleaved, dqn, dkn, y_dt, rows, H, Hk, C, &a);
  if (rc != BZPF_OK) return rc;
  REQUIRE_EL(dq, x_dt);
  REQUIRE_EL(dk, x_dt);
  REQUIRE(aligned_el(dw_q, BZPF_F32) && aligned_el(dw_k, BZPF_F32) && aligned_el(ws, BZPF_F32),
          "bzpf_qk_norm_rope_bwd: dw_q, dw_k or ws misaligned");
  const int64_t need = dw_q || dw_k ? bzpf::qk_norm_ws_bytes(C) : 0;
  REQUIRE(need == 0 || (ws && ws_bytes >= need), "bzpf_qk_norm_rope_bwd: ws holds %lld bytes of %lld",
          (long long)(ws ? ws_bytes : 0), (long long)need);
  const int64_t wq = (int64_t)H * C, wk = (int64_t)Hk * C;
  const Range outs[] = {{dq, rows * wq * size_of(x_dt)}, {dk, rows * wk * size_of(x_dt)}, {dw_q, 4 * C}, {dw_k, 4 * C}, {ws, need}};
  const Range ins[] = {{q, extent(1, 0, rows, ldq, wq, x_dt)}, {k, extent(1, 0, rows, ldk, wk, x_dt)}, {w_q, 4 * C},
                       {w_k, 4 * C}, {pos, pos ? pos_rows * (wide ? 8 : 4) : 0}, {dqn, rows * wq * size_of(y_dt)},
                       {dkn, rows * wk * size_of(y_dt)}};
  REQUIRE(all_apart(outs, ins), "bzpf_qk_norm_rope_bwd: an output overlaps another tensor");
  a.dx[0] = dq, a.dx[1] = dk;
  a.ws = need ? ws : nullptr;
  return done(bzpf::launch_qk_norm_bwd(a, x_dt, y_dt, dw_q, dw_k, S(stream)), "bzpf_qk_norm_rope_bwd");
}

}  // extern "C"

namespace {

constexpr int64_t ATT_LEN = 1 << 22, ATT_PITCH = 1 << 23;  // what the kernels' 32-bit offsets within a block hold
constexpr int64_t WORKGROUPS = (1 << 24) - 8;              // a launch has fewer than 2^32 threads, 256 a workgroup

// Whether sizes are such that no product of them below overflows, and a launch holds them.
bool attn_sizes(int S, int H, int C, int64_t N, int64_t M) {
  if (S < 1 || H < 1 || H > 65535 || C < 8 || C > 128 || C % 8 || N < 1 || M < 1 || N > ATT_LEN || M > ATT_LEN) return false;
  const int64_t most = N > M ? N : M, groups = product(S, H, (most + 31) / 32, 1), chunks = product(S, H, N, (C + 7) / 8);
  return groups >= 0 && groups <= WORKGROUPS && chunks >= 0 && chunks < (int64_t)1 << 31 && product(S, H, N, M) >= 0 &&
         product(S, most, H, 4 * C) >= 0;
}

int make_attn(const char* who, const void* q, int64_t ldq, int64_t sq, const void* k, int64_t ldk, int64_t sk, const void* v,
              int64_t ldv, int64_t sv, const void* g, int64_t ldg, int64_t sg, const void* bias, int bias_dt, int mult,
              const float* mask, const void* out, const float* stats, int dt, int S, int H, int C, int64_t N, int64_t M,
              bzpf::Attn* a) {
  REQUIRE(dt3_ok(dt), "%s: bad dtype %d", who, dt);
  REQUIRE(!bias || bias_dt == dt || (dt == BZPF_F32 && dt3_ok(bias_dt)),
          "%s: a bias of the operands' type, or fp16 / bf16 with fp32 operands (%d with %d)", who, bias_dt, dt);
  REQUIRE(C >= 8 && C <= 128 && C % 8 == 0, "%s: heads of 8 to 128 channels, a multiple of 8 (C=%d)", who, C);
  REQUIRE(S >= 1 && H >= 1 && H <= 65535 && mult >= 1 && S % mult == 0, "%s: bad sample or head counts (S=%d H=%d mult=%d)",
          who, S, H, mult);
  REQUIRE(N >= 1 && M >= 1 && N <= ATT_LEN && M <= ATT_LEN, "%s: 1 to 2^22 queries and keys (N=%lld M=%lld)", who, (long long)N,
          (long long)M);
  REQUIRE(attn_sizes(S, H, C, N, M), "%s: too many samples, heads and rows for a launch (S=%d H=%d N=%lld M=%lld)", who, S, H, (long long)N, (long long)M);
  REQUIRE(q && k && v && out && stats, "%s: NULL pointer", who);
  for (const void* p : {q, k, v, g, out}) REQUIRE(aligned_el(p, dt), "%s: a tensor is misaligned", who);
  REQUIRE(aligned_el(bias, bias_dt) && aligned_el(mask, BZPF_F32) && aligned_el(stats, BZPF_F32), "%s: a tensor is misaligned", who);
  const int64_t w = (int64_t)H * C;
  REQUIRE((N == 1 || (ldq >= w && (!g || ldg >= w))) && (M == 1 || (ldk >= w && ldv >= w)), "%s: row pitches below a row's width", who);
  for (int64_t l : {w, ldq, ldk, ldv, ldg}) REQUIRE(l >= 0 && l < ATT_PITCH, "%s: rows of fewer than 2^23 elements", who);
  REQUIRE(sq >= 0 && sk >= 0 && sv >= 0 && sg >= 0, "%s: negative sample strides", who);
  for (int64_t s : {sq, sk, sv, sg}) REQUIRE(product(S, s, 4, 1) >= 0, "%s: bad strides", who);
  *a = bzpf::Attn{};
  a->q = q, a->k = k, a->v = v, a->g = g, a->bias = bias, a->mask = mask;
  a->ldq = ldq, a->ldk = ldk, a->ldv = ldv, a->ldg = ldg, a->sq = sq, a->sk = sk, a->sv = sv, a->sg = sg;
  a->N = N, a->M = M, a->S = S, a->H = H, a->C = C, a->mult = mult, a->dt = dt, a->bias_dt = bias ? bias_dt : dt;
  a->scale = (float)(1.0 / std::sqrt((double)C));
  a->out = const_cast<void*>(out), a->stats = const_cast<float*>(stats);
  return BZPF_OK;
}

}  // namespace

extern "C" {

int64_t bzpf_attention_ws(int S_, int H, int C, int64_t N, int64_t M) {
  if (!attn_sizes(S_, H, C, N, M)) return -1;
  bzpf::Attn a{};
  a.S = S_, a.H = H, a.C = C, a.N = N, a.M = M;
  return bzpf::attention_ws_bytes(a);
}

int bzpf_attention(const void* q, int64_t ldq, int64_t sq, const void* k, int64_t ldk, int64_t sk, const void* v, int64_t ldv,
                   int64_t sv, const void* g, int64_t ldg, int64_t sg, const void* bias, int bias_dt, int mult,
                   const float* mask, void* out, float* stats, void* ws, int64_t ws_bytes, int dt, int S_, int H, int C,
                   int64_t N, int64_t M, void* stream) {
  bzpf::Attn a;
  const int rc = make_attn("bzpf_attention", q, ldq, sq, k, ldk, sk, v, ldv, sv, g, ldg, sg, bias, bias_dt, mult, mask, out,
                           stats, dt, S_, H, C, N, M, &a);
  if (rc != BZPF_OK) return rc;
  const int64_t w = (int64_t)H * C;
  const int64_t need = bzpf::attention_ws_bytes(a);
  REQUIRE(ws_bytes >= need && (ws || !need), "bzpf_attention: ws holds %lld bytes of %lld", (long long)(ws ? ws_bytes : 0), (long long)need);
  REQUIRE(((uintptr_t)ws & 15) == 0, "bzpf_attention: ws must be 16-byte aligned");
  const Range outs[] = {{out, S_ * N * w * size_of(dt)}, {stats, (int64_t)S_ * H * N * 8}, {ws, need}};
  const Range ins[] = {{q, extent(S_, sq, N, ldq, w, dt)}, {k, extent(S_, sk, M, ldk, w, dt)}, {v, extent(S_, sv, M, ldv, w, dt)},
                       {g, extent(S_, sg, N, ldg, w, dt)}, {bias, (int64_t)(S_ / mult) * H * N * M * size_of(bias_dt)}, {mask, S_ * M * 4}};
  REQUIRE(all_apart(outs, ins), "bzpf_attention: out or stats overlaps another tensor");
  return done(bzpf::launch_attention(a, ws, S(stream)), "bzpf_attention");
}

int64_t bzpf_attention_bwd_ws(int dt, int S_, int H, int C, int64_t N, int64_t M, int gate) {
  if (!dt3_ok(dt) || !attn_sizes(S_, H, C, N, M)) return -1;
  return bzpf::attention_bwd_ws_bytes(dt, S_, N, H, C, gate != 0);
}

int bzpf_attention_bwd(const void* dout, const void* q, int64_t ldq, int64_t sq, const void* k, int64_t ldk, int64_t sk,
                       const void* v, int64_t ldv, int64_t sv, const void* g, int64_t ldg, int64_t sg, const void* bias,
                       int bias_dt, int mult, const float* mask, const void* out, const float* stats, void* dq, void* dk,
                       void* dv, void* dg, void* dbias, void* ws, int64_t ws_bytes, int dt, int S_, int H, int C, int64_t N,
                       int64_t M, void* stream) {
  bzpf::Attn a;
  const int rc = make_attn("bzpf_attention_bwd", q, ldq, sq, k, ldk, sk, v, ldv, sv, g, ldg, sg, bias, bias_dt, mult, mask, out,
                           stats, dt, S_, H, C, N, M, &a);
  if (rc != BZPF_OK) return rc;
  REQUIRE_EL(dout, dt);
  REQUIRE_EL(dq, dt);
  REQUIRE_EL(dk, dt);
  REQUIRE_EL(dv, dt);
  REQUIRE(!g == !dg && (bias || !dbias) && aligned_el(dg, dt) && aligned_el(dbias, bias_dt),
          "bzpf_attention_bwd: dg goes with g, dbias with bias");
  REQUIRE(!dbias || mult == 1 || product(S_ / mult, H, (N + 63) / 64, (M + 63) / 64) <= WORKGROUPS,
          "bzpf_attention_bwd: a shared bias of too many tiles for a launch");
  const int64_t need = bzpf::attention_bwd_ws_bytes(dt, S_, N, H, C, g != nullptr);
  REQUIRE_PTR(ws);
  REQUIRE(ws_bytes >= need, "bzpf_attention_bwd: ws holds %lld bytes of %lld", (long long)ws_bytes, (long long)need);
  const int64_t w = (int64_t)H * C, e = size_of(dt), qo = S_ * N * w * e, kv = S_ * M * w * e;
  const int64_t plane = (int64_t)(S_ / mult) * H * N * M * size_of(bias_dt);
  const Range outs[] = {{dq, qo}, {dk, kv}, {dv, kv}, {dg, qo}, {dbias, plane}, {ws, need}};
  const Range ins[] = {{q, extent(S_, sq, N, ldq, w, dt)}, {k, extent(S_, sk, M, ldk, w, dt)}, {v, extent(S_, sv, M, ldv, w, dt)},
                       {g, extent(S_, sg, N, ldg, w, dt)}, {bias, plane}, {mask, S_ * M * 4}, {out, qo},
                       {stats, (int64_t)S_ * H * N * 8}, {dout, qo}};
  REQUIRE(all_apart(outs, ins), "bzpf_attention_bwd: an output overlaps another tensor");
  a.dout = dout, a.dq = dq, a.dk = dk, a.dv = dv, a.dg = dg, a.dbias = dbias;
  return done(bzpf::launch_attention_bwd(a, ws, S(stream)), "bzpf_attention_bwd");
}

}  // extern "C"

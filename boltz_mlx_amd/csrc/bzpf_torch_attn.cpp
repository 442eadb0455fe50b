// torch binding of the sequence attention's training form: the position bias by buckets, the norms of queries and keys with
// the rotation, the attention, and their autograd nodes (bzpf_torch.cpp says why these are native).
//
// Arguments are checked before devices, so that what a call would refuse can be seen without a GPU.
#include "bzpf_torch.h"

namespace bzpf_torch {

namespace {

bool whole(const Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }

// ------------------------------------------------------------------------------------------------ position bias

// The buckets of a bias and the positions it is for, checked; positions are contiguous [n] or [B, n].
struct Rel {
  Tensor lut, pos_q, pos_k, group_q, group_k;
  int64_t lo, count, B = 1, N, M;
  bool other, batched = false;
  Rel(const char* name, Tensor lut_, int64_t lo_, int64_t count_, bool other_, Tensor pq, Tensor pk, Tensor gq, Tensor gk)
      : lut(lut_), pos_q(pq), pos_k(pk.defined() ? pk : pq), group_q(gq), group_k(gk.defined() || pk.defined() ? gk : gq),
        lo(lo_), count(count_), other(other_) {
    TORCH_CHECK_VALUE(lut.scalar_type() == at::kByte && lut.dim() == 1 && lut.is_contiguous() && lut.size(0) >= 1, name,
                      ": buckets must be made by rel_buckets");
    count_fits(name, "distances", lut.size(0));
    count_fits(name, "buckets", count);
    TORCH_CHECK_VALUE((pos_q.dim() == 1 || pos_q.dim() == 2) && (pos_k.dim() == 1 || pos_k.dim() == 2), name,
                      ": positions must be [n] or [B, n], got ", pos_q.sizes(), " and ", pos_k.sizes());
    TORCH_CHECK_VALUE(group_q.defined() == group_k.defined(), name, ": groups must be given for queries and keys, or for neither");
    for (const Tensor& t : {pos_q, pos_k, group_q, group_k})
      TORCH_CHECK_VALUE(!t.defined() || (whole(t) && t.scalar_type() == pos_q.scalar_type() && t.device() == lut.device()), name,
                        ": positions and groups must be of one integer type (int32 or int64) on ", lut.device());
    TORCH_CHECK_VALUE(!group_q.defined() || (group_q.sizes() == pos_q.sizes() && group_k.sizes() == pos_k.sizes()), name,
                      ": groups must have their positions' shapes");
    for (const Tensor& t : {pos_q, pos_k})
      if (t.dim() == 2) {
        TORCH_CHECK_VALUE(!batched || B == t.size(0), name, ": positions of different batch sizes: ", B, " and ", t.size(0));
        batched = true, B = t.size(0);
      }
    if (!other) group_q = group_k = Tensor();  // one bucket scheme for every pair
    N = pos_q.size(-1), M = pos_k.size(-1);
    for (Tensor* t : {&pos_q, &pos_k, &group_q, &group_k})
      if (t->defined()) *t = t->contiguous();
  }
  // What t ([H, N, M] or [B, H, N, M]) says of the batch; H.
  int64_t meet(const char* name, const Tensor& t, const char* what) {
    TORCH_CHECK_VALUE((t.dim() == 3 || t.dim() == 4) && t.size(-2) == N && t.size(-1) == M &&
                          (t.dim() == 4 ? !batched || t.size(0) == B : !batched),
                      name, ": ", what, " must be [", batched ? "B, " : "", "H, ", N, ", ", M, "], got ", t.sizes());
    TORCH_CHECK_VALUE(t.device() == lut.device(), name, ": ", what, " must be on ", lut.device());
    if (t.dim() == 4) batched = true, B = t.size(0);
    count_fits(name, "heads", t.size(-3));
    return t.size(-3);
  }
  bool wide() const { return pos_q.scalar_type() == at::kLong; }
  int64_t batch_q() const { return pos_q.dim() == 2 ? N : 0; }
  int64_t batch_k() const { return pos_k.dim() == 2 ? M : 0; }
};

Tensor rel_bias(const Tensor& table, Rel r, const Tensor& add_, at::ScalarType to) {
  const char* name = "rel_bias";
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) == r.count && table.size(1) >= 1 && table.device() == r.lut.device(), name,
                    ": table must be [", r.count, ", H] on ", r.lut.device(), ", got ", table.sizes());
  type_code(table);
  const int dt = type_code(to);
  const int64_t H = table.size(1);
  count_fits(name, "heads", H);
  if (add_.defined()) {
    TORCH_CHECK_VALUE(r.meet(name, add_, "add") == H && add_.scalar_type() == to, name, ": add must have ", H,
                      " heads and the output's type");
  }
  on_gpu(name, table, r.pos_q);
  const OnDevice dev(table);
  const Tensor w = param(table), add = add_.defined() ? add_.contiguous() : add_;
  const auto opt = table.options().dtype(to);
  const Tensor y = r.batched ? at::empty({r.B, H, r.N, r.M}, opt) : at::empty({H, r.N, r.M}, opt);
  if (y.numel())
    check(lib.rel_bias(f32(w), r.lut.const_data_ptr<uint8_t>(), r.lo, (int)r.lut.size(0), (int)r.count, in(r.pos_q), in(r.pos_k),
                       in(r.group_q), in(r.group_k), r.wide(), r.batch_q(), r.batch_k(), in(add), out(y), dt, r.B, (int)H, r.N,
                       r.M, dev.stream),
          "bzpf_rel_bias");
  return y;
}

Tensor rel_bias_bwd(const Tensor& dy_, Rel r) {
  const char* name = "rel_bias_bwd";
  const int64_t H = r.meet(name, dy_, "dbias");
  const int dt = type_code(dy_);
  on_gpu(name, dy_, r.pos_q);
  const OnDevice dev(dy_);
  const Tensor dy = dy_.contiguous();
  const auto opt = dy.options().dtype(at::kFloat);
  if (!dy.numel()) return at::zeros({r.count, H}, opt);
  const Tensor d = at::empty({r.count, H}, opt);
  const int64_t bytes = lib.rel_bias_bwd_ws(r.B, (int)H, r.N, r.M, (int)r.count);
  const Tensor ws = at::empty({bytes / 4}, opt);
  check(lib.rel_bias_bwd(in(dy), dt, r.lut.const_data_ptr<uint8_t>(), r.lo, (int)r.lut.size(0), (int)r.count, in(r.pos_q),
                         in(r.pos_k), in(r.group_q), in(r.group_k), r.wide(), r.batch_q(), r.batch_k(), f32_out(d),
                         f32_out(ws), bytes, r.B, (int)H, r.N, r.M, dev.stream),
        "bzpf_rel_bias_bwd");
  return d;
}

struct RelBiasNode : torch::autograd::Function<RelBiasNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, Opt add, const Tensor& lut, int64_t lo, int64_t count,
                        bool other, const Tensor& pq, Opt pk, Opt gq, Opt gk, at::ScalarType to) {
    const Rel r("rel_bias", lut, lo, count, other, pq, get(pk), get(gq), get(gk));
    ctx->save_for_backward({lut, r.pos_q, r.pos_k, r.group_q, r.group_k});
    ctx->saved_data["lo"] = lo;
    ctx->saved_data["count"] = count;
    ctx->saved_data["table"] = type_of(table);
    ctx->saved_data["add"] = add.has_value();
    return rel_bias(table, r, get(add), to);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    once("rel_bias");
    const variable_list s = ctx->get_saved_variables();
    variable_list d(11);
    if (ctx->needs_input_grad(0)) {
      const Rel r("rel_bias_bwd", s[0], ctx->saved_data["lo"].toInt(), ctx->saved_data["count"].toInt(), s[3].defined(), s[1],
                  s[2], s[3], s[4]);
      d[0] = as(rel_bias_bwd(g[0], r), ctx->saved_data["table"].toInt());
    }
    if (ctx->saved_data["add"].toBool()) d[1] = g[0];
    return d;
  }
};

// ------------------------------------------------------------------------------------------------ norms and rotation

// x [.., W] as rows of one pitch: itself where its leading dimensions step evenly, else a contiguous copy.
Tensor even_rows(const Tensor& x) {
  if (x.stride(-1) != 1 && x.size(-1) != 1) return x.contiguous();
  int64_t step = -1;  // the pitch times the rows of the dimensions seen so far
  for (int64_t i = x.dim() - 2; i >= 0; i--) {
    if (x.size(i) == 1) continue;
    if (step >= 0 ? x.stride(i) != step : x.stride(i) < x.size(-1)) return x.contiguous();
    step = x.stride(i) * x.size(i);
  }
  return x;
}
int64_t pitch(const Tensor& x) {  // of even_rows' result
  for (int64_t i = x.dim() - 2; i >= 0; i--)
    if (x.size(i) != 1) return x.stride(i);
  return x.size(-1);
}

struct QK {
  int64_t H, Hk, C, rows = 1, pos_rows = 0, rotary;
  double eps, base;
  bool inter, wide = false;
  Tensor pos, wq, wk;
  QK(const char* name, const Tensor& q, const Tensor& k, const Tensor& wq_, const Tensor& wk_, int64_t H_, const Tensor& pos_,
     double eps_, double base_, std::optional<int64_t> rotary_, bool inter_)
      : H(H_), eps(eps_), base(base_), inter(inter_) {
    TORCH_CHECK_VALUE(q.dim() >= 1 && q.dim() == k.dim() && H >= 1 && q.size(-1) > 0 && q.size(-1) % H == 0, name,
                      ": need q [.., H * C] and k [.., Hk * C], got ", q.sizes(), " and ", k.sizes(), " with H = ", H);
    C = q.size(-1) / H;
    TORCH_CHECK_VALUE(C % 2 == 0 && C <= 256, name, ": heads of an even 2 to 256 channels, got ", C);
    TORCH_CHECK_VALUE(k.size(-1) > 0 && k.size(-1) % C == 0 && q.sizes().slice(0, q.dim() - 1) == k.sizes().slice(0, k.dim() - 1),
                      name, ": k must have q's rows and heads of ", C, " channels, got ", k.sizes());
    TORCH_CHECK_VALUE(k.scalar_type() == q.scalar_type() && k.device() == q.device(), name, ": q and k must be of one type on one device");
    Hk = k.size(-1) / C;
    count_fits(name, "heads", H > Hk ? H : Hk);
    for (int64_t i = 0; i + 1 < q.dim(); i++) rows *= q.size(i);
    rotary = rotary_.value_or(C);
    TORCH_CHECK_VALUE(rotary >= 0 && rotary <= C && rotary % 2 == 0, name, ": rotary must be even, 0 to ", C, ", got ", rotary);
    TORCH_CHECK_VALUE(base > 0, name, ": base must be positive, got ", base);
    for (const Tensor& w : {wq_, wk_})
      TORCH_CHECK_VALUE(!w.defined() || (w.dim() == 1 && w.size(0) == C && w.device() == q.device()), name, ": weights must be [", C,
                        "] tensors on ", q.device());
    if (pos_.defined()) {
      const auto lead = q.sizes().slice(0, q.dim() - 1);
      const bool whole_rows = pos_.sizes() == lead, last = pos_.dim() == 1 && !lead.empty() && pos_.size(0) == lead.back();
      TORCH_CHECK_VALUE(whole(pos_) && (whole_rows || last) && pos_.device() == q.device(), name,
                        ": pos must hold an int32 or int64 for each row, or for each of the last ones, on ", q.device(), ", got ",
                        pos_.sizes());
      pos = pos_.contiguous();
      pos_rows = pos.numel();
      wide = pos.scalar_type() == at::kLong;
    }
    wq = param(wq_), wk = param(wk_);
  }
};

std::tuple<Tensor, Tensor> qk_norm_rope(const Tensor& q_, const Tensor& k_, const QK& a, at::ScalarType to) {
  const char* name = "qk_norm_rope";
  const int xt = type_code(q_), yt = type_code(to);
  on_gpu(name, q_);
  const OnDevice dev(q_);
  const Tensor q = even_rows(q_), k = even_rows(k_);
  const Tensor qn = at::empty(q.sizes(), q.options().dtype(to)), kn = at::empty(k.sizes(), k.options().dtype(to));
  if (a.rows)
    check(lib.qk_norm_rope(in(q), pitch(q), in(k), pitch(k), xt, f32(a.wq), f32(a.wk), (float)a.eps, in(a.pos), a.wide, a.pos_rows,
                           a.base, (int)a.rotary, a.inter, out(qn), out(kn), yt, a.rows, (int)a.H, (int)a.Hk, (int)a.C,
                           dev.stream),
          "bzpf_qk_norm_rope");
  return {qn, kn};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> qk_norm_rope_bwd(const Tensor& dqn_, const Tensor& dkn_, const Tensor& q_,
                                                            const Tensor& k_, const QK& a, bool need_wq, bool need_wk) {
  const char* name = "qk_norm_rope_bwd";
  TORCH_CHECK_VALUE(dqn_.sizes() == q_.sizes() && dkn_.sizes() == k_.sizes() && dqn_.scalar_type() == dkn_.scalar_type() &&
                        dqn_.device() == q_.device() && dkn_.device() == q_.device(),
                    name, ": the gradients must have the shapes of q and k and one type");
  const int xt = type_code(q_), yt = type_code(dqn_);
  on_gpu(name, q_);
  const OnDevice dev(q_);
  const Tensor q = even_rows(q_), k = even_rows(k_), dqn = dqn_.contiguous(), dkn = dkn_.contiguous();
  const Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
  const auto opt = q.options().dtype(at::kFloat);
  const auto grad = [&](bool need) { return !need ? Tensor() : a.rows ? at::empty({a.C}, opt) : at::zeros({a.C}, opt); };
  const Tensor dwq = grad(need_wq), dwk = grad(need_wk);
  if (a.rows) {
    const int64_t bytes = need_wq || need_wk ? lib.qk_norm_rope_bwd_ws((int)a.C) : 0;
    const Tensor ws = bytes ? at::empty({bytes / 4}, opt) : Tensor();
    check(lib.qk_norm_rope_bwd(in(dqn), in(dkn), yt, in(q), pitch(q), in(k), pitch(k), xt, f32(a.wq), f32(a.wk), (float)a.eps,
                               in(a.pos), a.wide, a.pos_rows, a.base, (int)a.rotary, a.inter, out(dq), out(dk), f32_out(dwq),
                               f32_out(dwk), f32_out(ws), bytes, a.rows, (int)a.H, (int)a.Hk, (int)a.C, dev.stream),
          "bzpf_qk_norm_rope_bwd");
  }
  return {dq, dk, dwq, dwk};
}

struct QKNormNode : torch::autograd::Function<QKNormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, Opt wq, Opt wk, int64_t H, Opt pos,
                               double eps, double base, std::optional<int64_t> rotary, bool inter, at::ScalarType to) {
    const QK a("qk_norm_rope", q, k, get(wq), get(wk), H, get(pos), eps, base, rotary, inter);
    ctx->save_for_backward({q, k, get(wq), get(wk), get(pos)});
    ctx->saved_data["H"] = H;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["base"] = base;
    ctx->saved_data["rotary"] = a.rotary;
    ctx->saved_data["inter"] = inter;
    auto [qn, kn] = qk_norm_rope(q, k, a, to);
    return {qn, kn};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    once("qk_norm_rope");
    const variable_list s = ctx->get_saved_variables();
    const QK a("qk_norm_rope_bwd", s[0], s[1], s[2], s[3], ctx->saved_data["H"].toInt(), s[4], ctx->saved_data["eps"].toDouble(),
               ctx->saved_data["base"].toDouble(), ctx->saved_data["rotary"].toInt(), ctx->saved_data["inter"].toBool());
    const bool need_wq = s[2].defined() && ctx->needs_input_grad(2);
    const bool need_wk = s[3].defined() && ctx->needs_input_grad(2 + s[2].defined());
    auto [dq, dk, dwq, dwk] = qk_norm_rope_bwd(g[0], g[1], s[0], s[1], a, need_wq, need_wk);
    variable_list d(11);
    d[0] = dq, d[1] = dk, d[2] = as(dwq, type_of(s[2])), d[3] = as(dwk, type_of(s[3]));
    return d;
  }
};

// ------------------------------------------------------------------------------------------------ attention

// An operand [S, n, H C] as the kernels take it: rows of unit stride (a copy where they are not).
Tensor operand(const Tensor& x) {
  const Tensor y = x.dim() == 2 ? x.unsqueeze(0) : x;
  return (y.stride(2) == 1 || y.size(2) == 1) && (y.size(1) == 1 || y.stride(1) >= y.size(2)) ? y : y.contiguous();
}

struct Att {
  Tensor q, k, v, g, bias, mask;
  int64_t S, H, C, N, M, mult;
  bool batched, bias4 = false;
  Att(const char* name, const Tensor& q_, const Tensor& k_, const Tensor& v_, int64_t H_, const Tensor& g_, const Tensor& bias_,
      const Tensor& mask_, int64_t mult_)
      : H(H_), mult(mult_) {
    TORCH_CHECK_VALUE((q_.dim() == 2 || q_.dim() == 3) && k_.dim() == q_.dim() && k_.sizes() == v_.sizes() && H >= 1 &&
                          q_.size(-1) > 0 && q_.size(-1) % H == 0 && k_.size(-1) == q_.size(-1) &&
                          (q_.dim() == 2 || q_.size(0) == k_.size(0)),
                      name, ": need q [(S,) N, H * C] and k, v [(S,) M, H * C], got ", q_.sizes(), ", ", k_.sizes(), " and ",
                      v_.sizes(), " with H = ", H);
    batched = q_.dim() == 3;
    S = batched ? q_.size(0) : 1, N = q_.size(-2), M = k_.size(-2), C = q_.size(-1) / H;
    TORCH_CHECK_VALUE(C % 8 == 0 && C <= 128, name, ": heads of 8 to 128 channels, a multiple of 8, got ", C);
    count_fits(name, "samples", S);
    count_fits(name, "heads", H);
    type_code(q_);
    TORCH_CHECK_VALUE(!g_.defined() || g_.sizes() == q_.sizes(), name, ": g must have q's shape");
    for (const Tensor& t : {k_, v_, g_})
      TORCH_CHECK_VALUE(!t.defined() || (t.scalar_type() == q_.scalar_type() && t.device() == q_.device()), name,
                        ": q, k, v and g must be of one type on one device");
    TORCH_CHECK_VALUE(mult >= 1 && S % mult == 0, name, ": multiplicity ", mult, " does not divide ", S, " samples");
    if (bias_.defined()) {
      bias4 = bias_.dim() == 4;
      TORCH_CHECK_VALUE((bias4 || (bias_.dim() == 3 && S == mult)) && (!bias4 || bias_.size(0) == S / mult) && bias_.size(-3) == H &&
                            bias_.size(-2) == N && bias_.size(-1) == M && bias_.device() == q_.device(),
                        name, ": bias must be [S / multiplicity, H, N, M] = [", S / mult, ", ", H, ", ", N, ", ", M, "] on ",
                        q_.device(), ", got ", bias_.sizes());
      TORCH_CHECK_TYPE(bias_.scalar_type() == q_.scalar_type() || (q_.scalar_type() == at::kFloat && type_code(bias_) >= 0), name,
                       ": bias must be of q's type, or fp16 / bf16 with fp32 q");
    }
    TORCH_CHECK_VALUE(!mask_.defined() || (mask_.scalar_type() == at::kFloat && mask_.numel() == S * M &&
                                           mask_.dim() <= 2 && mask_.dim() >= 1 && mask_.size(-1) == M && mask_.device() == q_.device()),
                      name, ": mask must be fp32 [", S, ", ", M, "] on ", q_.device());
    q = operand(q_), k = operand(k_), v = operand(v_);
    if (g_.defined()) g = operand(g_);
    if (bias_.defined()) bias = bias_.contiguous();
    if (mask_.defined()) mask = mask_.contiguous();
  }
  at::IntArrayRef shape(const Tensor& x) const { return batched ? x.sizes() : x.sizes().slice(1); }
  int bias_type() const { return bias.defined() ? type_code(bias) : type_code(q); }
};
// An operand's pointer, row pitch and sample stride (a dimension of one has any stride).
#define BZPF_ROWS(t)                                                              \
  in(t), !(t).defined() ? 0 : (t).size(1) == 1 ? (t).size(2) : (t).stride(1),     \
      !(t).defined() || (t).size(0) == 1 ? 0 : (t).stride(0)

std::tuple<Tensor, Tensor> attention(const Att& a) {
  on_gpu("attention", a.q);
  const OnDevice dev(a.q);
  const Tensor o = at::empty(a.shape(a.q), a.q.options());
  const auto opt = a.q.options().dtype(at::kFloat);
  const Tensor stats = a.batched ? at::empty({a.S, a.H, a.N, 2}, opt) : at::empty({a.H, a.N, 2}, opt);
  if (!o.numel()) return {o, stats};
  if (a.M == 0) {  // no key: as a row whose logits are all -inf
    o.zero_();
    stats.select(-1, 0).fill_(-std::numeric_limits<float>::infinity());
    stats.select(-1, 1).zero_();
    return {o, stats};
  }
  const int64_t bytes = lib.attention_ws((int)a.S, (int)a.H, (int)a.C, a.N, a.M);
  const Tensor ws = bytes > 0 ? at::empty({bytes}, a.q.options().dtype(at::kByte)) : Tensor();
  check(lib.attention(BZPF_ROWS(a.q), BZPF_ROWS(a.k), BZPF_ROWS(a.v), BZPF_ROWS(a.g), in(a.bias), a.bias_type(), (int)a.mult,
                      f32(a.mask), out(o), f32_out(stats), out(ws), bytes, type_code(a.q), (int)a.S, (int)a.H, (int)a.C, a.N, a.M, dev.stream),
        "bzpf_attention");
  return {o, stats};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> attention_bwd(const Tensor& dout_, const Att& a, const Tensor& o_,
                                                                 const Tensor& stats_, bool need_bias) {
  const char* name = "attention_bwd";
  for (const Tensor& t : {dout_, o_})
    TORCH_CHECK_VALUE(t.sizes() == a.shape(a.q) && t.scalar_type() == a.q.scalar_type() && t.device() == a.q.device(), name,
                      ": dout and out must be of q's shape and type on ", a.q.device());
  TORCH_CHECK_VALUE(stats_.scalar_type() == at::kFloat && stats_.numel() == a.S * a.H * a.N * 2 && stats_.dim() == (a.batched ? 4 : 3) &&
                        stats_.device() == a.q.device(),
                    name, ": stats must be those of the forward call");
  on_gpu(name, a.q);
  const OnDevice dev(a.q);
  const Tensor dout = dout_.contiguous(), o = o_.contiguous(), stats = stats_.contiguous();
  const Tensor dq = at::empty(a.shape(a.q), a.q.options()), dk = at::empty(a.shape(a.k), a.q.options());
  const Tensor dv = at::empty(a.shape(a.k), a.q.options()), dg = a.g.defined() ? at::empty(a.shape(a.q), a.q.options()) : Tensor();
  const Tensor db = need_bias && a.bias.defined() ? at::empty(a.bias.sizes(), a.bias.options()) : Tensor();
  if (!o.numel() || a.M == 0) {
    for (const Tensor& t : {dq, dk, dv, dg, db})
      if (t.defined()) t.zero_();
    return {dq, dk, dv, dg, db};
  }
  const int64_t bytes = lib.attention_bwd_ws(type_code(a.q), (int)a.S, (int)a.H, (int)a.C, a.N, a.M, a.g.defined());
  const Tensor ws = at::empty({bytes > 0 ? bytes : 0}, a.q.options().dtype(at::kByte));  // none for sizes that the call refuses
  check(lib.attention_bwd(in(dout), BZPF_ROWS(a.q), BZPF_ROWS(a.k), BZPF_ROWS(a.v), BZPF_ROWS(a.g), in(a.bias), a.bias_type(),
                          (int)a.mult, f32(a.mask), in(o), f32(stats), out(dq), out(dk), out(dv), out(dg), out(db), out(ws), bytes,
                          type_code(a.q), (int)a.S, (int)a.H, (int)a.C, a.N, a.M, dev.stream),
        "bzpf_attention_bwd");
  return {dq, dk, dv, dg, db};
}

struct AttentionNode : torch::autograd::Function<AttentionNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, int64_t H, Opt g, Opt bias, Opt mask,
                        int64_t mult) {
    const Att a("attention", q, k, v, H, get(g), get(bias), get(mask), mult);
    auto [o, stats] = attention(a);
    ctx->save_for_backward({q, k, v, get(g), get(bias), get(mask), o, stats});
    ctx->saved_data["H"] = H;
    ctx->saved_data["mult"] = mult;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grad) {
    once("attention");
    const variable_list s = ctx->get_saved_variables();
    const Att a("attention_bwd", s[0], s[1], s[2], ctx->saved_data["H"].toInt(), s[3], s[4], s[5], ctx->saved_data["mult"].toInt());
    const bool need_bias = s[4].defined() && ctx->needs_input_grad(3 + s[3].defined());
    auto [dq, dk, dv, dg, db] = attention_bwd(grad[0], a, s[6], s[7], need_bias);
    variable_list d(8);
    d[0] = dq, d[1] = dk, d[2] = dv, d[4] = dg, d[5] = db;
    return d;
  }
};

}  // namespace

void bind_attention(pybind11::module_& m) {
  namespace py = pybind11;
  typedef py::call_guard<py::gil_scoped_release> NoGil;
  typedef std::optional<at::ScalarType> Type;
  typedef std::optional<int64_t> Int;
  const auto bias_type = [](const Tensor& table, Opt add, Type to) {
    return to.value_or(add.has_value() ? add->scalar_type() : table.scalar_type());
  };

  m.def("rel_bias", [=](const Tensor& table, const Tensor& lut, int64_t lo, int64_t count, bool other, const Tensor& pq, Opt pk,
                        Opt gq, Opt gk, Opt add, Type to) {
    return rel_bias(table, Rel("rel_bias", lut, lo, count, other, pq, get(pk), get(gq), get(gk)), get(add),
                    bias_type(table, add, to));
  }, NoGil());
  m.def("rel_bias_bwd", [](const Tensor& dy, const Tensor& lut, int64_t lo, int64_t count, bool other, const Tensor& pq, Opt pk,
                           Opt gq, Opt gk) {
    return rel_bias_bwd(dy, Rel("rel_bias_bwd", lut, lo, count, other, pq, get(pk), get(gq), get(gk)));
  }, NoGil());
  m.def("grad_rel_bias", [=](const Tensor& table, const Tensor& lut, int64_t lo, int64_t count, bool other, const Tensor& pq,
                             Opt pk, Opt gq, Opt gk, Opt add, Type to) {
    return RelBiasNode::apply(table, add, lut, lo, count, other, pq, pk, gq, gk, bias_type(table, add, to));
  }, NoGil());
  m.def("qk_norm_rope", [](const Tensor& q, const Tensor& k, Opt wq, Opt wk, int64_t H, Opt pos, double eps, double base, Int rotary,
                           bool inter, Type to) {
    return qk_norm_rope(q, k, QK("qk_norm_rope", q, k, get(wq), get(wk), H, get(pos), eps, base, rotary, inter),
                        to.value_or(q.scalar_type()));
  }, NoGil());
  m.def("qk_norm_rope_bwd", [](const Tensor& dq, const Tensor& dk, const Tensor& q, const Tensor& k, Opt wq, Opt wk, int64_t H,
                               Opt pos, double eps, double base, Int rotary, bool inter, bool need_weights) {
    return qk_norm_rope_bwd(dq, dk, q, k, QK("qk_norm_rope_bwd", q, k, get(wq), get(wk), H, get(pos), eps, base, rotary, inter),
                            need_weights, need_weights);
  }, NoGil());
  m.def("grad_qk_norm_rope", [](const Tensor& q, const Tensor& k, Opt wq, Opt wk, int64_t H, Opt pos, double eps, double base,
                                Int rotary, bool inter, Type to) {
    const variable_list o = QKNormNode::apply(q, k, wq, wk, H, pos, eps, base, rotary, inter, to.value_or(q.scalar_type()));
    return std::make_tuple(o[0], o[1]);
  }, NoGil());
  m.def("attention", [](const Tensor& q, const Tensor& k, const Tensor& v, int64_t H, Opt g, Opt bias, Opt mask, int64_t mult) {
    return attention(Att("attention", q, k, v, H, get(g), get(bias), get(mask), mult));
  }, NoGil());
  m.def("attention_bwd", [](const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v, int64_t H, const Tensor& o,
                            const Tensor& stats, Opt g, Opt bias, Opt mask, int64_t mult, bool need_bias) {
    return attention_bwd(dout, Att("attention_bwd", q, k, v, H, get(g), get(bias), get(mask), mult), o, stats, need_bias);
  }, NoGil());
  m.def("grad_attention", [](const Tensor& q, const Tensor& k, const Tensor& v, int64_t H, Opt g, Opt bias, Opt mask, int64_t mult) {
    return AttentionNode::apply(q, k, v, H, g, bias, mask, mult);
  }, NoGil());
}

}  // namespace bzpf_torch

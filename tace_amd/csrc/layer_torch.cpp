// The routed layer's operators on torch tensors, beside rows_torch.cpp's: root-mean-square norm and the step of AdamW.
#include "rows_torch.h"

#include <algorithm>

namespace {

// ---------------------------------------------------------------------- norm ----
struct Norm {
  double eps;
  std::vector<int32_t> comps;
  int64_t rows;
  int channels;
  bool residual, timed;

  int blocks() const { return (int)comps.size(); }
};

// (y, h, factors of the rows)
struct Normed {
  Tensor y, h, inv;
};
Normed norm_rows(const Tensor& x, const Tensor& res, const Tensor& w, const Norm& a, bool want_inv) {
  Normed r{at::empty_like(x), a.residual ? at::empty_like(x) : Tensor(),
           want_inv ? at::empty({a.rows, a.blocks()}, x.options().dtype(sum_type(x))) : Tensor()};
  Launch l(x, "rms_norm_fwd", a.timed);
  l.done(tace_rms_norm_fwd(type_code(x.scalar_type()), ptr(x), ptr(res), ptr(w), w.scalar_type() == sum_type(x), a.rows,
                           a.channels, a.blocks(), a.comps.data(), a.eps, ptr(r.h), ptr(r.y), nullptr, ptr(r.inv),
                           l.stream), {x.numel()});
  return r;
}

// the gradients of h and of the weight in torch's operations, for a graph of them
std::pair<Tensor, Tensor> norm_gradients(const Tensor& gy, const Tensor& gh, const Tensor& h, const Tensor& w,
                                         const Norm& a) {
  const auto st = sum_type(h);
  const Tensor weight = w.to(st), gs = gy.to(st).reshape({-1}), hs = h.to(st).reshape({-1});
  std::vector<Tensor> dh, dw;
  int64_t at = 0;
  for (int b = 0; b < a.blocks(); ++b) {
    const int64_t d = a.comps[b], n = a.rows * d * a.channels;
    const Tensor g = gs.narrow(0, at, n).view({a.rows, d, a.channels}), hb = hs.narrow(0, at, n).view_as(g);
    const Tensor q = (hb.square().mean({1, 2}, true) + a.eps).rsqrt(), u = g * weight[b];
    dh.push_back((q * (u - hb * q.square() * (u * hb).mean({1, 2}, true))).reshape({-1}));
    dw.push_back((g * hb * q).sum(at::IntArrayRef({0, 1})));
    at += n;
  }
  Tensor dx = at::cat(dh).view(h.sizes());
  if (gh.defined()) dx = dx + gh.to(st);
  return {dx.to(h.scalar_type()), at::stack(dw).to(w.scalar_type())};
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& res, const Tensor& w,
                               const Norm& a) {
    const Normed r = norm_rows(x, res.value_or(Tensor()), w, a, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({a.residual ? r.h : x, w, r.inv});
    hold(ctx, a);
    return a.residual ? variable_list{r.y, r.h} : variable_list{r.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &h = saved[0], &w = saved[1], &inv = saved[2];
    const Norm& a = held<Norm>(ctx);
    const Tensor gh = a.residual && grads[1].defined() ? dense(grads[1]) : Tensor();
    // (edges are counted over the tensors that were given)
    const bool need_w = ctx->needs_input_grad(a.residual ? 2 : 1);
    Tensor dx, dw;
    if (!grads[0].defined()) {
      dx = gh;
      if (need_w) dw = at::zeros_like(w);
    } else {
      const Tensor gy = dense(grads[0]);
      if (a.rows == 0) {
        dx = at::empty_like(h);
        dw = at::zeros_like(w);
      } else if (tracked(gy) || tracked(gh) || tracked(h) || tracked(w)) {
        std::tie(dx, dw) = norm_gradients(gy, gh, h, w, a);
      } else {
        const int code = type_code(h.scalar_type());
        dx = at::empty_like(h);
        Tensor work;
        int64_t bytes = 0;
        if (need_w) {
          dw = at::empty_like(w);
          bytes = tace_rms_norm_bwd_work(code, a.rows, a.channels, a.blocks(), a.comps.data());
          work = at::empty({bytes}, h.options().dtype(at::kByte));
        }
        Launch l(h, "rms_norm_bwd", a.timed);
        l.done(tace_rms_norm_bwd(code, ptr(gy), ptr(gh), ptr(h), ptr(w), w.scalar_type() == sum_type(h), ptr(inv),
                                 a.rows, a.channels, a.blocks(), a.comps.data(), ptr(dx), ptr(dw), ptr(work), bytes,
                                 l.stream), {h.numel()});
      }
    }
    return {dx, a.residual ? dx : Tensor(), dw, Tensor()};
  }
};

// checks the arguments of both norms; x, weight and residual as the kernels read them
Norm norm_arguments(Tensor& x, Tensor& w, double eps, optional<Tensor>& residual,
                    const std::vector<int64_t>& components, bool timed) {
  want_rows(x, "x");
  Norm a{eps, {}, 0, 0, residual.has_value(), timed};
  bool ok = !components.empty() && components.size() <= TACE_ROW_MAX_BLOCKS;
  int64_t total = 0;
  for (int64_t c : components) {
    ok = ok && c >= 1 && c <= 1024;
    a.comps.push_back((int32_t)c);
    total += c;
  }
  TORCH_CHECK_VALUE(ok, "rms_norm: components ", components, " are not 1 to ", TACE_ROW_MAX_BLOCKS,
                    " blocks of 1 to 1024");
  TORCH_CHECK_VALUE(eps >= 0, "rms_norm: eps = ", eps, " is negative");
  const bool plain = components.size() == 1 && components[0] == 1;
  TORCH_CHECK_VALUE((plain ? x.dim() >= 1 : x.dim() == 2) && x.size(-1) >= 1 && x.size(-1) % total == 0,
                    "x has shape ", x.sizes(), ", expected [", plain ? "..." : "rows", ", ", total, " C]");
  const int64_t C = x.size(-1) / total;
  for (int64_t c : components)
    TORCH_CHECK_VALUE(c * C <= MAX_ROW, "rms_norm: a row of ", c * C, " elements, at most ", MAX_ROW);
  a.channels = (int)C;
  a.rows = x.numel() / x.size(-1);
  TORCH_CHECK_VALUE(a.rows <= MAX_INDEX, "rms_norm: rows exceed 32-bit indices");
  const int64_t B = (int64_t)components.size();
  TORCH_CHECK_VALUE((w.scalar_type() == x.scalar_type() || w.scalar_type() == sum_type(x)) &&
                    ((B == 1 && w.dim() == 1 && w.size(0) == C) || (w.dim() == 2 && w.size(0) == B && w.size(1) == C)),
                    "weight is ", w.scalar_type(), " ", w.sizes(), ", expected ", x.scalar_type(), " or ", sum_type(x),
                    " [", B, ", ", C, "]", B == 1 ? " or [C]" : "");
  want_device(w, x, "weight");
  if (residual) {
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type(), "residual is ",
                      residual->scalar_type(), " ", residual->sizes(), ", expected ", x.scalar_type(), " ", x.sizes());
    want_device(*residual, x, "residual");
    residual = dense(*residual);
  }
  x = dense(x);
  w = dense(w.dim() == 1 ? w.unsqueeze(0) : w);
  return a;
}

std::vector<Tensor> rms_norm(Tensor x, Tensor weight, double eps, optional<Tensor> residual,
                             const std::vector<int64_t>& components, bool timed) {
  const Norm a = norm_arguments(x, weight, eps, residual, components, timed);
  const Tensor res = residual.value_or(Tensor());
  if (tracked(x) || tracked(res) || tracked(weight)) return RmsNorm::apply(x, residual, weight, a);
  const Normed r = norm_rows(x, res, weight, a, false);
  return a.residual ? std::vector<Tensor>{r.y, r.h} : std::vector<Tensor>{r.y};
}

std::vector<Tensor> rms_norm_e4m3(Tensor x, Tensor weight, double eps, optional<Tensor> residual,
                                  const std::vector<int64_t>& components, bool timed) {
  TORCH_CHECK_VALUE(x.scalar_type() != at::kDouble, "rms_norm_e4m3: x has dtype Double, expected float32, bfloat16 or "
                    "float16");
  const Norm a = norm_arguments(x, weight, eps, residual, components, timed);
  const Tensor res = residual.value_or(Tensor());
  TORCH_CHECK_VALUE(!tracked(x) && !tracked(res) && !tracked(weight), "rms_norm_e4m3 has no gradient: call it under "
                    "torch.no_grad()");
  Tensor q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
  Tensor scales = at::empty({a.rows, a.blocks()}, x.options().dtype(at::kFloat));
  Tensor h = a.residual ? at::empty_like(x) : Tensor();
  Launch l(x, "rms_norm_fwd", timed);
  l.done(tace_rms_norm_fwd(type_code(x.scalar_type()), ptr(x), ptr(res), ptr(weight),
                           weight.scalar_type() == sum_type(x), a.rows, a.channels, a.blocks(), a.comps.data(), a.eps,
                           ptr(h), q.data_ptr(), scales.data_ptr<float>(), nullptr, l.stream), {x.numel()});
  return a.residual ? std::vector<Tensor>{q, scales, h} : std::vector<Tensor>{q, scales};
}

// ------------------------------------------------------------------- experts ----
struct Experts {
  Pinned rowptr;
  int64_t rows, experts;
  std::vector<int32_t> comps;
  int64_t total;   // components
  int64_t K, N;
  double scale;
  bool timed, flat;   // flat: weights [E, K, N]

  int blocks() const { return (int)comps.size(); }
  const int32_t* starts() const { return rowptr.get("plan.rowptr").data_ptr<int>(); }
};

Tensor expert_rows(bool transposed, const Tensor& x, const Tensor& w, const Experts& a) {
  Tensor out = at::empty({a.rows, a.total * (transposed ? a.K : a.N)}, x.options());
  Launch l(x, "expert_linear", a.timed);
  l.done(tace_expert_linear(type_code(x.scalar_type()), transposed, ptr(x), ptr(w), a.starts(), a.rows, (int)a.experts,
                            a.blocks(), a.comps.data(), (int)a.K, (int)a.N, a.scale, ptr(out), l.stream),
         {a.rows, a.total, a.K, a.N});
  return out;
}

Tensor expert_weights(const Tensor& x, const Tensor& g, const Experts& a) {
  Tensor dw = a.flat ? at::empty({a.experts, a.K, a.N}, x.options())
                     : at::empty({a.experts, a.blocks(), a.K, a.N}, x.options()), work;
  const int code = type_code(x.scalar_type());
  const int64_t bytes = tace_expert_linear_grad_work(code, a.rows, (int)a.experts, a.blocks(), a.comps.data(), (int)a.K,
                                                     (int)a.N);
  if (bytes > 0) work = at::empty({bytes}, x.options().dtype(at::kByte));
  Launch l(x, "expert_linear_grad", a.timed);
  l.done(tace_expert_linear_grad(code, ptr(x), ptr(g), a.starts(), a.rows, (int)a.experts, a.blocks(), a.comps.data(),
                                 (int)a.K, (int)a.N, a.scale, ptr(dw), ptr(work), bytes, l.stream),
         {a.rows, a.total, a.K, a.N});
  return dw;
}

// L(x, w) = s x w, T(g, w) = s g w^T and G(x, g) = s x^T g by expert are bilinear and each other's derivatives
Tensor rows_op(bool transposed, const Tensor& x, const Tensor& w, const Experts& a);
Tensor weights_op(const Tensor& x, const Tensor& g, const Experts& a);

template <bool TRANSPOSED>
struct ExpertRows : torch::autograd::Function<ExpertRows<TRANSPOSED>> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Experts& a) {
    ctx->save_for_backward({x, w});
    hold(ctx, a);
    return expert_rows(TRANSPOSED, x, w, a);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Experts& a = held<Experts>(ctx);
    const Tensor c = dense(grads[0]);
    variable_list out(3);
    if (ctx->needs_input_grad(0)) out[0] = rows_op(!TRANSPOSED, c, saved[1], a);
    if (ctx->needs_input_grad(1)) out[1] = TRANSPOSED ? weights_op(c, saved[0], a) : weights_op(saved[0], c, a);
    return out;
  }
};

struct ExpertWeights : torch::autograd::Function<ExpertWeights> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& g, const Experts& a) {
    ctx->save_for_backward({x, g});
    hold(ctx, a);
    return expert_weights(x, g, a);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Experts& a = held<Experts>(ctx);
    const Tensor v = dense(grads[0]);
    variable_list out(3);
    if (ctx->needs_input_grad(0)) out[0] = rows_op(true, saved[1], v, a);
    if (ctx->needs_input_grad(1)) out[1] = rows_op(false, saved[0], v, a);
    return out;
  }
};

Tensor rows_op(bool transposed, const Tensor& x, const Tensor& w, const Experts& a) {
  if (!tracked(x) && !tracked(w)) return expert_rows(transposed, x, w, a);
  return transposed ? ExpertRows<true>::apply(x, w, a) : ExpertRows<false>::apply(x, w, a);
}
Tensor weights_op(const Tensor& x, const Tensor& g, const Experts& a) {
  return tracked(x) || tracked(g) ? ExpertWeights::apply(x, g, a) : expert_weights(x, g, a);
}

void want_rowptr(const Tensor& rowptr, const Tensor& like, int64_t rows) {
  TORCH_CHECK_VALUE(rowptr.dim() == 1 && rowptr.numel() >= 1, "plan.rowptr is empty");
  want_int32(rowptr, rowptr.numel(), like, "plan.rowptr");
  TORCH_CHECK_VALUE(rows >= 0 && rows <= MAX_INDEX, "expert_linear: rows exceed 32-bit indices");
}

Tensor expert_linear(const Tensor& x, const Tensor& weight, const Tensor& rowptr, int64_t rows, double scale,
                     const std::vector<int64_t>& components, bool timed) {
  want_rows(x, "x");
  want_rowptr(rowptr, x, rows);
  Experts a{rowptr, rows, rowptr.numel() - 1, {}, 0, 0, 0, scale, timed, weight.dim() == 3};
  bool ok = !components.empty() && components.size() <= TACE_ROW_MAX_BLOCKS;
  for (int64_t c : components) {
    ok = ok && c >= 1 && c <= 1024;
    a.comps.push_back((int32_t)c);
    a.total += c;
  }
  TORCH_CHECK_VALUE(ok, "expert_linear: components ", components, " are not 1 to ", TACE_ROW_MAX_BLOCKS,
                    " blocks of 1 to 1024");
  const int64_t B = a.blocks();
  TORCH_CHECK_VALUE(weight.scalar_type() == x.scalar_type() &&
                    ((B == 1 && weight.dim() == 3) || (weight.dim() == 4 && weight.size(1) == B)) &&
                    weight.size(0) == a.experts,
                    "weight is ", weight.scalar_type(), " ", weight.sizes(), ", expected ", x.scalar_type(), " [",
                    a.experts, ", ", B, ", K, N]", B == 1 ? " or [E, K, N]" : "");
  want_device(weight, x, "weight");
  a.K = weight.size(-2);
  a.N = weight.size(-1);
  TORCH_CHECK_VALUE(a.K >= 1 && a.K <= 65536 && a.N >= 1 && a.N <= 65536, "weight has shape ", weight.sizes(),
                    ", expected K and N of 1 to 65536");
  TORCH_CHECK_VALUE(x.dim() == 2 && x.size(0) == rows && x.size(1) == a.total * a.K, "x has shape ", x.sizes(),
                    ", expected [", rows, ", ", a.total * a.K, "]");
  return rows_op(false, dense(x), dense(weight), a);
}

Tensor expert_linear_e4m3(const Tensor& q, const Tensor& q_scale, const Tensor& w, const Tensor& w_scale,
                          const Tensor& rowptr, const Tensor& order, int64_t tokens, int64_t k, bool gather,
                          at::ScalarType out_type, bool timed) {
  const int64_t rows = tokens * k, from = gather ? tokens : rows, E = rowptr.numel() - 1;
  TORCH_CHECK_VALUE(q.is_cuda(), "q must be a GPU tensor (got ", q.device(), ")");
  want_memory(q, "q");
  want_rowptr(rowptr, q, rows);
  if (gather) want_int32(order, rows, q, "plan.order");
  TORCH_CHECK_VALUE(out_type == at::kFloat || out_type == at::kBFloat16 || out_type == at::kHalf,
                    "expert_linear_e4m3: out_dtype ", out_type, ", expected float32, bfloat16 or float16");
  TORCH_CHECK_VALUE(w.scalar_type() == at::kFloat8_e4m3fn && w.dim() == 3 && w.size(0) == E && w.size(1) >= 1 &&
                    w.size(1) <= 65536 && w.size(2) >= 16 && w.size(2) <= 65536 && w.size(2) % 16 == 0, "weight is ",
                    w.scalar_type(), " ", w.sizes(), ", expected float8_e4m3fn [", E, ", N, K], K a multiple of 16");
  const int64_t N = w.size(1), K = w.size(2);
  TORCH_CHECK_VALUE(q.scalar_type() == at::kFloat8_e4m3fn && q.dim() == 2 && q.size(0) == from && q.size(1) == K, "q is ",
                    q.scalar_type(), " ", q.sizes(), ", expected float8_e4m3fn [", from, ", ", K, "]");
  TORCH_CHECK_VALUE(q_scale.scalar_type() == at::kFloat && q_scale.dim() >= 1 && q_scale.numel() == from &&
                    q_scale.size(0) == from,
                    "q_scale is ", q_scale.scalar_type(), " ", q_scale.sizes(), ", expected float32 [", from, "]");
  TORCH_CHECK_VALUE(w_scale.scalar_type() == at::kFloat && w_scale.dim() == 2 && w_scale.size(0) == E &&
                    w_scale.size(1) == N, "w_scale is ", w_scale.scalar_type(), " ", w_scale.sizes(),
                    ", expected float32 [", E, ", ", N, "]");
  want_device(w, q, "weight");
  want_device(q_scale, q, "q_scale");
  want_device(w_scale, q, "w_scale");
  TORCH_CHECK_VALUE(!tracked(q_scale) && !tracked(w_scale), "expert_linear_e4m3 has no gradient: call it under "
                    "torch.no_grad()");
  // (a view of codes may begin anywhere: 16-byte loads need a copy)
  auto codes = [](const Tensor& t) {
    const Tensor c = t.contiguous();
    return c.numel() && (uintptr_t)c.const_data_ptr() % 16 ? c.clone() : c;
  };
  const Tensor x = codes(q), wt = codes(w), xs = dense(q_scale), ws = dense(w_scale);
  Tensor out = at::empty({rows, N}, q_scale.options().dtype(out_type).requires_grad(false));
  Launch l(q, "expert_linear_e4m3", timed);
  l.done(tace_expert_linear_e4m3(type_code(out_type), x.const_data_ptr(), xs.const_data_ptr<float>(),
                                 gather ? order.const_data_ptr<int>() : nullptr, (int)k, wt.const_data_ptr(),
                                 ws.const_data_ptr<float>(), rowptr.const_data_ptr<int>(), rows, (int)E, (int)K, (int)N,
                                 out.data_ptr(), l.stream), {rows, K, N});
  return out;
}

// --------------------------------------------------------------------- AdamW ----
typedef std::vector<Tensor> Tensors;

void want_state(const Tensor& t, const Tensor& p, at::ScalarType type, const char* name, size_t i) {
  TORCH_CHECK_VALUE(t.scalar_type() == type && t.sizes() == p.sizes() && t.is_contiguous() && !t.is_neg(), name, "[", i,
                    "] is ", t.scalar_type(), " ", t.sizes(), ", expected a contiguous ", type, " ", p.sizes());
  want_device(t, p, name);
}

void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// gradients as the kernels read them (kept alive by `held`)
Tensor gradient_of(const Tensor& g, const Tensor& like, Tensors& held, size_t i) {
  TORCH_CHECK_VALUE(g.layout() == at::kStrided && g.scalar_type() == like.scalar_type() && g.sizes() == like.sizes(),
                    "grads[", i, "] is ", g.scalar_type(), " ", g.sizes(), ", expected ", like.scalar_type(), " ",
                    like.sizes());
  want_device(g, like, "grads");
  if (g.is_contiguous() && !g.is_neg()) return g;
  held.push_back(dense(g));
  return held.back();
}

Tensor norm_of(const std::vector<tace_adam_tensor>& table, const Tensor& like, int64_t* ticket, bool timed) {
  Tensor norm = at::empty({}, like.options().dtype(sum_type(like)).requires_grad(false));
  const int64_t bytes = tace_grad_norm_work(table.data(), (int64_t)table.size());
  Tensor work = at::empty({bytes}, norm.options().dtype(at::kByte));
  Launch l(like, "grad_norm", timed);
  l.done(tace_grad_norm(type_code(like.scalar_type()), table.data(), (int64_t)table.size(), ticket, norm.data_ptr(),
                        ptr(work), bytes, l.stream), {(int64_t)table.size()});
  return norm;
}

Tensor grad_norm(const Tensors& grads, bool timed) {
  TORCH_CHECK_VALUE(!grads.empty(), "grad_norm: no gradients");
  want_rows(grads[0], "grads[0]");
  Tensors held;
  std::vector<tace_adam_tensor> table;
  int64_t total = 0;
  for (size_t i = 0; i < grads.size(); ++i) {
    TORCH_CHECK_VALUE(grads[i].scalar_type() == grads[0].scalar_type(), "grads[", i, "] is ", grads[i].scalar_type(),
                      ", expected ", grads[0].scalar_type());
    table.push_back({nullptr, gradient_of(grads[i], grads[i], held, i).const_data_ptr(), nullptr, nullptr, nullptr,
                     nullptr, grads[i].numel()});
    TORCH_CHECK_VALUE(grads[i].device() == grads[0].device(), "grads[", i, "] is on ", grads[i].device(), ", expected ",
                      grads[0].device());
    total += grads[i].numel();
  }
  const auto opt = grads[0].options().requires_grad(false);
  if (total == 0) return at::zeros({}, opt.dtype(sum_type(grads[0])));
  Tensor ticket = at::zeros({1}, opt.dtype(at::kLong));
  return norm_of(table, grads[0], ticket.data_ptr<int64_t>(), timed);
}

// What a step writes shares no memory, and none with what it reads.
void want_apart(const std::vector<tace_adam_tensor>& table, at::ScalarType type, at::ScalarType wide, bool eight) {
  typedef std::pair<uintptr_t, uintptr_t> Span;   // first byte, end
  std::vector<Span> written;
  written.reserve(table.size() * 4);
  const int64_t b = (int64_t)c10::elementSize(type), state = eight ? 1 : (int64_t)c10::elementSize(wide);
  auto add = [&](const void* p, int64_t bytes) {
    if (p && bytes) written.emplace_back((uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes);
  };
  for (const auto& t : table) {
    add(t.p, t.n * b);
    add(t.m, t.n * state);
    add(t.s, t.n * state);
    add(t.master, t.n * 4);
    add(t.scales, (t.n + TACE_ADAM_BLOCK - 1) / TACE_ADAM_BLOCK * 8);
  }
  std::sort(written.begin(), written.end());
  for (size_t i = 1; i < written.size(); ++i)
    TORCH_CHECK_VALUE(written[i - 1].second <= written[i].first,
                      "adamw_step: parameters or states overlap (or one is given twice)");
  for (const auto& t : table) {
    if (t.n == 0) continue;
    const uintptr_t g = (uintptr_t)t.g;
    const auto after = std::lower_bound(written.begin(), written.end(), Span(g + (uintptr_t)(t.n * b), 0));
    TORCH_CHECK_VALUE(after == written.begin() || std::prev(after)->second <= g,
                      "adamw_step: a gradient overlaps a parameter or state");
  }
}

optional<Tensor> adamw_step(const Tensors& params, const Tensors& grads, const Tensors& ms, const Tensors& ss,
                            const Tensor& counter, double lr, const optional<Tensor>& lr_at, double beta1, double beta2,
                            double eps, double decay, const optional<Tensors>& scales,
                            const optional<Tensors>& masters, optional<double> max_norm, const optional<Tensor>& norm_in,
                            int64_t seed, const optional<std::vector<int64_t>>& places, bool timed) {
  const size_t n = params.size();
  TORCH_CHECK_VALUE(n > 0, "adamw_step: no parameters");
  TORCH_CHECK_VALUE(grads.size() == n && ms.size() == n && ss.size() == n && (!scales || scales->size() == n) &&
                    (!masters || masters->size() == n), "adamw_step: lists of different lengths");
  const Tensor& first = params[0];
  want_rows(first, "params[0]");
  const auto type = first.scalar_type(), wide = sum_type(first);
  TORCH_CHECK_VALUE(!scales || type != at::kDouble, "adamw_step: float64 parameters have no states of 8 bits");
  TORCH_CHECK_VALUE(!masters || (type != at::kDouble && type != at::kFloat),
                    "adamw_step: parameters of 16 bits have masters");
  TORCH_CHECK_VALUE(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, "adamw_step: betas (", beta1, ", ", beta2,
                    ") are not in [0, 1)");
  TORCH_CHECK_VALUE(eps >= 0 && decay >= 0 && (lr_at || lr >= 0), "adamw_step: lr, eps and weight_decay are not negative");
  TORCH_CHECK_VALUE(!max_norm || *max_norm > 0, "adamw_step: max_norm is not positive");
  TORCH_CHECK_VALUE(!norm_in || max_norm, "adamw_step: a norm without max_norm");
  if (places) {
    bool ok = places->size() == n && places->front() >= 0 && places->back() < (1 << 20);
    for (size_t i = 1; i < places->size(); ++i) ok = ok && (*places)[i - 1] < (*places)[i];
    TORCH_CHECK_VALUE(ok, "adamw_step: places are one for each parameter, each larger than the one before, below 2^20");
  }
  TORCH_CHECK_VALUE(counter.scalar_type() == at::kLong && counter.dim() == 1 && counter.size(0) == 2 &&
                    counter.is_contiguous() && !counter.is_neg(), "counter must be a contiguous int64 tensor [2]");
  want_device(counter, first, "counter");
  if (lr_at) {
    TORCH_CHECK_VALUE(lr_at->numel() == 1 && (lr_at->scalar_type() == at::kFloat || lr_at->scalar_type() == at::kDouble)
                      && !lr_at->is_neg(), "lr must be a number or a float32 or float64 tensor of one element");
    want_device(*lr_at, first, "lr");
  }
  Tensors held;
  std::vector<tace_adam_tensor> table(n);
  int64_t total = 0;
  for (size_t i = 0; i < n; ++i) {
    const Tensor& p = params[i];
    TORCH_CHECK_VALUE(p.scalar_type() == type && p.is_contiguous() && !p.is_neg(), "params[", i, "] is ", p.scalar_type(),
                      " ", p.sizes(), ", expected a contiguous ", type);
    want_device(p, first, "params");
    want_state(ms[i], p, scales ? at::kFloat8_e4m3fn : wide, "exp_avgs", i);
    want_state(ss[i], p, scales ? at::kFloat8_e4m3fn : wide, "exp_avg_sqs", i);
    const int64_t count = p.numel();
    if (scales) {
      const Tensor& s = (*scales)[i];
      const int64_t blocks = (count + TACE_ADAM_BLOCK - 1) / TACE_ADAM_BLOCK;
      TORCH_CHECK_VALUE(s.scalar_type() == at::kFloat && s.dim() == 2 && s.size(0) == blocks && s.size(1) == 2 &&
                        s.is_contiguous() && !s.is_neg() && (uintptr_t)s.const_data_ptr() % 8 == 0, "scales[", i,
                        "] must be a contiguous float32 tensor [", blocks, ", 2] at a multiple of 8 bytes");
      want_device(s, p, "scales");
    }
    if (masters) want_state((*masters)[i], p, at::kFloat, "masters", i);
    const Tensor g = gradient_of(grads[i], p, held, i);
    table[i] = {p.data_ptr(), g.const_data_ptr(), ms[i].data_ptr(), ss[i].data_ptr(),
                masters ? (*masters)[i].data_ptr() : nullptr, scales ? (*scales)[i].data_ptr() : nullptr, count};
    total += count;
  }
  want_apart(table, type, wide, scales.has_value());
  if (total == 0) return max_norm ? optional<Tensor>(at::zeros({}, first.options().dtype(wide).requires_grad(false)))
                                  : std::nullopt;
  Tensor norm;
  if (norm_in) {
    TORCH_CHECK_VALUE(norm_in->numel() == 1 && norm_in->scalar_type() == wide && !norm_in->is_neg(),
                      "norm must be a tensor of one ", wide);
    want_device(*norm_in, first, "norm");
    norm = *norm_in;
  } else if (max_norm) {
    norm = norm_of(table, first, counter.data_ptr<int64_t>() + 1, timed);
  }
  if (places && scales) {   // (draws are numbered by the table's rows: empty ones between)
    std::vector<tace_adam_tensor> spread((size_t)places->back() + 1);
    for (size_t i = 0; i < n; ++i) spread[(size_t)(*places)[i]] = table[i];
    table = std::move(spread);
  }
  {
    Launch l(first, "adamw", timed);
    l.done(tace_adamw(type_code(type), scales.has_value(), table.data(), (int64_t)table.size(), counter.data_ptr<int64_t>(), lr,
                      lr_at ? lr_at->const_data_ptr() : nullptr, lr_at && lr_at->scalar_type() == at::kDouble, beta1,
                      beta2, eps, decay, norm.defined() ? norm.const_data_ptr() : nullptr, max_norm.value_or(0),
                      (uint64_t)seed, l.stream), {total});
  }
  for (size_t i = 0; i < n; ++i) {
    written(params[i]);
    written(ms[i]);
    written(ss[i]);
    if (scales) written((*scales)[i]);
    if (masters) written((*masters)[i]);
  }
  written(counter);
  return maybe(norm);
}

}  // namespace

void bind_layer(py::module_& mod) {
  mod.def("rms_norm", torch::wrap_pybind_function(rms_norm));
  mod.def("rms_norm_e4m3", torch::wrap_pybind_function(rms_norm_e4m3));
  mod.def("expert_linear", torch::wrap_pybind_function(expert_linear));
  mod.def("expert_linear_e4m3", torch::wrap_pybind_function(expert_linear_e4m3));
  mod.def("grad_norm", torch::wrap_pybind_function(grad_norm));
  mod.def("adamw_step", torch::wrap_pybind_function(adamw_step));
}

// The row operators on torch tensors: argument checks, outputs and workspaces
// from torch's allocator, launches on torch's current stream of the tensors'
// device, and autograd nodes whose backward is made of the same operators (so
// each differentiates any number of times).
//
// Host time, not the kernels, is what small calls take: with the nodes in
// Python a forward and backward of dropout on [1024, 128] took 157 us (45 of
// them Python in the forward, 95 in the backward's thread).
#include "rows_torch.h"

namespace {

// positions grouped by key: rowptr [n_keys + 1], order [n] and, where wanted, place [n]
struct Groups {
  Tensor rowptr, order, place;
};
Groups group(const Tensor& keys, int64_t n_keys, bool want_place, bool timed) {
  const int64_t n = keys.numel();
  const auto opt = keys.options().dtype(at::kInt);
  Groups g{at::empty({n_keys + 1}, opt), at::empty({n}, opt), want_place ? at::empty({n}, opt) : Tensor()};
  Tensor work = at::empty({tace_route_group_work(n, n_keys)}, opt);
  Launch l(keys, "route_group", timed);
  l.done(tace_route_group((int)keys.element_size(), ptr(keys), n ? keys.stride(0) : 1, n, n_keys, ints(g.rowptr),
                          ints(g.order), ints(g.place), work.data_ptr<int>(), l.stream), {n, n_keys});
  return g;
}

// ----------------------------------------------------------------- embedding ----
struct Lookup {
  int64_t vocab;
  double scale;
  Pinned rowptr, order;   // the tokens' grouping, where the caller gave it
  bool timed;
};

Tensor embed_rows(const Tensor& table, const Tensor& tokens, const Lookup& a) {
  Tensor out = at::empty({tokens.numel(), table.size(1)}, table.options());
  Launch l(table, "embed_fwd", a.timed);
  l.done(tace_embed_fwd(type_code(table.scalar_type()), (int)tokens.element_size(), ptr(table), ptr(tokens),
                        tokens.numel(), a.vocab, (int)table.size(1), a.scale, ptr(out), l.stream),
         {tokens.numel(), table.size(1)});
  return out;
}

Tensor embed_grad(const Tensor& g, const Tensor& tokens, const Lookup& a) {
  const int64_t n = tokens.numel(), C = g.size(1);
  if (n == 0) return at::zeros({a.vocab, C}, g.options());
  const int code = type_code(g.scalar_type());
  Tensor grad = at::empty({a.vocab, C}, g.options()), rowptr, order, work;
  if (a.order.t.defined()) {
    rowptr = a.rowptr.get("groups[0]");
    order = a.order.get("groups[1]");
  } else if (tace_embed_grad_grouped(n, a.vocab)) {
    const Groups by = group(tokens, a.vocab, false, a.timed);
    rowptr = by.rowptr;
    order = by.order;
  }
  const int64_t bytes = tace_embed_grad_work(code, n, a.vocab, (int)C, order.defined());
  if (bytes > 0) work = at::empty({bytes}, g.options().dtype(at::kByte));
  Launch l(g, "embed_grad", a.timed);
  l.done(tace_embed_grad(code, (int)tokens.element_size(), ptr(g), ptr(tokens), ints(order), ints(rowptr), n, a.vocab,
                         (int)C, a.scale, ptr(grad), ptr(work), bytes, l.stream), {n, a.vocab, C});
  return grad;
}

struct EmbeddingGrad;
struct Embedding : torch::autograd::Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& tokens, const Lookup& a) {
    ctx->save_for_backward({tokens});
    hold(ctx, a);
    return embed_rows(table, tokens, a);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads);
};

struct EmbeddingGrad : torch::autograd::Function<EmbeddingGrad> {
  static Tensor forward(AutogradContext* ctx, const Tensor& g, const Tensor& tokens, const Lookup& a) {
    ctx->save_for_backward({tokens});
    hold(ctx, a);
    return embed_grad(g, tokens, a);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor g = dense(grads[0]), tokens = ctx->get_saved_variables()[0];
    const Lookup& a = held<Lookup>(ctx);
    return {tracked(g) ? Embedding::apply(g, tokens, a) : embed_rows(g, tokens, a), Tensor(), Tensor()};
  }
};

variable_list Embedding::backward(AutogradContext* ctx, variable_list grads) {
  const Tensor g = dense(grads[0]), tokens = ctx->get_saved_variables()[0];
  const Lookup& a = held<Lookup>(ctx);
  return {tracked(g) ? EmbeddingGrad::apply(g, tokens, a) : embed_grad(g, tokens, a), Tensor(), Tensor()};
}

Tensor embedding(const Tensor& table, const Tensor& tokens, double scale, const optional<Tensor>& rowptr,
                 const optional<Tensor>& order, bool timed) {
  want_rows(table, "table");
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(1) >= 1 && table.size(1) <= MAX_ROW, "table has shape ",
                    table.sizes(), ", expected [V, C] with C of 1 to ", MAX_ROW);
  want_indices(tokens, "tokens");
  want_device(tokens, table, "tokens");
  const int64_t n = tokens.numel(), V = table.size(0);
  TORCH_CHECK_VALUE(n <= MAX_INDEX && V <= MAX_INDEX, "embedding: tokens or table rows exceed 32-bit indices");
  Lookup a{V, scale, {}, {}, timed};
  TORCH_CHECK_VALUE(rowptr.has_value() == order.has_value(), "groups: one of (rowptr, order) is None");
  if (order) {
    want_int32(*rowptr, V + 1, table, "groups[0] (rowptr)");
    want_int32(*order, n, table, "groups[1] (order)");
    a.rowptr = *rowptr;
    a.order = *order;
  }
  const Tensor tab = dense(table), flat = dense(tokens.reshape({-1}));
  const Tensor out = tracked(tab) ? Embedding::apply(tab, flat, a) : embed_rows(tab, flat, a);
  if (tokens.dim() == 1) return out;
  auto shape = tokens.sizes().vec();
  shape.push_back(table.size(1));
  return out.view(shape);
}

// ------------------------------------------------------------------- routing ----
struct Routed {
  Pinned place, rowptr;
  int64_t tokens;
  int k;
  std::vector<int64_t> widths;
  bool timed;

  const int32_t* places() const { return place.get("plan.place").data_ptr<int>(); }
  const int32_t* end() const { return rowptr.get("plan.rowptr").data_ptr<int>() + (rowptr.t.numel() - 1); }
};

Tensor dispatch_rows(const Tensor& x, const Tensor& w, const Routed& r) {
  Tensor out = at::empty({r.tokens * r.k, x.size(1)}, x.options());
  Launch l(x, "route_dispatch", r.timed);
  l.done(tace_route_dispatch(type_code(x.scalar_type()), ptr(x), ptr(w), r.places(), r.end(), r.tokens, r.k,
                             (int)r.widths.size(), r.widths.data(), ptr(out), l.stream), {r.tokens, r.k, x.size(1)});
  return out;
}

Tensor combine_rows(const Tensor& y, const Tensor& w, const Routed& r) {
  Tensor out = at::empty({r.tokens, y.size(1)}, y.options());
  Launch l(y, "route_combine", r.timed);
  l.done(tace_route_combine(type_code(y.scalar_type()), ptr(y), ptr(w), r.places(), r.end(), r.tokens, r.k,
                            (int)r.widths.size(), r.widths.data(), ptr(out), l.stream), {r.tokens, r.k, y.size(1)});
  return out;
}

// (as dispatch_rows of x by w where want_rows, <x row, y row> per slot)
std::pair<Tensor, Tensor> dots_of(const Tensor& x, const Tensor& y, const Tensor& w, const Routed& r, bool want) {
  Tensor gy = want ? at::empty_like(y) : Tensor();
  Tensor dots = at::empty({r.tokens, r.k}, x.options().dtype(sum_type(x)));
  Launch l(x, "route_dots", r.timed);
  l.done(tace_route_dots(type_code(x.scalar_type()), ptr(x), ptr(y), ptr(w), r.places(), r.end(), r.tokens, r.k,
                         (int)r.widths.size(), r.widths.data(), ptr(gy), ptr(dots), l.stream),
         {r.tokens, r.k, x.size(1)});
  return {gy, dots};
}

// The three of them are bilinear and each other's derivatives:
// D(x, w)[place[s]] = w_s x[t(s)],  C(y, w)[t] = sum_s w_s y[place[s]],
// P(x, y)[s] = <x[t(s)], y[place[s]]>
Tensor dispatch_op(const Tensor& x, const Tensor& w, const Routed& r);
Tensor combine_op(const Tensor& y, const Tensor& w, const Routed& r);
Tensor dots_op(const Tensor& x, const Tensor& y, const Routed& r);

struct Dispatch : torch::autograd::Function<Dispatch> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& w, const Routed& r) {
    ctx->save_for_backward({w ? x : Tensor(), w.value_or(Tensor())});
    hold(ctx, r);
    return dispatch_rows(x, w.value_or(Tensor()), r);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Routed& r = held<Routed>(ctx);
    const Tensor g = dense(grads[0]), &x = saved[0], &w = saved[1];
    variable_list out(3);
    if (ctx->needs_input_grad(0)) out[0] = combine_op(g, w, r);
    if (w.defined() && ctx->needs_input_grad(1)) out[1] = dots_op(x, g, r);
    return out;
  }
};

struct Combine : torch::autograd::Function<Combine> {
  static Tensor forward(AutogradContext* ctx, const Tensor& y, const optional<Tensor>& w, const Routed& r) {
    ctx->save_for_backward({w ? y : Tensor(), w.value_or(Tensor())});
    hold(ctx, r);
    return combine_rows(y, w.value_or(Tensor()), r);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Routed& r = held<Routed>(ctx);
    const Tensor g = dense(grads[0]), &y = saved[0], &w = saved[1];
    const bool need_y = ctx->needs_input_grad(0), need_w = w.defined() && ctx->needs_input_grad(1);
    variable_list out(3);
    if (need_w && !tracked(g) && !tracked(y) && !tracked(w)) {   // both in one pass
      std::tie(out[0], out[1]) = dots_of(g, y, w, r, need_y);
      return out;
    }
    if (need_y) out[0] = dispatch_op(g, w, r);
    if (need_w) out[1] = dots_op(g, y, r);
    return out;
  }
};

struct RowDots : torch::autograd::Function<RowDots> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& y, const Routed& r) {
    ctx->save_for_backward({x, y});
    hold(ctx, r);
    return dots_of(x, y, Tensor(), r, false).second;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Routed& r = held<Routed>(ctx);
    const Tensor g = dense(grads[0]), &x = saved[0], &y = saved[1];
    variable_list out(3);
    if (ctx->needs_input_grad(0)) out[0] = combine_op(y, g, r);
    if (ctx->needs_input_grad(1)) out[1] = dispatch_op(x, g, r);
    return out;
  }
};

Tensor dispatch_op(const Tensor& x, const Tensor& w, const Routed& r) {
  return tracked(x) || tracked(w) ? Dispatch::apply(x, maybe(w), r) : dispatch_rows(x, w, r);
}
Tensor combine_op(const Tensor& y, const Tensor& w, const Routed& r) {
  return tracked(y) || tracked(w) ? Combine::apply(y, maybe(w), r) : combine_rows(y, w, r);
}
Tensor dots_op(const Tensor& x, const Tensor& y, const Routed& r) {
  return tracked(x) || tracked(y) ? RowDots::apply(x, y, r) : dots_of(x, y, Tensor(), r, false).second;
}

// (rowptr, order, place, tokens, k)
std::tuple<Tensor, Tensor, Tensor, int64_t, int64_t> route_plan(const Tensor& experts, int64_t n_experts,
                                                                bool timed) {
  TORCH_CHECK_VALUE(experts.is_cuda(), "experts must be a GPU tensor (got ", experts.device(), ")");
  want_indices(experts, "experts");
  TORCH_CHECK_VALUE(experts.dim() == 1 || (experts.dim() == 2 && experts.size(1) >= 1), "experts has shape ",
                    experts.sizes(), ", expected [T] or [T, k]");
  const int64_t T = experts.size(0), k = experts.dim() == 1 ? 1 : experts.size(1);
  TORCH_CHECK_VALUE(n_experts >= 0 && n_experts <= MAX_INDEX && k <= MAX_INDEX && T * k <= MAX_INDEX,
                    "route_plan: slots or experts exceed 32-bit indices");
  const Groups g = group(signed_values(experts).reshape({-1}), n_experts, true, timed);
  return {g.rowptr, g.order, g.place, T, k};
}

Tensor route(bool combine, const Tensor& x, const Tensor& place, const Tensor& rowptr, int64_t tokens, int64_t k,
             const optional<Tensor>& weights, const optional<std::vector<int64_t>>& widths, bool timed) {
  const char* name = combine ? "y" : "x";
  const int64_t rows = combine ? tokens * k : tokens;
  want_rows(x, name);
  TORCH_CHECK_VALUE(x.dim() == 2 && x.size(0) == rows && x.size(1) >= 1 && x.size(1) <= MAX_ROW, name, " has shape ",
                    x.sizes(), ", expected [", rows, ", D] with D of 1 to ", MAX_ROW);
  want_device(x, place, name);
  want_int32(place, tokens * k, x, "plan.place");
  want_int32(rowptr, rowptr.numel(), x, "plan.rowptr");
  TORCH_CHECK_VALUE(rowptr.numel() >= 1, "plan.rowptr is empty");
  Routed r{place, rowptr, tokens, (int)k, widths ? *widths : std::vector<int64_t>{x.size(1)}, timed};
  int64_t total = 0;
  bool positive = true;
  for (int64_t v : r.widths) {
    total += v;
    positive = positive && v > 0 && v <= MAX_ROW;
  }
  TORCH_CHECK_VALUE(!r.widths.empty() && r.widths.size() <= TACE_ROW_MAX_BLOCKS && positive && total == x.size(1),
                    "widths ", r.widths, " are not 1 to ", TACE_ROW_MAX_BLOCKS, " blocks of ", x.size(1), " elements");
  Tensor w;
  if (weights) {
    w = *weights;
    TORCH_CHECK_VALUE(w.is_floating_point() && ((w.dim() == 2 && w.size(0) == tokens && w.size(1) == k) ||
                                                (w.dim() == 1 && k == 1 && w.size(0) == tokens)),
                      "weights must be floating point [", tokens, ", ", k, "], got ", w.scalar_type(), " ", w.sizes());
    want_device(w, x, "weights");
    w = dense(w.reshape({tokens, k}).to(sum_type(x)));
  }
  return combine ? combine_op(dense(x), w, r) : dispatch_op(dense(x), w, r);
}

// ------------------------------------------------------------------- dropout ----
struct Mask {
  int64_t seed, offset, site;
  int threshold, channels;
  std::vector<int32_t> comps;
  int total;   // components
  bool timed, residual;
};

Tensor masked(const Tensor& x, const Tensor& residual, const Tensor& state, const Mask& m) {
  Tensor out = at::empty_like(x);
  Launch l(x, "dropout", m.timed);
  l.done(tace_dropout(type_code(x.scalar_type()), ptr(x), ptr(residual),
                      state.defined() ? state.data_ptr<int64_t>() : nullptr, m.seed, m.offset, (uint32_t)m.site, m.threshold, x.numel() / ((int64_t)m.channels * m.total),
                      m.channels, (int)m.comps.size(), m.comps.data(), ptr(out), l.stream), {x.numel()});
  return out;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& residual,
                        const optional<Tensor>& state, const Mask& m) {
    ctx->save_for_backward({state.value_or(Tensor())});
    hold(ctx, m);
    return masked(x, residual.value_or(Tensor()), state.value_or(Tensor()), m);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor state = ctx->get_saved_variables()[0];
    Mask m = held<Mask>(ctx);
    variable_list out(4);
    if (m.residual && ctx->needs_input_grad(1)) out[1] = grads[0];
    m.residual = false;
    if (ctx->needs_input_grad(0)) {
      const Tensor g = dense(grads[0]);
      out[0] = tracked(g) ? Dropout::apply(g, std::nullopt, maybe(state), m) : masked(g, Tensor(), state, m);
    }
    return out;
  }
};

Tensor dropout(const Tensor& x, double p, const optional<Tensor>& state, int64_t seed, int64_t offset, int64_t site,
               const std::vector<int64_t>& components, const optional<Tensor>& residual, bool timed) {
  want_rows(x, "x");
  const double t = p >= 0.0 && p <= 1.0 ? std::nearbyint(65536 * p) : -1;
  TORCH_CHECK_VALUE(t >= 0 && (t == 0) == (p == 0.0) && (t == 65536) == (p == 1.0), "dropout: p = ", p,
                    " is outside [0, 1] or nearer to its ends than the mask's 2^-16");
  TORCH_CHECK_VALUE(site >= 0 && site <= UINT32_MAX, "dropout: site ", site, " is outside 0 .. 2^32 - 1");
  Mask m{seed, offset, site, (int)t, 1, {}, 0, timed, residual.has_value()};
  bool ok = !components.empty() && components.size() <= TACE_ROW_MAX_BLOCKS;
  for (int64_t c : components) {
    ok = ok && c >= 1 && c <= 1024;
    m.comps.push_back((int32_t)c);
    m.total += (int)c;
  }
  TORCH_CHECK_VALUE(ok, "dropout: components ", components, " are not 1 to ", TACE_ROW_MAX_BLOCKS,
                    " blocks of 1 to 1024");
  if (m.comps.size() > 1 || m.comps[0] > 1) {
    TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) >= 1 && x.size(1) % m.total == 0 && x.size(1) <= INT32_MAX,
                      "x has shape ", x.sizes(), ", expected [rows, ", m.total, " C]");
    m.channels = (int)(x.size(1) / m.total);
  }
  TORCH_CHECK_VALUE(x.numel() / m.total * (int64_t)m.comps.size() <= (int64_t)1 << 34, "dropout: over 2^34 draws");
  if (state) {
    TORCH_CHECK_VALUE(state->scalar_type() == at::kLong && state->dim() == 1 && state->size(0) == 2 &&
                      state->is_contiguous() && !state->is_neg(), "rng must be a contiguous int64 tensor [2] or two integers");
    want_device(*state, x, "rng");
  }
  Tensor res;
  if (residual) {
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type(), "residual is ",
                      residual->scalar_type(), " ", residual->sizes(), ", expected ", x.scalar_type(), " ", x.sizes());
    want_device(*residual, x, "residual");
    res = dense(*residual);
  }
  const Tensor in = dense(x);
  if (tracked(in) || tracked(res)) return Dropout::apply(in, maybe(res), state, m);
  return masked(in, res, state.value_or(Tensor()), m);
}

}  // namespace

PYBIND11_MODULE(_rows, mod) {
  mod.attr("BUILT_FOR") = TACE_ROWS_ABI_VERSION;   // (the library's own may differ)
  mod.def("timer", [](py::object start, py::object stop) {
    Launch::start = start.release().ptr();
    Launch::stop = stop.release().ptr();
  });
  mod.def("embedding", torch::wrap_pybind_function(embedding));
  mod.def("route_plan", torch::wrap_pybind_function(route_plan));
  mod.def("route", torch::wrap_pybind_function(route));
  mod.def("dropout", torch::wrap_pybind_function(dropout));
  bind_layer(mod);
}

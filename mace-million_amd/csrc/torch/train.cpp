// PyTorch functions of the operators that train a head: group norm, linear cross entropy, orthogonalisation.
#include "checks.h"

namespace {
// ------------------------------------------------------------------------------------------------ group norm
struct GroupSizes { long rows, structs, C, groups; };

Tensor group_workspace(const GroupSizes& n, bool ragged, int code, int backward, const Tensor& like) {
  size_t bytes = 0;
  done(mm_groupnorm_workspace(n.rows, (int)n.structs, ragged, (int)n.C, (int)n.groups, code, backward, &bytes));
  return bytes ? f32({(int64_t)(bytes / sizeof(float))}, like) : Tensor();
}

struct GroupNormFn : torch::autograd::Function<GroupNormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& w, const Maybe& b, const Maybe& offsets,
                        int64_t structs, int64_t groups, double eps, int64_t act, int64_t code, int64_t p_code) {
    const Tensor weight = value(w), bias = value(b), offs = value(offsets);
    auto [x2, ldx] = as_rows(x);
    const GroupSizes n{x2.size(0), structs, x2.size(1), groups};
    Tensor stats = f32({structs, groups, 2}, x);
    Tensor y = run(x, x2, ldx, weight, bias, offs, n, eps, (int)act, (int)code, (int)p_code, stats);
    ctx->save_for_backward({x2, weight, bias, offs, stats});
    ctx->saved_data["args"] = std::vector<int64_t>{structs, groups, act, code, p_code};
    ctx->saved_data["shape"] = x.sizes().vec();
    return y;
  }

  static Tensor run(const Tensor& x, const Tensor& x2, long ldx, const Tensor& weight, const Tensor& bias,
                    const Tensor& offsets, const GroupSizes& n, double eps, int act, int code, int p_code,
                    Tensor stats) {
    Tensor y = at::empty(x.sizes(), x.options());
    const Tensor w = weight.defined() ? weight.contiguous() : weight, b = bias.defined() ? bias.contiguous() : bias;
    const Tensor ws = group_workspace(n, offsets.defined(), code, 0, x);
    if (ws.defined() && !stats.defined()) stats = f32({n.structs, n.groups, 2}, x);
    done(mm_groupnorm_fwd(ptr(x2), ldx, code, n.rows, (int)n.structs, iptr(offsets), (int)n.C, (int)n.groups, ptr(w),
                          ptr(b), p_code, (float)eps, act, ptr(y), n.C, fptr(stats), fptr(ws), stream()));
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto args = ctx->saved_data["args"].toIntVector();
    const int code = (int)args[3], p_code = (int)args[4];
    auto [dy, lddy] = as_rows(plain(grads[0]));
    const GroupSizes n{dy.size(0), args[0], dy.size(1), args[1]};
    const auto p_type = type_of(p_code);
    auto [x, ldx] = as_rows(unpacked(saved[0], {n.rows, n.C}, type_of(code), dy, "x"));
    const Tensor w = unpacked_dense(saved[1], {n.C}, p_type, dy, "weight");
    const Tensor b = unpacked_dense(saved[2], {n.C}, p_type, dy, "bias");
    const Tensor offsets = unpacked_dense(saved[3], {n.structs + 1}, at::kInt, dy, "offsets");
    const Tensor stats = unpacked_dense(saved[4], {n.structs, n.groups, 2}, at::kFloat, dy, "statistics");
    Tensor dx, dw, db;
    if (ctx->needs_input_grad(0)) dx = at::empty(ctx->saved_data["shape"].toIntVector(), x.options());
    const int at_bias = w.defined() ? 2 : 1;   // autograd counts the tensors that are there
    if (w.defined() && ctx->needs_input_grad(1)) dw = at::empty({n.C}, x.options().dtype(p_type));
    if (b.defined() && ctx->needs_input_grad(at_bias)) db = at::empty({n.C}, x.options().dtype(p_type));
    const Tensor ws = group_workspace(n, offsets.defined(), code, 1, x);
    done(mm_groupnorm_bwd(ptr(dy), lddy, ptr(x), ldx, code, n.rows, (int)n.structs, iptr(offsets), (int)n.C,
                          (int)n.groups, ptr(w), ptr(b), p_code, (int)args[2], fptr(stats), ptr(dx), n.C, ptr(dw),
                          ptr(db), fptr(ws), stream()));
    variable_list out(10);
    out[0] = dx;
    out[1] = dw;
    out[2] = db;
    return once(out, "group_norm");
  }
};

Tensor group_norm(const Tensor& x0, int64_t groups, const Maybe& weight, const Maybe& bias, double eps,
                  const std::optional<std::string>& activation, const Maybe& offsets0) {
  const Tensor x = plain(x0);
  const int code = check_gpu(x, "x");
  if (x.dim() < 2 || x.size(-1) == 0)
    throw py::value_error(text("x must be [structures, ..., C] (or [rows, C] with offsets), got ", x.sizes()));
  const long C = x.size(-1);
  if (groups < 1 || C % groups) throw py::value_error(text("groups must divide the ", C, " channels, got ", groups));
  if (groups > 65535) throw py::value_error(text("at most 65535 groups are supported, got ", groups));
  if (C / groups * x.element_size() > kMaxDim)
    throw py::value_error(text("groups of more than ", kMaxDim / x.element_size(), " channels are not supported, got ",
                               C / groups));
  int64_t act = 0;
  if (activation) {
    if (*activation == "silu") act = 1;
    else if (*activation == "gelu") act = 2;
    else throw py::value_error(text("activation must be None, 'silu' or 'gelu', got '", *activation, "'"));
  }
  int p_code = code;
  auto param = [&](const Maybe& p, const char* name) {
    if (!p) return Tensor();
    p_code = check_gpu(*p, name);
    if (p_code != code && p_code != 0)
      throw py::type_error(text(name, " must be ", type_name(x.scalar_type()), " (as x) or float32, got ",
                                type_name(p->scalar_type())));
    if (p->dim() != 1 || p->size(0) != C) throw py::value_error(text(name, " must be [", C, "], got ", p->sizes()));
    return plain(*p);
  };
  const Tensor w = param(weight, "weight"), b = param(bias, "bias");
  if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type())
    throw py::type_error(text("weight and bias must have one type, got ", type_name(w.scalar_type()), " and ",
                              type_name(b.scalar_type())));
  const long rows = x.numel() / C;
  if (rows >= kMaxRows) throw py::value_error(text(rows, " rows: fewer than 2^31 - 2^16 are supported"));
  long structs = x.size(0);
  Tensor offsets;
  if (offsets0) {
    const Tensor o = plain(*offsets0);
    if (!o.is_cuda()) throw py::type_error("offsets must be a GPU tensor");
    if (o.scalar_type() != at::kInt && o.scalar_type() != at::kLong)
      throw py::type_error(text("offsets must be int32 or int64, got ", type_name(o.scalar_type())));
    if (o.device() != x.device()) throw py::value_error("x and offsets must be on one device");
    if (x.dim() != 2 || o.dim() != 1 || o.size(0) < 2)
      throw py::value_error(text("with offsets [structures + 1], x must be [rows, C], got ", o.sizes(), " and ",
                                 x.sizes()));
    structs = o.size(0) - 1;
    // values outside int32 must not wrap into the rows
    offsets = (o.scalar_type() == at::kLong ? o.clamp(0, rows).to(at::kInt) : o).contiguous();
  }
  if (structs > kInt32Max - 1) throw py::value_error(text("too many structures: ", structs));
  refuse_modes("group_norm", {&x, &w, &b});
  if (rows == 0) structs = offsets.defined() ? structs : 0;
  if (needs_grad({&x, &w, &b}))
    return GroupNormFn::apply(x, maybe(w), maybe(b), maybe(offsets), (int64_t)structs, groups, eps, act, (int64_t)code,
                              (int64_t)p_code);
  auto [x2, ldx] = as_rows(x);
  return GroupNormFn::run(x, x2, ldx, w, b, offsets, GroupSizes{rows, structs, C, groups}, eps, (int)act, code, p_code,
                          Tensor());
}

// ------------------------------------------------------------------------------------------------ cross entropy
Tensor bytes_like(size_t n, const Tensor& like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }

struct LossSizes { long T, D, V; };

struct CrossEntropyFn : torch::autograd::Function<CrossEntropyFn> {
  struct Result { Tensor loss, stats, rows; };

  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& targets,
                        int64_t ignore, int64_t reduction, int64_t code) {
    auto [x2, ldx] = as_rows(x);
    const Tensor w = weight.contiguous();
    Result r = run(x2, ldx, w, targets, ignore, (int)reduction, (int)code);
    ctx->save_for_backward({x2, w, r.stats, r.rows});
    ctx->saved_data["args"] = std::vector<int64_t>{reduction, code, x2.size(0), x2.size(1), w.size(0)};
    ctx->saved_data["shape"] = x.sizes().vec();
    return r.loss;
  }

  static Result run(const Tensor& x2, long ldx, const Tensor& w, const Tensor& targets, int64_t ignore, int reduction,
                    int code) {
    const LossSizes n{x2.size(0), x2.size(1), w.size(0)};
    const Tensor y = targets.contiguous();
    Result r{reduction ? f32({}, x2) : f32(targets.sizes(), x2), f32({2, n.T}, x2), i32({4 + 3 * n.T}, x2)};
    size_t bytes = 0;
    done(mm_ce_workspace(n.T, n.D, n.V, code, ptr(w), 0, 0, &bytes));
    const Tensor ws = bytes_like(bytes, x2);
    if (n.T || reduction)
      done(mm_ce_fwd(ptr(x2), ldx, code, n.T, n.D, ptr(w), n.V, ptr(y), y.scalar_type() == at::kLong, ignore, reduction,
                     fptr(r.loss), fptr(r.stats), iptr(r.rows), ptr(ws), stream()));
    return r;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto args = ctx->saved_data["args"].toIntVector();
    const int reduction = (int)args[0], code = (int)args[1];
    const LossSizes n{args[2], args[3], args[4]};
    const Tensor dloss = plain(grads[0]).contiguous();
    const auto type = type_of(code);
    auto [x, ldx] = as_rows(unpacked(saved[0], {n.T, n.D}, type, dloss, "x"));
    const Tensor w = unpacked_dense(saved[1], {n.V, n.D}, type, dloss, "weight");
    const Tensor stats = unpacked_dense(saved[2], {2, n.T}, at::kFloat, dloss, "statistics");
    const Tensor rows = unpacked_dense(saved[3], {4 + 3 * n.T}, at::kInt, dloss, "rows");
    Tensor dx, dw;
    if (ctx->needs_input_grad(0)) dx = at::empty(ctx->saved_data["shape"].toIntVector(), x.options());
    if (ctx->needs_input_grad(1)) dw = n.T ? at::empty({n.V, n.D}, x.options()) : at::zeros({n.V, n.D}, x.options());
    if (n.T && (dx.defined() || dw.defined())) {
      size_t bytes = 0;
      done(mm_ce_workspace(n.T, n.D, n.V, code, ptr(w), dx.defined(), dw.defined(), &bytes));
      const Tensor ws = bytes_like(bytes, x);
      done(mm_ce_bwd(ptr(x), ldx, code, n.T, n.D, ptr(w), n.V, reduction, fptr(stats), iptr(rows), fptr(dloss), ptr(dx),
                     ptr(dw), ptr(ws), stream()));
    }
    variable_list out(6);
    out[0] = dx;
    out[1] = dw;
    return once(out, "linear_cross_entropy");
  }
};

Tensor linear_cross_entropy(const Tensor& x0, const Tensor& weight0, const Tensor& targets0, int64_t ignore,
                            const std::string& reduction) {
  const Tensor x = plain(x0), weight = plain(weight0), targets = plain(targets0);
  const int code = check_gpu(x, "x");
  if (check_gpu(weight, "weight") != code)
    throw py::type_error(text("weight must be ", type_name(x.scalar_type()), " (as x), got ",
                              type_name(weight.scalar_type())));
  if (x.dim() < 1 || x.size(-1) == 0) throw py::value_error(text("x must be [..., D] with D > 0, got ", x.sizes()));
  const long D = x.size(-1), T = x.numel() / D;
  if (weight.dim() != 2 || weight.size(1) != D || weight.size(0) == 0)
    throw py::value_error(text("weight must be [classes, ", D, "], got ", weight.sizes()));
  if (!targets.is_cuda()) throw py::type_error("targets must be a GPU tensor");
  if (targets.scalar_type() != at::kInt && targets.scalar_type() != at::kLong)
    throw py::type_error(text("targets must be int32 or int64, got ", type_name(targets.scalar_type())));
  if (targets.device() != x.device()) throw py::value_error("x and targets must be on one device");
  if (targets.sizes() != x.sizes().slice(0, x.dim() - 1))
    throw py::value_error(text("targets must be ", x.sizes().slice(0, x.dim() - 1), ", got ", targets.sizes()));
  const long V = weight.size(0);
  if (T >= kMaxRows || V >= kMaxRows || D >= kMaxRows)
    throw py::value_error(text("sizes of 2^31 - 2^16 or more are not supported, got ", x.sizes(), " and ",
                               weight.sizes()));
  int64_t how = 0;
  if (reduction == "sum") how = 1;
  else if (reduction == "mean") how = 2;
  else if (reduction != "none")
    throw py::value_error(text("reduction must be 'mean', 'sum' or 'none', got '", reduction, "'"));
  refuse_modes("linear_cross_entropy", {&x, &weight});
  if (needs_grad({&x, &weight})) return CrossEntropyFn::apply(x, weight, targets, ignore, how, (int64_t)code);
  auto [x2, ldx] = as_rows(x);
  return CrossEntropyFn::run(x2, ldx, weight.contiguous(), targets, ignore, (int)how, code).loss;
}

// ------------------------------------------------------------------------------------------------ orthogonalisation
Tensor orthogonalize(const Tensor& m0, const std::vector<float>& coefficients, double eps) {
  const Tensor m1 = plain(m0);
  const int code = check_gpu(m1, "m");
  if (m1.dim() < 2 || m1.size(-1) == 0 || m1.size(-2) == 0)
    throw py::value_error(text("m must be [..., rows, columns], got ", m1.sizes()));
  if (coefficients.size() % 3) throw py::value_error("coefficients must be triples (a, b, c)");
  if (!(eps >= 0.) || !std::isfinite((float)eps)) throw py::value_error(text("eps must be finite and >= 0, got ", eps));
  const long rows = m1.size(-2), cols = m1.size(-1), batch = m1.numel() / (rows * cols);
  if (rows > 65536 || cols > 65536)
    throw py::value_error(text("matrices of more than 65536 rows or columns are not supported, got ", m1.sizes()));
  refuse_modes("orthogonalize", {&m1});
  if (needs_grad({&m1}))
    throw std::runtime_error("orthogonalize has no derivative: call it under torch.no_grad() or on a detached tensor");
  const Tensor m = m1.contiguous();
  Tensor out = at::empty(m.sizes(), m.options());
  if (batch == 0) return out;
  const long step = rows * cols * (long)m.element_size();
  Tensor ws;
  for (long i = 0; i < batch; i += 65535) {   // of a launch's grid
    const long n = std::min(batch - i, 65535L);
    size_t bytes = 0;
    done(mm_orthogonalize_workspace_steps(n, rows, cols, code, (int)(coefficients.size() / 3), &bytes));
    if (!ws.defined() || bytes > (size_t)ws.numel()) ws = bytes_like(bytes, m);
    done(mm_orthogonalize((const char*)ptr(m) + i * step, code, n, rows, cols, (int)(coefficients.size() / 3),
                          coefficients.data(), (float)eps, (char*)ptr(out) + i * step, ptr(ws), stream()));
  }
  return out;
}
}  // namespace

void bind_train(py::module_& m) {
  m.def("group_norm", &group_norm);
  m.def("linear_cross_entropy", &linear_cross_entropy);
  m.def("orthogonalize", &orthogonalize);
}

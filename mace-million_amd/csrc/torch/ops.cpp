// PyTorch functions of the layer norm, routing and expert kernels: argument checks, output and workspace tensors, the
// calls of the C ABI on torch's current stream, and their place in autograd.
//
// In C++ because small calls are bound by the host: with the forward and backward as Python functions, a training call
// took 130 - 210 us whatever its kernels took, most of it the hand-over of the interpreter to autograd's thread and
// back.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/sub.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cmath>
#include <memory>
#include <optional>
#include <sstream>
#include <string>
#include <tuple>
#include <vector>

#include "../../../include/mace_million_amd.h"

namespace {
namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr long kInt32Max = 2147483647L, kMaxRows = 2147483648L - 65536;
constexpr int kMaxDim = 16384, kMaxExperts = 1024, kMaxK = 32, kMaxGroups = 64;

template <typename... A>
std::string text(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  return s.str();
}

void done(int rc) {
  if (rc != 0) throw std::runtime_error(mm_last_error());
}

mm_stream_t stream() { return (mm_stream_t)c10::hip::getCurrentHIPStream().stream(); }

// Fake, wrapped and zero tensors pass for GPU tensors and have no memory.
void* ptr(const Tensor& t) {
  if (!t.defined()) return nullptr;
  void* p = t.numel() ? t.data_ptr() : nullptr;
  if (!p && t.numel()) throw py::type_error("a tensor without memory (fake, wrapped or zero tensor) cannot be read");
  return p;
}
float* fptr(const Tensor& t) { return (float*)ptr(t); }
int* iptr(const Tensor& t) { return (int*)ptr(t); }

const char* type_name(at::ScalarType t) { return c10::toString(t); }

// dtype code of a floating tensor of the current GPU
int check_gpu(const Tensor& t, const char* name) {
  if (!t.is_cuda()) throw py::type_error(text(name, " must be a GPU tensor"));
  if (t.device().index() != c10::hip::current_device())
    throw py::value_error(text(name, " is on ", t.device(), ", the current device is cuda:",
                               (int)c10::hip::current_device()));
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default:
      throw py::type_error(text(name, " must be float32, bfloat16 or float16, got ", type_name(t.scalar_type())));
  }
}

Tensor f32(at::IntArrayRef size, const Tensor& like) { return at::empty(size, like.options().dtype(at::kFloat)); }
Tensor i32(at::IntArrayRef size, const Tensor& like) { return at::empty(size, like.options().dtype(at::kInt)); }

// The values of a lazily negated view (of a conjugate's imaginary part, say) are not those of its memory.
Tensor plain(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }

// Autograd takes absent tensors as empty optionals.
using Maybe = std::optional<Tensor>;
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }
Tensor value(const Maybe& t) { return t ? *t : Tensor(); }

bool needs_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// Forward-mode derivatives and traces go through dispatched operations only, so they would miss these functions without
// a word: the result would pass for a constant, the trace would hold memory that nothing writes.
void refuse_modes(const char* what, std::initializer_list<const Tensor*> ts) {
  if (torch::jit::tracer::isTracing()) throw std::runtime_error(text(what, " cannot be traced (torch.jit.trace)"));
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(0).defined())
      throw std::runtime_error(text(what, " has no forward-mode derivative: its inputs must not be dual tensors"));
}

// Gradients that raise when they are differentiated again, instead of passing for constants.
variable_list once(variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads)
    if (g.defined()) g = g.detach().requires_grad_(true);
  auto error = std::make_shared<torch::autograd::DelayedError>(text(what, " can be differentiated once only"),
                                                               (int64_t)grads.size());
  return (*error)(std::move(grads));
}

// t as rows with a contiguous last axis, and the distance of rows
std::pair<Tensor, long> as_rows(Tensor t) {
  const long D = t.size(-1);
  if (t.dim() != 2) t = t.reshape({-1, D});
  if (D > 1 && t.stride(1) != 1) t = t.contiguous();
  return {t, t.size(0) > 1 ? t.stride(0) : D};
}

// A saved tensor as its node gets it back.  Hooks on saved tensors (offloading, compression) may return it with any
// strides, so its layout is taken from what comes back; sizes and type have to be those that were saved.
Tensor unpacked(const Tensor& t, at::IntArrayRef size, at::ScalarType type, const Tensor& like,
                       const char* name) {
  if (t.defined() && (t.sizes() != size || t.scalar_type() != type || t.device() != like.device()))
    throw std::runtime_error(text(name, " was saved for the backward as ", type_name(type), " ", size, " on ",
                                  like.device(), " and came back as ", type_name(t.scalar_type()), " ", t.sizes(),
                                  " on ", t.device()));
  return plain(t);
}

Tensor unpacked_dense(const Tensor& t, at::IntArrayRef size, at::ScalarType type, const Tensor& like,
                      const char* name) {
  const Tensor u = unpacked(t, size, type, like, name);
  return u.defined() ? u.contiguous() : u;
}

at::ScalarType type_of(int64_t code) { return code == 0 ? at::kFloat : code == 1 ? at::kBFloat16 : at::kHalf; }

// ------------------------------------------------------------------------------------------------ layer norm
struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& w, const Maybe& b, double eps, int64_t code,
                        int64_t p_code) {
    const Tensor weight = value(w), bias = value(b);
    Tensor stats;
    auto [x2, ldx] = as_rows(x);
    Tensor y = run(x, x2, ldx, weight, bias, eps, (int)code, (int)p_code, &stats);
    ctx->save_for_backward({x2, weight, stats});
    ctx->saved_data["bias"] = bias.defined();
    ctx->saved_data["codes"] = code * 4 + p_code;
    ctx->saved_data["shape"] = x.sizes().vec();
    return y;
  }

  static Tensor run(const Tensor& x, const Tensor& x2, long ldx, const Tensor& weight, const Tensor& bias, double eps,
                    int code, int p_code, Tensor* stats) {
    const long rows = x2.size(0), D = x2.size(1);
    Tensor y = at::empty(x.sizes(), x.options());
    const Tensor w = weight.defined() ? weight.contiguous() : weight, b = bias.defined() ? bias.contiguous() : bias;
    if (stats) *stats = f32({2, rows}, x);
    float* mean = stats ? fptr(*stats) : nullptr;
    done(mm_layernorm_fwd(ptr(x2), ldx, code, rows, (int)D, ptr(w), ptr(b), p_code, (float)eps, ptr(y), D, mean,
                          mean ? mean + rows : nullptr, stream()));
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const int64_t codes = ctx->saved_data["codes"].toInt();
    const int code = (int)(codes / 4), p_code = (int)(codes % 4);
    auto [dy, lddy] = as_rows(plain(grads[0]));
    const long rows = dy.size(0), D = dy.size(1);
    const auto p_type = type_of(p_code);
    auto [x, ldx] = as_rows(unpacked(saved[0], {rows, D}, type_of(code), dy, "x"));
    const Tensor w = unpacked_dense(saved[1], {D}, p_type, dy, "weight");
    const Tensor stats = unpacked_dense(saved[2], {2, rows}, at::kFloat, dy, "statistics");
    Tensor dx, dw, db, ws;
    if (ctx->needs_input_grad(0)) dx = at::empty(ctx->saved_data["shape"].toIntVector(), x.options());
    const int at_bias = w.defined() ? 2 : 1;   // autograd counts the tensors that are there
    if (w.defined() && ctx->needs_input_grad(1)) dw = at::empty({D}, x.options().dtype(p_type));
    if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(at_bias))
      db = at::empty({D}, x.options().dtype(p_type));
    if (dw.defined() || db.defined()) {
      size_t bytes = 0;
      done(mm_layernorm_workspace(rows, (int)D, code, &bytes));
      ws = f32({(int64_t)(bytes / sizeof(float))}, x);
    }
    const float* mean = fptr(stats);
    done(mm_layernorm_bwd(ptr(dy), lddy, ptr(x), ldx, code, rows, (int)D, ptr(w), p_code, mean, mean + rows, ptr(dx), D,
                          ptr(dw), ptr(db), fptr(ws), stream()));
    return once({dx, dw, db, Tensor(), Tensor(), Tensor()}, "layer_norm");
  }
};

Tensor layer_norm(const Tensor& x0, const Maybe& weight, const Maybe& bias, double eps) {
  const Tensor x = plain(x0);
  const int code = check_gpu(x, "x");
  if (x.dim() < 1 || x.size(-1) == 0)
    throw py::value_error(text("x must be [..., D] with D > 0, got ", x.sizes()));
  const long D = x.size(-1);
  if (D > kMaxDim)
    throw py::value_error(text("rows of more than ", kMaxDim, " values are not supported, got ", D));
  int p_code = code;
  auto param = [&](const Maybe& p, const char* name) {
    if (!p) return Tensor();
    p_code = check_gpu(*p, name);
    if (p_code != code && p_code != 0)
      throw py::type_error(text(name, " must be ", type_name(x.scalar_type()), " (as x) or float32, got ",
                                type_name(p->scalar_type())));
    if (p->dim() != 1 || p->size(0) != D) throw py::value_error(text(name, " must be [", D, "], got ", p->sizes()));
    return plain(*p);
  };
  const Tensor w = param(weight, "weight"), b = param(bias, "bias");
  if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type())
    throw py::type_error(text("weight and bias must have one type, got ", type_name(w.scalar_type()), " and ",
                              type_name(b.scalar_type())));
  refuse_modes("layer_norm", {&x, &w, &b});
  if (needs_grad({&x, &w, &b})) return LayerNormFn::apply(x, maybe(w), maybe(b), eps, (int64_t)code, (int64_t)p_code);
  auto [x2, ldx] = as_rows(x);
  return LayerNormFn::run(x, x2, ldx, w, b, eps, code, p_code, nullptr);
}

// ------------------------------------------------------------------------------------------------ routing
struct RouteFn : torch::autograd::Function<RouteFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Maybe& bias, int64_t code, int64_t k,
                               int64_t scoring, int64_t groups, int64_t top_groups, int64_t renorm, double scale) {
    const Tensor x = rows(logits);
    auto [gates, experts] = run(x, value(bias), code, k, scoring, groups, top_groups, renorm, scale);
    ctx->save_for_backward({x, gates, experts});
    ctx->saved_data["args"] = std::vector<int64_t>{code, scoring, renorm, x.size(1), k};
    ctx->saved_data["scale"] = scale;
    ctx->mark_non_differentiable({experts});
    return {gates, experts};
  }

  static Tensor rows(const Tensor& t) {
    const bool ok = (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
    return ok ? t : t.contiguous();
  }

  static long distance(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

  static std::pair<Tensor, Tensor> run(const Tensor& x, const Tensor& bias, int64_t code, int64_t k, int64_t scoring,
                                       int64_t groups, int64_t top_groups, int64_t renorm, double scale) {
    const long T = x.size(0), E = x.size(1);
    Tensor gates = f32({T, k}, x), experts = i32({T, k}, x);
    done(mm_route_fwd(ptr(x), distance(x), (int)code, T, (int)E, (int)k, (int)scoring, fptr(bias), (int)groups,
                      (int)top_groups, (int)renorm, (float)scale, fptr(gates), iptr(experts), stream()));
    return {gates, experts};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto args = ctx->saved_data["args"].toIntVector();
    const Tensor dg = plain(grads[0]).contiguous();
    const long T = dg.size(0), E = args[3], k = args[4];
    const Tensor x = rows(unpacked(saved[0], {T, E}, type_of(args[0]), dg, "logits"));
    const Tensor gates = unpacked_dense(saved[1], {T, k}, at::kFloat, dg, "gates");
    const Tensor experts = unpacked_dense(saved[2], {T, k}, at::kInt, dg, "experts");
    Tensor dl = at::empty({T, E}, x.options());
    done(mm_route_bwd(ptr(x), distance(x), (int)args[0], T, (int)E, (int)k, (int)args[1], (int)args[2],
                      (float)ctx->saved_data["scale"].toDouble(), fptr(gates), iptr(experts), fptr(dg), ptr(dl),
                      stream()));
    variable_list out(9);
    out[0] = dl;
    return once(out, "route");
  }
};

std::tuple<Tensor, Tensor> route(const Tensor& logits0, int64_t k, const std::string& scoring,
                                 const Maybe& bias, int64_t groups, std::optional<int64_t> top,
                                 bool renormalize, double scale) {
  const Tensor logits = plain(logits0);
  const int code = check_gpu(logits, "logits");
  if (logits.dim() != 2 || logits.size(1) == 0)
    throw py::value_error(text("logits must be [rows, experts], got ", logits.sizes()));
  const long E = logits.size(1), most = std::min<long>(E, kMaxK);
  if (E > kMaxExperts) throw py::value_error(text("at most ", kMaxExperts, " experts are supported, got ", E));
  if (k < 1 || k > most) throw py::value_error(text("k must be 1 .. ", most, ", got ", k));
  if (scoring != "softmax" && scoring != "sigmoid")
    throw py::value_error(text("scoring must be 'softmax' or 'sigmoid', got '", scoring, "'"));
  if (groups < 1 || groups > kMaxGroups || E % groups)
    throw py::value_error(text("groups must divide the ", E, " experts and be at most ", kMaxGroups, ", got ", groups));
  const int64_t top_groups = top.value_or(groups);
  if (top_groups < 1 || top_groups > groups)
    throw py::value_error(text("top_groups must be 1 .. ", groups, ", got ", top_groups));
  if (!((float)scale != 0.f) || !std::isfinite((float)scale))
    throw py::value_error(text("scale must be finite and not 0, got ", scale));
  Tensor b;
  if (bias) {
    check_gpu(*bias, "bias");
    if (bias->scalar_type() != at::kFloat)
      throw py::type_error(text("bias must be float32, got ", type_name(bias->scalar_type())));
    if (bias->dim() != 1 || bias->size(0) != E)
      throw py::value_error(text("bias must be [", E, "], got ", bias->sizes()));
    b = plain(bias->detach()).contiguous();
  }
  refuse_modes("route", {&logits});
  const int64_t s = scoring == "sigmoid", r = renormalize;
  if (needs_grad({&logits})) {
    const variable_list out = RouteFn::apply(logits, maybe(b), (int64_t)code, k, s, groups, top_groups, r, scale);
    return {out[0], out[1]};
  }
  auto [gates, experts] = RouteFn::run(RouteFn::rows(logits), b, code, k, s, groups, top_groups, r, scale);
  return {gates, experts};
}

// ------------------------------------------------------------------------------------------------ plan
struct Lists { Tensor offsets, order; };

Lists make_lists(const Tensor& experts, long E) {
  const long S = experts.numel();
  long scratch = 0;
  done(mm_expert_plan_scratch((int)S, (int)E, &scratch));
  const Tensor buf = i32({S + E + 1 + scratch}, experts);
  int* p = iptr(buf);
  done(mm_expert_plan(iptr(experts), (int)S, (int)E, p, p + E + 1, scratch ? p + E + 1 + S : nullptr, stream()));
  return {buf.narrow(0, 0, E + 1), buf.narrow(0, E + 1, S)};
}

// rows of two choices sorted by the pair of their experts
Lists make_pairs(const Tensor& experts, long E) {
  const long T = experts.size(0), buckets = (E + 1) * (E + 2) / 2;
  long scratch = 0;
  done(mm_expert_plan_scratch((int)T, (int)buckets - 1, &scratch));
  const Tensor buf = i32({T + buckets + scratch}, experts);
  int* p = iptr(buf);
  done(mm_expert_plan_pairs(iptr(experts), (int)T, (int)E, p, p + buckets, scratch ? p + buckets + T : nullptr,
                            stream()));
  return {buf.narrow(0, 0, buckets), buf.narrow(0, buckets, T)};
}

hipStream_t raw_stream() { return c10::hip::getCurrentHIPStream().stream(); }

// the graph capture that a stream is part of
std::optional<unsigned long long> capture(hipStream_t s = raw_stream()) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  C10_HIP_CHECK(hipStreamGetCaptureInfo(s, &status, &id));
  if (status == hipStreamCaptureStatusNone) return std::nullopt;
  return id;
}

c10::Stream current_stream(const Tensor& t) {
  return c10::impl::VirtualGuardImpl(t.device().type()).getStream(t.device());
}

// The sorts wait until a product (or the caller) needs one: few rows need none, and rows of two choices may need the
// pairs' instead of the slots'.  The caller cannot see which call sorts and so cannot order another stream behind it:
// every stream sorts its own lists (an event for each sort costs every training call 5 us of the host, sorting once
// more only those that use several streams, 5 - 12 us of the GPU).  Under graph capture the slots are sorted at once,
// so that a captured plan follows every replay.  Outside that capture such a plan is sorted anew by every call: its
// experts change with the replays, and what its graph sorted holds nothing before the first.  A capture takes the lists
// that an older plan has from a stream outside the capture; those it has to sort are its own and are not kept.
struct Plan {
  struct Kept {
    hipStream_t stream;
    Lists lists;
  };
  Tensor experts;
  long T, k, E;
  std::optional<unsigned long long> made_in;   // the capture that the plan was made in, and its slots
  Lists captured;
  long version = 0;   // of experts
  std::vector<Kept> slots, rows;
  std::vector<c10::Stream> streams;   // that the allocator knows to use experts, which may be the plan's own copy

  // The lists and the experts are read together, and experts may be the caller's tensor: one that was written since the
  // plan was made is refused instead of being read beside older lists.  (A replay changes the experts of a captured
  // plan with its lists, and elsewhere such a plan is sorted anew; tensors of inference mode have no version.)
  void check() {
    if (experts.is_inference() || (made_in && made_in != capture())) return;
    if ((long)experts._version() != version)
      throw std::runtime_error("the experts of this plan were changed in place after plan_experts: make a new plan");
  }

  void use() {
    check();
    const c10::Stream s = current_stream(experts);
    if (std::find(streams.begin(), streams.end(), s) != streams.end()) return;
    experts.record_stream(s);
    streams.push_back(s);
  }

  template <typename F>
  Lists keep(std::vector<Kept>& kept, F make) {
    const hipStream_t s = raw_stream();
    if (made_in) return make(experts, E);
    if (capture()) {
      const c10::hip::HIPStreamCaptureModeGuard relaxed(hipStreamCaptureModeRelaxed);
      for (const Kept& q : kept) {
        if (q.stream == s || capture(q.stream)) continue;
        C10_HIP_CHECK(hipStreamSynchronize(q.stream));   // a capture cannot wait for work outside it: the host does
        return q.lists;
      }
      return make(experts, E);
    }
    for (const Kept& q : kept)
      if (q.stream == s) return q.lists;
    kept.push_back({s, make(experts, E)});
    return kept.back().lists;
  }
  Lists lists() {
    check();
    return made_in && made_in == capture() ? captured : keep(slots, make_lists);
  }
  Lists pairs() { return keep(rows, make_pairs); }
};

std::shared_ptr<Plan> plan_experts(const Tensor& experts0, int64_t E) {
  const Tensor experts = plain(experts0);
  if (!experts.is_cuda()) throw py::type_error("experts must be a GPU tensor");
  if (experts.scalar_type() != at::kInt && experts.scalar_type() != at::kLong)
    throw py::type_error(text("experts must be int32 or int64, got ", type_name(experts.scalar_type())));
  if (experts.device().index() != c10::hip::current_device())
    throw py::value_error(text("experts is on ", experts.device(), ", the current device is cuda:",
                               (int)c10::hip::current_device()));
  if (experts.dim() != 2 || experts.size(1) == 0)
    throw py::value_error(text("experts must be [rows, k], got ", experts.sizes()));
  if (E < 1 || E > kMaxExperts) throw py::value_error(text("n_experts must be 1 .. ", kMaxExperts, ", got ", E));
  refuse_modes("plan_experts", {});
  const long S = experts.numel();
  if (S > kInt32Max) throw py::value_error(text("more than 2^31 - 1 slots (", S, ")"));
  auto p = std::make_shared<Plan>();
  // values outside int32 must not wrap into the range of the experts
  p->experts = (experts.scalar_type() == at::kLong ? experts.clamp(-1, E).to(at::kInt) : experts).contiguous();
  p->T = experts.size(0);
  p->k = experts.size(1);
  p->E = E;
  if (!p->experts.is_inference()) p->version = (long)p->experts._version();
  p->streams = {current_stream(p->experts)};
  p->made_in = capture();
  if (p->made_in) p->captured = make_lists(p->experts, E);
  return p;
}

// ------------------------------------------------------------------------------------------------ products
struct Sizes { long T, M, D, F, E, k; };

// Whether rows go straight through their blocks (mm_expert_few), without a plan and without joining slots: while the
// blocks' bytes that they read, mostly from the L2s, stay below 64 MB.  Measured (us, straight against sorted): 128 ->
// 128 float, 2 of 8 experts: 1 row 3.5 / 13, 128 rows (17 MB) 4.5 / 15, 512 rows (67 MB) 10 / 15, 1000 rows 18 / 16;
// 1024 -> 1024 bfloat16, 4 of 64: 1 row 8 / 22, 8 rows (67 MB) 22 / 27, 16 rows 38 / 29, 64 rows 139 / 32; the same in
// float: 4 rows (67 MB) 21 / 70, 8 rows 39 / 72.
bool few_rows(const Sizes& n, int code) {
  const double bytes = (double)n.T * n.M * n.k * n.D * n.F * (code == 0 ? 4 : 2);
  return bytes <= 64e6 && n.T <= 65535 && n.M <= 65535;
}

// t [T, D] or [T, M, D] as [T, M, D] with a contiguous last axis.  Taken inside the autograd function, where a view
// costs no node of its own (two views outside took 6 - 10 us of a training call).
Tensor inner(const Tensor& t0) {
  const Tensor t = t0.dim() == 2 ? t0.unsqueeze(1) : t0;
  return t.size(2) > 1 && t.stride(2) != 1 ? t.contiguous() : t;
}

// Whether the choices of a row are joined before they are written (mm_expert_joined) instead of through fp32 rows of
// the slots; K values a row go in, N come out.  One choice: always (65,536 rows, 8 experts, us, joined / slots: 128 ->
// 128 float 25 / 37, bfloat16 16 / 29; 16,384 rows 1024 -> 1024 float 259 / 270, bfloat16 59 / 99).  Two choices:
// where every pair of experts fills tiles of rows and enough values are not written and read again to pay for the
// pairs' plan (15 us): float up to 128 values from 2 M results on (98,304 rows 128 -> 128: 44 / 70), beyond that
// splitting the operands of the small tiles costs more (256 -> 256, 65,536 rows: 159 / 173, 1024 -> 1024 521 / 484);
// 16-bit types from 16 M results on (65,536 rows 256 -> 256: 52 / 84; 98,304 rows 128 -> 128: 39 / 56).
bool join_rows(const Sizes& n, long K, long N, int code) {
  if (n.M > 64) return false;
  if (n.k == 1) return true;
  const long pairs = (n.E + 1) * (n.E + 2) / 2, results = n.T * n.M * N;
  if (n.k != 2 || n.E > 21 || n.T * n.M < 128 * pairs) return false;
  return code == 0 ? K <= 128 && n.M <= 16 && results >= 2000000 : results >= 16000000;
}

// dx with dgates likewise: all columns in one workgroup, two choices for float only (bfloat16, DG: 57 / 67, but 41 /
// 36 with 3 components)
bool join_gradients(const Sizes& n, int code, bool dgates) {
  return join_rows(n, n.F, n.D, code) && (!dgates || (n.D <= 128 && (n.k == 1 || code == 0)));
}

struct ExpertLinearFn : torch::autograd::Function<ExpertLinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Maybe& gates,
                        const std::shared_ptr<Plan>& plan, int64_t code) {
    const Tensor w = weight.contiguous(), g = gates ? gates->contiguous() : Tensor();
    const Sizes n = sizes(x, w, plan->experts);
    // Asked of the caller's tensors: copies made in here have no gradient.  The backward takes its path from what is
    // saved, as it has only these lists.
    const bool dg = gates && gates->requires_grad(), dxg = x.requires_grad() || dg;
    const bool joined = join_gradients(n, (int)code, dg);
    Lists l, p;   // the backward's
    if (weight.requires_grad() || (dxg && !(joined && n.k == 2))) l = plan->lists();
    if (dxg && joined && n.k == 2) p = plan->pairs();
    ctx->save_for_backward({x, w, g, plan->experts, l.offsets, l.order, p.offsets, p.order});
    ctx->saved_data["args"] = std::vector<int64_t>{code, joined, n.T, n.M, n.D, n.F, n.E, n.k};
    return run(x, w, g, *plan, (int)code);
  }

  static Sizes sizes(const Tensor& x, const Tensor& w, const Tensor& experts) {
    return Sizes{x.size(0), x.dim() == 2 ? 1 : x.size(1), x.size(-1), w.size(2), w.size(0), experts.size(1)};
  }

  static Tensor run(const Tensor& x0, const Tensor& w, const Tensor& gates, Plan& plan, int code) {
    const Tensor& experts = plan.experts;
    plan.use();
    const Sizes n = sizes(x0, w, experts);
    const Tensor x = inner(x0);
    Tensor y = x0.dim() == 2 ? at::empty({n.T, n.F}, x.options()) : at::empty({n.T, n.M, n.F}, x.options());
    const int T = (int)n.T, k = (int)n.k, M = (int)n.M, D = (int)n.D, F = (int)n.F, E = (int)n.E;
    if (few_rows(n, code)) {
      done(mm_expert_few(ptr(x), x.stride(0), x.stride(1), code, T, k, M, D, F, ptr(w), E, fptr(gates),
                         iptr(experts), ptr(y), stream()));
      return y;
    }
    if (join_rows(n, n.D, n.F, code)) {
      const Lists l = k == 2 ? plan.pairs() : plan.lists();
      done(mm_expert_joined(ptr(x), x.stride(0), x.stride(1), code, T, k, M, D, F, ptr(w), 0, E, fptr(gates),
                            iptr(experts), iptr(l.offsets), iptr(l.order), ptr(y), nullptr, 0, 0, nullptr, stream()));
      return y;
    }
    const Lists l = plan.lists();
    const Tensor rows = f32({n.T * n.k, n.M, n.F}, x);
    done(mm_expert_rows(ptr(x), x.stride(0), x.stride(1), code, T * k, k, M, D, F, ptr(w), 0, E, iptr(l.offsets),
                        iptr(l.order), fptr(rows), stream()));
    done(mm_expert_combine(fptr(rows), fptr(gates), iptr(experts), code, n.T, k, M, F, E, ptr(y), stream()));
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto args = ctx->saved_data["args"].toIntVector();
    const int code = (int)args[0];
    const Sizes n{args[2], args[3], args[4], args[5], args[6], args[7]};
    const Tensor dy = inner(plain(grads[0]));
    const auto type = type_of(code);
    const Tensor x = inner(grads[0].dim() == 2 ? unpacked(saved[0], {n.T, n.D}, type, dy, "x")
                                               : unpacked(saved[0], {n.T, n.M, n.D}, type, dy, "x"));
    const Tensor w = unpacked_dense(saved[1], {n.E, n.D, n.F}, type, dy, "weight");
    const Tensor gates = unpacked_dense(saved[2], {n.T, n.k}, at::kFloat, dy, "gates");
    const Tensor experts = unpacked_dense(saved[3], {n.T, n.k}, at::kInt, dy, "experts");
    const Tensor offsets = unpacked_dense(saved[4], {n.E + 1}, at::kInt, dy, "offsets");
    const Tensor order = unpacked_dense(saved[5], {n.T * n.k}, at::kInt, dy, "order");
    const Tensor pair_offsets = unpacked_dense(saved[6], {(n.E + 1) * (n.E + 2) / 2}, at::kInt, dy, "pairs");
    const Tensor pair_order = unpacked_dense(saved[7], {n.T}, at::kInt, dy, "pairs' order");
    const int S = (int)(n.T * n.k), k = (int)n.k, M = (int)n.M, D = (int)n.D, F = (int)n.F, E = (int)n.E;
    Tensor dx, dw, dg;
    if (ctx->needs_input_grad(0)) dx = at::empty(saved[0].sizes(), x.options());
    if (ctx->needs_input_grad(1)) dw = at::empty({n.E, n.D, n.F}, x.options());
    if (gates.defined() && ctx->needs_input_grad(2)) dg = f32({n.T, n.k}, x);
    if ((dx.defined() || dg.defined()) && args[1]) {
      const bool pairs = k == 2;
      done(mm_expert_joined(ptr(dy), dy.stride(0), dy.stride(1), code, (int)n.T, k, M, F, D, ptr(w), 1, E, fptr(gates),
                            iptr(experts), iptr(pairs ? pair_offsets : offsets), iptr(pairs ? pair_order : order),
                            ptr(dx), ptr(x), x.stride(0), x.stride(1), fptr(dg), stream()));
    } else if (dx.defined() || dg.defined()) {
      const Tensor rows = f32({S, M, D}, x);
      done(mm_expert_rows(ptr(dy), dy.stride(0), dy.stride(1), code, S, k, M, F, D, ptr(w), 1, E, iptr(offsets),
                          iptr(order), fptr(rows), stream()));
      done(mm_expert_combine_bwd(fptr(rows), fptr(gates), iptr(experts), ptr(x), x.stride(0), x.stride(1), code, n.T, k,
                                 M, D, E, ptr(dx), fptr(dg), stream()));
    }
    if (dw.defined()) {
      size_t bytes = 0;
      done(mm_expert_wgrad_workspace(S, M, D, F, E, &bytes));
      Tensor ws;
      if (bytes) ws = f32({(int64_t)(bytes / sizeof(float))}, x);
      done(mm_expert_wgrad(ptr(x), x.stride(0), x.stride(1), ptr(dy), dy.stride(0), dy.stride(1), code, S, k, M, D, F,
                           E, fptr(gates), iptr(offsets), iptr(order), ptr(dw), fptr(ws), stream()));
    }
    variable_list out(5);
    out[0] = dx;
    out[1] = dw;
    out[2] = dg;
    return once(out, "expert_linear");
  }
};

Tensor expert_linear(const Tensor& x1, const Tensor& weight1, const Maybe& gates, const std::shared_ptr<Plan>& plan) {
  const Tensor x0 = plain(x1), weight = plain(weight1);
  const int code = check_gpu(x0, "x");
  if (check_gpu(weight, "weight") != code)
    throw py::type_error(text("weight must be ", type_name(x0.scalar_type()), " (as x), got ",
                              type_name(weight.scalar_type())));
  if ((x0.dim() != 2 && x0.dim() != 3) || weight.dim() != 3)
    throw py::value_error(text("x must be [rows, D] or [rows, components, D] and weight [experts, D, F], got ",
                               x0.sizes(), " and ", weight.sizes()));
  if (!plan) throw py::type_error("plan must be an ExpertPlan (plan_experts)");
  const long T = plan->T, k = plan->k, E = plan->E;
  if (x0.size(0) != T) throw py::value_error(text("x has ", x0.size(0), " rows, the plan ", T));
  if (weight.size(0) != E || weight.size(1) != x0.size(-1) || weight.size(1) == 0 || weight.size(2) == 0)
    throw py::value_error(text("weight must be [", E, ", ", x0.size(-1), ", F], got ", weight.sizes()));
  if (x0.dim() == 3 && x0.size(1) == 0) throw py::value_error("x has no components");
  if (weight.size(1) > kMaxRows || weight.size(2) > kMaxRows) throw py::value_error("weight blocks are too large");
  Tensor g;
  if (gates) {
    g = plain(*gates);
    check_gpu(g, "gates");
    if (g.scalar_type() != at::kFloat)
      throw py::type_error(text("gates must be float32, got ", type_name(g.scalar_type())));
    if (g.dim() != 2 || g.size(0) != T || g.size(1) != k)
      throw py::value_error(text("gates must be [", T, ", ", k, "], got ", g.sizes()));
  }
  const Tensor& experts = plan->experts;
  if (experts.device() != x0.device()) throw py::value_error("x and the plan must be on one device");
  const long slots = T * k * (x0.dim() == 2 ? 1 : x0.size(1));
  if (slots > kMaxRows) throw py::value_error(text(slots, " rows: more than 2^31 - 2^16 are not supported"));
  refuse_modes("expert_linear", {&x0, &weight, &g});
  if (needs_grad({&x0, &weight, &g})) return ExpertLinearFn::apply(x0, weight, maybe(g), plan, (int64_t)code);
  return ExpertLinearFn::run(x0, weight.contiguous(), g.defined() ? g.contiguous() : g, *plan, code);
}
}  // namespace

PYBIND11_MODULE(mm_torch_ops, m) {
  m.def("version", []() { return mm_version(); });
  m.def("layer_norm", &layer_norm);
  m.def("route", &route);
  py::class_<Plan, std::shared_ptr<Plan>>(m, "ExpertPlan")
      .def_property_readonly("experts", [](Plan& p) { return p.experts; })
      .def_property_readonly("n_experts", [](Plan& p) { return p.E; })
      .def_property_readonly("offsets", [](Plan& p) { return p.lists().offsets; })
      .def_property_readonly("order", [](Plan& p) { return p.lists().order; })
      .def_property_readonly("counts", [](Plan& p) {
        const Tensor o = p.lists().offsets;
        return at::sub(o.narrow(0, 1, p.E), o.narrow(0, 0, p.E));
      });
  m.def("plan_experts", &plan_experts);
  m.def("expert_linear", &expert_linear);
}

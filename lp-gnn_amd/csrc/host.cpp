// lpgnn._host: the host side of calls that are bound by it.
//
// A layer norm of a small graph or the optimizer step of a small model is a few microseconds of GPU time;
// checking the arguments, the autograd node and the launch from Python took 14 us a layer norm, 142 its
// training pass (a Python node in the engine's thread waits for the interpreter lock) and 42 a step over 24
// tensors.  Here the same checks, the autograd node and the call of the C entry (include/lpgnn.h, resolved
// from the library that lpgnn._lib loads) run in C++: 5, 30 to 65 (the engine's hand-over between threads;
// 14 of it are this file's and the launches) and 6 us.
//
// Every refusal is a RuntimeError before any device work; device, stream and allocator are torch's current
// ones of the tensors' device.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <optional>
#include <stdexcept>
#include <unordered_set>
#include <vector>

#include "lpgnn.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

#define REQUIRE(cond, ...)                                   \
  do {                                                       \
    if (!(cond)) throw std::runtime_error(c10::str(__VA_ARGS__)); \
  } while (0)

// ------------------------------------------------------------------ the library
struct Lib {
  decltype(&lpg_last_error) last_error = nullptr;
  decltype(&lpg_layer_norm_fwd) layer_norm_fwd = nullptr;
  decltype(&lpg_layer_norm_bwd_workspace_bytes) layer_norm_bwd_workspace_bytes = nullptr;
  decltype(&lpg_layer_norm_bwd) layer_norm_bwd = nullptr;
  decltype(&lpg_adamw) adamw = nullptr;
  decltype(&lpg_adamw8) adamw8 = nullptr;
  decltype(&lpg_grad_norm_workspace_bytes) grad_norm_workspace_bytes = nullptr;
  decltype(&lpg_grad_norm) grad_norm = nullptr;
  decltype(&lpg_i8_chunk_rows) i8_chunk_rows = nullptr;
  decltype(&lpg_quant_i8) quant_i8 = nullptr;
  decltype(&lpg_fc_i8) fc_i8 = nullptr;
  decltype(&lpg_fc_i8_rows) fc_i8_rows = nullptr;
} L;

void open(const std::string &path) {
  void *h = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);  // (the one lpgnn._lib holds already)
  REQUIRE(h, "lpgnn: ", dlerror());
#define SYM(name)                                                               \
  L.name = reinterpret_cast<decltype(L.name)>(dlsym(h, "lpg_" #name));          \
  REQUIRE(L.name, "lpgnn: ", path, " has no lpg_" #name)
  SYM(last_error);
  SYM(layer_norm_fwd);
  SYM(layer_norm_bwd_workspace_bytes);
  SYM(layer_norm_bwd);
  SYM(adamw);
  SYM(adamw8);
  SYM(grad_norm_workspace_bytes);
  SYM(grad_norm);
  SYM(i8_chunk_rows);
  SYM(quant_i8);
  SYM(fc_i8);
  SYM(fc_i8_rows);
#undef SYM
}

void check(lpg_status st, const char *what) {  // lpgnn._lib.check
  if (st == LPG_OK) return;
  const char *kind = st == LPG_ERR_INVALID ? "invalid argument" : st == LPG_ERR_HIP ? "HIP error" : "unsupported";
  throw std::runtime_error(c10::str(what, ": ", kind, ": ", L.last_error()));
}

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
template <typename T>
T *ptr_of(const Tensor &t) {
  return static_cast<T *>(ptr(t));
}

int32_t code_of(at::ScalarType t) {
  return t == at::kBFloat16 ? LPG_BF16 : t == at::kHalf ? LPG_F16 : t == at::kFloat ? LPG_F32 : -1;
}

// the row stride of a matrix (that of a single row says nothing)
int64_t ld(const Tensor &t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// a call's workspace on the current device: torch's allocator without a tensor around it, given back in stream order
c10::DataPtr workspace(int64_t bytes) { return c10::GetAllocator(c10::DeviceType::CUDA)->allocate((size_t)bytes); }

// The operators have no forward-mode derivative: a dual tensor's tangent would be dropped, which reads as a derivative
// of zero.  (No tensor has one while no level of the mode is open: one look a call, not one a tensor -- 22 parameters'
// lists 7.6 us with the latter, 6.0 with the former.)
bool forward_mode() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }
void no_tangent(const char *what, const Tensor &t) {
  REQUIRE(!t.defined() || !t._fw_grad(0).defined(), "lpgnn ", what, ": there is no forward-mode derivative");
}
void no_tangent(const char *what, const OptTensor &t) {
  if (t) no_tangent(what, *t);
}

// t as [rows, D] with contiguous rows (a copy only where its strides allow no view)
Tensor rows(const Tensor &t) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return (r.stride(1) == 1 || r.size(1) == 1) && ld(r) >= r.size(1) ? r : r.contiguous();
}

bool capturing() {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  return hipStreamIsCapturing(c10::hip::getCurrentHIPStream().stream(), &st) == hipSuccess &&
         st != hipStreamCaptureStatusNone;
}

// ------------------------------------------------------------------ layer norm
int32_t weight_code(const Tensor &w, const Tensor &b) {
  return w.defined() ? code_of(w.scalar_type()) : b.defined() ? code_of(b.scalar_type()) : LPG_F32;
}

Tensor norm_forward(const Tensor &x, const Tensor &w, const Tensor &b, double eps, bool relu, Tensor *stats) {
  const c10::DeviceGuard guard(x.device());
  const int64_t M = x.size(0), D = x.size(1);
  Tensor y = at::empty({M, D}, x.options());
  if (stats) *stats = at::empty({2, M}, x.options().dtype(at::kFloat));
  float *mean = stats ? stats->data_ptr<float>() : nullptr;
  check(L.layer_norm_fwd(code_of(x.scalar_type()), weight_code(w, b), M, D, x.data_ptr(), ld(x), ptr(w), ptr(b),
                         (float)eps, relu ? LPG_NORM_RELU : 0, y.data_ptr(), D, mean, mean ? mean + M : nullptr,
                         stream_of(x)),
        "lpg_layer_norm_fwd");
  return y;
}

// What a backward under create_graph hands on: a gradient that depends on what it was computed from by an error
// (without it a loss that holds a gradient's norm beside other terms would just miss that term's part).
struct NoSecond : torch::autograd::Function<NoSecond> {
  static Tensor forward(torch::autograd::AutogradContext *, const Tensor &t, const Tensor &, const Tensor &,
                        const OptTensor &, const OptTensor &) {
    return t.view_as(t);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *, torch::autograd::variable_list) {
    throw std::runtime_error("lpgnn layer_norm: there is no second derivative");
  }
};

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const OptTensor &weight,
                        const OptTensor &bias, double eps, bool relu) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    Tensor stats;
    Tensor y = norm_forward(x, w, b, eps, relu, &stats);
    ctx->save_for_backward({x, w, b, stats});
    ctx->saved_data["relu"] = relu;
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &stats = saved[3];
    const c10::DeviceGuard guard(x.device());
    const int64_t M = x.size(0), D = x.size(1);
    const Tensor dy = rows(grads[0]);
    Tensor dx, dw, db;
    c10::DataPtr ws;
    const size_t bi = w.defined() ? 2 : 1;  // (the node's edges are its tensors: one less without a weight)
    if (ctx->needs_input_grad(0)) dx = at::empty({M, D}, x.options());
    if (w.defined() && ctx->needs_input_grad(1)) dw = at::empty({D}, w.options());
    if (b.defined() && ctx->needs_input_grad(bi)) db = at::empty({D}, b.options());
    if (dw.defined() || db.defined())
      ws = workspace(L.layer_norm_bwd_workspace_bytes(M, D));
    const float *mean = stats.data_ptr<float>();
    check(L.layer_norm_bwd(code_of(x.scalar_type()), weight_code(w, b), M, D, x.data_ptr(), ld(x), dy.data_ptr(),
                           ld(dy), ptr(w), ptr(b), mean, mean + M,
                           ctx->saved_data["relu"].toBool() ? LPG_NORM_RELU : 0, ptr(dx), D, ptr(dw), ptr(db), ws.get(),
                           stream_of(x)),
          "lpg_layer_norm_bwd");
    if (at::GradMode::is_enabled()) {
      const auto opt = [](const Tensor &t) { return t.defined() ? OptTensor(t) : std::nullopt; };
      for (Tensor *t : {&dx, &dw, &db})
        if (t->defined()) *t = NoSecond::apply(*t, x, grads[0], opt(w), opt(b));
    }
    return {dx, dw, db, Tensor(), Tensor()};
  }
};

// A backward that is captured while an eager graph of the same leaves lives would add to their gradients on the eager
// graph's stream, out of the capture, which ends the process: refused in the forward, before there is one.  The leaves
// are those behind t's whole graph (a view or a cast of a parameter has the parameter's).
void no_eager_leaf(const Tensor &t) {
  using torch::autograd::Node;
  const auto id = c10::hip::getCurrentHIPStream(t.get_device()).id();
  const auto check_leaf = [&](Node *acc) {
    const auto stream = acc->stream();
    REQUIRE(!stream || stream->id() == id,
            "lpgnn layer_norm: captured while an eager autograd graph of the same parameters lives; drop it first");
  };
  if (t.is_leaf()) {
    if (const auto acc = torch::autograd::impl::try_get_grad_accumulator(t)) check_leaf(acc.get());
    return;
  }
  std::unordered_set<Node *> seen{t.grad_fn().get()};
  std::vector<Node *> todo(seen.begin(), seen.end());
  while (!todo.empty()) {
    Node *const n = todo.back();
    todo.pop_back();
    if (dynamic_cast<torch::autograd::AccumulateGrad *>(n)) check_leaf(n);
    for (const auto &e : n->next_edges())
      if (e.function && seen.insert(e.function.get()).second) todo.push_back(e.function.get());
  }
}

Tensor layer_norm(const Tensor &x, const OptTensor &weight, const OptTensor &bias, double eps, bool relu) {
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  if (forward_mode())
    for (const Tensor *t : {&x, &w, &b}) no_tangent("layer_norm", *t);
  REQUIRE(x.is_cuda(), "lpgnn layer_norm: runs on a HIP device only (no CPU path)");
  REQUIRE(code_of(x.scalar_type()) >= 0, "lpgnn layer_norm: x must be float32, bfloat16 or float16, got ",
          x.scalar_type());
  REQUIRE(x.dim() > 0 && x.size(-1) > 0, "lpgnn layer_norm: x needs a last dimension to normalise, got shape ", x.sizes());
  REQUIRE(eps >= 0, "lpgnn layer_norm: eps must not be negative, got ", eps);
  for (const Tensor &p : {w, b}) {
    if (!p.defined()) continue;
    const char *name = p.is_same(w) ? "weight" : "bias";
    REQUIRE(p.dim() == 1 && p.size(0) == x.size(-1) && p.device() == x.device(), "lpgnn layer_norm: ", name, " must be [",
            x.size(-1), "] on ", x.device(), ", got ", p.sizes(), " on ", p.device());
    REQUIRE(p.scalar_type() == at::kFloat || p.scalar_type() == x.scalar_type(), "lpgnn layer_norm: ", name,
            " must be float32 or ", x.scalar_type(), ", got ", p.scalar_type());
  }
  REQUIRE(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(),
          "lpgnn layer_norm: weight and bias must share a type, got ", w.scalar_type(), " and ", b.scalar_type());
  const auto grad = [](const Tensor &t) { return t.defined() && t.requires_grad(); };
  const c10::DeviceGuard guard(x.device());
  if (at::GradMode::is_enabled() && capturing())
    for (const Tensor *t : {&x, &w, &b})
      if (grad(*t)) no_eager_leaf(*t);
  const auto packed = [](const OptTensor &t) { return t ? OptTensor(t->contiguous()) : t; };
  const Tensor xr = rows(x);
  const OptTensor wc = packed(weight), bc = packed(bias);
  const bool graph = at::GradMode::is_enabled() && (grad(x) || grad(w) || grad(b));
  const Tensor y = graph ? LayerNorm::apply(xr, wc, bc, eps, relu)
                         : norm_forward(xr, wc.value_or(Tensor()), bc.value_or(Tensor()), eps, relu, nullptr);
  return x.dim() == 2 ? y : y.view(x.sizes());
}

// ------------------------------------------------------------------ many tensors
// A Python list or tuple of tensors, borrowed for the call (which keeps the interpreter lock and the list): no
// reference counts, no vector of copies.
struct Tensors {
  pybind11::object fast;
  PyObject **items = nullptr;
  size_t n = 0;
  Tensors(pybind11::handle list, const char *what) {
    fast = pybind11::reinterpret_steal<pybind11::object>(PySequence_Fast(list.ptr(), "lpgnn: a list of tensors"));
    if (!fast) throw pybind11::error_already_set();
    n = (size_t)PySequence_Fast_GET_SIZE(fast.ptr());
    items = PySequence_Fast_ITEMS(fast.ptr());
    for (size_t i = 0; i < n; ++i)
      if (!THPVariable_Check(items[i])) throw pybind11::type_error(c10::str("lpgnn ", what, ": the lists hold tensors"));
  }
  size_t size() const { return n; }
  bool empty() const { return n == 0; }
  const Tensor &operator[](size_t i) const { return THPVariable_Unpack(items[i]); }
};

void no_tangents(const char *what, std::initializer_list<const Tensors *> lists, const OptTensor &scale = std::nullopt) {
  if (!forward_mode()) return;
  for (const Tensors *ts : lists)
    for (size_t i = 0; i < ts->size(); ++i) no_tangent(what, (*ts)[i]);
  no_tangent(what, scale);
}

// `ts` beside the parameters `ps`: as many, one type, the parameters' device, contiguous, their sizes (or,
// scales, one number a block of 256)
void same(const char *what, const char *name, const Tensors &ts, const Tensors &ps, at::ScalarType type,
          bool blocks = false) {
  REQUIRE(ts.size() == ps.size(), "lpgnn ", what, ": ", ps.size(), " params and ", ts.size(), " ", name);
  for (size_t i = 0; i < ts.size(); ++i) {
    const Tensor &t = ts[i];
    REQUIRE(t.scalar_type() == type, "lpgnn ", what, ": ", name, " must be ", type, ", got ", t.scalar_type());
    REQUIRE(t.device() == ps[0].device(), "lpgnn ", what, ": ", name, " must be on the parameters' device");
    REQUIRE(t.layout() == at::kStrided && t.is_contiguous(), "lpgnn ", what, ": ", name, " must be contiguous");
    const int64_t n = ps[i].numel();
    REQUIRE(t.numel() == (blocks ? (n + 255) / 256 : n), "lpgnn ", what, ": ", name,
            " do not have the parameters' sizes");
  }
}

int32_t params(const char *what, const Tensors &ps) {
  REQUIRE(ps[0].is_cuda(), "lpgnn ", what, ": runs on a HIP device only (no CPU path)");
  const auto type = ps[0].scalar_type();
  REQUIRE(type == at::kFloat || type == at::kBFloat16, "lpgnn ", what, ": parameters must be float32 or bfloat16, got ",
          type);
  same(what, "params", ps, ps, type);
  return code_of(type);
}

// No memory that the step writes is another tensor's of the call (two blocks would race for it); read-only
// tensors may share.
struct Spans {
  struct Span {
    const char *at, *end;
    bool out;
  };
  std::vector<Span> list;
  void add(const Tensors &ts, bool out) {
    for (size_t i = 0; i < ts.size(); ++i) {
      const Tensor &t = ts[i];
      const char *p = static_cast<const char *>(t.data_ptr());
      if (t.numel() > 0) list.push_back({p, p + t.numel() * t.element_size(), out});
    }
  }
  void check(const char *what) {
    std::sort(list.begin(), list.end(), [](const Span &a, const Span &b) { return a.at < b.at; });
    const char *any = nullptr, *out = nullptr;  // the furthest ends so far
    for (const Span &s : list) {
      REQUIRE(s.at >= out && !(s.out && s.at < any), "lpgnn ", what,
              ": tensors of the call overlap (a parameter or a state tensor is in it twice?)");
      any = std::max(any, s.end);
      if (s.out) out = std::max(out, s.end);
    }
  }
};
void apart(const char *what, const Tensors &gs, const float *scale, std::initializer_list<const Tensors *> written) {
  Spans s;
  s.list.reserve(gs.size() * (1 + written.size()));
  s.add(gs, false);
  for (const Tensors *ts : written) s.add(*ts, true);
  s.check(what);
  if (!scale) return;
  const char *p = reinterpret_cast<const char *>(scale);
  for (const Spans::Span &x : s.list)
    REQUIRE(!x.out || p + sizeof(float) <= x.at || p >= x.end, "lpgnn ", what, ": grad_scale overlaps a tensor that is written");
}

lpg_adamw_hyper hyper(const char *what, int64_t step, double lr, std::pair<double, double> betas, double eps,
                      double weight_decay) {
  const double b1 = betas.first, b2 = betas.second;
  REQUIRE(step >= 1, "lpgnn ", what, ": step counts from 1, got ", step);
  REQUIRE(lr >= 0 && eps >= 0 && weight_decay >= 0 && b1 >= 0 && b1 < 1 && b2 >= 0 && b2 < 1, "lpgnn ", what,
          ": need lr, eps, weight_decay >= 0 and 0 <= betas < 1, got lr=", lr, " betas=(", b1, ", ", b2, ") eps=", eps,
          " weight_decay=", weight_decay);
  return {(float)b1, (float)(1 - b1), (float)b2, (float)(1 - b2), (float)(1 / std::sqrt(1 - std::pow(b2, (double)step))),
          (float)eps, (float)(1 - lr * weight_decay), (float)(lr / (1 - std::pow(b1, (double)step)))};
}

const float *scale_ptr(const char *what, const OptTensor &s, const Tensors &ps) {
  if (!s) return nullptr;
  REQUIRE(s->scalar_type() == at::kFloat && s->numel() == 1 && s->device() == ps[0].device(), "lpgnn ", what,
          ": grad_scale must be one float32 number on the parameters' device");
  return s->data_ptr<float>();
}

// the kernels write through pointers: tell autograd (and whatever keeps values by version), as an in-place op
void written(const Tensors &ts) {
  for (size_t i = 0; i < ts.size(); ++i)
    if (!ts[i].is_inference()) ts[i].unsafeGetTensorImpl()->bump_version();
}

using pybind11::handle;

void adamw_step(handle params_, handle grads, handle exp_avgs, handle exp_avg_sqs, int64_t step, double lr,
                std::pair<double, double> betas, double eps, double weight_decay, const OptTensor &grad_scale,
                bool check_only) {
  const char *what = "adamw_step";
  const Tensors ps(params_, what), gs(grads, what), ms(exp_avgs, what), vs(exp_avg_sqs, what);
  const lpg_adamw_hyper h = hyper(what, step, lr, betas, eps, weight_decay);
  no_tangents(what, {&ps, &gs, &ms, &vs}, grad_scale);
  if (ps.empty()) return;
  const int32_t type = params(what, ps);
  same(what, "grads", gs, ps, ps[0].scalar_type());
  same(what, "exp_avgs", ms, ps, at::kFloat);
  same(what, "exp_avg_sqs", vs, ps, at::kFloat);
  const float *scale = scale_ptr(what, grad_scale, ps);
  apart(what, gs, scale, {&ps, &ms, &vs});
  if (check_only) return;
  std::vector<lpg_adamw_tensor> tab(ps.size());
  for (size_t i = 0; i < ps.size(); ++i)
    tab[i] = {ps[i].data_ptr(), gs[i].data_ptr(), ptr_of<float>(ms[i]), ptr_of<float>(vs[i]), ps[i].numel()};
  const c10::DeviceGuard guard(ps[0].device());
  check(L.adamw(type, (int64_t)tab.size(), tab.data(), &h, scale, stream_of(ps[0])), "lpg_adamw");
  written(ps), written(ms), written(vs);
}

// The 32-bit integer hash of the kernels' random bits (fc_common.h lowbias32), for the rounding key of a
// tensor: of the seed, the step and the tensor's place in the list.
uint32_t mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0x7feb352du;
  x ^= x >> 15;
  x *= 0x846ca68bu;
  return x ^ (x >> 16);
}
uint32_t step_key(int64_t step, uint64_t seed) {
  return mix((uint32_t)seed ^ mix((uint32_t)(seed >> 32) ^ mix((uint32_t)step)));
}
int64_t rounding_key(int64_t place, int64_t step, uint64_t seed) {
  return mix(step_key(step, seed) + 0x9e3779b9u * (uint32_t)(place + 1));
}

void adamw_step_8bit(handle params_, handle grads, handle m8_, handle m_scales, handle r8_, handle r_scales,
                     const std::optional<std::vector<int64_t>> &places, uint64_t seed, int64_t step, double lr,
                     std::pair<double, double> betas, double eps, double weight_decay, const OptTensor &grad_scale,
                     bool check_only) {
  const char *what = "adamw_step_8bit";
  const Tensors ps(params_, what), gs(grads, what), m8(m8_, what), ms(m_scales, what), r8(r8_, what), rs(r_scales, what);
  const lpg_adamw_hyper h = hyper(what, step, lr, betas, eps, weight_decay);
  no_tangents(what, {&ps, &gs, &m8, &ms, &r8, &rs}, grad_scale);
  if (ps.empty()) return;
  const int32_t type = params(what, ps);
  REQUIRE(!places || places->size() == ps.size(), "lpgnn ", what, ": ", ps.size(), " params and ", places->size(),
          " places");
  same(what, "grads", gs, ps, ps[0].scalar_type());
  same(what, "m8", m8, ps, at::kFloat8_e4m3fn);
  same(what, "m_scales", ms, ps, at::kFloat, true);
  same(what, "r8", r8, ps, at::kFloat8_e4m3fn);
  same(what, "r_scales", rs, ps, at::kFloat, true);
  const float *scale = scale_ptr(what, grad_scale, ps);
  apart(what, gs, scale, {&ps, &m8, &ms, &r8, &rs});
  if (check_only) return;
  std::vector<lpg_adamw8_tensor> tab(ps.size());
  for (size_t i = 0; i < ps.size(); ++i)
    tab[i] = {ps[i].data_ptr(), gs[i].data_ptr(),      m8[i].data_ptr(), ptr_of<float>(ms[i]),
              r8[i].data_ptr(), ptr_of<float>(rs[i]), ps[i].numel(),
              rounding_key(places ? (*places)[i] : (int64_t)i, step, seed)};
  const c10::DeviceGuard guard(ps[0].device());
  check(L.adamw8(type, (int64_t)tab.size(), tab.data(), &h, scale, stream_of(ps[0])), "lpg_adamw8");
  written(ps), written(m8), written(ms), written(r8), written(rs);
}

std::pair<Tensor, Tensor> clip_scale(handle grads, double max_norm) {
  const char *what = "clip_scale";
  const Tensors gs(grads, what);
  no_tangents(what, {&gs});
  REQUIRE(!gs.empty(), "lpgnn clip_scale: no gradients");
  REQUIRE(max_norm >= 0, "lpgnn clip_scale: max_norm must not be negative, got ", max_norm);
  const int32_t type = params(what, gs);
  std::vector<lpg_tensor> tab(gs.size());
  for (size_t i = 0; i < gs.size(); ++i) tab[i] = {gs[i].data_ptr(), gs[i].numel()};
  const c10::DeviceGuard guard(gs[0].device());
  const auto f32 = gs[0].options().dtype(at::kFloat);
  Tensor norm = at::empty({}, f32), scale = at::empty({}, f32);
  const c10::DataPtr ws = workspace(L.grad_norm_workspace_bytes((int64_t)tab.size(), tab.data()));
  check(L.grad_norm(type, (int64_t)tab.size(), tab.data(), max_norm, norm.data_ptr<float>(), scale.data_ptr<float>(),
                    ws.get(), stream_of(norm)),
        "lpg_grad_norm");
  return {norm, scale};
}

// ------------------------------------------------------------------ 8-bit integers
// whole numbers have no derivative: nothing a call computes from may want one
void no_gradient(const char *what, const OptTensor &t) {
  if (forward_mode()) no_tangent(what, t);
  REQUIRE(!at::GradMode::is_enabled() || !t || !t->requires_grad(), "lpgnn ", what,
          ": 8-bit integers have no gradient (call it under torch.no_grad())");
}

// x [.., K1] (and x2 [.., K2], the same rows) as row matrices
std::pair<Tensor, Tensor> i8_rows(const char *what, const Tensor &x, const OptTensor &x2) {
  no_gradient(what, x);
  no_gradient(what, x2);
  REQUIRE(x.is_cuda(), "lpgnn ", what, ": runs on a HIP device only (no CPU path)");
  REQUIRE(code_of(x.scalar_type()) >= 0, "lpgnn ", what, ": x must be float32, bfloat16 or float16, got ",
          x.scalar_type());
  REQUIRE(x.dim() > 0 && x.size(-1) > 0, "lpgnn ", what, ": x needs columns, got shape ", x.sizes());
  if (!x2) return {rows(x), Tensor()};
  REQUIRE(x2->device() == x.device() && x2->scalar_type() == x.scalar_type() && x2->dim() == x.dim() &&
              x2->sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1) && x2->size(-1) > 0,
          "lpgnn ", what, ": x2 must have x's rows, type and device, got ", x2->sizes(), " ", x2->scalar_type(), " beside ",
          x.sizes(), " ", x.scalar_type());
  return {rows(x), rows(*x2)};
}

// rows [at, at + M) of [x | x2] into q [M, ldq] and s [M]
void quant(const Tensor &x, const Tensor &x2, int64_t at, int64_t M, int8_t *q, int64_t ldq, float *s) {
  const auto row = [&](const Tensor &t) { return static_cast<char *>(t.data_ptr()) + at * ld(t) * t.element_size(); };
  const bool two = x2.defined();
  check(L.quant_i8(code_of(x.scalar_type()), M, x.size(1), row(x), ld(x), two ? x2.size(1) : 0, two ? row(x2) : nullptr,
                   two ? ld(x2) : 0, q, ldq, s, stream_of(x)),
        "lpg_quant_i8");
}

int64_t code_pitch(const Tensor &x, const Tensor &x2) {
  return (x.size(1) + (x2.defined() ? x2.size(1) : 0) + 127) / 128 * 128;
}

std::pair<Tensor, Tensor> quantize_i8(const Tensor &x, const OptTensor &x2) {
  const auto [a, b] = i8_rows("quantize_i8", x, x2);
  const c10::DeviceGuard guard(x.device());
  const int64_t M = a.size(0), ldq = code_pitch(a, b);
  Tensor q = at::empty({M, ldq}, a.options().dtype(at::kChar)), s = at::empty({M}, a.options().dtype(at::kFloat));
  quant(a, b, 0, M, ptr_of<int8_t>(q), ldq, ptr_of<float>(s));
  return {q.narrow(1, 0, a.size(1) + (b.defined() ? b.size(1) : 0)), s};
}

Tensor linear_i8(const Tensor &x, const Tensor &wq, const Tensor &ws, const OptTensor &bias, const OptTensor &x2,
                 bool relu) {
  const char *what = "linear_i8";
  no_gradient(what, ws);
  no_gradient(what, bias);
  const auto [a, b] = i8_rows(what, x, x2);
  const int64_t M = a.size(0), K1 = a.size(1), K2 = b.defined() ? b.size(1) : 0, K = K1 + K2;
  REQUIRE(wq.dim() == 2 && wq.scalar_type() == at::kChar && wq.device() == x.device() && wq.size(1) == K && wq.size(0) > 0,
          "lpgnn linear_i8: wq must be int8 [N, ", K, "] on ", x.device(), ", got ", wq.scalar_type(), " ", wq.sizes(),
          " on ", wq.device());
  const int64_t N = wq.size(0);
  const auto vec = [&](const char *name, const Tensor &t) {
    REQUIRE(t.dim() == 1 && t.size(0) == N && t.scalar_type() == at::kFloat && t.device() == x.device(),
            "lpgnn linear_i8: ", name, " must be float32 [", N, "] on ", x.device(), ", got ", t.scalar_type(), " ",
            t.sizes(), " on ", t.device());
    return t.contiguous();
  };
  const Tensor scale = vec("ws", ws), bb = bias ? vec("bias", *bias) : Tensor();
  const c10::DeviceGuard guard(x.device());
  // rows of w on 16-byte borders, each readable to the next one, within the kernel's pitch (quantize_i8's are);
  // else a copy that is
  Tensor w = wq;
  const int64_t k16 = (K + 15) / 16 * 16;
  int64_t ldw = N > 1 ? w.stride(0) : k16;
  const bool room = (w.storage_offset() + (N - 1) * ldw + k16) <= (int64_t)w.storage().nbytes();
  if ((w.stride(1) != 1 && K > 1) || ldw < k16 || ldw % 16 || ldw > (1 << 22) || !room ||
      reinterpret_cast<uintptr_t>(w.data_ptr()) % 16) {
    w = at::empty({N, k16}, wq.options()).narrow(1, 0, K);
    w.copy_(wq);
    ldw = k16;
  }
  auto shape = x.sizes().vec();
  shape.back() = N;
  Tensor y = at::empty({M, N}, x.options());
  const int32_t type = code_of(x.scalar_type()), flags = relu ? LPG_FC_RELU : 0;
  if (M > 0) {
    const lpg_status st =
        L.fc_i8_rows(type, M, N, K1, a.data_ptr(), ld(a), K2, ptr(b), K2 ? ld(b) : 0, ptr_of<int8_t>(w),
                     ldw, ptr_of<float>(scale), ptr_of<float>(bb), flags, y.data_ptr(), N, stream_of(x));
    if (st != LPG_ERR_UNSUPPORTED) {  // (else: too many rows for one launch)
      check(st, "lpg_fc_i8_rows");
      return y.view(shape);
    }
  }
  if (M > 0) {
    const int64_t rows = L.i8_chunk_rows(M, N, K), most = rows < M ? rows + rows / 4 : M, ldq = code_pitch(a, b);
    const c10::DataPtr codes = workspace(most * ldq), scales = workspace(most * 4);
    int8_t *const q = static_cast<int8_t *>(codes.get());
    float *const s = static_cast<float *>(scales.get());
    for (int64_t at = 0, m; at < M; at += m) {
      m = std::min(L.i8_chunk_rows(M - at, N, K), most);
      quant(a, b, at, m, q, ldq, s);
      check(L.fc_i8(type, m, N, K, q, ldq, s, ptr_of<int8_t>(w), ldw, ptr_of<float>(scale),
                    ptr_of<float>(bb), flags, static_cast<char *>(y.data_ptr()) + at * N * y.element_size(), N,
                    stream_of(x)),
            "lpg_fc_i8");
    }
  }
  return y.view(shape);
}

}  // namespace

PYBIND11_MODULE(_host, m) {
  m.def("open", &open);
  m.def("layer_norm", &layer_norm);
  m.def("rounding_key", &rounding_key);
  m.def("adamw_step", &adamw_step);
  m.def("adamw_step_8bit", &adamw_step_8bit);
  m.def("clip_scale", &clip_scale);
  m.def("quantize_i8", &quantize_i8);
  m.def("linear_i8", &linear_i8);
}

// disco_torch.cpp -- torch's side of the residual join and the gradient norm (host code; the kernels are libdisco_hip.so's).
//
//   residual_norm, gradient_norm                                        what Python calls: checks of layout, the autograd nodes
//   residual_norm_forward, residual_norm_backward, grad_norm, grad_clip  what a trace holds: each is one call of a C entry
//
// A training pass over few rows is bound by what the host does around two launches: with the node in Python, whose backward
// has to take the interpreter from the thread that waits for it, a pass of forward and eight gradients took 213 us of host
// time, and takes 116 here (the forward 46 and 17).  Arguments are checked in disco_amd/residual.py (4 of the 10.4 us of a join of
// one row; the operators, two allocations and the launch are the rest); this file allocates, calls the C entries and keeps what
// the backward reads.  A list of gradients is read here too: an attribute of every tensor costs in Python what a launch does
// (norm and clipping of ten: 17 and 26 us, 12 and 13 here).  The entries' addresses come from the loaded library (bind), so
// there is one copy of it in the process.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/util/SmallVector.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include <algorithm>
#include <cstdint>
#include <memory>
#include <optional>
#include <utility>
#include <vector>

#include "../../include/disco_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

decltype(&disco_residual_norm_forward) g_forward = nullptr;
decltype(&disco_residual_norm_backward) g_backward = nullptr;
decltype(&disco_residual_norm_workspace_bytes) g_workspace = nullptr;
decltype(&disco_status_string) g_status = nullptr;
decltype(&disco_grad_norm) g_norm = nullptr;
decltype(&disco_grad_clip) g_clip = nullptr;
decltype(&disco_grad_norm_workspace_bytes) g_norm_workspace = nullptr;

void bind(int64_t forward, int64_t backward, int64_t workspace, int64_t status, int64_t norm, int64_t clip, int64_t norm_workspace) {
  g_norm = reinterpret_cast<decltype(g_norm)>(norm);
  g_clip = reinterpret_cast<decltype(g_clip)>(clip);
  g_norm_workspace = reinterpret_cast<decltype(g_norm_workspace)>(norm_workspace);
  g_forward = reinterpret_cast<decltype(g_forward)>(forward);
  g_backward = reinterpret_cast<decltype(g_backward)>(backward);
  g_workspace = reinterpret_cast<decltype(g_workspace)>(workspace);
  g_status = reinterpret_cast<decltype(g_status)>(status);
}

// The stream that is current where the call happens.  (A handle among the operator's arguments would become a constant of a
// traced module, which then launches on the stream of its tracing.)
void* stream_of(const at::Device& device) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(device.index()).stream(); }

// Without this a tensor that carries a tangent but needs no gradient would come back without one.
void refuse_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), what, " has no forward-mode derivatives");
}

void check(int status, const char* what) { TORCH_CHECK(status == DISCO_OK, what, ": ", g_status(status)); }

// What a call does besides its tensors, as residual.py packs it: two bits each of the post norm, the pre norm, the gate, its
// activation, the block's and the parameters' type, and one for the block itself.
struct Plan {
  int post, pre, gate, act, block_type, param_type, block;
  explicit Plan(int64_t p)
      : post(p & 3), pre(p >> 2 & 3), gate(p >> 4 & 3), act(p >> 6 & 3), block_type(p >> 8 & 3), param_type(p >> 10 & 3), block(p >> 12 & 1) {}
};

int type_code(const Tensor& t) {
  const auto s = t.scalar_type();
  return s == at::kFloat ? DISCO_F32 : s == at::kHalf ? DISCO_F16 : DISCO_BF16;
}
at::ScalarType type_of(int code) { return code == DISCO_F32 ? at::kFloat : code == DISCO_F16 ? at::kHalf : at::kBFloat16; }
const void* read(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* write(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
int64_t pitch(const Tensor& t, int64_t width) { return t.defined() ? t.stride(0) : width; }

// x, y, gate, scale, post weight and bias, pre weight and bias; an absent one is undefined
struct Operands { Tensor x, y, gate, scale, w1, b1, w2, b2; };
using Maybe = std::optional<Tensor>;
Operands operands(const Tensor& x, const Maybe& y, const Maybe& gate, const Maybe& scale, const Maybe& w1, const Maybe& b1, const Maybe& w2,
                  const Maybe& b2) {
  const auto get = [](const Maybe& t) { return t.has_value() ? *t : Tensor(); };
  return {x, get(y), get(gate), get(scale), get(w1), get(b1), get(w2), get(b2)};
}

disco_residual_norm describe(const Plan& p, const Operands& o, double scale, double eps) {
  disco_residual_norm d{};
  d.rows = o.x.size(0); d.width = o.x.size(1);
  d.ldx = o.x.stride(0); d.ldy = o.y.defined() ? o.y.stride(0) : 0; d.ld_gate = o.gate.defined() ? o.gate.stride(0) : 0;
  d.x = read(o.x); d.y = read(o.y); d.gate = read(o.gate);
  d.post_weight = read(o.w1); d.post_bias = read(o.b1); d.pre_weight = read(o.w2); d.pre_bias = read(o.b2); d.scale_vector = read(o.scale);
  d.stream_type = type_code(o.x); d.block_type = p.block_type; d.param_type = p.param_type;
  d.has_block = p.block; d.post_norm = p.post; d.pre_norm = p.pre; d.gate_kind = p.gate; d.gate_act = p.act;
  d.scale = (float)scale; d.eps = (float)eps;
  return d;
}

void bound() { TORCH_CHECK(g_forward && g_backward && g_workspace && g_status && g_norm && g_clip && g_norm_workspace, "disco_torch: not bound to libdisco_hip.so"); }

// ---- operators of the dispatcher: what a tracer, a fake tensor or a mode sees of a call ---------------------------------
// A call that went to the kernels around the dispatcher would leave nothing behind in a trace but its uninitialised outputs.

// out, h and, where the backward wants them, the rows' statistics.  Output rows lie densely: columns that nothing writes
// between them leave cache lines half written (the norm of 2.4 M rows of 41 floats: 268 us with rows padded to 44, 170 dense).
variable_list forward_outputs(const Plan& p, const Tensor& x, bool keep) {
  variable_list r;
  if (p.block) r.push_back(at::empty_symint(x.sym_sizes(), x.options()));
  if (p.pre) r.push_back(at::empty_symint(x.sym_sizes(), x.options().dtype(type_of(p.block_type))));
  if (keep) r.push_back(at::empty_symint({4 * x.sym_size(0)}, x.options().dtype(at::kFloat)));
  return r;
}

variable_list forward_op(const Tensor& x, const Maybe& y, const Maybe& gate, const Maybe& scale, const Maybe& w1, const Maybe& b1, const Maybe& w2,
                         const Maybe& b2, int64_t plan, double factor, double eps, bool keep) {
  bound();
  const Plan p(plan);
  const Operands o = operands(x, y, gate, scale, w1, b1, w2, b2);
  const c10::DeviceGuard guard(x.device());
  variable_list r = forward_outputs(p, x, keep);
  const Tensor out = p.block ? r[0] : Tensor(), h = p.pre ? r[p.block] : Tensor(), stats = keep ? r.back() : Tensor();
  const disco_residual_norm d = describe(p, o, factor, eps);
  check(g_forward(&d, write(out), pitch(out, 0), write(h), pitch(h, 0), static_cast<float*>(write(stats)), stream_of(x.device())),
        "disco_residual_norm_forward");
  return r;
}

variable_list forward_meta(const Tensor& x, const Maybe&, const Maybe&, const Maybe&, const Maybe&, const Maybe&, const Maybe&, const Maybe&, int64_t plan,
                           double, double, bool keep) {
  return forward_outputs(Plan(plan), x, keep);
}

// Rows with unit column stride that do not overlap, or one row for all: the tensor or a copy.
Tensor rows(const Tensor& t) {
  if (!t.defined() || t.is_contiguous()) return t;
  const int64_t n = t.size(0), width = t.size(1), r = t.stride(0), c = t.stride(1);
  return (width > 1 && c != 1) || (n > 1 && r > 0 && r < width) ? t.contiguous() : t;
}

// The operands' gradients that `wanted` names (a bit for each operand, in the operator's order), in that order.
variable_list backward_outputs(const Plan& p, const Operands& o, int64_t wanted) {
  variable_list r;
  const Tensor* all[] = {&o.x, &o.y, &o.gate, &o.scale, &o.w1, &o.b1, &o.w2, &o.b2};
  for (int i = 0; i < 8; ++i) {
    const Tensor& t = all[i]->defined() ? *all[i] : o.x;      // y, where it was not kept
    if (wanted >> i & 1) r.push_back(at::empty_symint(t.sym_sizes(), i == 1 ? t.options().dtype(type_of(p.block_type)) : t.options()));
  }
  return r;
}

variable_list backward_op(const Maybe& dout_, const Maybe& dh_, const Maybe& stats, const Maybe& x, const Maybe& y, const Maybe& gate, const Maybe& scale,
                          const Maybe& w1, const Maybe& b1, const Maybe& w2, const Maybe& b2, int64_t plan, double factor, double eps, int64_t wanted) {
  bound();
  const Plan p(plan);
  const Tensor dout = rows(dout_.value_or(Tensor())), dh = rows(dh_.value_or(Tensor()));
  const Operands o = operands(x.value_or(dout), y, gate, scale, w1, b1, w2, b2);      // dout: of x's shape and type
  const c10::DeviceGuard guard(o.x.device());
  const int64_t n = o.x.size(0), width = o.x.size(1);
  variable_list r = backward_outputs(p, o, wanted);
  size_t next = 0;
  const auto gradient = [&](int i) { return wanted >> i & 1 ? r[next++] : Tensor(); };
  const Tensor dx = gradient(0), dy = gradient(1), dgate = gradient(2), dscale = gradient(3), dw1 = gradient(4), db1 = gradient(5), dw2 = gradient(6),
               db2 = gradient(7);
  const size_t bytes = g_workspace(n, width);
  const Tensor ws = at::empty({(int64_t)bytes}, o.x.options().dtype(at::kByte));
  const disco_residual_norm d = describe(p, o, factor, eps);
  disco_residual_norm_grads g{};
  g.dout = read(dout); g.dh = read(dh);
  g.dx = write(dx); g.dy = write(dy); g.dgate = write(dgate); g.dscale = write(dscale);
  g.dpost_weight = write(dw1); g.dpost_bias = write(db1); g.dpre_weight = write(dw2); g.dpre_bias = write(db2);
  g.ld_dout = pitch(dout, width); g.ld_dh = pitch(dh, width); g.ld_dx = pitch(dx, width); g.ld_dy = pitch(dy, width); g.ld_dgate = pitch(dgate, width);
  // autograd makes the forward's stream current for its node, whichever one the caller of the backward is on
  check(g_backward(&d, static_cast<const float*>(read(stats.value_or(Tensor()))), &g, write(ws), bytes, stream_of(o.x.device())),
        "disco_residual_norm_backward");
  return r;
}

variable_list backward_meta(const Maybe& dout, const Maybe&, const Maybe&, const Maybe& x, const Maybe& y, const Maybe& gate, const Maybe& scale,
                            const Maybe& w1, const Maybe& b1, const Maybe& w2, const Maybe& b2, int64_t plan, double, double, int64_t wanted) {
  return backward_outputs(Plan(plan), operands(x.has_value() ? *x : *dout, y, gate, scale, w1, b1, w2, b2), wanted);
}

// The tensors of a list as the C entries take them.
struct List {
  std::vector<const void*> src;
  std::vector<void*> dst;
  std::vector<int64_t> numel;
  std::vector<int> type, out_type;
  Tensor ws, norm;
  List(at::TensorList grads, const at::TensorList* out) : src(grads.size()), dst(out ? grads.size() : 0), numel(grads.size()), type(grads.size()),
                                                          out_type(out ? grads.size() : 0) {
    bound();
    const auto options = at::TensorOptions().device(grads[0].device());
    ws = at::empty({(int64_t)g_norm_workspace((int64_t)grads.size())}, options.dtype(at::kByte));
    norm = at::empty({}, options.dtype(at::kFloat));
    for (size_t i = 0; i < grads.size(); ++i) {
      src[i] = grads[i].const_data_ptr();
      numel[i] = grads[i].numel();
      type[i] = type_code(grads[i]);
      if (!out) continue;
      dst[i] = (*out)[i].mutable_data_ptr();
      out_type[i] = type_code((*out)[i]);
    }
  }
};

constexpr const char* kShared = "clip_grads: two tensors share memory; each gradient may be scaled only once";

Tensor norm_op(at::TensorList grads, int64_t norm_type) {
  const c10::DeviceGuard guard(grads[0].device());
  const List l(grads, nullptr);
  check(g_norm(l.src.data(), l.numel.data(), l.type.data(), (int64_t)grads.size(), (int)norm_type, static_cast<float*>(write(l.norm)), write(l.ws),
               (size_t)l.ws.numel(), stream_of(grads[0].device())), "disco_grad_norm");
  return l.norm;
}

Tensor clip_op(at::TensorList grads, at::TensorList out, int64_t norm_type, double max_norm) {
  const c10::DeviceGuard guard(grads[0].device());
  const List l(grads, &out);
  const int status = g_clip(l.src.data(), l.dst.data(), l.numel.data(), l.type.data(), l.out_type.data(), (int64_t)grads.size(), (int)norm_type, max_norm,
                            static_cast<float*>(write(l.norm)), write(l.ws), (size_t)l.ws.numel(), stream_of(grads[0].device()));
  TORCH_CHECK_VALUE(status != DISCO_EINVAL, kShared);
  check(status, "disco_grad_clip");
  return l.norm;
}

Tensor norm_meta(at::TensorList grads, int64_t) { return at::empty({}, grads[0].options().dtype(at::kFloat)); }
Tensor clip_meta(at::TensorList grads, at::TensorList, int64_t, double) { return at::empty({}, grads[0].options().dtype(at::kFloat)); }

template <typename F> c10::TypedOperatorHandle<F> handle(const char* name, F*) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").template typed<F>();
}
template <typename F, typename... Args> auto below_autograd(const c10::TypedOperatorHandle<F>& op, const Args&... args) {
  const at::AutoDispatchBelowADInplaceOrView guard;
  return op.call(args...);
}

// ---- what Python calls ------------------------------------------------------------------------------------------------

variable_list call_forward(const Operands& o, int64_t plan, double factor, double eps, bool keep) {
  static const auto op = handle("disco_amd::residual_norm_forward", &forward_op);
  const auto maybe = [](const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); };
  return below_autograd(op, o.x, maybe(o.y), maybe(o.gate), maybe(o.scale), maybe(o.w1), maybe(o.b1), maybe(o.w2), maybe(o.b2), plan, factor, eps, keep);
}

class ResidualNorm : public torch::autograd::Function<ResidualNorm> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& y, const Maybe& gate, const Maybe& scale, const Maybe& w1,
                               const Maybe& b1, const Maybe& w2, const Maybe& b2, int64_t plan, double factor, double eps) {
    const Plan p(plan);
    const Operands o = operands(x, y, gate, scale, w1, b1, w2, b2);
    variable_list outputs = call_forward(o, plan, factor, eps, true);
    ctx->set_materialize_grads(false);
    // what no gradient reads is not kept, and may change: x without a next norm, y in out = x + factor * y
    const bool reads_y = p.post || p.pre || p.gate || o.scale.defined();
    ctx->save_for_backward({p.pre ? o.x : Tensor(), reads_y ? o.y : Tensor(), o.gate, o.scale, o.w1, o.b1, o.w2, o.b2, outputs.back()});
    outputs.pop_back();
    ctx->saved_data["plan"] = plan;
    ctx->saved_data["floats"] = std::vector<double>{factor, eps};
    return outputs;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op = handle("disco_amd::residual_norm_backward", &backward_op);
    variable_list result(11);
    const int64_t plan = ctx->saved_data["plan"].toInt();
    const auto floats = ctx->saved_data["floats"].toDoubleVector();
    const Plan p(plan);
    const Tensor dout = p.block ? grads[0] : Tensor(), dh = p.pre ? grads[p.block ? 1 : 0] : Tensor();
    if (!dout.defined() && !dh.defined()) return result;
    const variable_list s = ctx->get_saved_variables();
    const auto present = [&](size_t i) { return i == 0 || (i == 1 ? p.block : s[i].defined()); };
    // without a gradient of h the stream's gradient is that of out itself
    const bool through = !dh.defined();
    int64_t wanted = 0;
    for (size_t i = 0, edge = 0; i < 8; ++i) {      // edges are numbered over the operands that are there
      if (!present(i) || !ctx->needs_input_grad(edge++)) continue;
      if (through && (i == 0 || i >= 6)) continue;
      wanted |= (int64_t)1 << i;
    }
    if (wanted) {
      const auto maybe = [](const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); };
      const variable_list got = below_autograd(op, maybe(dout), maybe(dh), maybe(s[8]), maybe(s[0]), maybe(s[1]), maybe(s[2]), maybe(s[3]), maybe(s[4]),
                                               maybe(s[5]), maybe(s[6]), maybe(s[7]), plan, floats[0], floats[1], wanted);
      for (size_t i = 0, next = 0; i < 8; ++i)
        if (wanted >> i & 1) result[i] = got[next++];
    }
    if (through && ctx->needs_input_grad(0)) result[0] = dout;
    if (at::GradMode::is_enabled()) {      // the gradients have no formula of their own: whoever differentiates them is told
      for (Tensor& t : result)
        if (t.defined()) t = t.detach().requires_grad_();
      const auto refuse = std::make_shared<torch::autograd::DelayedError>("residual_norm has no second derivatives", 11);
      return (*refuse)(std::move(result));
    }
    return result;
  }
};

variable_list residual_norm(const Tensor& x, const Maybe& y, const Maybe& gate, const Maybe& scale, const Maybe& w1, const Maybe& b1, const Maybe& w2,
                            const Maybe& b2, int64_t plan, double factor, double eps, int64_t /*stream: unused*/) {
  const Operands o = operands(x, y, gate, scale, w1, b1, w2, b2);
  bool grad = false;
  for (const Tensor* t : {&o.x, &o.y, &o.gate, &o.scale, &o.w1, &o.b1, &o.w2, &o.b2}) {
    refuse_tangent(*t, "residual_norm");
    grad = grad || (t->defined() && t->requires_grad());
  }
  TORCH_CHECK(x.is_cuda(), "x is on ", x.device(), ": disco_amd runs on the GPU only, there is no CPU fallback");
  if (grad && at::GradMode::is_enabled()) return ResidualNorm::apply(x, y, gate, scale, w1, b1, w2, b2, plan, factor, eps);
  return call_forward(o, plan, factor, eps, false);
}

// The norm has no derivative here.  Of gradients that are differentiated again it is a node that says so, not a constant.
class GradientNorm : public torch::autograd::Function<GradientNorm> {
 public:
  static Tensor forward(AutogradContext*, at::TensorList grads, int64_t norm_type) {
    static const auto op = handle("disco_amd::grad_norm", &norm_op);
    return below_autograd(op, grads, norm_type);
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "grad_norm has no derivative: detach the gradients, or compute their norm with torch");
  }
};

bool known(const Tensor& t) {
  const auto s = t.scalar_type();
  return s == at::kFloat || s == at::kHalf || s == at::kBFloat16;
}

// A gradient without gaps, in any order of its dimensions, and its destination (itself or another tensor) in the same order:
// the kernels may walk the pair as it lies.
bool walkable(const Tensor& g, const Tensor& o) {
  if (g.is_neg() || o.is_neg()) return false;      // negated when read: an operator that writes cannot take them
  if (g.sym_numel() == 0) return true;
  return g.is_non_overlapping_and_dense() && (o.is_same(g) || o.sym_strides() == g.sym_strides() || (o.is_contiguous() && g.is_contiguous()));
}

// The norm over the gradients; with `out` also their clipping into it (out may be the list itself).  No value where the
// tensors are not what the kernels read -- on one GPU, of a known type, without gaps, each output of its gradient's shape,
// strides and type or float32: gradients.py then says what is wrong, or makes copies.
std::optional<Tensor> gradient_norm(const std::vector<Tensor>& grads, const std::optional<std::vector<Tensor>>& out, int64_t norm_type, double max_norm,
                                    int64_t /*stream: unused*/) {
  for (const Tensor& t : grads) refuse_tangent(t, "gradient_norm");
  if (out)
    for (const Tensor& t : *out) refuse_tangent(t, "gradient_norm");
  const size_t n = grads.size();
  if (n == 0 || !grads[0].is_cuda() || (out && out->size() != n)) return std::nullopt;
  const auto device = grads[0].device();
  for (size_t i = 0; i < n; ++i) {
    const Tensor& g = grads[i];
    if (g.layout() != at::kStrided || g.device() != device || !known(g) || (g.sym_numel() > 0 && !g.is_non_overlapping_and_dense())) return std::nullopt;
    if (!out) continue;
    const Tensor& o = (*out)[i];
    if (!o.is_same(g) && (o.layout() != at::kStrided || o.device() != device || (o.scalar_type() != g.scalar_type() && o.scalar_type() != at::kFloat) ||
                          o.sym_sizes() != g.sym_sizes()))
      return std::nullopt;
    if (!walkable(g, o)) return std::nullopt;
  }
  if (!out) {
    const bool grad = at::GradMode::is_enabled() && std::any_of(grads.begin(), grads.end(), [](const Tensor& g) { return g.requires_grad(); });
    return grad ? GradientNorm::apply(at::TensorList(grads), norm_type) : GradientNorm::forward(nullptr, grads, norm_type);
  }
  static const auto op = handle("disco_amd::grad_clip", &clip_op);
  const Tensor norm = below_autograd(op, at::TensorList(grads), at::TensorList(*out), norm_type, max_norm);
  for (const Tensor& o : *out)      // written behind autograd's back: whoever saved one of them must notice
    if (!o.is_inference()) torch::autograd::impl::bump_version(o);
  return norm;
}

// Places of a view in memory: the bytes at + sum of stride_k * x_k + u, 0 <= x_k <= most_k, with u inside an element; the
// strides fall and end with u's 1.
struct Term { int64_t stride, most; };
struct Places {
  int64_t at, last;      // last byte
  c10::SmallVector<Term, 6> terms;
  Places(int64_t at_, c10::IntArrayRef size, c10::IntArrayRef stride, int64_t item) : at(at_), last(at_ + item - 1) {
    for (size_t d = 0; d < size.size(); ++d)
      if (size[d] > 1 && stride[d] > 0) {
        terms.push_back({stride[d] * item, size[d] - 1});
        last += terms.back().stride * terms.back().most;
      }
    std::sort(terms.begin(), terms.end(), [](const Term& p, const Term& q) { return p.stride > q.stride; });
    terms.push_back({1, item - 1});
  }
};
Places places(const Tensor& t) { return {(int64_t)reinterpret_cast<uintptr_t>(t.const_data_ptr()), t.sizes(), t.strides(), (int64_t)t.element_size()}; }

// A sum of the terms from k on that is `target`; strides fall and end with 1.  After `work` steps the answer is yes: views that
// nobody can tell apart are not told apart here.
bool reaches(c10::ArrayRef<Term> terms, c10::ArrayRef<int64_t> rest, size_t k, int64_t target, int64_t& work) {
  if (target < 0 || target > rest[k]) return false;
  if (k + 1 == terms.size()) return true;
  const int64_t s = terms[k].stride;
  for (int64_t x = std::min(terms[k].most, target / s); x >= 0 && target - x * s <= rest[k + 1]; --x)
    if (--work < 0 || reaches(terms, rest, k + 1, target - x * s, work)) return true;
  return false;
}

// Whether two views have a byte in common.  With b's indices counted from their ends, a place of each is one sum of terms:
// sum_a + sum_b' = (b's last byte) - (a's first).
bool meet(const Places& a, const Places& b) {
  if (a.last < b.at || b.last < a.at) return false;
  c10::SmallVector<Term, 12> terms;
  for (size_t i = 0, j = 0; i < a.terms.size() || j < b.terms.size();) {
    const bool first = j == b.terms.size() || (i < a.terms.size() && a.terms[i].stride >= b.terms[j].stride);
    const Term& t = first ? a.terms[i++] : b.terms[j++];
    if (!terms.empty() && terms.back().stride == t.stride) terms.back().most += t.most;
    else terms.push_back(t);
  }
  c10::SmallVector<int64_t, 12> rest(terms.size());
  int64_t sum = 0;
  for (size_t k = terms.size(); k-- > 0;) rest[k] = sum += terms[k].stride * terms[k].most;
  int64_t work = 100000;
  return reaches(terms, rest, 0, b.last - a.at, work);
}

// Two elements of one view at the same place: their indices differ first in some dimension d, and there it is enough to set
// index 0 against the others.
bool meets_itself(const Tensor& t) {
  const int64_t item = (int64_t)t.element_size(), at = (int64_t)reinterpret_cast<uintptr_t>(t.const_data_ptr());
  for (int64_t d = 0; d < t.dim(); ++d) {
    if (t.size(d) == 1) continue;
    c10::SmallVector<int64_t, 6> size(t.sizes().begin() + d, t.sizes().end());
    const auto stride = t.strides().slice(d);
    size[0] = 1;
    const Places first(at, size, stride, item);
    size[0] = t.size(d) - 1;
    if (meet(first, Places(at + stride[0] * item, size, stride, item))) return true;
  }
  return false;
}

// Whether an element would be written with two values: by two gradients, or by one into a view that meets itself.  Gradients
// that are scaled where they lie may meet, since each writes what the other writes.
bool written_twice(const std::vector<Tensor>& grads, const std::vector<Tensor>& out) {
  std::vector<std::pair<Places, bool>> all;
  for (size_t i = 0; i < out.size(); ++i) {
    if (out[i].numel() == 0 || out[i].key_set().has(c10::DispatchKey::Python)) continue;      // a fake tensor has no memory
    const bool in_place = out[i].is_same(grads[i]);
    if (!in_place && !out[i].is_non_overlapping_and_dense() && meets_itself(out[i])) return true;
    all.emplace_back(places(out[i]), in_place);
  }
  std::sort(all.begin(), all.end(), [](const auto& a, const auto& b) { return a.first.at < b.first.at; });
  for (size_t i = 0; i < all.size(); ++i)
    for (size_t j = i + 1; j < all.size() && all[j].first.at <= all[i].first.last; ++j)
      if (!(all[i].second && all[j].second) && meet(all[i].first, all[j].first)) return true;
  return false;
}

// Which pairs go through contiguous copies, because the kernels cannot walk them as they lie.
std::vector<int64_t> copied_pairs(const std::vector<Tensor>& grads, const std::vector<Tensor>& out) {
  TORCH_CHECK(grads.size() == out.size(), "copied_pairs: a destination for each gradient");
  std::vector<int64_t> r;
  bool in_place = true;
  for (size_t i = 0; i < out.size(); ++i) {
    in_place = in_place && out[i].is_same(grads[i]);
    if (!walkable(grads[i], out[i])) r.push_back((int64_t)i);
  }
  TORCH_CHECK_VALUE(in_place || !written_twice(grads, out), kShared);
  return r;
}

}  // namespace

// `stream` is not read: it stands for callers that still pass one.
TORCH_LIBRARY(disco_amd, m) {
  m.def("bind(int forward, int backward, int workspace, int status, int norm, int clip, int norm_workspace) -> ()", &bind);
  m.def("gradient_norm(Tensor[] grads, Tensor[]? out, int norm_type, float max_norm, int stream=0) -> Tensor?", &gradient_norm);
  m.def(
      "residual_norm(Tensor x, Tensor? y, Tensor? gate, Tensor? scale, Tensor? post_weight, Tensor? post_bias, Tensor? pre_weight, "
      "Tensor? pre_bias, int plan, float factor, float eps, int stream=0) -> Tensor[]",
      &residual_norm);
  m.def(
      "residual_norm_forward(Tensor x, Tensor? y, Tensor? gate, Tensor? scale, Tensor? post_weight, Tensor? post_bias, Tensor? pre_weight, "
      "Tensor? pre_bias, int plan, float factor, float eps, bool keep) -> Tensor[]");
  m.def(
      "residual_norm_backward(Tensor? dout, Tensor? dh, Tensor? stats, Tensor? x, Tensor? y, Tensor? gate, Tensor? scale, Tensor? post_weight, "
      "Tensor? post_bias, Tensor? pre_weight, Tensor? pre_bias, int plan, float factor, float eps, int wanted) -> Tensor[]");
  m.def("copied_pairs(Tensor[] grads, Tensor[] out) -> int[]", &copied_pairs);
  m.def("grad_norm(Tensor[] grads, int norm_type) -> Tensor");
  m.def("grad_clip(Tensor[] grads, Tensor(a!)[] out, int norm_type, float max_norm) -> Tensor");
}

TORCH_LIBRARY_IMPL(disco_amd, CUDA, m) {
  m.impl("residual_norm_forward", &forward_op);
  m.impl("residual_norm_backward", &backward_op);
  m.impl("grad_norm", &norm_op);
  m.impl("grad_clip", &clip_op);
}

// Called by themselves (a recorded graph that is differentiated again) they have no derivative, and say so.
TORCH_LIBRARY_IMPL(disco_amd, Autograd, m) {
  m.impl("residual_norm_forward", torch::autograd::autogradNotImplementedFallback());
  m.impl("residual_norm_backward", torch::autograd::autogradNotImplementedFallback());
  m.impl("grad_norm", torch::autograd::autogradNotImplementedFallback());
}

TORCH_LIBRARY_IMPL(disco_amd, Meta, m) {
  m.impl("residual_norm_forward", &forward_meta);
  m.impl("residual_norm_backward", &backward_meta);
  m.impl("grad_norm", &norm_meta);
  m.impl("grad_clip", &clip_meta);
}

// csn_torch.cpp -- PyTorch binding of the gated recurrent and linear-attention blocks' entry points (python module
// csn_b200._gated).
//
// The other entry points are bound with ctypes and torch.autograd.Function.  These are called once a token or once a
// layer on small tensors, where the host's time for a call is the call's time, so their argument checks, allocations
// and autograd nodes are C++: a training call of the scan costs the host 60 us less than from Python.  The kernels are
// reached through the C ABI alone.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <initializer_list>
#include <optional>
#include <string>
#include <tuple>

#include "../../include/csn_b200.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = optional<Tensor>;

// a status of the library other than CSN_OK; csn_b200._lib.CsnError in Python
struct Failure : std::runtime_error {
  std::string entry, text;
  int code;
  Failure(const char* e, int c) : std::runtime_error(std::string(e) + " failed: " + csn_last_error()), entry(e), text(csn_last_error()), code(c) {}
};
void check(const char* entry, int code) {
  if (code != CSN_OK) throw Failure(entry, code);
}

bool there(const Maybe& t) { return t.has_value() && t->defined(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* ptr(const Maybe& t) { return there(t) ? t->data_ptr() : nullptr; }

int code_of(at::ScalarType t) {
  return t == at::kFloat ? CSN_F32 : t == at::kBFloat16 ? CSN_BF16 : t == at::kHalf ? CSN_F16 : -1;
}

void on_one_device(const char* name, std::initializer_list<const Tensor*> ts) {
  const Tensor& first = **ts.begin();
  for (const Tensor* t : ts) {
    if (!t) continue;
    TORCH_CHECK(t->is_cuda(), "csn_b200 ops need CUDA tensors: the library has no CPU path");
    TORCH_CHECK_VALUE(t->device() == first.device(), name, ": tensors are on different devices");
  }
}
void of_one_type(const char* name, bool floats, std::initializer_list<const Tensor*> ts) {
  const Tensor& first = **ts.begin();
  const int c = code_of(first.scalar_type());
  TORCH_CHECK_VALUE(c >= (floats ? 0 : 1), name, ": tensors of one type among ", floats ? "float32, " : "",
                    "bfloat16, float16 expected, got ", first.scalar_type());
  for (const Tensor* t : ts)
    if (t) TORCH_CHECK_VALUE(t->scalar_type() == first.scalar_type(), name, ": tensors of one type expected, got ",
                             first.scalar_type(), " and ", t->scalar_type());
}
const Tensor* at_of(const Maybe& t) { return there(t) ? &*t : nullptr; }

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t && t->requires_grad()) return true;
  return false;
}

// The kernels read and write through pointers, past which a forward-mode tangent would be lost without a word.
void no_tangent(const char* name, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t || !t->defined() || !t->_fw_grad(0).defined(), name, ": forward-mode derivatives are not available");
}

// t with a contiguous last axis (itself where it has one)
Tensor rows(const Tensor& t) { return !t.defined() || t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }
Tensor rows(const Maybe& t) { return there(t) ? rows(*t) : Tensor(); }
// t contiguous and 16-byte aligned (itself where it is)
Tensor packed(const Tensor& t) {
  if (!t.defined()) return t;
  Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
}
Tensor packed(const Maybe& t) { return there(t) ? packed(*t) : Tensor(); }

Tensor room(const Tensor& like, at::IntArrayRef sizes) { return at::empty(sizes, like.options()); }
Tensor floats(const Tensor& like, at::IntArrayRef sizes) { return at::empty(sizes, like.options().dtype(at::kFloat)); }
Tensor bytes(const Tensor& like, size_t n) {
  return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor();
}

void* stream(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// Gradients are first-order: where a second backward pass could follow, what comes out raises in it.
variable_list first_order(const char* name, variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string(name) + " is differentiable once: a second backward pass through it is not available", grads.size());
  return (*error)(std::move(grads));
}

// ------------------------------------------------------------- gated recurrence
struct Sizes {
  int64_t S, T, C;
  Sizes(const Tensor& f, bool cut, const Maybe& cu)
      : S(cut ? cu->size(0) - 1 : f.size(0)), T(cut ? f.size(0) : f.size(1)), C(f.size(-1)) {}
};

// strides of every axis but the last, 0 where an axis has one entry; a matrix has (0, row)
void put_strides(int64_t* to, const Tensor& t) {
  to[0] = to[1] = 0;
  if (!t.defined()) return;
  const int64_t n = t.dim();
  for (int64_t i = 0; i < n - 1; ++i) to[2 - (n - 1) + i] = t.size(i) > 1 ? t.stride(i) : 0;
}

Sizes scan_sizes(const Tensor& f, const Tensor& x, const Maybe& gate, const Maybe& cu) {
  of_one_type("gated_scan", true, {&f, &x, at_of(gate)});
  const bool shapes = f.dim() == (there(cu) ? 2 : 3) && x.sizes() == f.sizes() && (!there(gate) || gate->sizes() == f.sizes());
  TORCH_CHECK_VALUE(shapes, "gated_scan: f, x and gate [B, T, C], or [L, C] with cu_seqlens, of one shape expected, got ",
                    f.sizes(), " and ", x.sizes());
  TORCH_CHECK_VALUE(!there(cu) || (cu->scalar_type() == at::kInt && cu->dim() == 1 && cu->size(0) >= 2 && cu->is_contiguous()),
                    "gated_scan: cu_seqlens is a contiguous int32 vector of at least 2 row numbers");
  return Sizes(f, there(cu), cu);
}

void check_state(const char* what, const Maybe& h, const Sizes& n) {
  TORCH_CHECK_VALUE(!there(h) || (h->dim() == 2 && h->size(0) == n.S && h->size(1) == n.C && at::isFloatingType(h->scalar_type())),
                    "gated_scan: ", what, " [", n.S, ", ", n.C, "] of a floating type expected");
}

void check_scan(const Tensor& f, const Tensor& x, const Maybe& h0, const Maybe& gate, const Maybe& cu) {
  no_tangent("gated_scan", {&f, &x, at_of(h0), at_of(gate)});
  check_state("h0", h0, scan_sizes(f, x, gate, cu));
  on_one_device("gated_scan", {&f, &x, at_of(h0), at_of(gate), at_of(cu)});
}

std::tuple<Tensor, Tensor, Tensor> scan_forward(const Tensor& f_, const Tensor& x_, const Maybe& h0_, const Maybe& gate_,
                                                const Maybe& cu, bool keep) {
  const c10::cuda::CUDAGuard guard(f_.device());
  const Tensor f = rows(f_), x = rows(x_), gate = rows(gate_), h0 = packed(h0_);
  const bool cut = there(cu);
  const Sizes n(f, cut, cu);
  const int code = code_of(f.scalar_type());
  Tensor y = room(f, f.sizes()), last = floats(f, {n.S, n.C});
  Tensor marks = keep ? floats(f, {csn_gated_scan_marks(n.S, n.T, n.C, cut)}) : Tensor();
  const size_t nb = csn_gated_scan_workspace_bytes(n.S, n.T, n.C, cut, code, 0);
  const Tensor ws = bytes(f, nb);
  int64_t st[6];
  put_strides(st, f), put_strides(st + 2, x), put_strides(st + 4, gate);
  check("csn_gated_scan_fwd",
        csn_gated_scan_fwd(ptr(f), ptr(x), ptr(gate), st, static_cast<const float*>(ptr(h0)), static_cast<const int32_t*>(ptr(cu)),
                           ptr(y), static_cast<float*>(ptr(last)), static_cast<float*>(ptr(marks)), n.S, n.T, n.C, code, ptr(ws),
                           nb, stream(f)));
  return {y, last, marks};
}

// (df, dx, dh0 where it is wanted, dgate where there is a gate)
std::tuple<Tensor, Tensor, Tensor, Tensor> scan_backward(const Tensor& f_, const Tensor& x_, const Maybe& gate_, const Maybe& cu,
                                                         const Tensor& marks, const Maybe& dy_, const Maybe& dlast_,
                                                         bool want_h0) {
  const c10::cuda::CUDAGuard guard(f_.device());
  const Tensor f = rows(f_), x = rows(x_), gate = rows(gate_), dlast = packed(dlast_);
  // only the last states are used: a zero for every place
  const Tensor dy = there(dy_) ? rows(*dy_) : rows(at::zeros(std::vector<int64_t>(f.dim(), 1), f.options()).expand(f.sizes()));
  const bool cut = there(cu);
  const Sizes n(f, cut, cu);
  const int code = code_of(f.scalar_type());
  Tensor df = room(f, f.sizes()), dx = room(f, f.sizes());
  Tensor dgate = gate.defined() ? room(f, f.sizes()) : Tensor(), dh0 = want_h0 ? floats(f, {n.S, n.C}) : Tensor();
  const size_t nb = csn_gated_scan_workspace_bytes(n.S, n.T, n.C, cut, code, 1);
  const Tensor ws = bytes(f, nb);
  int64_t st[8];
  put_strides(st, f), put_strides(st + 2, x), put_strides(st + 4, gate), put_strides(st + 6, dy);
  check("csn_gated_scan_bwd",
        csn_gated_scan_bwd(ptr(f), ptr(x), ptr(gate), ptr(dy), st, static_cast<const int32_t*>(ptr(cu)),
                           static_cast<const float*>(ptr(marks)), static_cast<const float*>(ptr(dlast)), ptr(df), ptr(dx),
                           ptr(dgate), static_cast<float*>(ptr(dh0)), n.S, n.T, n.C, code, ptr(ws), nb, stream(f)));
  return {df, dx, dh0, dgate};
}

// The backward pass on tensors of any origin, which are looked at first.
std::tuple<Tensor, Tensor, Tensor, Tensor> gated_scan_backward(const Tensor& f, const Tensor& x, const Maybe& gate, const Maybe& cu,
                                                               const Tensor& marks, const Tensor& dy, const Tensor& dlast) {
  no_tangent("gated_scan", {&f, &x, at_of(gate), &marks, &dy, &dlast});
  const Sizes n = scan_sizes(f, x, gate, cu);
  of_one_type("gated_scan", true, {&f, &dy});
  TORCH_CHECK_VALUE(dy.sizes() == f.sizes(), "gated_scan: dy of f's shape expected, got ", dy.sizes(), " and ", f.sizes());
  check_state("dh_last", dlast, n);
  const int64_t room = csn_gated_scan_marks(n.S, n.T, n.C, there(cu));
  TORCH_CHECK_VALUE(marks.scalar_type() == at::kFloat && marks.dim() == 1 && marks.size(0) == room && marks.is_contiguous() &&
                        reinterpret_cast<uintptr_t>(ptr(marks)) % 16 == 0,
                    "gated_scan: marks are the ", room, " numbers that the forward pass kept");
  on_one_device("gated_scan", {&f, &x, at_of(gate), at_of(cu), &marks, &dy, &dlast});
  return scan_backward(f, x, gate, cu, marks, dy, dlast.to(at::kFloat), true);
}

struct GatedScan : torch::autograd::Function<GatedScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& f, const Tensor& x, const Maybe& h0, const Maybe& gate,
                               const Maybe& cu) {
    ctx->set_materialize_grads(false);
    auto [y, last, marks] = scan_forward(f, x, h0, gate, cu, true);
    ctx->save_for_backward({f, x, there(gate) ? *gate : Tensor(), there(cu) ? *cu : Tensor(), marks});
    ctx->saved_data["h0"] = there(h0) && h0->requires_grad();
    return {y, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined() && !g[1].defined()) return variable_list(5);
    no_tangent("gated_scan", {&g[0], &g[1]});
    const auto s = ctx->get_saved_variables();
    auto [df, dx, dh0, dgate] = [&] {
      at::AutoGradMode off(false);
      return scan_backward(s[0], s[1], s[2], s[3], s[4], g[0], g[1], ctx->saved_data["h0"].toBool());
    }();
    return first_order("gated_scan", {df, dx, dh0, dgate, Tensor()});
  }
};

std::tuple<Tensor, Tensor> gated_scan(const Tensor& f, const Tensor& x, const Maybe& h0_, const Maybe& gate, const Maybe& cu) {
  check_scan(f, x, h0_, gate, cu);
  const Maybe h0 = there(h0_) && h0_->scalar_type() != at::kFloat ? Maybe(h0_->to(at::kFloat)) : h0_;
  if (!wants_grad({&f, &x, at_of(h0), at_of(gate)})) {
    auto [y, last, marks] = scan_forward(f, x, h0, gate, cu, false);
    return {y, last};
  }
  variable_list out = GatedScan::apply(f, x, h0, gate, cu);
  return {out[0], out[1]};
}

Tensor gated_step(const Tensor& f_, const Tensor& x_, const Tensor& h, const Maybe& gate_) {
  no_tangent("gated_step", {&f_, &x_, &h, at_of(gate_)});
  on_one_device("gated_step", {&f_, &x_, &h, at_of(gate_)});
  of_one_type("gated_step", true, {&f_, &x_, at_of(gate_)});
  TORCH_CHECK_VALUE(f_.dim() == 2 && x_.sizes() == f_.sizes() && h.sizes() == f_.sizes() && (!there(gate_) || gate_->sizes() == f_.sizes()),
                    "gated_step: f, x, h and gate [B, C] of one shape expected");
  TORCH_CHECK_VALUE(h.scalar_type() == at::kFloat && h.is_contiguous() && reinterpret_cast<uintptr_t>(h.data_ptr()) % 16 == 0,
                    "gated_step: h is a contiguous float32 state, 16-byte aligned");
  TORCH_CHECK_VALUE(!wants_grad({&f_, &x_, &h, at_of(gate_)}),
                    "gated_step: not differentiable; call it under torch.no_grad() or use gated_scan");
  const c10::cuda::CUDAGuard guard(f_.device());
  const Tensor f = rows(f_), x = rows(x_), gate = rows(gate_);
  Tensor y = room(f, f.sizes());
  h.unsafeGetTensorImpl()->bump_version();  // first: it raises where h may not be changed
  const int64_t st[3] = {f.stride(0), x.stride(0), gate.defined() ? gate.stride(0) : 0};
  check("csn_gated_step", csn_gated_step(ptr(f), ptr(x), ptr(gate), st, static_cast<float*>(ptr(h)), ptr(y), f.size(0), f.size(1),
                                         code_of(f.scalar_type()), stream(f)));
  return y;
}

// ---------------------------------------------------- gated feed-forward product
// From this width on the products are kept in float32 (8 bytes an element of the result, what keeping both and the gate
// in their own type would take) instead of being formed again in the backward pass.  Forward and backward, R = 8192,
// F = 2 C, bf16, formed again / kept: C = 512 99.5 / 103 us, C = 1024 250 / 244, C = 2048 887 / 784, C = 4096 3240 / 2737;
// F = 3136, C = 1536 551 / 502.  Below, what little it brings is not worth the memory.
constexpr int64_t KEEP = 1536;

// (y, both products where they are to be kept)
std::tuple<Tensor, Tensor> ffn_forward(const Tensor& x_, const Tensor& wg_, const Tensor& wu_, bool keep) {
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = rows(x_), wg = rows(wg_), wu = rows(wu_);
  const int64_t R = x.size(0), C = x.size(1), F = wg.size(0), ldx = x.stride(0), ldg = wg.stride(0), ldu = wu.stride(0);
  Tensor y = room(x, {R, F}), pre = keep ? floats(x, {2, R, F}) : Tensor();
  const size_t nb = csn_silu_gated_linear_workspace_bytes(
      R, C, F, csn_silu_gated_linear_copies(ptr(x), ldx, ptr(wg), ldg, ptr(wu), ldu, R, C, F), 0);
  const Tensor ws = bytes(x, nb);
  check("csn_silu_gated_linear_fwd", csn_silu_gated_linear_fwd(ptr(x), ldx, ptr(wg), ldg, ptr(wu), ldu, ptr(y),
                                                               static_cast<float*>(ptr(pre)), R, C, F, code_of(x.scalar_type()),
                                                               ptr(ws), nb, stream(x)));
  return {y, pre};
}

std::tuple<Tensor, Tensor, Tensor> ffn_backward(const Tensor& x_, const Tensor& wg_, const Tensor& wu_, const Tensor& dy_,
                                                const Maybe& pre, bool need_x, bool need_g, bool need_u) {
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = rows(x_), wg = rows(wg_), wu = rows(wu_), dy = rows(dy_);
  const int64_t R = x.size(0), C = x.size(1), F = wg.size(0), ldx = x.stride(0), ldg = wg.stride(0), ldu = wu.stride(0);
  Tensor dx = need_x ? room(x, {R, C}) : Tensor(), dg = need_g ? room(x, {F, C}) : Tensor(), du = need_u ? room(x, {F, C}) : Tensor();
  const size_t nb = csn_silu_gated_linear_workspace_bytes(
      R, C, F, csn_silu_gated_linear_copies(ptr(x), ldx, ptr(wg), ldg, ptr(wu), ldu, R, C, F), 1);
  const Tensor ws = bytes(x, nb);
  check("csn_silu_gated_linear_bwd",
        csn_silu_gated_linear_bwd(ptr(x), ldx, ptr(wg), ldg, ptr(wu), ldu, ptr(dy), dy.stride(0),
                                  static_cast<const float*>(ptr(pre)), ptr(dx), ptr(dg), ptr(du), R, C, F,
                                  code_of(x.scalar_type()), ptr(ws), nb, stream(x)));
  return {dx, dg, du};
}

struct SiluGatedLinear : torch::autograd::Function<SiluGatedLinear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu) {
    auto [y, pre] = ffn_forward(x, wg, wu, x.size(1) >= KEEP && x.size(0) > 64);
    ctx->save_for_backward({x, wg, wu, pre});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    no_tangent("silu_gated_linear", {&g[0]});
    auto [dx, dg, du] = [&] {
      at::AutoGradMode off(false);
      return ffn_backward(s[0], s[1], s[2], g[0], s[3], ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2));
    }();
    return first_order("silu_gated_linear", {dx, dg, du});
  }
};

void check_ffn(const Tensor& x, const Tensor& wg, const Tensor& wu) {
  of_one_type("silu_gated_linear", false, {&x, &wg, &wu});
  TORCH_CHECK_VALUE(x.dim() >= 1 && wg.dim() == 2 && wu.sizes() == wg.sizes() && x.size(-1) == wg.size(1),
                    "silu_gated_linear: x [..., C] and w_gate, w_up [F, C] expected, got ", x.sizes(), ", ", wg.sizes(), ", ", wu.sizes());
}

// t [..., n] as a matrix
Tensor flat(const Tensor& t) {
  if (t.dim() == 2) return t;
  int64_t n = 1;
  for (int64_t i = 0; i < t.dim() - 1; ++i) n *= t.size(i);
  return t.reshape({n, t.size(-1)});
}

Tensor silu_gated_linear(const Tensor& x, const Tensor& wg, const Tensor& wu) {
  no_tangent("silu_gated_linear", {&x, &wg, &wu});
  check_ffn(x, wg, wu);
  on_one_device("silu_gated_linear", {&x, &wg, &wu});
  const Tensor r = flat(x);
  Tensor y = wants_grad({&x, &wg, &wu}) ? SiluGatedLinear::apply(r, wg, wu) : std::get<0>(ffn_forward(r, wg, wu, false));
  if (x.dim() == 2) return y;
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = wg.size(0);
  return y.view(shape);
}

// The backward pass on tensors of any origin, which are looked at first; both products are formed again.
std::tuple<Tensor, Tensor, Tensor> silu_gated_linear_backward(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& dy) {
  no_tangent("silu_gated_linear", {&x, &wg, &wu, &dy});
  check_ffn(x, wg, wu);
  of_one_type("silu_gated_linear", false, {&x, &dy});
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  TORCH_CHECK_VALUE(dy.dim() == x.dim() && dy.sizes().slice(0, lead.size()) == lead && dy.size(-1) == wg.size(0),
                    "silu_gated_linear: dy of the result's shape expected, got ", dy.sizes(), " for ", x.sizes(), " and ", wg.sizes());
  on_one_device("silu_gated_linear", {&x, &wg, &wu, &dy});
  auto [dx, dg, du] = ffn_backward(flat(x), wg, wu, flat(dy), std::nullopt, true, true, true);
  return {dx.view(x.sizes()), dg, du};
}

// -------------------------------------------------------------- linear attention
struct Heads {
  int64_t S, T, H, Hk, Dk, Dv;
  Heads(const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& cu)
      : S(there(cu) ? cu->size(0) - 1 : q.size(0)), T(there(cu) ? q.size(0) : q.size(1)), H(q.size(-2)), Hk(k.size(-2)), Dk(q.size(-1)),
        Dv(v.size(-1)) {}
};

// strides of sequence, row and head, 0 where an axis has one entry
void put_head_strides(int64_t* to, const Tensor& t) {
  to[0] = 0;
  const int64_t n = t.dim() - 1;
  for (int64_t i = 0; i < n; ++i) to[3 - n + i] = t.size(i) > 1 ? t.stride(i) : 0;
}

// `lead`: axes before the heads
void check_heads(const char* name, const char* form, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, int64_t lead) {
  of_one_type(name, true, {&q, &k, &v});
  bool fits = q.dim() == lead + 2 && k.dim() == q.dim() && v.dim() == q.dim();
  for (int64_t i = 0; fits && i < lead; ++i) fits = k.size(i) == q.size(i) && v.size(i) == q.size(i);
  TORCH_CHECK_VALUE(fits && k.size(-1) == q.size(-1) && v.size(-2) == k.size(-2), name, ": q ", form, " k and v with the same rows, k of q's last size, v of "
                    "k's heads expected, got ", q.sizes(), ", ", k.sizes(), " and ", v.sizes());
  TORCH_CHECK_VALUE(q.size(-2) >= 1 && k.size(-2) >= 1 && q.size(-2) % k.size(-2) == 0, name, ": the heads of k and v (", k.size(-2),
                    ") have to divide those of q (", q.size(-2), ")");
  TORCH_CHECK_VALUE(q.size(-1) >= 1 && q.size(-1) <= 128 && v.size(-1) >= 1 && v.size(-1) <= 128, name, ": head sizes of 1 to 128 expected, got ",
                    q.size(-1), " and ", v.size(-1));
  TORCH_CHECK_VALUE(log_decay.scalar_type() == at::kFloat && log_decay.dim() == 1 && log_decay.size(0) == q.size(-2) && log_decay.is_contiguous(),
                    name, ": log_decay is a contiguous float32 vector with a number for each of the ", q.size(-2), " heads");
  TORCH_CHECK_VALUE(!wants_grad({&log_decay}), name, ": log_decay has no gradient here: pass it detached");
}

Heads attention_sizes(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Maybe& cu) {
  TORCH_CHECK_VALUE(!there(cu) || (cu->scalar_type() == at::kInt && cu->dim() == 1 && cu->size(0) >= 2 && cu->is_contiguous()),
                    "linear_attention: cu_seqlens is a contiguous int32 vector of at least 2 row numbers");
  check_heads("linear_attention", "[B, T, H, D], or [L, H, D] with cu_seqlens,", q, k, v, log_decay, there(cu) ? 1 : 2);
  return Heads(q, k, v, cu);
}

void check_states(const char* what, const Maybe& s, const Heads& n) {
  TORCH_CHECK_VALUE(!there(s) || (s->dim() == 4 && s->size(0) == n.S && s->size(1) == n.H && s->size(2) == n.Dk && s->size(3) == n.Dv &&
                                  at::isFloatingType(s->scalar_type())),
                    "linear_attention: ", what, " [", n.S, ", ", n.H, ", ", n.Dk, ", ", n.Dv, "] of a floating type expected");
}

void check_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Maybe& s0, const Maybe& cu) {
  no_tangent("linear_attention", {&q, &k, &v, &log_decay, at_of(s0)});
  check_states("s0", s0, attention_sizes(q, k, v, log_decay, cu));
  on_one_device("linear_attention", {&q, &k, &v, &log_decay, at_of(s0), at_of(cu)});
}

double scale_of(const optional<double>& scale, int64_t Dk) { return scale ? *scale : 1.0 / std::sqrt((double)Dk); }

std::tuple<Tensor, Tensor> attention_forward(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& log_decay, const Maybe& s0_,
                                             const Maybe& cu, double scale) {
  const c10::cuda::CUDAGuard guard(q_.device());
  const Tensor q = rows(q_), k = rows(k_), v = rows(v_), s0 = packed(s0_);
  const Heads n(q, k, v, cu);
  const int code = code_of(q.scalar_type());
  std::vector<int64_t> shape(q.sizes().begin(), q.sizes().end());
  shape.back() = n.Dv;
  Tensor o = room(q, shape), last = floats(q, {n.S, n.H, n.Dk, n.Dv});
  int64_t st[9];
  put_head_strides(st, q), put_head_strides(st + 3, k), put_head_strides(st + 6, v);
  const int copies = csn_linear_attention_copies(ptr(q), ptr(k), ptr(v), nullptr, st, n.S, n.T, n.H, n.Hk, n.Dk, n.Dv, there(cu), code);
  const size_t nb = csn_linear_attention_workspace_bytes(n.S, n.T, n.H, n.Hk, n.Dk, n.Dv, there(cu), code, copies, 0);
  const Tensor ws = bytes(q, nb);
  check("csn_linear_attention_fwd",
        csn_linear_attention_fwd(ptr(q), ptr(k), ptr(v), st, static_cast<const float*>(ptr(log_decay)), static_cast<const float*>(ptr(s0)),
                                 static_cast<const int32_t*>(ptr(cu)), ptr(o), static_cast<float*>(ptr(last)), n.S, n.T, n.H, n.Hk, n.Dk,
                                 n.Dv, (float)scale, code, ptr(ws), nb, stream(q)));
  return {o, last};
}

// (dq, dk, dv, ds0), those that are wanted
std::tuple<Tensor, Tensor, Tensor, Tensor> attention_backward(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& log_decay,
                                                              const Maybe& s0_, const Maybe& cu, const Maybe& do_, const Maybe& dlast_,
                                                              double scale, bool want_q, bool want_k, bool want_v, bool want_s0) {
  const c10::cuda::CUDAGuard guard(q_.device());
  const Tensor q = rows(q_), k = rows(k_), v = rows(v_), s0 = packed(s0_), dlast = packed(dlast_);
  const Heads n(q, k, v, cu);
  std::vector<int64_t> shape(q.sizes().begin(), q.sizes().end());
  shape.back() = n.Dv;
  // only the last states are used: a zero for every place
  const Tensor d = there(do_) ? rows(*do_) : at::zeros(std::vector<int64_t>(q.dim() - 1, 1), q.options()).unsqueeze(-1).expand(shape).contiguous();
  const int code = code_of(q.scalar_type());
  Tensor dq = want_q ? room(q, q.sizes()) : Tensor(), dk = want_k ? room(k, k.sizes()) : Tensor();
  Tensor dv = want_v || want_s0 ? room(v, v.sizes()) : Tensor(), ds0 = want_s0 ? floats(q, {n.S, n.H, n.Dk, n.Dv}) : Tensor();
  int64_t st[12];
  put_head_strides(st, q), put_head_strides(st + 3, k), put_head_strides(st + 6, v), put_head_strides(st + 9, d);
  const int copies = csn_linear_attention_copies(ptr(q), ptr(k), ptr(v), ptr(d), st, n.S, n.T, n.H, n.Hk, n.Dk, n.Dv, there(cu), code);
  const size_t nb = csn_linear_attention_workspace_bytes(n.S, n.T, n.H, n.Hk, n.Dk, n.Dv, there(cu), code, copies, 1);
  const Tensor ws = bytes(q, nb);
  check("csn_linear_attention_bwd",
        csn_linear_attention_bwd(ptr(q), ptr(k), ptr(v), ptr(d), st, static_cast<const float*>(ptr(log_decay)),
                                 static_cast<const float*>(ptr(s0)), static_cast<const int32_t*>(ptr(cu)),
                                 static_cast<const float*>(ptr(dlast)), ptr(dq), ptr(dk), ptr(dv), static_cast<float*>(ptr(ds0)), n.S, n.T,
                                 n.H, n.Hk, n.Dk, n.Dv, (float)scale, code, ptr(ws), nb, stream(q)));
  return {dq, dk, want_v ? dv : Tensor(), ds0};
}

// The backward pass on tensors of any origin, which are looked at first.
std::tuple<Tensor, Tensor, Tensor, Tensor> linear_attention_backward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay,
                                                                     const Maybe& s0, const Maybe& cu, const Tensor& d, const Tensor& dlast,
                                                                     optional<double> scale) {
  no_tangent("linear_attention", {&q, &k, &v, &log_decay, at_of(s0), &d, &dlast});
  const Heads n = attention_sizes(q, k, v, log_decay, cu);
  check_states("s0", s0, n);
  check_states("ds_last", dlast, n);
  of_one_type("linear_attention", true, {&q, &d});
  std::vector<int64_t> shape(q.sizes().begin(), q.sizes().end());
  shape.back() = n.Dv;
  TORCH_CHECK_VALUE(d.sizes() == at::IntArrayRef(shape), "linear_attention: do of the result's shape expected, got ", d.sizes());
  on_one_device("linear_attention", {&q, &k, &v, &log_decay, at_of(s0), at_of(cu), &d, &dlast});
  return attention_backward(q, k, v, log_decay, there(s0) ? Maybe(s0->to(at::kFloat)) : s0, cu, d, dlast.to(at::kFloat), scale_of(scale, n.Dk),
                            true, true, true, true);
}

struct LinearAttention : torch::autograd::Function<LinearAttention> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay,
                               const Maybe& s0, const Maybe& cu, double scale) {
    ctx->set_materialize_grads(false);
    auto [o, last] = attention_forward(q, k, v, log_decay, s0, cu, scale);
    ctx->save_for_backward({q, k, v, log_decay, there(s0) ? *s0 : Tensor(), there(cu) ? *cu : Tensor()});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["s0"] = there(s0) && s0->requires_grad();
    return {o, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined() && !g[1].defined()) return variable_list(7);
    no_tangent("linear_attention", {&g[0], &g[1]});
    const auto s = ctx->get_saved_variables();
    auto [dq, dk, dv, ds0] = [&] {
      at::AutoGradMode off(false);
      return attention_backward(s[0], s[1], s[2], s[3], s[4], s[5], g[0], g[1], ctx->saved_data["scale"].toDouble(), ctx->needs_input_grad(0),
                                ctx->needs_input_grad(1), ctx->needs_input_grad(2), ctx->saved_data["s0"].toBool());
    }();
    return first_order("linear_attention", {dq, dk, dv, Tensor(), ds0, Tensor(), Tensor()});
  }
};

std::tuple<Tensor, Tensor> linear_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Maybe& s0_,
                                            const Maybe& cu, optional<double> scale_) {
  check_attention(q, k, v, log_decay, s0_, cu);
  const Maybe s0 = there(s0_) && s0_->scalar_type() != at::kFloat ? Maybe(s0_->to(at::kFloat)) : s0_;
  const double scale = scale_of(scale_, q.size(-1));
  if (!wants_grad({&q, &k, &v, at_of(s0)})) return attention_forward(q, k, v, log_decay, s0, cu, scale);
  variable_list out = LinearAttention::apply(q, k, v, log_decay, s0, cu, scale);
  return {out[0], out[1]};
}

Tensor linear_attention_step(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& log_decay, const Tensor& s,
                             optional<double> scale) {
  no_tangent("linear_attention_step", {&q_, &k_, &v_, &log_decay, &s});
  check_heads("linear_attention_step", "[B, H, D],", q_, k_, v_, log_decay, 1);
  const int64_t B = q_.size(0), H = q_.size(1), Hk = k_.size(1), Dk = q_.size(2), Dv = v_.size(2);
  TORCH_CHECK_VALUE(s.dim() == 4 && s.size(0) == B && s.size(1) == H && s.size(2) == Dk && s.size(3) == Dv && s.scalar_type() == at::kFloat &&
                        s.is_contiguous() && reinterpret_cast<uintptr_t>(s.data_ptr()) % 16 == 0,
                    "linear_attention_step: s is a contiguous float32 state [", B, ", ", H, ", ", Dk, ", ", Dv, "], 16-byte aligned");
  TORCH_CHECK_VALUE(!wants_grad({&q_, &k_, &v_, &s}),
                    "linear_attention_step: not differentiable; call it under torch.no_grad() or use linear_attention");
  on_one_device("linear_attention_step", {&q_, &k_, &v_, &log_decay, &s});
  const c10::cuda::CUDAGuard guard(q_.device());
  const Tensor q = rows(q_), k = rows(k_), v = rows(v_);
  Tensor o = room(q, {B, H, Dv});
  s.unsafeGetTensorImpl()->bump_version();  // first: it raises where s may not be changed
  const int64_t st[6] = {q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1)};
  check("csn_linear_attention_step",
        csn_linear_attention_step(ptr(q), ptr(k), ptr(v), st, static_cast<const float*>(ptr(log_decay)), static_cast<float*>(ptr(s)), ptr(o), B,
                                  H, Hk, Dk, Dv, (float)scale_of(scale, Dk), code_of(q.scalar_type()), stream(q)));
  return o;
}

// --------------------------------------------------------- layer norm of 16-bit rows
std::tuple<Tensor, Tensor> norm_forward(const Tensor& x, const Tensor& w_, const Tensor& b_, double eps, bool keep) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor w = w_.contiguous(), b = b_.contiguous();
  const int64_t R = x.size(0), C = x.size(1);
  Tensor y = room(x, {R, C}), kept = keep ? floats(x, {2, R}) : Tensor();
  float* k = static_cast<float*>(ptr(kept));
  check("csn_layer_norm_rows_fwd", csn_layer_norm_rows_fwd(ptr(x), x.stride(0), ptr(w), ptr(b), ptr(y), k, k ? k + R : nullptr, R, C, (float)eps,
                                                           code_of(x.scalar_type()), code_of(w.scalar_type()), stream(x)));
  return {y, kept};
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& b, double eps) {
    auto [y, kept] = norm_forward(x, w, b, eps, true);
    ctx->save_for_backward({x, w, kept});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    no_tangent("layer_norm", {&g[0]});
    auto [dx, dw, db] = [&] {
      at::AutoGradMode off(false);
      const Tensor &x = s[0], w = s[1].contiguous(), &kept = s[2], dy = rows(g[0]);
      const c10::cuda::CUDAGuard guard(x.device());
      const int64_t R = x.size(0), C = x.size(1);
      Tensor dx = ctx->needs_input_grad(0) ? room(x, {R, C}) : Tensor(), dw = ctx->needs_input_grad(1) ? room(w, {C}) : Tensor();
      Tensor db = ctx->needs_input_grad(2) ? room(w, {C}) : Tensor();
      const size_t nb = dw.defined() || db.defined() ? csn_layer_norm_rows_bwd_workspace_bytes(R, C) : 0;
      const Tensor ws = bytes(x, nb);
      const float* k = static_cast<const float*>(ptr(kept));
      check("csn_layer_norm_rows_bwd",
            csn_layer_norm_rows_bwd(ptr(dy), dy.stride(0), ptr(x), x.stride(0), k, k + R, ptr(w), ptr(dx), ptr(dw), ptr(db), R, C,
                                    code_of(x.scalar_type()), code_of(w.scalar_type()), ptr(ws), nb, stream(x)));
      return std::make_tuple(dx, dw, db);
    }();
    return first_order("layer_norm", {dx, dw, db, Tensor()});
  }
};

Tensor layer_norm_rows(const Tensor& x, const Tensor& w_, const Tensor& b_, double eps) {
  no_tangent("layer_norm", {&x, &w_, &b_});
  of_one_type("layer_norm", false, {&x});
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && w_.dim() == 1 && b_.dim() == 1 && w_.size(0) == x.size(-1) && b_.size(0) == x.size(-1),
                    "layer_norm: x [..., C], weight and bias [C] expected, got ", x.sizes(), ", ", w_.sizes(), " and ", b_.sizes());
  TORCH_CHECK_VALUE(at::isFloatingType(w_.scalar_type()) && at::isFloatingType(b_.scalar_type()), "layer_norm: weight and bias of a floating type expected");
  on_one_device("layer_norm", {&x, &w_, &b_});
  // weights of another type than the rows' are taken as float32
  const bool same = w_.scalar_type() == x.scalar_type() && b_.scalar_type() == x.scalar_type();
  const Tensor w = same ? w_ : w_.to(at::kFloat), b = same ? b_ : b_.to(at::kFloat);
  const Tensor r = rows(flat(x));
  Tensor y = wants_grad({&x, &w, &b}) ? LayerNorm::apply(r, w, b, eps) : std::get<0>(norm_forward(r, w, b, eps, false));
  return x.dim() == 2 ? y : y.view(x.sizes());
}

// ------------------------------------------------------------------------ dropout
Tensor dropout_run(const Tensor& x_, const Maybe& residual_, int64_t cut, const Tensor& rng) {
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = packed(x_), residual = packed(residual_);
  Tensor y = room(x, x.sizes());
  check("csn_dropout_add", csn_dropout_add(ptr(x), ptr(residual), static_cast<const int64_t*>(ptr(rng)), ptr(y), x.numel(), (int)cut,
                                           code_of(x.scalar_type()), stream(x)));
  return y;
}

struct DropoutAdd : torch::autograd::Function<DropoutAdd> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& residual, int64_t cut, const Tensor& rng) {
    ctx->save_for_backward({rng});  // changing rng in place before the backward pass raises there
    ctx->saved_data["cut"] = cut;
    ctx->saved_data["x"] = x.requires_grad();
    ctx->saved_data["residual"] = there(residual) && residual->requires_grad();
    return dropout_run(x, residual, cut, rng);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const Tensor rng = ctx->get_saved_variables()[0];
    no_tangent("dropout_add", {&g[0]});
    Tensor dx;
    if (ctx->saved_data["x"].toBool()) {
      at::AutoGradMode off(false);
      dx = dropout_run(g[0], std::nullopt, ctx->saved_data["cut"].toInt(), rng);
    }
    return first_order("dropout_add", {dx, ctx->saved_data["residual"].toBool() ? g[0] : Tensor(), Tensor(), Tensor()});
  }
};

Tensor dropout_add(const Tensor& x, const Maybe& residual, double p, const Tensor& rng) {
  no_tangent("dropout_add", {&x, at_of(residual)});
  on_one_device("dropout_add", {&x, at_of(residual), &rng});
  of_one_type("dropout_add", true, {&x, at_of(residual)});
  TORCH_CHECK_VALUE(!there(residual) || residual->sizes() == x.sizes(), "dropout_add: x and residual of one shape expected");
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "dropout_add: 0 <= p <= 1 expected, got ", p);
  TORCH_CHECK_VALUE(rng.scalar_type() == at::kLong && rng.dim() == 1 && rng.size(0) == 2 && rng.is_contiguous(),
                    "dropout_add: rng is a contiguous int64 tensor (seed, offset)");
  const int64_t cut = std::llrint(p * 65536.0);
  return wants_grad({&x, at_of(residual)}) ? DropoutAdd::apply(x, residual, cut, rng) : dropout_run(x, residual, cut, rng);
}

}  // namespace

PYBIND11_MODULE(_gated, m) {
  namespace py = pybind11;
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Failure& e) {
      py::object type = py::module_::import("csn_b200._lib").attr("CsnError");
      PyErr_SetObject(type.ptr(), type(e.entry, e.code, e.text).ptr());
    }
  });
  m.def("gated_scan", &gated_scan);
  m.def("gated_scan_check", &check_scan);
  m.def("gated_scan_forward", &scan_forward);
  m.def("gated_scan_backward", &gated_scan_backward);
  m.def("gated_step", &gated_step);
  m.def("silu_gated_linear", &silu_gated_linear);
  m.def("silu_gated_linear_backward", &silu_gated_linear_backward);
  m.def("dropout_add", &dropout_add);
  m.def("linear_attention", &linear_attention);
  m.def("linear_attention_check", &check_attention);
  m.def("linear_attention_forward", [](const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Maybe& s0,
                                       const Maybe& cu, optional<double> scale) {
    return attention_forward(q, k, v, log_decay, s0, cu, scale_of(scale, q.size(-1)));
  });
  m.def("linear_attention_backward", &linear_attention_backward);
  m.def("linear_attention_step", &linear_attention_step);
  m.def("layer_norm_rows", &layer_norm_rows);
}

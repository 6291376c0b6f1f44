// The Python module scao_amd._torch_host: what would cost more host time in
// Python than the kernels take.
//
//   grad_norm, grad_clip
//               the norm of a model's gradients and their clipping as operators of
//               torch's dispatcher: reading six properties of 332 tensors from
//               Python takes 125 us, their norm and scaling 25
//   gated_ffn   the feed-forward block as an operator of torch's dispatcher, its
//               backward pass without the interpreter: a small block's training
//               step took 145 us of host time as a Python function
//   orthogonalize, muon_step
//               matrix updates orthogonalised, and the step of the optimiser that is
//               built on it, as operators of the dispatcher over lists of tensors
//   qk_norm_rope
//               norms of queries and keys with their rotation, forward and backward
//   bind        the addresses of the C ABI's entry points, which the caller has
//               loaded (so that one library is used, whichever it is)
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "../../include/scao_train.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Entries {
  decltype(&scao_last_error) last_error;
  decltype(&scao_ffn_saved_bytes) saved_bytes;
  decltype(&scao_ffn_forward_workspace) forward_workspace;
  decltype(&scao_ffn_forward) forward;
  decltype(&scao_ffn_backward_workspace) backward_workspace;
  decltype(&scao_ffn_backward) backward;
  decltype(&scao_grad_norm_workspace) grad_norm_workspace;
  decltype(&scao_grad_norm) grad_norm;
  decltype(&scao_grad_clip) grad_clip;
  decltype(&scao_orthogonalize_workspace) orthogonalize_workspace;
  decltype(&scao_orthogonalize) orthogonalize;
  decltype(&scao_muon_workspace) muon_workspace;
  decltype(&scao_muon_step) muon_step;
  decltype(&scao_qk_rope_forward) rope_forward;
  decltype(&scao_qk_rope_backward_workspace) rope_backward_workspace;
  decltype(&scao_qk_rope_backward) rope_backward;
} lib;

void check(int rc, const char* who) {
  TORCH_CHECK(rc == SCAO_OK, who, " failed (", rc, "): ", lib.last_error());
}

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return SCAO_F32;
    case at::kBFloat16: return SCAO_BF16;
    case at::kHalf: return SCAO_F16;
    default: return -1;
  }
}

void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}
Tensor bytes(int64_t n, const Tensor& like) {
  return at::empty({n}, like.options().dtype(at::kByte));
}

// whether any tensor may have a tangent (asking a view takes a lock)
bool forward_mode() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }

// ------------------------------------------------------------- gated_ffn ---
// Operators of torch's dispatcher, so that what follows a program by its
// operators (tracers, dispatch modes, negated views, tensor subclasses) finds the
// block among them, or refuses it:
//   gated_ffn           without a gradient
//   gated_ffn_save      the same, and what the backward pass needs
//   gated_ffn_backward  the wanted gradients (bits SCAO_FFN_DX ...) in order
constexpr int64_t MAX_STRIDE = (int64_t)1 << 21;   // of rows that scao_ffn_* take

Tensor op_gated_ffn(const Tensor& x, const Tensor& g, const Tensor& u, const Tensor& d,
                    int64_t act) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("scao_amd::gated_ffn", "")
                             .typed<decltype(op_gated_ffn)>();
  return op.call(x, g, u, d, act);
}
std::tuple<Tensor, Tensor> op_gated_ffn_save(const Tensor& x, const Tensor& g, const Tensor& u,
                                             const Tensor& d, int64_t act) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("scao_amd::gated_ffn_save", "")
                             .typed<decltype(op_gated_ffn_save)>();
  return op.call(x, g, u, d, act);
}
std::vector<Tensor> op_gated_ffn_backward(const Tensor& dy, const Tensor& saved, const Tensor& x,
                                          const Tensor& g, const Tensor& u, const Tensor& d,
                                          int64_t act, int64_t wanted) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("scao_amd::gated_ffn_backward", "")
                             .typed<decltype(op_gated_ffn_backward)>();
  return op.call(dy, saved, x, g, u, d, act, wanted);
}

// sizes, types and devices, whoever calls
void check_block(const Tensor& x, const Tensor& g, const Tensor& u, const Tensor& d) {
  TORCH_CHECK(lib.forward, "gated_ffn: scao_amd has not loaded its library");
  TORCH_CHECK(x.dim() == 2 && g.dim() == 2 && u.dim() == 2 && d.dim() == 2,
              "gated_ffn takes matrices");
  TORCH_CHECK(x.sym_size(1) == g.sym_size(1) && u.sym_sizes() == g.sym_sizes() &&
                  d.sym_size(0) == g.sym_size(1) && d.sym_size(1) == g.sym_size(0),
              "gated_ffn: shape mismatch: x ", x.sym_sizes(), ", w_gate ", g.sym_sizes(),
              ", w_up ", u.sym_sizes(), ", w_down ", d.sym_sizes());
  for (const Tensor* t : {&x, &g, &u, &d})
    TORCH_CHECK(code_of(t->scalar_type()) >= 0 && t->scalar_type() == x.scalar_type() &&
                    t->device() == x.device(),
                "gated_ffn takes float32, bfloat16 or float16 tensors of one type and device");
}

// t with unit column stride and rows that do not overlap and that scao_ffn_* take.
// (A single column may have any stride: torch calls it contiguous, and a copy
// would keep it.)
Tensor rows(const Tensor& t) {
  const bool unit = t.stride(1) == 1 || t.size(1) == 1;
  const bool apart = t.size(0) <= 1 || (t.stride(0) >= t.size(1) && t.stride(0) < MAX_STRIDE);
  return unit && apart ? t : t.contiguous();
}

// of matrices that rows() has made
scao_ffn_desc describe(const Tensor& x, const Tensor& g, const Tensor& u, const Tensor& d,
                       int64_t act) {
  return scao_ffn_desc{x.data_ptr(),  g.data_ptr(),  u.data_ptr(),        d.data_ptr(),
                       x.stride(0),   g.stride(0),   u.stride(0),         d.stride(0),
                       x.size(0),     g.size(1),     g.size(0),           code_of(x.scalar_type()),
                       (int32_t)act};
}

std::tuple<Tensor, Tensor> forward(const Tensor& x_, const Tensor& g_, const Tensor& u_,
                                   const Tensor& d_, int64_t act, bool save) {
  check_block(x_, g_, u_, d_);
  const c10::DeviceGuard guard(x_.device());
  const Tensor x = rows(x_), g = rows(g_), u = rows(u_), d = rows(d_);
  const scao_ffn_desc desc = describe(x, g, u, d, act);
  Tensor y = at::empty({x.size(0), x.size(1)}, x.options()), saved;
  if (save) saved = bytes(lib.saved_bytes(&desc), x);
  const Tensor work = bytes(lib.forward_workspace(&desc, save), x);
  check(lib.forward(&desc, y.data_ptr(), save ? saved.data_ptr() : nullptr, work.data_ptr(),
                    stream_of(x)),
        "scao_ffn_forward");
  return {y, saved};
}
Tensor gated_ffn_hip(const Tensor& x, const Tensor& g, const Tensor& u, const Tensor& d,
                     int64_t act) {
  return std::get<0>(forward(x, g, u, d, act, false));
}
std::tuple<Tensor, Tensor> gated_ffn_save_hip(const Tensor& x, const Tensor& g, const Tensor& u,
                                              const Tensor& d, int64_t act) {
  return forward(x, g, u, d, act, true);
}

std::vector<Tensor> gated_ffn_backward_hip(const Tensor& dy_, const Tensor& saved,
                                           const Tensor& x_, const Tensor& g_, const Tensor& u_,
                                           const Tensor& d_, int64_t act, int64_t wanted) {
  check_block(x_, g_, u_, d_);
  TORCH_CHECK(dy_.sizes() == x_.sizes() && dy_.scalar_type() == x_.scalar_type() &&
                  dy_.device() == x_.device(),
              "gated_ffn_backward: dy is not like x");
  const c10::DeviceGuard guard(x_.device());
  const Tensor x = rows(x_), g = rows(g_), u = rows(u_), d = rows(d_), dy = rows(dy_);
  const scao_ffn_desc desc = describe(x, g, u, d, act);
  TORCH_CHECK(saved.scalar_type() == at::kByte && saved.device() == x.device() &&
                  saved.is_contiguous() && saved.numel() == lib.saved_bytes(&desc),
              "gated_ffn_backward: saved is not what gated_ffn_save returned");
  static_assert(SCAO_FFN_DX == 1 && SCAO_FFN_DGATE == 2 && SCAO_FFN_DUP == 4 &&
                    SCAO_FFN_DDOWN == 8,
                "the inputs' order");
  std::vector<Tensor> out;
  const Tensor* like[4] = {&x, &g, &u, &d};
  void* to[4] = {};
  for (int i = 0; i < 4; ++i) {
    if (!(wanted >> i & 1)) continue;
    out.push_back(at::empty({like[i]->size(0), like[i]->size(1)}, x.options()));
    to[i] = out.back().data_ptr();
  }
  const Tensor work =
      bytes(lib.backward_workspace(&desc, dy.data_ptr(), dy.stride(0), (int)wanted & 15), x);
  check(lib.backward(&desc, dy.data_ptr(), dy.stride(0), saved.data_ptr(), to[0], to[1], to[2],
                     to[3], work.data_ptr(), stream_of(x)),
        "scao_ffn_backward");
  return out;
}

// shapes alone, for tensors without memory
Tensor like(const Tensor& t) { return at::empty_symint(t.sym_sizes(), t.options()); }
Tensor gated_ffn_meta(const Tensor& x, const Tensor& g, const Tensor& u, const Tensor& d,
                      int64_t) {
  check_block(x, g, u, d);
  return like(x);
}
std::tuple<Tensor, Tensor> gated_ffn_save_meta(const Tensor& x, const Tensor& g, const Tensor& u,
                                               const Tensor& d, int64_t act) {
  check_block(x, g, u, d);
  scao_ffn_desc desc{};
  desc.tokens = x.sym_size(0).guard_int(__FILE__, __LINE__);
  desc.d = g.sym_size(1).guard_int(__FILE__, __LINE__);
  desc.f = g.sym_size(0).guard_int(__FILE__, __LINE__);
  desc.dtype = code_of(x.scalar_type());
  desc.act = (int32_t)act;
  return {like(x), bytes(lib.saved_bytes(&desc), x)};
}
std::vector<Tensor> gated_ffn_backward_meta(const Tensor&, const Tensor&, const Tensor& x,
                                            const Tensor& g, const Tensor& u, const Tensor& d,
                                            int64_t, int64_t wanted) {
  std::vector<Tensor> out;
  int i = 0;
  for (const Tensor* t : {&x, &g, &u, &d})
    if (wanted >> i++ & 1) out.push_back(like(*t));
  return out;
}

struct GatedFFN : torch::autograd::Function<GatedFFN> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& g, const Tensor& u,
                        const Tensor& d, int64_t act) {
    const at::AutoDispatchBelowADInplaceOrView below;
    auto [y, saved] = op_gated_ffn_save(x, g, u, d, act);
    ctx->save_for_backward({x, g, u, d, saved});
    ctx->saved_data["act"] = act;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    // (hooks on saved tensors may have moved them: their addresses are new)
    const variable_list t = ctx->get_saved_variables();
    variable_list out(5);
    if (!grads[0].defined()) return out;
    int64_t wanted = 0;
    for (int i = 0; i < 4; ++i) wanted |= (int64_t)ctx->needs_input_grad(i) << i;
    variable_list have;
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      have = op_gated_ffn_backward(grads[0], t[4], t[0], t[1], t[2], t[3],
                                   ctx->saved_data["act"].toInt(), wanted);
    }
    if (at::GradMode::is_enabled()) {   // a gradient of these gradients is an error, not a zero
      const auto error = std::make_shared<torch::autograd::DelayedError>(
          "gated_ffn is differentiable once", 4);
      for (Tensor& g : have) g.requires_grad_(true);
      have = (*error)(std::move(have));
    }
    for (int i = 0, k = 0; i < 4; ++i)
      if (wanted >> i & 1) out[i] = have[k++];
    return out;
  }
};

Tensor gated_ffn_autograd(const Tensor& x, const Tensor& g, const Tensor& u, const Tensor& d,
                          int64_t act) {
  check_block(x, g, u, d);
  if (forward_mode())   // a tangent would be lost
    for (const Tensor* t : {&x, &g, &u, &d})
      TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(),
                                  "gated_ffn has no forward-mode derivative");
  if (at::GradMode::is_enabled() && (x.requires_grad() || g.requires_grad() ||
                                     u.requires_grad() || d.requires_grad()))
    // (what rows() copies, it copies here once for both passes)
    return GatedFFN::apply(rows(x), rows(g), rows(u), rows(d), act);
  const at::AutoDispatchBelowADInplaceOrView below;
  return op_gated_ffn(x, g, u, d, act);
}

TORCH_LIBRARY(scao_amd, m) {
#define SCAO_BLOCK "Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, int activation"
  m.def("gated_ffn(" SCAO_BLOCK ") -> Tensor");
  m.def("gated_ffn_save(" SCAO_BLOCK ") -> (Tensor, Tensor)");
  m.def("gated_ffn_backward(Tensor dy, Tensor saved, " SCAO_BLOCK ", int wanted) -> Tensor[]");
#undef SCAO_BLOCK
}
TORCH_LIBRARY_IMPL(scao_amd, CUDA, m) {
  m.impl("gated_ffn", gated_ffn_hip);
  m.impl("gated_ffn_save", gated_ffn_save_hip);
  m.impl("gated_ffn_backward", gated_ffn_backward_hip);
}
TORCH_LIBRARY_IMPL(scao_amd, Meta, m) {
  m.impl("gated_ffn", gated_ffn_meta);
  m.impl("gated_ffn_save", gated_ffn_save_meta);
  m.impl("gated_ffn_backward", gated_ffn_backward_meta);
}
TORCH_LIBRARY_IMPL(scao_amd, Autograd, m) { m.impl("gated_ffn", gated_ffn_autograd); }

PyObject* gated_ffn(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 5, "gated_ffn() takes five arguments");
  for (int i = 0; i < 4; ++i)
    TORCH_CHECK_TYPE(THPVariable_Check(args[i]), "gated_ffn() takes tensors");
  const long act = PyLong_AsLong(args[4]);
  if (act == -1 && PyErr_Occurred()) return nullptr;
  return THPVariable_Wrap(op_gated_ffn(THPVariable_Unpack(args[0]), THPVariable_Unpack(args[1]),
                                       THPVariable_Unpack(args[2]), THPVariable_Unpack(args[3]),
                                       act));
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------- gradient norm, clipping ---
// Operators of the dispatcher, as the block is:
//   grad_norm   the norm of a list of gradients, a 0-dim fp32 tensor
//   grad_clip_  the same, and the gradients scaled in place
// norm types as in scao_train.h
Tensor op_grad_norm(at::TensorList grads, int64_t norm_type, double scale) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("scao_amd::grad_norm", "")
                             .typed<decltype(op_grad_norm)>();
  return op.call(grads, norm_type, scale);
}
Tensor op_grad_clip_(at::TensorList grads, int64_t norm_type, double scale, double max_norm) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("scao_amd::grad_clip_", "")
                             .typed<decltype(op_grad_clip_)>();
  return op.call(grads, norm_type, scale, max_norm);
}

bool regular(const Tensor& g, c10::Device on) {
  return g.layout() == at::kStrided && code_of(g.scalar_type()) >= 0 && g.device() == on;
}
void check_gradient(const Tensor& g, c10::Device on) {
  TORCH_CHECK(regular(g, on), "gradients must be dense float32, bfloat16 or float16 tensors on "
              "one device (got ", g.scalar_type(), ", ", g.layout(), ", ", g.device(), ")");
}
void check_call(at::TensorList grads) {
  TORCH_CHECK(lib.grad_clip, "clip_grad_norm_: scao_amd has not loaded its library");
  TORCH_CHECK(!grads.empty(), "clip_grad_norm_: no gradients");
}

// The table of the gradients; those with gaps in their memory take part through
// a contiguous copy.
struct Gradients {
  std::vector<scao_tensor_desc> table;
  std::vector<std::pair<Tensor, Tensor>> copies;   // gradient, copy
  Tensor norm, work;

  explicit Gradients(at::TensorList grads) {
    table.reserve(grads.size());
    const c10::Device on = grads[0].device();
    for (const Tensor& g : grads) {
      check_gradient(g, on);
      // every element of its memory range once, in any order
      const bool dense = g.is_non_overlapping_and_dense();
      if (!dense) copies.emplace_back(g, g.contiguous());
      const Tensor& t = dense ? g : copies.back().second;
      table.push_back({t.data_ptr(), t.numel(), code_of(t.scalar_type()), 0});
    }
    norm = at::empty({}, grads[0].options().dtype(at::kFloat));
    work = bytes(lib.grad_norm_workspace(table.data(), (int)table.size()), grads[0]);
  }
};

Tensor grad_norm_hip(at::TensorList grads, int64_t norm_type, double scale) {
  check_call(grads);
  const c10::DeviceGuard guard(grads[0].device());
  const Gradients g(grads);
  check(lib.grad_norm(g.table.data(), (int)g.table.size(), (int)norm_type, scale,
                      (float*)g.norm.data_ptr(), g.work.data_ptr(), stream_of(g.norm)),
        "scao_grad_norm");
  return g.norm;
}

// Where the bytes of a tensor lie: begin + sum of i_k stride_k, 0 <= i_k < size_k.
struct Bytes {
  int64_t begin, end;
  std::vector<std::pair<int64_t, int64_t>> dims;   // size, stride
  explicit Bytes(const Tensor& t) : begin((int64_t)(uintptr_t)t.data_ptr()) {
    const int64_t item = (int64_t)t.element_size();
    if (t.is_non_overlapping_and_dense()) {
      dims = {{t.numel() * item, 1}};
    } else {
      for (int64_t k = 0; k < t.dim(); ++k)
        if (t.size(k) > 1) dims.emplace_back(t.size(k), t.stride(k) * item);
      dims.emplace_back(item, 1);
    }
    end = begin + 1;
    for (const auto& [size, stride] : dims) end += (size - 1) * stride;
  }
};
// Solutions of sum t_k stride_k = to with lo_k <= t_k <= hi_k, up to `enough`: term
// by term from the largest stride on, taking only what the others can make up
// for. That is one or two values of t where the strides are those of one buffer's
// parts; with others it may take too long to tell, which counts as enough.
struct Sums {
  struct Term {
    int64_t stride, lo, hi;
  };
  std::vector<Term> terms;
  int enough, found = 0, steps = 0;
  explicit Sums(int n) : enough(n) {}
  void add(int64_t stride, int64_t lo, int64_t hi) {
    for (Term& t : terms)
      if (t.stride == stride) {
        t.lo += lo;
        t.hi += hi;
        return;
      }
    terms.push_back({stride, lo, hi});
  }
  bool reach(int64_t to) {
    std::sort(terms.begin(), terms.end(),
              [](const Term& a, const Term& b) { return a.stride > b.stride; });
    walk(0, to);
    return found >= enough;
  }
  void walk(size_t k, int64_t to) {
    if (++steps > 1 << 16) found = enough;
    if (found >= enough) return;
    if (k == terms.size()) {
      found += to == 0;
      return;
    }
    int64_t low = 0, high = 0;   // what the terms behind this one can add up to
    for (size_t j = k + 1; j < terms.size(); ++j) {
      low += terms[j].lo * terms[j].stride;
      high += terms[j].hi * terms[j].stride;
    }
    const auto [stride, lo, hi] = terms[k];
    auto floor = [s = stride](int64_t x) { return x / s - (x % s < 0); };
    const int64_t last = std::min(hi, floor(to - low));
    for (int64_t t = std::max(lo, -floor(high - to)); t <= last && found < enough; ++t)
      walk(k + 1, to - t * stride);
  }
};
bool share_memory(const Bytes& a, const Bytes& b) {
  if (a.end <= b.begin || b.end <= a.begin) return false;
  Sums s(1);
  for (const auto& [size, stride] : a.dims) s.add(stride, 0, size - 1);
  for (const auto& [size, stride] : b.dims) s.add(stride, 1 - size, 0);
  return s.reach(b.begin - a.begin);
}
// two elements of one tensor: all t_k zero is one solution (and each term stands
// for itself, so that two of one stride have others)
bool share_memory(const Bytes& a) {
  Sums s(2);
  for (const auto& [size, stride] : a.dims) s.terms.push_back({stride, 1 - size, size - 1});
  return s.reach(0);
}
// Gradients with gaps: scao_grad_clip sees their copies and cannot tell.
void check_apart(at::TensorList grads, const std::vector<std::pair<Tensor, Tensor>>& copies) {
  if (copies.empty()) return;
  std::vector<Bytes> gaps, all;
  for (const Tensor& g : grads) {
    if (g.numel() == 0) continue;
    (g.is_non_overlapping_and_dense() ? all : gaps).emplace_back(g);
  }
  for (size_t i = 0; i < gaps.size(); ++i) {
    TORCH_CHECK_VALUE(!share_memory(gaps[i]), "elements of a gradient share memory");
    for (const Bytes& b : all)
      TORCH_CHECK_VALUE(!share_memory(gaps[i], b), "two gradients share memory");
    all.push_back(gaps[i]);
  }
}

Tensor grad_clip_hip_(at::TensorList grads, int64_t norm_type, double scale, double max_norm) {
  check_call(grads);
  const c10::DeviceGuard guard(grads[0].device());
  const Gradients g(grads);
  for (const auto& [to, copy] : g.copies)
    TORCH_CHECK_VALUE(at::has_internal_overlap(to) != at::MemOverlap::Yes,
                      "a gradient whose elements share memory (an expanded tensor) cannot be "
                      "scaled in place");
  check_apart(grads, g.copies);
  const int rc = lib.grad_clip(g.table.data(), (int)g.table.size(), (int)norm_type, scale, max_norm,
                               (float*)g.norm.data_ptr(), g.work.data_ptr(), stream_of(g.norm));
  TORCH_CHECK_VALUE(rc == SCAO_OK || !strstr(lib.last_error(), "share memory"), lib.last_error());
  check(rc, "scao_grad_clip");
  for (const auto& [to, copy] : g.copies) to.copy_(copy);
  return g.norm;
}

// a graph that holds a gradient has to see that it changed
Tensor grad_clip_version_(at::TensorList grads, int64_t norm_type, double scale, double max_norm) {
  Tensor norm;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    norm = op_grad_clip_(grads, norm_type, scale, max_norm);
  }
  for (const Tensor& g : grads)
    if (!g.is_inference()) g.unsafeGetTensorImpl()->bump_version();
  return norm;
}

Tensor grad_norm_meta(at::TensorList grads, int64_t, double) {
  check_call(grads);
  for (const Tensor& g : grads) check_gradient(g, grads[0].device());
  return at::empty({}, grads[0].options().dtype(at::kFloat));
}
Tensor grad_clip_meta_(at::TensorList grads, int64_t norm_type, double scale, double) {
  return grad_norm_meta(grads, norm_type, scale);
}

TORCH_LIBRARY_FRAGMENT(scao_amd, m) {
  m.def("grad_norm(Tensor[] grads, int norm_type, float scale) -> Tensor");
  m.def("grad_clip_(Tensor(a!)[] grads, int norm_type, float scale, float max_norm) -> Tensor");
}
TORCH_LIBRARY_IMPL(scao_amd, CUDA, m) {
  m.impl("grad_norm", grad_norm_hip);
  m.impl("grad_clip_", grad_clip_hip_);
}
TORCH_LIBRARY_IMPL(scao_amd, Meta, m) {
  m.impl("grad_norm", grad_norm_meta);
  m.impl("grad_clip_", grad_clip_meta_);
}
TORCH_LIBRARY_IMPL(scao_amd, ADInplaceOrView, m) { m.impl("grad_clip_", grad_clip_version_); }
// neither depends on the sign of what is held
TORCH_LIBRARY_IMPL(scao_amd, Negative, m) {
  m.impl("grad_norm", torch::CppFunction::makeFallthrough());
  m.impl("grad_clip_", torch::CppFunction::makeFallthrough());
}

// The gradients of a list or tuple of tensors, those that have one; false where
// any of them is not a dense fp32, bf16 or fp16 tensor on the first one's GPU,
// for the caller to refuse.
bool collect(PyObject* parameters, std::vector<Tensor>& grads) {
  const THPObjectPtr seq(PySequence_Fast(parameters, "a list or a tuple of parameters"));
  if (!seq) throw python_error();
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq.get());
  grads.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PySequence_Fast_GET_ITEM(seq.get(), i);
    if (!THPVariable_Check(o)) return false;
    const Tensor& g = THPVariable_Unpack(o).grad();
    if (!g.defined()) continue;
    if (!g.is_cuda() || !regular(g, grads.empty() ? g.device() : grads[0].device())) return false;
    grads.push_back(g);
  }
  return true;
}

// grad_norm(parameters, norm_type, scale), grad_clip(parameters, norm_type, scale,
// max_norm) -> the norm; None where there is no gradient, False where one is not
// as collect() says
PyObject* call_on_gradients(PyObject* const* args, Py_ssize_t n, bool clip) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == (clip ? 4 : 3), "wrong number of arguments");
  std::vector<Tensor> grads;
  if (!collect(args[0], grads)) Py_RETURN_FALSE;
  const long norm_type = PyLong_AsLong(args[1]);
  const double scale = PyFloat_AsDouble(args[2]);
  const double max_norm = clip ? PyFloat_AsDouble(args[3]) : 0;
  if (PyErr_Occurred()) return nullptr;
  if (grads.empty()) Py_RETURN_NONE;
  if (forward_mode())   // a tangent would be lost
    for (const Tensor& g : grads)
      TORCH_CHECK_NOT_IMPLEMENTED(!g._fw_grad(0).defined(),
                                  "the gradients' norm has no forward-mode derivative");
  const at::AutoDispatchBelowAutograd below;
  return THPVariable_Wrap(clip ? op_grad_clip_(grads, norm_type, scale, max_norm)
                               : op_grad_norm(grads, norm_type, scale));
  END_HANDLE_TH_ERRORS
}
PyObject* grad_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return call_on_gradients(args, n, false);
}
PyObject* grad_clip(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return call_on_gradients(args, n, true);
}

// -------------------------------------------------- orthogonalised updates ---
// Operators of the dispatcher over lists of matrices and stacks of matrices:
//   orthogonalize  fresh results of one type
//   muon_step_     parameters and momenta written in place
std::vector<Tensor> op_orthogonalize(at::TensorList updates, at::ArrayRef<double> coefficients,
                                     double eps, std::optional<at::ScalarType> dtype,
                                     std::optional<at::ScalarType> ns_dtype) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("scao_amd::orthogonalize", "")
                             .typed<decltype(op_orthogonalize)>();
  return op.call(updates, coefficients, eps, dtype, ns_dtype);
}
void op_muon_step_(at::TensorList params, at::TensorList grads, at::TensorList momenta,
                   at::ArrayRef<double> rates, at::ArrayRef<double> decays, double momentum,
                   bool nesterov, at::ArrayRef<double> coefficients, double eps,
                   at::IntArrayRef precisions) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("scao_amd::muon_step_", "")
                             .typed<decltype(op_muon_step_)>();
  op.call(params, grads, momenta, rates, decays, momentum, nesterov, coefficients, eps, precisions);
}

void check_matrices(at::TensorList list, const char* name, c10::Device on) {
  for (const Tensor& t : list) {
    TORCH_CHECK(t.layout() == at::kStrided && code_of(t.scalar_type()) >= 0 && t.device() == on,
                name, " must be dense float32, bfloat16 or float16 tensors on one device (got ",
                t.scalar_type(), ", ", t.layout(), ", ", t.device(), ")");
    TORCH_CHECK(t.dim() >= 2, name, " must be matrices or stacks of matrices (got ",
                t.sym_sizes(), ")");
    const auto rows = t.sym_size(-2), cols = t.sym_size(-1);
    constexpr int64_t SIDE = (int64_t)1 << 20, SMALLER = (int64_t)1 << 15;   // scao_train.h's
    TORCH_CHECK(t.sym_numel() == 0 ||
                    (rows < SIDE && cols < SIDE && (rows <= SMALLER || cols <= SMALLER)), name,
                " must have sides below 2^20, the smaller one up to 2^15 (got ", t.sym_sizes(), ")");
  }
}
void check_result(std::optional<at::ScalarType> dtype, std::optional<at::ScalarType> ns_dtype) {
  TORCH_CHECK(!dtype || code_of(*dtype) >= 0, "orthogonalize: no result of type ", *dtype);
  TORCH_CHECK(!ns_dtype || *ns_dtype == at::kFloat || *ns_dtype == at::kBFloat16,
              "orthogonalize: no products of type ", *ns_dtype);
}
void check_scheme(at::ArrayRef<double> coefficients) {
  TORCH_CHECK(lib.orthogonalize, "orthogonalize: scao_amd has not loaded its library");
  TORCH_CHECK(!coefficients.empty() && coefficients.size() % 3 == 0 &&
                  coefficients.size() <= 3 * 64,
              "orthogonalize: three coefficients a step, up to 64 steps");
}

// the matrices of a stack, whose rows are unit-strided and apart
template <class F>
void for_matrices(const Tensor& t, F&& f) {
  const int64_t n = t.dim(), rows = t.size(n - 2), cols = t.size(n - 1);
  int64_t many = 1;
  for (int64_t k = 0; k < n - 2; ++k) many *= t.size(k);
  if (many * rows * cols == 0) return;
  char* base = (char*)t.data_ptr();
  for (int64_t i = 0; i < many; ++i) {
    int64_t at = 0, left = i;
    for (int64_t k = n - 3; k >= 0; --k) {
      at += left % t.size(k) * t.stride(k);
      left /= t.size(k);
    }
    f(base + at * (int64_t)t.element_size(), rows, cols, t.stride(n - 2));
  }
}
Tensor row_strided(const Tensor& t) {
  const int64_t n = t.dim();
  const bool unit = t.stride(n - 1) == 1 || t.size(n - 1) == 1;
  return unit && (t.size(n - 2) <= 1 || (t.stride(n - 2) >= t.size(n - 1) &&
                                         t.stride(n - 2) <= 0x7fffffff))
             ? t
             : t.contiguous();
}

std::vector<Tensor> orthogonalize_hip(at::TensorList updates, at::ArrayRef<double> coefficients,
                                      double eps, std::optional<at::ScalarType> dtype,
                                      std::optional<at::ScalarType> ns_dtype) {
  check_scheme(coefficients);
  std::vector<Tensor> out;
  if (updates.empty()) return out;
  check_matrices(updates, "updates", updates[0].device());
  check_result(dtype, ns_dtype);
  const c10::DeviceGuard guard(updates[0].device());
  std::vector<Tensor> in;
  std::vector<scao_ortho_desc> table;
  for (const Tensor& t : updates) {
    in.push_back(row_strided(t.resolve_neg()));
    const at::ScalarType type = dtype.value_or(t.scalar_type());
    out.push_back(at::empty(t.sizes(), t.options().dtype(type)));
    // by default one word an element where the result has fewer bits than it
    const int precision =
        ns_dtype.value_or(type) == at::kBFloat16 ? SCAO_ORTHO_FAST : SCAO_ORTHO_FP32;
    char* to = (char*)out.back().data_ptr();
    for_matrices(in.back(), [&](char* p, int64_t rows, int64_t cols, int64_t ld) {
      table.push_back({p, to, rows, cols, ld, cols, code_of(t.scalar_type()), code_of(type),
                       precision, 0});
      to += rows * cols * (int64_t)out.back().element_size();
    });
  }
  const int steps = (int)coefficients.size() / 3, n = (int)table.size();
  const Tensor work = bytes(lib.orthogonalize_workspace(table.data(), n, steps), updates[0]);
  check(lib.orthogonalize(table.data(), n, coefficients.data(), steps, eps, work.data_ptr(),
                          stream_of(updates[0])),
        "scao_orthogonalize");
  return out;
}

void check_step(at::TensorList params, at::TensorList grads, at::TensorList momenta,
                at::ArrayRef<double> rates, at::ArrayRef<double> decays,
                at::IntArrayRef precisions) {
  const size_t n = params.size();
  TORCH_CHECK(grads.size() == n && momenta.size() == n && rates.size() == n && decays.size() == n &&
                  precisions.size() == n,
              "muon_step_: lists of different lengths");
  if (!n) return;
  const c10::Device on = params[0].device();
  check_matrices(params, "parameters", on);
  check_matrices(grads, "gradients", on);
  for (size_t i = 0; i < n; ++i) {
    const Tensor &p = params[i], &m = momenta[i];
    TORCH_CHECK(p.is_contiguous() && !p.is_neg() && m.is_contiguous() && !m.is_neg() &&
                    m.scalar_type() == at::kFloat && m.device() == on &&
                    m.sym_sizes() == p.sym_sizes() && grads[i].sym_sizes() == p.sym_sizes(),
                "muon_step_: a parameter and its momentum must be contiguous, the momentum "
                "float32, and both and the gradient of one shape");
  }
}
void muon_step_hip_(at::TensorList params, at::TensorList grads, at::TensorList momenta,
                    at::ArrayRef<double> rates, at::ArrayRef<double> decays, double momentum,
                    bool nesterov, at::ArrayRef<double> coefficients, double eps,
                    at::IntArrayRef precisions) {
  check_scheme(coefficients);
  check_step(params, grads, momenta, rates, decays, precisions);
  const size_t n = params.size();
  if (!n) return;
  const c10::Device on = params[0].device();
  const c10::DeviceGuard guard(on);
  std::vector<Tensor> copies;
  std::vector<scao_muon_desc> table;
  for (size_t i = 0; i < n; ++i) {
    const Tensor &p = params[i], &m = momenta[i];
    copies.push_back(grads[i].resolve_neg().contiguous());
    const char* g = (const char*)copies.back().data_ptr();
    float* buf = (float*)m.data_ptr();
    const int64_t g_size = (int64_t)copies.back().element_size();
    for_matrices(p, [&](char* at, int64_t rows, int64_t cols, int64_t) {
      table.push_back({at, g, buf, rows, cols, code_of(p.scalar_type()),
                       code_of(copies.back().scalar_type()), (float)rates[i], (float)decays[i],
                       (int32_t)precisions[i], 0});
      g += rows * cols * g_size;
      buf += rows * cols;
    });
  }
  const int steps = (int)coefficients.size() / 3, many = (int)table.size();
  const Tensor work = bytes(lib.muon_workspace(table.data(), many, steps), params[0]);
  check(lib.muon_step(table.data(), many, momentum, nesterov, coefficients.data(), steps, eps,
                      work.data_ptr(), stream_of(params[0])),
        "scao_muon_step");
}
// a graph that holds a parameter has to see that it changed
void muon_step_version_(at::TensorList params, at::TensorList grads, at::TensorList momenta,
                        at::ArrayRef<double> rates, at::ArrayRef<double> decays, double momentum,
                        bool nesterov, at::ArrayRef<double> coefficients, double eps,
                        at::IntArrayRef precisions) {
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    op_muon_step_(params, grads, momenta, rates, decays, momentum, nesterov, coefficients, eps,
                  precisions);
  }
  for (const at::TensorList list : {params, momenta})
    for (const Tensor& t : list)
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

std::vector<Tensor> orthogonalize_meta(at::TensorList updates, at::ArrayRef<double> coefficients,
                                       double, std::optional<at::ScalarType> dtype,
                                       std::optional<at::ScalarType> ns_dtype) {
  check_scheme(coefficients);
  std::vector<Tensor> out;
  if (!updates.empty()) check_matrices(updates, "updates", updates[0].device());
  check_result(dtype, ns_dtype);
  for (const Tensor& t : updates)
    out.push_back(at::empty_symint(t.sym_sizes(), t.options().dtype(dtype.value_or(t.scalar_type()))));
  return out;
}
void muon_step_meta_(at::TensorList params, at::TensorList grads, at::TensorList momenta,
                     at::ArrayRef<double> rates, at::ArrayRef<double> decays, double, bool,
                     at::ArrayRef<double> coefficients, double, at::IntArrayRef precisions) {
  check_scheme(coefficients);
  check_step(params, grads, momenta, rates, decays, precisions);
}

bool tangent(at::TensorList list) {
  if (forward_mode())
    for (const Tensor& t : list)
      if (t._fw_grad(0).defined()) return true;
  return false;
}
std::vector<Tensor> orthogonalize_autograd(at::TensorList updates,
                                           at::ArrayRef<double> coefficients, double eps,
                                           std::optional<at::ScalarType> dtype,
                                           std::optional<at::ScalarType> ns_dtype) {
  bool wanted = tangent(updates);
  if (at::GradMode::is_enabled())
    for (const Tensor& t : updates) wanted = wanted || t.requires_grad();
  TORCH_CHECK_NOT_IMPLEMENTED(!wanted, "orthogonalize has no derivative: detach the updates");
  const at::AutoDispatchBelowADInplaceOrView below;
  return op_orthogonalize(updates, coefficients, eps, dtype, ns_dtype);
}

TORCH_LIBRARY_FRAGMENT(scao_amd, m) {
  m.def("orthogonalize(Tensor[] updates, float[] coefficients, float eps, ScalarType? dtype, "
        "ScalarType? ns_dtype=None) -> Tensor[]");
  m.def("muon_step_(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] momenta, float[] rates, "
        "float[] decays, float momentum, bool nesterov, float[] coefficients, float eps, "
        "int[] precisions) -> ()");
}
TORCH_LIBRARY_IMPL(scao_amd, CUDA, m) {
  m.impl("orthogonalize", orthogonalize_hip);
  m.impl("muon_step_", muon_step_hip_);
}
TORCH_LIBRARY_IMPL(scao_amd, Meta, m) {
  m.impl("orthogonalize", orthogonalize_meta);
  m.impl("muon_step_", muon_step_meta_);
}
TORCH_LIBRARY_IMPL(scao_amd, Autograd, m) { m.impl("orthogonalize", orthogonalize_autograd); }
TORCH_LIBRARY_IMPL(scao_amd, ADInplaceOrView, m) { m.impl("muon_step_", muon_step_version_); }
// (torch's fallback does not look into lists; the kernels above do)
TORCH_LIBRARY_IMPL(scao_amd, Negative, m) {
  m.impl("orthogonalize", torch::CppFunction::makeFallthrough());
  m.impl("muon_step_", torch::CppFunction::makeFallthrough());
}

std::vector<Tensor> tensors(PyObject* list) {
  const THPObjectPtr seq(PySequence_Fast(list, "a list of tensors"));
  if (!seq) throw python_error();
  std::vector<Tensor> out;
  for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(seq.get()); ++i) {
    PyObject* o = PySequence_Fast_GET_ITEM(seq.get(), i);
    TORCH_CHECK_TYPE(THPVariable_Check(o), "a list of tensors");
    out.push_back(THPVariable_Unpack(o));
  }
  return out;
}
std::vector<double> numbers(PyObject* list) {
  const THPObjectPtr seq(PySequence_Fast(list, "a list of numbers"));
  if (!seq) throw python_error();
  std::vector<double> out;
  for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(seq.get()); ++i)
    out.push_back(PyFloat_AsDouble(PySequence_Fast_GET_ITEM(seq.get(), i)));
  if (PyErr_Occurred()) throw python_error();
  return out;
}
// muon_step(parameters, gradients, momenta, rates, decays, momentum, nesterov,
// coefficients, eps, precisions)
PyObject* muon_step(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 10, "muon_step() takes ten arguments");
  const std::vector<Tensor> params = tensors(args[0]), grads = tensors(args[1]),
                            momenta = tensors(args[2]);
  const std::vector<double> rates = numbers(args[3]), decays = numbers(args[4]),
                            coefficients = numbers(args[7]);
  const double momentum = PyFloat_AsDouble(args[5]), eps = PyFloat_AsDouble(args[8]);
  const int nesterov = PyObject_IsTrue(args[6]);
  std::vector<int64_t> precisions;
  for (const double p : numbers(args[9])) precisions.push_back((int64_t)p);
  if (PyErr_Occurred()) return nullptr;
  const at::AutoDispatchBelowAutograd below;
  op_muon_step_(params, grads, momenta, rates, decays, momentum, nesterov != 0, coefficients, eps,
                precisions);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------- norms of queries and keys, rotation ---
//   qk_norm_rope           both outputs
//   qk_norm_rope_backward  dq, dk, dw_q, dw_k: the wanted ones (bits 1, 2, 4, 8) in order
#define ROPE_PARAMS                                                                    \
  const Tensor &q, const Tensor &k, const std::optional<Tensor>&wq,                    \
      const std::optional<Tensor>&wk, const Tensor &cos, const Tensor &sin,            \
      const std::optional<Tensor>&positions, double eps, bool interleaved
#define ROPE_ARGS q, k, wq, wk, cos, sin, positions, eps, interleaved

std::tuple<Tensor, Tensor> op_qk_norm_rope(ROPE_PARAMS) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("scao_amd::qk_norm_rope", "")
                             .typed<decltype(op_qk_norm_rope)>();
  return op.call(ROPE_ARGS);
}
std::vector<Tensor> op_qk_norm_rope_backward(const Tensor& dq, const Tensor& dk, ROPE_PARAMS,
                                             int64_t wanted) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("scao_amd::qk_norm_rope_backward", "")
                             .typed<decltype(op_qk_norm_rope_backward)>();
  return op.call(dq, dk, ROPE_ARGS, wanted);
}

// q and k: batch x tokens x heads x columns
void check_rope(ROPE_PARAMS) {
  TORCH_CHECK(lib.rope_forward, "qk_norm_rope: scao_amd has not loaded its library");
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && q.sym_size(0) == k.sym_size(0) &&
                  q.sym_size(1) == k.sym_size(1) && q.sym_size(3) == k.sym_size(3),
              "qk_norm_rope: shape mismatch: q ", q.sym_sizes(), ", k ", k.sym_sizes());
  auto on = [&](const Tensor& t) { return t.layout() == at::kStrided && t.device() == q.device(); };
  TORCH_CHECK(on(q) && on(k) && code_of(q.scalar_type()) >= 0 && k.scalar_type() == q.scalar_type(),
              "qk_norm_rope takes q and k of one type of float32, bfloat16 and float16 on one device");
  for (const auto* w : {&wq, &wk})
    TORCH_CHECK(!*w || (on(**w) && code_of((*w)->scalar_type()) >= 0 && (*w)->dim() == 1 &&
                        (*w)->sym_size(0) == q.sym_size(3)),
                "qk_norm_rope: a weight is not a vector of a head's size on q's device");
  TORCH_CHECK(on(cos) && on(sin) && cos.scalar_type() == at::kFloat &&
                  sin.scalar_type() == at::kFloat && cos.dim() == 2 &&
                  cos.sym_sizes() == sin.sym_sizes() && cos.sym_size(1) * 2 <= q.sym_size(3),
              "qk_norm_rope: cos and sin must be float32 tables of at most half a head's columns "
              "on q's device");
  TORCH_CHECK(q.sym_size(3) >= 1 && q.sym_size(3) <= 512 && q.sym_size(2) >= 1 &&
                  k.sym_size(2) >= 1,
              "qk_norm_rope takes heads of 1 to 512 columns, one at least: q ", q.sym_sizes(),
              ", k ", k.sym_sizes());
  TORCH_CHECK(eps >= 0 && std::isfinite(eps), "qk_norm_rope: eps ", eps);
  TORCH_CHECK(positions || cos.sym_size(1) == 0 || q.sym_size(1) <= cos.sym_size(0),
              "qk_norm_rope: ", q.sym_size(1), " tokens and tables of ", cos.sym_size(0),
              " positions");
  TORCH_CHECK(!positions || (on(*positions) && positions->dim() == 2 &&
                             (positions->scalar_type() == at::kLong ||
                              positions->scalar_type() == at::kInt) &&
                             positions->sym_size(0) == q.sym_size(0) &&
                             positions->sym_size(1) == q.sym_size(1)),
              "qk_norm_rope: positions must be int64 or int32, one a token, on q's device");
}

void check_rope_gradients(const Tensor& dq, const Tensor& dk, const Tensor& q, const Tensor& k,
                          const std::optional<Tensor>& wq, const std::optional<Tensor>& wk,
                          int64_t wanted) {
  TORCH_CHECK(dq.sym_sizes() == q.sym_sizes() && dk.sym_sizes() == k.sym_sizes() &&
                  dq.scalar_type() == q.scalar_type() && dk.scalar_type() == k.scalar_type() &&
                  dq.device() == q.device() && dk.device() == q.device(),
              "qk_norm_rope_backward: the gradients are not like q and k");
  TORCH_CHECK((wq || !(wanted & 4)) && (wk || !(wanted & 8)),
              "qk_norm_rope_backward: no weight, no gradient");
}

Tensor unit_columns(const Tensor& t) {
  return t.stride(-1) == 1 || t.size(-1) <= 1 ? t : t.contiguous();
}
// Fresh memory for what the kernels write of t's shape: in t's order where the columns
// come out with unit stride, which is how they are written.  (Of a view whose tokens or
// sequences overlap, empty_like may put the columns outside of them.)
Tensor empty_columns(const Tensor& t) {
  const Tensor out = at::empty_like(t);
  return out.stride(-1) == 1 || out.size(-1) <= 1
             ? out
             : at::empty_like(t, t.options(), at::MemoryFormat::Contiguous);
}
scao_rope_tensor rope_tensor(const Tensor& t) {
  return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}
struct Rope {
  Tensor q, k, wq, wk, cos, sin, at;
  scao_rope_desc d{};
  Rope(const Tensor& q_, const Tensor& k_, const std::optional<Tensor>& wq_,
       const std::optional<Tensor>& wk_, const Tensor& cos_, const Tensor& sin_,
       const std::optional<Tensor>& positions, double eps, bool interleaved)
      : q(unit_columns(q_)), k(unit_columns(k_)) {
    // rows of one stride for both tables
    const bool same = cos_.stride(1) == 1 && sin_.stride(1) == 1 && cos_.stride(0) == sin_.stride(0) &&
                      cos_.stride(0) >= cos_.size(1);
    cos = same ? cos_ : cos_.contiguous();
    sin = same ? sin_ : sin_.contiguous();
    if (wq_) wq = wq_->contiguous();
    if (wk_) wk = wk_->contiguous();
    d.x[0] = rope_tensor(q);
    d.x[1] = rope_tensor(k);
    int i = 0;
    for (const Tensor* w : {&wq, &wk}) {
      if (w->defined()) {
        d.w[i] = w->data_ptr();
        d.w_dtype[i] = code_of(w->scalar_type());
      }
      ++i;
    }
    d.cos = (const float*)cos.data_ptr();
    d.sin = (const float*)sin.data_ptr();
    if (positions) {
      at = *positions;
      d.positions = at.data_ptr();
      d.wide_positions = at.scalar_type() == at::kLong;
      d.position_strides[0] = at.stride(0);
      d.position_strides[1] = at.stride(1);
    }
    d.batch = q.size(0);
    d.seq = q.size(1);
    d.table_rows = cos.size(0);
    d.ld_table = cos.stride(0);
    d.heads[0] = (int32_t)q.size(2);
    d.heads[1] = (int32_t)k.size(2);
    d.dim = (int32_t)q.size(3);
    d.rotary = (int32_t)cos.size(1) * 2;
    d.dtype = code_of(q.scalar_type());
    d.interleaved = interleaved;
    d.eps = (float)eps;
  }
};

std::tuple<Tensor, Tensor> qk_norm_rope_hip(ROPE_PARAMS) {
  check_rope(ROPE_ARGS);
  const c10::DeviceGuard guard(q.device());
  const Rope r(ROPE_ARGS);
  const Tensor yq = empty_columns(r.q), yk = empty_columns(r.k);
  const scao_rope_tensor y[2] = {rope_tensor(yq), rope_tensor(yk)};
  check(lib.rope_forward(&r.d, y, stream_of(q)), "scao_qk_rope_forward");
  return {yq, yk};
}

std::vector<Tensor> qk_norm_rope_backward_hip(const Tensor& dq_, const Tensor& dk_, ROPE_PARAMS,
                                              int64_t wanted) {
  check_rope(ROPE_ARGS);
  check_rope_gradients(dq_, dk_, q, k, wq, wk, wanted);
  const c10::DeviceGuard guard(q.device());
  const Rope r(ROPE_ARGS);
  const Tensor dq = unit_columns(dq_), dk = unit_columns(dk_);
  std::vector<Tensor> out;
  scao_rope_tensor dx[2] = {};
  void* dw[2] = {};
  for (int i = 0; i < 2; ++i)
    if (wanted >> i & 1) {
      out.push_back(empty_columns(i ? r.k : r.q));
      dx[i] = rope_tensor(out.back());
    }
  for (int i = 0; i < 2; ++i)
    if (wanted >> i & 4) {
      out.push_back(at::empty_like(i ? r.wk : r.wq));
      dw[i] = out.back().data_ptr();
    }
  const scao_rope_tensor dy[2] = {rope_tensor(dq), rope_tensor(dk)};
  const Tensor work = bytes(wanted & 12 ? lib.rope_backward_workspace(&r.d) : 0, q);
  check(lib.rope_backward(&r.d, dy, dx, dw[0], dw[1], work.data_ptr(), stream_of(q)),
        "scao_qk_rope_backward");
  return out;
}

std::tuple<Tensor, Tensor> qk_norm_rope_meta(ROPE_PARAMS) {
  check_rope(ROPE_ARGS);
  return {empty_columns(unit_columns(q)), empty_columns(unit_columns(k))};
}
std::vector<Tensor> qk_norm_rope_backward_meta(const Tensor& dq, const Tensor& dk, ROPE_PARAMS,
                                               int64_t wanted) {
  check_rope(ROPE_ARGS);
  check_rope_gradients(dq, dk, q, k, wq, wk, wanted);
  std::vector<Tensor> out;
  if (wanted & 1) out.push_back(empty_columns(unit_columns(q)));
  if (wanted & 2) out.push_back(empty_columns(unit_columns(k)));
  if (wanted & 4) out.push_back(at::empty_like(*wq));
  if (wanted & 8) out.push_back(at::empty_like(*wk));
  return out;
}

struct QkNormRope : torch::autograd::Function<QkNormRope> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k,
                               const std::optional<Tensor>& wq, const std::optional<Tensor>& wk,
                               const Tensor& cos, const Tensor& sin,
                               const std::optional<Tensor>& positions, double eps,
                               bool interleaved) {
    const at::AutoDispatchBelowADInplaceOrView below;
    auto [yq, yk] = op_qk_norm_rope(ROPE_ARGS);
    ctx->save_for_backward({q, k, wq.value_or(Tensor()), wk.value_or(Tensor()), cos, sin,
                            positions.value_or(Tensor())});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    return {yq, yk};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list t = ctx->get_saved_variables();
    variable_list out(9);
    auto given = [](const Tensor& x) { return x.defined() ? std::optional<Tensor>(x) : std::nullopt; };
    int64_t wanted = 0;
    for (int i = 0, edge = 0; i < 4; ++i)   // (a weight that is not given has no edge)
      if (t[i].defined()) wanted |= (int64_t)ctx->needs_input_grad(edge++) << i;
    variable_list have;
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      have = op_qk_norm_rope_backward(
          grads[0].defined() ? grads[0] : at::zeros_like(t[0]),
          grads[1].defined() ? grads[1] : at::zeros_like(t[1]), t[0], t[1], given(t[2]), given(t[3]),
          t[4], t[5], given(t[6]), ctx->saved_data["eps"].toDouble(),
          ctx->saved_data["interleaved"].toBool(), wanted);
    }
    if (at::GradMode::is_enabled()) {   // a gradient of these gradients is an error, not a zero
      const auto error = std::make_shared<torch::autograd::DelayedError>(
          "qk_norm_rope is differentiable once", (int64_t)have.size());
      for (Tensor& g : have) g.requires_grad_(true);
      have = (*error)(std::move(have));
    }
    for (int i = 0, n = 0; i < 4; ++i)
      if (wanted >> i & 1) out[i] = have[n++];
    return out;
  }
};

std::tuple<Tensor, Tensor> qk_norm_rope_autograd(ROPE_PARAMS) {
  check_rope(ROPE_ARGS);
  const Tensor none;
  const Tensor* inputs[6] = {&q, &k, wq ? &*wq : &none, wk ? &*wk : &none, &cos, &sin};
  bool wanted = false;
  for (int i = 0; i < 6; ++i) {
    if (!inputs[i]->defined()) continue;
    if (forward_mode())   // a tangent would be lost
      TORCH_CHECK_NOT_IMPLEMENTED(!inputs[i]->_fw_grad(0).defined(),
                                  "qk_norm_rope has no forward-mode derivative");
    if (!at::GradMode::is_enabled() || !inputs[i]->requires_grad()) continue;
    TORCH_CHECK_NOT_IMPLEMENTED(i < 4, "qk_norm_rope: cos and sin have no gradient");
    wanted = true;
  }
  if (wanted) {
    const variable_list y = QkNormRope::apply(unit_columns(q), unit_columns(k), wq, wk, cos, sin,
                                              positions, eps, interleaved);
    return {y[0], y[1]};
  }
  const at::AutoDispatchBelowADInplaceOrView below;
  return op_qk_norm_rope(ROPE_ARGS);
}

TORCH_LIBRARY_FRAGMENT(scao_amd, m) {
#define SCAO_ROPE                                                                       \
  "Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor cos, Tensor sin, "    \
  "Tensor? positions, float eps, bool interleaved"
  m.def("qk_norm_rope(" SCAO_ROPE ") -> (Tensor, Tensor)");
  m.def("qk_norm_rope_backward(Tensor dq, Tensor dk, " SCAO_ROPE ", int wanted) -> Tensor[]");
#undef SCAO_ROPE
}
TORCH_LIBRARY_IMPL(scao_amd, CUDA, m) {
  m.impl("qk_norm_rope", qk_norm_rope_hip);
  m.impl("qk_norm_rope_backward", qk_norm_rope_backward_hip);
}
TORCH_LIBRARY_IMPL(scao_amd, Meta, m) {
  m.impl("qk_norm_rope", qk_norm_rope_meta);
  m.impl("qk_norm_rope_backward", qk_norm_rope_backward_meta);
}
TORCH_LIBRARY_IMPL(scao_amd, Autograd, m) { m.impl("qk_norm_rope", qk_norm_rope_autograd); }

// qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved), tensors
// or None
PyObject* qk_norm_rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 9, "qk_norm_rope() takes nine arguments");
  std::optional<Tensor> t[7];
  for (int i = 0; i < 7; ++i) {
    if (args[i] == Py_None && (i == 2 || i == 3 || i == 6)) continue;
    TORCH_CHECK_TYPE(THPVariable_Check(args[i]), "qk_norm_rope() takes tensors");
    t[i] = THPVariable_Unpack(args[i]);
  }
  const double eps = PyFloat_AsDouble(args[7]);
  const int interleaved = PyObject_IsTrue(args[8]);
  if (PyErr_Occurred()) return nullptr;
  auto [yq, yk] = op_qk_norm_rope(*t[0], *t[1], t[2], t[3], *t[4], *t[5], t[6], eps, interleaved != 0);
  const THPObjectPtr a(THPVariable_Wrap(yq)), b(THPVariable_Wrap(yk));
  if (!a || !b) return nullptr;
  return PyTuple_Pack(2, a.get(), b.get());
  END_HANDLE_TH_ERRORS
}

// bind({name: address})
PyObject* bind(PyObject*, PyObject* arg) {
  auto at = [&](const char* name, auto& entry) {
    PyObject* v = PyDict_Check(arg) ? PyDict_GetItemString(arg, name) : nullptr;
    void* p = v ? PyLong_AsVoidPtr(v) : nullptr;
    if (!p && !PyErr_Occurred()) PyErr_Format(PyExc_KeyError, "bind() has no %s", name);
    entry = reinterpret_cast<std::decay_t<decltype(entry)>>(p);
    return p != nullptr;
  };
  if (!(at("scao_last_error", lib.last_error) && at("scao_ffn_saved_bytes", lib.saved_bytes) &&
        at("scao_ffn_forward_workspace", lib.forward_workspace) &&
        at("scao_ffn_forward", lib.forward) &&
        at("scao_ffn_backward_workspace", lib.backward_workspace) &&
        at("scao_ffn_backward", lib.backward) &&
        at("scao_grad_norm_workspace", lib.grad_norm_workspace) &&
        at("scao_grad_norm", lib.grad_norm) && at("scao_grad_clip", lib.grad_clip) &&
        at("scao_orthogonalize_workspace", lib.orthogonalize_workspace) &&
        at("scao_orthogonalize", lib.orthogonalize) &&
        at("scao_muon_workspace", lib.muon_workspace) && at("scao_muon_step", lib.muon_step) &&
        at("scao_qk_rope_forward", lib.rope_forward) &&
        at("scao_qk_rope_backward_workspace", lib.rope_backward_workspace) &&
        at("scao_qk_rope_backward", lib.rope_backward)))
    return nullptr;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
#define SCAO_FASTCALL(f) \
  {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
    SCAO_FASTCALL(gated_ffn),
    SCAO_FASTCALL(grad_norm),
    SCAO_FASTCALL(grad_clip),
    SCAO_FASTCALL(muon_step),
    SCAO_FASTCALL(qk_norm_rope),
#undef SCAO_FASTCALL
    {"bind", bind, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_host", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_host(void) { return PyModule_Create(&module); }

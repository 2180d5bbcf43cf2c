// blocks_autograd.cpp — the autograd side of lidarseg3d_amd/blocks.py: output allocation, saved tensors, forward and backward calls of the
// training-block operators (include/ls3d.h).  No arithmetic here; blocks.py checks the arguments and says what they mean.
//
// In Python this took most of a small call's time: a 68 x 96 dropout, forward and backward, 89 us on the host for two kernels of 3 us each.  What is left is
// torch's own engine (a backward pass on the GPU runs on a thread of its own: two wake-ups).
//
// The kernels are reached through addresses that _lib hands over (bind), so that the library a process works with stays _lib's choice.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include <torch/csrc/jit/frontend/tracer.h>

#include "../../../include/ls3d.h"

namespace {
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef c10::optional<Tensor> Optional;

struct {
  decltype(&ls3d_dropout_forward) dropout_forward;
  decltype(&ls3d_dropout_backward) dropout_backward;
  decltype(&ls3d_residual_norm_forward) norm_forward;
  decltype(&ls3d_residual_norm_workspace_bytes) norm_workspace;
  decltype(&ls3d_residual_norm_backward) norm_backward;
  decltype(&ls3d_embedding_forward) embedding_forward;
  decltype(&ls3d_embedding_workspace_bytes) embedding_workspace;
  decltype(&ls3d_embedding_backward) embedding_backward;
} api;

template <typename F>
void bind_one(F &f, const std::map<std::string, uint64_t> &a, const char *name) {
  const auto it = a.find(name);
  TORCH_CHECK(it != a.end() && it->second, name, " is missing");
  f = reinterpret_cast<F>(it->second);
}
void bind(const std::map<std::string, uint64_t> &a) {
  bind_one(api.dropout_forward, a, "ls3d_dropout_forward");
  bind_one(api.dropout_backward, a, "ls3d_dropout_backward");
  bind_one(api.norm_forward, a, "ls3d_residual_norm_forward");
  bind_one(api.norm_workspace, a, "ls3d_residual_norm_workspace_bytes");
  bind_one(api.norm_backward, a, "ls3d_residual_norm_backward");
  bind_one(api.embedding_forward, a, "ls3d_embedding_forward");
  bind_one(api.embedding_workspace, a, "ls3d_embedding_workspace_bytes");
  bind_one(api.embedding_backward, a, "ls3d_embedding_backward");
}

void check(int rc, const char *what) {
  TORCH_CHECK(rc == LS3D_OK, what, " failed: ",
              rc == LS3D_ERR_ARG ? "LS3D_ERR_ARG" : rc == LS3D_ERR_LAUNCH ? "LS3D_ERR_LAUNCH" : rc == LS3D_ERR_UNSUPPORTED ? "LS3D_ERR_UNSUPPORTED" : "LS3D_ERR_WORKSPACE");
}
void once(const char *what) { TORCH_CHECK(!at::GradMode::is_enabled(), what, " is differentiable once (backward with create_graph=True)"); }

int code(const Tensor &t) {
  const auto s = t.scalar_type();
  TORCH_CHECK(s == at::kFloat || s == at::kBFloat16 || s == at::kHalf, "float32, bfloat16 or float16 needed");
  return s == at::kFloat ? LS3D_DTYPE_F32 : s == at::kBFloat16 ? LS3D_DTYPE_BF16 : LS3D_DTYPE_F16;
}
// the values themselves: memory may hold them with the other sign (the imaginary part of a conjugate)
Tensor values(const Tensor &t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
// [..., c] as rows the kernels take: a view where the rows are contiguous, else a copy
Tensor rows(const Tensor &x) {
  const Tensor t = values(x);
  const int64_t c = t.size(-1);
  Tensor r = t.dim() == 2 ? t : t.reshape({c ? t.numel() / c : 0, c});
  if (r.is_contiguous()) return r;
  return (c > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < c) ? r.contiguous() : r;
}
long long ld(const Tensor &t) { return t.defined() ? (t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(t.size(1), 1)) : 0; }
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor fresh(const Tensor &like, at::IntArrayRef sizes) { return at::empty(sizes, like.options()); }
Tensor tensor(const Optional &t) { return t.has_value() ? *t : Tensor(); }
Optional maybe(const Tensor &t) { return t.defined() ? Optional(t) : c10::nullopt; }  // (a Function's absent inputs: they have no place among its edges)
void *stream(const Tensor &t) { return t.is_cuda() ? (void *)c10::hip::getCurrentHIPStream(t.device().index()).stream() : nullptr; }  // (the host emulation: none)
int count(int64_t n) {
  TORCH_CHECK(n >= 0 && n <= 0x7FFFFFFF, "more than 2^31 - 1 rows");
  return (int)n;
}
void same_device(const Tensor &ref, std::initializer_list<const Tensor *> others) {
  for (const Tensor *t : others) TORCH_CHECK(!t->defined() || t->device() == ref.device(), "tensors on different devices: ", ref.device(), " and ", t->device());
}

// A tracer sees the allocation of an output and not the kernel that fills it: what it records returns memory that nobody wrote
bool traced() {
  if (torch::jit::tracer::isTracing()) return true;
  typedef c10::impl::TorchDispatchModeTLS Modes;
  typedef c10::impl::TorchDispatchModeKey Key;
  return Modes::any_modes_set() && (Modes::get_mode(Key::PROXY).has_value() || Modes::get_mode(Key::FAKE).has_value() || Modes::get_mode(Key::FUNCTIONAL).has_value());
}
// fake tensors, the wrappers of vmap, grad and functionalization
bool in_memory(const Tensor &t) { return t.numel() == 0 || (t.has_storage() && t.storage().unsafeGetStorageImpl()->_mutable_data_ptr_no_checks().get()); }

// What would give wrong answers or be lost without a word, of a call's inputs and of the gradients that come into a backward pass: a tracer that records,
// tensors without memory of their own, tangents of forward-mode differentiation
void usable(const char *what, at::ArrayRef<Tensor> tensors) {
  TORCH_CHECK(!traced(), what, " cannot be traced (torch.jit.trace, make_fx, torch.export, fake tensors): a tracer does not see its kernels");
  for (const Tensor &t : tensors) {
    if (!t.defined()) continue;
    TORCH_CHECK(in_memory(t), what, " needs tensors in memory: fake tensors and the wrappers of torch.func (vmap, grad, jvp, functionalize) and batched gradients have none");
    TORCH_CHECK(!t._fw_grad(0).defined(), what, " has no forward-mode derivative (an input carries a tangent)");
  }
}

// ---------------------------------------------------------------------------------------------- dropout
Tensor dropout_raw(const Tensor &x, double p, const Tensor &state, int64_t call, bool relu, Tensor *bits) {
  same_device(x, {&state});
  const c10::DeviceGuard guard(x.device());
  const Tensor r = rows(x);
  Tensor y = fresh(x, x.sizes());
  if (bits) *bits = at::empty({r.size(0), (r.size(1) + 7) / 8}, x.options().dtype(at::kByte));
  check(api.dropout_forward(ptr(r), ld(r), r.size(0), r.size(1), code(x), (float)p, state.data_ptr<int64_t>(), (uint32_t)call, relu, ptr(y),
                            bits ? bits->data_ptr<uint8_t>() : nullptr, stream(x)), "ls3d_dropout_forward");
  return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, double p, const Tensor &state, int64_t call, bool relu) {
    Tensor bits;
    Tensor y = dropout_raw(x, p, state, call, relu, relu ? &bits : nullptr);
    ctx->save_for_backward({state, bits});
    ctx->saved_data["a"] = std::vector<double>{p, (double)call, (double)relu};
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    once("dropout");
    usable("dropout", grads);
    const auto saved = ctx->get_saved_variables();
    const auto a = ctx->saved_data["a"].toDoubleVector();
    const c10::DeviceGuard guard(grads[0].device());
    const Tensor g = rows(grads[0]);
    Tensor dx = fresh(g, grads[0].sizes());
    check(api.dropout_backward(ptr(g), ld(g), saved[1].defined() ? saved[1].data_ptr<uint8_t>() : nullptr, g.size(0), g.size(1), code(g), (float)a[0],
                               saved[0].data_ptr<int64_t>(), (uint32_t)a[1], a[2] != 0.0, ptr(dx), stream(g)), "ls3d_dropout_backward");
    return {dx, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor dropout(const Tensor &x, double p, const Tensor &state, int64_t call, bool relu) {
  usable("dropout", {x, state});
  if (at::GradMode::is_enabled() && x.requires_grad()) return Dropout::apply(x, p, state, call, relu);
  return dropout_raw(x, p, state, call, relu, nullptr);
}

// ---------------------------------------------------------------------------------------------- residual, dropout, gate and norms
struct NormForm {  // what residual_norm does, beside its tensors
  int64_t kind_in, kind_out, call;
  double eps_in, eps_out, alpha, p;
  bool want_sum;
  std::vector<double> pack() const { return {(double)kind_in, (double)kind_out, (double)call, eps_in, eps_out, alpha, p, (double)want_sum}; }
  static NormForm unpack(const std::vector<double> &v) {
    return {(int64_t)v[0], (int64_t)v[1], (int64_t)v[2], v[3], v[4], v[5], v[6], v[7] != 0.0};
  }
};

ls3d_norm_t norm_of(int64_t kind, const Tensor &w, const Tensor &b, double eps) {
  return ls3d_norm_t{ptr(w), ptr(b), (int32_t)kind, w.defined() ? code(w) : 0, b.defined() ? code(b) : 0, (float)eps};
}
ls3d_residual_norm_t descriptor(const NormForm &f, const Tensor &x, const Tensor &residual, const Tensor &gate, const Tensor &w_in, const Tensor &b_in, const Tensor &w_out,
                                const Tensor &b_out, const Tensor &state) {
  ls3d_residual_norm_t d = {};
  d.in = norm_of(f.kind_in, w_in, b_in, f.eps_in);
  d.out = norm_of(f.kind_out, w_out, b_out, f.eps_out);
  if (gate.defined()) {
    d.gate = ptr(gate);
    d.gate_kind = gate.dim() == 1 ? LS3D_GATE_CHANNEL : LS3D_GATE_FULL;
    d.gate_ld = gate.dim() == 1 ? 0 : ld(gate);
    d.gate_dtype = code(gate);
  }
  d.state = state.defined() ? state.data_ptr<int64_t>() : nullptr;
  d.dtype = code(x);
  d.stream_dtype = residual.defined() ? code(residual) : d.dtype;
  d.alpha = (float)f.alpha;
  d.p = (float)f.p;
  d.call = (uint32_t)f.call;
  return d;
}

// x, residual, gate: rows [n, c] (gate also [c]) -> y, s of the caller's shape, stats (undefined where not wanted)
std::array<Tensor, 3> norm_raw(const NormForm &f, at::IntArrayRef shape, const Tensor &x, const Tensor &residual, const Tensor &gate, const Tensor &w_in, const Tensor &b_in, const Tensor &w_out,
                               const Tensor &b_out, const Tensor &state, bool want_stats) {
  same_device(x, {&residual, &gate, &w_in, &b_in, &w_out, &b_out, &state});
  const c10::DeviceGuard guard(x.device());
  const ls3d_residual_norm_t d = descriptor(f, x, residual, gate, w_in, b_in, w_out, b_out, state);
  Tensor y, s, stats;
  if (f.kind_out) y = fresh(x, shape);
  if (f.want_sum || !f.kind_out) s = fresh(residual.defined() ? residual : x, shape);
  if (want_stats) stats = at::empty({x.size(0), 4}, x.options().dtype(at::kFloat));
  check(api.norm_forward(ptr(x), ld(x), ptr(residual), ld(residual), count(x.size(0)), count(x.size(1)), &d, ptr(y), ptr(s), stats.defined() ? stats.data_ptr<float>() : nullptr,
                         stream(x)), "ls3d_residual_norm_forward");
  return {y, s, stats};
}
variable_list norm_outputs(const NormForm &f, const std::array<Tensor, 3> &o) {
  if (f.kind_out && f.want_sum) return {o[0], o[1]};
  return {f.kind_out ? o[0] : o[1]};
}

Tensor gate_rows(const Tensor &g) { return g.defined() ? g.dim() == 1 ? values(g).contiguous() : rows(g) : Tensor(); }

// Takes the caller's tensors and makes rows of them inside: a gradient goes back as the one tensor that the kernel wrote.  Views of it, as a reshape before the
// Function would make, look like tensors of their own to the engine, which then keeps and adds to each as if no other shared its memory.
struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Optional &residual, const Optional &gate, const Optional &w_in, const Optional &b_in,
                               const Optional &w_out, const Optional &b_out, const Optional &state, const NormForm &f) {
    const Tensor t[] = {rows(x), residual ? rows(*residual) : Tensor(), gate_rows(tensor(gate)), values(tensor(w_in)), values(tensor(b_in)), values(tensor(w_out)), values(tensor(b_out)), tensor(state)};
    const auto o = norm_raw(f, x.sizes(), t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7], true);
    ctx->save_for_backward({t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7], o[2]});
    ctx->saved_data["f"] = f.pack();
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->set_materialize_grads(false);
    return norm_outputs(f, o);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    once("residual_norm");
    usable("residual_norm", grads);
    const NormForm f = NormForm::unpack(ctx->saved_data["f"].toDoubleVector());
    Tensor dy, ds;
    if (f.kind_out) {
      dy = grads[0];
      if (grads.size() > 1) ds = grads[1];
    } else ds = grads[0];
    variable_list out(9);
    if (!dy.defined() && !ds.defined()) return out;
    const auto v = ctx->get_saved_variables();
    const auto shape = ctx->saved_data["shape"].toIntVector();
    const Tensor &x = v[0], &residual = v[1], &gate = v[2];
    const c10::DeviceGuard guard(x.device());
    if (dy.defined()) dy = rows(dy);
    if (ds.defined()) ds = rows(ds);
    bool want[7];
    for (int i = 0, edge = 0; i < 7; ++i) want[i] = v[i].defined() && ctx->needs_input_grad(edge++);
    // s = residual + x: one gradient for both, written once
    const bool same = want[0] && want[1] && !gate.defined() && !f.kind_in && f.p == 0.0 && f.alpha == 1.0 && x.scalar_type() == residual.scalar_type();
    if (same) want[0] = false;
    for (int i = 0; i < 7; ++i)
      if (want[i]) out[i] = fresh(v[i], i < 2 || (i == 2 && gate.dim() > 1) ? at::IntArrayRef(shape) : v[i].sizes());
    const int n = count(x.size(0)), c = count(x.size(1));
    const size_t bytes = api.norm_workspace(n, c);
    Tensor ws;
    if (want[3] || want[4] || want[5] || want[6] || (want[2] && gate.dim() == 1)) ws = at::empty({(int64_t)std::max<size_t>(bytes, 256)}, x.options().dtype(at::kByte));
    const ls3d_residual_norm_t d = descriptor(f, x, residual, gate, v[3], v[4], v[5], v[6], v[7]);
    check(api.norm_backward(ptr(x), ld(x), ptr(residual), ld(residual), n, c, &d, v[8].data_ptr<float>(), ptr(dy), ld(dy), ptr(ds), ld(ds), ptr(out[0]), ptr(out[1]), ptr(out[2]),
                            ptr(out[3]), ptr(out[4]), ptr(out[5]), ptr(out[6]), ptr(ws), ws.defined() ? (size_t)ws.numel() : 0, stream(x)), "ls3d_residual_norm_backward");
    if (same) out[0] = out[1];
    return out;
  }
};

variable_list residual_norm(const Tensor &x, const Optional &residual, const Optional &gate, const Optional &w_in, const Optional &b_in, const Optional &w_out, const Optional &b_out,
                            const Optional &state, int64_t kind_in, double eps_in, int64_t kind_out, double eps_out, double alpha, double p, int64_t call, bool want_sum) {
  const NormForm f = {kind_in, kind_out, call, eps_in, eps_out, alpha, p, want_sum};
  const Tensor t[] = {x, tensor(residual), tensor(gate), tensor(w_in), tensor(b_in), tensor(w_out), tensor(b_out)};
  usable("residual_norm", t);
  usable("residual_norm", tensor(state));
  bool grad = false;
  for (const Tensor &u : t) grad = grad || (u.defined() && u.requires_grad());
  if (grad && at::GradMode::is_enabled()) return ResidualNorm::apply(x, maybe(t[1]), maybe(t[2]), maybe(t[3]), maybe(t[4]), maybe(t[5]), maybe(t[6]), state, f);
  return norm_outputs(f, norm_raw(f, x.sizes(), rows(x), t[1].defined() ? rows(t[1]) : Tensor(), gate_rows(t[2]), values(tensor(w_in)), values(tensor(b_in)), values(tensor(w_out)), values(tensor(b_out)), tensor(state), false));
}

// ---------------------------------------------------------------------------------------------- row lookup
Tensor embedding_raw(const Tensor &table, const Tensor &weight, const Tensor &idx, double scale) {
  same_device(table, {&weight, &idx});
  const c10::DeviceGuard guard(table.device());
  Tensor out = fresh(table, {idx.size(0), table.size(1)});
  check(api.embedding_forward(ptr(table), ld(table), table.size(0), count(table.size(1)), code(table), ptr(idx), idx.scalar_type() == at::kLong, count(idx.size(0)), count(idx.size(1)),
                              weight.defined() ? weight.data_ptr<float>() : nullptr, (float)scale, ptr(out), stream(table)), "ls3d_embedding_forward");
  return out;
}

struct Embedding : torch::autograd::Function<Embedding> {
  static Tensor forward(AutogradContext *ctx, const Tensor &table, const Optional &weight, const Tensor &idx, double scale, int64_t padding) {
    ctx->save_for_backward({table, tensor(weight), idx});
    ctx->saved_data["a"] = std::vector<double>{scale, (double)padding};
    return embedding_raw(table, tensor(weight), idx, scale);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    once("embedding");
    usable("embedding", grads);
    const auto v = ctx->get_saved_variables();
    const auto a = ctx->saved_data["a"].toDoubleVector();
    const Tensor &table = v[0], &weight = v[1], &idx = v[2];
    const c10::DeviceGuard guard(table.device());
    const Tensor g = rows(grads[0]);
    const int n = count(idx.size(0)), k = count(idx.size(1)), c = count(table.size(1));
    variable_list out(5);
    Tensor ws;
    if (ctx->needs_input_grad(0)) {
      out[0] = fresh(table, table.sizes());
      ws = at::empty({(int64_t)std::max<size_t>(api.embedding_workspace(n, k, c), 256)}, table.options().dtype(at::kByte));
    }
    if (weight.defined() && ctx->needs_input_grad(1)) out[1] = fresh(weight, weight.sizes());
    check(api.embedding_backward(ptr(table), ld(table), table.size(0), c, code(table), ptr(idx), idx.scalar_type() == at::kLong, n, k,
                                 weight.defined() ? weight.data_ptr<float>() : nullptr, (float)a[0], (long long)a[1], ptr(g), ld(g), ptr(out[0]),
                                 out[1].defined() ? out[1].data_ptr<float>() : nullptr, ptr(ws), ws.defined() ? (size_t)ws.numel() : 0, stream(table)),
          "ls3d_embedding_backward");
    return out;
  }
};

// idx [n, k], weight [n, k] or none -> [n, c]
Tensor embedding(const Tensor &table, const Optional &weight, const Tensor &idx, double scale, int64_t padding) {
  usable("embedding", {table, tensor(weight), idx});
  const Tensor t = rows(table), w = values(tensor(weight));
  if (at::GradMode::is_enabled() && (t.requires_grad() || (w.defined() && w.requires_grad()))) return Embedding::apply(t, maybe(w), idx, scale, padding);
  return embedding_raw(t, w, idx, scale);
}
}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("dropout", &dropout);
  m.def("residual_norm", &residual_norm);
  m.def("embedding", &embedding);
}

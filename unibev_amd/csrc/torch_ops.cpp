// Tensor-level entries of the dense-attention decoder operators: argument checks, workspaces and autograd nodes around the C ABI.
//
// One call of a small operator is host time: a Python autograd function takes ~30 us forward and, with the interpreter lock handed
// to the engine's thread, ~60 us backward, the node below 7 and 15.  The kernels are reached through the addresses of the loaded
// libunibev_hip.so (bind), so that this module follows whichever build of the library the process has loaded.
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>

#include "unibev_hip.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

#define UBV_ENTRIES(DO)                                                                                        \
  DO(ubv_last_error) DO(ubv_dropout) DO(ubv_layer_norm_forward) DO(ubv_layer_norm_backward_workspace)          \
  DO(ubv_layer_norm_backward) DO(ubv_diff_attention_forward_workspace) DO(ubv_diff_attention_forward)          \
  DO(ubv_diff_attention_backward_workspace) DO(ubv_diff_attention_backward)

struct {
#define DO(name) decltype(&::name) name = nullptr;
  UBV_ENTRIES(DO)
#undef DO
} api;

struct HipError : std::runtime_error { using std::runtime_error::runtime_error; };
PyObject* g_error = nullptr;      // UniBEVHipError
PyObject* g_hook = nullptr;       // called with the entry's name before every launch, or null

std::vector<std::string> entries() {
  std::vector<std::string> v;
#define DO(name) v.push_back(#name);
  UBV_ENTRIES(DO)
#undef DO
  return v;
}

void bind(const std::map<std::string, uintptr_t>& at, py::object error) {
#define DO(name) api.name = reinterpret_cast<decltype(&::name)>(at.at(#name));
  UBV_ENTRIES(DO)
#undef DO
  Py_XDECREF(g_error);
  g_error = error.release().ptr();
}

void set_hook(py::object fn) {
  Py_XDECREF(g_hook);
  g_hook = fn.is_none() ? nullptr : fn.release().ptr();
}

template <typename F, typename... A> void launch(const char* name, F f, A... a) {
  if (g_hook != nullptr) {
    py::gil_scoped_acquire gil;
    py::reinterpret_borrow<py::object>(g_hook)(name);
  }
  const int rc = f(a...);
  if (rc != 0) throw HipError(std::string(name + 4) + " failed (status " + std::to_string(rc) + "): " + api.ubv_last_error());
}

// The bodies run below autograd on the tensors' memory and hang their node on the result by hand: what else would follow an
// operation from its inputs to its result is refused (a forward-mode tangent or a trace would lose it without a word).
void plain(const char* who, std::initializer_list<const Tensor*> ts) {
  using Modes = c10::impl::TorchDispatchModeTLS;
  if (torch::jit::tracer::isTracing() || Modes::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value() ||
      Modes::get_mode(c10::impl::TorchDispatchModeKey::FAKE).has_value())
    throw std::runtime_error(std::string(who) + ": a trace cannot record this operator");
  const c10::DispatchKeySet wrapped = c10::python_ks | c10::DispatchKeySet({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                                                            c10::DispatchKey::Batched, c10::DispatchKey::Functionalize});
  for (const Tensor* t : ts) {
    if (!t->defined()) continue;
    if (t->layout() != at::kStrided || !t->has_storage() || t->key_set().has_any(wrapped))
      throw std::runtime_error(std::string(who) + ": takes ordinary tensors with memory (no sparse, batched or otherwise wrapped ones)");
    if (t->_fw_grad(/*level=*/0).defined()) throw std::runtime_error(std::string(who) + ": has no forward-mode derivative");
  }
}

// every given tensor on ONE GPU
c10::Device one_gpu(std::initializer_list<const Tensor*> ts) {
  std::optional<c10::Device> dev;
  for (const Tensor* t : ts) {
    if (!t->defined()) continue;
    if (!t->is_cuda()) throw std::runtime_error("unibev_amd ops run on the GPU only (got a CPU tensor); there is no CPU fallback");
    if (!dev) dev = t->device();
    else if (*dev != t->device())
      throw std::runtime_error("unibev_amd op: operands on different devices (" + dev->str() + " and " + t->device().str() + ")");
  }
  return *dev;
}

int type_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return UBV_F32;
    case at::kHalf: return UBV_F16;
    case at::kBFloat16: return UBV_BF16;
    default: throw py::type_error(std::string("unsupported dtype ") + c10::toString(t.scalar_type()) + "; expected float32, float16 or bfloat16");
  }
}

std::string shape(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

void* stream_of(const c10::Device& d) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(d.index()).stream(); }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
template <typename T = void> T* out_ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.mutable_data_ptr()) : nullptr; }
const float* f32_ptr(const Tensor& t) { return static_cast<const float*>(ptr(t)); }
Tensor f32(const Tensor& t) { return t.defined() ? t.to(at::kFloat).contiguous() : t; }
Tensor given(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
Tensor bytes(int64_t n, const Tensor& like) { return n > 0 ? at::empty({n}, like.options().dtype(at::kByte)) : Tensor(); }

// the gradients of a node that is differentiated once only (create_graph = True may ask for more and gets an error there)
variable_list once(const char* name, variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  auto err = std::make_shared<torch::autograd::DelayedError>(
      std::string("trying to differentiate twice a function that was marked with once_differentiable: ") + name, (int64_t)grads.size());
  return (*err)(std::move(grads));
}

template <typename N> std::shared_ptr<N> make_node(std::initializer_list<Tensor> inputs) {
  std::shared_ptr<N> n(new N(), torch::autograd::deleteNode);
  torch::autograd::edge_list edges;
  for (const Tensor& t : inputs) edges.push_back(t.defined() ? torch::autograd::impl::gradient_edge(t) : torch::autograd::Edge());
  n->set_next_edges(std::move(edges));
  return n;
}

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// ---- dropout --------------------------------------------------------------------------------------------------------------------
struct Drop {
  double p = 0.0;
  uint64_t seed = 0;
  Tensor base;
  const uint64_t* dev() const { return static_cast<const uint64_t*>(ptr(base)); }
};

Tensor dropout_raw(const Tensor& x, const Tensor& identity, at::ScalarType out_type, const Drop& d) {
  const c10::Device dev = x.device();
  c10::DeviceGuard guard(dev);
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor xc = x.contiguous(), ic = identity.defined() ? identity.contiguous() : identity;
  Tensor y = at::empty(x.sizes(), x.options().dtype(out_type));
  launch("ubv_dropout", api.ubv_dropout, ptr(xc), ptr(ic), out_ptr(y), xc.numel(), (float)d.p, d.seed, d.dev(), type_code(xc), type_code(y),
         stream_of(dev));
  return y;
}

struct DropoutBackward : Node {
  Drop drop;
  SavedVariable base_;              // (to notice that the base was changed: the mask is drawn again from it)
  at::ScalarType x_type;
  std::string name() const override { return "UbvDropoutBackward"; }
  variable_list apply(variable_list&& g) override {
    variable_list out(2);
    if (!g[0].defined()) return out;
    plain("dropout's gradient", {&g[0]});
    if (drop.base.defined()) base_.unpack();
    if (task_should_compute_output(0)) out[0] = dropout_raw(g[0], Tensor(), x_type, drop);
    if (task_should_compute_output(1)) out[1] = g[0];
    return once("dropout", std::move(out));
  }
};

Tensor dropout(const Tensor& x, double p, const OptTensor& identity_, uint64_t seed, const OptTensor& base) {
  const Tensor identity = given(identity_);
  Drop d{p, seed, given(base)};
  plain("dropout", {&x, &identity});
  one_gpu({&x, &identity, &d.base});
  type_code(x);
  if (identity.defined()) {
    if (!identity.sizes().equals(x.sizes()))
      throw py::value_error("dropout: identity " + shape(identity) + " must have the shape of x " + shape(x));
    if (identity.scalar_type() != x.scalar_type() && identity.scalar_type() != at::kFloat)
      throw py::type_error(std::string("dropout: identity of ") + c10::toString(identity.scalar_type()) + " beside x of " +
                           c10::toString(x.scalar_type()));
  }
  Tensor y = dropout_raw(x, identity, identity.defined() ? identity.scalar_type() : x.scalar_type(), d);
  if (wants_grad({&x, &identity})) {
    auto n = make_node<DropoutBackward>({x, identity});
    if (d.base.defined()) n->base_ = SavedVariable(d.base, false);
    n->drop = std::move(d);
    n->x_type = x.scalar_type();
    torch::autograd::set_history(y, n);
  }
  return y;
}

// ---- layer norm -----------------------------------------------------------------------------------------------------------------
struct LayerNormBackward : Node {
  SavedVariable x_, gamma_;
  Tensor stat;
  bool has_gamma = false;
  at::ScalarType gamma_type = at::kFloat, beta_type = at::kFloat;
  std::string name() const override { return "UbvLayerNormBackward"; }
  void release_variables() override {
    x_.reset_data();
    gamma_.reset_data();
    stat.reset();
  }
  variable_list apply(variable_list&& g) override {
    variable_list out(3);
    if (!g[0].defined()) return out;
    plain("layer_norm's gradient", {&g[0]});
    const Tensor x = x_.unpack(), gamma = has_gamma ? gamma_.unpack() : Tensor();
    const bool nx = task_should_compute_output(0), ng = task_should_compute_output(1), nb = task_should_compute_output(2);
    const int64_t C = x.size(-1), R = x.numel() / C;
    const c10::Device dev = x.device();
    c10::DeviceGuard guard(dev);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const auto fo = x.options().dtype(at::kFloat);
      Tensor gx, dg, db;
      if (nx) gx = at::empty_like(x);
      if (ng) dg = R > 0 ? at::empty({C}, fo) : at::zeros({C}, fo);
      if (nb) db = R > 0 ? at::empty({C}, fo) : at::zeros({C}, fo);
      if (R > 0 && (nx || ng || nb)) {
        const Tensor gy = g[0].contiguous();
        const int64_t nws = ng || nb ? api.ubv_layer_norm_backward_workspace(R, (int)C) : 0;
        const Tensor ws = bytes(nws, x);
        launch("ubv_layer_norm_backward", api.ubv_layer_norm_backward, ptr(gy), ptr(x), f32_ptr(gamma), f32_ptr(stat), f32_ptr(stat) + R,
               out_ptr(gx), out_ptr<float>(dg), out_ptr<float>(db), R, (int)C, type_code(x), out_ptr(ws), nws, stream_of(dev));
      }
      out[0] = gx;
      out[1] = ng ? dg.to(gamma_type) : dg;
      out[2] = nb ? db.to(beta_type) : db;
    }
    return once("layer_norm", std::move(out));
  }
};

Tensor layer_norm(const Tensor& x, const OptTensor& gamma_, const OptTensor& beta_, double eps) {
  const Tensor gamma = given(gamma_), beta = given(beta_);
  plain("layer_norm", {&x, &gamma, &beta});
  const c10::Device dev = one_gpu({&x, &gamma, &beta});
  const int dt = type_code(x);
  if (x.dim() < 1 || x.size(-1) < 1) throw py::value_error("layer_norm: x " + shape(x) + " has no last axis to normalise");
  const int64_t C = x.size(-1), R = x.numel() / C;
  if (C > (1 << 29)) throw py::value_error("layer_norm: rows of " + std::to_string(C) + " (at most 2^29)");
  if (!(eps >= 0.0)) throw py::value_error("layer_norm: eps " + std::to_string(eps) + " must not be negative");
  for (const Tensor* w : {&gamma, &beta}) {
    if (!w->defined()) continue;
    if (w->dim() != 1 || w->size(0) != C)
      throw py::value_error(std::string("layer_norm: ") + (w == &gamma ? "gamma " : "beta ") + shape(*w) + " must be (" + std::to_string(C) + ",)");
    type_code(*w);
  }
  const bool need = wants_grad({&x, &gamma, &beta});
  c10::DeviceGuard guard(dev);
  Tensor y, xc, g, stat;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    xc = x.contiguous();
    g = f32(gamma);
    const Tensor b = f32(beta);
    y = at::empty_like(xc);
    if (need) stat = at::empty({2, R}, x.options().dtype(at::kFloat));
    float* s = out_ptr<float>(stat);
    launch("ubv_layer_norm_forward", api.ubv_layer_norm_forward, ptr(xc), f32_ptr(g), f32_ptr(b), out_ptr(y), s, need ? s + R : nullptr, R,
           (int)C, (float)eps, dt, stream_of(dev));
  }
  if (need) {
    auto n = make_node<LayerNormBackward>({x, gamma, beta});
    n->x_ = SavedVariable(xc, false);
    n->has_gamma = gamma.defined();
    if (n->has_gamma) {
      n->gamma_ = SavedVariable(g, false);
      n->gamma_type = gamma.scalar_type();
    }
    if (beta.defined()) n->beta_type = beta.scalar_type();
    n->stat = stat;
    torch::autograd::set_history(y, n);
  }
  return y;
}

// ---- differential attention -----------------------------------------------------------------------------------------------------
struct Attn {
  int B, H, Hk, Nq, Nk, Dh, Dv;
  float scale;
  bool causal;
  Drop drop;
  Tensor padding, mask;             // padding (B, Nk) contiguous bool; mask expanded to (B, H, Nq, Nk), bool or f32
  int mask_kind() const { return !mask.defined() ? 0 : mask.scalar_type() == at::kBool ? 1 : 2; }
  bool empty() const { return B == 0 || H == 0 || Nq == 0 || Nk == 0; }
};

// t as the kernels take it — last axis contiguous and whole 16-byte pieces, every row 16-byte aligned, strides in reach — as it is
// where it already is so (views, expanded axes), else a copy (zero-padded last axis)
Tensor operand(const Tensor& t) {
  const int64_t size = t.element_size(), vec = 16 / size, D = t.size(-1);
  if (D % vec) {                                       // (constant_pad_nd would keep a channels-last order of t)
    auto sizes = t.sizes().vec();
    sizes.back() += vec - D % vec;
    Tensor p = at::zeros(sizes, t.options());
    p.narrow(-1, 0, D).copy_(t);
    return p;
  }
  bool fits = (t.stride(-1) == 1 || D == 1) && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) fits = fits && (t.size(i) <= 1 || t.stride(i) % vec == 0);
  fits = fits && (t.size(1) <= 1 || t.stride(1) * size < (1 << 24)) && (t.dim() < 5 || t.stride(3) * size < (1 << 28));
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

void strides(int64_t (&s)[18], const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& go, const Tensor& mask) {
  int at = 0;
  const std::pair<const Tensor*, int> order[] = {{&q, 4}, {&k, 4}, {&v, 3}, {&go, 3}, {&mask, 4}};
  for (const auto& [t, n] : order)
    for (int i = 0; i < n; ++i) s[at++] = t->defined() && t->size(i) > 1 ? t->stride(i) : 0;
}

struct DiffAttentionBackward : Node {
  SavedVariable q_, k_, v_, lam_, mask_, padding_, base_;      // the caller's masks and seed base: to notice that one was changed
  Attn a;
  Tensor stat, maps;
  at::ScalarType lam_type = at::kFloat;
  std::string name() const override { return "UbvDiffAttentionBackward"; }
  void release_variables() override {
    for (SavedVariable* s : {&q_, &k_, &v_, &lam_, &mask_, &padding_}) s->reset_data();
    stat.reset(); maps.reset();
    a.mask.reset(); a.padding.reset();
  }
  variable_list apply(variable_list&& g) override {
    variable_list out(4);
    if (!g[0].defined()) return out;
    plain("diff_attention's gradient", {&g[0]});
    const Tensor q = q_.unpack(), k = k_.unpack(), v = v_.unpack(), lam = lam_.unpack();
    if (a.mask.defined()) mask_.unpack();
    if (a.padding.defined()) padding_.unpack();
    if (a.drop.base.defined()) base_.unpack();
    const bool nq = task_should_compute_output(0), nk = task_should_compute_output(1), nv = task_should_compute_output(2),
               nl = task_should_compute_output(3);
    const c10::Device dev = q.device();
    c10::DeviceGuard guard(dev);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const auto o = q.options();
      auto make = [&](at::IntArrayRef s, const at::TensorOptions& opt) { return a.empty() ? at::zeros(s, opt) : at::empty(s, opt); };
      Tensor gq, gk, gv, gl;
      if (nq) gq = make({a.B, a.Nq, a.H, 2, a.Dh}, o);
      if (nk || nv) {
        gk = make({a.B, a.Nk, a.Hk, 2, a.Dh}, o);
        gv = make({a.B, a.Nk, a.Hk, a.Dv}, o);
      }
      if (nl) gl = make({a.H}, o.dtype(at::kFloat));
      if (!a.empty() && (nq || nk || nv || nl)) {
        const Tensor go = operand(g[0]);
        const int64_t nws = api.ubv_diff_attention_backward_workspace(a.B, a.H, a.Hk, a.Nq, a.Nk, a.Dh, a.Dv, (int)a.causal, type_code(q));
        const Tensor ws = bytes(nws, q);
        int64_t s[18];
        strides(s, q, k, v, go, a.mask);
        launch("ubv_diff_attention_backward", api.ubv_diff_attention_backward, ptr(go), ptr(q), ptr(k), ptr(v), f32_ptr(lam),
               static_cast<const uint8_t*>(ptr(a.padding)), ptr(a.mask), a.mask_kind(), f32_ptr(stat), f32_ptr(maps), out_ptr(gq),
               out_ptr(gk), out_ptr(gv), out_ptr<float>(gl), static_cast<const int64_t*>(s), a.B, a.H, a.Hk, a.Nq, a.Nk, a.Dh, a.Dv, a.scale,
               (int)a.causal, (float)a.drop.p, a.drop.seed, a.drop.dev(), type_code(q), out_ptr(ws), nws, stream_of(dev));
      }
      out[0] = gq;
      if (nk) out[1] = gk;
      if (nv) out[2] = gv;
      if (nl) out[3] = gl.to(lam_type);
    }
    return once("diff_attention", std::move(out));
  }
};

Tensor diff_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam_in, const OptTensor& attn_mask,
                      const OptTensor& key_padding_mask, bool causal, std::optional<double> scale, double p, uint64_t seed,
                      const OptTensor& base) {
  const Tensor mask_in = given(attn_mask), padding = given(key_padding_mask), seed_base = given(base);
  plain("diff_attention", {&q, &k, &v, &lam_in, &mask_in, &padding});
  const c10::Device dev = one_gpu({&q, &k, &v, &lam_in, &mask_in, &padding, &seed_base});
  const std::string who = "diff_attention: ";
  const std::string three = "q " + shape(q) + ", k " + shape(k) + ", v " + shape(v);
  if (q.dim() != 5 || k.dim() != 5 || v.dim() != 4 || q.size(3) != 2 || k.size(3) != 2)
    throw py::value_error(who + three + " must be (B, Nq, H, 2, Dh), (B, Nk, Hk, 2, Dh), (B, Nk, Hk, Dv)");
  const int64_t B = q.size(0), Nq = q.size(1), H = q.size(2), Dh = q.size(4), Nk = k.size(1), Hk = k.size(2), Dv = v.size(3);
  if (k.size(0) != B || k.size(4) != Dh || v.size(0) != B || v.size(1) != Nk || v.size(2) != Hk)
    throw py::value_error(who + three + " do not belong together");
  if (Hk < 1 || H % Hk != 0)
    throw py::value_error(who + std::to_string(H) + " query heads do not share " + std::to_string(Hk) + " key heads evenly");
  if (Dh < 1 || Dh > 128 || Dv < 1 || Dv > 256)
    throw py::value_error(who + "head widths " + std::to_string(Dh) + " and " + std::to_string(Dv) + " (at most 128 and 256)");
  const int64_t most = (int64_t(1) << 31) - 256;
  if (B * H > most || Nk > most || Nq * std::max<int64_t>(1, H / Hk) > most) throw py::value_error(who + three + " out of range");
  const int dt = type_code(q);
  if (q.scalar_type() != k.scalar_type() || q.scalar_type() != v.scalar_type())
    throw py::type_error(who + "q, k and v of " + c10::toString(q.scalar_type()) + ", " + c10::toString(k.scalar_type()) + " and " +
                         c10::toString(v.scalar_type()));
  if (!lam_in.is_floating_point() || (lam_in.numel() != 1 && !(lam_in.dim() == 1 && lam_in.size(0) == H)))
    throw py::value_error(who + "lam " + shape(lam_in) + " of " + c10::toString(lam_in.scalar_type()) + " must be (" + std::to_string(H) +
                          ",) or one value");
  const Tensor lam = lam_in.numel() == 1 && H != 1 ? lam_in.reshape({1}).expand({H}) : lam_in.dim() == 1 ? lam_in : lam_in.reshape({1});
  const double sc = scale.has_value() ? *scale : 1.0 / std::sqrt((double)Dh);
  if (!(sc >= 1e-30 && sc < 1e30)) throw py::value_error(who + "scale " + std::to_string(sc) + " must be in [1e-30, 1e30)");
  if (causal && Nq + Nk > most) throw py::value_error(who + three + " out of range");

  Attn a{(int)B, (int)H, (int)Hk, (int)Nq, (int)Nk, (int)Dh, (int)Dv, (float)sc, causal, Drop{p, seed, seed_base}, Tensor(), Tensor()};
  const bool need = wants_grad({&q, &k, &v, &lam});
  c10::DeviceGuard guard(dev);
  Tensor out, qc, kc, vc, lc, stat, maps;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    if (mask_in.defined()) {
      if (mask_in.requires_grad()) throw py::value_error(who + "attn_mask gets no gradient; detach it");
      if (mask_in.scalar_type() != at::kBool) type_code(mask_in);      // (f64's lowest value would become f32's -inf)
      Tensor m = mask_in.scalar_type() == at::kBool ? mask_in : mask_in.to(at::kFloat);
      if (m.dim() == 3 && m.size(0) == B * H && m.size(1) == Nq && m.size(2) == Nk) m = m.reshape({B, H, Nq, Nk});
      const int64_t full[4] = {B, H, Nq, Nk};
      bool fits = m.dim() == 2 || m.dim() == 4;
      for (int64_t i = 0; fits && i < m.dim(); ++i) fits = m.size(i) == 1 || m.size(i) == full[4 - m.dim() + i];
      if (!fits) throw py::value_error(who + "attn_mask " + shape(mask_in) + " does not broadcast to (B, H, Nq, Nk) of " + three);
      a.mask = m.expand({B, H, Nq, Nk});
    }
    if (padding.defined()) {
      if (padding.scalar_type() != at::kBool || padding.dim() != 2 || padding.size(0) != B || padding.size(1) != Nk)
        throw py::value_error(who + "key_padding_mask " + shape(padding) + " of " + c10::toString(padding.scalar_type()) + " must be bool (" +
                              std::to_string(B) + ", " + std::to_string(Nk) + ")");
      a.padding = padding.contiguous();
    }
    if (a.empty()) {                                   // no row, or nothing to see
      out = at::zeros({B, Nq, H, Dv}, q.options());
      qc = q; kc = k; vc = v; lc = lam;
    } else {
      qc = operand(q); kc = operand(k); vc = operand(v); lc = f32(lam);
      out = at::empty({B, Nq, H, Dv}, q.options());
      if (need) {
        stat = at::empty({B, H, Nq, 4}, q.options().dtype(at::kFloat));
        maps = at::empty({2, B, H, Nq, Dv}, q.options().dtype(at::kFloat));
      }
      const int64_t nws = api.ubv_diff_attention_forward_workspace(a.B, a.H, a.Hk, a.Nq, a.Nk, a.Dh, a.Dv, (int)causal, dt);
      const Tensor ws = bytes(nws, q);
      int64_t s[18];
      strides(s, qc, kc, vc, Tensor(), a.mask);
      launch("ubv_diff_attention_forward", api.ubv_diff_attention_forward, ptr(qc), ptr(kc), ptr(vc), f32_ptr(lc),
             static_cast<const uint8_t*>(ptr(a.padding)), ptr(a.mask), a.mask_kind(), out_ptr(out), out_ptr<float>(stat), out_ptr<float>(maps),
             static_cast<const int64_t*>(s), a.B, a.H, a.Hk, a.Nq, a.Nk, a.Dh, a.Dv, a.scale, (int)causal, (float)p, seed, a.drop.dev(), dt,
             out_ptr(ws), nws, stream_of(dev));
    }
  }
  if (need) {
    auto n = make_node<DiffAttentionBackward>({q, k, v, lam});
    n->q_ = SavedVariable(qc, false);
    n->k_ = SavedVariable(kc, false);
    n->v_ = SavedVariable(vc, false);
    n->lam_ = SavedVariable(lc, false);
    if (mask_in.defined()) n->mask_ = SavedVariable(mask_in, false);
    if (padding.defined()) n->padding_ = SavedVariable(padding, false);
    if (a.drop.base.defined()) n->base_ = SavedVariable(a.drop.base, false);
    n->lam_type = lam.scalar_type();
    n->a = std::move(a);
    n->stat = stat;
    n->maps = maps;
    torch::autograd::set_history(out, n);
  }
  return out;
}

}  // namespace

PYBIND11_MODULE(_native, m) {
  py::register_exception_translator([](std::exception_ptr e) {
    try {
      if (e) std::rethrow_exception(e);
    } catch (const HipError& err) {
      PyErr_SetString(g_error != nullptr ? g_error : PyExc_RuntimeError, err.what());
    }
  });
  m.def("entries", &entries);
  m.def("bind", &bind);
  m.def("set_hook", &set_hook);
  m.def("dropout", &dropout);
  m.def("layer_norm", &layer_norm);
  m.def("diff_attention", &diff_attention);
}

// Host side of cross_hip.py: the checks, descriptors and autograd nodes of the conditioned block's
// operators (mdg_attn_cross_*, mdg_rope_axes, mdg_gate_res_norm*), as a torch extension module.
// In Python a small call took 14-20 us of host time and a small training pass 100-130 us, most of
// it on the autograd engine's thread; the kernels of such calls take 3-10 us.
//
// The kernels stay behind the C ABI: bind() receives the addresses of the entry points that
// _lib.load() resolved, so this module links to nothing of libmdgen_hip.so.  Argument errors raise
// TypeError / ValueError before any launch, a failed call RuntimeError with the library's text.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <initializer_list>
#include <sstream>

#include "../../include/mdgen_hip.h"

namespace {

using torch::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using MaybeTensor = c10::optional<Tensor>;
namespace ag = torch::autograd;

struct Entry {
  size_t (*cross_ws)(const mdg_attn_cross*, int32_t);
  int (*cross_fwd)(const mdg_attn_cross*, void*, size_t, void*);
  int (*cross_bwd)(const mdg_attn_cross*, void*, size_t, void*);
  int (*rope)(const mdg_rope_axes_desc*, void*);
  int (*grn)(const mdg_gate_res_norm_desc*, void*);
  size_t (*grn_ws)(const mdg_gate_res_norm_desc*);
  int (*grn_bwd)(const mdg_gate_res_norm_desc*, void*, size_t, void*);
  const char* (*error)();
};
Entry lib = {};

template <typename F>
void set(F& f, uintptr_t address) { f = reinterpret_cast<F>(address); }

void bind(const std::vector<uintptr_t>& a) {
  if (a.size() != 8) throw py::value_error("bind: 8 entry points");
  set(lib.cross_ws, a[0]), set(lib.cross_fwd, a[1]), set(lib.cross_bwd, a[2]), set(lib.rope, a[3]);
  set(lib.grn, a[4]), set(lib.grn_ws, a[5]), set(lib.grn_bwd, a[6]), set(lib.error, a[7]);
}

// ------------------------------------------------------------------------------------------ helpers
struct Text {
  std::ostringstream s;
  template <typename T>
  Text& operator<<(const T& v) { s << v; return *this; }
  Text& operator<<(const Tensor& t) { s << t.scalar_type() << " " << t.sizes(); return *this; }
  operator std::string() const { return s.str(); }
};
[[noreturn]] void value_error(const Text& t) { throw py::value_error(t.s.str()); }
[[noreturn]] void type_error(const Text& t) { throw py::type_error(t.s.str()); }

void check_rc(int rc, const char* what) {
  if (rc != 0) throw std::runtime_error(Text() << what << " failed (code " << rc << "): " << lib.error());
}

bool known(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16; }
int code(at::ScalarType t) { return t == at::kBFloat16 ? MDG_BF16 : MDG_F32; }

// values as they lie in memory (a view such as z.conj().imag holds them negated)
Tensor plain(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }

// the tensor with its last dim contiguous (a copy only where it is not)
Tensor unit(const Tensor& t) { return plain(t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous()); }

mdg_heads heads(const Tensor& t) { return mdg_heads{t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)}; }

template <typename T = void>
T* address(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }

Tensor value(const MaybeTensor& t) { return t.has_value() ? *t : Tensor(); }

void check_device(const Tensor& t, std::initializer_list<const Tensor*> others) {
  if (!t.is_cuda()) {
    std::ostringstream s;
    s << "mdgen_finetune_amd.cross_hip runs on a ROCm device; got a tensor on " << t.device();
    throw std::runtime_error(s.str());
  }
  for (const Tensor* o : others)
    if (o->defined() && o->device() != t.device()) value_error(Text() << "tensors on " << t.device() << " and " << o->device());
}

void* current_stream(const at::Device& d) { return c10::hip::getCurrentHIPStream(d.index()).stream(); }

Tensor bytes(size_t n, const Tensor& like) {
  return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor();
}

// forward-mode tangents have no rule here and must not be dropped (no_grad leaves forward mode on)
void refuse_tangents(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(0).defined())
      throw std::runtime_error("mdgen_finetune_amd.cross_hip: no forward-mode derivative, detach the tangent first");
}

// A recording of torch operations holds the allocation of an output and not the call that fills it: what is traced
// (torch.jit.trace, make_fx) would return memory as it was found.  Fake tensors have no memory at all.
void refuse_tracing() {
  using Mode = c10::impl::TorchDispatchModeKey;
  if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::get_mode(Mode::PROXY).has_value() ||
      c10::impl::TorchDispatchModeTLS::get_mode(Mode::FAKE).has_value())
    throw std::runtime_error("mdgen_finetune_amd.cross_hip: its calls cannot be traced or run on fake tensors");
}

bool any_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

SavedVariable save(const Tensor& t) { return t.defined() ? SavedVariable(t, false) : SavedVariable(); }

// A node whose backward has no derivative of its own: gradients asked for with create_graph carry a node that
// raises when it is differentiated. That node leads to all that the gradients depend on (the node's inputs and
// the incoming gradients), so torch.autograd.grad with respect to any of them reaches it.
struct OnceNode : ag::Node {
  variable_list apply(variable_list&& grads) override {
    variable_list out;
    {
      at::AutoGradMode off(false);
      out = backward(grads);
    }
    if (!at::GradMode::is_enabled()) return out;
    ag::edge_list edges = next_edges();
    for (const Tensor& g : grads)
      if (g.defined() && g.requires_grad()) edges.push_back(ag::impl::gradient_edge(g));
    auto node = std::shared_ptr<ag::Error>(
        new ag::Error("trying to differentiate twice a function that was marked with @once_differentiable", std::move(edges)), ag::deleteNode);
    for (Tensor& g : out)
      if (g.defined()) {
        g = g.detach();
        ag::set_history(g, node);
      }
    return out;
  }
  virtual variable_list backward(const variable_list& grads) = 0;
};

// ------------------------------------------------------------------------------------------ cross attention
struct CrossArgs {
  Tensor q, k, v, mask, q_len, kv_len;
  double scale;
};

mdg_attn_cross cross_desc(const CrossArgs& c, const Tensor& o, const Tensor& side, int64_t low) {
  mdg_attn_cross d = {};
  const auto& q = c.q;
  d.dtype = code(q.scalar_type());
  d.B = (int)q.size(0), d.Nq = (int)q.size(1), d.Nk = (int)c.k.size(1), d.H = (int)q.size(2), d.Hk = (int)c.k.size(2);
  d.D = (int)q.size(3), d.scale = (float)c.scale;
  d.q = heads(q), d.k = heads(c.k), d.v = heads(c.v), d.o = heads(o);
  if (side.defined()) {  // lse [B, H, Nq] fp32, then (low >= 0) o's rounding residual, contiguous as o
    d.lse = static_cast<float*>(side.data_ptr());
    if (low >= 0)
      d.o_lo = mdg_heads{static_cast<char*>(side.data_ptr()) + low, q.size(1) * q.size(2) * q.size(3), q.size(2) * q.size(3), q.size(3)};
  }
  if (c.mask.defined()) {
    d.mask = c.mask.data_ptr(), d.mask_sb = c.mask.stride(0), d.mask_sn = c.mask.stride(1);
    d.mask_type = c.mask.scalar_type() == at::kFloat ? MDG_MASK_F32 : MDG_MASK_U8;
  }
  d.q_len = address<int32_t>(c.q_len), d.kv_len = address<int32_t>(c.kv_len);
  return d;
}

void cross_forward(const CrossArgs& c, const Tensor& o, const Tensor& side, int64_t low) {
  if (!o.numel()) return;
  const mdg_attn_cross d = cross_desc(c, o, side, low);
  const size_t n = lib.cross_ws(&d, 0);
  if (n == (size_t)-1) check_rc(1, "mdg_attn_cross_workspace_bytes");
  const Tensor ws = bytes(n, o);
  check_rc(lib.cross_fwd(&d, address(ws), n, current_stream(o.device())), "mdg_attn_cross_fwd");
}

struct CrossNode : OnceNode {
  SavedVariable q, k, v, o, side, mask, q_len, kv_len;  // (all of them, so that saved-tensor hooks see what is kept)
  int64_t low = -1;
  double scale = 1.0;
  std::string name() const override { return "CrossAttentionBackward"; }
  void release_variables() override {
    for (SavedVariable* s : {&q, &k, &v, &o, &side, &mask, &q_len, &kv_len}) s->reset_data();
  }
  variable_list backward(const variable_list& grads) override {
    variable_list out(3);
    if (!grads[0].defined()) return out;
    const CrossArgs c{unit(q.unpack()), unit(k.unpack()), unit(v.unpack()), mask.unpack(), q_len.unpack(), kv_len.unpack(), scale};
    const Tensor ou = unit(o.unpack(shared_from_this())), kept = side.unpack();
    const c10::DeviceGuard guard(c.q.device());
    const bool keys = should_compute_output(1) || should_compute_output(2);  // (a frozen encoder: dq alone)
    const Tensor dq = at::empty(c.q.sizes(), c.q.options());
    Tensor dk, dv;
    if (keys) dk = at::empty(c.k.sizes(), c.k.options()), dv = at::empty(c.v.sizes(), c.v.options());
    if (c.q.numel()) {
      const Tensor g = unit(grads[0]);
      mdg_attn_cross d = cross_desc(c, ou, kept, low);
      d.dout = heads(g), d.dq = heads(dq);
      if (keys) d.dk = heads(dk), d.dv = heads(dv);
      const size_t n = lib.cross_ws(&d, 1);
      if (n == (size_t)-1) check_rc(1, "mdg_attn_cross_workspace_bytes");
      const Tensor ws = bytes(n, dq);
      check_rc(lib.cross_bwd(&d, address(ws), n, current_stream(dq.device())), "mdg_attn_cross_bwd");
    } else if (keys) {
      dk.zero_(), dv.zero_();
    }
    if (should_compute_output(0)) out[0] = dq;
    if (should_compute_output(1)) out[1] = dk;
    if (should_compute_output(2)) out[2] = dv;
    return out;
  }
};

void check_len(const char* name, const Tensor& t, int64_t B) {
  if (t.defined() && (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != B || !t.is_contiguous()))
    value_error(Text() << "cross_attention: " << name << " must be a contiguous int32 [" << B << "], got " << t);
}

Tensor cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& mask_, const MaybeTensor& q_len_,
                       const MaybeTensor& kv_len_, c10::optional<double> scale_) {
  Tensor mask = value(mask_);
  const Tensor q_len = value(q_len_), kv_len = value(kv_len_);
  if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4)
    value_error(Text() << "cross_attention: q, k, v must be [B, N, heads, D], got " << q.sizes() << ", " << k.sizes() << ", " << v.sizes());
  if (!known(q.scalar_type()) || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
    type_error(Text() << "cross_attention: q, k, v must be fp32 or bf16 of one type, got " << q.scalar_type() << ", " << k.scalar_type()
                      << ", " << v.scalar_type());
  const int64_t B = q.size(0), H = q.size(2), D = q.size(3), Nk = k.size(1), Hk = k.size(2);
  if (k.sizes() != v.sizes() || k.size(0) != B || k.size(3) != D || Hk == 0 || H % Hk || D < 1 || D > 128 ||
      B > INT32_MAX || q.size(1) > INT32_MAX || Nk > INT32_MAX || H > INT32_MAX)
    value_error(Text() << "cross_attention: q " << q.sizes() << ", k " << k.sizes() << ", v " << v.sizes());
  refuse_tracing();
  refuse_tangents({&q, &k, &v});
  check_device(q, {&k, &v, &mask, &q_len, &kv_len});
  if (mask.defined()) {
    const auto t = mask.scalar_type();
    if ((t != at::kBool && t != at::kByte && t != at::kFloat) || mask.dim() != 2 || mask.size(1) != Nk || (mask.size(0) != 1 && mask.size(0) != B))
      value_error(Text() << "cross_attention: mask must be bool, uint8 or fp32 [" << B << " or 1, " << Nk << "], got " << mask);
    if (!Nk) mask = Tensor();  // (an encoder without states has nothing to mask, and an empty mask no address)
    else if (mask.size(0) != B) mask = mask.expand({B, Nk});
  }
  check_len("q_len", q_len, B), check_len("kv_len", kv_len, B);
  const double scale = scale_.has_value() ? *scale_ : 1.0 / std::sqrt((double)D);
  if (!(scale >= 1e-18 && scale <= 1e18)) value_error(Text() << "cross_attention: scale " << scale);

  const c10::DeviceGuard guard(q.device());
  const bool grad = any_grad({&q, &k, &v});
  std::shared_ptr<CrossNode> node;
  if (grad) {
    node = std::shared_ptr<CrossNode>(new CrossNode(), ag::deleteNode);
    node->set_next_edges(ag::collect_next_edges(q, k, v));
  }
  at::AutoGradMode off(false);
  const CrossArgs c{unit(q), unit(k), unit(v), mask, q_len, kv_len, scale};
  Tensor o = at::empty(q.sizes(), q.options());
  if (!grad) {
    cross_forward(c, o, Tensor(), -1);
    return o;
  }
  // what the backward reads beside o, one allocation
  const bool bf16 = q.scalar_type() == at::kBFloat16;
  const int64_t n = q.numel(), rows = (n / D + 3) / 4 * 16;
  const Tensor side = at::empty({rows + (bf16 ? 2 * n : 0) + 16}, q.options().dtype(at::kByte));
  node->low = bf16 ? rows : -1, node->scale = scale;
  cross_forward(c, o, side, node->low);
  node->side = save(side), node->q = save(c.q), node->k = save(c.k), node->v = save(c.v);
  node->mask = save(mask), node->q_len = save(q_len), node->kv_len = save(kv_len);
  ag::set_history(o, node);
  node->o = SavedVariable(o, true);
  return o;
}

// ------------------------------------------------------------------------------------------ rotary
struct RopePlan {
  Tensor turns, axis, cols;
  std::vector<int64_t> sections;
  int64_t pairs, npairs;
};

void rope_launch(const RopePlan& p, const Tensor& pos, const variable_list& x, const variable_list& y, bool inverse) {
  const Tensor& q = x[0];
  if (!q.size(0) || !q.size(1)) return;
  mdg_rope_axes_desc d = {};
  d.dtype = code(q.scalar_type()), d.pairs = (int)p.pairs, d.nseg = (int)x.size();
  d.B = (int)q.size(0), d.N = (int)q.size(1), d.D = (int)q.size(3), d.npairs = (int)p.npairs, d.naxes = (int)p.sections.size();
  d.pos_i64 = pos.scalar_type() == at::kLong, d.inverse = inverse;
  for (size_t i = 0; i < p.sections.size(); ++i) d.section[i] = (int)p.sections[i];
  d.pos = pos.data_ptr(), d.pos_sb = pos.size(0) == 1 ? 0 : pos.stride(0), d.pos_sn = pos.stride(1);
  d.turns = address<double>(p.turns), d.axis = address<int32_t>(p.axis), d.cols = address<int32_t>(p.cols);
  for (size_t i = 0; i < x.size(); ++i) d.H[i] = (int)x[i].size(2), d.x[i] = heads(x[i]), d.out[i] = heads(y[i]);
  check_rc(lib.rope(&d, current_stream(q.device())), "mdg_rope_axes");
}

variable_list rope_new(const RopePlan& p, const Tensor& pos, variable_list x, bool inverse) {
  variable_list y;
  for (Tensor& t : x) {
    t = unit(t);
    y.push_back(at::empty(t.sizes(), t.options()));
  }
  rope_launch(p, pos, x, y, inverse);
  return y;
}

struct RopeNode : OnceNode {
  RopePlan plan;
  SavedVariable pos;
  bool inverse = false;
  std::string name() const override { return "RopeAxesBackward"; }
  void release_variables() override { pos.reset_data(); }
  variable_list backward(const variable_list& grads) override {  // the transpose: the rotation by the negative angle
    variable_list some, out(grads.size());
    for (const Tensor& g : grads)
      if (g.defined()) some.push_back(g);
    if (some.empty()) return out;
    const c10::DeviceGuard guard(some[0].device());
    const variable_list r = rope_new(plan, unit(pos.unpack()), some, !inverse);
    for (size_t i = 0, j = 0; i < grads.size(); ++i)
      if (grads[i].defined()) out[i] = r[j++];
    return out;
  }
};

// Writing in place, each element must be one memory location.  Dims are told apart by their strides, each
// of which must span all that lies inside it (other layouts are taken to overlap).
struct Dim {
  int64_t stride, nx, ny;
};
using Dims = std::array<Dim, 4>;
bool nested(Dims& dims) {  // sorts them, strides descending
  std::sort(dims.begin(), dims.end(), [](const Dim& a, const Dim& b) { return a.stride > b.stride; });
  int64_t reach = 0;
  for (int i = 3; i >= 0; --i) {
    const int64_t n = std::max(dims[i].nx, dims[i].ny);
    if (n > 1 && dims[i].stride <= reach) return false;
    reach += (n - 1) * dims[i].stride;
  }
  return true;
}
// whether sum (i_x - i_y) stride = d for some indices
bool meets(const Dims& dims, int i, int64_t d) {
  if (i == 4) return d == 0;
  const int64_t s = dims[i].stride;
  if (s == 0) return meets(dims, i + 1, d);
  const int64_t f = d >= 0 ? d / s : -((-d + s - 1) / s);
  for (int64_t n : {f, f + 1})
    if (n < dims[i].nx && -n < dims[i].ny && meets(dims, i + 1, d - n * s)) return true;
  return false;
}
bool may_share(const Tensor& x, const Tensor& y) {
  if (!x.numel() || !y.numel()) return false;
  const int64_t e = x.element_size(), d = static_cast<char*>(y.data_ptr()) - static_cast<char*>(x.data_ptr());
  int64_t xend = e, yend = e;
  for (int i = 0; i < 4; ++i) xend += (x.size(i) - 1) * x.stride(i) * e, yend += (y.size(i) - 1) * y.stride(i) * e;
  if (d >= xend || -d >= yend) return false;
  Dims dims;
  for (int i = 0; i < 4; ++i) {
    if (x.size(i) > 1 && y.size(i) > 1 && x.stride(i) != y.stride(i)) return true;
    dims[i] = {x.size(i) > 1 ? x.stride(i) : y.size(i) > 1 ? y.stride(i) : 0, x.size(i), y.size(i)};
  }
  return d % e || !nested(dims) || meets(dims, 0, d / e);
}
bool apart(const Tensor& t) {
  Dims dims;
  for (int i = 0; i < 4; ++i) dims[i] = {t.size(i) > 1 ? t.stride(i) : 0, t.size(i), 1};
  return nested(dims);
}

py::object rope_axes(const RopePlan& plan, Tensor pos, const Tensor& q, const MaybeTensor& k_, bool inverse, bool inplace) {
  variable_list x = {q};
  if (k_.has_value()) x.push_back(*k_);
  for (const Tensor& t : x) {
    if (t.dim() != 4 || !known(t.scalar_type()) || t.scalar_type() != q.scalar_type())
      type_error(Text() << "rope_axes: tensors must be fp32 or bf16 [B, N, heads, D] of one type, got " << t);
    if (t.size(0) != q.size(0) || t.size(1) != q.size(1) || t.size(3) != q.size(3) || t.size(2) < 1 || t.size(2) > 1024)
      value_error(Text() << "rope_axes: q " << q.sizes() << ", k " << t.sizes());
  }
  const int64_t B = q.size(0), N = q.size(1), D = q.size(3), axes = (int64_t)plan.sections.size();
  if (2 * plan.npairs > D || D > 1024 || B > INT32_MAX || N > INT32_MAX) value_error(Text() << "rope_axes: " << plan.npairs << " pairs in q " << q.sizes());
  refuse_tracing();
  refuse_tangents({&x.front(), &x.back()});
  check_device(q, {&x.back(), &pos, &plan.turns});
  if (pos.scalar_type() != at::kInt && pos.scalar_type() != at::kLong)
    type_error(Text() << "rope_axes: pos must be int32 or int64, got " << pos.scalar_type());
  if (pos.dim() == 2) pos = pos.unsqueeze(0);
  if (pos.dim() != 3 || (pos.size(0) != 1 && pos.size(0) != B) || pos.size(1) != N || pos.size(2) != axes)
    value_error(Text() << "rope_axes: pos " << pos.sizes() << " for tokens [" << B << ", " << N << "] on " << axes << " axes");
  pos = unit(pos);
  const c10::DeviceGuard guard(q.device());
  const bool grad = any_grad({&x.front(), &x.back()});
  variable_list y;
  if (inplace) {
    if (grad) value_error(Text() << "rope_axes: inplace on a tensor that requires grad");
    for (const Tensor& t : x)
      if ((t.stride(3) != 1 && D != 1) || !apart(t))
        value_error(Text() << "rope_axes: inplace needs a contiguous head dim and no memory shared between tokens or heads");
    if (x.size() == 2 && may_share(x[0], x[1])) value_error(Text() << "rope_axes: inplace on q and k that share memory");
    rope_launch(plan, pos, x, x, inverse);
    for (const Tensor& t : x)
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    y = x;
  } else {
    std::shared_ptr<RopeNode> node;
    if (grad) {
      node = std::shared_ptr<RopeNode>(new RopeNode(), ag::deleteNode);
      node->set_next_edges(x.size() == 2 ? ag::collect_next_edges(x[0], x[1]) : ag::collect_next_edges(x[0]));
    }
    at::AutoGradMode off(false);
    y = rope_new(plan, pos, x, inverse);
    if (grad) {
      node->plan = plan, node->pos = save(pos), node->inverse = inverse;
      for (Tensor& t : y) ag::set_history(t, node);
    }
  }
  if (y.size() == 1) return py::cast(y[0]);
  return py::make_tuple(y[0], y[1]);
}

// ------------------------------------------------------------------------------------------ norms
enum { kH, kY, kGate, kShift, kScale, kPostW, kPostB, kPreW, kPreB, kIns };
bool pre_side(int i) { return i == kShift || i == kScale || i == kPreW || i == kPreB; }

struct GrnCfg {
  int32_t post, pre;
  int64_t R;
  double rs, eps;
  at::ScalarType xt;
};

// rows [M, C] with a contiguous last dim, and their stride
Tensor rows2d(const Tensor& t, int64_t C, int64_t& ld) {
  ld = C;
  if (!t.defined() || t.is_contiguous()) return t;
  Tensor r = t.reshape({-1, C});
  if ((r.stride(1) == 1 || C == 1) && (r.size(0) == 1 || r.stride(0) >= C)) {
    if (r.size(0) > 1) ld = r.stride(0);
    return r;
  }
  return r.contiguous();
}

// the inputs' part of the descriptor; ins is left holding the tensors that it points into
mdg_gate_res_norm_desc grn_desc(const GrnCfg& c, std::array<Tensor, kIns>& ins) {
  mdg_gate_res_norm_desc d = {};
  for (Tensor& t : ins)
    if (t.defined() && t.is_neg()) t = t.resolve_neg();
  const int64_t C = ins[kH].size(-1);
  d.res_dtype = code(ins[kH].scalar_type()), d.dtype = code(c.xt);
  d.M = (int)(ins[kH].numel() / C), d.C = (int)C, d.rows_per_mod = (int)c.R, d.post = c.post, d.pre = c.pre;
  d.resid_scale = (float)c.rs, d.eps = (float)c.eps;
  int64_t ld;
  ins[kH] = rows2d(ins[kH], C, ld), d.ldh = ld;
  ins[kY] = rows2d(ins[kY], C, ld), d.ldy = ld;
  // gate / shift / scale with one common row stride (copied where they differ)
  const Tensor* some = nullptr;
  bool same = true;
  for (int i : {kGate, kShift, kScale}) {
    const Tensor& t = ins[i];
    if (!t.defined()) continue;
    if (!some) some = &t;
    same = same && (t.stride(1) == 1 || C == 1) && t.stride(0) >= C && t.stride(0) == some->stride(0);
  }
  if (some) {
    if (!same)
      for (int i : {kGate, kShift, kScale})
        if (ins[i].defined()) ins[i] = ins[i].contiguous();
    d.mod_stride = same ? some->stride(0) : C;
  }
  d.h = address(ins[kH]), d.y = address(ins[kY]);
  d.gate = address<float>(ins[kGate]), d.shift = address<float>(ins[kShift]), d.scale = address<float>(ins[kScale]);
  d.post_w = address<float>(ins[kPostW]), d.post_b = address<float>(ins[kPostB]);
  d.pre_w = address<float>(ins[kPreW]), d.pre_b = address<float>(ins[kPreB]);
  return d;
}

struct GrnNode : OnceNode {
  GrnCfg cfg;
  std::array<SavedVariable, kIns> saved;
  std::vector<int64_t> shape;
  bool has_h = true;  // output 0 is h_out, then xn (else xn alone)
  std::string name() const override { return "GateResidualNormBackward"; }
  void release_variables() override {
    for (SavedVariable& s : saved) s.reset_data();
  }
  variable_list backward(const variable_list& grads) override {
    variable_list out(kIns);
    const Tensor gh = has_h ? grads[0] : Tensor(), gx = has_h ? (grads.size() > 1 ? grads[1] : Tensor()) : grads[0];
    if (!gh.defined() && !gx.defined()) return out;
    std::array<Tensor, kIns> ins;
    for (int i = 0; i < kIns; ++i) ins[i] = saved[i].unpack();
    const c10::DeviceGuard guard(ins[kH].device());
    const Tensor like = ins[kH];
    const bool rows = like.numel() > 0;
    mdg_gate_res_norm_desc d = grn_desc(cfg, ins);
    const Tensor dho = plain(gh.defined() ? gh.contiguous() : gh), dxn = plain(gx.defined() ? gx.contiguous() : gx);
    const auto f32 = like.options().dtype(at::kFloat);
    if (should_compute_output(kH)) out[kH] = at::empty(shape, like.options());
    if (should_compute_output(kY)) out[kY] = at::empty(shape, ins[kY].options());
    // the rows' gradients in one allocation, the weights' in another; the pre norm's are zero without dxn
    for (const auto& part : {std::pair<int, int>{kGate, kPostW}, std::pair<int, int>{kPostW, kIns}}) {
      std::vector<int> live;
      for (int i = part.first; i < part.second; ++i) {
        if (!should_compute_output(i)) continue;
        if (rows && !(pre_side(i) && !dxn.defined())) live.push_back(i);
        else out[i] = at::zeros(ins[i].sizes(), f32);
      }
      if (live.empty()) continue;
      std::vector<int64_t> size = ins[live[0]].sizes().vec();
      size.insert(size.begin(), (int64_t)live.size());
      const Tensor all = at::empty(size, f32);
      for (size_t j = 0; j < live.size(); ++j) out[live[j]] = live.size() == 1 ? all.view(ins[live[0]].sizes()) : all.select(0, (int64_t)j);
      float* at0 = static_cast<float*>(all.data_ptr());
      const int64_t n = ins[live[0]].numel();
      for (size_t j = 0; j < live.size(); ++j) {
        float* p = at0 + j * n;
        switch (live[j]) {
          case kGate: d.dgate = p; break;
          case kShift: d.dshift = p; break;
          case kScale: d.dscale = p; break;
          case kPostW: d.dpost_w = p; break;
          case kPostB: d.dpost_b = p; break;
          case kPreW: d.dpre_w = p; break;
          default: d.dpre_b = p; break;
        }
      }
    }
    if (!rows) return out;
    d.dh_out = address(dho), d.dxn = address(dxn), d.dh = address(out[kH]), d.dy = address(out[kY]);
    d.dmod_stride = like.size(-1);
    const size_t n = lib.grn_ws(&d);
    if (n == (size_t)-1) check_rc(1, "mdg_gate_res_norm_bwd_workspace_bytes");
    const Tensor ws = bytes(n, like);
    check_rc(lib.grn_bwd(&d, address(ws), n, current_stream(like.device())), "mdg_gate_res_norm_bwd");
    return out;
  }
};

int norm_code(const std::string& s) {
  return s == "none" ? MDG_NORM_NONE : s == "rms" ? MDG_NORM_RMS : s == "layer" ? MDG_NORM_LAYER : -1;
}

py::tuple gate_residual_norm(const Tensor& h, const MaybeTensor& y_, const MaybeTensor& gate_, const MaybeTensor& shift_,
                             const MaybeTensor& scale_, double rs, const std::string& post_, const std::string& pre_,
                             const MaybeTensor& post_w_, const MaybeTensor& post_b_, const MaybeTensor& pre_w_,
                             const MaybeTensor& pre_b_, double eps) {
  std::array<Tensor, kIns> ins = {h, value(y_), value(gate_), value(shift_), value(scale_), value(post_w_), value(post_b_), value(pre_w_), value(pre_b_)};
  const Tensor& y = ins[kY];
  if (h.dim() < 1 || !known(h.scalar_type())) type_error(Text() << "gate_residual_norm: h must be fp32 or bf16 [..., C], got " << h);
  const int64_t C = h.size(-1);
  if (C < 1 || C > 8192) value_error(Text() << "gate_residual_norm: C = " << C);
  GrnCfg cfg;
  cfg.post = norm_code(post_), cfg.pre = norm_code(pre_);
  if (cfg.post < 0 || cfg.pre < 0)
    value_error(Text() << "gate_residual_norm: post '" << post_ << "', pre '" << pre_ << "' (one of none, rms, layer)");
  if (!y.defined()) {
    if (cfg.post || ins[kGate].defined()) value_error(Text() << "gate_residual_norm: a post norm or gate without y");
    if (!cfg.pre) value_error(Text() << "gate_residual_norm: nothing to do without y and a pre norm");
  } else if (y.sizes() != h.sizes() || !known(y.scalar_type()) || (h.scalar_type() != at::kFloat && h.scalar_type() != y.scalar_type())) {
    type_error(Text() << "gate_residual_norm: h " << h << ", y " << y);
  }
  if (!cfg.post && (ins[kPostW].defined() || ins[kPostB].defined())) value_error(Text() << "gate_residual_norm: post weights without a post norm");
  if (!cfg.pre)
    for (int i = 0; i < kIns; ++i)
      if (pre_side(i) && ins[i].defined()) value_error(Text() << "gate_residual_norm: pre weights or modulation without a pre norm");
  refuse_tracing();
  refuse_tangents({&ins[0], &ins[1], &ins[2], &ins[3], &ins[4], &ins[5], &ins[6], &ins[7], &ins[8]});
  check_device(h, {&ins[1], &ins[2], &ins[3], &ins[4], &ins[5], &ins[6], &ins[7], &ins[8]});
  const int64_t M = h.numel() / C;
  int64_t G = 0;
  for (int i : {kGate, kShift, kScale}) {
    const Tensor& t = ins[i];
    if (!t.defined()) continue;
    if (t.scalar_type() != at::kFloat || t.dim() != 2 || t.size(1) != C || t.size(0) < 1 || (G && t.size(0) != G))
      value_error(Text() << "gate_residual_norm: gate, shift and scale must be fp32 [G, " << C << "], got " << t);
    G = t.size(0);
  }
  if (!G) G = 1;
  if (M % G || M > INT32_MAX || (M == 0 && G > 1 && h.size(0) != G)) value_error(Text() << "gate_residual_norm: " << M << " rows in " << G << " groups");
  for (int i = kPostW; i < kIns; ++i)
    if (ins[i].defined() && (ins[i].scalar_type() != at::kFloat || ins[i].dim() != 1 || ins[i].size(0) != C || !ins[i].is_contiguous()))
      value_error(Text() << "gate_residual_norm: weights must be contiguous fp32 [" << C << "], got " << ins[i]);
  if (!(eps >= 0 && std::isfinite(eps) && std::isfinite(rs))) value_error(Text() << "gate_residual_norm: eps " << eps << ", resid_scale " << rs);
  cfg.R = M / G ? M / G : 1, cfg.rs = rs, cfg.eps = eps, cfg.xt = y.defined() ? y.scalar_type() : h.scalar_type();

  const c10::DeviceGuard guard(h.device());
  const bool grad = any_grad({&ins[0], &ins[1], &ins[2], &ins[3], &ins[4], &ins[5], &ins[6], &ins[7], &ins[8]});
  std::shared_ptr<GrnNode> node;
  if (grad) {
    node = std::shared_ptr<GrnNode>(new GrnNode(), ag::deleteNode);
    node->set_next_edges(ag::collect_next_edges(ins[0], ins[1], ins[2], ins[3], ins[4], ins[5], ins[6], ins[7], ins[8]));
  }
  at::AutoGradMode off(false);
  const bool same = !y.defined() && rs == 1.0;  // the norm before a block: h itself goes on
  mdg_gate_res_norm_desc d = grn_desc(cfg, ins);
  Tensor ho = same ? Tensor() : at::empty(h.sizes(), h.options());
  Tensor xn = cfg.pre ? at::empty(h.sizes(), h.options().dtype(cfg.xt)) : Tensor();
  if (M) {
    d.h_out = address(ho), d.xn = address(xn);
    check_rc(lib.grn(&d, current_stream(h.device())), "mdg_gate_res_norm");
  }
  if (grad) {
    node->cfg = cfg, node->shape = h.sizes().vec(), node->has_h = !same;
    for (int i = 0; i < kIns; ++i) node->saved[i] = save(ins[i]);
    if (!same) ag::set_history(ho, node);
    if (xn.defined()) ag::set_history(xn, node);
  }
  return py::make_tuple(same ? h : ho, xn.defined() ? py::cast(xn) : py::none());
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  py::class_<RopePlan>(m, "RopePlan").def(py::init([](Tensor turns, Tensor axis, Tensor cols, std::vector<int64_t> sections, int64_t pairs) {
    int64_t n = 0;
    for (int64_t s : sections) n += s;
    return RopePlan{std::move(turns), std::move(axis), std::move(cols), std::move(sections), pairs, n};
  }));
  m.def("cross_attention", &cross_attention);
  m.def("rope_axes", &rope_axes);
  m.def("gate_residual_norm", &gate_residual_norm);
}

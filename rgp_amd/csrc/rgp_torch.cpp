// rgp_torch.cpp -- the sequence operators' torch side: argument checks, allocation, autograd nodes.  Python module rgp_amd._seq.
// A single step or a norm of a few rows runs for 2 to 4 us on the device; filling the argument structs from Python and a backward pass that
// re-enters the interpreter on the engine's thread cost several times that.  Everything here ends in the C entries of include/rgp_hip.h,
// whose addresses rgp_amd/seq_ops.py hands over (bind).  A call whose operands are not all as the entries take them returns None; seq_ops.py
// then names what is wrong with them, or copies what only has to be contiguous and calls again.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/SavedTensorHooks.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/Device.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <algorithm>
#include <array>
#include <memory>
#include <string>
#include <vector>

#include "../../include/rgp_hip.h"

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

namespace {

struct Entries {
#define ENTRY(name) decltype(&::name) name
  ENTRY(rgp_last_error);
  ENTRY(rgp_ssm_scan_states_bytes); ENTRY(rgp_ssm_scan_workspace); ENTRY(rgp_ssm_scan_forward); ENTRY(rgp_ssm_scan_backward); ENTRY(rgp_ssm_scan_step);
  ENTRY(rgp_ssm_conv_workspace); ENTRY(rgp_ssm_conv_forward); ENTRY(rgp_ssm_conv_backward); ENTRY(rgp_ssm_conv_step);
  ENTRY(rgp_rms_norm_workspace); ENTRY(rgp_rms_norm_forward); ENTRY(rgp_rms_norm_backward);
  ENTRY(rgp_grad_workspace); ENTRY(rgp_grad_sumsq); ENTRY(rgp_grad_clip);
#undef ENTRY
} lib;
PyObject* rgp_error = nullptr;                      // rgp_amd._lib.RgpError
PyObject *s_h, *s_device, *s_off, *s_n_seq, *s_rows, *s_max_len;

struct Failed { int code; std::string msg; };      // a status of the library

struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

// ---- what a call is made with ---------------------------------------------------------------------------------------------------------
PyObject* attr(PyObject* o, PyObject* name) {
  PyObject* r = PyObject_GetAttr(o, name);
  if (!r) throw python_error();
  return r;
}
int64_t attr_int(PyObject* o, PyObject* name) {
  PyObject* r = attr(o, name);
  const int64_t v = PyLong_AsLongLong(r);
  Py_DECREF(r);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

// Where a Handle's c_void_p holds the library's pointer; nullptr for None.
void* const* cell_of(PyObject* p) {
  if (p == Py_None) return nullptr;
  Py_buffer b;
  if (PyObject_GetBuffer(p, &b, PyBUF_SIMPLE) != 0) throw python_error();
  void* const* at = b.len == sizeof(void*) ? (void* const*)b.buf : nullptr;
  PyBuffer_Release(&b);
  return at;
}

// A Handle: the library's pointer, its device, and the Python object, which a graph keeps alive.
struct Handle {
  rgp_handle h = nullptr;                           // for the length of a call
  at::Device device = at::kCPU;
  PyObject* object;
  explicit Handle(PyObject* o) : object(o) {
    PyObject* d = attr(o, s_device);
    if (THPDevice_Check(d)) device = ((THPDevice*)d)->device;
    Py_DECREF(d);
    PyObject* p = attr(o, s_h);
    void* const* at = cell_of(p);
    if (at) h = (rgp_handle)*at;
    Py_DECREF(p);
  }
  void* stream() const { return c10::hip::getCurrentHIPStream(device.index()).stream(); }
  void check(rgp_status st) const {
    if (st != RGP_OK) throw Failed{(int)st, h ? lib.rgp_last_error(h) : "the handle is closed"};
  }
};
// What a graph, which may end on any thread, keeps of it.  close() clears the pointer in the c_void_p before it destroys the context, so a pass
// that comes later finds none there; the place itself lives as long as the c_void_p.
struct KeptHandle {
  at::Device device;
  std::shared_ptr<PyObject> owner;                  // the Handle and its c_void_p
  void* const* cell = nullptr;
  explicit KeptHandle(const Handle& from) : device(from.device) {
    PyObject* p = attr(from.object, s_h);
    PyObject* both = PyTuple_Pack(2, from.object, p);
    Py_DECREF(p);
    if (!both) throw python_error();
    owner = std::shared_ptr<PyObject>(both, [](PyObject* q) {
      if (!Py_IsInitialized()) return;
      const PyGILState_STATE s = PyGILState_Ensure();
      Py_DECREF(q);
      PyGILState_Release(s);
    });
    cell = cell_of(PyTuple_GET_ITEM(both, 1));
  }
  rgp_handle get() const {
    rgp_handle h = cell ? (rgp_handle)__atomic_load_n(cell, __ATOMIC_ACQUIRE) : nullptr;
    if (!h) throw std::runtime_error("librgp_hip: the handle of this graph is closed");
    return h;
  }
  void* stream() const { return c10::hip::getCurrentHIPStream(device.index()).stream(); }
};

int type_code(at::ScalarType t) {
  switch (t) {
    case at::kDouble: return RGP_F64;
    case at::kFloat: return RGP_F32;
    case at::kBFloat16: return RGP_BF16;
    case at::kHalf: return RGP_F16;
    default: return -1;
  }
}
at::ScalarType acc_of(at::ScalarType t) { return t == at::kDouble ? at::kDouble : at::kFloat; }

// While torch records a function (torch.jit.trace, make_fx), it would see the allocation of a result and nothing that fills it.
bool recording() {
  using Modes = c10::impl::TorchDispatchModeTLS;
  return c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::Tracer) || (Modes::any_modes_set() && Modes::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value());
}

// Forward-mode derivatives: a tensor may carry its tangent beside its values, and no result here would get one.
bool dual_level() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
thread_local bool duals = false;                    // a call made while there is a dual level
void seen(const Tensor& t) {
  if (duals && has_tangent(t)) throw Failed{RGP_ERR_BAD_ARG, "the sequence operators have no forward-mode derivatives: an operand carries a tangent"};
}
// None -> an undefined tensor; false: no tensor, or one whose memory does not hold its values (a view of a conjugate with the negation pending)
bool tensor(PyObject* o, Tensor& t, bool optional = false) {
  if (o == Py_None) return optional;
  if (!THPVariable_Check(o)) return false;
  t = THPVariable_Unpack(o);
  seen(t);
  return t.layout() == at::kStrided && !t.is_neg();
}
bool like(const Tensor& t, const Tensor& x) { return t.scalar_type() == x.scalar_type() && t.device() == x.device(); }
bool inner(const Tensor& t, int dims) {              // the last dims dimensions contiguous
  int64_t want = 1;
  for (int i = 1; i <= dims; ++i) {
    if (t.size(-i) != 1 && t.stride(-i) != want) return false;
    want *= t.size(-i);
  }
  return true;
}
Tensor rows_of(const Tensor& g) {                    // a gradient as the kernels read it
  const Tensor t = g.is_neg() ? g.resolve_neg() : g;
  return inner(t, 1) ? t : t.contiguous();
}
Tensor whole(const Tensor& t) { return t.defined() ? (t.is_neg() ? t.resolve_neg() : t).contiguous() : t; }
bool param(const Tensor& t, const Tensor& x, at::IntArrayRef shape) {
  return t.scalar_type() == acc_of(x.scalar_type()) && t.device() == x.device() && t.sizes() == shape && t.is_contiguous();
}
Tensor fresh(const Tensor& t) { return t.defined() ? at::empty(t.sizes(), t.options()) : Tensor(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor work_of(const Tensor& x, int64_t bytes, void*& work, int64_t& work_bytes) {
  if (bytes <= 0) return Tensor();
  Tensor w = at::empty({bytes}, x.options().dtype(at::kByte));
  work = w.data_ptr();
  work_bytes = bytes;
  return w;
}
void updated(const Tensor& t) {                      // a graph that saved the tensor notices the update
  if (!t.is_inference()) torch::autograd::impl::bump_version(t);
}
template <typename... Ts>
bool wants_grad(const Ts&... t) {
  return at::GradMode::is_enabled() && ((t.defined() && t.requires_grad()) || ...);
}

struct Geo {
  int n_seq = 0, dims = 0;                           // dims: leading dimensions of an activation
  int64_t T = 0, rows = 0, max_len = 0;
  Tensor off;
};
bool geometry(const Handle& h, const Tensor& x, PyObject* seqs, Geo& g) {
  if (!x.is_cuda() || x.device() != h.device || type_code(x.scalar_type()) < 0) return false;
  if (seqs == Py_None) {
    if (x.dim() != 3 || x.size(0) < 1 || x.size(1) < 1 || x.size(2) < 1 || x.size(1) > INT32_MAX) return false;
    g.dims = 2; g.T = g.max_len = x.size(0); g.n_seq = (int)x.size(1); g.rows = g.T * g.n_seq;
    return true;
  }
  if (x.dim() != 2 || x.size(1) < 1) return false;
  PyObject* off = attr(seqs, s_off);
  const bool ok = tensor(off, g.off);
  Py_DECREF(off);
  if (!ok || g.off.device() != x.device()) return false;
  g.dims = 1; g.n_seq = (int)attr_int(seqs, s_n_seq); g.rows = attr_int(seqs, s_rows); g.max_len = attr_int(seqs, s_max_len);
  return g.rows == x.size(0);
}
template <typename S>
void put_geo(S& a, const Geo& g, const Tensor& x, int reverse) {
  a.dtype = type_code(x.scalar_type());
  a.n_seq = g.n_seq; a.T = g.off.defined() ? 0 : g.T; a.rows = g.rows; a.max_len = g.max_len; a.reverse = reverse;
  a.off = (const int64_t*)ptr(g.off);
}
void put_stride(const Tensor& t, const Geo& g, int64_t& st, int64_t& sb) {
  st = t.defined() ? t.stride(0) : 0;
  sb = t.defined() && g.dims == 2 ? t.stride(1) : 0;
}

// A node of the graph: what both passes need besides the saved operands.
struct OpNode : torch::autograd::Node {
  KeptHandle handle;
  Geo geo;
  int reverse = 0;
  bool hooked;                                       // the user's hooks have what the node saves
  explicit OpNode(const Handle& h) : handle(h), hooked(at::SavedTensorDefaultHooks::get_hooks().has_value()) {}
  // What a backward pass has to refuse.  The engine hands a gradient on to the stream on which the node that takes it was made: during a capture
  // that must be the captured one.  A leaf that an eager graph still holds has its node on the eager stream, and an event from the capture to
  // there ends the capture, and the process with it.
  void begin(const variable_list& grads) const {
    if (at::GradMode::is_enabled()) throw std::runtime_error("the sequence operators have no second derivatives (create_graph=True)");
    if (recording()) throw std::runtime_error("the sequence operators cannot be recorded: leave their backward passes out of make_fx");
    if (dual_level())
      for (const Tensor& g : grads)
        if (has_tangent(g)) throw std::runtime_error("the sequence operators have no second derivatives: a gradient carries a forward-mode tangent");
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing((hipStream_t)handle.stream(), &capture) != hipSuccess || capture == hipStreamCaptureStatusNone) return;
    const c10::Stream here = c10::impl::VirtualGuardImpl(handle.device.type()).getStream(handle.device);
    for (const auto& e : next_edges()) {
      const auto there = e.function ? e.function->stream() : std::nullopt;
      if (there && *there != here)
        throw std::runtime_error("a captured backward pass cannot reach a leaf that a graph made outside the capture still holds: drop that graph first");
    }
  }
  // What a graph saved may come back through the user's hooks (torch.autograd.graph.saved_tensors_hooks): in another memory order, which the passes
  // lay out again, or as something else, which the kernels must not be given.  Asked only where there were hooks: the checks cost a small
  // backward pass 2 to 3 us.
  static void came_back(bool ok) {
    if (!ok) throw std::runtime_error("a saved operand of the sequence operators came back with another type, shape or device");
  }
  static void check(rgp_handle h, rgp_status st) {
    if (st != RGP_OK) throw std::runtime_error("librgp_hip status " + std::to_string((int)st) + ": " + lib.rgp_last_error(h));
  }
};
template <typename N>
std::shared_ptr<N> new_node(const Handle& h) { return std::shared_ptr<N>(new N(h), torch::autograd::deleteNode); }

// ---- convolution ------------------------------------------------------------------------------------------------------------------------
struct ConvOps { Tensor x, w, b; };
bool conv_ops(PyObject* const* o, ConvOps& c) {      // x, weight, bias
  return tensor(o[0], c.x) && tensor(o[1], c.w) && tensor(o[2], c.b, true);
}
bool conv_ok(const ConvOps& c) {
  const int64_t D = c.x.size(-1);
  return inner(c.x, 1) && c.w.dim() == 2 && c.w.size(1) >= 2 && c.w.size(1) <= 8 && param(c.w, c.x, {D, c.w.size(1)}) && (!c.b.defined() || param(c.b, c.x, {D})) && D <= INT32_MAX;
}
rgp_ssm_conv conv_args(const ConvOps& c, const Geo& g, int reverse) {
  rgp_ssm_conv a{};
  put_geo(a, g, c.x, reverse);
  a.D = (int)c.x.size(-1); a.W = (int)c.w.size(1);
  a.x = c.x.data_ptr(); a.w = c.w.data_ptr(); a.bias = ptr(c.b);
  put_stride(c.x, g, a.x_st, a.x_sb);
  return a;
}
struct ConvNode : OpNode {
  using OpNode::OpNode;
  SavedVariable x, w, b, init;
  std::string name() const override { return "SsmConvBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data(); w.reset_data(); b.reset_data(); init.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    begin(grads);
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(3);
    if (!grads[0].defined()) return out;
    ConvOps c{x.unpack(), w.unpack(), b.unpack()};
    Tensor before = init.unpack();
    const Tensor gv = rows_of(grads[0]);
    if (hooked) {
      c = ConvOps{rows_of(c.x), whole(c.w), whole(c.b)};
      before = whole(before);
      came_back(like(c.x, gv) && c.x.sizes() == gv.sizes() && conv_ok(c) &&
                (!before.defined() || (like(before, gv) && before.sizes() == at::IntArrayRef({geo.n_seq, c.w.size(1) - 1, c.x.size(-1)}))));
    }
    rgp_ssm_conv a = conv_args(c, geo, reverse);
    out[0] = fresh(c.x); out[1] = fresh(c.w); out[2] = fresh(c.b);
    a.init = ptr(before); a.gv = gv.data_ptr(); a.gx = out[0].data_ptr(); a.gw = out[1].data_ptr(); a.gbias = ptr(out[2]);
    put_stride(gv, geo, a.gv_st, a.gv_sb);
    const Tensor work = work_of(c.x, lib.rgp_ssm_conv_workspace(&a, 1), a.work, a.work_bytes);
    const rgp_handle h = handle.get();
    check(h, lib.rgp_ssm_conv_backward(h, handle.stream(), &a));
    return out;
  }
};

// (handle, x, weight, bias, seqs, init, reverse, return_state) -> (v, state or None)
PyObject* conv(PyObject* const* o) {
  Handle h(o[0]);
  ConvOps c;
  Geo g;
  Tensor init, last;
  if (!conv_ops(o + 1, c) || !tensor(o[5], init, true) || !geometry(h, c.x, o[4], g) || !conv_ok(c)) return nullptr;
  const int reverse = o[6] == Py_True, W = (int)c.w.size(1);
  if (init.defined() && (init.requires_grad() || !like(init, c.x) || init.sizes() != at::IntArrayRef({g.n_seq, W - 1, c.x.size(-1)}) || !init.is_contiguous())) return nullptr;
  Tensor v = fresh(c.x);
  if (o[7] == Py_True) last = at::empty({g.n_seq, W - 1, c.x.size(-1)}, c.x.options());
  rgp_ssm_conv a = conv_args(c, g, reverse);
  a.init = ptr(init); a.v = v.data_ptr(); a.last = ptr(last);
  {
    NoGil gil;
    h.check(lib.rgp_ssm_conv_forward(h.h, h.stream(), &a));
  }
  if (wants_grad(c.x, c.w, c.b)) {
    auto node = new_node<ConvNode>(h);
    node->set_next_edges(torch::autograd::collect_next_edges(c.x, c.w, c.b));
    node->geo = g; node->reverse = reverse;
    node->init = SavedVariable(init, false);
    node->x = SavedVariable(c.x, false); node->w = SavedVariable(c.w, false); node->b = SavedVariable(c.b, false);
    torch::autograd::set_history(v, node);
  }
  return Py_BuildValue("NN", THPVariable_Wrap(v), THPVariable_Wrap(last));
}
// (handle, x, weight, bias, state) -> v
PyObject* conv_step(PyObject* const* o) {
  Handle h(o[0]);
  ConvOps c;
  Tensor st;
  if (!conv_ops(o + 1, c) || !tensor(o[4], st) || !c.x.is_cuda() || c.x.device() != h.device || type_code(c.x.scalar_type()) < 0 || c.x.dim() != 2 ||
      c.x.numel() == 0 || c.x.size(0) > INT32_MAX || !conv_ok(c) || wants_grad(c.x, c.w, c.b))
    return nullptr;
  Geo g;
  g.T = g.max_len = 1; g.rows = c.x.size(0); g.n_seq = (int)g.rows;
  if (!like(st, c.x) || st.sizes() != at::IntArrayRef({g.rows, c.w.size(1) - 1, c.x.size(1)}) || !st.is_contiguous() || st.requires_grad()) return nullptr;
  Tensor v = fresh(c.x);
  rgp_ssm_conv a = conv_args(c, g, 0);
  a.x_st = 0; a.x_sb = c.x.stride(0);
  a.v = v.data_ptr(); a.last = st.data_ptr(); a.init = a.last;
  updated(st);
  {
    NoGil gil;
    h.check(lib.rgp_ssm_conv_step(h.h, h.stream(), &a));
  }
  return THPVariable_Wrap(v);
}

// ---- scan -------------------------------------------------------------------------------------------------------------------------------
struct ScanOps { Tensor u, delta, A, B, C, skip, z, bias; };
bool scan_ops(PyObject* const* o, ScanOps& s) {      // u, delta, A, B, C, D, z, delta_bias
  return tensor(o[0], s.u) && tensor(o[1], s.delta) && tensor(o[2], s.A) && tensor(o[3], s.B) && tensor(o[4], s.C) && tensor(o[5], s.skip, true) &&
         tensor(o[6], s.z, true) && tensor(o[7], s.bias, true);
}
bool scan_ok(const ScanOps& s, int dims, int& G) {   // dims: leading dimensions
  const Tensor& u = s.u;
  const int64_t n = u.size(-1);
  if (n > INT32_MAX || !inner(u, 1) || !like(s.delta, u) || s.delta.sizes() != u.sizes() || !inner(s.delta, 1)) return false;
  if (s.z.defined() && (!like(s.z, u) || s.z.sizes() != u.sizes() || !inner(s.z, 1))) return false;
  if (s.A.dim() != 2 || s.A.size(1) < 1 || s.A.size(1) > 64 || !param(s.A, u, {n, s.A.size(1)})) return false;
  if ((s.skip.defined() && !param(s.skip, u, {n})) || (s.bias.defined() && !param(s.bias, u, {n}))) return false;
  const int more = (int)s.B.dim() - dims;
  if (more < 1 || more > 2 || s.B.sizes() != s.C.sizes() || !like(s.B, u) || !like(s.C, u) || !inner(s.B, more) || !inner(s.C, more)) return false;
  for (int i = 0; i < dims; ++i)
    if (s.B.size(i) != u.size(i)) return false;
  G = more == 2 ? (int)s.B.size(-2) : 1;
  return s.B.size(-1) == s.A.size(1) && G >= 1 && n % G == 0;
}
rgp_ssm_scan scan_args(const ScanOps& s, const Geo& g, int G, int reverse) {
  rgp_ssm_scan a{};
  put_geo(a, g, s.u, reverse);
  a.D = (int)s.u.size(-1); a.N = (int)s.A.size(1); a.G = G;
  a.u = s.u.data_ptr(); a.delta = s.delta.data_ptr(); a.z = ptr(s.z); a.B = s.B.data_ptr(); a.C = s.C.data_ptr();
  put_stride(s.u, g, a.u_st, a.u_sb); put_stride(s.delta, g, a.delta_st, a.delta_sb); put_stride(s.z, g, a.z_st, a.z_sb);
  put_stride(s.B, g, a.B_st, a.B_sb); put_stride(s.C, g, a.C_st, a.C_sb);
  a.A = s.A.data_ptr(); a.skip = ptr(s.skip); a.bias = ptr(s.bias);
  return a;
}
struct ScanNode : OpNode {
  using OpNode::OpNode;
  SavedVariable u, delta, A, B, C, skip, z, bias;
  Tensor states;
  int G = 1;
  int64_t N = 0;
  std::string name() const override { return "SsmScanBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&u, &delta, &A, &B, &C, &skip, &z, &bias}) v->reset_data();
    states.reset();
  }
  variable_list apply(variable_list&& grads) override {
    begin(grads);
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(8);
    if (!grads[0].defined()) return out;
    ScanOps s{u.unpack(), delta.unpack(), A.unpack(), B.unpack(), C.unpack(), skip.unpack(), z.unpack(), bias.unpack()};
    const Tensor gy = rows_of(grads[0]);
    if (hooked) {
      s.u = rows_of(s.u); s.delta = rows_of(s.delta); s.z = s.z.defined() ? rows_of(s.z) : s.z;
      s.A = whole(s.A); s.skip = whole(s.skip); s.bias = whole(s.bias);
      for (Tensor* t : {&s.B, &s.C})
        if (t->is_neg() || t->dim() <= geo.dims || !inner(*t, (int)t->dim() - geo.dims)) *t = whole(*t);
      int groups = 0;
      came_back(like(s.u, gy) && s.u.sizes() == gy.sizes() && scan_ok(s, geo.dims, groups) && groups == G && s.A.size(1) == N);
    }
    rgp_ssm_scan a = scan_args(s, geo, G, reverse);
    const Tensor* in[8] = {&s.u, &s.delta, &s.A, &s.B, &s.C, &s.skip, &s.z, &s.bias};
    for (int i = 0; i < 8; ++i) out[i] = fresh(*in[i]);
    a.states = states.data_ptr(); a.gy = gy.data_ptr();
    a.gu = out[0].data_ptr(); a.gdelta = out[1].data_ptr(); a.gA = out[2].data_ptr(); a.gB = out[3].data_ptr(); a.gC = out[4].data_ptr();
    a.gskip = ptr(out[5]); a.gz = ptr(out[6]); a.gbias = ptr(out[7]);
    put_stride(gy, geo, a.gy_st, a.gy_sb);
    const Tensor work = work_of(s.u, lib.rgp_ssm_scan_workspace(&a, 1), a.work, a.work_bytes);
    const rgp_handle h = handle.get();
    check(h, lib.rgp_ssm_scan_backward(h, handle.stream(), &a));
    return out;
  }
};

// (handle, u, delta, A, B, C, D, z, delta_bias, seqs, init, reverse, return_state) -> (y, state or None)
PyObject* scan(PyObject* const* o) {
  Handle h(o[0]);
  ScanOps s;
  Geo g;
  Tensor init, last, states;
  int G = 1;
  if (!scan_ops(o + 1, s) || !tensor(o[10], init, true) || !geometry(h, s.u, o[9], g) || !scan_ok(s, g.dims, G)) return nullptr;
  const int reverse = o[11] == Py_True;
  const int64_t D = s.u.size(-1), N = s.A.size(1);
  if (init.defined() && (init.requires_grad() || !param(init, s.u, {g.n_seq, D, N}))) return nullptr;
  const bool train = wants_grad(s.u, s.delta, s.A, s.B, s.C, s.skip, s.z, s.bias);
  Tensor y = fresh(s.u);
  if (o[12] == Py_True) last = at::empty({g.n_seq, D, N}, s.A.options());
  rgp_ssm_scan a = scan_args(s, g, G, reverse);
  if (train) {
    const int64_t bytes = lib.rgp_ssm_scan_states_bytes(&a);
    states = at::empty({bytes > 0 ? bytes : 0}, s.u.options().dtype(at::kByte));
    a.states = states.data_ptr();
  }
  a.init = ptr(init); a.y = y.data_ptr(); a.last = ptr(last);
  const Tensor work = work_of(s.u, lib.rgp_ssm_scan_workspace(&a, 0), a.work, a.work_bytes);
  {
    NoGil gil;
    h.check(lib.rgp_ssm_scan_forward(h.h, h.stream(), &a));
  }
  if (train) {
    auto node = new_node<ScanNode>(h);
    node->set_next_edges(torch::autograd::collect_next_edges(s.u, s.delta, s.A, s.B, s.C, s.skip, s.z, s.bias));
    node->geo = g; node->reverse = reverse; node->G = G; node->N = N; node->states = states;
    node->u = SavedVariable(s.u, false); node->delta = SavedVariable(s.delta, false); node->A = SavedVariable(s.A, false);
    node->B = SavedVariable(s.B, false); node->C = SavedVariable(s.C, false); node->skip = SavedVariable(s.skip, false);
    node->z = SavedVariable(s.z, false); node->bias = SavedVariable(s.bias, false);
    torch::autograd::set_history(y, node);
  }
  return Py_BuildValue("NN", THPVariable_Wrap(y), THPVariable_Wrap(last));
}
// (handle, u, delta, A, B, C, D, z, delta_bias, state) -> y
PyObject* scan_step(PyObject* const* o) {
  Handle h(o[0]);
  ScanOps s;
  Tensor st;
  int G = 1;
  if (!scan_ops(o + 1, s) || !tensor(o[9], st) || !s.u.is_cuda() || s.u.device() != h.device || type_code(s.u.scalar_type()) < 0 || s.u.dim() != 2 ||
      s.u.numel() == 0 || s.u.size(0) > INT32_MAX || !scan_ok(s, 1, G) || wants_grad(s.u, s.delta, s.A, s.B, s.C, s.skip, s.z, s.bias))
    return nullptr;
  Geo g;
  g.dims = 1; g.T = g.max_len = 1; g.rows = s.u.size(0); g.n_seq = (int)g.rows;
  if (!param(st, s.u, {g.rows, s.u.size(1), s.A.size(1)}) || st.requires_grad()) return nullptr;
  Tensor y = fresh(s.u);
  rgp_ssm_scan a = scan_args(s, g, G, 0);
  for (auto p : {std::make_pair(&a.u_st, &a.u_sb), std::make_pair(&a.delta_st, &a.delta_sb), std::make_pair(&a.z_st, &a.z_sb), std::make_pair(&a.B_st, &a.B_sb),
                 std::make_pair(&a.C_st, &a.C_sb)}) {
    *p.second = *p.first;                            // the batch's rows are sequences of one step
    *p.first = 0;
  }
  a.y = y.data_ptr(); a.last = st.data_ptr(); a.init = a.last;
  updated(st);
  {
    NoGil gil;
    h.check(lib.rgp_ssm_scan_step(h.h, h.stream(), &a));
  }
  return THPVariable_Wrap(y);
}

// ---- norm -------------------------------------------------------------------------------------------------------------------------------
rgp_rms_norm rms_args(const Tensor& x, const Tensor& residual, const Tensor& w, double eps) {
  rgp_rms_norm a{};
  a.dtype = type_code(x.scalar_type());
  a.rows = x.size(0); a.C = x.size(1); a.eps = eps;
  a.x = x.data_ptr(); a.residual = ptr(residual); a.w = w.data_ptr();
  a.x_st = x.stride(0); a.residual_st = residual.defined() ? residual.stride(0) : 0;
  return a;
}
struct RmsNode : OpNode {
  using OpNode::OpNode;
  // 16-bit types: the backward pass adds x and residual again, hid's rounding would show in the weight's gradient; 32 and 64 bits: hid is that sum
  SavedVariable x, residual, w;
  Tensor rstd;
  double eps = 0.0;
  bool two = false, of_hid = false;
  std::string name() const override { return "RmsNormBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data(); residual.reset_data(); w.reset_data(); rstd.reset();
  }
  variable_list apply(variable_list&& grads) override {      // of y and, with a residual, of hid
    begin(grads);
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(3);                            // x, weight, residual
    const Tensor ghid = two ? grads[1] : Tensor();
    if (!grads[0].defined()) {                       // only the sum was used further on
      out[0] = out[2] = ghid;
      return out;
    }
    Tensor xs = x.unpack(of_hid ? shared_from_this() : nullptr), rs = residual.unpack(), ws = w.unpack();
    const Tensor gy = rows_of(grads[0]), gh = ghid.defined() ? rows_of(ghid) : ghid;
    if (hooked) {
      xs = rows_of(xs); rs = rs.defined() ? rows_of(rs) : rs; ws = whole(ws);
      came_back(like(xs, gy) && xs.sizes() == gy.sizes() && param(ws, gy, {gy.size(1)}) && (!rs.defined() || (like(rs, gy) && rs.sizes() == gy.sizes())));
    }
    rgp_rms_norm a = rms_args(xs, rs, ws, eps);
    out[0] = fresh(xs); out[1] = fresh(ws);
    if (two) out[2] = out[0];
    a.rstd = rstd.data_ptr(); a.gy = gy.data_ptr(); a.gy_st = gy.stride(0); a.ghid = ptr(gh); a.ghid_st = gh.defined() ? gh.stride(0) : 0;
    a.gx = out[0].data_ptr(); a.gw = out[1].data_ptr();
    const Tensor work = work_of(xs, lib.rgp_rms_norm_workspace(&a, 1), a.work, a.work_bytes);
    const rgp_handle h = handle.get();
    check(h, lib.rgp_rms_norm_backward(h, handle.stream(), &a));
    return out;
  }
};
// (handle, x, weight, residual, eps) -> (y, hid or None); x, residual (rows, C)
PyObject* rms(PyObject* const* o) {
  Handle h(o[0]);
  Tensor x, w, r, hid, rstd;
  const double eps = PyFloat_AsDouble(o[4]);
  if (eps == -1.0 && PyErr_Occurred()) throw python_error();
  if (!tensor(o[1], x) || !tensor(o[2], w) || !tensor(o[3], r, true) || !x.is_cuda() || x.device() != h.device || type_code(x.scalar_type()) < 0 ||
      x.dim() != 2 || x.size(1) < 1 || !inner(x, 1) || !param(w, x, {x.size(1)}) || !(eps > 0.0) || std::isinf(eps) ||
      (r.defined() && (!like(r, x) || r.sizes() != x.sizes() || !inner(r, 1))))
    return nullptr;
  const bool train = wants_grad(x, w, r);
  Tensor y = fresh(x);
  if (r.defined()) hid = fresh(x);
  if (train) rstd = at::empty({x.size(0)}, w.options());
  rgp_rms_norm a = rms_args(x, r, w, eps);
  a.y = y.data_ptr(); a.hid = ptr(hid); a.rstd = ptr(rstd);
  {
    NoGil gil;
    h.check(lib.rgp_rms_norm_forward(h.h, h.stream(), &a));
  }
  if (train) {
    auto node = new_node<RmsNode>(h);
    node->set_next_edges(torch::autograd::collect_next_edges(x, w, r));
    node->rstd = rstd; node->eps = eps; node->two = r.defined();
    torch::autograd::set_history(y, node);
    if (r.defined()) torch::autograd::set_history(hid, node);
    const bool again = r.defined() && x.element_size() == 2;
    node->of_hid = r.defined() && !again;
    node->x = SavedVariable(node->of_hid ? hid : x, node->of_hid);
    node->residual = SavedVariable(again ? r : Tensor(), false);
    node->w = SavedVariable(w, false);
  }
  return Py_BuildValue("NN", THPVariable_Wrap(y), THPVariable_Wrap(hid));
}

// ---- gradient norm ------------------------------------------------------------------------------------------------------------------------
struct Grads {
  std::vector<void*> p;
  std::vector<int64_t> n;
  std::vector<int32_t> dt;
};
bool grads_ok(const Handle& h, PyObject* list, Grads& g) {
  if (!PyList_Check(list)) return false;
  const Py_ssize_t n = PyList_GET_SIZE(list);
  std::vector<std::pair<char*, char*>> range(n);
  g.p.resize(n); g.n.resize(n); g.dt.resize(n);
  for (Py_ssize_t i = 0; i < n; ++i)
    if (THPVariable_Check(PyList_GET_ITEM(list, i))) seen(THPVariable_Unpack(PyList_GET_ITEM(list, i)));
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PyList_GET_ITEM(list, i);
    if (!THPVariable_Check(o)) return false;
    const Tensor& t = THPVariable_Unpack(o);
    const int code = type_code(t.scalar_type());
    if (code < 0 || !t.is_cuda() || t.device() != h.device || t.layout() != at::kStrided || t.is_neg() || !t.is_non_overlapping_and_dense()) return false;
    g.p[i] = t.data_ptr(); g.n[i] = t.numel(); g.dt[i] = code;
    range[i] = {(char*)g.p[i], (char*)g.p[i] + t.nbytes()};
  }
  std::sort(range.begin(), range.end());
  char* end = nullptr;
  for (const auto& r : range) {
    if (r.first < end && r.second > r.first) return false;       // two tensors share memory
    end = std::max(end, r.second);
  }
  return true;
}
Tensor scalars(const Handle& h, int64_t bytes) {      // one result and the places behind it
  return at::empty({1 + bytes / 8}, at::TensorOptions().dtype(at::kDouble).device(h.device));
}
// (handle, list of tensors) -> sum of squares
PyObject* sumsq(PyObject* const* o) {
  Handle h(o[0]);
  Grads g;
  if (!grads_ok(h, o[1], g) || !h.device.is_cuda()) return nullptr;
  const int n = (int)g.p.size();
  const int64_t bytes = lib.rgp_grad_workspace(n, g.n.data(), g.dt.data());
  Tensor buf = scalars(h, bytes);
  double* const p = buf.data_ptr<double>();
  {
    NoGil gil;
    h.check(lib.rgp_grad_sumsq(h.h, h.stream(), n, g.p.data(), g.n.data(), g.dt.data(), p, p + 1, bytes));
  }
  return THPVariable_Wrap(buf.select(0, 0));
}
// (handle, list of tensors, max_norm, sum of squares or None) -> norm
PyObject* clip(PyObject* const* o) {
  Handle h(o[0]);
  Grads g;
  Tensor sum;
  const double most = PyFloat_AsDouble(o[2]);
  if (most == -1.0 && PyErr_Occurred()) throw python_error();
  if (!(most > 0.0) || !tensor(o[3], sum, true) || !grads_ok(h, o[1], g) || !h.device.is_cuda()) return nullptr;
  if (sum.defined() && (sum.scalar_type() != at::kDouble || sum.numel() != 1 || sum.device() != h.device)) return nullptr;
  const int n = (int)g.p.size();
  const int64_t bytes = sum.defined() ? 0 : lib.rgp_grad_workspace(n, g.n.data(), g.dt.data());
  Tensor buf = scalars(h, bytes);
  double* const p = buf.data_ptr<double>();
  for (Py_ssize_t i = 0; i < n; ++i) updated(THPVariable_Unpack(PyList_GET_ITEM(o[1], i)));
  {
    NoGil gil;
    h.check(lib.rgp_grad_clip(h.h, h.stream(), n, g.p.data(), g.n.data(), g.dt.data(), (const double*)ptr(sum), most, p, bytes ? p + 1 : nullptr, bytes));
  }
  return THPVariable_Wrap(buf.select(0, 0));
}

// ---- module -------------------------------------------------------------------------------------------------------------------------------
// Calls f with exactly N arguments; a status of the library becomes an RgpError, "not as the entries take them" None.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments expected, %zd given", N, n);
    return nullptr;
  }
  try {
    if (recording()) throw Failed{RGP_ERR_BAD_ARG, "the sequence operators cannot be recorded: leave them out of torch.jit.trace and make_fx"};
    duals = dual_level();
    PyObject* r = F(args);
    if (r || PyErr_Occurred()) return r;
    Py_RETURN_NONE;
  } catch (const Failed& e) {
    PyObject* x = PyObject_CallFunction(rgp_error ? rgp_error : PyExc_RuntimeError, "is", e.code, e.msg.c_str());
    if (x) PyErr_SetObject((PyObject*)Py_TYPE(x), x);
    Py_XDECREF(x);
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// bind(error class, {entry: address})
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2 || !PyDict_Check(args[1])) {
    PyErr_SetString(PyExc_TypeError, "bind(error class, {entry: address})");
    return nullptr;
  }
  const std::pair<const char*, void**> want[] = {
#define ENTRY(name) {#name, (void**)&lib.name}
      ENTRY(rgp_last_error), ENTRY(rgp_ssm_scan_states_bytes), ENTRY(rgp_ssm_scan_workspace), ENTRY(rgp_ssm_scan_forward), ENTRY(rgp_ssm_scan_backward),
      ENTRY(rgp_ssm_scan_step), ENTRY(rgp_ssm_conv_workspace), ENTRY(rgp_ssm_conv_forward), ENTRY(rgp_ssm_conv_backward), ENTRY(rgp_ssm_conv_step),
      ENTRY(rgp_rms_norm_workspace), ENTRY(rgp_rms_norm_forward), ENTRY(rgp_rms_norm_backward), ENTRY(rgp_grad_workspace), ENTRY(rgp_grad_sumsq),
      ENTRY(rgp_grad_clip)
#undef ENTRY
  };
  for (const auto& w : want) {
    PyObject* v = PyDict_GetItemString(args[1], w.first);
    if (!v || !(*w.second = PyLong_AsVoidPtr(v))) {
      if (!PyErr_Occurred()) PyErr_Format(PyExc_KeyError, "%s", w.first);
      return nullptr;
    }
  }
  Py_INCREF(args[0]);
  Py_XSETREF(rgp_error, args[0]);
  Py_RETURN_NONE;
}

#define FAST(f) (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"bind", FAST(bind)},
                         {"conv", FAST((call<conv, 8>))},
                         {"conv_step", FAST((call<conv_step, 5>))},
                         {"scan", FAST((call<scan, 13>))},
                         {"scan_step", FAST((call<scan_step, 10>))},
                         {"rms", FAST((call<rms, 5>))},
                         {"sumsq", FAST((call<sumsq, 2>))},
                         {"clip", FAST((call<clip, 4>))},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_seq", "The sequence operators on torch tensors; use rgp_amd.seq_ops.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__seq() {
  const std::pair<PyObject**, const char*> names[] = {{&s_h, "h"}, {&s_device, "device"}, {&s_off, "off"}, {&s_n_seq, "n_seq"}, {&s_rows, "rows"},
                                                      {&s_max_len, "max_len"}};
  for (const auto& n : names)
    if (!(*n.first = PyUnicode_InternFromString(n.second))) return nullptr;
  return PyModule_Create(&module);
}

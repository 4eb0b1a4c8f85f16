// The token operators' calls from Python, for arguments that need nothing but the launch: tensors of the accepted types on
// a ROCm device, laid out as the kernels read them.  Everything else - copies, refusals and their messages - is left to
// the Python functions of reid_gan_amd.attention, which these return None to.  The kernels stay behind the C ABI; this
// file calls its entry points at the addresses that the Python binding found (reid_gan_amd._bind.connect).
//
// Why it is there: a layer norm of 16 rows takes 3 us on the GPU, its call from Python 10, and a forward and backward pass
// through a Python autograd node 50 to 115 (the engine runs the node on a thread of its own, where Python code costs the
// most).
#include <Python.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/torch.h>

#include "../../include/ried_gan.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct {
  decltype(&ried_last_error) last_error;
  decltype(&ried_layer_norm_fwd) layer_norm_fwd;
  decltype(&ried_layer_norm_bwd_scratch_floats) layer_norm_bwd_scratch_floats;
  decltype(&ried_layer_norm_bwd) layer_norm_bwd;
  decltype(&ried_rotary) rotary;
  decltype(&ried_xattn_fwd_scratch_floats) xattn_fwd_scratch_floats;
  decltype(&ried_xattn_fwd) xattn_fwd;
  decltype(&ried_xattn_bwd_scratch_floats) xattn_bwd_scratch_floats;
  decltype(&ried_xattn_bwd) xattn_bwd;
} abi;
bool connected = false;

int type_of(const Tensor& t) {                       // the C ABI's element types
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: return -1;
  }
}
ried_stream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
bool capturing(const Tensor& t) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  return hipStreamIsCapturing(stream_of(t), &status) == hipSuccess && status != hipStreamCaptureStatusNone;
}
void check(const char* what, int rc) { TORCH_CHECK(rc == 0, what, " failed (", rc, "): ", abi.last_error()); }
void not_captured(const char* what, const Tensor& t) {
  TORCH_CHECK(!capturing(t), what, ": gradients are not taken under graph capture; capture the forward and backward functions of reid_gan_amd.ops instead");
}
// Whether torch records the operations of this thread (jit.trace, make_fx): the recording would hold the allocation of a result
// and not the kernel that writes it.
bool traced() {
  return torch::jit::tracer::isTracing() ||
         c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value();
}
// A tensor with a forward-mode tangent: the kernels have no derivative in that direction, and a result without a tangent would
// stand for a derivative of zero.
bool dual(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
void one_way(const char* what, const Tensor& grad) {
  TORCH_CHECK(!dual(grad), what, ": there is no forward-mode derivative of its gradients, and the incoming one has a tangent");
}
const void* address(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
Tensor floats(const Tensor& like, at::IntArrayRef shape) { return at::empty(shape, like.options().dtype(at::kFloat)); }
Tensor fresh(const Tensor& like) { return at::empty(like.sizes(), like.options()); }

// Gradients have no second derivative: with create_graph they carry a node that says so.
variable_list once(variable_list out, const variable_list& grads) {
  if (!at::GradMode::is_enabled()) return out;
  bool any = false;
  for (const Tensor& g : grads) any |= g.defined() && g.requires_grad();
  if (!any) return out;
  for (Tensor& t : out)
    if (t.defined()) t = t.detach().set_requires_grad(true);
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable", static_cast<int64_t>(out.size()));
  return (*node)(std::move(out));
}

// ---------------------------------------------------------------------------------------------------------- layer norm
int parameter_type(const Tensor& w, const Tensor& b) { return w.defined() ? type_of(w) : b.defined() ? type_of(b) : 0; }

Tensor layer_norm(const Tensor& x, const Tensor& w, const Tensor& b, double eps, float* stats) {
  Tensor y = fresh(x);
  const int64_t C = x.size(-1), rows = x.numel() / C;
  check("ried_layer_norm_fwd", abi.layer_norm_fwd(address(x), C, address(w), address(b), y.mutable_data_ptr(), C, stats,
                                                  stats ? stats + rows : nullptr, rows, static_cast<int>(C),
                                                  static_cast<float>(eps), type_of(x), parameter_type(w, b), stream_of(x)));
  return y;
}

// (Only tensors that are there are inputs of a node: an absent weight or bias has no edge, and the edges of those behind it
// move up.)
struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    Tensor stats = floats(x, {2, x.numel() / x.size(-1)});
    Tensor y = layer_norm(x, w, b, eps, static_cast<float*>(stats.mutable_data_ptr()));
    ctx->save_for_backward({x, w, stats});
    ctx->saved_data["bias"] = b.defined() ? static_cast<int64_t>(b.scalar_type()) : -1;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
    c10::DeviceGuard guard(x.device());
    not_captured("layer_norm", x);
    one_way("layer_norm", grads[0]);
    Tensor dy = grads[0].contiguous();
    const int64_t C = x.size(-1), rows = x.numel() / C;
    Tensor dx = fresh(x), dw, db, scratch;
    const int64_t bias = ctx->saved_data["bias"].toInt();
    if (w.defined() && ctx->needs_input_grad(1)) dw = fresh(w);
    if (bias >= 0 && ctx->needs_input_grad(w.defined() ? 2 : 1)) db = at::empty({C}, x.options().dtype(static_cast<at::ScalarType>(bias)));
    float* work = nullptr;
    if (dw.defined() || db.defined()) {
      scratch = floats(x, {abi.layer_norm_bwd_scratch_floats(rows, static_cast<int>(C), type_of(x))});
      work = static_cast<float*>(scratch.mutable_data_ptr());
    }
    const float* mean = static_cast<const float*>(stats.const_data_ptr());
    check("ried_layer_norm_bwd",
          abi.layer_norm_bwd(address(dy), C, address(x), C, address(w), mean, mean + rows, dx.mutable_data_ptr(), C,
                             dw.defined() ? dw.mutable_data_ptr() : nullptr, db.defined() ? db.mutable_data_ptr() : nullptr, work, rows,
                             static_cast<int>(C), type_of(x), w.defined() ? type_of(w) : parameter_type(dw, db), stream_of(x)));
    if (!ctx->needs_input_grad(0)) dx = Tensor();
    return once({dx, dw, db, Tensor()}, grads);
  }
};

// ---------------------------------------------------------------------------------------------------- rotary positions
struct Turn { Tensor pos, freqs; int sections[4]; bool interleaved, inverse; };   // (no input of the node: nothing to differentiate)

Tensor turned(const Tensor& x, const Turn& t, bool inverse) {
  Tensor y = fresh(x);
  const Tensor &pos = t.pos, &freqs = t.freqs;
  const auto xs = x.strides(), ys = y.strides(), ps = pos.strides();
  const int ptype = pos.scalar_type() == at::kInt ? 0 : pos.scalar_type() == at::kLong ? 1 : 2;
  check("ried_rotary", abi.rotary(address(x), xs[0], xs[1], xs[2], y.mutable_data_ptr(), ys[0], ys[1], ys[2], address(pos), ptype,
                                  ps[0], ps[1], ps[2], static_cast<const double*>(freqs.const_data_ptr()), t.sections[0],
                                  t.sections[1], t.sections[2], t.sections[3], static_cast<int>(x.size(0)),
                                  static_cast<int>(x.size(1)), static_cast<int>(x.size(2)), static_cast<int>(x.size(3)),
                                  t.interleaved, inverse, type_of(x), stream_of(x)));
  return y;
}

struct Rotary : torch::autograd::Function<Rotary> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Turn& t) {
    ctx->save_for_backward({t.pos, t.freqs});
    ctx->saved_data["turn"] = std::vector<int64_t>{t.sections[0], t.sections[1], t.sections[2], t.sections[3], t.interleaved, t.inverse};
    return turned(x, t, t.inverse);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    c10::DeviceGuard guard(grads[0].device());
    not_captured("rotary", grads[0]);
    one_way("rotary", grads[0]);
    const std::vector<int64_t> v = ctx->saved_data["turn"].toIntVector();
    Turn t = {saved[0], saved[1]};
    for (int i = 0; i < 4; ++i) t.sections[i] = static_cast<int>(v[i]);
    t.interleaved = v[4];
    Tensor dy = grads[0].stride(-1) == 1 ? grads[0] : grads[0].contiguous();
    return once({turned(dy, t, !v[5]), Tensor()}, grads);
  }
};

// ----------------------------------------------------------------------------------------------------- cross attention
bool laid_out(const Tensor& t) {
  const auto s = t.strides();
  return s[3] == 1 && ((s[0] | s[1] | s[2]) & 7) == 0 && s[0] >= 0 && s[1] >= 0 && s[1] <= (1 << 23) && s[2] >= 0 &&
         (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0;
}
// The gradients' kernels reach the heads that share a key head (`share` of them) by 32-bit offsets in q and in dout.
bool far(const Tensor& t, int64_t share) { return (t.size(1) * t.stride(1) + share * t.stride(2)) * 2 >= (1ll << 31); }
void strides(long long (&to)[3], const Tensor& t) {
  for (int i = 0; i < 3; ++i) to[i] = t.stride(i);
}
ried_xattn_t attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& lse, const Tensor& lengths,
                       const Tensor& mask, double scale) {
  ried_xattn_t d = {};
  d.q = address(q); d.k = address(k); d.v = address(v); d.o = const_cast<void*>(address(o));
  d.lse = static_cast<float*>(const_cast<void*>(address(lse)));
  d.lengths = static_cast<const int*>(address(lengths));
  d.key_mask = static_cast<const unsigned char*>(address(mask));
  strides(d.q_stride, q); strides(d.k_stride, k); strides(d.v_stride, v); strides(d.o_stride, o);
  d.mask_stride = mask.defined() ? mask.stride(0) : 0;
  d.batch = q.size(0); d.queries = q.size(1); d.keys = k.size(1); d.heads = q.size(2); d.groups = k.size(2); d.dim = q.size(3);
  d.type = type_of(q);
  d.scale = scale;
  return d;
}

Tensor attend(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lse, const Tensor& lengths, const Tensor& mask, double scale) {
  Tensor o = fresh(q), scratch;
  ried_xattn_t d = attention(q, k, v, o, lse, lengths, mask, scale);
  const long long n = abi.xattn_fwd_scratch_floats(d.batch, d.queries, d.keys, static_cast<int>(d.heads), static_cast<int>(d.groups), static_cast<int>(d.dim));
  if (n) {
    scratch = floats(q, {n});
    d.scratch = static_cast<float*>(scratch.mutable_data_ptr());
  }
  check("ried_xattn_fwd", abi.xattn_fwd(&d, stream_of(q)));
  return o;
}

struct Keys { Tensor lengths, mask; };                               // (no inputs of the node)
struct Cross : torch::autograd::Function<Cross> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Keys& keys, double scale) {
    Tensor lse = floats(q, {q.size(0), q.size(2), q.size(1)});
    Tensor o = attend(q, k, v, lse, keys.lengths, keys.mask, scale);
    ctx->save_for_backward({q, k, v, o, lse, keys.lengths, keys.mask});
    ctx->saved_data["scale"] = scale;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &o = saved[3], &lse = saved[4];
    c10::DeviceGuard guard(q.device());
    not_captured("cross_attention", q);
    one_way("cross_attention", grads[0]);
    Tensor dq = fresh(q), dk = fresh(k), dv = fresh(v);
    if (q.size(1) == 0) {
      dk.zero_();
      dv.zero_();
    } else {
      const bool there = laid_out(grads[0]) && !far(grads[0], q.size(2) / k.size(2));
      Tensor dout = there ? grads[0] : grads[0].clone(at::MemoryFormat::Contiguous);
      ried_xattn_t d = attention(q, k, v, o, lse, saved[5], saved[6], ctx->saved_data["scale"].toDouble());
      d.dout = address(dout);
      d.dq = dq.mutable_data_ptr(); d.dk = dk.mutable_data_ptr(); d.dv = dv.mutable_data_ptr();
      strides(d.dout_stride, dout); strides(d.dq_stride, dq); strides(d.dk_stride, dk); strides(d.dv_stride, dv);
      Tensor scratch = floats(q, {abi.xattn_bwd_scratch_floats(d.batch, d.queries, d.keys, static_cast<int>(d.heads),
                                                               static_cast<int>(d.groups), static_cast<int>(d.dim))});
      d.scratch = static_cast<float*>(scratch.mutable_data_ptr());
      check("ried_xattn_bwd", abi.xattn_bwd(&d, stream_of(q)));
    }
    return once({dq, dk, dv, Tensor(), Tensor()}, grads);
  }
};

// ----------------------------------------------------------------------------------------------- called from Python
// Takes `o` when it is a plain tensor (no subclass) or, where `optional`, None.
bool take(PyObject* o, Tensor& t, bool optional = false) {
  if (optional && o == Py_None) return true;
  if (!THPVariable_CheckExact(o)) return false;
  t = THPVariable_Unpack(o);
  return t.layout() == at::kStrided && !t.is_neg();
}
bool number(PyObject* o, double& v) {
  if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return false;
  v = PyFloat_AsDouble(o);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}
// ready for a call: a ROCm tensor, outside a trace
bool ready(const Tensor& t) { return connected && t.is_cuda() && !traced(); }
bool wanted(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// layer_norm(x, weight, bias, eps)
PyObject* py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x, w, b;
  double eps;
  if (n != 4 || !take(a[0], x) || !take(a[1], w, true) || !take(a[2], b, true) || !number(a[3], eps) || !(eps >= 0)) Py_RETURN_NONE;
  if (!ready(x) || type_of(x) < 0 || x.dim() == 0 || x.size(-1) == 0 || x.size(-1) > (1 << 24) || !x.is_contiguous()) Py_RETURN_NONE;
  for (const Tensor* t : {&w, &b})
    if (t->defined() && (t->device() != x.device() || t->dim() != 1 || t->size(0) != x.size(-1) || !t->is_contiguous() ||
                         (t->scalar_type() != at::kFloat && t->scalar_type() != x.scalar_type())))
      Py_RETURN_NONE;
  if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type()) Py_RETURN_NONE;
  if (dual(x) || dual(w) || dual(b)) Py_RETURN_NONE;
  c10::DeviceGuard guard(x.device());
  if (!wanted({&x, &w, &b})) return THPVariable_Wrap(layer_norm(x, w, b, eps, nullptr));
  if (capturing(x)) Py_RETURN_NONE;
  const auto some = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
  return THPVariable_Wrap(LayerNorm::apply(x, some(w), some(b), eps));
  END_HANDLE_TH_ERRORS
}

// rotary(x, positions, freqs, sections, interleaved, inverse)
PyObject* py_rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x, pos, freqs;
  if (n != 6 || !take(a[0], x) || !take(a[1], pos) || !take(a[2], freqs) || !PyTuple_CheckExact(a[3])) Py_RETURN_NONE;
  Turn t = {};
  const Py_ssize_t axes = PyTuple_GET_SIZE(a[3]);
  int64_t pairs = 0;
  if (axes < 1 || axes > 4) Py_RETURN_NONE;
  for (Py_ssize_t i = 0; i < axes; ++i) {
    if (!PyLong_CheckExact(PyTuple_GET_ITEM(a[3], i))) Py_RETURN_NONE;
    int over = 0;
    const long v = PyLong_AsLongAndOverflow(PyTuple_GET_ITEM(a[3], i), &over);
    if (over || v < 0 || v > 65536) Py_RETURN_NONE;
    t.sections[i] = static_cast<int>(v);
    pairs += v;
  }
  for (int i = 4; i < 6; ++i)
    if (a[i] != Py_True && a[i] != Py_False) Py_RETURN_NONE;
  t.interleaved = a[4] == Py_True;
  t.inverse = a[5] == Py_True;
  if (!ready(x) || type_of(x) < 0 || x.dim() != 4 || x.stride(3) != 1 || pairs == 0 || 2 * pairs > x.size(3)) Py_RETURN_NONE;
  if (pos.device() != x.device() || pos.dim() != 3 || pos.size(0) != x.size(0) || pos.size(1) != x.size(1) || pos.size(2) != axes ||
      (pos.scalar_type() != at::kInt && pos.scalar_type() != at::kLong && pos.scalar_type() != at::kFloat))
    Py_RETURN_NONE;
  if (freqs.device() != x.device() || freqs.dim() != 1 || freqs.size(0) != pairs || freqs.scalar_type() != at::kDouble || !freqs.is_contiguous())
    Py_RETURN_NONE;
  for (int i = 0; i < 4; ++i)
    if (x.size(i) > 0x7fffffff) Py_RETURN_NONE;
  if (dual(x) || dual(pos) || dual(freqs) || wanted({&pos, &freqs})) Py_RETURN_NONE;   // (the tables have no gradient)
  t.pos = pos;
  t.freqs = freqs;
  c10::DeviceGuard guard(x.device());
  if (!wanted({&x})) return THPVariable_Wrap(turned(x, t, t.inverse));
  if (capturing(x)) Py_RETURN_NONE;
  return THPVariable_Wrap(Rotary::apply(x, t));
  END_HANDLE_TH_ERRORS
}

// cross_attention(q, k, v, lengths, key_mask, scale)
PyObject* py_cross_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor q, k, v, lengths, mask;
  double scale = 0;
  if (n != 6 || !take(a[0], q) || !take(a[1], k) || !take(a[2], v) || !take(a[3], lengths, true) || !take(a[4], mask, true)) Py_RETURN_NONE;
  if (a[5] != Py_None && !number(a[5], scale)) Py_RETURN_NONE;
  if (!ready(q) || type_of(q) < 1 || q.dim() != 4 || k.dim() != 4 || k.sizes() != v.sizes() || q.size(0) != k.size(0) || q.size(3) != k.size(3))
    Py_RETURN_NONE;
  const int64_t D = q.size(3);
  if (D % 8 || D < 8 || D > 128 || q.size(2) == 0 || k.size(2) == 0 || q.size(2) % k.size(2)) Py_RETURN_NONE;
  for (const Tensor* t : {&k, &v})
    if (t->device() != q.device() || t->scalar_type() != q.scalar_type()) Py_RETURN_NONE;
  if (!laid_out(q) || !laid_out(k) || !laid_out(v)) Py_RETURN_NONE;
  if (lengths.defined() && (lengths.device() != q.device() || lengths.scalar_type() != at::kInt || lengths.dim() != 1 ||
                            lengths.size(0) != q.size(0) || !lengths.is_contiguous()))
    Py_RETURN_NONE;
  if (mask.defined() && (mask.device() != q.device() || (mask.scalar_type() != at::kBool && mask.scalar_type() != at::kByte) ||
                         mask.dim() != 2 || mask.size(0) != q.size(0) || mask.size(1) != k.size(1) || mask.stride(0) < 0 ||
                         (mask.stride(1) != 1 && mask.size(1) > 1)))
    Py_RETURN_NONE;
  if (a[5] == Py_None) scale = 1.0 / std::sqrt(static_cast<double>(D));
  if (!(scale > 1e-37 && scale < 1e30)) Py_RETURN_NONE;
  if (dual(q) || dual(k) || dual(v)) Py_RETURN_NONE;
  c10::DeviceGuard guard(q.device());
  if (!wanted({&q, &k, &v})) return THPVariable_Wrap(attend(q, k, v, Tensor(), lengths, mask, scale));
  if (capturing(q) || far(q, q.size(2) / k.size(2))) Py_RETURN_NONE;
  return THPVariable_Wrap(Cross::apply(q, k, v, Keys{lengths, mask}, scale));
  END_HANDLE_TH_ERRORS
}

// dual(*tensors): whether one of the arguments is a tensor with a forward-mode tangent
PyObject* py_dual(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  for (Py_ssize_t i = 0; i < n; ++i)
    if (THPVariable_Check(a[i]) && dual(THPVariable_Unpack(a[i]))) Py_RETURN_TRUE;
  Py_RETURN_FALSE;
  END_HANDLE_TH_ERRORS
}

PyObject* py_traced(PyObject*, PyObject*) {
  HANDLE_TH_ERRORS
  if (traced()) Py_RETURN_TRUE;
  Py_RETURN_FALSE;
  END_HANDLE_TH_ERRORS
}

// A buffer of int64 (array.array('q')), released at the end of its scope
struct Words {
  Py_buffer view = {};
  bool ok = false;
  Words(PyObject* o, bool writable, Py_ssize_t n) {
    ok = PyObject_GetBuffer(o, &view, PyBUF_FORMAT | (writable ? PyBUF_WRITABLE : 0)) == 0;
    if (!ok) PyErr_Clear();
    else if (view.itemsize != 8 || view.len != n * 8) { PyBuffer_Release(&view); ok = false; }
  }
  ~Words() { if (ok) PyBuffer_Release(&view); }
  int64_t* data() { return static_cast<int64_t*>(view.buf); }
};

// gradients(params, addresses, sizes, out): out[i] = address of the i-th parameter's gradient (0: none).  False when a
// parameter does not lie at its address as it did, or a gradient is not a contiguous one of the parameter's type and size.
// Parameters with a gradient count as written (an earlier graph that saved one must not use it any more).
PyObject* py_gradients(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4 || !PyList_CheckExact(a[0])) Py_RETURN_FALSE;
  const Py_ssize_t many = PyList_GET_SIZE(a[0]);
  Words at(a[1], false, many), sizes(a[2], false, many), out(a[3], true, many);
  if (!at.ok || !sizes.ok || !out.ok) Py_RETURN_FALSE;
  for (Py_ssize_t i = 0; i < many; ++i) {
    PyObject* o = PyList_GET_ITEM(a[0], i);
    if (!THPVariable_Check(o)) Py_RETURN_FALSE;
    const Tensor& p = THPVariable_Unpack(o);
    if (reinterpret_cast<int64_t>(p.const_data_ptr()) != at.data()[i] || p.numel() != sizes.data()[i] || !p.is_contiguous() || p.is_neg())
      Py_RETURN_FALSE;
    const Tensor& g = p.grad();
    if (!g.defined()) {
      out.data()[i] = 0;
      continue;
    }
    if (g.layout() != at::kStrided || g.scalar_type() != p.scalar_type() || g.numel() != sizes.data()[i] || g.device() != p.device() ||
        !g.is_contiguous() || g.is_neg())
      Py_RETURN_FALSE;
    out.data()[i] = reinterpret_cast<int64_t>(g.const_data_ptr());
  }
  for (Py_ssize_t i = 0; i < many; ++i)
    if (out.data()[i]) torch::autograd::impl::bump_version(THPVariable_Unpack(PyList_GET_ITEM(a[0], i)));
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// connect({name: address}): the entry points of libried_gan.so
PyObject* py_connect(PyObject*, PyObject* table) {
  HANDLE_TH_ERRORS
  auto find = [&](const char* name, auto& fn) {
    PyObject* o = PyDict_Check(table) ? PyDict_GetItemString(table, name) : nullptr;
    TORCH_CHECK(o && PyLong_Check(o), "connect: no address of ", name);
    fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(PyLong_AsUnsignedLongLong(o));
  };
  find("ried_last_error", abi.last_error);
  find("ried_layer_norm_fwd", abi.layer_norm_fwd);
  find("ried_layer_norm_bwd_scratch_floats", abi.layer_norm_bwd_scratch_floats);
  find("ried_layer_norm_bwd", abi.layer_norm_bwd);
  find("ried_rotary", abi.rotary);
  find("ried_xattn_fwd_scratch_floats", abi.xattn_fwd_scratch_floats);
  find("ried_xattn_fwd", abi.xattn_fwd);
  find("ried_xattn_bwd_scratch_floats", abi.xattn_bwd_scratch_floats);
  find("ried_xattn_bwd", abi.xattn_bwd);
  connected = true;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL
PyMethodDef methods[] = {
    {"connect", py_connect, METH_O, "connect({name: address}): the entry points to call"},
    {"layer_norm", FAST(py_layer_norm), "layer_norm(x, weight, bias, eps), or None where more than the launch is needed"},
    {"rotary", FAST(py_rotary), "rotary(x, positions, freqs, sections, interleaved, inverse), or None"},
    {"cross_attention", FAST(py_cross_attention), "cross_attention(q, k, v, lengths, key_mask, scale), or None"},
    {"dual", FAST(py_dual), "dual(*tensors): whether one of them has a forward-mode tangent"},
    {"traced", py_traced, METH_NOARGS, "traced(): whether torch records the operations of this thread"},
    {"gradients", FAST(py_gradients), "gradients(params, addresses, sizes, out): whether out holds the gradients' addresses"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", "Direct calls of the token operators", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind() { return PyModule_Create(&module); }

// The operators' binding to torch tensors (module lama_b200._operators, used by
// lama_b200/operators.py): checks of arguments, outputs and workspaces from
// torch's allocator, torch's current stream, and the call of the C ABI
// (include/lama_b200.h).
//
// Native because the host is what bounds a small call: a single-token step
// takes the GPU 2.8 us and, with these checks and structures made in Python,
// took the host 17 us.
//
// The library is loaded by lama_b200.engine; its entry points come from there
// (setup), so this module links against torch alone.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <string>
#include <vector>

#include "lama_b200.h"

namespace {

using at::Tensor;

// ------------------------------------------------------------------ errors

PyObject* g_error = nullptr;  // lama_b200.LamaError(code, message)

struct Refusal {
  int code;
  std::string msg;
};

[[noreturn]] void refuse(const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  throw Refusal{LAMA_EINVAL, buf};
}

std::string text(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); i++) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + (s.size() == 1 ? ",)" : ")");
}

PyObject* raise(const Refusal& r) {
  PyObject* e = PyObject_CallFunction(g_error, "is", r.code, r.msg.c_str());
  if (e) {
    PyErr_SetObject(g_error, e);
    Py_DECREF(e);
  }
  return nullptr;
}

// ------------------------------------------------------------------ the library

struct Library {
  decltype(&lama_linear_attention_workspace) attention_workspace;
  decltype(&lama_linear_attention) attention;
  decltype(&lama_linear_attention_backward) attention_backward;
  decltype(&lama_linear_attention_step) attention_step;
  decltype(&lama_gated_residual_norm) norm;
  decltype(&lama_gated_residual_norm_workspace) norm_workspace;
  decltype(&lama_gated_residual_norm_backward) norm_backward;
  decltype(&lama_checkpoint_store) store;
  decltype(&lama_checkpoint_restore) restore;
} L;

// A call of the library without the interpreter's lock; its message on failure.
template <class F>
long long call(F&& f) {
  char err[256] = "";
  long long rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = f(err, (int)sizeof(err));
  Py_END_ALLOW_THREADS;
  if (rc < 0) throw Refusal{(int)rc, err};
  return rc;
}

// ------------------------------------------------------------------ arguments

// None of the operators has a forward-mode derivative: a dual tensor would lose its tangent here.
const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse("%s is not a tensor", name);
  const Tensor& t = THPVariable_Unpack(o);
  if (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
    refuse("%s has a tangent: the operators have no forward-mode derivative", name);
  return t;
}

int type_code(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat:
      return LAMA_F32;
    case at::kHalf:
      return LAMA_F16;
    case at::kBFloat16:
      return LAMA_BF16;
    default:
      refuse("%s has type %s; float32, float16 and bfloat16 are supported", name, at::toString(t.scalar_type()));
  }
}

// A call's first tensor: on a CUDA device, of a supported type.
const Tensor& first(PyObject* o, const char* name, int& dev, int& code) {
  const Tensor& t = tensor(o, name);
  if (!t.is_cuda() || t.layout() != at::kStrided) refuse("%s is not on a CUDA device", name);
  code = type_code(t, name);
  dev = t.get_device();
  return t;
}

// Another tensor of the call: same device, the given type and, unless null, shape.
const Tensor& also(PyObject* o, const char* name, int dev, at::ScalarType type, const at::IntArrayRef* shape = nullptr) {
  const Tensor& t = tensor(o, name);
  if (!t.is_cuda() || t.layout() != at::kStrided || t.get_device() != dev)
    refuse("%s is on %s, not on cuda:%d", name, t.device().str().c_str(), dev);
  if (t.scalar_type() != type)
    refuse("%s has type %s, not %s", name, at::toString(t.scalar_type()), at::toString(type));
  if (shape && t.sizes() != *shape) refuse("%s has shape %s, not %s", name, text(t.sizes()).c_str(), text(*shape).c_str());
  return t;
}

Tensor contiguous(const Tensor& t) { return t.is_contiguous() ? t : t.contiguous(); }

Tensor empty(at::IntArrayRef shape, at::ScalarType type, int dev) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(at::kCUDA, (c10::DeviceIndex)dev));
}

void* stream(int dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }

template <class T = void>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

PyObject* wrap(const Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}

PyObject* tuple(std::initializer_list<Tensor> ts) {
  PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
  if (!r) return nullptr;
  Py_ssize_t i = 0;
  for (const Tensor& t : ts) {
    PyObject* o = wrap(t);
    if (!o) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

double number(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse("%s is not a number", name);
  }
  return v;
}

// ------------------------------------------------------------------ linear attention

// The tensor itself where the kernels take its strides at full speed, else a
// contiguous copy: rows have to be contiguous, and 16-bit rows of a multiple
// of 8 channels on 16-byte boundaries (the copy then goes through the same
// kernel as a contiguous tensor, to the same bits).
Tensor unit(const Tensor& t, bool whole) {
  const auto n = t.sizes(), s = t.strides();
  const size_t d = n.size() - 1;
  if (s[d] != 1 && n[d] != 1) return t.contiguous();
  if (whole && t.scalar_type() != at::kFloat && n[d] % 8 == 0) {
    if (n[1] > 1 && s[1] == 0) return t.contiguous();
    bool fits = ((uintptr_t)t.data_ptr() & 15) == 0;
    for (size_t i = 0; i < d; i++) fits = fits && (s[i] % 8 == 0 || n[i] <= 1);
    if (!fits) return t.clone(at::MemoryFormat::Contiguous);
  }
  return t;
}

// [B,T,n,D] or [B,n,D]; a lone row's stride is arbitrary
lama_rows rows(const Tensor& t) {
  const auto n = t.sizes(), s = t.strides();
  const size_t h = n.size() - 2;
  lama_rows r;
  r.data = t.data_ptr();
  r.batch_stride = n[0] > 1 ? s[0] : 0;
  r.token_stride = n.size() == 4 && n[1] > 1 ? s[1] : 0;
  r.head_stride = n[h] > 1 ? s[h] : 0;
  r.heads = (int)n[h];
  return r;
}

struct Attention {
  Tensor q, k, v, decay, init, lengths;
  int dev, h, dk, dv;
  int64_t b, t;
  at::ScalarType type;
  lama_attention a{};

  // ndim 4: [B,T,n,D]; 3: [B,n,D], one token
  Attention(PyObject* oq, PyObject* ok, PyObject* ov, PyObject* od, PyObject* oscale, PyObject* oinit, PyObject* olen,
            int ndim) {
    int code;
    const Tensor& q0 = first(oq, "q", dev, code);
    type = q0.scalar_type();
    if (q0.dim() != ndim) refuse("q has %d dimensions, not %d", (int)q0.dim(), ndim);
    const Tensor &k0 = also(ok, "k", dev, type), &v0 = also(ov, "v", dev, type);
    const Tensor* kv[2] = {&k0, &v0};
    for (int i = 0; i < 2; i++)
      if (kv[i]->dim() != ndim || kv[i]->sizes().slice(0, ndim - 2) != q0.sizes().slice(0, ndim - 2))
        refuse("%s has shape %s, which does not go with q's %s", i ? "v" : "k", text(kv[i]->sizes()).c_str(),
               text(q0.sizes()).c_str());
    if (k0.size(-1) != q0.size(-1)) refuse("q has %lld channels a head and k %lld", (long long)q0.size(-1), (long long)k0.size(-1));
    const Tensor& d0 = also(od, "log_decay", dev, at::kFloat);
    if (d0.dim() != 1) refuse("log_decay has %d dimensions, not 1", (int)d0.dim());
    if (d0.requires_grad() && at::GradMode::is_enabled())
      refuse("log_decay has no gradient: the decays are constants of the layer");
    const int64_t heads = d0.size(0);
    const Tensor* all[3] = {&q0, &k0, &v0};
    const char* names[3] = {"q", "k", "v"};
    for (int i = 0; i < 3; i++) {
      const int64_t n = all[i]->size(-2);
      if (n < 1 || heads < n || heads % n)
        refuse("%s has %lld heads, which do not divide the %lld of log_decay", names[i], (long long)n, (long long)heads);
    }
    if (q0.size(-1) < 1 || q0.size(-1) > 128 || v0.size(-1) < 1 || v0.size(-1) > 128)
      refuse("head sizes %lld and %lld are not in 1..128", (long long)q0.size(-1), (long long)v0.size(-1));
    b = q0.size(0), t = ndim == 4 ? q0.size(1) : 1;
    if (b > 0x7fffffff || t > 0x7fffffff || heads > 0x7fffffff) refuse("a dimension exceeds 2^31 - 1");
    h = (int)heads, dk = (int)q0.size(-1), dv = (int)v0.size(-1);
    if (oinit != Py_None) {
      const int64_t s[4] = {b, h, dk, dv};
      const at::IntArrayRef shape(s, 4);
      init = contiguous(also(oinit, "initial_state", dev, at::kFloat, &shape));
    }
    if (olen != Py_None) {
      const int64_t s[1] = {b};
      const at::IntArrayRef shape(s, 1);
      lengths = contiguous(also(olen, "lengths", dev, at::kInt, &shape));
    }
    const bool whole = ndim == 4;
    q = unit(q0, whole), k = unit(k0, whole), v = unit(v0, whole), decay = contiguous(d0);
    a.dtype = code;
    a.batch = (int)b, a.tokens = (int)t, a.heads = h, a.dk = dk, a.dv = dv;
    a.q = rows(q), a.k = rows(k), a.v = rows(v);
    a.log_decay = ptr<float>(decay);
    a.initial_state = ptr<float>(init);
    a.lengths = ptr<int>(lengths);
    a.scale = oscale == Py_None ? (float)(1.0 / std::sqrt((double)dk)) : (float)number(oscale, "scale");
  }

  Tensor workspace(int backward, long long& bytes) const {
    char err[256] = "";
    bytes = L.attention_workspace(&a, backward, err, sizeof(err));
    if (bytes < 0) throw Refusal{(int)bytes, err};
    return bytes ? empty({(int64_t)bytes}, at::kByte, dev) : Tensor();
  }
};

Tensor attention_forward(const Attention& x, bool return_state, Tensor& state) {
  Tensor o = empty({x.b, x.t, x.h, x.dv}, x.type, x.dev);
  if (return_state) state = empty({x.b, x.h, x.dk, x.dv}, at::kFloat, x.dev);
  if (x.b == 0 || x.t == 0) {
    if (return_state) x.init.defined() ? state.copy_(x.init) : state.zero_();
    return o;
  }
  long long n;
  const Tensor w = x.workspace(0, n);
  const lama_rows out = rows(o);
  void* st = stream(x.dev);
  call([&](char* err, int len) { return L.attention(&x.a, &out, ptr<float>(state), ptr(w), n, x.dev, st, err, len); });
  return o;
}

// (q, k, v, log_decay, scale, initial_state, lengths, return_state) -> (o, state or None)
PyObject* py_attention(PyObject* const* p) {
  const Attention x(p[0], p[1], p[2], p[3], p[4], p[5], p[6], 4);
  Tensor state;
  const Tensor o = attention_forward(x, p[7] == Py_True, state);
  return tuple({o, state});
}

// (grad_o, q, k, v, log_decay, scale, initial_state, lengths, grad_state) -> (dq, dk, dv, ds or None)
PyObject* py_attention_backward(PyObject* const* p) {
  const Attention x(p[1], p[2], p[3], p[4], p[5], p[6], p[7], 4);
  const int64_t so[4] = {x.b, x.t, x.h, x.dv}, ss[4] = {x.b, x.h, x.dk, x.dv};
  const at::IntArrayRef oshape(so, 4), sshape(ss, 4);
  const Tensor go = unit(also(p[0], "grad_o", x.dev, x.type, &oshape), true);
  Tensor gs, ds;
  if (p[8] != Py_None) gs = contiguous(also(p[8], "grad_state", x.dev, at::kFloat, &sshape));
  Tensor dq = empty(x.q.sizes(), x.type, x.dev), dk = empty(x.k.sizes(), x.type, x.dev),
         dv = empty(x.v.sizes(), x.type, x.dev);
  if (x.init.defined()) ds = empty(sshape, at::kFloat, x.dev);
  if (x.b == 0 || x.t == 0) {
    if (ds.defined()) gs.defined() ? ds.copy_(gs) : ds.zero_();
    return tuple({dq, dk, dv, ds});
  }
  lama_attention_grads g{};
  g.grad_out = rows(go), g.grad_q = rows(dq), g.grad_k = rows(dk), g.grad_v = rows(dv);
  g.grad_final_state = ptr<float>(gs), g.grad_initial_state = ptr<float>(ds);
  long long n;
  const Tensor w = x.workspace(1, n);
  void* st = stream(x.dev);
  call([&](char* err, int len) { return L.attention_backward(&x.a, &g, ptr(w), n, x.dev, st, err, len); });
  return tuple({dq, dk, dv, ds});
}

// (q, k, v, log_decay, state, scale, slots, out_state) -> o
PyObject* py_attention_step(PyObject* const* p) {
  const Attention x(p[0], p[1], p[2], p[3], p[5], Py_None, Py_None, 3);
  const Tensor& state = also(p[4], "state", x.dev, at::kFloat);
  if (at::GradMode::is_enabled() && (x.q.requires_grad() || x.k.requires_grad() || x.v.requires_grad() || state.requires_grad()))
    refuse("a step has no gradient: call it under torch.no_grad() or use linear_attention");
  if (state.dim() != 4 || state.size(1) != x.h || state.size(2) != x.dk || state.size(3) != x.dv || !state.is_contiguous())
    refuse("state is not a contiguous tensor of shape (slots, %d, %d, %d)", x.h, x.dk, x.dv);
  Tensor out = state;
  if (p[7] != Py_None) {
    const at::IntArrayRef shape = state.sizes();
    out = also(p[7], "out_state", x.dev, at::kFloat, &shape);
    if (!out.is_contiguous()) refuse("out_state is not contiguous");
  }
  Tensor slots;
  if (p[6] != Py_None) {
    const int64_t s[1] = {x.b};
    const at::IntArrayRef shape(s, 1);
    slots = contiguous(also(p[6], "slots", x.dev, at::kInt, &shape));
  } else if (state.size(0) < x.b) {
    refuse("%lld states for %lld rows", (long long)state.size(0), (long long)x.b);
  }
  if (state.size(0) > 0x7fffffff) refuse("a dimension exceeds 2^31 - 1");
  Tensor o = empty({x.b, x.h, x.dv}, x.type, x.dev);
  if (x.b == 0) return wrap(o);
  if (state.size(0) == 0) return wrap(o.zero_());
  const lama_rows r = rows(o);
  void* st = stream(x.dev);
  call([&](char* err, int len) {
    return L.attention_step(&x.a, &r, ptr<float>(state), ptr<float>(out), (int)state.size(0), ptr<int>(slots), x.dev, st,
                            err, len);
  });
  // written behind autograd's back: a graph that saved the tensor has to see that it changed
  if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
  return wrap(o);
}

// ------------------------------------------------------------------ rows of channels

// [...,C] as a matrix of rows with one stride between them (a copy where its
// strides do not allow that).
struct Matrix {
  Tensor hold;
  void* p = nullptr;
  int64_t stride = 0;
  Matrix() = default;
  explicit Matrix(const Tensor& t) : hold(t) {
    const int64_t c = t.size(-1);
    stride = c;
    if (!t.is_contiguous()) {
      if (t.dim() != 2) hold = t.reshape({-1, c});
      const auto n = hold.sizes(), s = hold.strides();
      if ((n[1] > 1 && s[1] != 1) || (n[0] > 1 && s[0] < c))
        hold = hold.contiguous();
      else if (n[0] > 1)
        stride = s[0];
    }
    p = hold.data_ptr();
  }
};

constexpr int64_t GROUP = 128;

void empty_checkpoint(const Tensor& x, int dev, Tensor& codes, Tensor& scales) {
  codes = empty(x.sizes(), at::kChar, dev);
  c10::SmallVector<int64_t, 6> s(x.sizes().begin(), x.sizes().end());
  s.back() = (s.back() + GROUP - 1) / GROUP;
  scales = empty(s, at::kFloat, dev);
}

// (x) -> (codes, scales)
PyObject* py_store(PyObject* const* p) {
  int dev, code;
  if (THPVariable_Check(p[0]) && THPVariable_Unpack(p[0]).requires_grad() && at::GradMode::is_enabled())
    refuse("a checkpoint has no gradient: call it under torch.no_grad() or on x.detach()");
  const Tensor& x = first(p[0], "x", dev, code);
  if (x.dim() < 1 || x.size(-1) > 0x7fffffff) refuse("x has no channels, or more than 2^31 - 1");
  Tensor codes, scales;
  empty_checkpoint(x, dev, codes, scales);
  if (x.numel()) {
    const Matrix m(x);
    const int c = (int)x.size(-1);
    void* st = stream(dev);
    call([&](char* err, int len) {
      return L.store(m.p, code, x.numel() / c, c, m.stride, ptr<int8_t>(codes), ptr<float>(scales), dev, st, err, len);
    });
  }
  return tuple({codes, scales});
}

// (codes, scales, type code) -> x
PyObject* py_restore(PyObject* const* p) {
  const Tensor& codes0 = tensor(p[0], "codes");
  if (!codes0.is_cuda() || codes0.scalar_type() != at::kChar || codes0.dim() < 1 || codes0.size(-1) > 0x7fffffff)
    refuse("codes is not an int8 tensor of rows on a CUDA device");
  const int dev = codes0.get_device();
  c10::SmallVector<int64_t, 6> s(codes0.sizes().begin(), codes0.sizes().end());
  s.back() = (s.back() + GROUP - 1) / GROUP;
  const at::IntArrayRef shape(s);
  const Tensor scales = contiguous(also(p[1], "scales", dev, at::kFloat, &shape));
  const long code = PyLong_AsLong(p[2]);
  if (code < LAMA_F32 || code > LAMA_BF16) refuse("unknown element type");
  const at::ScalarType types[3] = {at::kFloat, at::kHalf, at::kBFloat16};
  const Tensor x = empty(codes0.sizes(), types[code], dev);
  if (x.numel()) {
    const Tensor codes = contiguous(codes0);
    const int c = (int)x.size(-1);
    void* st = stream(dev);
    call([&](char* err, int len) {
      return L.restore(ptr<int8_t>(codes), ptr<float>(scales), (int)code, x.numel() / c, c, c, ptr(x), dev, st, err, len);
    });
  }
  return wrap(x);
}

// ------------------------------------------------------------------ norms, gate and residual

Tensor vector(PyObject* o, const char* name, int dev, int64_t c) {
  const Tensor& w = tensor(o, name);
  if (!w.is_cuda() || w.get_device() != dev || w.dim() != 1 || w.size(0) != c)
    refuse("%s is not a tensor of %lld channels on cuda:%d", name, (long long)c, dev);
  type_code(w, name);
  return contiguous(w.scalar_type() == at::kFloat ? w : w.to(at::kFloat));
}

struct Norm {
  Tensor post, pre, scales;
  Matrix gate;
  Tensor gate0;
  lama_norm a{};
  // post, pre, gate, residual_scale, eps at p[0..4]
  Norm(PyObject* const* p, at::IntArrayRef shape, int64_t numel, at::ScalarType type, int code, int dev) {
    const int64_t c = shape.back();
    if (c > 0x7fffffff) refuse("x has more than 2^31 - 1 channels");
    a.dtype = code;
    a.channels = (int)c;
    a.rows = c ? numel / c : 0;
    if (p[0] != Py_None) post = vector(p[0], "post_weight", dev, c);
    if (p[1] != Py_None) pre = vector(p[1], "pre_weight", dev, c);
    if (THPVariable_Check(p[3]))
      scales = vector(p[3], "residual_scale", dev, c);
    else
      a.residual_scale = (float)number(p[3], "residual_scale");
    const double eps = number(p[4], "eps");
    if (!(eps >= 0)) refuse("eps must not be negative");
    a.eps = (float)eps;
    a.post_weight = ptr<float>(post), a.pre_weight = ptr<float>(pre), a.residual_scales = ptr<float>(scales);
    a.gate_rows = 1;
    if (p[2] != Py_None) {
      gate0 = also(p[2], "gate", dev, type);
      a.gate_rows = period(gate0.sizes(), shape);
      if (numel) {
        gate = Matrix(gate0);
        a.gate = gate.p;
        a.gate_stride = gate.stride;
      }
    }
  }
  // rows of x that share one row of a gate, whose dimensions of size 1 have to
  // be the innermost of x's row dimensions
  static int64_t period(at::IntArrayRef g, at::IntArrayRef x) {
    const int gd = (int)g.size(), xd = (int)x.size();
    if (gd < 1 || gd > xd || g[gd - 1] != x[xd - 1])
      refuse("a gate of shape %s does not broadcast over %s", text(g).c_str(), text(x).c_str());
    int64_t per = 1;
    bool whole = false;
    for (int i = 2; i <= xd; i++) {
      const int64_t n = i <= gd ? g[gd - i] : 1, m = x[xd - i];
      if (n == m && (m != 1 || whole))
        whole = true;
      else if (n == 1 && !whole)
        per *= m;
      else if (n != m)
        refuse("a gate of shape %s does not broadcast over %s one gate row to neighbouring rows; expand it",
               text(g).c_str(), text(x).c_str());
    }
    return per < 1 ? 1 : per;
  }
};

// (x, y, post, pre, gate, residual_scale, eps, save: 0 nothing, 1 statistics, 2 and 8-bit codes)
// -> (u, n, post_rstd, pre_rstd, y codes, y scales, u codes, u scales), None where not made
PyObject* py_norm(PyObject* const* p) {
  int dev, code;
  const Tensor& x = first(p[0], "x", dev, code);
  const at::IntArrayRef shape = x.sizes();
  if (shape.size() < 1 || shape.back() < 1) refuse("x has no channels");
  const Tensor& y = also(p[1], "y", dev, x.scalar_type(), &shape);
  const Norm a(p + 2, shape, x.numel(), x.scalar_type(), code, dev);
  const long save = PyLong_AsLong(p[7]);
  Tensor u = empty(shape, x.scalar_type(), dev), n, ry, ru, cy, sy, cu, su;
  const bool post = a.post.defined(), pre = a.pre.defined();
  if (pre) n = empty(shape, x.scalar_type(), dev);
  if (save) {
    const at::IntArrayRef lead = shape.slice(0, shape.size() - 1);
    if (post) ry = empty(lead, at::kFloat, dev);
    if (pre) ru = empty(lead, at::kFloat, dev);
    if (save == 2) {
      empty_checkpoint(x, dev, cy, sy);
      if (pre) empty_checkpoint(x, dev, cu, su);
    }
  }
  if (x.numel()) {
    const Matrix mx(x), my(y);
    void* st = stream(dev);
    call([&](char* err, int len) {
      return L.norm(&a.a, mx.p, mx.stride, my.p, my.stride, ptr(u), ptr(n), ptr<float>(ry), ptr<float>(ru),
                    ptr<int8_t>(cy), ptr<float>(sy), ptr<int8_t>(cu), ptr<float>(su), dev, st, err, len);
    });
  }
  return tuple({u, n, ry, ru, cy, sy, cu, su});
}

// (like: a tensor of the rows' shape, type code, grad_u, grad_n, post, pre, gate, residual_scale, eps, y, y scales, u, u scales,
//  post_rstd, pre_rstd) -> (dx, dy, dpost, dpre, dgate, dscale); with y scales, y and u are codes
PyObject* py_norm_backward(PyObject* const* p) {
  const Tensor& like = tensor(p[0], "y");
  const int dev = like.get_device();
  const long code = PyLong_AsLong(p[1]);
  if (!like.is_cuda() || code < LAMA_F32 || code > LAMA_BF16) refuse("the saved tensors are not on a CUDA device");
  const at::ScalarType types[3] = {at::kFloat, at::kHalf, at::kBFloat16}, type = types[code];
  const at::IntArrayRef shape = like.sizes();
  Tensor gu, gn;
  if (p[2] != Py_None) gu = also(p[2], "grad_u", dev, type, &shape);
  if (p[3] != Py_None) gn = also(p[3], "grad_n", dev, type, &shape);
  const Norm a(p + 4, shape, like.numel(), type, (int)code, dev);
  const int64_t c = shape.back();
  Tensor dx = empty(shape, type, dev), dy = empty(shape, type, dev), dpost, dpre, dgate, dscale;
  if (a.post.defined()) dpost = empty({c}, at::kFloat, dev);
  if (a.pre.defined()) dpre = empty({c}, at::kFloat, dev);
  if (a.scales.defined()) dscale = empty({c}, at::kFloat, dev);
  if (a.gate0.defined()) dgate = empty(a.gate0.sizes(), type, dev);
  if (!like.numel()) {
    for (Tensor* t : {&dpost, &dpre, &dscale, &dgate})
      if (t->defined()) t->zero_();
    return tuple({dx, dy, dpost, dpre, dgate, dscale});
  }
  lama_norm_grads g{};
  Matrix mu, mn, my, mz;
  if (gu.defined()) mu = Matrix(gu);
  if (gn.defined()) mn = Matrix(gn);
  g.grad_u = mu.p, g.grad_u_stride = mu.stride;
  g.grad_n = mn.p, g.grad_n_stride = mn.stride;
  Tensor ys, us, cy, cu;
  if (p[10] != Py_None) {
    cy = contiguous(also(p[9], "y's codes", dev, at::kChar, &shape));
    ys = contiguous(also(p[10], "y's scales", dev, at::kFloat));
    g.y_codes = ptr<int8_t>(cy), g.y_scales = ptr<float>(ys);
    if (p[11] != Py_None) {
      cu = contiguous(also(p[11], "u's codes", dev, at::kChar, &shape));
      us = contiguous(also(p[12], "u's scales", dev, at::kFloat));
      g.u_codes = ptr<int8_t>(cu), g.u_scales = ptr<float>(us);
    }
  } else {
    my = Matrix(also(p[9], "y", dev, type, &shape));
    g.y = my.p, g.y_stride = my.stride;
    if (p[11] != Py_None) {
      mz = Matrix(also(p[11], "u", dev, type, &shape));
      g.u = mz.p, g.u_stride = mz.stride;
    }
  }
  Tensor ry, ru;
  if (p[13] != Py_None) ry = contiguous(also(p[13], "post_rstd", dev, at::kFloat));
  if (p[14] != Py_None) ru = contiguous(also(p[14], "pre_rstd", dev, at::kFloat));
  const int64_t nrows = like.numel() / c, groups = (c + GROUP - 1) / GROUP;
  if ((ry.defined() && ry.numel() != nrows) || (ru.defined() && ru.numel() != nrows) ||
      (ys.defined() && ys.numel() != nrows * groups) || (us.defined() && us.numel() != nrows * groups))
    refuse("the saved statistics or scales do not have one entry a row or group");
  g.post_rstd = ptr<float>(ry), g.pre_rstd = ptr<float>(ru);
  g.grad_x = ptr(dx), g.grad_y = ptr(dy), g.grad_gate = ptr(dgate);
  g.grad_post_weight = ptr<float>(dpost), g.grad_pre_weight = ptr<float>(dpre), g.grad_residual_scales = ptr<float>(dscale);
  char err[256] = "";
  const long long n = L.norm_workspace(&a.a, err, sizeof(err));
  if (n < 0) throw Refusal{(int)n, err};
  const Tensor w = empty({(int64_t)n}, at::kByte, dev);
  void* st = stream(dev);
  call([&](char* e, int len) { return L.norm_backward(&a.a, &g, ptr(w), n, dev, st, e, len); });
  return tuple({dx, dy, dpost, dpre, dgate, dscale});
}

// ------------------------------------------------------------------ module

// (LamaError, addresses of the entry points in the order of Library)
PyObject* py_setup(PyObject* const* p) {
  void* at[9];
  for (int i = 0; i < 9; i++) {
    at[i] = PyLong_AsVoidPtr(p[1 + i]);
    if (!at[i]) return PyErr_Occurred() ? nullptr : raise(Refusal{LAMA_EINVAL, "an entry point is missing"});
  }
  static_assert(sizeof(L) == sizeof(at), "one address an entry point");
  memcpy(&L, at, sizeof(at));
  Py_INCREF(p[0]);
  Py_XSETREF(g_error, p[0]);
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments expected, %zd given", N, n);
    return nullptr;
  }
  HANDLE_TH_ERRORS
  try {
    at::AutoDispatchBelowADInplaceOrView plain;  // outputs and copies are no part of autograd's graph here
    return F(args);
  } catch (const Refusal& r) {
    return raise(r);
  }
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject* const*), int N>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<F, N>)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<py_setup, 10>("setup"),
                         method<py_attention, 8>("attention"),
                         method<py_attention_backward, 9>("attention_backward"),
                         method<py_attention_step, 8>("attention_step"),
                         method<py_store, 1>("store"),
                         method<py_restore, 3>("restore"),
                         method<py_norm, 8>("norm"),
                         method<py_norm_backward, 15>("norm_backward"),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_operators", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__operators(void) { return PyModule_Create(&module); }

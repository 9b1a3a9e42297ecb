// CPython side of the step operators (fused_adamw, fused_normed_update,
// fused_newton_schulz_heads): reads the tensors' pointers and sizes in C++ and
// makes the C-ABI call.  A list of small tensors is bound by this and not by the
// kernel: 20 vectors took 45 µs through Python's attribute calls and ctypes (7
// here), the kernel 4.  The tensors are not copied: their reference counts alone
// cost 3 µs.
//
// Only the plain case is handled here: ordinary CUDA tensors, the lists contiguous
// and of one device and type, that agree in their shapes.  For anything else a
// function returns None, and the Python front checks tensor by tensor, names what
// is wrong or takes the list apart.  Otherwise it returns the C call's status.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <exception>
#include <vector>

#include "../../include/fused_muon.h"

namespace {

using AdamwFn = decltype(&fm_adamw);
using NormedFn = decltype(&fm_muon_apply_normed);
using NormedSizeFn = decltype(&fm_normed_workspace_size);
using HeadsFn = decltype(&fm_newton_schulz_heads);
using HeadsSizeFn = decltype(&fm_heads_workspace_size);
AdamwFn g_adamw = nullptr;
NormedFn g_normed = nullptr;
NormedSizeFn g_normed_size = nullptr;
HeadsFn g_heads = nullptr;
HeadsSizeFn g_heads_size = nullptr;

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return FM_DT_F32;
    case at::kBFloat16: return FM_DT_BF16;
    case at::kHalf: return FM_DT_F16;
    default: return -1;
  }
}

// A list or tuple of ordinary contiguous CUDA tensors, all of one type, on one
// device; false where it is anything else.
class TensorList {
 public:
  explicit TensorList(PyObject* seq) {
    if (!PyList_Check(seq) && !PyTuple_Check(seq)) return;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
    PyObject** items = PySequence_Fast_ITEMS(seq);
    t_.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
      if (!THPVariable_CheckExact(items[i])) return;
      const at::Tensor& t = THPVariable_Unpack(items[i]);
      if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.is_inference() ||
          !t.is_contiguous() || t.is_neg() || t.is_conj())
        return;
      if (i > 0 && (t.scalar_type() != t_[0]->scalar_type() || t.device() != t_[0]->device())) return;
      t_.push_back(&t);
    }
    ok_ = true;
  }
  bool ok() const { return ok_; }
  size_t size() const { return t_.size(); }
  const at::Tensor& operator[](size_t i) const { return *t_[i]; }
  void bump() const {
    for (const at::Tensor* t : t_) t->unsafeGetTensorImpl()->bump_version();
  }

 private:
  std::vector<const at::Tensor*> t_;  // the Python objects hold them throughout the call
  bool ok_ = false;
};

bool same_shapes(const TensorList& a, const TensorList& b) {
  if (a.size() != b.size() || a[0].device() != b[0].device()) return false;
  for (size_t i = 0; i < a.size(); ++i)
    if (a[i].sizes() != b[i].sizes()) return false;
  return true;
}

void* current_stream(const at::Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

// adamw(params, grads, moments1, moments2, alphas, decay, w1, w2, eps, bump);
// alphas is a float for all or a list of one per tensor, bump whether autograd
// sees the writes.
PyObject* adamw(PyObject*, PyObject* args) {
  PyObject *po, *go, *mo, *vo, *ao;
  double decay, w1, w2, eps;
  int bump;
  if (!PyArg_ParseTuple(args, "OOOOOddddp", &po, &go, &mo, &vo, &ao, &decay, &w1, &w2, &eps, &bump))
    return nullptr;
  try {
    const TensorList p(po), g(go), m(mo), v(vo);
    if (!p.ok() || !g.ok() || !m.ok() || !v.ok() || p.size() == 0) Py_RETURN_NONE;
    if (!same_shapes(p, g) || !same_shapes(p, m) || !same_shapes(p, v)) Py_RETURN_NONE;
    const at::ScalarType pt = p[0].scalar_type(), mt = m[0].scalar_type();
    if (dtype_code(pt) < 0 || g[0].scalar_type() != pt || v[0].scalar_type() != mt ||
        (mt != pt && mt != at::kFloat))
      Py_RETURN_NONE;
    const bool one = PyFloat_Check(ao);
    if (!one && (!PyList_Check(ao) || PyList_GET_SIZE(ao) != Py_ssize_t(p.size()))) Py_RETURN_NONE;
    std::vector<fm_adamw_tensor> table(p.size());
    for (size_t i = 0; i < p.size(); ++i) {
      const double alpha = PyFloat_AsDouble(one ? ao : PyList_GET_ITEM(ao, i));
      if (alpha == -1.0 && PyErr_Occurred()) return nullptr;
      table[i] = {p[i].data_ptr(), g[i].data_ptr(), m[i].data_ptr(),
                  v[i].data_ptr(), p[i].numel(),    static_cast<float>(alpha)};
    }
    const c10::cuda::CUDAGuard guard(p[0].device());
    const int rc = g_adamw(table.data(), int64_t(table.size()), dtype_code(pt), dtype_code(mt),
                           float(decay), float(w1), float(w2), float(eps), current_stream(p[0]));
    if (rc == FM_OK && bump) {
      p.bump();
      m.bump();
      v.bump();
    }
    return PyLong_FromLong(rc);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// normed(params, updates, row_moments, decay, step_per_sqrt, beta2, eps,
// workspace or None); step_per_sqrt is lr·0.2.
PyObject* normed(PyObject*, PyObject* args) {
  PyObject *po, *uo, *vo, *wo;
  double decay, step, beta2, eps;
  if (!PyArg_ParseTuple(args, "OOOddddO", &po, &uo, &vo, &decay, &step, &beta2, &eps, &wo))
    return nullptr;
  try {
    const TensorList p(po), v(vo);
    if (!p.ok() || !v.ok() || p.size() == 0 || v.size() != p.size() || p[0].dim() < 2 ||
        p[0].numel() == 0 || dtype_code(p[0].scalar_type()) < 0 ||
        v[0].scalar_type() != at::kFloat || v[0].device() != p[0].device())
      Py_RETURN_NONE;
    const int64_t n = int64_t(p.size()), rows = p[0].size(0), numel = p[0].numel();
    std::vector<fm_normed_matrix> table(p.size());
    auto update_ok = [&](const at::Tensor& u) {
      return u.scalar_type() == at::kBFloat16 && u.device() == p[0].device();
    };
    if (THPVariable_CheckExact(uo)) {
      const at::Tensor& u = THPVariable_Unpack(uo);
      if (!u.is_cuda() || u.layout() != at::kStrided || !u.is_contiguous() || u.is_neg() ||
          !update_ok(u) || u.dim() < 2 || u.size(0) != n || u.size(1) != rows || u.numel() != n * numel)
        Py_RETURN_NONE;
      for (int64_t i = 0; i < n; ++i)
        table[i].update = static_cast<const char*>(u.data_ptr()) + 2 * i * numel;
    } else {
      const TensorList u(uo);
      if (!u.ok() || u.size() != p.size() || !update_ok(u[0])) Py_RETURN_NONE;
      for (int64_t i = 0; i < n; ++i) {
        if (u[i].numel() != numel || u[i].dim() == 0 || u[i].size(0) != rows) Py_RETURN_NONE;
        table[i].update = u[i].data_ptr();
      }
    }
    for (int64_t i = 0; i < n; ++i) {
      if (p[i].sizes() != p[0].sizes() || v[i].dim() != 1 || v[i].numel() != rows) Py_RETURN_NONE;
      table[i].param = p[i].data_ptr();
      table[i].row_moment = v[i].data_ptr<float>();
    }
    uint64_t need = 0;
    if (const int rc = g_normed_size(n, rows, &need)) return PyLong_FromLong(rc);
    at::Tensor ws;
    if (wo != Py_None) {
      if (!THPVariable_CheckExact(wo)) Py_RETURN_NONE;
      ws = THPVariable_Unpack(wo);
      if (!ws.is_cuda() || ws.device() != p[0].device() || !ws.is_contiguous() || ws.nbytes() < need)
        Py_RETURN_NONE;
    } else {
      ws = at::empty({int64_t(need)}, at::TensorOptions().dtype(at::kByte).device(p[0].device()));
    }
    const c10::cuda::CUDAGuard guard(p[0].device());
    const int rc = g_normed(table.data(), n, rows, numel / rows, dtype_code(p[0].scalar_type()),
                            float(decay), float(step * std::sqrt(double(numel))), beta2,
                            float(eps), ws.data_ptr(), ws.nbytes(), current_stream(p[0]));
    if (rc == FM_OK) {
      p.bump();
      v.bump();
    }
    return PyLong_FromLong(rc);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// heads(G, heads, dim, steps, workspace or None, out or None): the result tensor,
// or the C call's status where it failed.
PyObject* heads(PyObject*, PyObject* args) {
  PyObject *go, *wo, *oo;
  long long nheads;
  int dim, steps;
  if (!PyArg_ParseTuple(args, "OLiiOO", &go, &nheads, &dim, &steps, &wo, &oo)) return nullptr;
  try {
    if (!THPVariable_CheckExact(go)) Py_RETURN_NONE;
    const at::Tensor& g = THPVariable_Unpack(go);
    if (!g.defined() || !g.is_cuda() || g.layout() != at::kStrided || g.is_neg() || g.is_conj() ||
        (g.dim() != 2 && g.dim() != 3) || g.numel() == 0)
      Py_RETURN_NONE;
    const int code = g.scalar_type() == at::kDouble ? FM_DT_F64 : dtype_code(g.scalar_type());
    if (code < 0) Py_RETURN_NONE;
    const int64_t rows = g.size(-2), cols = g.size(-1), ld = g.stride(-2);
    const int64_t batch = g.dim() == 3 ? g.size(0) : 1, bs = g.dim() == 3 ? g.stride(0) : 0;
    if ((g.stride(-1) != 1 && cols > 1) || ld < cols ||
        (batch > 1 && bs < (rows - 1) * ld + cols))
      Py_RETURN_NONE;
    uint64_t need = 0;
    if (const int rc = g_heads_size(batch, rows, cols, nheads, dim, &need)) return PyLong_FromLong(rc);
    const c10::cuda::CUDAGuard guard(g.device());
    const auto options = at::TensorOptions().device(g.device());
    at::Tensor out, ws;
    if (oo != Py_None) {
      if (!THPVariable_CheckExact(oo)) Py_RETURN_NONE;
      out = THPVariable_Unpack(oo);
      if (out.scalar_type() != at::kBFloat16 || out.device() != g.device() ||
          out.layout() != at::kStrided || !out.is_contiguous() || out.is_neg() ||
          out.sizes() != g.sizes())
        Py_RETURN_NONE;
    } else {
      out = at::empty(g.sizes(), options.dtype(at::kBFloat16));
    }
    if (wo != Py_None) {
      if (!THPVariable_CheckExact(wo)) Py_RETURN_NONE;
      ws = THPVariable_Unpack(wo);
      if (!ws.is_cuda() || ws.device() != g.device() || ws.layout() != at::kStrided ||
          !ws.is_contiguous() || ws.nbytes() < need)
        Py_RETURN_NONE;
    } else {
      ws = at::empty({int64_t(need)}, options.dtype(at::kByte));
    }
    const int rc = g_heads(g.data_ptr(), code, batch, rows, cols, ld, bs, nheads, dim,
                           out.data_ptr(), steps, ws.data_ptr(), ws.nbytes(), current_stream(g));
    if (rc != FM_OK) return PyLong_FromLong(rc);
    if (oo != Py_None) {
      if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
      Py_INCREF(oo);
      return oo;
    }
    return THPVariable_Wrap(out);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// bind(fm_adamw, fm_muon_apply_normed, fm_normed_workspace_size,
// fm_newton_schulz_heads, fm_heads_workspace_size): addresses of the loaded
// library's entries.
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long a, b, c, d, e;
  if (!PyArg_ParseTuple(args, "KKKKK", &a, &b, &c, &d, &e)) return nullptr;
  g_adamw = reinterpret_cast<AdamwFn>(static_cast<uintptr_t>(a));
  g_normed = reinterpret_cast<NormedFn>(static_cast<uintptr_t>(b));
  g_normed_size = reinterpret_cast<NormedSizeFn>(static_cast<uintptr_t>(c));
  g_heads = reinterpret_cast<HeadsFn>(static_cast<uintptr_t>(d));
  g_heads_size = reinterpret_cast<HeadsSizeFn>(static_cast<uintptr_t>(e));
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"adamw", adamw, METH_VARARGS, nullptr},
    {"normed", normed, METH_VARARGS, nullptr},
    {"heads", heads, METH_VARARGS, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_step_ext", nullptr, -1, g_methods,
                        nullptr,               nullptr,     nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__step_ext(void) { return PyModule_Create(&g_module); }

// vitfp4._fast: the plain calls of the FP8 block ops, the gated residual norm and cross attention in one C++ step.
//
// The small calls of these ops take 2 to 10 us on the GPU, and the Python path (argument checks, strides, three
// allocations, a ctypes call) 11 to 22 us on the host.  Each function here checks its arguments, allocates the outputs,
// calls the C ABI of libvitfp4.so on torch's current stream and returns the outputs -- or returns None, without having
// done anything, for whatever is not the plain case: then the caller goes the Python path, which copes with it
// (copies, other devices, the probe, torch.library where gradients are recorded) or says what is wrong.  Plain means:
// exact tensors on the current CUDA device, no dispatch mode, no gradients recorded, layouts that the kernels read as they are (more than
// two dimensions: contiguous).
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>

#include "vitfp4.h"

namespace {

int g_launched = 0;   // kernels that the last call launched (under the interpreter's lock)

bool plain(PyObject* o) { return THPVariable_CheckExact(o); }

// A call's tensors: unpacked, checked for their device and gradients.
struct Args {
  bool ok = !c10::impl::dispatch_mode_enabled();   // a tracer would not see the call
  const bool grad = at::GradMode::is_enabled();
  int device = -1;

  // The tensor behind o; with optional, None stays undefined.
  at::Tensor get(PyObject* o, bool optional = false) {
    if (o == Py_None) {
      ok = ok && optional;
      return {};
    }
    if (!ok || !plain(o)) {
      ok = false;
      return {};
    }
    at::Tensor t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.layout() != at::kStrided || (grad && t.requires_grad())) {
      ok = false;
      return t;
    }
    if (device < 0) {
      device = t.get_device();
      ok = device == c10::cuda::current_device();
    } else {
      ok = t.get_device() == device;
    }
    return t;
  }
};

int code_of(const at::Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? VF4_BF16 : t.scalar_type() == at::kFloat ? VF4_F32 : -1;
}

// Rows with unit column stride that do not overlap; their stride.
bool rows_ok(const at::Tensor& t, int64_t* ld) {
  if (t.dim() != 2) return false;
  const int64_t rows = t.size(0), cols = t.size(1), s0 = t.stride(0);
  if (rows < 1 || cols < 1 || (t.stride(1) != 1 && cols > 1) || (s0 < cols && rows > 1)) return false;
  *ld = rows > 1 || s0 > cols ? s0 : cols;
  return true;
}

// (..., K) as rows: a contiguous tensor of more dimensions as (rows, K); others as they are.
at::Tensor rows_of(const at::Tensor& t) {
  return t.defined() && t.dim() > 2 && t.numel() > 0 && t.is_contiguous() ? t.view({-1, t.size(-1)}) : t;
}

// Rows (rows, n) of an output with x's leading dimensions.
at::Tensor like_x(const at::Tensor& rows, const at::Tensor& x) {
  if (x.dim() == 2) return rows;
  c10::SmallVector<int64_t, 6> size(x.sizes().begin(), x.sizes().end());
  size.back() = rows.size(1);
  return rows.view(size);
}

bool vector_ok(const at::Tensor& t, int64_t n) { return !t.defined() || (t.dim() == 1 && t.size(0) == n && (n == 1 || t.stride(0) == 1)); }

const void* ptr(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

vf4_stream_t stream(int device) { return reinterpret_cast<vf4_stream_t>(c10::cuda::getCurrentCUDAStream(device).stream()); }

at::Tensor make(at::IntArrayRef size, at::IntArrayRef strides, at::ScalarType type, const at::Tensor& like) {
  return at::empty_strided(size, strides, like.options().dtype(type).requires_grad(false));
}

PyObject* pair(const at::Tensor& a, const at::Tensor& b) {
  PyObject* r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(a));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(b));
  return r;
}

// Nothing may throw into Python: an exception (out of memory) becomes None, and the Python path raises it anew.
template <typename F>
PyObject* guarded(F&& f) {
  try {
    PyObject* r = f();
    if (r) return r;
    if (PyErr_Occurred()) return nullptr;
  } catch (...) {
  }
  Py_RETURN_NONE;
}

// Code rows of K bytes, each starting on 16 bytes: the first K columns of padded rows.
at::Tensor make_codes(int64_t M, int64_t K, int64_t ldc, const at::Tensor& like) {
  const at::Tensor t = make({M, ldc}, {ldc, 1}, at::kFloat8_e4m3fn, like);
  return ldc == K ? t : t.narrow(1, 0, K);
}

// cast(x) -> (codes, scale): activations
PyObject* cast(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 1) return nullptr;
    Args in;
    const at::Tensor x0 = in.get(a[0]), x = rows_of(x0);
    int64_t ld;
    if (!in.ok || code_of(x) < 0 || !rows_ok(x, &ld)) return nullptr;
    const int64_t M = x.size(0), K = x.size(1), kb = (K + 127) / 128, ldc = (K + 15) / 16 * 16;
    at::Tensor codes = make_codes(M, K, ldc, x), scale = make({M, kb}, {1, M}, at::kFloat, x);
    if (vf4_cast_fp8_block(x.const_data_ptr(), code_of(x), M, K, ld, 1, static_cast<uint8_t*>(codes.mutable_data_ptr()), ldc,
                           static_cast<float*>(scale.mutable_data_ptr()), 1, M, stream(in.device)))
      return nullptr;
    g_launched = 1;
    return pair(like_x(codes, x0), like_x(scale, x0));
  });
}

// linear(x, w, w_scale, bias) -> y
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 4) return nullptr;
    Args in;
    const at::Tensor x0 = in.get(a[0]), x = rows_of(x0), w = in.get(a[1]), ws = in.get(a[2]), bias = in.get(a[3], true);
    int64_t ld, ldw;
    if (!in.ok || code_of(x) < 0 || !rows_ok(x, &ld) || w.scalar_type() != at::kFloat8_e4m3fn || !rows_ok(w, &ldw) ||
        ldw % 16 || reinterpret_cast<uintptr_t>(w.const_data_ptr()) % 16)
      return nullptr;
    const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
    if (w.size(1) != K || ws.dim() != 2 || ws.scalar_type() != at::kFloat || ws.size(0) != (N + 127) / 128 ||
        ws.size(1) != (K + 127) / 128 || !vector_ok(bias, N) || (bias.defined() && code_of(bias) < 0))
      return nullptr;
    at::Tensor y = make({M, N}, {N, 1}, x.scalar_type(), x), work;
    const int64_t need = vf4_linear_fp8_block_workspace_size(M, N, K);
    if (need) work = make({need}, {1}, at::kByte, x);
    if (vf4_linear_fp8_block(x.const_data_ptr(), code_of(x), M, K, ld, static_cast<const uint8_t*>(w.const_data_ptr()), ldw,
                             static_cast<const float*>(ws.const_data_ptr()), ws.stride(0), ws.stride(1), N, ptr(bias),
                             bias.defined() ? code_of(bias) : VF4_BF16, y.mutable_data_ptr(), N,
                             need ? work.mutable_data_ptr() : nullptr, need, stream(in.device)))
      return nullptr;
    g_launched = need ? 2 : 1;
    return THPVariable_Wrap(like_x(y, x0));
  });
}

// norm(x, y, gate, residual_scale, kind, post_w, post_b, pre_w, pre_b, eps, fp8) -> (x', h | (codes, scale)):
// both norms, of one kind (1 LayerNorm, 2 RMSNorm)
PyObject* norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 11) return nullptr;
    Args in;
    const at::Tensor x0 = in.get(a[0]), y0 = in.get(a[1]), x = rows_of(x0), y = rows_of(y0), gate = in.get(a[2], true);
    at::Tensor p[4];
    for (int i = 0; i < 4; ++i) p[i] = in.get(a[5 + i], true);
    const double rs = PyFloat_AsDouble(a[3]), eps = PyFloat_AsDouble(a[9]);
    const long kind = PyLong_AsLong(a[4]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      return nullptr;
    }
    if (kind != 1 && kind != 2) return nullptr;
    const bool fp8 = a[10] == Py_True;
    int64_t ldx, ldy;
    if (!in.ok || code_of(x) < 0 || !rows_ok(x, &ldx) || !rows_ok(y, &ldy) || y0.sizes() != x0.sizes() ||
        y.scalar_type() != x.scalar_type())
      return nullptr;
    const int64_t M = x.size(0), K = x.size(1), kb = (K + 127) / 128, ldc = (K + 15) / 16 * 16;
    int64_t groups = 1;
    int pcode = -1;
    if (gate.defined()) {
      if (gate.dim() < 1 || gate.dim() > 2 || gate.size(-1) != K || !gate.is_contiguous()) return nullptr;
      groups = gate.dim() == 1 ? 1 : gate.size(0);
      if (groups < 1 || M % groups) return nullptr;
      pcode = code_of(gate);
      if (pcode < 0) return nullptr;
    }
    for (const at::Tensor& t : p) {
      if (!t.defined()) continue;
      if (!vector_ok(t, K) || code_of(t) < 0 || (pcode >= 0 && code_of(t) != pcode)) return nullptr;
      pcode = code_of(t);
    }
    if (pcode < 0) pcode = code_of(x);
    if (pcode != VF4_F32 && pcode != code_of(x)) return nullptr;
    at::Tensor out = make({M, K}, {K, 1}, x.scalar_type(), x), h, scale;
    h = fp8 ? make_codes(M, K, ldc, x) : make({M, K}, {K, 1}, x.scalar_type(), x);
    if (fp8) scale = make({M, kb}, {1, M}, at::kFloat, x);
    if (vf4_gated_residual_norm(x.const_data_ptr(), ldx, y.const_data_ptr(), ldy, code_of(x), M, K, ptr(gate), groups,
                                (float)rs, (int)kind, ptr(p[0]), ptr(p[1]), (int)kind, ptr(p[2]), ptr(p[3]), pcode,
                                (float)eps, out.mutable_data_ptr(), h.mutable_data_ptr(), fp8, fp8 ? ldc : 0,
                                fp8 ? static_cast<float*>(scale.mutable_data_ptr()) : nullptr, 1, M, stream(in.device)))
      return nullptr;
    g_launched = 1;
    if (!fp8) return pair(like_x(out, x0), like_x(h, x0));
    PyObject* codes = pair(like_x(h, x0), like_x(scale, x0));
    PyObject* r = codes ? PyTuple_New(2) : nullptr;
    if (!r) {
      Py_XDECREF(codes);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(like_x(out, x0)));
    PyTuple_SET_ITEM(r, 1, codes);
    return r;
  });
}

// Stride of dimension d; of one with a single entry, whose stride may be anything, 0.
int64_t step(const at::Tensor& t, int d) { return t.size(d) > 1 ? t.stride(d) : 0; }

// cross(q, k, v, kv_lens, key_mask, scale | None) -> out: 4-D bf16 in layouts that the kernels read in place
PyObject* cross(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 6) return nullptr;
    Args in;
    const at::Tensor q = in.get(a[0]), k = in.get(a[1]), v = in.get(a[2]), lens = in.get(a[3], true), mask = in.get(a[4], true);
    if (!in.ok || q.dim() != 4) return nullptr;
    const int64_t B = q.size(0), H = q.size(1), Sq = q.size(2), D = q.size(3);
    for (const at::Tensor* t : {&q, &k, &v}) {
      if (t->scalar_type() != at::kBFloat16 || t->dim() != 4 || t->size(0) != B || t->size(3) != D || t->numel() == 0 ||
          t->stride(3) != 1 || ((step(*t, 0) | step(*t, 1) | step(*t, 2)) & 7) || (t->size(2) > 1 && t->stride(2) < D) ||
          (reinterpret_cast<uintptr_t>(t->const_data_ptr()) & 15))
        return nullptr;
    }
    const int64_t Hkv = k.size(1), Skv = k.size(2);
    if (v.size(1) != Hkv || v.size(2) != Skv || H % Hkv || D % 8 || D > 128) return nullptr;
    if (lens.defined() && (lens.dim() != 1 || lens.size(0) != B || lens.scalar_type() != at::kInt || !lens.is_contiguous())) return nullptr;
    if (mask.defined() && (mask.dim() != 2 || mask.size(0) != B || mask.size(1) != Skv || mask.scalar_type() != at::kBool ||
                           (mask.stride(1) != 1 && Skv > 1)))
      return nullptr;
    double scale = 1.0 / std::sqrt((double)D);
    if (a[5] != Py_None) {
      scale = PyFloat_AsDouble(a[5]);
      if (PyErr_Occurred()) {
        PyErr_Clear();
        return nullptr;
      }
    }
    if (!std::isfinite(scale)) return nullptr;
    at::Tensor out = make({B, H, Sq, D}, {Sq * H * D, D, H * D, 1}, at::kBFloat16, q), work;
    const int64_t need = vf4_cross_attn_workspace_size(B, H, Hkv, Sq, Skv, D);
    if (need) work = make({need}, {1}, at::kByte, q);
    if (vf4_cross_attn(q.const_data_ptr(), step(q, 0), step(q, 1), step(q, 2), k.const_data_ptr(), step(k, 0), step(k, 1),
                       step(k, 2), v.const_data_ptr(), step(v, 0), step(v, 1), step(v, 2), B, H, Hkv, Sq, Skv, D,
                       (float)scale, static_cast<const int32_t*>(ptr(lens)), static_cast<const uint8_t*>(ptr(mask)),
                       mask.defined() ? mask.stride(0) : 0, out.mutable_data_ptr(), Sq * H * D, D, H * D,
                       need ? work.mutable_data_ptr() : nullptr, need, stream(in.device)))
      return nullptr;
    g_launched = need ? 2 : 1;
    return THPVariable_Wrap(out);
  });
}

PyObject* launched(PyObject*, PyObject*) { return PyLong_FromLong(g_launched); }

PyMethodDef methods[] = {
    {"launched", launched, METH_NOARGS, nullptr},
    {"cast", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cast)), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear)), METH_FASTCALL, nullptr},
    {"norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(norm)), METH_FASTCALL, nullptr},
    {"cross", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cross)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// built_for: torch's release (its C++ interface); the package loads no module that names another.  Nothing of torch is
// called before that.
PyMODINIT_FUNC PyInit__fast(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for", VF4_BUILT_FOR)) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}

// CPython module over the library's MXFP4 entry points for torch tensors: looks at the arguments, makes the results and
// calls the C entry point, without the interpreter between these steps.  A decode-sized product takes the GPU less time
// than the same steps take in Python.
//
// The module computes nothing and knows no entry points but those of b200gemm.h.  What does not belong together
// raises ValueError, and so does a tensor whose gradient the call would drop; a failing entry point raises the
// exception type that capi.py hands over (B200Error).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>

#include "b200gemm.h"

namespace {

PyObject* g_error = nullptr;  // B200Error(status, message)

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return B200_F32;
    case at::kHalf: return B200_F16;
    case at::kBFloat16: return B200_BF16;
    default: return -1;
  }
}

// Spreads positional and keyword arguments over `names`; missing ones stay null.  False with an exception set.
bool spread(const char* fn, std::initializer_list<const char*> names, size_t required, PyObject* const* args, Py_ssize_t n,
            PyObject* kwnames, PyObject** out) {
  if (size_t(n) > names.size()) {
    PyErr_Format(PyExc_TypeError, "%s() takes at most %zu arguments (%zd given)", fn, names.size(), n);
    return false;
  }
  for (size_t i = 0; i < names.size(); ++i) out[i] = i < size_t(n) ? args[i] : nullptr;
  const Py_ssize_t nkw = kwnames ? PyTuple_GET_SIZE(kwnames) : 0;
  for (Py_ssize_t k = 0; k < nkw; ++k) {
    PyObject* name = PyTuple_GET_ITEM(kwnames, k);
    size_t i = 0;
    for (const char* have : names) {
      if (PyUnicode_CompareWithASCIIString(name, have) == 0) break;
      ++i;
    }
    if (i == names.size() || out[i]) {
      PyErr_Format(PyExc_TypeError, "%s() got an unexpected or repeated argument '%U'", fn, name);
      return false;
    }
    out[i] = args[n + k];
  }
  for (size_t i = 0; i < required; ++i)
    if (!out[i]) {
      PyErr_Format(PyExc_TypeError, "%s() misses argument '%s'", fn, *(names.begin() + i));
      return false;
    }
  return true;
}

PyObject* refuse(const char* text) {
  PyErr_SetString(PyExc_ValueError, text);
  return nullptr;
}

// Null for what is no tensor, and for one whose memory holds the negatives of its values (a view that torch resolves
// later, such as the imaginary part of a conjugate).
const at::Tensor* tensor(PyObject* o) {
  const at::Tensor* t = o && THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
  return t && !t->is_neg() ? t : nullptr;
}
bool given(PyObject* o) { return o && o != Py_None; }

// A packed matrix whose two tensors belong together: rows and K in whole blocks.
bool operand(PyObject* q_, PyObject* s_, const at::Tensor** q, const at::Tensor** s, int64_t* rows, int64_t* K) {
  *q = tensor(q_);
  *s = tensor(s_);
  if (!*q || !(*q)->is_cuda() || (*q)->scalar_type() != at::kByte || (*q)->dim() != 2 || !(*q)->is_contiguous() ||
      (*q)->size(0) == 0 || (*q)->size(1) == 0 || (*q)->size(1) % 16) {
    refuse("packed elements are a contiguous uint8 CUDA tensor [rows, whole blocks of 16 bytes]");
    return false;
  }
  *rows = (*q)->size(0);
  *K = 2 * (*q)->size(1);
  const at::Tensor* t = *s;
  if (!t || t->scalar_type() != at::kByte || t->dim() != 5 || t->size(0) != (*rows + 127) / 128 ||
      t->size(1) != (*K + 127) / 128 || t->size(2) != 32 || t->size(3) != 4 || t->size(4) != 4 || !t->is_contiguous() ||
      t->device() != (*q)->device()) {
    refuse("scales are a contiguous uint8 tensor [ceil(rows / 128), ceil(K / 128), 32, 4, 4] beside the packed elements");
    return false;
  }
  return true;
}

// The given result tensor, or a new one.
bool result(PyObject* given_out, int64_t rows, int64_t cols, at::ScalarType dtype, const at::Device& device, at::Tensor* out) {
  if (!given(given_out)) {
    *out = at::detail::empty_cuda({rows, cols}, dtype, device, std::nullopt);
    return true;
  }
  const at::Tensor* t = tensor(given_out);
  if (!t || t->scalar_type() != dtype || t->dim() != 2 || t->size(0) != rows || t->size(1) != cols || !t->is_contiguous() ||
      t->device() != device) {
    refuse("out: a contiguous tensor of the result's type and shape on the operands' device");
    return false;
  }
  *out = *t;
  return true;
}

// The operators have no derivative, and a result without one would end a gradient in silence: what autograd follows, or
// would follow into a given result, is refused.
bool untracked(std::initializer_list<const at::Tensor*> tensors) {
  for (const at::Tensor* t : tensors)
    if (t && ((c10::GradMode::is_enabled() && t->requires_grad()) || t->_fw_grad(0).defined())) {
      refuse("a tensor requires a gradient: the MXFP4 operators have none (call them on detached tensors or under torch.no_grad())");
      return false;
    }
  return true;
}

// A given result was written in place: autograd has to know, should it have kept the values for a backward pass.
void written(PyObject* given_out, const at::Tensor& out) {
  if (given(given_out) && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
}

// A given result that shares memory with an operand would be written while other CTAs still read it.
bool apart(const at::Tensor& out, std::initializer_list<const at::Tensor*> operands) {
  const auto begin = [](const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()); };
  for (const at::Tensor* t : operands)
    if (t && begin(*t) < begin(out) + out.nbytes() && begin(out) < begin(*t) + t->nbytes()) {
      refuse("out: must not share memory with an operand");
      return false;
    }
  return true;
}

// dtype argument: bf16 if not given.
bool wanted_dtype(PyObject* o, at::ScalarType* dtype) {
  *dtype = at::kBFloat16;
  if (!given(o)) return true;
  if (!THPDtype_Check(o) || dtype_code(reinterpret_cast<THPDtype*>(o)->scalar_type) < 0) {
    refuse("dtype: torch.float32, torch.float16 or torch.bfloat16");
    return false;
  }
  *dtype = reinterpret_cast<THPDtype*>(o)->scalar_type;
  return true;
}

// Runs `call(stream)` with the tensors' device current, on its current stream.  False with an exception set.
template <typename F>
bool run(const at::Device& device, F&& call) {
  int status;
  {
    c10::cuda::OptionalCUDAGuard guard;
    if (device.index() != c10::cuda::current_device()) guard.set_device(device);
    void* stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    PyThreadState* gil = PyEval_SaveThread();
    status = call(stream);
    PyEval_RestoreThread(gil);
  }
  if (status == B200_OK) return true;
  PyObject* e = g_error ? PyObject_CallFunction(g_error, "is", status, b200_last_error()) : nullptr;
  if (e) {
    PyErr_SetObject(g_error, e);
    Py_DECREF(e);
  } else if (!PyErr_Occurred()) {
    PyErr_SetString(PyExc_RuntimeError, b200_last_error());
  }
  return false;
}

PyObject* quantize_mxfp4(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
  HANDLE_TH_ERRORS
  PyObject* a[2];
  if (!spread("quantize_mxfp4", {"x", "along"}, 1, args, n, kw, a)) return nullptr;
  const at::Tensor* x = tensor(a[0]);
  const int code = x ? dtype_code(x->scalar_type()) : -1;
  if (code < 0 || !x->is_cuda() || x->dim() != 2) return refuse("x: a 2-D fp32, fp16 or bf16 CUDA tensor");
  const int64_t R = x->size(0), C = x->size(1);
  if (R == 0 || C == 0) return refuse("x: sizes must be positive");
  const int64_t ldx = R == 1 ? C : x->stride(0);
  if ((x->stride(1) != 1 && C != 1) || ldx < C)
    return refuse("x: the elements of a row must be neighbours, and rows must not overlap");
  if (!untracked({x})) return nullptr;
  long along = 0;
  if (a[1]) {
    along = PyLong_AsLong(a[1]);
    if (along == -1 && PyErr_Occurred()) return nullptr;
    if (along != 0 && along != 1) return refuse("along: 0 (blocks in rows) or 1 (blocks in columns)");
  }
  const int64_t rows = along ? C : R, K = along ? R : C;
  const at::Device device = x->device();
  at::Tensor q = at::detail::empty_cuda({rows, (K + 31) / 32 * 16}, at::kByte, device, std::nullopt);
  at::Tensor s = at::detail::empty_cuda({(rows + 127) / 128, (K + 127) / 128, 32, 4, 4}, at::kByte, device, std::nullopt);
  const void* px = x->const_data_ptr();
  void *pq = q.mutable_data_ptr(), *ps = s.mutable_data_ptr();
  if (!run(device, [&](void* st) { return b200_quantize_mxfp4(code, px, pq, ps, R, C, ldx, int(along), st); })) return nullptr;
  PyObject* pair = PyTuple_New(2);
  if (!pair) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(q)));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(s)));
  return pair;
  END_HANDLE_TH_ERRORS
}

PyObject* dequantize_mxfp4(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
  HANDLE_TH_ERRORS
  PyObject* a[5];
  if (!spread("dequantize_mxfp4", {"q", "scale", "K", "dtype", "out"}, 2, args, n, kw, a)) return nullptr;
  const at::Tensor *q, *s;
  int64_t rows, width;
  if (!operand(a[0], a[1], &q, &s, &rows, &width)) return nullptr;
  int64_t K = width;
  if (given(a[2])) {
    K = PyLong_AsLongLong(a[2]);
    if (K == -1 && PyErr_Occurred()) return nullptr;
    if (K <= width - 32 || K > width) return refuse("K: the row length that was quantised, in the last block of the packed rows");
  }
  at::ScalarType dtype;
  if (!wanted_dtype(a[3], &dtype)) return nullptr;
  const at::Device device = q->device();
  at::Tensor out;
  if (!result(a[4], rows, K, dtype, device, &out) || !untracked({&out}) || !apart(out, {q, s})) return nullptr;
  const void *pq = q->const_data_ptr(), *ps = s->const_data_ptr();
  void* po = out.mutable_data_ptr();
  if (!run(device, [&](void* st) { return b200_dequantize_mxfp4(dtype_code(dtype), pq, ps, po, rows, K, 0, st); })) return nullptr;
  written(a[4], out);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyObject* gemm_mxfp4(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
  HANDLE_TH_ERRORS
  PyObject* v[6];
  if (!spread("gemm_mxfp4", {"a", "a_scale", "b", "b_scale", "dtype", "out"}, 4, args, n, kw, v)) return nullptr;
  const at::Tensor *a, *sa, *b, *sb;
  int64_t M, N, K, K2;
  if (!operand(v[0], v[1], &a, &sa, &M, &K) || !operand(v[2], v[3], &b, &sb, &N, &K2)) return nullptr;
  const at::Device device = a->device();
  if (K != K2 || b->device() != device) return refuse("a and b do not fit: their inner dimensions or devices differ");
  at::ScalarType dtype;
  if (!wanted_dtype(v[4], &dtype)) return nullptr;
  at::Tensor out;
  if (!result(v[5], M, N, dtype, device, &out) || !untracked({&out}) || !apart(out, {a, sa, b, sb})) return nullptr;
  const void *pa = a->const_data_ptr(), *psa = sa->const_data_ptr(), *pb = b->const_data_ptr(), *psb = sb->const_data_ptr();
  void* po = out.mutable_data_ptr();
  if (!run(device, [&](void* st) { return b200_gemm_mxfp4(dtype_code(dtype), pa, psa, pb, psb, po, M, N, K, 0, st); }))
    return nullptr;
  written(v[5], out);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyObject* linear_mxfp4(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
  HANDLE_TH_ERRORS
  PyObject* v[6];
  if (!spread("linear_mxfp4", {"x", "w", "w_scale", "bias", "relu", "out"}, 3, args, n, kw, v)) return nullptr;
  const at::Tensor* x = tensor(v[0]);
  const int code = x ? dtype_code(x->scalar_type()) : -1;
  if (code < 0 || !x->is_cuda() || x->dim() != 2 || !x->is_contiguous() || x->size(0) == 0)
    return refuse("x: a contiguous 2-D fp32, fp16 or bf16 CUDA tensor");
  const int64_t batch = x->size(0), in_f = x->size(1);
  const at::Tensor *w, *sw;
  int64_t out_f, K;
  if (!operand(v[1], v[2], &w, &sw, &out_f, &K)) return nullptr;
  const at::Device device = x->device();
  if (in_f <= K - 32 || in_f > K || w->device() != device)
    return refuse("x and w do not fit: their inner dimensions or devices differ");
  const float* bias = nullptr;
  const at::Tensor* b = nullptr;
  if (given(v[3])) {
    b = tensor(v[3]);
    if (!b || b->scalar_type() != at::kFloat || b->dim() != 1 || b->size(0) != out_f || !b->is_contiguous() || b->device() != device)
      return refuse("bias: a contiguous fp32 tensor [out] on the operands' device");
    bias = static_cast<const float*>(b->const_data_ptr());
  }
  const int relu = v[4] ? PyObject_IsTrue(v[4]) : 0;
  if (relu < 0) return nullptr;
  at::Tensor out, ws;
  if (!result(v[5], batch, out_f, x->scalar_type(), device, &out) || !untracked({x, b, &out}) || !apart(out, {x, w, sw, b}))
    return nullptr;
  const size_t need = b200_linear_mxfp4_workspace(batch, in_f, out_f);
  void* pws = nullptr;
  if (need) {
    ws = at::detail::empty_cuda({int64_t(need)}, at::kByte, device, std::nullopt);
    pws = ws.mutable_data_ptr();
  }
  const void *px = x->const_data_ptr(), *pw = w->const_data_ptr(), *psw = sw->const_data_ptr();
  void* po = out.mutable_data_ptr();
  if (!run(device, [&](void* st) {
        return b200_linear_mxfp4(code, px, pw, psw, bias, po, batch, in_f, out_f, relu ? B200_LINEAR_RELU : 0, pws, need, st);
      }))
    return nullptr;
  written(v[5], out);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyObject* set_error(PyObject*, PyObject* type) {
  Py_XINCREF(type);
  Py_XSETREF(g_error, type);
  Py_RETURN_NONE;
}

#define ENTRY(name, text) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL | METH_KEYWORDS, text}
PyMethodDef g_methods[] = {
    ENTRY(quantize_mxfp4,
          "quantize_mxfp4(x, along=0)\n--\n\n"
          "x: [R, C] fp32, fp16 or bf16 CUDA tensor (rows may be strided) -> (q, scale) with blocks of 32 along the\n"
          "rows (along = 0: q is uint8 [R, 16 * ceil(C / 32)]) or down the columns (along = 1: the result is\n"
          "transposed, q is uint8 [C, 16 * ceil(R / 32)]).  scale: uint8 [bands of 128 rows, tiles of 4 blocks, 32, 4, 4],\n"
          "the byte of (row, block) at [row // 128, block // 4, row % 32, row % 128 // 32, block % 4]."),
    ENTRY(dequantize_mxfp4,
          "dequantize_mxfp4(q, scale, K=None, dtype=None, out=None)\n--\n\n"
          "(q, scale) -> [rows, K] values in `dtype` (bf16 if not given).  K: the row length that was quantised (whole\n"
          "blocks if not given)."),
    ENTRY(gemm_mxfp4,
          "gemm_mxfp4(a, a_scale, b, b_scale, dtype=None, out=None)\n--\n\n"
          "a [M, K] times b [N, K] transposed, both packed 4-bit, fp32 sums, result in `dtype` (bf16 if not given)."),
    ENTRY(linear_mxfp4,
          "linear_mxfp4(x, w, w_scale, bias=None, relu=False, out=None)\n--\n\n"
          "Fully connected layer on 4-bit weights: act(Q(x) @ W^T + bias), x [batch, in] fp32, fp16 or bf16 quantised\n"
          "along its rows on the way, (w, w_scale) the quantised [out, in] weights, bias fp32 [out].  relu is fmaxf(0, .): it\n"
          "makes 0 of NaN."),
    {"_set_error", set_error, METH_O, "The exception type of failing entry points, called with (status, message)."},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_torch_binding", "MXFP4 entry points of libb200gemm on torch tensors.", -1,
                        g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// The torch and the Python this was compiled for; the build looks for this text in the file.
const char g_built_for[] = "\0" B200_BUILT_FOR;

PyMODINIT_FUNC PyInit__torch_binding(void) {
  PyObject* module = PyModule_Create(&g_module);
  if (module && PyModule_AddStringConstant(module, "built_for", g_built_for + 1) < 0) {
    Py_DECREF(module);
    return nullptr;
  }
  return module;
}

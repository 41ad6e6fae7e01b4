// aklr_amd._host: the ops' per-call host work in native code, for the calls a serving loop makes.
//
// Each function takes a call's positional and keyword arguments as the op received them and returns its
// outputs, or None where the general Python path has to decide: a call outside the contract, a disabled or
// traced op, out=, trans_b=False, a tensor subclass, an active torch mode, a missing or unknown argument.
// It serves exactly what that path would serve, in the same way: the checks of aklr_amd/gemm.py, quant.py, rotary.py,
// kv_cache.py, attention.py, drafts.py, kv_pages.py and lora.py, then torch's allocator for outputs and scratch and the C ABI
// on the current stream.
// Nothing is kept between calls, and the GIL is released around allocation and launch.
//
// Why: a decode GEMM takes 3 to 20 us on the GPU, and its call took 12 to 17 us on the host (argument
// binding, about forty tensor attribute reads, two environment lookups, a ctypes call of 21 arguments), so
// a loop of layers was bound by Python. One quantizer call of 8 x 7168 12.4 -> 4.6 us, one GEMM call of
// 333 x 3072 x 1536 17.5 -> 7.6 (the GPU's time now), quantizer and MXFP4 GEMM of 8 x 10240 x 8192 31.0 -> 14.1.
#include <ATen/Context.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <initializer_list>
#include <optional>

#include "../../../include/aklr_amd.h"

namespace {

constexpr int64_t kMaxM = 1 << 20, kMaxN = 262144, kMaxK = 65536;              // aklr_amd/gemm.py
constexpr int64_t kMaxTokens = 131072, kMaxHidden = 21504, kMaxHidden4 = 65536;  // aklr_amd/quant.py

// The arguments of one call by parameter position, nullptr where not given. False: the general path binds
// them (and raises what it raises).
bool bind(PyObject* const* argv, Py_ssize_t argc, const char* const* names, int count, int positional, int required,
          PyObject** out) {
  if (argc != 2 || !PyTuple_CheckExact(argv[0]) || !PyDict_CheckExact(argv[1])) return false;
  for (int i = 0; i < count; ++i) out[i] = nullptr;
  const Py_ssize_t n = PyTuple_GET_SIZE(argv[0]);
  if (n > positional) return false;
  for (Py_ssize_t i = 0; i < n; ++i) out[i] = PyTuple_GET_ITEM(argv[0], i);
  PyObject *key, *value;
  Py_ssize_t pos = 0;
  while (PyDict_Next(argv[1], &pos, &key, &value)) {
    int at = -1;
    for (int i = 0; i < count && at < 0; ++i)
      if (PyUnicode_CompareWithASCIIString(key, names[i]) == 0) at = i;
    if (at < 0 || out[at]) return false;
    out[at] = value;
  }
  for (int i = 0; i < required; ++i)
    if (!out[i]) return false;
  return true;
}

bool set_and_not_zero(const char* name) {
  const char* v = std::getenv(name);
  return v && *v && std::strcmp(v, "0") != 0;
}

// Whether anything may look at, or change, what a call does: the general path's business.
bool watched() {
  return set_and_not_zero("AKLR_DISABLE") || set_and_not_zero("AKLR_TRACE") || at::impl::torch_function_mode_enabled() ||
         c10::impl::TorchDispatchModeTLS::any_modes_set() || at::globalContext().deterministicAlgorithms();
}

// A plain dense GPU tensor (no subclass, no functional wrapper).
const at::Tensor* dense(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || t.layout() != at::kStrided || !t.device().is_cuda() || !t.has_storage()) return nullptr;
  return t.unsafeGetTensorImpl()->is_python_dispatch() ? nullptr : &t;
}

bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0; }

// The same, 16-byte aligned.
const at::Tensor* plain(PyObject* o) {
  const at::Tensor* t = dense(o);
  return t && aligned16(*t) ? t : nullptr;
}

bool is_true_attr(PyObject* o, PyObject* name, bool* out) {
  PyObject* v = nullptr;
#if PY_VERSION_HEX >= 0x030D0000
  if (PyObject_GetOptionalAttr(o, name, &v) < 0) return false;
#else
  if (_PyObject_LookupAttr(o, name, &v) < 0) return false;  // the same function before it was public
#endif
  *out = v == Py_True;
  Py_XDECREF(v);
  return true;
}

PyObject *s_is_shuffled, *s_is_row_major;

bool str_is(PyObject* o, const char* s) { return PyUnicode_CheckExact(o) && PyUnicode_CompareWithASCIIString(o, s) == 0; }

bool is_none(PyObject* o) { return o == nullptr || o == Py_None; }

// block_size: the default, or a tuple of two ints equal to it
bool block_ok(PyObject* o) {
  if (!o) return true;
  if (!PyTuple_CheckExact(o) || PyTuple_GET_SIZE(o) != 2) return false;
  for (int i = 0; i < 2; ++i) {
    PyObject* v = PyTuple_GET_ITEM(o, i);
    if (!PyLong_CheckExact(v) || PyLong_AsLong(v) != 128) return PyErr_Clear(), false;
  }
  return true;
}

bool out_type(PyObject* o, at::ScalarType* t) {
  if (is_none(o)) return *t = at::kBFloat16, true;
  if (!THPDtype_Check(o)) return false;
  *t = reinterpret_cast<THPDtype*>(o)->scalar_type;
  return *t == at::kBFloat16 || *t == at::kHalf;
}

int out_code(at::ScalarType t) { return t == at::kBFloat16 ? AKLR_OUT_BF16 : AKLR_OUT_F16; }

hipStream_t stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

at::Tensor make(at::IntArrayRef size, at::ScalarType type, const at::Tensor& like) {
  return at::empty(size, at::TensorOptions().dtype(type).device(like.device()));
}

// The outputs of a launch, or the exception aklr_amd._lib.check raises for its status.
PyObject* status_error(int status, const char* what) {
  PyObject* m = PyImport_ImportModule("aklr_amd._lib");
  if (!m) return nullptr;
  PyObject* r = PyObject_CallMethod(m, "check", "is", status, what);
  Py_DECREF(m);
  if (r) {
    Py_DECREF(r);
    PyErr_Format(PyExc_RuntimeError, "%s: status %d", what, status);
  }
  return nullptr;
}

PyObject* pair(const at::Tensor& a, const at::Tensor& b) {
  PyObject* x = THPVariable_Wrap(a);
  PyObject* y = THPVariable_Wrap(b);
  PyObject* r = x && y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return r;
}

// ---------------------------------------------------------------------------------------------
// quantizers
const at::Tensor* activations(PyObject* o, int64_t multiple, int64_t max_hidden) {
  const at::Tensor* x = plain(o);
  if (!x || x->dim() != 2 || x->scalar_type() != at::kBFloat16 || !x->is_contiguous()) return nullptr;
  const int64_t t = x->size(0), h = x->size(1);
  return t >= 1 && t <= kMaxTokens && h >= multiple && h <= max_hidden && h % multiple == 0 ? x : nullptr;
}

PyObject* quant_fp8(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  static const char* const names[] = {"x"};
  PyObject* a[1];
  if (!bind(argv, argc, names, 1, 1, 1, a) || watched()) Py_RETURN_NONE;
  const at::Tensor* x = activations(a[0], 128, kMaxHidden);
  if (!x) Py_RETURN_NONE;
  const int64_t t = x->size(0), h = x->size(1);
  at::Tensor q, s;
  int st;
  {
    pybind11::gil_scoped_release no_gil;
    q = make({t, h}, at::kFloat8_e4m3fn, *x);
    s = make({h / 128, t}, at::kFloat, *x);
    st = aklr_per_group_quant_fp8(x->const_data_ptr(), h, q.mutable_data_ptr(), static_cast<float*>(s.mutable_data_ptr()),
                                  t, h, stream_of(*x));
  }
  return st == AKLR_OK ? pair(q, s) : status_error(st, "per_group_quant_fp8");
  END_HANDLE_TH_ERRORS
}

PyObject* quant_mxfp8(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  static const char* const names[] = {"x"};
  PyObject* a[1];
  if (!bind(argv, argc, names, 1, 1, 1, a) || watched()) Py_RETURN_NONE;
  const at::Tensor* x = activations(a[0], 32, kMaxHidden);
  if (!x) Py_RETURN_NONE;
  const int64_t t = x->size(0), h = x->size(1);
  at::Tensor q, s;
  int st;
  {
    pybind11::gil_scoped_release no_gil;
    q = make({t, h}, at::kFloat8_e4m3fn, *x);
    s = make({t, h / 32}, at::kByte, *x);
    st = aklr_per_group_quant_mxfp8(x->const_data_ptr(), h, q.mutable_data_ptr(),
                                    static_cast<uint8_t*>(s.mutable_data_ptr()), t, h, stream_of(*x));
  }
  return st == AKLR_OK ? pair(q, s) : status_error(st, "per_group_quant_mxfp8");
  END_HANDLE_TH_ERRORS
}

PyObject* quant_mxfp4(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  static const char* const names[] = {"x", "shuffle"};
  PyObject* a[2];
  if (!bind(argv, argc, names, 2, 2, 1, a) || watched()) Py_RETURN_NONE;
  if (a[1] && a[1] != Py_True && a[1] != Py_False) Py_RETURN_NONE;
  const bool shuffle = a[1] == Py_True;
  const at::Tensor* x = activations(a[0], 32, kMaxHidden4);
  if (!x) Py_RETURN_NONE;
  const int64_t t = x->size(0), h = x->size(1), g = h / 32;
  at::Tensor q, s;
  int st;
  {
    pybind11::gil_scoped_release no_gil;
    q = make({t, h / 2}, at::kFloat4_e2m1fn_x2, *x);
    s = make({shuffle ? (t + 255) / 256 * 256 : t, shuffle ? (g + 7) / 8 * 8 : g}, at::kFloat8_e8m0fnu, *x);
    st = aklr_dynamic_mxfp4_quant(x->const_data_ptr(), h, static_cast<uint8_t*>(q.mutable_data_ptr()),
                                  static_cast<uint8_t*>(s.mutable_data_ptr()), t, h,
                                  shuffle ? AKLR_SCALES_SHUFFLED : AKLR_SCALES_ROW_MAJOR, stream_of(*x));
  }
  return st == AKLR_OK ? pair(q, s) : status_error(st, "dynamic_mxfp4_quant");
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------
// GEMMs
bool gemm_dims(int64_t m, int64_t n, int64_t k, int64_t k_multiple) {
  return m >= 1 && m <= kMaxM && n >= 16 && n <= kMaxN && n % 16 == 0 && k >= k_multiple && k <= kMaxK && k % k_multiple == 0;
}

// bias: none, or fp32 [n] on the operands' device
bool bias_ok(PyObject* o, int64_t n, const at::Tensor& like, const float** data) {
  *data = nullptr;
  if (is_none(o)) return true;
  const at::Tensor* b = plain(o);
  if (!b || b->scalar_type() != at::kFloat || b->dim() != 1 || b->size(0) != n || !b->is_contiguous() ||
      b->device() != like.device())
    return false;
  *data = static_cast<const float*>(b->const_data_ptr());
  return true;
}

bool shape_is(const at::Tensor& t, int64_t r, int64_t c) { return t.dim() == 2 && t.size(0) == r && t.size(1) == c; }

PyObject* gemm_fp8(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  static const char* const names[] = {"a", "b", "a_scale", "b_scale", "block_size", "scale_major_mode", "trans_b",
                                      "bias", "out_dtype", "out", "operand_format"};
  PyObject* p[11];
  if (!bind(argv, argc, names, 11, 10, 4, p) || watched()) Py_RETURN_NONE;
  if (!block_ok(p[4]) || (p[6] && p[6] != Py_True) || !is_none(p[9])) Py_RETURN_NONE;
  const bool mn = p[5] && str_is(p[5], "MN");
  if (p[5] && !mn && !str_is(p[5], "K")) Py_RETURN_NONE;
  const bool pre = p[10] && str_is(p[10], "none:preshuffled");
  if (p[10] && !pre && !str_is(p[10], "none:none")) Py_RETURN_NONE;
  at::ScalarType ot;
  const at::Tensor *a = plain(p[0]), *b = plain(p[1]), *sa = plain(p[2]), *sb = plain(p[3]);
  if (!a || !b || !sa || !sb || !out_type(p[8], &ot)) Py_RETURN_NONE;
  bool shuffled = false, row_major_scale = false;
  if (!is_true_attr(p[1], s_is_shuffled, &shuffled) || !is_true_attr(p[2], s_is_row_major, &row_major_scale)) return nullptr;
  if (!pre && shuffled) Py_RETURN_NONE;
  const auto type = a->scalar_type();
  if ((type != at::kFloat8_e4m3fn && type != at::kFloat8_e5m2) || b->scalar_type() != type) Py_RETURN_NONE;
  if (pre && (mn || !is_none(p[7]) || type != at::kFloat8_e4m3fn)) Py_RETURN_NONE;
  if (sa->scalar_type() != at::kFloat || sb->scalar_type() != at::kFloat || a->dim() != 2 || b->dim() != 2) Py_RETURN_NONE;
  const int64_t m = a->size(0), k = a->size(1), n = b->size(0), kb = k / 128;
  if (b->size(1) != k || !gemm_dims(m, n, k, 128) || !a->is_contiguous() || !b->is_contiguous()) Py_RETURN_NONE;
  // preshuffled weights with a_scale not marked row-major: the column-major bytes in the logical shape
  const bool column_major = pre && !row_major_scale;
  if (!shape_is(*sa, mn ? kb : m, mn ? m : kb) || !sa->is_contiguous()) Py_RETURN_NONE;
  if (!shape_is(*sb, (n + 127) / 128, kb) || !sb->is_contiguous()) Py_RETURN_NONE;
  if (b->device() != a->device() || sa->device() != a->device() || sb->device() != a->device()) Py_RETURN_NONE;
  const float* bias;
  if (!bias_ok(p[7], n, *a, &bias)) Py_RETURN_NONE;
  at::Tensor out, ws;
  int st;
  {
    pybind11::gil_scoped_release no_gil;
    out = make({m, n}, ot, *a);
    const size_t bytes = aklr_gemm_a8w8_blockscale_workspace_bytes(m, n, k);
    if (bytes) ws = make({static_cast<int64_t>(bytes)}, at::kByte, *a);
    st = aklr_gemm_a8w8_blockscale(
        a->const_data_ptr(), a->stride(0), b->const_data_ptr(), pre ? k : b->stride(0),
        static_cast<const float*>(sa->const_data_ptr()),
        mn || column_major ? 1 : kb, mn || column_major ? m : 1, static_cast<const float*>(sb->const_data_ptr()),
        sb->stride(0), bias, out.mutable_data_ptr(), n, m, n, k,
        type == at::kFloat8_e4m3fn ? AKLR_FP8_E4M3FN : AKLR_FP8_E5M2, pre ? AKLR_B_PRESHUFFLE_16x16 : AKLR_B_ROW_MAJOR,
        out_code(ot), bytes ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(*a));
  }
  return st == AKLR_OK ? THPVariable_Wrap(out) : status_error(st, "gemm_a8w8_blockwise_scaled");
  END_HANDLE_TH_ERRORS
}

PyObject* quant_gemm_fp8(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  static const char* const names[] = {"x", "b", "b_scale", "bias", "out_dtype", "out", "operand_format"};
  PyObject* p[7];
  if (!bind(argv, argc, names, 7, 6, 3, p) || watched()) Py_RETURN_NONE;
  if (!is_none(p[5])) Py_RETURN_NONE;
  const bool pre = p[6] && str_is(p[6], "none:preshuffled");
  if (p[6] && !pre && !str_is(p[6], "none:none")) Py_RETURN_NONE;
  at::ScalarType ot;
  const at::Tensor *x = plain(p[0]), *b = plain(p[1]), *sb = plain(p[2]);
  if (!x || !b || !sb || !out_type(p[4], &ot)) Py_RETURN_NONE;
  bool shuffled = false;
  if (!is_true_attr(p[1], s_is_shuffled, &shuffled)) return nullptr;
  if (!pre && shuffled) Py_RETURN_NONE;
  if (x->scalar_type() != at::kBFloat16 || b->scalar_type() != at::kFloat8_e4m3fn || sb->scalar_type() != at::kFloat ||
      x->dim() != 2 || b->dim() != 2)
    Py_RETURN_NONE;
  const int64_t m = x->size(0), k = x->size(1), n = b->size(0);
  if (b->size(1) != k || !gemm_dims(m, n, k, 128)) Py_RETURN_NONE;
  if (!shape_is(*sb, (n + 127) / 128, k / 128) || !sb->is_contiguous() || !b->is_contiguous()) Py_RETURN_NONE;
  if (x->stride(1) != 1 || x->stride(0) < k || x->stride(0) % 8 != 0) Py_RETURN_NONE;
  if (b->device() != x->device() || sb->device() != x->device()) Py_RETURN_NONE;
  const float* bias;
  if (!bias_ok(p[3], n, *x, &bias)) Py_RETURN_NONE;
  at::Tensor out, ws;
  int st;
  {
    pybind11::gil_scoped_release no_gil;
    out = make({m, n}, ot, *x);
    const size_t bytes = aklr_quant_gemm_a8w8_blockscale_workspace_bytes(m, n, k);
    if (bytes) ws = make({static_cast<int64_t>(bytes)}, at::kByte, *x);
    st = aklr_quant_gemm_a8w8_blockscale(x->const_data_ptr(), x->stride(0), b->const_data_ptr(),
                                         pre ? k : b->stride(0), static_cast<const float*>(sb->const_data_ptr()), sb->stride(0), bias,
                                         out.mutable_data_ptr(), n, m, n, k,
                                         pre ? AKLR_B_PRESHUFFLE_16x16 : AKLR_B_ROW_MAJOR, out_code(ot),
                                         bytes ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(*x));
  }
  return st == AKLR_OK ? THPVariable_Wrap(out) : status_error(st, "quant_gemm_a8w8_blockwise_scaled");
  END_HANDLE_TH_ERRORS
}

bool float_is(PyObject* o, double v) { return !o || (PyFloat_CheckExact(o) && PyFloat_AS_DOUBLE(o) == v); }

PyObject* gemm_mxfp4(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  static const char* const names[] = {"a", "b", "a_scale", "b_scale", "alpha", "beta", "trans_b", "bias", "out_dtype",
                                      "out", "operand_format"};
  PyObject* p[11];
  if (!bind(argv, argc, names, 11, 10, 4, p) || watched()) Py_RETURN_NONE;
  if (!float_is(p[4], 1.0) || !float_is(p[5], 0.0) || (p[6] && p[6] != Py_True) || !is_none(p[9])) Py_RETURN_NONE;
  const bool pre = !p[10] || str_is(p[10], "none:preshuffled");
  if (!pre && !str_is(p[10], "none:none")) Py_RETURN_NONE;
  at::ScalarType ot;
  const at::Tensor *a = plain(p[0]), *b = plain(p[1]), *sa = plain(p[2]), *sb = plain(p[3]);
  if (!a || !b || !sa || !sb || !out_type(p[8], &ot)) Py_RETURN_NONE;
  const auto code = [](const at::Tensor& t) { return t.scalar_type() == at::kFloat4_e2m1fn_x2 || t.scalar_type() == at::kByte; };
  const auto scale = [](const at::Tensor& t) { return t.scalar_type() == at::kFloat8_e8m0fnu || t.scalar_type() == at::kByte; };
  if (!code(*a) || !code(*b) || !scale(*sa) || !scale(*sb) || a->dim() != 2 || b->dim() != 2) Py_RETURN_NONE;
  const int64_t m = a->size(0), kh = a->size(1), n = b->size(0), k = 2 * kh, g = k / 32;
  if (b->size(1) != kh || !gemm_dims(m, n, k, 64)) Py_RETURN_NONE;
  const int64_t cols = pre ? (g + 7) / 8 * 8 : g;
  if (!shape_is(*sa, pre ? (m + 255) / 256 * 256 : m, cols) || !shape_is(*sb, pre ? (n + 255) / 256 * 256 : n, cols)) Py_RETURN_NONE;
  for (const at::Tensor* t : {a, b, sa, sb})
    if (!t->is_contiguous() || t->device() != a->device()) Py_RETURN_NONE;
  const float* bias;
  if (!bias_ok(p[7], n, *a, &bias)) Py_RETURN_NONE;
  at::Tensor out, ws;
  int st;
  {
    pybind11::gil_scoped_release no_gil;
    out = make({m, n}, ot, *a);
    const size_t bytes = aklr_gemm_a4w4_mxfp4_workspace_bytes(m, n, k);
    if (bytes) ws = make({static_cast<int64_t>(bytes)}, at::kByte, *a);
    const auto u8 = [](const at::Tensor& t) { return static_cast<const uint8_t*>(t.const_data_ptr()); };
    st = aklr_gemm_a4w4_mxfp4(u8(*a), a->stride(0), u8(*b), b->stride(0), u8(*sa), sa->stride(0), u8(*sb), sb->stride(0),
                              bias, out.mutable_data_ptr(), n, m, n, k,
                              pre ? AKLR_B_PRESHUFFLE_16x16 : AKLR_B_ROW_MAJOR,
                              pre ? AKLR_SCALES_SHUFFLED : AKLR_SCALES_ROW_MAJOR, out_code(ot),
                              bytes ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(*a));
  }
  return st == AKLR_OK ? THPVariable_Wrap(out) : status_error(st, "gemm_a4w4_mxfp4");
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------
// rotary positions, FP8 cache, attention over it: the checks of aklr_amd/rotary.py, kv_cache.py and attention.py
using Tensor = at::Tensor;

int64_t span(const Tensor& t, int64_t from) {
  int64_t n = 1;
  for (int64_t d = from; d < t.dim(); ++d) n += (t.size(d) - 1) * t.stride(d);
  return n * t.element_size();
}

bool apart(const Tensor* a, const Tensor* b) {
  if (!a || !b || a->numel() == 0 || b->numel() == 0) return true;
  const int64_t pa = reinterpret_cast<int64_t>(a->const_data_ptr()), pb = reinterpret_cast<int64_t>(b->const_data_ptr());
  if (pa + span(*a, 0) <= pb || pb + span(*b, 0) <= pa) return true;
  if (a->dim() < 2 || b->dim() < 2) return false;
  const int64_t row = a->stride(0) * a->element_size();
  if (row == 0 || row != b->stride(0) * b->element_size()) return false;
  const int64_t gap = ((pb - pa) % row + row) % row;
  return span(*a, 1) <= gap && gap + span(*b, 1) <= row;
}

bool apart_all(const Tensor* a, std::initializer_list<const Tensor*> others) {
  return std::all_of(others.begin(), others.end(), [a](const Tensor* b) { return apart(a, b); });
}

bool same_place(const Tensor& a, const Tensor& b) {
  return a.const_data_ptr() == b.const_data_ptr() && a.sizes() == b.sizes() && a.strides() == b.strides() &&
         a.scalar_type() == b.scalar_type();
}

bool no_inner_overlap(const Tensor& t) {
  int64_t reach = 1, done = 0;  // dimensions by ascending stride
  for (int64_t n = 0; n < t.dim(); ++n) {
    int64_t at = -1;
    for (int64_t d = 0; d < t.dim(); ++d)
      if (t.size(d) > 1 && !(done >> d & 1) && (at < 0 || t.stride(d) < t.stride(at))) at = d;
    if (at < 0) break;
    done |= int64_t{1} << at;
    if (t.stride(at) < reach) return false;
    reach += (t.size(at) - 1) * t.stride(at);
  }
  return true;
}

bool wants_grad(const Tensor* t) {
  return t && ((t->requires_grad() && c10::GradMode::is_enabled()) || t->_fw_grad(/*level=*/0).defined());
}

int float_code(at::ScalarType t) {
  return t == at::kBFloat16 ? AKLR_OUT_BF16 : t == at::kHalf ? AKLR_OUT_F16 : t == at::kFloat ? AKLR_F32 : -1;
}

bool vectors_ok(const Tensor& t, int64_t tokens, int64_t heads, int64_t dim, at::ScalarType type) {
  if (t.dim() != 3 || t.size(0) != tokens || t.size(1) != heads || t.size(2) != dim || t.scalar_type() != type) return false;
  const int64_t size = t.element_size();
  return t.stride(2) == 1 && aligned16(t) && t.stride(0) * size % 16 == 0 && t.stride(1) * size % 16 == 0;
}

bool index_ok(const Tensor& t, int64_t n) {
  return (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) && t.dim() == 1 && t.size(0) == n && t.is_contiguous();
}

bool flag(PyObject* o, bool* out) {
  *out = o == Py_True;
  return !o || o == Py_True || o == Py_False;
}

bool number(PyObject* o, double* out) {
  if (!o) return true;
  if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return false;
  *out = PyFloat_AsDouble(o);
  if (PyErr_Occurred()) return PyErr_Clear(), false;
  return std::fabs(*out) <= 0x1p127;  // what fp32 holds, with room for a factor of log2(e)
}

struct Turn {  // what a rotation takes beside its vectors
  const Tensor *positions, *frequencies;
  bool interleaved;
  double magnitude = 1.0;
  int64_t rot;
  bool read(PyObject* pos, PyObject* freq, PyObject* inter, PyObject* mag, int64_t tokens, int64_t dim) {
    positions = dense(pos);
    frequencies = dense(freq);
    if (!positions || !frequencies || !flag(inter, &interleaved) || !number(mag, &magnitude)) return false;
    if (!index_ok(*positions, tokens) || frequencies->scalar_type() != at::kDouble || frequencies->dim() != 1 ||
        !frequencies->is_contiguous() || wants_grad(frequencies))
      return false;
    rot = 2 * frequencies->numel();
    return rot >= 16 && rot <= dim && rot % 16 == 0;
  }
};

struct Cache {
  const Tensor* t[4];  // k codes, v codes, k scales, v scales
  int64_t step[4];
  int64_t pages, heads, page, dim;
  bool read(PyObject* const* o) {
    for (int i = 0; i < 4; ++i)
      if (!(t[i] = plain(o[i])) || t[i]->dim() != (i < 2 ? 4 : 3) || t[i]->device() != t[0]->device() ||
          t[i]->scalar_type() != (i < 2 ? at::kFloat8_e4m3fn : at::kFloat) || wants_grad(t[i]))
        return false;
    pages = t[0]->size(0), heads = t[0]->size(1), page = t[0]->size(2), dim = t[0]->size(3);
    if ((dim != 64 && dim != 128 && dim != 256) || page < 16 || page > 1024 || page % 16 || heads < 1 || heads > 1024 ||
        pages < 1 || pages * page >= (int64_t{1} << 31))
      return false;
    for (int i = 0; i < 4; ++i) {
      if (!(i < 2 ? t[i]->sizes() == t[0]->sizes() : t[i]->sizes() == t[0]->sizes().slice(0, 3))) return false;
      int64_t inner = 1;
      for (int64_t d = t[i]->dim() - 1; d > 0; --d) {
        if (t[i]->size(d) != 1 && t[i]->stride(d) != inner) return false;
        inner *= t[i]->size(d);
      }
      step[i] = pages == 1 ? inner : t[i]->stride(0);
      if (step[i] < inner || step[i] % (i < 2 ? 16 : 4)) return false;
    }
    return true;
  }
  bool clear_of(const Tensor* x) const { return apart_all(x, {t[0], t[1], t[2], t[3]}); }
  float* scales(int i) const { return static_cast<float*>(t[i]->mutable_data_ptr()); }
};

bool starts_ok(const Tensor& t) { return t.scalar_type() == at::kInt && t.dim() == 1 && t.numel() >= 1 && t.is_contiguous(); }

bool table_ok(const Tensor& t, int64_t batch) {
  return t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) == batch && (t.size(1) <= 1 || t.stride(1) == 1) &&
         (batch <= 1 || t.stride(0) >= t.size(1));
}

int64_t table_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

template <typename... T>
bool one_device(const Tensor& first, T... rest) {
  return (... && (!rest || rest->device() == first.device()));
}

// An output that the caller gave (or none): its place, or a new one.
bool given(PyObject* o, const Tensor** t) {
  *t = nullptr;
  return is_none(o) || (*t = dense(o)) != nullptr;
}

const void* at_or_null(const Tensor* t) { return t ? t->const_data_ptr() : nullptr; }

PyObject* rotary(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  static const char* const names[] = {"q", "k", "positions", "frequencies", "interleaved", "magnitude", "out_q", "out_k"};
  PyObject* p[8];
  if (!bind(argv, argc, names, 8, 4, 4, p) || watched()) Py_RETURN_NONE;
  const Tensor *q = dense(p[0]), *k, *oq, *ok;
  if (!q || !given(p[1], &k) || !given(p[6], &oq) || !given(p[7], &ok) || (!k && ok) || q->dim() != 3) Py_RETURN_NONE;
  const int64_t tokens = q->size(0), heads = q->size(1), dim = q->size(2);
  const auto type = q->scalar_type();
  if (float_code(type) < 0 || heads < 1 || heads > 32768 || dim < 16 || dim > 1024 || dim % 16 || tokens < 1 ||
      tokens >= (int64_t{1} << 31) || !vectors_ok(*q, tokens, heads, dim, type))
    Py_RETURN_NONE;
  if (k && (k->dim() != 3 || k->size(1) < 1 || k->size(1) > 32768 || !vectors_ok(*k, tokens, k->size(1), dim, type))) Py_RETURN_NONE;
  Turn turn;
  if (!turn.read(p[2], p[3], p[4], p[5], tokens, dim)) Py_RETURN_NONE;
  for (const Tensor* t : {q, k, oq, ok})
    if (wants_grad(t)) Py_RETURN_NONE;
  if (!one_device(*q, k, turn.positions, turn.frequencies, oq, ok)) Py_RETURN_NONE;
  for (int i = 0; i < 2; ++i) {
    const Tensor *out = i ? ok : oq, *like = i ? k : q, *other = i ? q : k;
    if (!out) continue;
    if (!vectors_ok(*out, tokens, like->size(1), dim, type) || !no_inner_overlap(*out)) Py_RETURN_NONE;
    if (!apart_all(out, {other, turn.positions, turn.frequencies}) || !(same_place(*out, *like) || apart(out, like))) Py_RETURN_NONE;
  }
  if (!apart(oq, ok)) Py_RETURN_NONE;
  Tensor a, b;
  int st;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::DeviceGuard on(q->device());
    a = oq ? *oq : make(q->sizes(), type, *q);
    if (k) b = ok ? *ok : make(k->sizes(), type, *q);
    st = aklr_rotary_embedding(q->const_data_ptr(), q->stride(0), q->stride(1), a.mutable_data_ptr(), a.stride(0), a.stride(1),
                               heads, at_or_null(k), k ? k->stride(0) : 0, k ? k->stride(1) : 0,
                               k ? b.mutable_data_ptr() : nullptr, k ? b.stride(0) : 0, k ? b.stride(1) : 0,
                               k ? k->size(1) : 0, turn.positions->const_data_ptr(), turn.positions->scalar_type() == at::kLong,
                               static_cast<const double*>(turn.frequencies->const_data_ptr()), tokens, dim, turn.rot,
                               turn.interleaved, static_cast<float>(turn.magnitude), float_code(type), stream_of(*q));
  }
  if (st != AKLR_OK) return status_error(st, "rotary_embedding");
  PyObject* x = oq ? (Py_INCREF(p[6]), p[6]) : THPVariable_Wrap(a);
  PyObject* y = !k ? (Py_INCREF(Py_None), Py_None) : ok ? (Py_INCREF(p[7]), p[7]) : THPVariable_Wrap(b);
  PyObject* r = x && y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return r;
  END_HANDLE_TH_ERRORS
}

// Both writes: with q, rotated.
PyObject* write_cache(PyObject* qo, PyObject* ko, PyObject* vo, PyObject* const* cache_objects, PyObject* slots_object,
                      PyObject* const* turn_objects, PyObject* out_object, const char* what) {
  Cache c;
  const Tensor *q = nullptr, *out = nullptr, *k = dense(ko), *v = dense(vo), *slots = dense(slots_object);
  if (!k || !v || !slots || !c.read(cache_objects) || k->dim() != 3) Py_RETURN_NONE;
  const int64_t tokens = k->size(0);
  const auto type = k->scalar_type();
  if (float_code(type) < 0 || tokens < 1 || tokens >= (int64_t{1} << 31) || !vectors_ok(*k, tokens, c.heads, c.dim, type) ||
      !vectors_ok(*v, tokens, c.heads, c.dim, type) || !index_ok(*slots, tokens))
    Py_RETURN_NONE;
  if (!one_device(*k, v, slots, c.t[0]) || wants_grad(k) || wants_grad(v)) Py_RETURN_NONE;
  for (const Tensor* t : {k, v, slots})
    if (!c.clear_of(t)) Py_RETURN_NONE;
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < i; ++j)
      if (!apart(c.t[i], c.t[j])) Py_RETURN_NONE;
  Turn turn{};
  if (qo) {
    q = dense(qo);
    if (!q || !given(out_object, &out) || q->dim() != 3 || q->size(1) < 1 || q->size(1) > 32768 ||
        !vectors_ok(*q, tokens, q->size(1), c.dim, type))
      Py_RETURN_NONE;
    if (!turn.read(turn_objects[0], turn_objects[1], turn_objects[2], turn_objects[3], tokens, c.dim) || wants_grad(q) || wants_grad(out))
      Py_RETURN_NONE;
    if (!one_device(*k, q, turn.positions, turn.frequencies, out)) Py_RETURN_NONE;
    for (const Tensor* t : {q, turn.positions, turn.frequencies, out})
      if (t && !c.clear_of(t)) Py_RETURN_NONE;
    if (out) {
      if (!vectors_ok(*out, tokens, q->size(1), c.dim, type) || !no_inner_overlap(*out)) Py_RETURN_NONE;
      if (!(same_place(*out, *q) || apart(out, q)) || !apart_all(out, {k, v, turn.positions, turn.frequencies, slots})) Py_RETURN_NONE;
    }
  }
  Tensor a;
  int st;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::DeviceGuard on(k->device());
    if (q) a = out ? *out : make(q->sizes(), type, *q);
    st = aklr_kv_cache_write_fp8(
        at_or_null(q), q ? q->stride(0) : 0, q ? q->stride(1) : 0, q ? a.mutable_data_ptr() : nullptr, q ? a.stride(0) : 0,
        q ? a.stride(1) : 0, q ? q->size(1) : 0, k->const_data_ptr(), k->stride(0), k->stride(1), v->const_data_ptr(),
        v->stride(0), v->stride(1), at_or_null(turn.positions), q && turn.positions->scalar_type() == at::kLong,
        static_cast<const double*>(at_or_null(turn.frequencies)), turn.rot, turn.interleaved,
        static_cast<float>(turn.magnitude), slots->const_data_ptr(), slots->scalar_type() == at::kLong,
        c.t[0]->mutable_data_ptr(), c.t[1]->mutable_data_ptr(), c.scales(2), c.scales(3), c.step[0], c.step[1], c.step[2],
        c.step[3], tokens, c.heads, c.dim, c.pages, c.page, float_code(type), stream_of(*k));
  }
  if (st != AKLR_OK) return status_error(st, what);
  if (!q) return PyTuple_Pack(4, cache_objects[0], cache_objects[1], cache_objects[2], cache_objects[3]);
  if (out) return Py_INCREF(out_object), out_object;
  return THPVariable_Wrap(a);
}

PyObject* kv_write(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  static const char* const names[] = {"k", "v", "k_cache", "v_cache", "k_scale", "v_scale", "slots"};
  PyObject* p[7];
  if (!bind(argv, argc, names, 7, 7, 7, p) || watched()) Py_RETURN_NONE;
  return write_cache(nullptr, p[0], p[1], p + 2, p[6], nullptr, nullptr, "kv_cache_write_fp8");
  END_HANDLE_TH_ERRORS
}

PyObject* rotary_kv_write(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  static const char* const names[] = {"q", "k", "v", "positions", "frequencies", "k_cache", "v_cache", "k_scale", "v_scale",
                                      "slots", "interleaved", "magnitude", "out"};
  PyObject* p[13];
  if (!bind(argv, argc, names, 13, 10, 10, p) || watched()) Py_RETURN_NONE;
  PyObject* const turn[] = {p[3], p[4], p[10], p[11]};
  return write_cache(p[0], p[1], p[2], p + 5, p[9], turn, p[12], "rotary_kv_cache_write_fp8");
  END_HANDLE_TH_ERRORS
}

PyObject* kv_read(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  static const char* const names[] = {"k_cache", "v_cache", "k_scale", "v_scale", "block_table", "starts", "total",
                                      "out_dtype", "out_k", "out_v"};
  PyObject* p[10];
  if (!bind(argv, argc, names, 10, 7, 7, p) || watched()) Py_RETURN_NONE;
  Cache c;
  at::ScalarType type;
  const Tensor *table = dense(p[4]), *starts = dense(p[5]);
  if (!table || !starts || !c.read(p) || !is_none(p[8]) || !is_none(p[9]) || !out_type(p[7], &type) || !PyLong_CheckExact(p[6]))
    Py_RETURN_NONE;
  const int64_t total = PyLong_AsLongLong(p[6]);
  if (total < 1 || total >= (int64_t{1} << 31)) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  if (!starts_ok(*starts) || !table_ok(*table, starts->numel() - 1) || !one_device(*c.t[0], table, starts)) Py_RETURN_NONE;
  Tensor k, v;
  int st;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::DeviceGuard on(c.t[0]->device());
    k = make({total, c.heads, c.dim}, type, *c.t[0]);
    v = make({total, c.heads, c.dim}, type, *c.t[0]);
    st = aklr_kv_cache_read_fp8(c.t[0]->const_data_ptr(), c.t[1]->const_data_ptr(), c.scales(2), c.scales(3), c.step[0],
                                c.step[1], c.step[2], c.step[3], static_cast<const int32_t*>(table->const_data_ptr()),
                                table_stride(*table), table->size(1), static_cast<const int32_t*>(starts->const_data_ptr()),
                                starts->numel() - 1, total, k.mutable_data_ptr(), v.mutable_data_ptr(), c.heads, c.dim,
                                c.pages, c.page, out_code(type), stream_of(*c.t[0]));
  }
  return st == AKLR_OK ? pair(k, v) : status_error(st, "kv_cache_read_fp8");
  END_HANDLE_TH_ERRORS
}

PyObject* tree_attention(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  static const char* const names[] = {"q", "k_cache", "v_cache", "k_scale", "v_scale", "block_table", "seq_lens", "starts",
                                      "tree_mask", "softmax_scale", "return_lse", "out"};
  PyObject* p[12];
  if (!bind(argv, argc, names, 12, 9, 8, p) || watched()) Py_RETURN_NONE;
  Cache c;
  bool with_lse;
  double scale = 0;
  const Tensor *q = dense(p[0]), *table = dense(p[5]), *lens = dense(p[6]), *starts = dense(p[7]), *mask, *out;
  if (!q || !table || !lens || !starts || !c.read(p + 1) || !given(p[8], &mask) || !given(p[11], &out) || !flag(p[10], &with_lse) ||
      q->dim() != 3)
    Py_RETURN_NONE;
  const int64_t tokens = q->size(0), heads = q->size(1), dim = q->size(2), batch = lens->numel();
  const auto type = q->scalar_type();
  if ((type != at::kBFloat16 && type != at::kHalf) || dim != c.dim || heads < c.heads || heads % c.heads || heads > 65536 ||
      tokens < 1 || batch < 1 || !vectors_ok(*q, tokens, heads, dim, type) || tokens * heads >= (int64_t{1} << 28))
    Py_RETURN_NONE;
  if (lens->scalar_type() != at::kInt || lens->dim() != 1 || !lens->is_contiguous() || batch > 65536 || !starts_ok(*starts) ||
      starts->numel() != batch + 1 || !table_ok(*table, batch) || table->size(1) * c.page > (int64_t{1} << 28) ||
      c.step[0] != c.step[1] || c.step[2] != c.step[3] || c.step[0] >= (int64_t{1} << 32) || c.step[2] >= (int64_t{1} << 30))
    Py_RETURN_NONE;
  if (mask && ((mask->scalar_type() != at::kBool && mask->scalar_type() != at::kByte) || mask->dim() != 2 ||
               mask->size(0) != tokens || (mask->size(1) > 1 && mask->stride(1) != 1)))
    Py_RETURN_NONE;
  if (is_none(p[9]))
    scale = 1 / std::sqrt(static_cast<double>(dim));
  else if (!number(p[9], &scale))
    Py_RETURN_NONE;
  if (!one_device(*q, c.t[0], table, lens, starts, mask, out) || wants_grad(q) || wants_grad(out)) Py_RETURN_NONE;
  if (out && (out->sizes() != q->sizes() || out->scalar_type() != type || !out->is_contiguous() || !aligned16(*out) ||
              !c.clear_of(out) || !apart_all(out, {q, table, lens, starts, mask})))
    Py_RETURN_NONE;
  if (!aklr_tree_attention_fp8_rows(tokens, batch, heads, c.heads, dim, table->size(1) * c.page, nullptr)) Py_RETURN_NONE;
  Tensor o, l, ws;
  int st;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::DeviceGuard on(q->device());
    o = out ? *out : make({tokens, heads, dim}, type, *q);
    if (with_lse) l = make({tokens, heads}, at::kFloat, *q);
    const size_t bytes = aklr_tree_attention_fp8_workspace_bytes(tokens, batch, heads, c.heads, dim, table->size(1) * c.page);
    if (bytes) ws = make({static_cast<int64_t>(bytes)}, at::kByte, *q);
    const auto ints = [](const Tensor* t) { return static_cast<const int32_t*>(t->const_data_ptr()); };
    st = aklr_tree_attention_fp8(q->const_data_ptr(), q->stride(0), q->stride(1), c.t[0]->const_data_ptr(),
                                 c.t[1]->const_data_ptr(), c.scales(2), c.scales(3), c.step[0], c.step[2], ints(table),
                                 table_stride(*table), table->size(1), ints(lens), ints(starts),
                                 at_or_null(mask), mask ? mask->stride(0) : 0, mask ? mask->size(1) : 0, o.mutable_data_ptr(),
                                 with_lse ? static_cast<float*>(l.mutable_data_ptr()) : nullptr, tokens, batch, heads, c.heads,
                                 dim, c.pages, c.page, static_cast<float>(scale), out_code(type),
                                 bytes ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(*q));
  }
  if (st != AKLR_OK) return status_error(st, "tree_attention_fp8");
  PyObject* x = out ? (Py_INCREF(p[11]), p[11]) : THPVariable_Wrap(o);
  if (!with_lse || !x) return x;
  PyObject* y = THPVariable_Wrap(l);
  PyObject* r = y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_DECREF(x);
  Py_XDECREF(y);
  return r;
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------
// drafted tokens, pages of the cache, adapters: the checks of aklr_amd/drafts.py, kv_pages.py and lora.py
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

bool rows_ok(const Tensor& t) {
  return t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1) && row_stride(t) >= t.size(1) &&
         reinterpret_cast<uintptr_t>(t.const_data_ptr()) % t.element_size() == 0;
}

bool vector_ok(const Tensor& t, int64_t n, at::ScalarType type) {
  return t.scalar_type() == type && t.dim() == 1 && t.size(0) == n && t.is_contiguous();
}

bool whole(PyObject* o, int64_t least, int64_t most, int64_t* out) {
  if (!PyLong_CheckExact(o)) return false;
  *out = PyLong_AsLongLong(o);
  if (*out == -1 && PyErr_Occurred()) return PyErr_Clear(), false;
  return *out >= least && *out <= most;
}

const int32_t* ints(const Tensor* t) { return t ? static_cast<const int32_t*>(t->const_data_ptr()) : nullptr; }
const float* floats(const Tensor* t) { return t ? static_cast<const float*>(t->const_data_ptr()) : nullptr; }

at::Tensor scratch(size_t bytes, const Tensor& like) {
  return bytes ? make({static_cast<int64_t>(bytes)}, at::kByte, like) : at::Tensor();
}
void* data_or_null(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

PyObject* tuple_of(std::initializer_list<const Tensor*> ts) {
  PyObject* r = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  if (!r) return nullptr;
  Py_ssize_t i = 0;
  for (const Tensor* t : ts) {
    PyObject* o = THPVariable_Wrap(*t);
    if (!o) return Py_DECREF(r), nullptr;
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

PyObject* verify(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  static const char* const names[] = {"target_probs", "draft_tokens", "starts", "accept_uniforms", "sample_uniforms",
                                      "most", "draft_probs", "parents"};
  PyObject* p[8];
  if (!bind(argv, argc, names, 8, 6, 6, p) || watched()) Py_RETURN_NONE;
  const Tensor *target = dense(p[0]), *tokens = dense(p[1]), *starts = dense(p[2]), *accept = dense(p[3]),
               *sample = dense(p[4]), *draft, *parents;
  int64_t most;
  if (!target || !tokens || !starts || !accept || !sample || !given(p[6], &draft) || !given(p[7], &parents) ||
      !whole(p[5], 1, 1024, &most) || !rows_ok(*target))
    Py_RETURN_NONE;
  const int64_t n = target->size(0), vocab = target->size(1);
  const auto type = target->scalar_type();
  if (float_code(type) < 0 || n < 1 || n >= (int64_t{1} << 31) || vocab < 8 || vocab > (1 << 24) || !starts_ok(*starts)) Py_RETURN_NONE;
  const int64_t batch = starts->numel() - 1;
  if (batch < 1 || batch > 65536 || !index_ok(*tokens, n) || !vector_ok(*accept, n, at::kFloat) ||
      !vector_ok(*sample, batch, at::kFloat) || (parents && !vector_ok(*parents, n, at::kInt)))
    Py_RETURN_NONE;
  if (draft && (!rows_ok(*draft) || draft->sizes() != target->sizes() || draft->scalar_type() != type)) Py_RETURN_NONE;
  if (!one_device(*target, tokens, starts, accept, sample, draft, parents)) Py_RETURN_NONE;
  for (const Tensor* t : {target, accept, sample, draft})
    if (wants_grad(t)) Py_RETURN_NONE;
  Tensor out, path, counts, ws;
  int st;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::DeviceGuard on(target->device());
    out = make({batch, most}, tokens->scalar_type(), *target);
    path = make({batch, most}, at::kInt, *target);
    counts = make({batch}, at::kInt, *target);
    const size_t bytes = aklr_verify_drafts_workspace_bytes(batch, vocab, most);
    ws = scratch(bytes, *target);
    st = aklr_verify_drafts(target->const_data_ptr(), row_stride(*target), at_or_null(draft), draft ? row_stride(*draft) : 0, n,
                            vocab, tokens->const_data_ptr(), tokens->scalar_type() == at::kLong, ints(parents), ints(starts),
                            floats(accept), floats(sample), batch, most, out.mutable_data_ptr(),
                            static_cast<int32_t*>(path.mutable_data_ptr()), static_cast<int32_t*>(counts.mutable_data_ptr()),
                            float_code(type), data_or_null(ws), bytes, stream_of(*target));
  }
  return st == AKLR_OK ? tuple_of({&out, &path, &counts}) : status_error(st, "verify_drafts");
  END_HANDLE_TH_ERRORS
}

// The cache and what a call reads beside it share no memory, nor do the cache's tensors.
bool cache_apart(const Cache& c, std::initializer_list<const Tensor*> others) {
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < i; ++j)
      if (!apart(c.t[i], c.t[j])) return false;
  return std::all_of(others.begin(), others.end(),
                     [&](const Tensor* t) { return t->device() == c.t[0]->device() && c.clear_of(t); });
}

PyObject* kv_copy(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  static const char* const names[] = {"k_cache", "v_cache", "k_scale", "v_scale", "src", "dst"};
  PyObject* p[6];
  if (!bind(argv, argc, names, 6, 6, 6, p) || watched()) Py_RETURN_NONE;
  Cache c;
  const Tensor *src = dense(p[4]), *dst = dense(p[5]);
  if (!src || !dst || src->dim() != 1 || src->numel() < 1 || src->numel() >= (int64_t{1} << 31) || !index_ok(*src, src->numel()) ||
      !vector_ok(*dst, src->numel(), src->scalar_type()) || !c.read(p) || !cache_apart(c, {src, dst}))
    Py_RETURN_NONE;
  int st;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::DeviceGuard on(c.t[0]->device());
    st = aklr_kv_cache_copy_pages_fp8(c.t[0]->mutable_data_ptr(), c.t[1]->mutable_data_ptr(), c.scales(2), c.scales(3),
                                      c.step[0], c.step[1], c.step[2], c.step[3], src->const_data_ptr(), dst->const_data_ptr(),
                                      src->scalar_type() == at::kLong, src->numel(), c.heads, c.dim, c.pages, c.page,
                                      stream_of(*c.t[0]));
  }
  return st == AKLR_OK ? PyTuple_Pack(4, p[0], p[1], p[2], p[3]) : status_error(st, "kv_cache_copy_pages_fp8");
  END_HANDLE_TH_ERRORS
}

PyObject* kv_compact(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  static const char* const names[] = {"k_cache", "v_cache", "k_scale", "v_scale", "block_table", "seq_lens", "starts", "path",
                                      "counts"};
  PyObject* p[9];
  if (!bind(argv, argc, names, 9, 9, 9, p) || watched()) Py_RETURN_NONE;
  Cache c;
  const Tensor *table = dense(p[4]), *lens = dense(p[5]), *starts = dense(p[6]), *path = dense(p[7]), *counts = dense(p[8]);
  if (!table || !lens || !starts || !path || !counts || lens->dim() != 1) Py_RETURN_NONE;
  const int64_t batch = lens->numel();
  if (batch < 1 || batch > 65536 || !starts_ok(*starts) || starts->numel() != batch + 1 || !table_ok(*table, batch) ||
      table->size(1) < 1 || !vector_ok(*lens, batch, at::kInt) || !vector_ok(*counts, batch, at::kInt) || !table_ok(*path, batch) ||
      path->size(1) < 1 || path->size(1) > (int64_t{1} << 28))
    Py_RETURN_NONE;
  if (!c.read(p) || !cache_apart(c, {table, lens, starts, path, counts}) || table->size(1) * c.page > (int64_t{1} << 28)) Py_RETURN_NONE;
  const int64_t most = path->size(1);
  int st;
  Tensor ws;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::DeviceGuard on(c.t[0]->device());
    const size_t bytes = aklr_kv_cache_compact_fp8_workspace_bytes(batch, most, c.heads, c.dim);
    ws = scratch(bytes, *c.t[0]);
    st = aklr_kv_cache_compact_fp8(c.t[0]->mutable_data_ptr(), c.t[1]->mutable_data_ptr(), c.scales(2), c.scales(3), c.step[0],
                                   c.step[1], c.step[2], c.step[3], ints(table), table_stride(*table), table->size(1), ints(lens),
                                   ints(starts), ints(path), row_stride(*path), most, ints(counts), batch, c.heads, c.dim, c.pages,
                                   c.page, data_or_null(ws), bytes, stream_of(*c.t[0]));
  }
  return st == AKLR_OK ? PyTuple_Pack(4, p[0], p[1], p[2], p[3]) : status_error(st, "kv_cache_compact_fp8");
  END_HANDLE_TH_ERRORS
}

PyObject* kv_update(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  static const char* const names[] = {"page_refs", "block_table", "lens", "new_lens", "page_size", "parents"};
  PyObject* p[6];
  if (!bind(argv, argc, names, 6, 6, 5, p) || watched()) Py_RETURN_NONE;
  const Tensor *refs = plain(p[0]), *table = dense(p[1]), *lens = dense(p[2]), *wants = dense(p[3]), *parents;
  int64_t page;
  if (!refs || !table || !lens || !wants || !given(p[5], &parents) || !whole(p[4], 1, int64_t{1} << 31, &page) || lens->dim() != 1)
    Py_RETURN_NONE;
  const int64_t batch = lens->numel(), pages = refs->numel();
  if (batch < 1 || batch > 65536 || pages < 1 || pages * page >= (int64_t{1} << 31) || !table_ok(*table, batch)) Py_RETURN_NONE;
  const int64_t cols = table->size(1);
  if (cols * page > (int64_t{1} << 28) || batch * cols >= (int64_t{1} << 31) || !vector_ok(*refs, pages, at::kInt) ||
      !vector_ok(*lens, batch, at::kInt) || !vector_ok(*wants, batch, at::kInt) || (parents && !vector_ok(*parents, batch, at::kInt)))
    Py_RETURN_NONE;
  if (!one_device(*refs, table, lens, wants, parents) || !apart_all(refs, {table, lens, wants, parents})) Py_RETURN_NONE;
  Tensor out, granted, src, dst, ws;
  int st;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::DeviceGuard on(refs->device());
    out = make({batch, cols}, at::kInt, *refs);
    granted = make({batch}, at::kInt, *refs);
    src = make({batch}, at::kInt, *refs);
    dst = make({batch}, at::kInt, *refs);
    const size_t bytes = aklr_kv_cache_update_pages_workspace_bytes(batch);
    ws = scratch(bytes, *refs);
    const auto to = [](const Tensor& t) { return static_cast<int32_t*>(t.mutable_data_ptr()); };
    st = aklr_kv_cache_update_pages(to(*refs), pages, ints(table), table_stride(*table), cols, ints(lens), ints(wants),
                                    ints(parents), batch, page, to(out), to(granted), to(src), to(dst), data_or_null(ws), bytes,
                                    stream_of(*refs));
  }
  return st == AKLR_OK ? tuple_of({&out, &granted, &src, &dst}) : status_error(st, "kv_cache_update_pages");
  END_HANDLE_TH_ERRORS
}

// A tensor of 16-byte pieces along its last dimension.
bool pieces_ok(const Tensor& t, at::ScalarType type, at::IntArrayRef shape) {
  if (t.scalar_type() != type || t.sizes() != shape || t.stride(-1) != 1 || !aligned16(t)) return false;
  for (int64_t d = 0; d + 1 < t.dim(); ++d)
    if (t.stride(d) % 8) return false;
  return true;
}

PyObject* lora(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  static const char* const names[] = {"x", "a", "b", "adapters", "base", "scales", "ranks", "out"};
  PyObject* p[8];
  if (!bind(argv, argc, names, 8, 5, 5, p) || watched()) Py_RETURN_NONE;
  const Tensor *x = dense(p[0]), *a = dense(p[1]), *b = dense(p[2]), *ids = dense(p[3]), *base = dense(p[4]), *scales, *ranks, *out;
  if (!x || !a || !b || !ids || !base || !given(p[5], &scales) || !given(p[6], &ranks) || !given(p[7], &out) || x->dim() != 2 ||
      b->dim() != 3)
    Py_RETURN_NONE;
  const int64_t tokens = x->size(0), k = x->size(1), count = b->size(0), n = b->size(1), rank = b->size(2);
  const auto type = x->scalar_type();
  if ((type != at::kBFloat16 && type != at::kHalf) || k < 8 || k > 65536 || k % 8 || n < 8 || n > 262144 || n % 8 || rank < 8 ||
      rank > 128 || rank % 8 || tokens < 1 || tokens > (1 << 20) || count < 1 || count > 4096)
    Py_RETURN_NONE;
  if (!pieces_ok(*x, type, {tokens, k}) || !pieces_ok(*a, type, {count, rank, k}) || !pieces_ok(*b, type, {count, n, rank}) ||
      !pieces_ok(*base, type, {tokens, n}) || !index_ok(*ids, tokens) || (scales && !vector_ok(*scales, count, at::kFloat)) ||
      (ranks && !vector_ok(*ranks, count, at::kInt)))
    Py_RETURN_NONE;
  if (!one_device(*x, a, b, ids, base, scales, ranks, out)) Py_RETURN_NONE;
  for (const Tensor* t : {x, a, b, base, scales, out})
    if (wants_grad(t)) Py_RETURN_NONE;
  if (out && (!pieces_ok(*out, type, {tokens, n}) || !no_inner_overlap(*out) || !(same_place(*out, *base) || apart(out, base)) ||
              !(apart(out, x) || (same_place(*out, *x) && same_place(*out, *base))) ||
              !apart_all(out, {a, b, ids, scales, ranks})))
    Py_RETURN_NONE;
  Tensor o, ws;
  int st;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::DeviceGuard on(x->device());
    o = out ? *out : make({tokens, n}, type, *x);
    const size_t bytes = aklr_lora_project_workspace_bytes(tokens, k, n, rank, count);
    ws = scratch(bytes, *x);
    st = aklr_lora_project(x->const_data_ptr(), x->stride(0), a->const_data_ptr(), a->stride(0), a->stride(1), b->const_data_ptr(),
                           b->stride(0), b->stride(1), ids->const_data_ptr(), ids->scalar_type() == at::kLong, floats(scales),
                           ints(ranks), base->const_data_ptr(), base->stride(0), o.mutable_data_ptr(), o.stride(0), tokens, k, n, rank,
                           count, out_code(type), data_or_null(ws), bytes, stream_of(*x));
  }
  if (st != AKLR_OK) return status_error(st, "lora_project");
  if (out) return Py_INCREF(p[7]), p[7];
  return THPVariable_Wrap(o);
  END_HANDLE_TH_ERRORS
}

#define AKLR_HOST_FN(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {AKLR_HOST_FN(quant_fp8), AKLR_HOST_FN(quant_mxfp8), AKLR_HOST_FN(quant_mxfp4),
                          AKLR_HOST_FN(gemm_fp8), AKLR_HOST_FN(quant_gemm_fp8), AKLR_HOST_FN(gemm_mxfp4),
                          AKLR_HOST_FN(rotary), AKLR_HOST_FN(kv_write), AKLR_HOST_FN(rotary_kv_write),
                          AKLR_HOST_FN(kv_read), AKLR_HOST_FN(tree_attention), AKLR_HOST_FN(verify),
                          AKLR_HOST_FN(kv_copy), AKLR_HOST_FN(kv_compact), AKLR_HOST_FN(kv_update), AKLR_HOST_FN(lora),
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_host", "the ops' per-call host work", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

// The checks above read torch's own objects, whose layout belongs to one version.
static bool same_torch() {
  PyObject* torch = PyImport_ImportModule("torch");
  PyObject* version = torch ? PyObject_GetAttrString(torch, "__version__") : nullptr;
  Py_XDECREF(torch);
  if (!version) return false;
  const bool same = PyUnicode_Check(version) && PyUnicode_CompareWithASCIIString(version, AKLR_TORCH_VERSION) == 0;
  if (!same) PyErr_Format(PyExc_ImportError, "built with torch %s, not %S", AKLR_TORCH_VERSION, version);
  Py_DECREF(version);
  return same;
}

PyMODINIT_FUNC PyInit__host() {
  if (!same_torch()) return nullptr;
  if (aklr_abi_version() != 1) {
    PyErr_SetString(PyExc_ImportError, "libaklr_amd.so ABI version does not match aklr_amd._host");
    return nullptr;
  }
  s_is_shuffled = PyUnicode_InternFromString("is_shuffled");
  s_is_row_major = PyUnicode_InternFromString("is_row_major");
  if (!s_is_shuffled || !s_is_row_major) return nullptr;
  return PyModule_Create(&kModule);
}

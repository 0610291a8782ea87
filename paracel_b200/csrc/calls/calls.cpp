// Python module `_pcl_calls`: the plain calls of the products by group and of the four-bit matrices without Python's part of their cost.
//
// A call of these takes the device a few microseconds at the smallest sizes, and looking at the tensors, two torch.empty and a foreign call
// through ctypes took the host more than the launches themselves.  Every function here looks at its arguments, and where they are
// as they mostly are (one device, the current one; contiguous columns; a new result) makes the result and launches; for anything else, an error
// among it, it returns None, and the caller goes the long way.  The launchers are the extern "C" ones of libpcl_kernels.so, bound
// by address.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

namespace {

using Rows = int (*)(int, int, int, const void*, long long, const void*, long long, long long, const void*, int, void*, long long,
                     long long, int, int, int, int, cudaStream_t);
using Tn = int (*)(int, int, const void*, long long, const void*, long long, const void*, int, void*, long long, int, int, int,
                   cudaStream_t);
using PadFn = int (*)(const void*, long long, long long, long long, long long, int, void*, const void*, long long, long long, long long, long long, int,
                      void*, const void*, int, cudaStream_t);
using Quantize = int (*)(const void*, long long, int, void*, void*, long long, int, cudaStream_t);
using Dequantize = int (*)(const void*, const void*, void*, long long, int, long long, int, cudaStream_t);
using Mx4Rows = int (*)(const void*, long long, int, void*, void*, const void*, const void*, const void*, int, void*, long long, int, long long,
                        int, int, int, int, cudaStream_t);
using Mx4Room = long long (*)(int, long long, int, int, int);
using ErrorString = const char* (*)(int);

Rows rows_fn;
Tn tn_fn;
PadFn pad_fn;
Quantize quantize_fn;
Dequantize dequantize_fn;
Mx4Rows mx4_rows_fn;
Mx4Room mx4_room_fn;
ErrorString error_fn;

constexpr int64_t MAX_GROUPS = 1024, MAX_ROWS = (1ll << 31) - 512, MAX_SIZE = 1ll << 30;

// number of a type as the launchers have it, -1 for others
int type_of(at::ScalarType t) {
  return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1;
}

bool is_tensor(PyObject* o) { return THPVariable_Check(o); }
const at::Tensor& tensor(PyObject* o) { return THPVariable_Unpack(o); }

// out_dtype or, for None, `own`; false for what is neither
bool type_arg(PyObject* o, at::ScalarType own, at::ScalarType* t) {
  *t = own;
  if (o == Py_None) return true;
  if (!THPDtype_Check(o)) return false;
  *t = reinterpret_cast<THPDtype*>(o)->scalar_type;
  return true;
}

// on the current device
bool here(const at::Tensor& t, int device) { return t.is_cuda() && t.get_device() == device; }

bool plain_offsets(const at::Tensor& o, int device) {
  return o.dim() == 1 && (o.scalar_type() == at::kInt || o.scalar_type() == at::kLong) && o.size(0) >= 2 &&
         o.size(0) <= MAX_GROUPS + 1 && o.is_contiguous() && here(o, device);
}

// A 16-bit operand [mats, rows, cols] with contiguous columns: as it lies where its rows start at multiples of 16 bytes, else with a copy to be made
struct Operand {
  const void* at;
  int64_t mats, rows, cols, step_e, step;
  bool plain, copy;

  explicit Operand(const at::Tensor& t) : at(t.data_ptr()) {
    const int64_t d = t.dim();
    mats = d == 3 ? t.size(0) : 1;
    rows = t.size(d - 2);
    cols = t.size(d - 1);
    step = rows > 1 ? t.stride(d - 2) : pitch();   // a dimension of one index may report any stride
    step_e = mats > 1 ? t.stride(0) : rows * step;
    plain = t.stride(d - 1) == 1 || cols == 1;
    copy = (reinterpret_cast<uintptr_t>(at) & 15) || step <= 0 || (step & 7) || step_e <= 0 || (step_e & 7);
  }
  int64_t pitch() const { return (cols + 7) / 8 * 8; }
  int64_t bytes() const { return copy ? mats * rows * pitch() * 2 : 0; }
  Operand copied(void* to) const {
    Operand o = *this;
    if (copy) { o.at = to; o.step = pitch(); o.step_e = rows * o.step; }
    return o;
  }
};

// Buffer for the copies of what has to be copied
at::Tensor room_for(const Operand& a, const Operand& b, const at::TensorOptions& options) {
  return a.copy || b.copy ? at::empty({a.bytes() + b.bytes()}, options.dtype(at::kByte)) : at::Tensor();
}

// Copies it there, and points the operands to it; `offsets`: b has a matrix for each group of them
int copy_operands(Operand& a, Operand& b, const at::Tensor& room, const at::Tensor* offsets, cudaStream_t stream) {
  if (!a.copy && !b.copy) return 0;
  char* to = static_cast<char*>(room.data_ptr());
  const Operand na = a.copied(to), nb = b.copied(to + a.bytes());
  const int rc = pad_fn(a.copy ? a.at : nullptr, a.step_e, a.step, a.mats, a.rows, (int)a.cols, const_cast<void*>(na.at), b.copy ? b.at : nullptr, b.step_e,
                        b.step, b.mats, b.rows, (int)b.cols, const_cast<void*>(nb.at), offsets ? offsets->data_ptr() : nullptr,
                        offsets && offsets->scalar_type() == at::kLong, stream);
  a = na;
  b = nb;
  return rc;
}

bool size_ok(int64_t v) { return v > 0 && v < MAX_SIZE; }

template <class F>
PyObject* launched(const char* name, F&& launch, const at::Tensor& result) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = launch();
  Py_END_ALLOW_THREADS
  if (rc != 0) return PyErr_Format(PyExc_RuntimeError, "%s failed: CUDA error %d (%s)", name, rc, error_fn(rc));
  return THPVariable_Wrap(result);
}

// bind(rows, tn, pad, quantize, dequantize, mx4_rows, mx4_room, error_string): addresses
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  constexpr int COUNT = 8;
  if (n != COUNT) return PyErr_Format(PyExc_TypeError, "%d addresses are wanted", COUNT);
  void* p[COUNT];
  for (int i = 0; i < COUNT; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (p[i] == nullptr) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "address %d is null", i);
  }
  rows_fn = reinterpret_cast<Rows>(p[0]);
  tn_fn = reinterpret_cast<Tn>(p[1]);
  pad_fn = reinterpret_cast<PadFn>(p[2]);
  quantize_fn = reinterpret_cast<Quantize>(p[3]);
  dequantize_fn = reinterpret_cast<Dequantize>(p[4]);
  mx4_rows_fn = reinterpret_cast<Mx4Rows>(p[5]);
  mx4_room_fn = reinterpret_cast<Mx4Room>(p[6]);
  error_fn = reinterpret_cast<ErrorString>(p[7]);
  Py_RETURN_NONE;
}

// grouped_rows(mode, X, W, offsets, out_dtype)
PyObject* grouped_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5 || rows_fn == nullptr || !is_tensor(a[1]) || !is_tensor(a[2]) || !is_tensor(a[3])) Py_RETURN_NONE;
  const long mode = PyLong_AsLong(a[0]);
  const at::Tensor &X = tensor(a[1]), &W = tensor(a[2]), &offsets = tensor(a[3]);
  if ((mode != 0 && mode != 1) || X.dim() != 2 || W.dim() != 3 || !X.is_cuda()) Py_RETURN_NONE;
  const int device = c10::cuda::current_device();
  const at::ScalarType type = X.scalar_type();
  const int in = type_of(type);
  at::ScalarType out_type;
  const int64_t T = X.size(0), E = W.size(0), N = W.size(1), K = W.size(2);
  if (in < 1 || W.scalar_type() != type || !type_arg(a[4], type, &out_type) || (out_type != type && out_type != at::kFloat) || T < 1 ||
      T >= MAX_ROWS || !size_ok(N) || !size_ok(K) || X.size(1) != (mode == 0 ? K : N) || !plain_offsets(offsets, device) ||
      offsets.size(0) != E + 1 || !here(X, device) || !here(W, device))
    Py_RETURN_NONE;
  Operand x(X), w(W);
  if (!x.plain || !w.plain) Py_RETURN_NONE;
  const int64_t cols = mode == 0 ? N : K;
  const at::Tensor out = at::empty({T, cols}, X.options().dtype(out_type));
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device).stream();
  const at::Tensor room = room_for(x, w, X.options());
  return launched("pcl_grouped_rows", [&] {
    const int rc = copy_operands(x, w, room, &offsets, stream);
    return rc ? rc : rows_fn((int)mode, in, type_of(out_type), x.at, x.step, w.at, w.step_e, w.step, offsets.data_ptr(),
                             offsets.scalar_type() == at::kLong, out.data_ptr(), cols, T, (int)E, (int)N, (int)K, 1, stream);
  }, out);
  END_HANDLE_TH_ERRORS
}

// grouped_tn(dY, X, offsets, out_dtype)
PyObject* grouped_tn(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4 || tn_fn == nullptr || !is_tensor(a[0]) || !is_tensor(a[1]) || !is_tensor(a[2])) Py_RETURN_NONE;
  const at::Tensor &Y = tensor(a[0]), &X = tensor(a[1]), &offsets = tensor(a[2]);
  if (X.dim() != 2 || Y.dim() != 2 || !X.is_cuda()) Py_RETURN_NONE;
  const int device = c10::cuda::current_device();
  const at::ScalarType type = X.scalar_type();
  const int in = type_of(type);
  at::ScalarType out_type;
  const int64_t T = X.size(0), K = X.size(1), N = Y.size(1);
  if (in < 1 || Y.scalar_type() != type || !type_arg(a[3], type, &out_type) || (out_type != type && out_type != at::kFloat) || T < 1 ||
      T >= MAX_ROWS || Y.size(0) != T || !size_ok(N) || !size_ok(K) || !plain_offsets(offsets, device) || !here(X, device) || !here(Y, device))
    Py_RETURN_NONE;
  Operand x(X), y(Y);
  if (!x.plain || !y.plain) Py_RETURN_NONE;
  const int64_t E = offsets.size(0) - 1;
  const at::Tensor out = at::empty({E, N, K}, X.options().dtype(out_type));
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device).stream();
  const at::Tensor room = room_for(x, y, X.options());
  return launched("pcl_grouped_tn", [&] {
    const int rc = copy_operands(x, y, room, nullptr, stream);
    return rc ? rc : tn_fn(in, type_of(out_type), y.at, y.step, x.at, x.step, offsets.data_ptr(), offsets.scalar_type() == at::kLong, out.data_ptr(), T,
                           (int)E, (int)N, (int)K, stream);
  }, out);
  END_HANDLE_TH_ERRORS
}

// rows of a matrix that is quantised: contiguous values, any distance
bool plain_rows(const at::Tensor& x) { return x.dim() == 2 && (x.stride(1) == 1 || x.size(1) == 1); }

int64_t data_bytes(int64_t rows, int64_t cols) { return rows * ((cols + 31) / 32 * 16); }
int64_t scale_bytes(int64_t rows, int64_t cols) { return rows * ((cols + 127) / 128 * 4); }

// quantize(X) -> (bytes of data and scales, device, rows, cols, address of data, of scales)
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 1 || quantize_fn == nullptr || !is_tensor(a[0])) Py_RETURN_NONE;
  const at::Tensor& X = tensor(a[0]);
  if (!X.is_cuda() || type_of(X.scalar_type()) < 0 || !(plain_rows(X) || (X.dim() == 3 && X.is_contiguous()))) Py_RETURN_NONE;
  const int device = c10::cuda::current_device();
  const int64_t d = X.dim(), K = X.size(d - 1);
  if (!size_ok(K) || !here(X, device)) Py_RETURN_NONE;
  const int64_t rows = d == 2 ? X.size(0) : X.size(0) * X.size(1);
  if (rows < 1 || rows >= MAX_ROWS) Py_RETURN_NONE;
  const at::Tensor buf = at::empty({data_bytes(rows, K) + scale_bytes(rows, K)}, X.options().dtype(at::kByte));
  uint8_t* data = static_cast<uint8_t*>(buf.data_ptr());
  uint8_t* scales = data + data_bytes(rows, K);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device).stream();
  // a contiguous stack has rows of K values one behind the other, whatever a dimension of one index reports as its stride
  const int64_t ldx = d == 2 ? X.stride(0) : K;
  PyObject* t = launched("pcl_mx4_quantize", [&] {
    return quantize_fn(X.data_ptr(), ldx, type_of(X.scalar_type()), data, scales, rows, (int)K, stream);
  }, buf);
  if (t == nullptr) return nullptr;
  return Py_BuildValue("(NiLLKK)", t, device, (long long)rows, (long long)K, (unsigned long long)(uintptr_t)data,
                       (unsigned long long)(uintptr_t)scales);
  END_HANDLE_TH_ERRORS
}

// dequantize(a tensor on the matrix's device, address of data, of scales, rows, cols, dtype)
PyObject* dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  at::ScalarType type;
  if (n != 6 || dequantize_fn == nullptr || !is_tensor(a[0]) || a[5] == Py_None || !type_arg(a[5], at::kFloat, &type)) Py_RETURN_NONE;
  const at::Tensor& base = tensor(a[0]);
  if (!base.is_cuda() || type_of(type) < 0) Py_RETURN_NONE;
  const int device = c10::cuda::current_device();
  const long long rows = PyLong_AsLongLong(a[3]), cols = PyLong_AsLongLong(a[4]);
  void *data = PyLong_AsVoidPtr(a[1]), *scales = PyLong_AsVoidPtr(a[2]);
  if (PyErr_Occurred()) return nullptr;
  if (rows < 1 || !size_ok(cols) || !here(base, device)) Py_RETURN_NONE;
  const at::Tensor out = at::empty({rows, cols}, base.options().dtype(type));
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device).stream();
  return launched("pcl_mx4_dequantize", [&] { return dequantize_fn(data, scales, out.data_ptr(), cols, type_of(type), rows, (int)cols, stream); }, out);
  END_HANDLE_TH_ERRORS
}

// mx4_rows(A, address of B's data, of its scales, B's rows, cols, device, offsets or None, out_dtype): A is quantised in the call
PyObject* mx4_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8 || mx4_rows_fn == nullptr || !is_tensor(a[0]) || !(a[6] == Py_None || is_tensor(a[6]))) Py_RETURN_NONE;
  const at::Tensor& A = tensor(a[0]);
  at::ScalarType out_type;
  if (!A.is_cuda() || !plain_rows(A) || type_of(A.scalar_type()) < 0 || !type_arg(a[7], A.scalar_type(), &out_type) || type_of(out_type) < 0)
    Py_RETURN_NONE;
  void *data = PyLong_AsVoidPtr(a[1]), *scales = PyLong_AsVoidPtr(a[2]);
  const long long rows = PyLong_AsLongLong(a[3]), K = PyLong_AsLongLong(a[4]), b_device = PyLong_AsLongLong(a[5]);
  if (PyErr_Occurred()) return nullptr;
  const int device = c10::cuda::current_device();
  const int64_t T = A.size(0);
  if (A.size(1) != K || !here(A, device) || b_device != device || T < 1 || T >= MAX_ROWS) Py_RETURN_NONE;
  int64_t groups = 1;
  const void* offsets = nullptr;
  bool wide = false;
  if (a[6] != Py_None) {
    const at::Tensor& o = tensor(a[6]);
    if (!plain_offsets(o, device)) Py_RETURN_NONE;
    groups = o.size(0) - 1;
    offsets = o.data_ptr();
    wide = o.scalar_type() == at::kLong;
  }
  if (rows < 1 || rows % groups) Py_RETURN_NONE;
  const int64_t N = rows / groups;
  const at::Tensor out = at::empty({T, N}, A.options().dtype(out_type));
  at::Tensor work;
  const int64_t room = mx4_room_fn(type_of(A.scalar_type()), T, (int)groups, (int)N, (int)K);
  if (room > 0) work = at::empty({room}, A.options().dtype(at::kByte));
  uint8_t* qa = room > 0 ? static_cast<uint8_t*>(work.data_ptr()) : nullptr;
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device).stream();
  return launched("pcl_mx4_rows", [&] {
    return mx4_rows_fn(A.data_ptr(), A.stride(0), type_of(A.scalar_type()), qa, qa ? qa + data_bytes(T, K) : nullptr, data, scales, offsets, wide,
                       out.data_ptr(), N, type_of(out_type), T, (int)groups, (int)N, (int)K, 1, stream);
  }, out);
  END_HANDLE_TH_ERRORS
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(bind), FAST(grouped_rows), FAST(grouped_tn), FAST(quantize), FAST(dequantize), FAST(mx4_rows),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pcl_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__pcl_calls(void) { return PyModule_Create(&module); }

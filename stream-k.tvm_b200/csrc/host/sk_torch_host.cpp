// Host fast path of the 8-bit integer and grouped entry points: a CPython module that goes from
// torch tensors to the C ABI in one step.
//
// The Python layer (ops.py) checks arguments, copies what has to be copied and calls the C ABI
// through ctypes; that costs 11 to 14 us a call, several times what the small kernels take.  The
// functions here do the same for the plain case -- every argument in order, nothing to copy, no
// options -- in about a third of the time, and return None for anything else: the caller then
// takes the Python path, which knows how to help or what to raise.  They hold no state but the
// addresses of the C functions and of the workspaces that the Python layer registers (one per
// device and stream, as there), and on which devices that layer holds workspaces of a capture.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <map>
#include <set>
#include <utility>

#include "../../../include/streamk_b200.h"

namespace {

using QuantizeFn = int (*)(const void*, int, int, int, int, void*, int, float*, void*);
using GemmI8Fn = int (*)(const sk_problem*, const void*, const void*, const float*, const float*, void*, void*, size_t, void*);
using GroupedFn = int (*)(const sk_grouped_problem*, const void*, const void*, const void*, void*, void*, size_t, void*);

QuantizeFn g_quantize = nullptr;
GemmI8Fn g_gemm_i8 = nullptr;
GroupedFn g_grouped = nullptr;
struct Workspace { void* ptr; size_t bytes; };
std::map<std::pair<int, void*>, Workspace> g_workspaces;   // (device, stream); under the GIL
std::set<int> g_captured;   // devices with workspaces of a capture to be let go; under the GIL

// A plain CUDA tensor (torch.Tensor or Parameter), or null.
const at::Tensor* cuda_tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided) return nullptr;
  return &t;   // (FakeTensor and the like are subclasses: not these)
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool fits_int(int64_t v) { return v > 0 && v <= 0x7fffffff; }

// Row-major matrix whose rows start on 16 bytes: its pitch in elements, or 0.
int64_t pitch16(const at::Tensor& t, int dim0, int64_t elem) {
  const int64_t cols = t.size(dim0 + 1), ld = t.stride(dim0);
  if (t.stride(dim0 + 1) != 1 || ld < cols || (ld * elem) % 16 != 0 || !aligned16(t.const_data_ptr())) return 0;
  return ld;
}

at::Tensor empty(at::IntArrayRef sizes, at::IntArrayRef strides, at::ScalarType type, const at::Device& device) {
  return at::Tensor(at::detail::empty_strided_cuda(sizes, strides, type, device));
}

bool half_type(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }

// The workspace of an eager call; none (a null address) while the stream captures (a graph has one of its own, which
// the Python path makes) and for the first call behind a capture (the Python path lets go of that).
Workspace workspace(int device, void* stream) {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return {nullptr, 0};
  if (g_captured.count(device) != 0) return {nullptr, 0};
  const auto it = g_workspaces.find({device, stream});
  return it == g_workspaces.end() ? Workspace{nullptr, 0} : it->second;
}

// Lets other threads have the interpreter for as long as it lives: an allocation may wait for the
// device and a launch for room in its queue, and what they wait for may need another thread of this
// process (a callback on the host, the launch of a kernel that the queued ones wait for).  Whatever
// belongs to Python or to the maps above is read before.
class Unlocked {
 public:
  Unlocked() : state_(PyEval_SaveThread()) {}
  ~Unlocked() { PyEval_RestoreThread(state_); }
  Unlocked(const Unlocked&) = delete;
  Unlocked& operator=(const Unlocked&) = delete;

 private:
  PyThreadState* state_;
};

#define SK_MISS Py_RETURN_NONE

// quantize(X) -> (Q, scale)
PyObject* quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 1 || g_quantize == nullptr) SK_MISS;
  const at::Tensor* x = cuda_tensor(args[0]);
  if (x == nullptr || x->dim() != 2 || !half_type(x->scalar_type())) SK_MISS;
  const int64_t M = x->size(0), K = x->size(1);
  const int64_t pitch = (K + 15) / 16 * 16;
  if (!fits_int(M) || !fits_int(pitch) || x->stride(1) != 1) SK_MISS;
  const int64_t ld = M > 1 ? x->stride(0) : K;
  if (ld < K || !fits_int(ld)) SK_MISS;
  const at::Device device = x->device();
  const c10::cuda::CUDAGuard guard(device);
  void* stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
  const int flags = SK_FLAG_PDL | (x->scalar_type() == at::kBFloat16 ? SK_FLAG_BF16 : 0);
  const void* X = x->const_data_ptr();
  at::Tensor Q, scale;
  int status;
  {
    const Unlocked unlocked;
    Q = empty({M, K}, {pitch, 1}, at::kChar, device);
    scale = empty({M}, {1}, at::kFloat, device);
    status = g_quantize(X, static_cast<int>(M), static_cast<int>(K), static_cast<int>(ld), flags, Q.mutable_data_ptr(),
                        static_cast<int>(pitch), static_cast<float*>(scale.mutable_data_ptr()), stream);
  }
  if (status != SK_OK) SK_MISS;
  PyObject* q = THPVariable_Wrap(std::move(Q));
  PyObject* s = THPVariable_Wrap(std::move(scale));
  if (q == nullptr || s == nullptr) { Py_XDECREF(q); Py_XDECREF(s); return nullptr; }
  PyObject* r = PyTuple_New(2);
  if (r == nullptr) { Py_DECREF(q); Py_DECREF(s); return nullptr; }
  PyTuple_SET_ITEM(r, 0, q);
  PyTuple_SET_ITEM(r, 1, s);
  return r;
}

// A scale vector of n elements, or null.
const float* scale_of(PyObject* o, int64_t n, const at::Device& device) {
  const at::Tensor* s = cuda_tensor(o);
  if (s == nullptr || s->scalar_type() != at::kFloat || s->device() != device || s->dim() != 1 || s->size(0) != n ||
      (n > 1 && s->stride(0) != 1))
    return nullptr;
  return static_cast<const float*>(s->const_data_ptr());
}

// gemm_i8(A, B, scale_a, scale_b, bf16) -> C
PyObject* gemm_i8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5 || g_gemm_i8 == nullptr) SK_MISS;
  const at::Tensor *a = cuda_tensor(args[0]), *b = cuda_tensor(args[1]);
  if (a == nullptr || b == nullptr || a->dim() != 2 || b->dim() != 2 || a->scalar_type() != at::kChar ||
      b->scalar_type() != at::kChar || a->device() != b->device())
    SK_MISS;
  const int64_t M = a->size(0), K = a->size(1), N = b->size(0);
  if (b->size(1) != K || !fits_int(M) || !fits_int(N) || !fits_int(K)) SK_MISS;
  const int64_t lda = pitch16(*a, 0, 1), ldb = pitch16(*b, 0, 1);
  if (!fits_int(lda) || !fits_int(ldb)) SK_MISS;
  const at::Device device = a->device();
  const float *sa = scale_of(args[2], M, device), *sb = scale_of(args[3], N, device);
  if (sa == nullptr || sb == nullptr) SK_MISS;
  const bool bf16 = args[4] == Py_True;
  const c10::cuda::CUDAGuard guard(device);
  void* stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
  const Workspace ws = workspace(device.index(), stream);
  if (ws.ptr == nullptr) SK_MISS;
  sk_problem p = {};
  p.M = static_cast<int32_t>(M); p.N = static_cast<int32_t>(N); p.K = static_cast<int32_t>(K);
  p.lda = static_cast<int32_t>(lda); p.ldb = static_cast<int32_t>(ldb); p.ldc = static_cast<int32_t>(N);
  p.layout = SK_LAYOUT_NT; p.schedule = SK_SCHED_AUTO; p.fixup = SK_FIXUP_BLOCK_REDUCE;
  p.flags = SK_FLAG_PDL | (bf16 ? SK_FLAG_BF16 : 0);
  const void *A = a->const_data_ptr(), *B = b->const_data_ptr();
  at::Tensor C;
  int status;
  {
    const Unlocked unlocked;
    C = empty({M, N}, {N, 1}, bf16 ? at::kBFloat16 : at::kHalf, device);
    status = g_gemm_i8(&p, A, B, sa, sb, C.mutable_data_ptr(), ws.ptr, ws.bytes, stream);
  }
  if (status != SK_OK) SK_MISS;
  return THPVariable_Wrap(std::move(C));
}

// grouped(kind, A, B, offsets, fp32) -> C
PyObject* grouped(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5 || g_grouped == nullptr) SK_MISS;
  const long kind = PyLong_AsLong(args[0]);
  if (kind == -1 && PyErr_Occurred()) return nullptr;
  const at::Tensor *a = cuda_tensor(args[1]), *b = cuda_tensor(args[2]), *off = cuda_tensor(args[3]);
  if (a == nullptr || b == nullptr || off == nullptr || a->dim() != 2 || !half_type(a->scalar_type()) ||
      b->scalar_type() != a->scalar_type() || a->device() != b->device() || a->device() != off->device())
    SK_MISS;
  const bool off64 = off->scalar_type() == at::kLong;
  if ((!off64 && off->scalar_type() != at::kInt) || off->dim() != 1 || off->size(0) < 2 || off->stride(0) != 1) SK_MISS;
  const int64_t T = a->size(0), K = a->size(1), E = off->size(0) - 1;
  const bool tn = kind == SK_GROUPED_TN, fp32 = args[4] == Py_True;
  if (fp32 && !tn) SK_MISS;
  int64_t N, ldb, stride_b = 0;
  const int64_t lda = pitch16(*a, 0, 2);
  if (tn) {
    if (b->dim() != 2 || b->size(0) != T) SK_MISS;
    N = b->size(1);
    ldb = pitch16(*b, 0, 2);
  } else {
    if (b->dim() != 3 || b->size(0) != E || b->size(kind == SK_GROUPED_NT ? 2 : 1) != K) SK_MISS;
    N = b->size(kind == SK_GROUPED_NT ? 1 : 2);
    ldb = pitch16(*b, 1, 2);
    stride_b = b->stride(0);
    if (E > 1 && (stride_b % 8 != 0 || stride_b < b->size(1) * ldb)) SK_MISS;
  }
  if (lda == 0 || ldb == 0 || !fits_int(T) || !fits_int(N) || !fits_int(K) || !fits_int(E)) SK_MISS;
  const at::Device device = a->device();
  const c10::cuda::CUDAGuard guard(device);
  void* stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
  const Workspace ws = workspace(device.index(), stream);
  if (ws.ptr == nullptr) SK_MISS;
  const at::ScalarType type = fp32 ? at::kFloat : a->scalar_type();
  sk_grouped_problem g = {};
  g.kind = static_cast<int32_t>(kind);
  g.T = static_cast<int32_t>(T); g.E = static_cast<int32_t>(E);
  g.N = static_cast<int32_t>(N); g.K = static_cast<int32_t>(K);
  g.flags = SK_FLAG_PDL | (a->scalar_type() == at::kBFloat16 ? SK_FLAG_BF16 : 0) | (off64 ? SK_FLAG_OFFSETS_64 : 0) |
            (fp32 ? SK_FLAG_OUT_F32 : 0) | (tn ? 0 : SK_FLAG_ZERO_REST);
  g.lda = lda; g.ldb = ldb; g.ldc = N; g.stride_b = stride_b; g.stride_c = tn ? K * N : 0;
  const void *A = a->const_data_ptr(), *B = b->const_data_ptr(), *offsets = off->const_data_ptr();
  at::Tensor C;
  int status;
  {
    const Unlocked unlocked;
    C = tn ? empty({E, K, N}, {K * N, N, 1}, type, device) : empty({T, N}, {N, 1}, type, device);
    status = g_grouped(&g, A, B, offsets, C.mutable_data_ptr(), ws.ptr, ws.bytes, stream);
  }
  if (status != SK_OK) SK_MISS;
  return THPVariable_Wrap(std::move(C));
}

// No C++ exception leaves: where an allocation fails, say, the Python path meets the same and raises.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  try {
    return F(self, args, n);
  } catch (...) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
}

// bind(quantize, gemm_i8, grouped): addresses of the C functions
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 3) { PyErr_SetString(PyExc_TypeError, "bind takes three addresses"); return nullptr; }
  void* p[3];
  for (int i = 0; i < 3; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (p[i] == nullptr && PyErr_Occurred()) return nullptr;
  }
  g_quantize = reinterpret_cast<QuantizeFn>(p[0]);
  g_gemm_i8 = reinterpret_cast<GemmI8Fn>(p[1]);
  g_grouped = reinterpret_cast<GroupedFn>(p[2]);
  Py_RETURN_NONE;
}

// set_workspace(device, stream, address, bytes)
PyObject* set_workspace(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 4) { PyErr_SetString(PyExc_TypeError, "set_workspace takes four numbers"); return nullptr; }
  const long device = PyLong_AsLong(args[0]);
  void* stream = PyLong_AsVoidPtr(args[1]);
  void* ptr = PyLong_AsVoidPtr(args[2]);
  const size_t bytes = PyLong_AsSize_t(args[3]);
  if (PyErr_Occurred()) return nullptr;
  g_workspaces[{static_cast<int>(device), stream}] = Workspace{ptr, bytes};
  Py_RETURN_NONE;
}

// set_captured(device, held)
PyObject* set_captured(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2) { PyErr_SetString(PyExc_TypeError, "set_captured takes a device and a truth value"); return nullptr; }
  const long device = PyLong_AsLong(args[0]);
  if (PyErr_Occurred()) return nullptr;
  if (args[1] == Py_True) g_captured.insert(static_cast<int>(device));
  else g_captured.erase(static_cast<int>(device));
  Py_RETURN_NONE;
}

PyObject* clear_workspaces(PyObject*, PyObject* const*, Py_ssize_t) {
  g_workspaces.clear();
  g_captured.clear();
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"quantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&guarded<quantize>)), METH_FASTCALL, nullptr},
    {"gemm_i8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&guarded<gemm_i8>)), METH_FASTCALL, nullptr},
    {"grouped", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&guarded<grouped>)), METH_FASTCALL, nullptr},
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&bind)), METH_FASTCALL, nullptr},
    {"set_workspace", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&set_workspace)), METH_FASTCALL, nullptr},
    {"set_captured", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&set_captured)), METH_FASTCALL, nullptr},
    {"clear_workspaces", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&clear_workspaces)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "sk_torch_host", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_sk_torch_host(void) { return PyModule_Create(&kModule); }

// The torch side of uwc_b200.paged: checks of tensors, outputs, streams and workspaces, and the calls of
// the C ABI (include/uwc_b200.h). A paged call is a few microseconds of GPU work, of which the checks would
// take twice as long in Python (15 us a call, launch included; 7 to 9 us here). Refusals are AssertionErrors as everywhere in the
// package, CUDA problems RuntimeErrors.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAStream.h>

#include <map>
#include <stdexcept>
#include <string>
#include <utility>

#include "../../include/uwc_b200.h"

namespace {

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};
void require(bool ok, const char* what) {
  if (!ok) throw Refused(what);
}

constexpr int64_t kHd = 128;
constexpr long long kMost = 1ll << 30;   // longest length, window and sinks

const at::Tensor& tensor(PyObject* o, const char* what) {
  require(THPVariable_Check(o), what);
  return THPVariable_Unpack(o);
}
long long integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw std::bad_cast();
  return v;
}
int length(PyObject* o, const char* what) {
  const long long v = integer(o);
  require(v >= 0 && v <= kMost, what);
  return (int)v;
}
// A window or a number of sinks: more than any position is as good as kMost.
int reach(PyObject* o, const char* what) {
  const long long v = integer(o);
  require(v >= 0, what);
  return (int)std::min(v, kMost);
}
double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw std::bad_cast();
  return v;
}

// What every call has: the pages and the batch's description.
struct Call {
  int dev;
  int8_t *k, *v;
  float *sk, *sv;
  int pages, ps, Hkv, seqs, width;
  const int *table, *start, *cu;
  at::Device device;

  bool on(const at::Tensor& t, at::ScalarType type) const {
    return t.is_cuda() && t.get_device() == dev && t.scalar_type() == type && t.is_contiguous();
  }
  // k, v, sk, sv, table, start, cu
  explicit Call(PyObject* const* a) : device(at::kCPU) {
    const at::Tensor& kt = tensor(a[0], "the cache holds tensors");
    const at::Tensor& vt = tensor(a[1], "the cache holds tensors");
    const at::Tensor& skt = tensor(a[2], "the cache holds tensors");
    const at::Tensor& svt = tensor(a[3], "the cache holds tensors");
    const at::Tensor& tt = tensor(a[4], "table is a tensor");
    const at::Tensor& st = tensor(a[5], "start is a tensor");
    const at::Tensor& ct = tensor(a[6], "cu is a tensor");
    require(kt.is_cuda(), "the cache lies on a CUDA device");
    device = kt.device();
    dev = kt.get_device();
    require(dev == c10::cuda::current_device(), "the cache's device is the current one");
    require(kt.dim() == 4 && kt.size(3) == kHd, "pages are (pages, Hkv, page_size, 128)");
    require(vt.sizes() == kt.sizes(), "keys and values have the same pages");
    require(skt.dim() == 2 && skt.size(0) == kt.size(0) && skt.size(1) == kt.size(1) && svt.sizes() == skt.sizes(),
            "scales are (pages, Hkv)");
    require(on(kt, at::kChar) && on(vt, at::kChar), "pages are contiguous int8 on one device");
    require(on(skt, at::kFloat) && on(svt, at::kFloat), "scales are contiguous float32 on the pages' device");
    require(tt.dim() == 2 && st.dim() == 1 && ct.dim() == 1 && st.size(0) == tt.size(0) && ct.size(0) == tt.size(0) + 1,
            "table is (sequences, width), start (sequences), cu (sequences + 1)");
    require(on(tt, at::kInt) && on(st, at::kInt) && on(ct, at::kInt),
            "the batch's description is contiguous int32 on the pages' device");
    require(kt.size(0) <= kMost && kt.size(1) <= kMost && tt.size(0) <= kMost && tt.size(1) <= kMost, "too large");
    pages = (int)kt.size(0);
    Hkv = (int)kt.size(1);
    ps = (int)kt.size(2);
    seqs = (int)tt.size(0);
    width = (int)tt.size(1);
    k = (int8_t*)kt.data_ptr();
    v = (int8_t*)vt.data_ptr();
    sk = (float*)skt.data_ptr();
    sv = (float*)svt.data_ptr();
    table = (const int*)tt.data_ptr();
    start = (const int*)st.data_ptr();
    cu = (const int*)ct.data_ptr();
  }
};

int type_code(at::ScalarType t) {
  require(t == at::kBFloat16 || t == at::kHalf, "rows are bfloat16 or float16");
  return t == at::kBFloat16 ? UWC_T_BF16 : UWC_T_F16;
}

struct Rows {
  const void* p;
  long long tok, head;
  int n, heads;
};
Rows rows_of(const Call& c, const at::Tensor& t, at::ScalarType type) {
  require(t.dim() == 3 && t.size(2) == kHd && t.stride(2) == 1, "rows are (n, heads, 128), a head's values contiguous");
  require(t.is_cuda() && t.get_device() == c.dev && t.scalar_type() == type, "rows have one type, on the pages' device");
  require(t.size(0) <= kMost && t.size(1) <= kMost, "too many rows");
  return Rows{t.data_ptr(), t.stride(0), t.stride(1), (int)t.size(0), (int)t.size(1)};
}

void check(int rc, const char* what) {
  if (rc == UWC_OK) return;
  const std::string msg = std::string(what) + ": " + uwc_status_string(rc) + " (status " + std::to_string(rc) + ")";
  if (rc == UWC_ERR_ARG || rc == UWC_ERR_SHAPE || rc == UWC_ERR_ALIGN || rc == UWC_ERR_SCRATCH) throw Refused(msg);
  throw std::runtime_error(msg);
}

template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_AssertionError, e.what());
  } catch (const std::bad_cast&) {
    // the Python error is set
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// k, v, sk, sv, table, start, cu, max_new, rows k, rows v, cos, sin, q, q_norm, k_norm, eps -> rotated q or None
PyObject* py_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    require(n == 16, "append takes 16 arguments");
    const Call c(a);
    const int max_new = length(a[7], "max_new is not negative");
    const at::Tensor& kt = tensor(a[8], "k is a tensor");
    const at::ScalarType type = kt.scalar_type();
    const int code = type_code(type);
    const Rows k = rows_of(c, kt, type), v = rows_of(c, tensor(a[9], "v is a tensor"), type);
    require(k.heads == c.Hkv && v.heads == c.Hkv && v.n == k.n, "k and v are (n, Hkv, 128)");
    const at::Tensor &cos = tensor(a[10], "cos is a tensor"), &sin = tensor(a[11], "sin is a tensor");
    require(cos.dim() == 2 && cos.size(1) == kHd && sin.sizes() == cos.sizes() && cos.size(0) <= kMost &&
                c.on(cos, at::kFloat) && c.on(sin, at::kFloat),
            "cos and sin are contiguous float32 (positions, 128) on the pages' device");
    const float* norm[2] = {nullptr, nullptr};
    for (int i = 0; i < 2; i++)
      if (a[13 + i] != Py_None) {
        const at::Tensor& w = tensor(a[13 + i], "a norm's weights are a tensor");
        require(w.dim() == 1 && w.size(0) == kHd && c.on(w, at::kFloat), "a norm's weights are contiguous float32 (128) on the pages' device");
        norm[i] = (const float*)w.data_ptr();
      }
    const double eps = real(a[15]);
    at::Tensor out;
    Rows q = {nullptr, 0, 0, 0, 0};
    if (a[12] != Py_None) {
      q = rows_of(c, tensor(a[12], "q is a tensor"), type);
      require(q.n == k.n, "q has k's rows");
      out = at::empty({q.n, q.heads, kHd}, kt.options());
    }
    check(uwc_paged_append(c.k, c.sk, c.v, c.sv, c.pages, c.ps, c.Hkv, c.table, c.start, c.cu, c.seqs, c.width, k.n, max_new,
                           code, k.p, k.tok, k.head, v.p, v.tok, v.head, q.p, q.tok, q.head, q.p ? out.data_ptr() : nullptr,
                           q.heads, (const float*)cos.data_ptr(), (const float*)sin.data_ptr(), (int)cos.size(0), norm[0],
                           norm[1], eps, c10::cuda::getCurrentCUDAStream(c.dev).stream()),
          "paged append");
    if (a[12] == Py_None) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
  });
}

// k, v, sk, sv, table, first, cu, n, max_rows, type (0 bf16, 1 fp16, 2 float32) -> (keys, values)
PyObject* py_gather(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    require(n == 10, "gather takes 10 arguments");
    const Call c(a);
    const int rows = length(a[7], "n is not negative"), most = length(a[8], "max_rows is not negative");
    const int code = (int)integer(a[9]);
    require(code >= 0 && code <= 2, "values are bfloat16, float16 or float32");
    const at::TensorOptions opt =
        at::TensorOptions().device(c.device).dtype(code == 0 ? at::kBFloat16 : code == 1 ? at::kHalf : at::kFloat);
    at::Tensor k = at::empty({rows, c.Hkv, kHd}, opt), v = at::empty({rows, c.Hkv, kHd}, opt);
    check(uwc_paged_gather(c.k, c.sk, c.v, c.sv, c.pages, c.ps, c.Hkv, c.table, c.start, c.cu, c.seqs, c.width, rows, most,
                           code, k.data_ptr(), v.data_ptr(), c10::cuda::getCurrentCUDAStream(c.dev).stream()),
          "paged gather");
    PyObject* r = PyTuple_New(2);
    if (!r) return nullptr;
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(k)));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(v)));
    return r;
  });
}

// A stream's workspace, as large as any call on the device needs (40 MB), its counters zeroed once: a call
// leaves them so. A captured call gets one of its own size, whose counters the graph zeroes. (The map is
// never destroyed: its tensors would outlive the CUDA context. The caller holds the GIL.)
constexpr int64_t kCounters = 4096;
at::Tensor workspace(const Call& c, cudaStream_t stream, int max_new, int max_len, int H, int window, int sinks) {
  static auto* kept = new std::map<std::pair<int, cudaStream_t>, at::Tensor>;
  const bool captured = c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None;
  const at::TensorOptions opt = at::TensorOptions().device(c.device).dtype(at::kByte);
  uint64_t bytes = 0;
  if (captured) {
    bytes = uwc_paged_attention_workspace_bytes(c.seqs, max_new, max_len, H, c.Hkv, window, sinks);
  } else {
    const auto it = kept->find({c.dev, stream});
    if (it != kept->end()) return it->second;
    for (const int rows : {8, 16, 1 << 30})
      bytes = std::max<uint64_t>(bytes, uwc_paged_attention_workspace_bytes(1, rows, 1 << 30, 1, 1, -1, 0));
  }
  at::Tensor ws = at::empty({(int64_t)std::max<uint64_t>(bytes, kCounters)}, opt);
  ws.narrow(0, 0, kCounters).zero_();
  if (!captured) (*kept)[{c.dev, stream}] = ws;
  return ws;
}

// k, v, sk, sv, table, start, cu, max_new, q, max_len, scale, window or None, sinks, out or None -> out
PyObject* py_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    require(n == 14, "attention takes 14 arguments");
    const Call c(a);
    const int max_new = length(a[7], "max_new is not negative"), max_len = length(a[9], "max_len is not negative");
    const at::Tensor& qt = tensor(a[8], "q is a tensor");
    const at::ScalarType type = qt.scalar_type();
    const int code = type_code(type);
    const Rows q = rows_of(c, qt, type);
    const double scale = real(a[10]);
    const int window = a[11] == Py_None ? -1 : reach(a[11], "window is not negative");
    const int sinks = reach(a[12], "sinks is not negative");
    at::Tensor out;
    if (a[13] == Py_None) {
      out = at::empty({q.n, q.heads, kHd}, qt.options());
    } else {
      out = tensor(a[13], "out is a tensor");
      require(out.sizes() == qt.sizes() && c.on(out, type), "out is contiguous, of q's shape and type, on the pages' device");
    }
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(c.dev).stream();
    const at::Tensor ws = workspace(c, stream, max_new, max_len, q.heads, window, sinks);
    check(uwc_paged_attention(c.k, c.sk, c.v, c.sv, c.pages, c.ps, c.Hkv, c.table, c.start, c.cu, c.seqs, c.width, q.n, max_new,
                              max_len, code, q.p, q.tok, q.head, out.data_ptr(), q.heads, (float)scale, window, sinks,
                              ws.data_ptr(), (uint64_t)ws.numel(), stream),
          "paged attention");
    if (a[13] != Py_None) {
      Py_INCREF(a[13]);
      return a[13];
    }
    return THPVariable_Wrap(std::move(out));
  });
}

PyMethodDef kMethods[] = {
    {"append", (PyCFunction)(void (*)(void))py_append, METH_FASTCALL, nullptr},
    {"gather", (PyCFunction)(void (*)(void))py_gather, METH_FASTCALL, nullptr},
    {"attention", (PyCFunction)(void (*)(void))py_attention, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_paged", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged(void) { return PyModule_Create(&kModule); }

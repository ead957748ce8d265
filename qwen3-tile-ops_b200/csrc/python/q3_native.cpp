// Python side of the rotary and paged-chunk operators: turns tensors (or
// MatrixView s) into the views of the C ABI and calls it, on the tensors' device
// and its current stream.  These calls take a few microseconds on the GPU for
// small batches; building a view with ctypes takes 2.4 us and a call of it 3 us more
// on the host, against about 1 us for a whole call here.
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <Python.h>

#include <climits>
#include <cstring>
#include <stdexcept>
#include <string>

#include "../../../include/q3_ops.h"

namespace {

struct PyError {};   // a Python exception is set

[[noreturn]] void refuse(const std::string &what) { throw std::invalid_argument(what); }

struct Call {
  PyObject *const *args;
  int dev = -1;
  c10::cuda::OptionalCUDAGuard guard;
  void *stream = nullptr;
  PyObject *given = nullptr;

  // device of the first operand, made current; the stream argument comes last
  Call(PyObject *const *a, Py_ssize_t n, Py_ssize_t want, int operand) : args(a) {
    if (n != want) refuse("wrong number of arguments");
    PyObject *x = a[operand];
    PyObject *owner = nullptr;
    if (!THPVariable_Check(x) && x != Py_None) {
      owner = PyObject_GetAttrString(x, "owner");
      if (!owner) throw PyError{};
      x = owner;
    }
    if (THPVariable_Check(x)) {
      const at::Tensor &t = THPVariable_Unpack(x);
      const bool cuda = t.is_cuda();
      if (cuda) dev = t.get_device();
      Py_XDECREF(owner);
      if (!cuda) refuse("MatrixView needs CUDA memory");
    } else {
      Py_XDECREF(owner);
      dev = c10::cuda::current_device();
    }
    if (dev != c10::cuda::current_device()) guard.set_index(dev);
    given = a[n - 1];
    if (given == Py_None) {
      given = nullptr;
      stream = c10::cuda::getCurrentCUDAStream(dev).stream();
    } else if (PyLong_Check(given)) {
      stream = PyLong_AsVoidPtr(given);
    } else {
      PyObject *s = PyObject_GetAttrString(given, "cuda_stream");
      if (!s) throw PyError{};
      stream = PyLong_AsVoidPtr(s);
      Py_DECREF(s);
    }
    if (PyErr_Occurred()) throw PyError{};
  }

  // The stream given is being captured into a graph, the current one is not: what the allocator gives
  // now belongs to the current one, and is another tensor's when the graph is replayed.
  bool foreign_capture() const {
    return given && capturing(static_cast<cudaStream_t>(stream)) &&
           !capturing(c10::cuda::getCurrentCUDAStream(dev).stream());
  }
  static bool capturing(cudaStream_t s) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    const cudaError_t e = cudaStreamIsCapturing(s, &status);
    if (e == cudaErrorStreamCaptureImplicit) {   // the legacy stream beside a blocking captured one
      cudaGetLastError();
      return false;
    }
    C10_CUDA_CHECK(e);
    return status != cudaStreamCaptureStatusNone;
  }

  const at::Tensor &tensor(int i) const {
    const at::Tensor &t = THPVariable_Unpack(args[i]);
    if (!t.is_cuda() || t.get_device() != dev)
      refuse("operands on different devices: " + t.device().str() + " and cuda:" + std::to_string(dev));
    return t;
  }
  // an empty tensor has no address: any aligned one, of which nothing is read
  static void *address(const at::Tensor &t) {
    return t.numel() ? t.data_ptr() : reinterpret_cast<void *>(256);
  }
  uint32_t u32(int i) const {
    const unsigned long x = PyLong_AsUnsignedLong(args[i]);
    if (x == static_cast<unsigned long>(-1) && PyErr_Occurred()) throw PyError{};
    if (x > UINT32_MAX) refuse("a size is too large");
    return static_cast<uint32_t>(x);
  }
  int flag(int i) const {
    const int x = PyObject_IsTrue(args[i]);
    if (x < 0) throw PyError{};
    return x;
  }
  double number(int i) const {
    const double x = PyFloat_AsDouble(args[i]);
    if (x == -1.0 && PyErr_Occurred()) throw PyError{};
    return x;
  }
  // the view of an operand: v, or null for None
  const q3_view *view(int i, q3_view &v) const {
    if (args[i] == Py_None) return nullptr;
    std::memset(&v, 0, sizeof v);
    if (!THPVariable_Check(args[i])) {
      PyObject *owner = PyObject_GetAttrString(args[i], "owner");
      if (!owner) throw PyError{};
      const int at = THPVariable_Check(owner) ? THPVariable_Unpack(owner).get_device() : dev;
      Py_DECREF(owner);
      if (at != dev) refuse("operands on different devices");
      auto get = [&](const char *name) -> long long {
        PyObject *o = PyObject_GetAttrString(args[i], name);
        if (!o) throw PyError{};
        const long long x = static_cast<long long>(PyLong_AsLongLong(o));
        Py_DECREF(o);
        if (x == -1 && PyErr_Occurred()) throw PyError{};
        return x;
      };
      v.data = reinterpret_cast<void *>(get("data"));
      v.row_bytes = static_cast<int32_t>(get("row_bytes"));
      v.col_bytes = static_cast<int32_t>(get("col_bytes"));
      v.rows = static_cast<uint32_t>(get("rows"));
      v.cols = static_cast<uint32_t>(get("cols"));
      v.dtype = static_cast<uint8_t>(get("dtype"));
      return &v;
    }
    const at::Tensor &t = tensor(i);
    const int64_t dim = t.dim(), es = t.element_size();
    if (dim != 1 && dim != 2) refuse("MatrixView needs a 1-D or 2-D tensor");
    switch (t.scalar_type()) {
      case at::kChar: v.dtype = Q3_DT_I8; break;
      case at::kByte: v.dtype = Q3_DT_U8; break;
      case at::kInt: v.dtype = Q3_DT_I32; break;
      case at::kFloat: v.dtype = Q3_DT_F32; break;
      case at::kHalf: v.dtype = Q3_DT_F16; break;
      case at::kBFloat16: v.dtype = Q3_DT_BF16; break;
      default: refuse("MatrixView has no code for this dtype");
    }
    const int64_t rb = t.stride(0) * es, cb = dim == 2 ? t.stride(1) * es : es;
    const int64_t rows = t.size(0), cols = dim == 2 ? t.size(1) : 1;
    if (rb > INT32_MAX || rb < INT32_MIN || cb > INT32_MAX || cb < INT32_MIN || rows > UINT32_MAX ||
        cols > UINT32_MAX)
      refuse("a size or stride of a view is too large");
    v.data = address(t);
    v.row_bytes = static_cast<int32_t>(rb);
    v.col_bytes = static_cast<int32_t>(cb);
    v.rows = static_cast<uint32_t>(rows);
    v.cols = static_cast<uint32_t>(cols);
    return &v;
  }
  // address of a contiguous device array of at least n elements
  void *array(int i, bool sixteen, int64_t n, const char *what) const {
    const char *type = sixteen ? " 16-bit integers" : " int32";
    if (!THPVariable_Check(args[i])) refuse(std::string(what) + ": a tensor is needed");
    const at::Tensor &t = tensor(i);
    const bool ok = sixteen ? t.scalar_type() == at::kShort || t.scalar_type() == at::kUInt16
                            : t.scalar_type() == at::kInt;
    if (!ok || !t.is_contiguous() || t.numel() < n)
      refuse(std::string(what) + ": a contiguous array of at least " + std::to_string(n) + type +
             " is needed");
    return address(t);
  }
  q3_paged_kv pool(int i) const {
    Py_buffer b;
    if (PyObject_GetBuffer(args[i], &b, PyBUF_SIMPLE)) throw PyError{};
    q3_paged_kv kv;
    const bool ok = b.len == static_cast<Py_ssize_t>(sizeof kv);
    if (ok) std::memcpy(&kv, b.buf, sizeof kv);
    PyBuffer_Release(&b);
    if (!ok) refuse("kv: a PagedKV is needed");
    return kv;
  }
};

template <typename F>
PyObject *guarded(F f) {
  try {
    return PyLong_FromLong(f());
  } catch (const PyError &) {
  } catch (const std::invalid_argument &e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// theta, pos0, scaling, factor, original_max, beta_fast, beta_slow, attn_factor, cos, sin, stream
PyObject *rope_tables(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&] {
    Call c(a, n, 11, 8);
    q3_rope_spec s{c.number(0), c.number(3), c.number(4), c.number(5), c.number(6), c.number(7),
                   static_cast<int32_t>(c.u32(2))};
    q3_view cos, sin;
    const q3_view *pc = c.view(8, cos), *ps = c.view(9, sin);
    return q3_rope_tables(&s, c.u32(1), pc, ps, c.stream);
  });
}

// x, nw, pos, cos, sin, out, scale, heads, head_dim, interleaved, inv_hd, stream
PyObject *rope_rows(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&] {
    Call c(a, n, 12, 0);
    q3_view x, nw, cos, sin, out, scale;
    const q3_view *px = c.view(0, x), *pn = c.view(1, nw);
    if (!px) return static_cast<int>(Q3_ERR_NULL);
    const void *pos = c.array(2, false, x.rows, "pos");
    const q3_view *pc = c.view(3, cos), *ps = c.view(4, sin), *po = c.view(5, out);
    const q3_view *pl = c.view(6, scale);
    return q3_rope_rows(px, pn, static_cast<const int32_t *>(pos), pc, ps, po, pl, c.u32(7), c.u32(8),
                        c.flag(9), static_cast<float>(c.number(10)), c.stream);
  });
}

// k, v, nw, inv_hd, cos, sin, interleaved, kv, num_pages, tables, max_pages, row0, kv_len, n_seqs,
// kv_heads, head_dim, stream
PyObject *paged_kv_append(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&] {
    Call c(a, n, 17, 0);
    q3_view k, v, nw, cos, sin;
    const q3_view *pk = c.view(0, k), *pv = c.view(1, v), *pn = c.view(2, nw);
    const q3_view *pc = c.view(4, cos), *ps = c.view(5, sin);
    const q3_paged_kv kv = c.pool(7);
    const uint32_t pages = c.u32(8), mp = c.u32(10), seqs = c.u32(13);
    const void *tables = c.array(9, true, static_cast<int64_t>(seqs) * mp, "tables");
    const void *row0 = c.array(11, false, static_cast<int64_t>(seqs) + 1, "row0");
    const void *len = c.array(12, false, seqs, "kv_len");
    return q3_paged_kv_append_batch(pk, pv, pn, static_cast<float>(c.number(3)), pc, ps, c.flag(6), &kv,
                                    pages, static_cast<const uint16_t *>(tables), mp,
                                    static_cast<const int32_t *>(row0),
                                    static_cast<const int32_t *>(len), seqs, c.u32(14), c.u32(15),
                                    c.stream);
  });
}

// q, q_scale, kv, num_pages, tables, max_pages, row0, kv_len, n_seqs, max_rows, o, os, heads, kv_heads,
// head_dim, causal, window, qk_scale, workspace, stream
PyObject *attention_chunk(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&] {
    if (n == 20 && a[18] != Py_None && !THPVariable_Check(a[18])) refuse("workspace: a tensor is needed");
    Call c(a, n, 20, 0);
    q3_view q, qs, o, os;
    const q3_view *pq = c.view(0, q), *pqs = c.view(1, qs), *po = c.view(10, o), *pos = c.view(11, os);
    if (!pq) return static_cast<int>(Q3_ERR_NULL);
    const q3_paged_kv kv = c.pool(2);
    const uint32_t pages = c.u32(3), mp = c.u32(5), seqs = c.u32(8), max_rows = c.u32(9);
    const uint32_t heads = c.u32(12), kvh = c.u32(13), hd = c.u32(14);
    const void *tables = c.array(4, true, static_cast<int64_t>(seqs) * mp, "tables");
    const void *row0 = c.array(6, false, static_cast<int64_t>(seqs) + 1, "row0");
    const void *len = c.array(7, false, seqs, "kv_len");
    at::Tensor ws;
    void *at_ = nullptr;
    size_t bytes = 0;
    if (a[18] != Py_None) {
      const at::Tensor &t = c.tensor(18);
      if (!t.is_contiguous()) refuse("workspace: a contiguous tensor is needed");
      at_ = t.data_ptr();
      bytes = t.nbytes();
    } else if ((bytes = q3_attention_chunk_workspace_bytes(q.rows, seqs, max_rows, mp * kv.page_tokens,
                                                           heads, kvh, hd))) {
      if (c.foreign_capture())
        refuse("workspace: needed where the stream given is being captured and the current one is not");
      ws = at::empty({static_cast<int64_t>(bytes)},
                     at::TensorOptions().dtype(at::kByte).device(at::kCUDA, c.dev));
      at_ = ws.data_ptr();
      if (c.given)   // the allocator's stream is another one
        c10::cuda::CUDACachingAllocator::recordStream(
            ws.storage().data_ptr(),
            c10::cuda::getStreamFromExternal(static_cast<cudaStream_t>(c.stream), c.dev));
    }
    return q3_attention_chunk_batch(pq, pqs, &kv, pages, static_cast<const uint16_t *>(tables), mp,
                                    static_cast<const int32_t *>(row0),
                                    static_cast<const int32_t *>(len), seqs, max_rows, po, pos, heads,
                                    kvh, hd, c.flag(15), c.u32(16), static_cast<float>(c.number(17)), at_,
                                    bytes, c.stream);
  });
}

PyMethodDef methods[] = {
    {"rope_tables", reinterpret_cast<PyCFunction>(rope_tables), METH_FASTCALL, nullptr},
    {"rope_rows", reinterpret_cast<PyCFunction>(rope_rows), METH_FASTCALL, nullptr},
    {"paged_kv_append", reinterpret_cast<PyCFunction>(paged_kv_append), METH_FASTCALL, nullptr},
    {"attention_chunk", reinterpret_cast<PyCFunction>(attention_chunk), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods,
                      nullptr,               nullptr,   nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&module); }

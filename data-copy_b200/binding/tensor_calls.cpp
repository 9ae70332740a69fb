// dcopy._tensor_calls: the model operators' C ABI called on torch tensors.
//
// Reads rows, pitch and type of each tensor, takes torch's current stream of the
// tensors' device (made current for the call) unless one is given, and a workspace
// from torch's allocator unless one is given.  The same in Python took 5 us a call
// besides the launch, more than the smallest operators run on the GPU; here it is
// under 1 us.  The functions of libdcopy.so are handed over by address (bind), so
// that one copy of the library is loaded.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>
#include <string>

#include "dcopy/dcopy.h"

namespace {

#define DCOPY_CALLS(X)                                                                     \
  X(dcopy_last_error_message)                                                              \
  X(dcopy_embedding_lookup) X(dcopy_embedding_grad) X(dcopy_embedding_grad_workspace)      \
  X(dcopy_expert_sort) X(dcopy_expert_sort_workspace) X(dcopy_expert_dispatch)             \
  X(dcopy_expert_combine) X(dcopy_expert_combine_grad)                                     \
  X(dcopy_grad_sum_squares) X(dcopy_grad_clip) X(dcopy_clip_grad_norm)

struct Library {
#define X(name) decltype(&::name) name = nullptr;
  DCOPY_CALLS(X)
#undef X
} lib;
PyObject *error_class = nullptr;  // dcopy.DcopyError

// A Python exception is set; carried to the entry point as a C++ one.
struct Raised {};

[[noreturn]] void value_error(const char *name, const std::string &what) {
  PyErr_Format(PyExc_ValueError, "%s: %s", name, what.c_str());
  throw Raised{};
}

[[noreturn]] void dcopy_error(int code, const std::string &message, const char *func) {
  PyObject *e = PyObject_CallFunction(error_class, "iss", code, message.c_str(), func);
  if (e) {
    PyErr_SetObject(error_class, e);
    Py_DECREF(e);
  }
  throw Raised{};
}

int32_t type_code(at::ScalarType t) {  // the GE DataType; -1, which the library refuses
  switch (t) {
    case at::kFloat: return 0;
    case at::kHalf: return 1;
    case at::kChar: return 2;
    case at::kInt: return 3;
    case at::kByte: case at::kFloat8_e4m3fn: case at::kFloat8_e5m2: return 4;
    case at::kLong: return 9;
    case at::kBFloat16: return 27;
    default: return -1;
  }
}

const at::Tensor &unpack(PyObject *o, const char *name) {
  if (!THPVariable_Check(o)) value_error(name, "expected a tensor");
  return THPVariable_Unpack(o);
}

// A tensor as rows of its last dimension; the other dimensions must step evenly.
DcopyMatrix layout(const at::Tensor &t, const char *name) {
  DcopyMatrix m{};
  const auto shape = t.sizes(), stride = t.strides();
  const int64_t d = (int64_t)shape.size();
  int64_t unit = 1;
  if (d < 2) {
    m.rows = 1;
    m.cols = t.numel();
    unit = d ? stride[0] : 1;
    if (unit != 1) {  // a strided vector: rows of one element
      m.rows = m.cols, m.cols = 1, m.pitch = unit, unit = 1;
      if (m.pitch < 1 && m.rows > 1) value_error(name, "elements repeat");
    }
  } else {
    m.cols = shape[d - 1];
    unit = stride[d - 1];
    m.pitch = stride[d - 2];
    m.rows = 1;
    for (int64_t k = d - 2; k >= 0; --k) {
      if (shape[k] > 1 && t.numel()) {  // without elements strides mean nothing
        if (m.rows == 1) m.pitch = stride[k];
        else if (stride[k] != m.rows * m.pitch) value_error(name, "rows do not lie at one pitch");
      }
      m.rows *= shape[k];
    }
  }
  if (unit != 1 && m.cols > 1 && t.numel()) value_error(name, "the last dimension must be dense");
  m.data = const_cast<void *>(t.const_data_ptr());
  m.type = type_code(t.scalar_type());
  return m;
}

int64_t as_int(PyObject *o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return v;
}
double as_double(PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised{};
  return v;
}

bool as_bool(PyObject *o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised{};
  return v != 0;
}

// One call: its device, which all its tensors share, and its stream.
class Call {
 public:
  Call(const char *func, PyObject *stream) : func_(func), given_(stream) {}

  const at::Tensor &tensor(PyObject *o, const char *name) {
    const at::Tensor &t = unpack(o, name);
    if (!t.is_cuda()) value_error(name, "expected a CUDA tensor");
    if (device_ < 0) device_ = t.get_device();
    else if (t.get_device() != device_) value_error(name, "tensors are on different devices");
    return t;
  }
  DcopyMatrix matrix(PyObject *o, const char *name) { return layout(tensor(o, name), name); }
  // A dense tensor of one type, or None (nullptr).
  void *vector(PyObject *o, const char *name, at::ScalarType type, int64_t *count = nullptr) {
    if (o == Py_None) return nullptr;
    const at::Tensor &t = tensor(o, name);
    if (!t.is_contiguous() || t.scalar_type() != type)
      value_error(name, std::string("expected a contiguous CUDA tensor of type ") +
                            c10::toString(type));
    if (count) *count = t.numel();
    return const_cast<void *>(t.const_data_ptr());
  }
  void on_device(int64_t device) { device_ = device; }

  // Fixes device and stream; after the tensors were read.  A given stream is torch's
  // current one for the rest of the call.
  dcopy_stream_t stream() {
    guard_.emplace((c10::DeviceIndex)device_);
    if (given_ == Py_None)
      return reinterpret_cast<dcopy_stream_t>(
          c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device_).stream());
    PyObject *value = PyLong_Check(given_) ? Py_NewRef(given_)
                                           : PyObject_GetAttrString(given_, "cuda_stream");
    if (!value) throw Raised{};
    const unsigned long long raw = PyLong_AsUnsignedLongLong(value);
    Py_DECREF(value);
    if (PyErr_Occurred()) throw Raised{};
    const auto s = reinterpret_cast<dcopy_stream_t>((uintptr_t)raw);
    on_stream_.emplace(torch_stream(s));
    return s;
  }
  c10::cuda::CUDAStream torch_stream(dcopy_stream_t s) const {
    return c10::cuda::getStreamFromExternal(reinterpret_cast<cudaStream_t>(s),
                                            (c10::DeviceIndex)device_);
  }
  // The given workspace, or one from the allocator: of the pool of the call's stream, so
  // that neither a block's last user nor its next can meet the call's kernels.
  void *workspace(PyObject *o, uint64_t need, uint64_t *bytes) {
    if (o != Py_None) {
      const at::Tensor &t = tensor(o, "workspace");
      if (!t.is_contiguous()) value_error("workspace", "expected a contiguous tensor");
      *bytes = t.nbytes();
      return const_cast<void *>(t.const_data_ptr());
    }
    scratch_ = at::empty({(int64_t)need}, at::TensorOptions().dtype(at::kByte).device(
                                              at::Device(at::kCUDA, (c10::DeviceIndex)device_)));
    *bytes = need;
    return scratch_.mutable_data_ptr();
  }
  const at::Tensor &taken() const { return scratch_; }
  void check(int rc) {
    if (rc) dcopy_error(rc, lib.dcopy_last_error_message(), func_);
  }
  const char *func() const { return func_; }

 private:
  const char *func_;
  PyObject *given_;
  int64_t device_ = -1;
  std::optional<c10::cuda::CUDAGuard> guard_;
  std::optional<c10::cuda::CUDAStreamGuard> on_stream_;
  at::Tensor scratch_;
};

// Runs a call's body; C++ exceptions end here.
template <typename F>
PyObject *run(const char *func, PyObject *const *a, Py_ssize_t n, Py_ssize_t want, F &&body) {
  if (n != want) {
    PyErr_Format(PyExc_TypeError, "%s takes %zd arguments", func, want);
    return nullptr;
  }
  if (!lib.dcopy_last_error_message) {
    PyErr_SetString(PyExc_RuntimeError, "dcopy._tensor_calls is not bound to the library");
    return nullptr;
  }
  try {
    Call call(func, a[n - 1]);  // the stream comes last
    body(call);
    Py_RETURN_NONE;
  } catch (const Raised &) {
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "internal exception");
  }
  return nullptr;
}

// Without the interpreter's lock: a launch may wait for room in the stream's queue.
template <typename F>
int unlocked(F &&f) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f();
  Py_END_ALLOW_THREADS
  return rc;
}

PyObject *embedding_lookup(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return run("dcopy_embedding_lookup", a, n, 6, [&](Call &c) {
    const DcopyMatrix out = c.matrix(a[0], "out"), table = c.matrix(a[1], "table"),
                      ids = c.matrix(a[2], "ids");
    const float scale = (float)as_double(a[3]);
    const int64_t first = as_int(a[4]);
    dcopy_stream_t s = c.stream();
    c.check(unlocked([&] { return lib.dcopy_embedding_lookup(&out, &table, &ids, first, scale, s); }));
  });
}

PyObject *embedding_grad(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return run("dcopy_embedding_grad", a, n, 8, [&](Call &c) {
    const DcopyMatrix grad = c.matrix(a[0], "grad"), dout = c.matrix(a[1], "dout"),
                      ids = c.matrix(a[2], "ids");
    const float scale = (float)as_double(a[3]);
    const int64_t first = as_int(a[4]);
    const int accumulate = as_bool(a[5]);
    dcopy_stream_t s = c.stream();
    uint64_t need = 0, bytes = 0;
    if (a[6] == Py_None)
      c.check(lib.dcopy_embedding_grad_workspace(ids.rows * ids.cols, grad.rows, grad.cols, &need));
    void *space = c.workspace(a[6], need, &bytes);
    c.check(unlocked([&] {
      return lib.dcopy_embedding_grad(&grad, &dout, &ids, first, scale, accumulate, space, bytes, s);
    }));
  });
}

PyObject *expert_sort(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return run("dcopy_expert_sort", a, n, 7, [&](Call &c) {
    int64_t entries = 0, rows = 0, ends = 0;
    auto *dest = (int32_t *)c.vector(a[0], "dest", at::kInt, &entries);
    auto *source = (int32_t *)c.vector(a[1], "source", at::kInt, &rows);
    auto *offsets = (int32_t *)c.vector(a[2], "offsets", at::kInt, &ends);
    const DcopyMatrix ids = c.matrix(a[3], "expert_ids");
    if (entries != ids.rows * ids.cols)
      dcopy_error(DCOPY_ERR_SHAPE_INVALID, "dest has " + std::to_string(entries) + " values for " +
                  std::to_string(ids.rows * ids.cols) + " choices", c.func());
    const int32_t align = (int32_t)as_int(a[4]), experts = (int32_t)(ends - 1);
    dcopy_stream_t s = c.stream();
    uint64_t need = 0, bytes = 0;
    if (a[5] == Py_None) c.check(lib.dcopy_expert_sort_workspace(entries, experts, &need));
    void *space = c.workspace(a[5], need, &bytes);
    c.check(unlocked([&] {
      return lib.dcopy_expert_sort(dest, source, rows, offsets, &ids, experts, align, space, bytes, s);
    }));
  });
}

// dest and source of a routing of `tokens` tokens into `rows` rows.  A flat dest has as
// many slots as divide it over the tokens, without tokens those of the weights.
struct Routing {
  const int32_t *dest, *source;
  int64_t slots;
};
Routing routing(Call &c, PyObject *dest, PyObject *source, int64_t tokens, int64_t rows,
                const DcopyMatrix &weights) {
  Routing r{};
  int64_t n = 0, held = rows;
  const at::Tensor &d = unpack(dest, "dest");
  r.dest = (const int32_t *)c.vector(dest, "dest", at::kInt, &n);
  r.source = (const int32_t *)c.vector(source, "source", at::kInt, &held);
  if (d.dim() > 1) r.slots = d.size(-1);
  else r.slots = tokens ? n / tokens : weights.cols;
  if (r.slots * tokens != n)
    dcopy_error(DCOPY_ERR_SHAPE_INVALID, "dest has " + std::to_string(n) + " values for " +
                std::to_string(tokens) + " tokens", c.func());
  if (held != rows)
    dcopy_error(DCOPY_ERR_SHAPE_INVALID, "source has " + std::to_string(held) + " values for " +
                std::to_string(rows) + " rows", c.func());
  return r;
}

PyObject *expert_dispatch(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return run("dcopy_expert_dispatch", a, n, 6, [&](Call &c) {
    const DcopyMatrix out = c.matrix(a[0], "out"), x = c.matrix(a[1], "x");
    DcopyMatrix weights{};
    const bool weighted = a[4] != Py_None;
    if (weighted) weights = c.matrix(a[4], "weights");
    const Routing r = routing(c, a[2], a[3], x.rows, out.rows, weights);
    dcopy_stream_t s = c.stream();
    c.check(unlocked([&] {
      return lib.dcopy_expert_dispatch(&out, &x, r.dest, r.slots, r.source,
                                       weighted ? &weights : nullptr, s);
    }));
  });
}

PyObject *expert_combine(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return run("dcopy_expert_combine", a, n, 5, [&](Call &c) {
    const DcopyMatrix out = c.matrix(a[0], "out"), y = c.matrix(a[1], "y");
    DcopyMatrix weights{};
    const bool weighted = a[3] != Py_None;
    if (weighted) weights = c.matrix(a[3], "weights");
    const Routing r = routing(c, a[2], Py_None, out.rows, y.rows, weights);
    dcopy_stream_t s = c.stream();
    c.check(unlocked([&] {
      return lib.dcopy_expert_combine(&out, &y, r.dest, r.slots, weighted ? &weights : nullptr, s);
    }));
  });
}

PyObject *expert_combine_grad(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return run("dcopy_expert_combine_grad", a, n, 8, [&](Call &c) {
    const DcopyMatrix dy = c.matrix(a[0], "dy"), dw = c.matrix(a[1], "dweights"),
                      dout = c.matrix(a[2], "dout"), y = c.matrix(a[3], "y"),
                      weights = c.matrix(a[5], "weights");
    const Routing r = routing(c, a[4], a[6], dout.rows, dy.rows, weights);
    dcopy_stream_t s = c.stream();
    c.check(unlocked([&] {
      return lib.dcopy_expert_combine_grad(&dy, &dw, &dout, &y, r.dest, r.slots, r.source, &weights,
                                           s);
    }));
  });
}

// A list of gradients as Python holds it: (address of the DcopyGradList, device, the tensors
// that it keeps, the streams they are known to be used on).
struct Gradients {
  const DcopyGradList *list;
  PyObject *tensors, *streams;
};
Gradients gradients(Call &c, PyObject *o) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4 || !PyList_Check(PyTuple_GET_ITEM(o, 2)) ||
      !PySet_Check(PyTuple_GET_ITEM(o, 3)))
    value_error("gradients", "expected a GradList");
  c.on_device(as_int(PyTuple_GET_ITEM(o, 1)));
  return {reinterpret_cast<const DcopyGradList *>((uintptr_t)as_int(PyTuple_GET_ITEM(o, 0))),
          PyTuple_GET_ITEM(o, 2), PyTuple_GET_ITEM(o, 3)};
}

// Tells the allocator of a list's first use on a stream: its memory, should the list be
// dropped, waits for what that stream holds by then.
void use_on(const Gradients &g, Call &c, dcopy_stream_t s) {
  PyObject *key = PyLong_FromVoidPtr(s);
  const int known = key ? PySet_Contains(g.streams, key) : -1;
  if (known == 0) {
    const auto stream = c.torch_stream(s);
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(g.tensors); ++i)
      c10::cuda::CUDACachingAllocator::recordStream(
          unpack(PyList_GET_ITEM(g.tensors, i), "gradient").storage().data_ptr(), stream);
  }
  const bool failed = known < 0 || (known == 0 && PySet_Add(g.streams, key));
  Py_XDECREF(key);
  if (failed) throw Raised{};
}

PyObject *grad_sum_squares(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return run("dcopy_grad_sum_squares", a, n, 3, [&](Call &c) {
    const Gradients g = gradients(c, a[0]);
    auto *total = (double *)c.vector(a[1], "total", at::kDouble);
    dcopy_stream_t s = c.stream();
    use_on(g, c, s);
    c.check(unlocked([&] { return lib.dcopy_grad_sum_squares(g.list, total, s); }));
  });
}

PyObject *grad_clip(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return run("dcopy_grad_clip", a, n, 6, [&](Call &c) {
    const Gradients g = gradients(c, a[0]);
    auto *total = (const double *)c.vector(a[1], "total", at::kDouble);
    const float max_norm = (float)as_double(a[2]), eps = (float)as_double(a[3]);
    auto *norm = (float *)c.vector(a[4], "norm", at::kFloat);
    dcopy_stream_t s = c.stream();
    use_on(g, c, s);
    c.check(unlocked([&] { return lib.dcopy_grad_clip(g.list, total, max_norm, eps, norm, s); }));
  });
}

PyObject *clip_grad_norm(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return run("dcopy_clip_grad_norm", a, n, 5, [&](Call &c) {
    const Gradients g = gradients(c, a[0]);
    const float max_norm = (float)as_double(a[1]), eps = (float)as_double(a[2]);
    auto *norm = (float *)c.vector(a[3], "norm", at::kFloat);
    dcopy_stream_t s = c.stream();
    use_on(g, c, s);
    c.check(unlocked([&] { return lib.dcopy_clip_grad_norm(g.list, max_norm, eps, norm, s); }));
  });
}

// scratch(bytes, device, stream) -> (tensor, the stream's handle): memory of that stream's
// pool, by default the current one's.
PyObject *scratch(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 3) {
    PyErr_SetString(PyExc_TypeError, "scratch takes 3 arguments");
    return nullptr;
  }
  try {
    Call c("scratch", a[2]);
    c.on_device(as_int(a[1]));
    dcopy_stream_t s = c.stream();
    uint64_t bytes = 0;
    c.workspace(Py_None, (uint64_t)as_int(a[0]), &bytes);
    return Py_BuildValue("NN", THPVariable_Wrap(c.taken()), PyLong_FromVoidPtr(s));
  } catch (const Raised &) {
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// fill_grads(address, grads, outs) -> device: DcopyGrad records of two lists of tensors.
PyObject *fill_grads(PyObject *, PyObject *const *a, Py_ssize_t n) {
  try {
    if (n != 3 || !PyList_Check(a[1]) || !PyList_Check(a[2]))
      value_error("fill_grads", "expected an address and two lists");
    auto *record = reinterpret_cast<DcopyGrad *>((uintptr_t)as_int(a[0]));
    const Py_ssize_t count = PyList_Size(a[1]);
    if (PyList_Size(a[2]) != count) value_error("out", "needs a tensor for each gradient");
    int64_t device = -1;
    for (Py_ssize_t i = 0; i < count; ++i) {
      const at::Tensor &g = unpack(PyList_GetItem(a[1], i), "gradient");
      const at::Tensor &o = unpack(PyList_GetItem(a[2], i), "out");
      const std::string name = "gradient " + std::to_string(i);
      if (!g.is_cuda() || !o.is_cuda() || !g.is_contiguous() || !o.is_contiguous())
        value_error(name.c_str(), "expected contiguous CUDA tensors");
      if (g.numel() != o.numel())
        value_error(name.c_str(), std::to_string(g.numel()) + " elements for " +
                                      std::to_string(o.numel()));
      if (device < 0) device = g.get_device();
      if (g.get_device() != device || o.get_device() != device)
        value_error(name.c_str(), "tensors are on different devices");
      record[i] = DcopyGrad{g.const_data_ptr(), const_cast<void *>(o.const_data_ptr()),
                            (uint64_t)g.numel(), type_code(g.scalar_type()),
                            type_code(o.scalar_type())};
    }
    return PyLong_FromLongLong(device);
  } catch (const Raised &) {
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// layout(tensor) -> (rows, cols, pitch, type): how a call sees a tensor, on any device.
PyObject *layout_of(PyObject *, PyObject *o) {
  try {
    const DcopyMatrix m = layout(unpack(o, "tensor"), "tensor");
    return Py_BuildValue("LLLi", (long long)m.rows, (long long)m.cols, (long long)m.pitch, m.type);
  } catch (const Raised &) {
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// bind({name: address}, DcopyError)
PyObject *bind(PyObject *, PyObject *args) {
  PyObject *addresses = nullptr, *error = nullptr;
  if (!PyArg_ParseTuple(args, "O!O", &PyDict_Type, &addresses, &error)) return nullptr;
  Library found;
#define X(name)                                                                 \
  {                                                                             \
    PyObject *v = PyDict_GetItemString(addresses, #name);                       \
    void *p = v ? PyLong_AsVoidPtr(v) : nullptr;                                \
    if (!p) {                                                                   \
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_KeyError, #name);            \
      return nullptr;                                                           \
    }                                                                           \
    found.name = reinterpret_cast<decltype(&::name)>(p);                        \
  }
  DCOPY_CALLS(X)
#undef X
  lib = found;
  Py_XSETREF(error_class, Py_NewRef(error));
  Py_RETURN_NONE;
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    FAST(embedding_lookup), FAST(embedding_grad), FAST(expert_sort), FAST(expert_dispatch),
    FAST(expert_combine), FAST(expert_combine_grad), FAST(grad_sum_squares), FAST(grad_clip),
    FAST(clip_grad_norm), FAST(fill_grads), FAST(scratch),
    {"layout", layout_of, METH_O, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_calls", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_calls(void) { return PyModule_Create(&module); }

// The operators' calls in native code: one object per bound kernel that takes the operand tensors, allocates the result and
// launches on torch's current stream.
//
// A small call is as long as its host code.  Of the 5 us that a call took from Python (softmax of 64 x 512 4.9 us), the HIP
// launch itself is 2.4; the rest was the allocation through torch's argument parser (0.9 to 1.4 us), packing the arguments, the
// foreign-function call and two look-ups of the stream.  This does them in one step.
//
//   Launch(entry, handle, dims, num_pointers, num_scalars, fail, keep)
//       entry      address of kcg_hip_launch_packed (include/kcg_hip.h): the library itself is not linked
//       handle     kernel handle
//       dims       seven whole numbers: grid, block, LDS bytes
//       fail       called with a status that is not 0; raises
//       keep       any object that has to live as long
//   launch(pointer, ..., number, ...)      pointers as whole numbers or tensors; numbers as fp32
//   launch.result(shape, dtype)            a Launch whose call leaves the last pointer out: call(tensor, ..., number, ...)
//                                          allocates it on the first tensor's device and returns it
//   launch.result(None, None)              the result is like the first tensor
//   launch.results((shape, dtype), ...)    a Launch whose call leaves the last pointers out and returns a tuple of their tensors,
//                                          parts of one allocation
//   signature(tensor or None, ...)         what a kernel can depend on of its operands, as bytes: device, type, sizes, strides and how
//                                          far each address is from a multiple of 16
//   row_signature(tensor or None, ...)     the same without the last size and the strides before the last
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <cstdint>
#include <cstring>
#include <vector>

namespace {

typedef int (*Entry)(void* handle, const uint32_t* dims, void* stream, const void* slots, int num_args);
constexpr int MAX_ARGS = 16;      // as many as the entry takes

struct Launch {
  PyObject_HEAD
  vectorcallfunc call;
  Entry entry;
  void* handle;
  uint32_t dims[7];
  int pointers, scalars;
  int result;                     // 0: no result, 1: shape and dtype, 2: like the first tensor, 3: several
  std::vector<std::pair<std::vector<int64_t>, at::ScalarType>>* several;
  std::vector<int64_t>* shape;
  at::ScalarType dtype;
  PyObject *fail, *keep;
};

// The launch on the current stream, without the GIL; the status of the entry.
int launch(const Launch* self, const uint64_t* slots) {
  void* stream = (void*)c10::hip::getCurrentHIPStream().stream();
  return self->entry(self->handle, self->dims, stream, slots, self->pointers + self->scalars);
}

// A new tensor on `like`'s device: on the part without the dispatcher, which takes as long as the allocation itself, unless a mode
// (torch.utils._python_dispatch) looks at what is called.
at::Tensor fresh(const at::Tensor& like, at::IntArrayRef shape, at::ScalarType dtype) {
  if (like.is_cuda() && !c10::impl::dispatch_mode_enabled()) return at::Tensor(at::detail::empty_cuda(shape, dtype, like.device(), std::nullopt));
  return at::empty(shape, like.options().dtype(dtype).requires_grad(false));
}

// The bytes of a result, up to the next multiple of 256.
int64_t bytesOf(const std::vector<int64_t>& shape, at::ScalarType dtype) {
  int64_t n = (int64_t)c10::elementSize(dtype);
  for (int64_t s : shape) n *= s;
  return (n + 255) / 256 * 256;
}

bool scalar(PyObject* o, uint64_t& slot) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) return false;
  // a number beyond the fp32 range is an infinity, as the conversion to a C float gives it
  const float f = v > 3.4028235677973366e38 ? INFINITY : v < -3.4028235677973366e38 ? -INFINITY : (float)v;
  slot = 0;
  memcpy(&slot, &f, sizeof f);
  return true;
}

PyObject* failed(Launch* self, int rc) {
  PyObject* r = PyObject_CallFunction(self->fail, "i", rc);
  if (r) {
    Py_DECREF(r);
    PyErr_Format(PyExc_RuntimeError, "kernel launch failed with status %d", rc);
  }
  return nullptr;
}

PyObject* callLaunch(PyObject* me, PyObject* const* args, size_t nargsf, PyObject* kwnames) {
  HANDLE_TH_ERRORS
  Launch* self = (Launch*)me;
  const Py_ssize_t n = PyVectorcall_NARGS(nargsf);
  const int given = self->pointers - (self->result == 3 ? (int)self->several->size() : self->result ? 1 : 0);
  if ((kwnames && PyTuple_GET_SIZE(kwnames)) || n != given + self->scalars) {
    PyErr_Format(PyExc_TypeError, "a launch of this kernel takes %d pointers and %d numbers", given, self->scalars);
    return nullptr;
  }
  uint64_t slots[MAX_ARGS];
  for (int i = 0; i < given; ++i) {
    if (THPVariable_Check(args[i])) {
      slots[i] = (uint64_t)(uintptr_t)THPVariable_Unpack(args[i]).data_ptr();
    } else {
      PyObject* whole = PyNumber_Index(args[i]);
      if (!whole) return nullptr;
      slots[i] = PyLong_AsUnsignedLongLong(whole);
      Py_DECREF(whole);
      if (slots[i] == (uint64_t)-1 && PyErr_Occurred()) return nullptr;
    }
  }
  for (int i = 0; i < self->scalars; ++i)
    if (!scalar(args[given + i], slots[self->pointers + i])) return nullptr;
  int rc;
  if (!self->result) {
    {
      pybind11::gil_scoped_release unlocked;      // (an exception takes it back)
      rc = launch(self, slots);
    }
    if (rc) return failed(self, rc);
    Py_RETURN_NONE;
  }
  if (!given || !THPVariable_Check(args[0])) {
    PyErr_SetString(PyExc_TypeError, "the first operand must be a tensor");
    return nullptr;
  }
  if (self->result == 3) {
    std::vector<at::Tensor> outs;
    outs.reserve(self->several->size());
    {
      const at::Tensor& like = THPVariable_Unpack(args[0]);
      pybind11::gil_scoped_release unlocked;
      // one allocation, of which each result is a part that begins at a multiple of 256 bytes: one each takes 0.6 us
      int64_t bytes = 0;
      for (const auto& [shape, dtype] : *self->several) bytes += bytesOf(shape, dtype);
      const at::Tensor all = fresh(like, {bytes}, at::kByte);
      int64_t at = 0;
      for (const auto& [shape, dtype] : *self->several) {
        auto part = c10::make_intrusive<at::TensorImpl>(c10::Storage(all.storage()), all.key_set(), c10::scalarTypeToTypeMeta(dtype));
        part->set_storage_offset(at / (int64_t)c10::elementSize(dtype));
        part->set_sizes_contiguous(shape);
        outs.emplace_back(std::move(part));
        slots[given + outs.size() - 1] = (uint64_t)(uintptr_t)all.data_ptr() + (uint64_t)at;
        at += bytesOf(shape, dtype);
      }
      rc = launch(self, slots);
    }
    if (rc) return failed(self, rc);
    PyObject* tuple = PyTuple_New((Py_ssize_t)outs.size());
    if (!tuple) return nullptr;
    for (size_t i = 0; i < outs.size(); ++i) {
      PyObject* o = THPVariable_Wrap(outs[i]);
      if (!o) {
        Py_DECREF(tuple);
        return nullptr;
      }
      PyTuple_SET_ITEM(tuple, (Py_ssize_t)i, o);
    }
    return tuple;
  }
  at::Tensor out;
  {
    const at::Tensor& like = THPVariable_Unpack(args[0]);
    pybind11::gil_scoped_release unlocked;
    out = self->result == 2 ? at::empty_like(like) : fresh(like, *self->shape, self->dtype);
    slots[given] = (uint64_t)(uintptr_t)out.data_ptr();
    rc = launch(self, slots);
  }
  if (rc) return failed(self, rc);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

PyTypeObject LaunchType = {PyVarObject_HEAD_INIT(nullptr, 0)};

PyObject* newLaunch(PyTypeObject* type, PyObject* args, PyObject* kwargs) {
  HANDLE_TH_ERRORS
  unsigned long long entry, handle;
  unsigned int d[7];
  int pointers, scalars;
  PyObject *fail, *keep;
  if ((kwargs && PyDict_GET_SIZE(kwargs)) ||
      !PyArg_ParseTuple(args, "KK(IIIIIII)iiOO", &entry, &handle, &d[0], &d[1], &d[2], &d[3], &d[4], &d[5], &d[6], &pointers, &scalars, &fail, &keep)) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "Launch takes no keyword arguments");
    return nullptr;
  }
  if (!entry || !handle || pointers < 1 || scalars < 0 || pointers + scalars > MAX_ARGS) {
    PyErr_SetString(PyExc_ValueError, "Launch: no entry, no kernel, or not 1 to 16 arguments");
    return nullptr;
  }
  Launch* self = (Launch*)type->tp_alloc(type, 0);
  if (!self) return nullptr;
  self->call = callLaunch;
  self->entry = (Entry)(uintptr_t)entry;
  self->handle = (void*)(uintptr_t)handle;
  memcpy(self->dims, d, sizeof d);
  self->pointers = pointers;
  self->scalars = scalars;
  self->result = 0;
  self->shape = nullptr;
  self->several = nullptr;
  Py_INCREF(fail);
  self->fail = fail;
  Py_INCREF(keep);
  self->keep = keep;
  return (PyObject*)self;
  END_HANDLE_TH_ERRORS
}

// The sizes and type of a result; false with an error set.
bool shapeOf(PyObject* shape, PyObject* dtype, std::vector<int64_t>& sizes) {
  PyObject* seq = PySequence_Fast(shape, "the shape is a sequence of whole numbers");
  if (!seq) return false;
  for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(seq); ++i) {
    const long long v = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(seq, i));
    if (v == -1 && PyErr_Occurred()) {
      Py_DECREF(seq);
      return false;
    }
    sizes.push_back(v);
  }
  Py_DECREF(seq);
  if (!THPDtype_Check(dtype)) {
    PyErr_SetString(PyExc_TypeError, "a shape needs a torch dtype");
    return false;
  }
  return true;
}

// A Launch of the same kernel; what it gives is set by the caller.
Launch* again(Launch* self) {
  Launch* made = (Launch*)LaunchType.tp_alloc(&LaunchType, 0);
  if (!made) return nullptr;
  made->call = callLaunch;
  made->entry = self->entry;
  made->handle = self->handle;
  memcpy(made->dims, self->dims, sizeof made->dims);
  made->pointers = self->pointers;
  made->scalars = self->scalars;
  made->result = 0;
  made->shape = nullptr;
  made->several = nullptr;
  Py_INCREF(self->fail);
  made->fail = self->fail;
  Py_INCREF(self->keep);
  made->keep = self->keep;
  return made;
}

PyObject* withResult(PyObject* me, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *shape, *dtype;
  if (!PyArg_ParseTuple(args, "OO", &shape, &dtype)) return nullptr;
  std::vector<int64_t> sizes;
  if (shape != Py_None && !shapeOf(shape, dtype, sizes)) return nullptr;
  Launch* made = again((Launch*)me);
  if (!made) return nullptr;
  made->result = shape == Py_None ? 2 : 1;
  if (shape != Py_None) {
    made->shape = new std::vector<int64_t>(std::move(sizes));
    made->dtype = ((THPDtype*)dtype)->scalar_type;
  }
  return (PyObject*)made;
  END_HANDLE_TH_ERRORS
}

PyObject* withResults(PyObject* me, PyObject* args) {
  HANDLE_TH_ERRORS
  std::vector<std::pair<std::vector<int64_t>, at::ScalarType>> several;
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args); ++i) {
    PyObject *shape, *dtype;
    if (!PyArg_ParseTuple(PyTuple_GET_ITEM(args, i), "OO", &shape, &dtype)) return nullptr;
    several.emplace_back();
    if (!shapeOf(shape, dtype, several.back().first)) return nullptr;
    several.back().second = ((THPDtype*)dtype)->scalar_type;
  }
  if (several.empty() || (int)several.size() >= ((Launch*)me)->pointers) {
    PyErr_SetString(PyExc_ValueError, "results: one or more, and fewer than the kernel has pointers");
    return nullptr;
  }
  Launch* made = again((Launch*)me);
  if (!made) return nullptr;
  made->result = 3;
  made->several = new std::vector<std::pair<std::vector<int64_t>, at::ScalarType>>(std::move(several));
  return (PyObject*)made;
  END_HANDLE_TH_ERRORS
}

// `rows`: without what a kernel takes as arguments of tensors whose rows it walks over, the length of a row and how far rows are apart.
// Rows of one element or none are rows of neighbouring elements.
template <bool rows>
PyObject* signatureOf(PyObject* const* args, Py_ssize_t n) {
  // (a tensor of d dimensions takes 2 d + 2 numbers of 8 bytes)
  int64_t out[256];
  size_t at = 0;
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (args[i] == Py_None) {
      if (at + 1 > 256) break;
      out[at++] = -1;
      continue;
    }
    if (!THPVariable_Check(args[i])) {
      PyErr_SetString(PyExc_TypeError, "operands must be tensors");
      return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(args[i]);
    const int64_t d = t.dim();
    if (at + 2 * d + 2 > 256) {
      PyErr_SetString(PyExc_ValueError, "too many dimensions");
      return nullptr;
    }
    const auto device = t.device();
    out[at++] = d | (int64_t)t.scalar_type() << 8 | (int64_t)device.type() << 16 | (int64_t)(uint8_t)device.index() << 24 |
                (int64_t)t.layout() << 32;
    if (rows) {
      for (int64_t j = 0; j + 1 < d; ++j) out[at++] = t.size(j);
      if (d) out[at++] = t.size(d - 1) > 1 ? t.stride(d - 1) : 1;
    } else {
      for (int64_t j = 0; j < d; ++j) out[at++] = t.size(j);
      for (int64_t j = 0; j < d; ++j) out[at++] = t.stride(j);
    }
    out[at++] = (int64_t)((uintptr_t)t.data_ptr() & 15);
  }
  return PyBytes_FromStringAndSize((const char*)out, (Py_ssize_t)(at * sizeof out[0]));
}

PyObject* signature(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  return signatureOf<false>(args, n);
  END_HANDLE_TH_ERRORS
}

PyObject* rowSignature(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  return signatureOf<true>(args, n);
  END_HANDLE_TH_ERRORS
}

void freeLaunch(PyObject* me) {
  Launch* self = (Launch*)me;
  delete self->shape;
  delete self->several;
  Py_XDECREF(self->fail);
  Py_XDECREF(self->keep);
  Py_TYPE(me)->tp_free(me);
}

PyMethodDef methods[] = {{"result", withResult, METH_VARARGS, "result(shape, dtype): a Launch that allocates and returns its last pointer's tensor"},
                         {"results", withResults, METH_VARARGS, "results((shape, dtype), ...): a Launch that allocates and returns its last pointers' tensors"},
                         {nullptr, nullptr, 0, nullptr}};
PyMethodDef functions[] = {{"signature", (PyCFunction)(void (*)(void))signature, METH_FASTCALL, "what a kernel can depend on of its operands"},
                           {"row_signature", (PyCFunction)(void (*)(void))rowSignature, METH_FASTCALL, "the same without the rows' length and distance"},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_launch", "bound kernel launches on torch tensors", -1, functions};

}  // namespace

PyMODINIT_FUNC PyInit__launch(void) {
  LaunchType.tp_name = "kernelcodegen_amd._launch.Launch";
  LaunchType.tp_basicsize = sizeof(Launch);
  LaunchType.tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL;
  LaunchType.tp_vectorcall_offset = offsetof(Launch, call);
  LaunchType.tp_call = PyVectorcall_Call;
  LaunchType.tp_new = newLaunch;
  LaunchType.tp_dealloc = freeLaunch;
  LaunchType.tp_methods = methods;
  if (PyType_Ready(&LaunchType) < 0) return nullptr;
  PyObject* m = PyModule_Create(&module);
  if (!m) return nullptr;
  Py_INCREF(&LaunchType);
  if (PyModule_AddObject(m, "Launch", (PyObject*)&LaunchType) < 0) {
    Py_DECREF(&LaunchType);
    Py_DECREF(m);
    return nullptr;
  }
  // the version whose headers this was built on (torch.__version__), for the importer to compare
  if (PyModule_AddStringConstant(m, "torch_version", KCG_TORCH_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}

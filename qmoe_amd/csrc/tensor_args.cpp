// What the Python side of a call does with its tensors, in C++: looks each of
// them over and hands back their addresses.
//
// A call on a small matrix or a few tokens takes as long as Python needs for it, and a
// layer of 128 experts has 768 tensors.  Looking at a tensor's type, device, strides and
// size from Python costs 0.4 us, here 0.03: the operator's six tensors 2.3 -> 0.4 us, a
// layer's 768 112 -> 22.
//
// Nothing is decided here: whatever is not plainly in order (no tensor, a subclass of
// one, another device, type, size or layout, no memory of its own) is answered with
// None or False, and the caller then takes its slow way, which raises the error that
// belongs to it.  No state is kept.
//
// The calls on microscaled 4-bit matrices go all the way here: tensors looked over, results
// made, the library's entry called (its address comes from the caller, which has the library).
// Host time of a product 8.7 -> 4.4 us, of a sparse MLP's call 36 -> 18 (14 with three launches).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>

#include <cstdint>

#include "sub1_hip.h"

namespace {

// The address of a plain contiguous tensor on GPU `device`, of this type and (unless negative)
// this number of elements and dimensions; null if it is anything else.  An empty tensor has
// no address to find: the caller learns that it is in order through `fine`.
void *address_of(PyObject *object, PyObject *dtype, int64_t numel, int64_t dims, int64_t device, bool *fine) {
  *fine = false;
  if (!THPVariable_CheckExact(object) || !THPDtype_Check(dtype)) return nullptr;
  try {
    const at::Tensor &t = THPVariable_Unpack(object);
    if (!t.defined() || !t.is_cuda() || t.device().index() != device ||
        t.scalar_type() != reinterpret_cast<THPDtype *>(dtype)->scalar_type || !t.is_contiguous() ||
        (numel >= 0 && t.numel() != numel) || (dims >= 0 && t.dim() != dims))
      return nullptr;
    void *p = t.data_ptr();
    *fine = true;
    return p;
  } catch (...) {   // a tensor without memory: the slow way has the error for it
    return nullptr;
  }
}

bool integer(PyObject *object, int64_t *out) {
  if (!PyLong_Check(object)) return false;
  *out = PyLong_AsLongLong(object);
  if (*out == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

// addresses(spec, tensors, numels, device): spec[i] = (dtype, name, dims), all of them tuples.
PyObject *addresses(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "addresses(spec, tensors, numels, device)");
    return nullptr;
  }
  PyObject *spec = args[0], *tensors = args[1], *numels = args[2];
  int64_t device;
  if (!PyTuple_Check(spec) || !PyTuple_Check(tensors) || !PyTuple_Check(numels) || !integer(args[3], &device) ||
      PyTuple_GET_SIZE(spec) != PyTuple_GET_SIZE(tensors) || PyTuple_GET_SIZE(numels) != PyTuple_GET_SIZE(tensors))
    Py_RETURN_NONE;
  const Py_ssize_t count = PyTuple_GET_SIZE(tensors);
  PyObject *out = PyTuple_New(count);
  if (!out) return nullptr;
  for (Py_ssize_t i = 0; i < count; i++) {
    PyObject *what = PyTuple_GET_ITEM(spec, i);
    int64_t numel, dims;
    bool fine = PyTuple_Check(what) && PyTuple_GET_SIZE(what) == 3 &&
                integer(PyTuple_GET_ITEM(numels, i), &numel) && integer(PyTuple_GET_ITEM(what, 2), &dims);
    void *p = fine ? address_of(PyTuple_GET_ITEM(tensors, i), PyTuple_GET_ITEM(what, 0), numel, dims, device, &fine)
                   : nullptr;
    if (!fine) {
      Py_DECREF(out);
      Py_RETURN_NONE;
    }
    PyObject *address = PyLong_FromUnsignedLongLong(reinterpret_cast<uintptr_t>(p));
    if (!address) {
      Py_DECREF(out);
      return nullptr;
    }
    PyTuple_SET_ITEM(out, i, address);
  }
  return out;
}

// layer_addresses(table, row, layers, spec, numels, device): the addresses of layers[e][c] into
// table[row + c][e], an int64 tensor in host memory with a column per layer; False if some are not
// in order (what the table then holds is not to be used).
PyObject *layer_addresses(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != 6) {
    PyErr_SetString(PyExc_TypeError, "layer_addresses(table, row, layers, spec, numels, device)");
    return nullptr;
  }
  PyObject *layers = args[2], *spec = args[3], *numels = args[4];
  int64_t row, device, want[8], dims[8];
  if (!THPVariable_CheckExact(args[0]) || !integer(args[1], &row) || !PyList_Check(layers) || !PyTuple_Check(spec) ||
      !PyTuple_Check(numels) || !integer(args[5], &device) || PyTuple_GET_SIZE(spec) > 8 ||
      PyTuple_GET_SIZE(numels) != PyTuple_GET_SIZE(spec))
    Py_RETURN_FALSE;
  const Py_ssize_t count = PyList_GET_SIZE(layers), columns = PyTuple_GET_SIZE(spec);
  int64_t *table = nullptr;
  try {
    const at::Tensor &t = THPVariable_Unpack(args[0]);
    if (!t.defined() || !t.is_cpu() || t.scalar_type() != at::kLong || t.dim() != 2 || !t.is_contiguous() ||
        t.size(1) != count || row < 0 || row > t.size(0) - columns)
      Py_RETURN_FALSE;
    table = static_cast<int64_t *>(t.data_ptr()) + row * count;
  } catch (...) {
    Py_RETURN_FALSE;
  }
  for (Py_ssize_t c = 0; c < columns; c++) {
    PyObject *what = PyTuple_GET_ITEM(spec, c);
    if (!PyTuple_Check(what) || PyTuple_GET_SIZE(what) != 3 || !integer(PyTuple_GET_ITEM(numels, c), &want[c]) ||
        !integer(PyTuple_GET_ITEM(what, 2), &dims[c]))
      Py_RETURN_FALSE;
  }
  for (Py_ssize_t e = 0; e < count; e++) {
    PyObject *layer = PyList_GET_ITEM(layers, e);
    if (!PyTuple_Check(layer) || PyTuple_GET_SIZE(layer) != columns) Py_RETURN_FALSE;
    for (Py_ssize_t c = 0; c < columns; c++) {
      bool fine;
      void *p = address_of(PyTuple_GET_ITEM(layer, c), PyTuple_GET_ITEM(PyTuple_GET_ITEM(spec, c), 0), want[c],
                           dims[c], device, &fine);
      if (!fine) Py_RETURN_FALSE;
      table[c * count + e] = static_cast<int64_t>(reinterpret_cast<uintptr_t>(p));
    }
  }
  Py_RETURN_TRUE;
}

// ---- calls on microscaled 4-bit matrices ----

// The tensor behind a plain one on GPU `device`; null if it is anything else, one whose values torch negates when it reads
// them among it.
const at::Tensor *plain(PyObject *object, int64_t device) {
  if (!THPVariable_CheckExact(object)) return nullptr;
  const at::Tensor &t = THPVariable_Unpack(object);
  return t.defined() && t.is_cuda() && t.device().index() == device && t.layout() == at::kStrided && !t.is_neg() ? &t : nullptr;
}

bool address(PyObject *object, void **out) {
  int64_t v;
  if (!integer(object, &v)) return false;
  *out = reinterpret_cast<void *>(v);
  return true;
}

constexpr int64_t blocks_of(int64_t width) { return (width + 31) / 32; }

// Rows that lie together, `ld` elements apart.
bool rows_of(const at::Tensor &x, int64_t *rows, int64_t *width, int64_t *ld) {
  if (x.dim() < 1) return false;
  *width = x.size(-1);
  if (*width < 1 || *width > SUB1_MX4_MAX_WIDTH) return false;
  *rows = x.numel() / *width;
  *ld = *width;
  if (x.is_contiguous()) return true;
  if (x.dim() != 2 || x.stride(1) != 1 || x.stride(0) < *width) return false;
  *ld = x.stride(0);
  return true;
}

bool matrix_in_format(const at::Tensor &codes, const at::Tensor &scales, int64_t width, int64_t dims) {
  if (codes.scalar_type() != at::kByte || scales.scalar_type() != at::kByte || codes.dim() != dims ||
      scales.dim() != dims || !codes.is_contiguous() || !scales.is_contiguous() || codes.size(-1) != 16 * blocks_of(width) ||
      scales.size(-1) != blocks_of(width) || reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16)
    return false;
  for (int64_t i = 0; i + 1 < dims; i++)
    if (codes.size(i) != scales.size(i) || codes.size(i) < 1 || codes.size(i) > (int64_t{1} << 30)) return false;
  return true;
}

at::Tensor like(const at::Tensor &x, int64_t last, at::ScalarType type) {
  auto sizes = x.sizes().vec();
  sizes.back() = last;
  return at::empty(sizes, x.options().dtype(type));
}

int type_of(const at::Tensor &x) {
  switch (x.scalar_type()) {
    case at::kBFloat16: return SUB1_MX4_BF16;
    case at::kHalf: return SUB1_MX4_FP16;
    case at::kFloat: return SUB1_MX4_FP32;
    default: return -1;
  }
}

// The results, or the status of a library's entry that refused.
PyObject *result(int status, std::initializer_list<at::Tensor> tensors) {
  if (status) return PyLong_FromLong(status);
  if (tensors.size() == 1) return THPVariable_Wrap(*tensors.begin());
  PyObject *out = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()));
  if (!out) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor &t : tensors) {
    PyObject *item = THPVariable_Wrap(t);
    if (!item) {
      Py_DECREF(out);
      return nullptr;
    }
    PyTuple_SET_ITEM(out, i++, item);
  }
  return out;
}

typedef decltype(&sub1_mx4_quantize) Quantize;
typedef decltype(&sub1_mx4_dequantize) Dequantize;
typedef decltype(&sub1_mx4_product) Product;
typedef decltype(&sub1_mx4_product_quantized) ProductQuantized;
typedef decltype(&sub1_mx4_layer_scratch_bytes) LayerBytes;
typedef decltype(&sub1_mx4_layer_forward) LayerForward;

int quantized(Quantize entry, const at::Tensor &x, int64_t rows, int64_t width, int64_t ld, void *stream, at::Tensor *codes,
              at::Tensor *scales) {
  *codes = like(x, 16 * blocks_of(width), at::kByte);
  *scales = like(x, blocks_of(width), at::kByte);
  return entry(x.data_ptr(), type_of(x), ld, rows, static_cast<int>(width), codes->data_ptr<uint8_t>(),
               scales->data_ptr<uint8_t>(), stream);
}

// mx4_quantize(entry, x, device, stream)
PyObject *mx4_quantize(PyObject *, PyObject *const *args, Py_ssize_t n) {
  void *entry, *stream;
  int64_t device, rows, width, ld;
  if (n != 4 || !address(args[0], &entry) || !integer(args[2], &device) || !address(args[3], &stream)) Py_RETURN_NONE;
  try {
    const at::Tensor *x = plain(args[1], device);
    if (!x || type_of(*x) < 0 || !rows_of(*x, &rows, &width, &ld) || rows < 1) Py_RETURN_NONE;
    at::Tensor codes, scales;
    const int status = quantized(reinterpret_cast<Quantize>(entry), *x, rows, width, ld, stream, &codes, &scales);
    return result(status, {codes, scales});
  } catch (...) {
    Py_RETURN_NONE;
  }
}

// mx4_dequantize(entry, codes, scales, width, dtype, device, stream)
PyObject *mx4_dequantize(PyObject *, PyObject *const *args, Py_ssize_t n) {
  void *entry, *stream;
  int64_t device, width;
  if (n != 7 || !address(args[0], &entry) || !integer(args[3], &width) || !THPDtype_Check(args[4]) ||
      !integer(args[5], &device) || !address(args[6], &stream) || width < 1 || width > SUB1_MX4_MAX_WIDTH)
    Py_RETURN_NONE;
  try {
    const at::Tensor *codes = plain(args[1], device), *scales = plain(args[2], device);
    if (!codes || !scales || codes->dim() < 1 || !matrix_in_format(*codes, *scales, width, codes->dim())) Py_RETURN_NONE;
    const at::ScalarType type = reinterpret_cast<THPDtype *>(args[4])->scalar_type;
    if (type != at::kBFloat16 && type != at::kHalf && type != at::kFloat) Py_RETURN_NONE;
    at::Tensor out = like(*codes, width, type);
    const int status = reinterpret_cast<Dequantize>(entry)(codes->data_ptr<uint8_t>(), scales->data_ptr<uint8_t>(),
                                                           out.numel() / width, static_cast<int>(width), out.data_ptr(),
                                                           type_of(out), width, stream);
    return result(status, {out});
  } catch (...) {
    Py_RETURN_NONE;
  }
}

// mx4_product(entry, None or the entry that quantizes x first, x, codes, scales, the matrix' width or 0 for x's, device,
// stream)
PyObject *mx4_product(PyObject *, PyObject *const *args, Py_ssize_t n) {
  void *entry, *quantize = nullptr, *stream;
  int64_t device, rows, width, ld, expected;
  if (n != 8 || !address(args[0], &entry) || (args[1] != Py_None && !address(args[1], &quantize)) ||
      !integer(args[5], &expected) || !integer(args[6], &device) || !address(args[7], &stream))
    Py_RETURN_NONE;
  try {
    const at::Tensor *x = plain(args[2], device), *codes = plain(args[3], device), *scales = plain(args[4], device);
    if (!x || !codes || !scales || x->scalar_type() != at::kBFloat16 || !rows_of(*x, &rows, &width, &ld) || rows < 1 ||
        rows > SUB1_MX4_MAX_TOKENS || (expected && width != expected) || !matrix_in_format(*codes, *scales, width, 2))
      Py_RETURN_NONE;
    const int64_t height = codes->size(0);
    if (height > SUB1_MX4_MAX_WIDTH) Py_RETURN_NONE;
    at::Tensor y = like(*x, height, at::kBFloat16);
    int status;
    if (quantize) {
      at::Tensor x_codes, x_scales;
      status = quantized(reinterpret_cast<Quantize>(quantize), *x, rows, width, ld, stream, &x_codes, &x_scales);
      if (status == SUB1_OK)
        status = reinterpret_cast<ProductQuantized>(entry)(
            codes->data_ptr<uint8_t>(), scales->data_ptr<uint8_t>(), static_cast<int>(height), static_cast<int>(width),
            x_codes.data_ptr<uint8_t>(), x_scales.data_ptr<uint8_t>(), y.data_ptr(), height, static_cast<int>(rows), stream);
    } else {
      status = reinterpret_cast<Product>(entry)(codes->data_ptr<uint8_t>(), scales->data_ptr<uint8_t>(),
                                                static_cast<int>(height), static_cast<int>(width), x->data_ptr(), ld,
                                                y.data_ptr(), height, static_cast<int>(rows), stream);
    }
    return result(status, {y});
  } catch (...) {
    Py_RETURN_NONE;
  }
}

// mx4_layer(entry, entry that says how much scratch memory, hidden, router, wi_codes, wi_scales, wo_codes,
// wo_scales, top_k, normalize, capacity, device, stream): (y, logits, index)
PyObject *mx4_layer(PyObject *, PyObject *const *args, Py_ssize_t n) {
  void *entry, *bytes_entry, *stream;
  int64_t top_k, normalize, capacity, device;
  if (n != 13 || !address(args[0], &entry) || !address(args[1], &bytes_entry) || !integer(args[8], &top_k) ||
      !integer(args[9], &normalize) || !integer(args[10], &capacity) || !integer(args[11], &device) ||
      !address(args[12], &stream) || capacity < 0 || capacity > (int64_t{1} << 30) || top_k < 1 ||
      top_k > SUB1_MX4_LAYER_TOP_K)
    Py_RETURN_NONE;
  try {
    const at::Tensor *t[6];
    for (int i = 0; i < 6; i++) {
      t[i] = plain(args[2 + i], device);
      if (!t[i] || !t[i]->is_contiguous()) Py_RETURN_NONE;
    }
    const at::Tensor &x = *t[0], &router = *t[1];
    if (x.scalar_type() != at::kBFloat16 || x.dim() < 2 || router.dim() != 2 || x.size(-1) != router.size(1) ||
        (router.scalar_type() != at::kBFloat16 && router.scalar_type() != at::kFloat))
      Py_RETURN_NONE;
    const int64_t experts = router.size(0), d_model = router.size(1);
    if (d_model < 1 || d_model > SUB1_MX4_MAX_WIDTH || experts < 1 || experts > SUB1_MX4_LAYER_EXPERTS) Py_RETURN_NONE;
    const int64_t tokens = x.numel() / d_model;
    if (tokens < 1 || tokens > SUB1_MX4_LAYER_TOKENS || t[2]->dim() != 3) Py_RETURN_NONE;
    const int64_t d_ff = t[2]->size(1);
    if (d_ff < 1 || d_ff > SUB1_MX4_MAX_WIDTH || !matrix_in_format(*t[2], *t[3], d_model, 3) ||
        !matrix_in_format(*t[4], *t[5], d_ff, 3) || t[2]->size(0) != experts || t[4]->size(0) != experts ||
        t[4]->size(1) != d_model)
      Py_RETURN_NONE;
    sub1_mx4_layer layer{router.data_ptr(), t[2]->data_ptr<uint8_t>(), t[3]->data_ptr<uint8_t>(), t[4]->data_ptr<uint8_t>(),
                         t[5]->data_ptr<uint8_t>(), static_cast<int32_t>(experts), static_cast<int32_t>(d_model),
                         static_cast<int32_t>(d_ff), static_cast<int32_t>(top_k), type_of(router),
                         normalize != 0, static_cast<int32_t>(capacity)};
    at::Tensor y = like(x, d_model, at::kBFloat16), logits = like(x, experts, at::kFloat), index = like(x, top_k, at::kLong);
    // of the call's own: two calls at once, on streams or in captured graphs, never share it
    at::Tensor scratch = at::empty({reinterpret_cast<LayerBytes>(bytes_entry)(&layer, static_cast<int>(tokens))},
                                   x.options().dtype(at::kByte));
    const int status = reinterpret_cast<LayerForward>(entry)(
        &layer, x.data_ptr(), static_cast<int>(tokens), capacity ? static_cast<int>(x.size(-2)) : 1, y.data_ptr(),
        logits.data_ptr<float>(), index.data_ptr<int64_t>(), scratch.data_ptr(), scratch.numel(), stream);
    return result(status, {y, logits, index});
  } catch (...) {
    Py_RETURN_NONE;
  }
}

PyMethodDef kMethods[] = {
    {"addresses", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(addresses)), METH_FASTCALL, nullptr},
    {"layer_addresses", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(layer_addresses)), METH_FASTCALL,
     nullptr},
    {"mx4_quantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(mx4_quantize)), METH_FASTCALL, nullptr},
    {"mx4_dequantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(mx4_dequantize)), METH_FASTCALL, nullptr},
    {"mx4_product", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(mx4_product)), METH_FASTCALL, nullptr},
    {"mx4_layer", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(mx4_layer)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_tensor_args", nullptr, -1, kMethods,
                       nullptr,               nullptr,        nullptr, nullptr};

}  // namespace

#ifndef SUB1_TORCH_VERSION
#error "the build says which torch these headers are of"
#endif
// The classes behind a tensor differ from one torch to the next and nothing in the library's symbols
// says so: whoever loads the module compares this with the torch it has.
PyMODINIT_FUNC PyInit__tensor_args() {
  PyObject *module = PyModule_Create(&kModule);
  if (module && PyModule_AddStringConstant(module, "built_against", "qmoe_amd, built against torch " SUB1_TORCH_VERSION) < 0) {
    Py_DECREF(module);
    return nullptr;
  }
  return module;
}

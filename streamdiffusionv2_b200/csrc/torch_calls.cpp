// PyTorch side of the 8-bit cache and key-span entry points: tensors in, the C ABI's views out.
//
// A call through ctypes costs 15 to 19 us of host time for these (eight tensors to look at, two dozen arguments to
// convert), more than their kernels take at the smallest sizes; from here it is a few.  Nothing is computed or kept:
// every tensor's shape, type, device and strides are compared, outputs and scratch come from PyTorch's allocator on the
// current stream (a recording graph's own pool while capturing, so that no two graphs share scratch), and the functions
// whose addresses bind() was given do the rest.
#include <Python.h>
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <initializer_list>
#include <string>

#include "../../include/sdv2.h"

namespace {

decltype(&sdv2_rope_kv_append_q8) g_append = nullptr;
decltype(&sdv2_kv_read_q8) g_read = nullptr;
decltype(&sdv2_attn_q8_scratch_bytes) g_q8_bytes = nullptr;
decltype(&sdv2_attn_kvcache_q8) g_q8 = nullptr;
decltype(&sdv2_attn_spans_scratch_bytes) g_spans_bytes = nullptr;
decltype(&sdv2_attn_spans) g_spans = nullptr;
PyObject* g_check = nullptr;  // check(code, what): raises for a negative code

struct Refused {  // a Python exception is set
};

[[noreturn]] void refuse(const std::string& what) {
  PyErr_SetString(PyExc_ValueError, what.c_str());
  throw Refused();
}

const at::Tensor& tensor(PyObject* o, const char* what, const char* name) {
  if (!THPVariable_Check(o)) refuse(std::string(what) + ": " + name + " must be a tensor");
  return THPVariable_Unpack(o);
}

std::string described(at::IntArrayRef shape, at::ScalarType type, const at::Device& device) {
  std::string s = std::string(at::toString(type)) + " [";
  for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
  return s + "] on " + device.str();
}

void expect(const at::Tensor& t, at::IntArrayRef shape, at::ScalarType type, const at::Device& device, const char* what,
            const char* name) {
  if (t.sizes() != shape || t.scalar_type() != type || t.device() != device)
    refuse(std::string(what) + ": " + name + " must be " + described(shape, type, device) + ", not " +
           described(t.sizes(), t.scalar_type(), t.device()));
}

// [rows, tokens, heads, head_dim] with contiguous head_dim.  A size-1 dimension may carry any stride: it gets a legal one.
sdv2_view view4(const at::Tensor& t, at::IntArrayRef shape, at::ScalarType type, const at::Device& device, const char* what,
                const char* name) {
  expect(t, shape, type, device, what, name);
  if (t.stride(3) != 1) refuse(std::string(what) + ": " + name + " must have a contiguous head_dim");
  const int64_t head = shape[2] > 1 ? t.stride(2) : shape[3];
  const int64_t tok = shape[1] > 1 ? t.stride(1) : shape[2] * head;
  return {t.data_ptr(), shape[0] > 1 ? t.stride(0) : shape[1] * tok, tok, head};
}

// exponents [rows, tokens, heads]
sdv2_view view3(const at::Tensor& t, at::IntArrayRef shape, const at::Device& device, const char* what, const char* name) {
  expect(t, shape, at::kChar, device, what, name);
  const int64_t head = shape[2] > 1 ? t.stride(2) : 1, tok = shape[1] > 1 ? t.stride(1) : shape[2] * head;
  return {t.data_ptr(), shape[0] > 1 ? t.stride(0) : shape[1] * tok, tok, head};
}

struct Cache {
  sdv2_view k, v, k_exp, v_exp;
  int64_t tokens;
};
Cache cache_of(PyObject* const* a, const at::Device& device, int64_t rows, int64_t heads, int64_t head_dim, const char* what) {
  if (head_dim != 128) refuse(std::string(what) + ": the 8-bit cache has head_dim 128, not " + std::to_string(head_dim));
  const at::Tensor& k = tensor(a[0], what, "k_cache");
  const int64_t tokens = k.dim() == 4 ? k.size(1) : 0;
  const int64_t shape[4] = {rows, tokens, heads, 128};
  const at::IntArrayRef s4(shape, 4), s3(shape, 3);
  return {view4(k, s4, at::kByte, device, what, "k_cache"),
          view4(tensor(a[1], what, "v_cache"), s4, at::kByte, device, what, "v_cache"),
          view3(tensor(a[2], what, "k_exp"), s3, device, what, "k_exp"),
          view3(tensor(a[3], what, "v_exp"), s3, device, what, "v_exp"), tokens};
}

template <typename T>
struct Ints {  // one number per row
  T v[SDV2_MAX_ROWS];
  Ints(PyObject* o, int64_t rows, const char* what) {
    if (rows > SDV2_MAX_ROWS) refuse(std::string(what) + ": at most " + std::to_string(SDV2_MAX_ROWS) + " rows");
    PyObject* seq = PySequence_Fast(o, "expected a sequence of ints");
    if (seq == nullptr) throw Refused();
    const bool enough = PySequence_Fast_GET_SIZE(seq) >= rows;
    for (int64_t i = 0; enough && i < rows; ++i) {
      const long long x = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(seq, i));
      v[i] = static_cast<T>(x);
      if (v[i] != x) v[i] = -1;  // out of the type's range: out of every other range too
    }
    Py_DECREF(seq);
    if (PyErr_Occurred()) throw Refused();
    if (!enough) refuse(std::string(what) + ": one entry per row is needed");
  }
};

long long int_of(PyObject* o) {
  const long long x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) throw Refused();
  return x;
}
int small_int(PyObject* o) {  // what does not fit becomes a value that the callee refuses
  const long long x = int_of(o);
  return x < 0 || x > 0x7FFFFFFF ? -1 : static_cast<int>(x);
}

int code_of(at::ScalarType t, const char* what) {
  if (t == at::kBFloat16) return SDV2_DTYPE_BF16;
  if (t == at::kFloat) return SDV2_DTYPE_F32;
  refuse(std::string(what) + ": unsupported dtype " + at::toString(t));
}

void on_cuda(const at::Device& d, const char* what) {
  if (!d.is_cuda()) refuse(std::string(what) + ": expected CUDA tensors (there is no CPU path)");
}

// Nothing here records a gradient: while gradients are recorded a tensor that wants one is refused, outputs too.
template <typename... Tensors>
void no_gradient(const char* what, const Tensors&... t) {
  if (c10::GradMode::is_enabled() && (t.requires_grad() || ...)) {
    PyErr_SetString(PyExc_RuntimeError, (std::string(what) + " records no gradient: call it under torch.no_grad()").c_str());
    throw Refused();
  }
}

float scale_of(PyObject* o, int64_t head_dim) {
  if (o == Py_None) return static_cast<float>(1.0 / std::sqrt(static_cast<double>(head_dim)));
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw Refused();
  return static_cast<float>(x);
}

const at::Tensor& four_dims(PyObject* o, const char* what, const char* name) {
  const at::Tensor& t = tensor(o, what, name);
  if (t.dim() != 4) refuse(std::string(what) + ": " + name + " must be [rows, tokens, heads, head_dim]");
  return t;
}

at::Tensor out_like(const at::Tensor& q, PyObject* given, const char* what) {
  if (given != Py_None) return tensor(given, what, "out");
  return at::empty(q.sizes(), q.options());
}

at::Tensor scratch_of(size_t bytes, const at::Device& device) {
  return bytes == 0 ? at::Tensor() : at::empty({static_cast<int64_t>(bytes)}, at::TensorOptions().dtype(at::kByte).device(device));
}

void* stream_of(const at::Device& d) { return c10::cuda::getCurrentCUDAStream(d.index()).stream(); }

void checked(int rc, const char* what) {
  if (rc == SDV2_OK) return;
  PyObject* r = PyObject_CallFunction(g_check, "is", rc, what);
  if (r == nullptr) throw Refused();
  Py_DECREF(r);
}

template <typename Call>
int without_gil(const Call& call) {
  PyThreadState* state = PyEval_SaveThread();
  const int rc = call();
  PyEval_RestoreThread(state);
  return rc;
}

template <typename Body>
PyObject* guarded(const Body& body) {
  HANDLE_TH_ERRORS
  try {
    return body();
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

PyObject* wrong_count() {
  PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
  return nullptr;
}

// q, k, v, k_cache, v_cache, k_exp, v_exp, table, grid, start_frames, dst_begin, q_out, index_tensors, index_values,
// step_params, status
PyObject* append_q8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 16) return wrong_count();
  return guarded([&]() -> PyObject* {
    const char* what = "rope_kv_append_q8";
    const at::Tensor& q = four_dims(a[0], what, "q");
    const at::Device dev = q.device();
    const int64_t rows = q.size(0), tokens = q.size(1), heads = q.size(2), dim = q.size(3);
    const auto type = q.scalar_type();
    const int dtype = code_of(type, what);
    const Cache c = cache_of(a + 3, dev, rows, heads, dim, what);
    const at::Tensor& table = tensor(a[7], what, "table");
    if (table.dim() != 3 || table.size(1) != dim / 2 || table.size(2) != 2 || table.scalar_type() != at::kDouble ||
        table.device() != dev || !table.is_contiguous())
      refuse("rope_kv_append_q8: the rope table must be a contiguous float64 [rows, 64, 2] tensor on " + dev.str());
    PyObject* grid = PySequence_Fast(a[8], "grid must be (frames, height, width)");
    if (grid == nullptr) throw Refused();
    int g[3] = {-1, -1, -1};
    const bool three = PySequence_Fast_GET_SIZE(grid) == 3;
    for (int i = 0; three && i < 3; ++i) {
      const long long x = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(grid, i));
      g[i] = x < 0 || x > 0x7FFFFFFF ? -1 : static_cast<int>(x);
    }
    Py_DECREF(grid);
    if (PyErr_Occurred()) throw Refused();
    if (!three) refuse("rope_kv_append_q8: grid must be (frames, height, width)");
    no_gradient(what, q, tensor(a[1], what, "k"), tensor(a[2], what, "v"));
    const at::Tensor out = a[11] != Py_None ? tensor(a[11], what, "q_out") : (on_cuda(dev, what), at::empty(q.sizes(), q.options()));
    no_gradient(what, out);
    const sdv2_view vq = view4(q, q.sizes(), type, dev, what, "q"), vk = view4(tensor(a[1], what, "k"), q.sizes(), type, dev, what, "k"),
                    vv = view4(tensor(a[2], what, "v"), q.sizes(), type, dev, what, "v"),
                    vo = view4(out, q.sizes(), type, dev, what, "q_out");
    int64_t* index[2] = {nullptr, nullptr};
    if (a[12] != Py_None) {
      PyObject* pair = PySequence_Fast(a[12], "index_tensors must be two tensors");
      if (pair == nullptr) throw Refused();
      bool good = PySequence_Fast_GET_SIZE(pair) == 2;
      for (int i = 0; good && i < 2; ++i) {
        PyObject* o = PySequence_Fast_GET_ITEM(pair, i);
        if (!THPVariable_Check(o)) {
          good = false;
          break;
        }
        const at::Tensor& t = THPVariable_Unpack(o);
        good = t.scalar_type() == at::kLong && t.numel() >= rows && t.is_contiguous() && t.device() == dev;
        index[i] = good ? static_cast<int64_t*>(t.data_ptr()) : nullptr;
      }
      Py_DECREF(pair);
      if (!good) refuse("rope_kv_append_q8: index tensors must be contiguous int64 with one entry per row, on q's device");
    }
    on_cuda(dev, what);
    void* status = PyLong_AsVoidPtr(a[15]);
    const c10::cuda::OptionalCUDAGuard guard(dev);
    auto run = [&](const int64_t* starts, const int64_t* slots, const int64_t* params, const int64_t* ge, const int64_t* le) {
      checked(without_gil([&] {
                return g_append(&vq, &vk, &vv, &vo, &c.k, &c.v, &c.k_exp, &c.v_exp, static_cast<int>(rows),
                                static_cast<int>(tokens), static_cast<int>(heads), 128, c.tokens,
                                static_cast<const double*>(table.data_ptr()), static_cast<int>(table.size(0)), g[0], g[1], g[2],
                                starts, slots, params, index[0], index[1], ge, le, dtype, static_cast<int*>(status),
                                stream_of(dev));
              }),
              what);
    };
    if (a[14] != Py_None) {
      const at::Tensor& params = tensor(a[14], what, "step_params");
      if (params.scalar_type() != at::kLong || !params.is_contiguous() || params.numel() != 4 * rows || params.device() != dev)
        refuse("rope_kv_append_q8: step_params must be a contiguous int64 [4, rows] tensor on the same device");
      run(nullptr, nullptr, static_cast<const int64_t*>(params.data_ptr()), nullptr, nullptr);
    } else {
      const Ints<int64_t> starts(a[9], rows, what), slots(a[10], rows, what);
      if (index[0] != nullptr) {
        PyObject* pair = a[13] == Py_None ? nullptr : PySequence_Fast(a[13], "index_values must be two sequences");
        if (pair == nullptr || PySequence_Fast_GET_SIZE(pair) != 2) {
          Py_XDECREF(pair);
          if (PyErr_Occurred()) throw Refused();
          refuse("rope_kv_append_q8: index_values need one entry per row");
        }
        struct Keep {
          PyObject* o;
          ~Keep() { Py_DECREF(o); }
        } keep{pair};
        const Ints<int64_t> ge(PySequence_Fast_GET_ITEM(pair, 0), rows, what), le(PySequence_Fast_GET_ITEM(pair, 1), rows, what);
        run(starts.v, slots.v, nullptr, ge.v, le.v);
      } else {
        run(starts.v, slots.v, nullptr, nullptr, nullptr);
      }
    }
    return THPVariable_Wrap(out);
  });
}

// k_cache, v_cache, k_exp, v_exp, begin, tokens, dtype, out
PyObject* read_q8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8) return wrong_count();
  return guarded([&]() -> PyObject* {
    const char* what = "kv_read_q8";
    const at::Tensor& kc = four_dims(a[0], what, "k_cache");
    const at::Device dev = kc.device();
    const int64_t rows = kc.size(0), heads = kc.size(2);
    const Cache c = cache_of(a, dev, rows, heads, kc.size(3), what);
    const long long tokens = int_of(a[5]);
    if (tokens < 0 || tokens > c.tokens) refuse("kv_read_q8: cannot read " + std::to_string(tokens) + " tokens of " + std::to_string(c.tokens));
    if (!THPDtype_Check(a[6])) refuse("kv_read_q8: dtype must be a torch.dtype");
    const auto type = reinterpret_cast<THPDtype*>(a[6])->scalar_type;
    const int dtype = code_of(type, what);
    const int64_t shape[4] = {rows, tokens, heads, 128};
    const at::IntArrayRef s4(shape, 4);
    const Ints<int64_t> begin(a[4], rows, what);
    at::Tensor out[2];
    if (a[7] != Py_None) {
      PyObject* pair = PySequence_Fast(a[7], "out must be two tensors");
      if (pair == nullptr) throw Refused();
      const bool two = PySequence_Fast_GET_SIZE(pair) == 2 && THPVariable_Check(PySequence_Fast_GET_ITEM(pair, 0)) &&
                       THPVariable_Check(PySequence_Fast_GET_ITEM(pair, 1));
      for (int i = 0; two && i < 2; ++i) out[i] = THPVariable_Unpack(PySequence_Fast_GET_ITEM(pair, i));
      Py_DECREF(pair);
      if (!two) refuse("kv_read_q8: out must be two tensors");
      no_gradient(what, out[0], out[1]);
      on_cuda(dev, what);
    } else {
      on_cuda(dev, what);
      for (auto& t : out) t = at::empty(s4, at::TensorOptions().dtype(type).device(dev));
    }
    const sdv2_view ko = view4(out[0], s4, type, dev, what, "out[0]"), vo = view4(out[1], s4, type, dev, what, "out[1]");
    if (out[0].numel() != 0) {
      const c10::cuda::OptionalCUDAGuard guard(dev);
      checked(without_gil([&] {
                return g_read(&c.k, &c.v, &c.k_exp, &c.v_exp, &ko, &vo, static_cast<int>(rows), static_cast<int>(tokens),
                              static_cast<int>(heads), 128, c.tokens, begin.v, dtype, stream_of(dev));
              }),
              what);
    }
    PyObject* first = THPVariable_Wrap(out[0]);
    PyObject* second = THPVariable_Wrap(out[1]);
    PyObject* both = first != nullptr && second != nullptr ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first);
    Py_XDECREF(second);
    return both;
  });
}

// q, k_cache, v_cache, k_exp, v_exp, seq_lens, out, softmax_scale, status
PyObject* attn_q8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 9) return wrong_count();
  return guarded([&]() -> PyObject* {
    const char* what = "attn_kvcache_q8";
    const at::Tensor& q = four_dims(a[0], what, "q");
    const at::Device dev = q.device();
    const int64_t rows = q.size(0), tokens = q.size(1), heads = q.size(2), dim = q.size(3);
    if (q.scalar_type() != at::kBFloat16) refuse("attn_kvcache_q8: the tensor-core attention kernel takes bf16");
    const Cache c = cache_of(a + 1, dev, rows, heads, dim, what);
    const Ints<int32_t> lens(a[5], rows, what);
    no_gradient(what, q);
    if (a[6] == Py_None) on_cuda(dev, what);
    const at::Tensor out = out_like(q, a[6], what);
    no_gradient(what, out);
    on_cuda(dev, what);
    const sdv2_view vq = view4(q, q.sizes(), at::kBFloat16, dev, what, "q"), vo = view4(out, q.sizes(), at::kBFloat16, dev, what, "out");
    const float scale = scale_of(a[7], dim);
    void* status = PyLong_AsVoidPtr(a[8]);
    const c10::cuda::OptionalCUDAGuard guard(dev);
    if (q.numel() == 0 || c.tokens == 0) return THPVariable_Wrap(const_cast<at::Tensor&>(out).zero_());
    const size_t bytes = g_q8_bytes(static_cast<int>(rows), static_cast<int>(tokens), static_cast<int>(heads), c.tokens, lens.v);
    const at::Tensor scratch = scratch_of(bytes, dev);
    checked(without_gil([&] {
              return g_q8(&vq, &c.k, &c.v, &c.k_exp, &c.v_exp, &vo, static_cast<int>(rows), static_cast<int>(tokens),
                          static_cast<int>(heads), 128, c.tokens, lens.v, scale, bytes ? scratch.data_ptr() : nullptr, bytes,
                          static_cast<int*>(status), stream_of(dev));
            }),
            what);
    return THPVariable_Wrap(out);
  });
}

// q, k, v, begin, end, out, softmax_scale, status
PyObject* spans(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8) return wrong_count();
  return guarded([&]() -> PyObject* {
    const char* what = "attn_spans";
    const at::Tensor& q = four_dims(a[0], what, "q");
    const at::Device dev = q.device();
    const int64_t rows = q.size(0), tokens = q.size(1), heads = q.size(2), dim = q.size(3);
    if (q.scalar_type() != at::kBFloat16) refuse("attn_spans: the tensor-core attention kernel takes bf16");
    const at::Tensor& k = four_dims(a[1], what, "k");
    const int64_t kv[4] = {rows, k.size(1), heads, dim}, sp[2] = {rows, tokens};
    const at::IntArrayRef s4(kv, 4), s2(sp, 2);
    const sdv2_view vk = view4(k, s4, at::kBFloat16, dev, what, "k"), vv = view4(tensor(a[2], what, "v"), s4, at::kBFloat16, dev, what, "v");
    if ((vk.stride_row == 0) != (vv.stride_row == 0)) refuse("attn_spans: k and v are broadcast over rows both or neither");
    const at::Tensor& end = tensor(a[4], what, "end");
    expect(end, s2, at::kInt, dev, what, "end");
    at::Tensor begin;
    if (a[3] != Py_None) {
      begin = tensor(a[3], what, "begin");
      expect(begin, s2, at::kInt, dev, what, "begin");
    }
    no_gradient(what, q, k, tensor(a[2], what, "v"));
    if (a[5] == Py_None) on_cuda(dev, what);
    const at::Tensor out = out_like(q, a[5], what);
    no_gradient(what, out);
    on_cuda(dev, what);
    const sdv2_view vq = view4(q, q.sizes(), at::kBFloat16, dev, what, "q"), vo = view4(out, q.sizes(), at::kBFloat16, dev, what, "out");
    const float scale = scale_of(a[6], dim);
    void* status = PyLong_AsVoidPtr(a[7]);
    const c10::cuda::OptionalCUDAGuard guard(dev);
    if (q.numel() == 0 || kv[1] == 0) return THPVariable_Wrap(const_cast<at::Tensor&>(out).zero_());
    const size_t bytes = g_spans_bytes(static_cast<int>(rows), static_cast<int>(tokens), static_cast<int>(heads), kv[1]);
    const at::Tensor scratch = scratch_of(bytes, dev);
    checked(without_gil([&] {
              return g_spans(&vq, &vk, &vv, &vo, static_cast<int>(rows), static_cast<int>(tokens), static_cast<int>(heads),
                             static_cast<int>(dim), kv[1], begin.defined() ? static_cast<const int32_t*>(begin.data_ptr()) : nullptr,
                             begin.defined() ? begin.stride(0) : 0, begin.defined() ? begin.stride(1) : 0,
                             static_cast<const int32_t*>(end.data_ptr()), end.stride(0), end.stride(1), scale,
                             bytes ? scratch.data_ptr() : nullptr, bytes, static_cast<int*>(status), stream_of(dev));
            }),
            what);
    return THPVariable_Wrap(out);
  });
}

// the six functions' addresses in the order of the declarations above, and check(code, what)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 7) return wrong_count();
  void* f[6];
  for (int i = 0; i < 6; ++i) {
    f[i] = PyLong_AsVoidPtr(a[i]);
    if (f[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "a function is missing");
      return nullptr;
    }
  }
  g_append = reinterpret_cast<decltype(g_append)>(f[0]);
  g_read = reinterpret_cast<decltype(g_read)>(f[1]);
  g_q8_bytes = reinterpret_cast<decltype(g_q8_bytes)>(f[2]);
  g_q8 = reinterpret_cast<decltype(g_q8)>(f[3]);
  g_spans_bytes = reinterpret_cast<decltype(g_spans_bytes)>(f[4]);
  g_spans = reinterpret_cast<decltype(g_spans)>(f[5]);
  Py_INCREF(a[6]);
  Py_XSETREF(g_check, a[6]);
  Py_RETURN_NONE;
}

template <PyObject* (*kFunction)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kFunction));
}

PyMethodDef g_methods[] = {{"append_q8", fast<append_q8>(), METH_FASTCALL, nullptr},
                           {"read_q8", fast<read_q8>(), METH_FASTCALL, nullptr},
                           {"attn_q8", fast<attn_q8>(), METH_FASTCALL, nullptr},
                           {"spans", fast<spans>(), METH_FASTCALL, nullptr},
                           {"bind", fast<bind>(), METH_FASTCALL, nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) { return PyModule_Create(&g_module); }

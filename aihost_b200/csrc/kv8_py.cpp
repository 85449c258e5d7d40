// kv8_py.cpp — the Python module _kv8: torch tensors in, C ABI calls of the 8-bit and the 4-bit cache out.
//
// A decode step makes a few calls per layer, each a few microseconds of GPU time; checking a dozen
// tensors and passing their pointers from Python takes several times that, so it is done here.
// Every check raises AttnError(EINVAL) with the argument's name; what the library refuses raises
// AttnError with its status and message.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/StreamGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdarg.h>
#include <stdio.h>

#include <initializer_list>
#include <type_traits>
#include <utility>

#include "../../include/aihost_attn.h"

namespace {

PyObject* g_error = nullptr;  // aihost_b200.AttnError

struct Raised {};  // a Python exception is set

[[noreturn]] void raise(int status, const char* fmt, ...) {
  char text[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(text, sizeof(text), fmt, ap);
  va_end(ap);
  PyObject* e = g_error ? PyObject_CallFunction(g_error, "is", status, text) : nullptr;
  if (e) {
    PyErr_SetObject(g_error, e);
    Py_DECREF(e);
  } else if (!PyErr_Occurred()) {
    PyErr_SetString(PyExc_RuntimeError, text);
  }
  throw Raised{};
}

void check(aihost_status s) {
  if (s != AIHOST_OK) raise(s, "%s", aihost_attn_last_error());
}

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return v;
}

int32_t int32_of(PyObject* o, const char* name) {
  const int64_t v = integer(o);
  if (v < INT32_MIN || v > INT32_MAX) raise(AIHOST_EINVAL, "%s does not fit 32 bits", name);
  return static_cast<int32_t>(v);
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) raise(AIHOST_EINVAL, "%s must be a tensor", name);
  return THPVariable_Unpack(o);
}

// What every call starts with: (context, device, address of the aihost_kv8_desc, stream or None).
struct Call {
  aihost_attn_ctx* ctx;
  int device;
  aihost_kv8_desc d;
  cudaStream_t stream;
  bool given;  // the stream was named, not torch's current one

  explicit Call(PyObject* const* a) {
    ctx = reinterpret_cast<aihost_attn_ctx*>(integer(a[0]));
    device = static_cast<int>(integer(a[1]));
    d = *reinterpret_cast<const aihost_kv8_desc*>(integer(a[2]));
    given = a[3] != Py_None;
    stream = !given ? c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream()
                             : reinterpret_cast<cudaStream_t>(integer(a[3]));
  }

  // A contiguous tensor of this type on the context's device: its pointer. shape: its exact sizes, or,
  // with at_least, one size that it has to reach.
  template <typename T>
  T* array(PyObject* o, const char* name, at::ScalarType type, std::initializer_list<int64_t> shape,
           bool at_least = false) const {
    const at::Tensor& t = tensor(o, name);
    if (t.scalar_type() != type || !t.is_cuda() || t.get_device() != device || !t.is_contiguous())
      raise(AIHOST_EINVAL, "%s must be a contiguous %s tensor on cuda:%d", name, c10::toString(type), device);
    if (at_least) {
      if (t.numel() < *shape.begin())
        raise(AIHOST_EINVAL, "%s must have at least %lld elements, not %lld", name,
              static_cast<long long>(*shape.begin()), static_cast<long long>(t.numel()));
    } else if (t.sizes() != at::IntArrayRef(shape)) {
      char want[96] = "";
      size_t n = 0;
      for (int64_t s : shape) n += snprintf(want + n, sizeof(want) - n, n ? ", %lld" : "%lld", static_cast<long long>(s));
      raise(AIHOST_EINVAL, "%s must have shape [%s]", name, want);
    }
    return static_cast<T*>(t.data_ptr());
  }
  template <typename T>
  T* maybe(PyObject* o, const char* name, at::ScalarType type, std::initializer_list<int64_t> shape,
           bool at_least = false) const {
    return o == Py_None ? nullptr : array<T>(o, name, type, shape, at_least);
  }

  at::ScalarType io() const { return d.io_dtype == AIHOST_F32 ? at::kFloat : at::kHalf; }

  // [n, heads, head_dim] with the heads packed within a token; tokens may lie apart (a fused
  // projection's output). Returns the bytes between tokens.
  int64_t rows(const at::Tensor& t, const char* name, int32_t heads) const {
    if (t.scalar_type() != io() || !t.is_cuda() || t.get_device() != device || t.dim() != 3 || t.size(1) != heads ||
        t.size(2) != d.head_dim)
      raise(AIHOST_EINVAL, "%s must be %s [n, %d, %d] on cuda:%d", name, c10::toString(io()), heads, d.head_dim, device);
    const int64_t n = t.size(0), packed = static_cast<int64_t>(heads) * d.head_dim;
    if (n > INT32_MAX) raise(AIHOST_EINVAL, "%s has too many tokens", name);
    if (n && (t.stride(2) != 1 || (heads > 1 && t.stride(1) != d.head_dim) || (n > 1 && t.stride(0) < packed)))
      raise(AIHOST_EINVAL, "%s must have its heads packed within a token, and tokens in order", name);
    return (n > 1 ? t.stride(0) : packed) * t.element_size();
  }

  // A pool and what its values are multiplied with: scales of the 8-bit cache, ranges of the 4-bit one.
  template <bool FOUR>
  std::conditional_t<FOUR, uint8_t, int8_t>* pool(PyObject* o, const char* name) const {
    if constexpr (FOUR) return array<uint8_t>(o, name, at::kByte, {d.n_pages, d.n_kv_heads, d.page_rows, d.head_dim / 2});
    else return array<int8_t>(o, name, at::kChar, {d.n_pages, d.n_kv_heads, d.page_rows, d.head_dim});
  }
  template <bool FOUR>
  std::conditional_t<FOUR, void, float>* factors(PyObject* o, const char* name) const {
    if constexpr (FOUR) return array<void>(o, name, at::kHalf, {d.n_pages, d.n_kv_heads, d.page_rows, 2});
    else return array<float>(o, name, at::kFloat, {d.n_pages, d.n_kv_heads});
  }
  at::Tensor make(at::IntArrayRef sizes, at::ScalarType type) const {
    c10::OptionalStreamGuard on;  // a result written on a stream of the caller's is that stream's memory
    if (given) on.reset_stream(c10::cuda::getStreamFromExternal(stream, static_cast<c10::DeviceIndex>(device)));
    return at::empty(sizes, at::TensorOptions().dtype(type).device(at::kCUDA, static_cast<c10::DeviceIndex>(device)));
  }
};

// n elements of `type` of base's storage from element `at` on (counted in that type).
at::Tensor part_of(const at::Tensor& base, at::ScalarType type, int64_t at, int64_t n) {
  auto impl = c10::make_intrusive<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(base.storage()), base.key_set(),
                                                   c10::scalarTypeToTypeMeta(type));
  impl->set_storage_offset(at);
  impl->set_sizes_contiguous({n});
  return at::Tensor(std::move(impl));
}

template <typename F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F&& f) {
  if (got != want) {
    PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd, are wanted", want, got);
    return nullptr;
  }
  try {
    return f();
  } catch (const Raised&) {
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyObject* map_pages(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded(n_args, 11, [&]() -> PyObject* {
    const Call c(a);
    const int32_t most = int32_of(a[4], "max_tokens");
    const at::Tensor& len = tensor(a[5], "seq_len");
    const int64_t n = len.numel();
    if (n > INT32_MAX) raise(AIHOST_EINVAL, "seq_len is too long");
    if (most < 0) raise(AIHOST_EINVAL, "max_tokens (%d) must be >= 0", most);
    const int32_t* seq_len = c.array<int32_t>(a[5], "seq_len", at::kInt, {n});
    const int32_t* n_new = c.array<int32_t>(a[6], "n_new", at::kInt, {n});
    const int32_t* free_pages = c.array<int32_t>(a[7], "free_pages", at::kInt, {c.d.n_pages}, true);
    const int32_t* free_count = c.array<int32_t>(a[8], "free_count", at::kInt, {1});
    int32_t* table = c.array<int32_t>(a[9], "block_table", at::kInt, {n, c.d.max_pages});
    PyObject* out[5];
    if (a[10] == Py_None) {
      // one allocation for the five: slots first, every part on a 16-byte boundary
      const int64_t pos_at = 2 * ((static_cast<int64_t>(most) + 1) / 2 * 2), len_at = pos_at + (most + 3) / 4 * 4;
      const int64_t start_at = len_at + (n + 3) / 4 * 4, count_at = start_at + (n + 4) / 4 * 4;
      const at::Tensor all = c.make({count_at / 2 + 2}, at::kLong);
      const at::Tensor t[5] = {part_of(all, at::kInt, len_at, n), part_of(all, at::kInt, start_at, n + 1),
                               part_of(all, at::kLong, 0, most), part_of(all, at::kInt, pos_at, most),
                               part_of(all, at::kInt, count_at, 1)};
      for (int i = 0; i < 5; ++i) out[i] = THPVariable_Wrap(t[i]);
    } else {
      if (!PyTuple_Check(a[10]) || PyTuple_GET_SIZE(a[10]) != 5) raise(AIHOST_EINVAL, "into must hold five tensors");
      for (int i = 0; i < 5; ++i) {
        out[i] = PyTuple_GET_ITEM(a[10], i);
        Py_INCREF(out[i]);
      }
    }
    PyObject* const result = PyTuple_New(5);
    for (int i = 0; i < 5; ++i) PyTuple_SET_ITEM(result, i, out[i]);
    try {
      check(aihost_page_map(c.ctx, static_cast<int32_t>(n), c.d.page_rows, c.d.n_pages, c.d.max_pages, most, seq_len, n_new,
                            free_pages, free_count, table, c.array<int32_t>(out[0], "kv_len", at::kInt, {n}),
                            c.array<int32_t>(out[1], "row_start", at::kInt, {n + 1}),
                            c.array<int64_t>(out[2], "slots", at::kLong, {most}, true),
                            c.array<int32_t>(out[3], "positions", at::kInt, {most}, true),
                            c.array<int32_t>(out[4], "free_count", at::kInt, {1}), c.stream));
    } catch (const Raised&) {
      Py_DECREF(result);
      throw;
    }
    return result;
  });
}

PyObject* release_pages(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded(n_args, 9, [&]() -> PyObject* {
    const Call c(a);
    const int64_t n = tensor(a[5], "seq_len").numel();
    if (n > INT32_MAX) raise(AIHOST_EINVAL, "seq_len is too long");
    check(aihost_page_release(c.ctx, static_cast<int32_t>(n), c.d.page_rows, c.d.n_pages, c.d.max_pages,
                              c.array<int32_t>(a[4], "done", at::kInt, {n}), c.array<int32_t>(a[5], "seq_len", at::kInt, {n}),
                              c.array<int32_t>(a[8], "block_table", at::kInt, {n, c.d.max_pages}),
                              c.array<int32_t>(a[6], "free_pages", at::kInt, {c.d.n_pages}, true),
                              c.array<int32_t>(a[7], "free_count", at::kInt, {1}), c.stream));
    Py_RETURN_NONE;
  });
}

// The C call of the cache that a function is instantiated for.
template <bool FOUR, typename A, typename B>
constexpr auto pick(A* eight, B* four) {
  if constexpr (FOUR) return four;
  else return eight;
}
#define FOUR_OR_EIGHT(name) pick<FOUR>(aihost_kv8_##name, aihost_kv4_##name)

template <bool FOUR>
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded(n_args, 12, [&]() -> PyObject* {
    Call c(a);
    const at::Tensor &k = tensor(a[4], "k_new"), &v = tensor(a[5], "v_new");
    c.d.kv_token_stride = c.rows(k, "k_new", c.d.n_kv_heads);
    if (c.rows(v, "v_new", c.d.n_kv_heads) != c.d.kv_token_stride || v.size(0) != k.size(0))
      raise(AIHOST_EINVAL, "k_new and v_new must have the same tokens and the same stride between them");
    const int64_t n = k.size(0);
    constexpr auto call = FOUR_OR_EIGHT(append);
    check(call(c.ctx, &c.d, static_cast<int32_t>(n), k.data_ptr(), v.data_ptr(),
               c.array<int64_t>(a[6], "slots", at::kLong, {n}, true),
               c.maybe<int32_t>(a[7], "positions", at::kInt, {n}, true), c.pool<FOUR>(a[8], "k_pool"),
               c.pool<FOUR>(a[9], "v_pool"), c.factors<FOUR>(a[10], FOUR ? "k_range" : "k_scale"),
               c.factors<FOUR>(a[11], FOUR ? "v_range" : "v_scale"), c.stream));
    Py_RETURN_NONE;
  });
}

template <bool FOUR>
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded(n_args, 9, [&]() -> PyObject* {
    const Call c(a);
    const int64_t n = tensor(a[6], "slots").numel();
    if (n > INT32_MAX) raise(AIHOST_EINVAL, "slots is too long");
    const int32_t dtype = int32_of(a[7], "dtype");
    const at::ScalarType type = dtype == AIHOST_F32 ? at::kFloat : at::kHalf;
    const at::Tensor out = a[8] == Py_None ? c.make({n, c.d.n_kv_heads, c.d.head_dim}, type) : tensor(a[8], "out");
    if (a[8] != Py_None) c.array<void>(a[8], "out", type, {n, c.d.n_kv_heads, c.d.head_dim});
    constexpr auto call = FOUR_OR_EIGHT(read);
    check(call(c.ctx, &c.d, static_cast<int32_t>(n), c.array<int64_t>(a[6], "slots", at::kLong, {n}, true),
               c.pool<FOUR>(a[4], "pool"), c.factors<FOUR>(a[5], FOUR ? "range" : "scale"), out.data_ptr(), dtype, c.stream));
    return THPVariable_Wrap(out);
  });
}

template <bool FOUR>
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded(n_args, 18, [&]() -> PyObject* {
    Call c(a);
    const at::Tensor& q = tensor(a[4], "q");
    c.d.q_token_stride = c.rows(q, "q", c.d.n_q_heads);
    const int64_t n = q.size(0), b = tensor(a[6], "kv_len").numel();
    if (b > INT32_MAX) raise(AIHOST_EINVAL, "kv_len is too long");
    const int32_t max_new = int32_of(a[12], "max_new"), max_kv = int32_of(a[13], "max_kv");
    const at::ScalarType type = c.d.out_dtype == AIHOST_F32 ? at::kFloat : at::kHalf;
    const at::Tensor out = a[17] == Py_None ? c.make({n, c.d.n_q_heads, c.d.head_dim}, type) : tensor(a[17], "out");
    if (a[17] != Py_None) c.array<void>(a[17], "out", type, {n, c.d.n_q_heads, c.d.head_dim});
    auto call = [&] {
      constexpr auto attention = FOUR_OR_EIGHT(attention);
      return attention(
          c.ctx, &c.d, static_cast<int32_t>(b), static_cast<int32_t>(n), max_new, max_kv, q.data_ptr(),
          c.array<int32_t>(a[5], "row_start", at::kInt, {b + 1}), c.array<int32_t>(a[6], "kv_len", at::kInt, {b}),
          c.array<int32_t>(a[7], "block_table", at::kInt, {b, c.d.max_pages}), c.pool<FOUR>(a[8], "k_pool"),
          c.pool<FOUR>(a[9], "v_pool"), c.factors<FOUR>(a[10], FOUR ? "k_range" : "k_scale"),
          c.factors<FOUR>(a[11], FOUR ? "v_range" : "v_scale"), c.maybe<int32_t>(a[14], "prefix_len", at::kInt, {b}),
          c.maybe<int32_t>(a[15], "row_first", at::kInt, {n}, true),
          c.maybe<float>(a[16], "alibi_slopes", at::kFloat, {c.d.n_q_heads}), out.data_ptr(), c.stream);
    };
    aihost_status s = call();
    if (s == AIHOST_ENOMEM) {  // the context's scratch is too small: grow it once
      size_t need = 0;
      check((FOUR_OR_EIGHT(plan))(c.ctx, &c.d, static_cast<int32_t>(b), static_cast<int32_t>(n), max_new, max_kv, &need, nullptr));
      check(aihost_attn_reserve(c.ctx, need));
      s = call();
    }
    check(s);
    return THPVariable_Wrap(out);
  });
}

PyObject* set_error(PyObject*, PyObject* cls) {
  Py_XDECREF(g_error);
  Py_INCREF(cls);
  g_error = cls;
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f))
PyMethodDef methods[] = {
    {"set_error", set_error, METH_O, nullptr},
    {"map_pages", FAST(map_pages), METH_FASTCALL, nullptr},
    {"release_pages", FAST(release_pages), METH_FASTCALL, nullptr},
    {"append", FAST(append<false>), METH_FASTCALL, nullptr},
    {"read", FAST(read<false>), METH_FASTCALL, nullptr},
    {"attend", FAST(attend<false>), METH_FASTCALL, nullptr},
    {"append4", FAST(append<true>), METH_FASTCALL, nullptr},
    {"read4", FAST(read<true>), METH_FASTCALL, nullptr},
    {"attend4", FAST(attend<true>), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kv8", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv8(void) { return PyModule_Create(&module); }

// Native call path of the operators between the projections (norm and rotation, the 4-bit cache, attention over it): from the Python
// arguments to the launch without Python code in between.  A call at decode sizes runs 5 to 10 us on the GPU and cost 25 us
// of host time through a Python wrapper (argument checks, torch.empty, a ctypes call of 20 arguments).
//
// Each function checks all that it needs to pass raw pointers on.  It returns None for whatever it does not take on itself -- a check that fails,
// an input off 16 bytes, nothing to do, another device than the current one: the Python function that called it then raises, or serves the call.
#pragma once

namespace attention {

decltype(&xqt_b200_qk_norm_rope) rope_entry = nullptr;
decltype(&xqt_b200_kv4_append) append_entry = nullptr;
decltype(&xqt_b200_kv4_gather) gather_entry = nullptr;
decltype(&xqt_b200_kv4_attention) attention_entry = nullptr;
decltype(&xqt_b200_kv4_attention_workspace_bytes) workspace_entry = nullptr;
PyObject* on_error = nullptr;          // called with (code, symbol): raises
const unsigned int volatile* status_words[64] = {};   // per device, in pinned host memory; null until the Python side has made it

struct NotServed {};

const at::Tensor& tensor(PyObject* o) {
  if (!THPVariable_Check(o)) throw NotServed();
  return THPVariable_Unpack(o);
}
const at::Tensor* maybe(PyObject* o) { return o == Py_None ? nullptr : &tensor(o); }
void need(bool ok) {
  if (!ok) throw NotServed();
}
int device_of(const at::Tensor& t) {
  need(t.is_cuda() && t.layout() == at::kStrided && t.device().index() == c10::cuda::current_device());
  return t.device().index();
}
void on(const at::Tensor& t, int device) { need(t.is_cuda() && t.layout() == at::kStrided && t.device().index() == device); }
bool aligned(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
bool half_type(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }
int code_of(at::ScalarType t) { return t == at::kHalf ? XQT_B200_FP16 : t == at::kBFloat16 ? XQT_B200_BF16 : XQT_B200_FP32; }
int small(int64_t v) {
  need(v >= 0 && v <= INT32_MAX);
  return (int)v;
}
// whether the address ranges that two tensors span meet (neither is empty)
bool overlap(const at::Tensor& a, const at::Tensor& b) {
  auto end = [](const at::Tensor& t) {
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    return reinterpret_cast<uintptr_t>(t.data_ptr()) + (uintptr_t)(last + 1) * t.element_size();
  };
  return reinterpret_cast<uintptr_t>(a.data_ptr()) < end(b) && reinterpret_cast<uintptr_t>(b.data_ptr()) < end(a);
}
// token and head stride of a [tokens, heads, dim] tensor whose channels are contiguous and start on 16 bytes
void rows(const at::Tensor& t, long long* strides) {
  const int64_t token = t.size(0) > 1 ? t.stride(0) : 0, head = t.size(1) > 1 ? t.stride(1) : 0;
  need((t.size(2) <= 1 || t.stride(2) == 1) && aligned(t) && ((token | head) & 7) == 0);
  strides[0] = token;
  strides[1] = head;
}
at::Tensor fresh(at::IntArrayRef shape, at::ScalarType type, int device) {
  return at::detail::empty_cuda(shape, type, c10::Device(c10::kCUDA, (c10::DeviceIndex)device), c10::nullopt);
}
cudaStream_t stream_of(int device) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }
bool failed(int code, const char* symbol) {
  if (code == 0) return false;
  THPObjectPtr r(PyObject_CallFunction(on_error, "is", code, symbol));
  if (r) PyErr_SetString(PyExc_RuntimeError, "library call failed");
  return true;
}
PyObject* pair(at::Tensor a, at::Tensor b, bool has_b) {
  THPObjectPtr x(THPVariable_Wrap(std::move(a)));
  if (!x) return nullptr;
  if (!has_b) return PyTuple_Pack(2, x.get(), Py_None);
  THPObjectPtr y(THPVariable_Wrap(std::move(b)));
  return y ? PyTuple_Pack(2, x.get(), y.get()) : nullptr;
}
template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const NotServed&) {
    Py_RETURN_NONE;
  } catch (...) {
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  }
}

// (q, k, positions, frequencies, axes, q_weight, k_weight, eps, interleaved) -> (q_out, k_out)
PyObject* qk_norm_rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n == 9 && rope_entry != nullptr);
    const at::Tensor& q = tensor(args[0]);
    const at::Tensor *k = maybe(args[1]), *axes = maybe(args[4]), *weights[2] = {maybe(args[5]), maybe(args[6])};
    const at::Tensor &positions = tensor(args[2]), &frequencies = tensor(args[3]);
    const double eps = PyFloat_AsDouble(args[7]);
    if (eps == -1.0 && PyErr_Occurred()) return nullptr;
    const int interleaved = PyObject_IsTrue(args[8]);
    if (interleaved < 0) return nullptr;
    const int device = device_of(q);
    const at::ScalarType type = q.scalar_type();
    need(q.dim() == 3 && half_type(type));
    const int tokens = small(q.size(0)), q_heads = small(q.size(1)), dim = small(q.size(2));
    need(tokens > 0 && q_heads > 0 && dim % 16 == 0 && dim >= 16 && dim <= 256);
    long long strides[10] = {};
    rows(q, strides);
    int k_heads = 0;
    if (k != nullptr) {
      on(*k, device);
      need(k->dim() == 3 && k->scalar_type() == type && k->size(0) == tokens && k->size(2) == dim && k->size(1) > 0);
      k_heads = small(k->size(1));
      rows(*k, strides + 4);
    }
    on(frequencies, device);
    need(frequencies.dim() == 1 && frequencies.scalar_type() == at::kDouble && frequencies.is_contiguous());
    const int pairs = small(frequencies.size(0));
    need(pairs % 8 == 0 && 2 * pairs <= dim);
    on(positions, device);
    const bool wide = positions.scalar_type() == at::kLong;
    const int64_t pd = positions.dim();
    need((wide || positions.scalar_type() == at::kInt) && (pd == 1 || pd == 2) && positions.size(pd - 1) == tokens && (pd == 1 || positions.size(0) > 0));
    strides[8] = pd == 2 ? positions.stride(0) : 0;
    strides[9] = positions.stride(pd - 1);
    if (axes != nullptr) {
      on(*axes, device);
      need(axes->dim() == 1 && axes->scalar_type() == at::kInt && axes->size(0) == pairs && axes->is_contiguous());
    }
    at::ScalarType weight_type = at::kFloat;
    need(k != nullptr || weights[1] == nullptr);
    for (int i = 0; i < 2; ++i) {
      if (weights[i] == nullptr) continue;
      on(*weights[i], device);
      const at::ScalarType t = weights[i]->scalar_type();
      need(weights[i]->dim() == 1 && weights[i]->size(0) == dim && weights[i]->is_contiguous() && (half_type(t) || t == at::kFloat));
      need(i == 0 || weights[0] == nullptr || t == weight_type);
      weight_type = t;
    }
    at::Tensor q_out = fresh({tokens, q_heads, dim}, type, device), k_out;
    rows(q_out, strides + 2);
    if (k != nullptr) {
      k_out = fresh({tokens, k_heads, dim}, type, device);
      rows(k_out, strides + 6);
    }
    int code;
    {
      const cudaStream_t stream = stream_of(device);
      const WithoutGil released;
      code = rope_entry(q.data_ptr(), k ? k->data_ptr() : nullptr, q_out.data_ptr(), k ? k_out.data_ptr() : nullptr,
                        weights[0] ? weights[0]->data_ptr() : nullptr, weights[1] ? weights[1]->data_ptr() : nullptr, positions.data_ptr(),
                        static_cast<const double*>(frequencies.data_ptr()), axes ? static_cast<const int*>(axes->data_ptr()) : nullptr, strides, tokens, q_heads,
                        k_heads, dim, 2 * pairs, pd == 2 ? small(positions.size(0)) : 1, wide, interleaved, code_of(type), code_of(weight_type), (float)eps, stream);
    }
    if (failed(code, "xqt_b200_qk_norm_rope")) return nullptr;
    return pair(std::move(q_out), std::move(k_out), k != nullptr);
  });
}

struct Cache {
  int device, heads, page_size, dim;
  long long pages;
  at::ScalarType type;
};
Cache cache(const at::Tensor& codes, const at::Tensor& params) {
  Cache c;
  c.device = device_of(codes);
  on(params, c.device);
  need(codes.dim() == 5 && codes.size(1) == 2 && codes.scalar_type() == at::kByte && codes.is_contiguous() && params.dim() == 5 && params.is_contiguous());
  c.pages = codes.size(0);
  c.heads = small(codes.size(2));
  c.page_size = small(codes.size(3));
  c.dim = small(2 * codes.size(4));
  c.type = params.scalar_type();
  need((c.dim == 64 || c.dim == 128 || c.dim == 256) && c.heads > 0 && c.pages > 0 && c.page_size >= 16 && c.page_size <= 4096 && (c.page_size & (c.page_size - 1)) == 0);
  need(half_type(c.type) && params.size(0) == c.pages && params.size(1) == 2 && params.size(2) == c.heads && params.size(3) == c.page_size && params.size(4) == 2);
  need(aligned(codes) && aligned(params));
  return c;
}
int slots_of(const at::Tensor& slots, int device) {
  on(slots, device);
  need(slots.dim() == 1 && slots.is_contiguous() && (slots.scalar_type() == at::kLong || slots.scalar_type() == at::kInt) && slots.size(0) > 0);
  return small(slots.size(0));
}

// (k, v, codes, params, slots) -> True
PyObject* kv4_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n == 5 && append_entry != nullptr);
    const at::Tensor &k = tensor(args[0]), &v = tensor(args[1]), &codes = tensor(args[2]), &params = tensor(args[3]), &slots = tensor(args[4]);
    const Cache c = cache(codes, params);
    const int tokens = slots_of(slots, c.device);
    long long strides[4];
    for (int i = 0; i < 2; ++i) {
      const at::Tensor& x = i ? v : k;
      on(x, c.device);
      need(x.dim() == 3 && x.scalar_type() == c.type && x.size(0) == tokens && x.size(1) == c.heads && x.size(2) == c.dim);
      rows(x, strides + 2 * i);
    }
    int code;
    {
      const cudaStream_t stream = stream_of(c.device);
      const WithoutGil released;
      code = append_entry(k.data_ptr(), v.data_ptr(), codes.data_ptr(), params.data_ptr(), slots.data_ptr(), strides, tokens, c.heads, c.dim, c.pages,
                          c.page_size, slots.scalar_type() == at::kLong, code_of(c.type), stream);
    }
    if (failed(code, "xqt_b200_kv4_append")) return nullptr;
    Py_RETURN_TRUE;
  });
}

// (codes, params, slots) -> (k, v)
PyObject* kv4_gather(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n == 3 && gather_entry != nullptr);
    const at::Tensor &codes = tensor(args[0]), &params = tensor(args[1]), &slots = tensor(args[2]);
    const Cache c = cache(codes, params);
    const int tokens = slots_of(slots, c.device);
    at::Tensor k = fresh({tokens, c.heads, c.dim}, c.type, c.device), v = fresh({tokens, c.heads, c.dim}, c.type, c.device);
    int code;
    {
      const cudaStream_t stream = stream_of(c.device);
      const WithoutGil released;
      code = gather_entry(codes.data_ptr(), params.data_ptr(), slots.data_ptr(), k.data_ptr(), v.data_ptr(), tokens, c.heads, c.dim, c.pages, c.page_size,
                          slots.scalar_type() == at::kLong, code_of(c.type), stream);
    }
    if (failed(code, "xqt_b200_kv4_gather")) return nullptr;
    return pair(std::move(k), std::move(v), true);
  });
}

// (q, codes, params, block_table, seq_lens, query_starts, scale, window, out) -> out
PyObject* kv4_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n == 9 && attention_entry != nullptr);
    const at::Tensor &q = tensor(args[0]), &codes = tensor(args[1]), &params = tensor(args[2]), &table = tensor(args[3]), &lens = tensor(args[4]);
    const at::Tensor *starts = maybe(args[5]), *given = maybe(args[8]);
    const Cache c = cache(codes, params);
    need(c.device < 64 && status_words[c.device] != nullptr && *status_words[c.device] == 0);      // (an earlier call's wait ran out: the Python function raises)
    on(q, c.device);
    need(q.dim() == 3 && q.scalar_type() == c.type && q.size(2) == c.dim);
    const int tokens = small(q.size(0)), q_heads = small(q.size(1));
    need(tokens > 0 && q_heads > 0 && q_heads % c.heads == 0);
    long long strides[4] = {};
    rows(q, strides);
    on(table, c.device);
    need(table.dim() == 2 && table.scalar_type() == at::kInt && (table.size(1) <= 1 || table.stride(1) == 1));
    const int batch = small(table.size(0)), width = small(table.size(1));
    strides[2] = table.stride(0);
    on(lens, c.device);
    need(batch > 0 && lens.dim() == 1 && lens.size(0) == batch && lens.scalar_type() == at::kInt && lens.is_contiguous());
    if (starts != nullptr) {
      on(*starts, c.device);
      need(starts->dim() == 1 && starts->size(0) == (int64_t)batch + 1 && starts->scalar_type() == at::kInt && starts->is_contiguous());
    } else {
      need(tokens == batch);
    }
    double scale = 1.0 / std::sqrt((double)c.dim);
    if (args[6] != Py_None) {
      scale = PyFloat_AsDouble(args[6]);
      if (scale == -1.0 && PyErr_Occurred()) return nullptr;
      need(std::fabs(scale) < 0x1p127);              // (false for NaN)
    }
    long long window = 0;
    if (args[7] != Py_None) {
      need(PyLong_Check(args[7]));
      int overflow = 0;
      window = PyLong_AsLongLongAndOverflow(args[7], &overflow);
      need(overflow == 0 && window >= 1);
      if (window > INT32_MAX) window = INT32_MAX;
    }
    at::Tensor out;
    if (given != nullptr) {
      on(*given, c.device);
      need(given->scalar_type() == c.type && given->sizes() == q.sizes() && given->is_contiguous() && aligned(*given));
      need((given->data_ptr() == q.data_ptr() && q.is_contiguous()) || !overlap(q, *given));
      out = *given;
    } else {
      out = fresh({tokens, q_heads, c.dim}, c.type, c.device);
    }
    const size_t bytes = workspace_entry(tokens, batch, q_heads, c.heads, c.dim, starts != nullptr);
    at::Tensor workspace = fresh({(int64_t)bytes}, at::kByte, c.device);       // the allocator's: each captured graph has its own
    int code;
    {
      const cudaStream_t stream = stream_of(c.device);
      const WithoutGil released;
      code = attention_entry(q.data_ptr(), codes.data_ptr(), params.data_ptr(), static_cast<const int*>(table.data_ptr()), static_cast<const int*>(lens.data_ptr()),
                             starts ? static_cast<const int*>(starts->data_ptr()) : nullptr, out.data_ptr(), strides, tokens, batch, q_heads, c.heads, c.dim, c.pages,
                             c.page_size, width, (int)window, code_of(c.type), (float)scale, workspace.data_ptr(), bytes, const_cast<unsigned int*>(status_words[c.device]), stream);
    }
    if (failed(code, "xqt_b200_kv4_attention")) return nullptr;
    if (given != nullptr) {
      Py_INCREF(args[8]);
      return args[8];
    }
    return THPVariable_Wrap(std::move(out));
  });
}

// set_attention_entries(rope, append, gather, attention, workspace_bytes, on_error): addresses in the library
PyObject* set_entries(PyObject*, PyObject* args) {
  unsigned long long at[5];
  PyObject* error;
  if (!PyArg_ParseTuple(args, "KKKKKO", &at[0], &at[1], &at[2], &at[3], &at[4], &error)) return nullptr;
  Py_INCREF(error);
  Py_XSETREF(on_error, error);
  rope_entry = reinterpret_cast<decltype(rope_entry)>(at[0]);
  append_entry = reinterpret_cast<decltype(append_entry)>(at[1]);
  gather_entry = reinterpret_cast<decltype(gather_entry)>(at[2]);
  attention_entry = reinterpret_cast<decltype(attention_entry)>(at[3]);
  workspace_entry = reinterpret_cast<decltype(workspace_entry)>(at[4]);
  Py_RETURN_NONE;
}

// set_status_word(device, address): of a pinned tensor that lives as long as the process
PyObject* set_status_word(PyObject*, PyObject* args) {
  int device;
  unsigned long long at;
  if (!PyArg_ParseTuple(args, "iK", &device, &at)) return nullptr;
  if (device >= 0 && device < 64) status_words[device] = reinterpret_cast<const unsigned int volatile*>(at);
  Py_RETURN_NONE;
}

#define XQT_FASTCALL(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)), METH_FASTCALL

}  // namespace attention

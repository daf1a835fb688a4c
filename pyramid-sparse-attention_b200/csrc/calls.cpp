// The ordinary calls of the answering operators from Python in one step: look at the tensors, make the outputs, launch.
//
// A single token's operators take 2 to 8 us on the device.  Looking at their tensors from Python, making outputs there and passing
// twenty arguments through ctypes took 17 to 22 us a call; here it is 1 to 2 us beside the launch.  Each function returns its result
// (tensors; a status code where the library refused the call), or None for whatever is out of the ordinary - a tensor on the CPU, rows
// that are not whole words, a wrong shape, a tangent - which the wrapper in ops.py then lays out or refuses with a reason.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <string>

#include "psa_b200.h"

namespace {

constexpr int kDevices = 64;
int32_t* status_words[kDevices];   // set by status(); never freed

// A plain strided CUDA tensor on the device of the given index (or any, where it is -1).
const at::Tensor* plain(PyObject* o, int index = -1) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage() || t.is_neg() || t.is_conj()) return nullptr;
  const int at = t.get_device();
  if (at < 0 || at >= kDevices || (index >= 0 && at != index)) return nullptr;
  return &t;
}

const at::Tensor* ints(PyObject* o, int index, int dims) {
  const at::Tensor* t = plain(o, index);
  return t && t->scalar_type() == at::kInt && t->dim() == dims && t->is_contiguous() ? t : nullptr;
}

int type_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return PSA_F32;
    case at::kHalf: return PSA_F16;
    case at::kBFloat16: return PSA_BF16;
    default: return -1;
  }
}

// [B, H, S, D] whose rows are whole 16-byte words wherever they lie -> its strides of batch, head and token.
bool rows_of(const at::Tensor& x, int64_t* strides) {
  if (x.dim() != 4 || x.stride(3) != 1 || ((uintptr_t)x.const_data_ptr() & 15)) return false;
  const int64_t word = 16 / x.element_size();
  for (int i = 0; i < 3; ++i) {
    if (x.size(i) == 0) return false;
    strides[i] = x.size(i) > 1 ? x.stride(i) : 0;
    if (strides[i] % word) return false;
  }
  return x.size(3) > 0;
}

// A new tensor in x's order of dimensions, as torch.empty_like makes it.
at::Tensor rows_like(const at::Tensor& x) {
  if (x.is_non_overlapping_and_dense()) return at::Tensor(at::detail::empty_strided_cuda(x.sizes(), x.strides(), x.scalar_type(), x.device()));
  return at::empty_like(x);
}

at::Tensor made(at::IntArrayRef sizes, at::ScalarType type, const at::Device& on) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, on, std::nullopt));
}

// n numbers of a vector, from number `at` on, as a tensor of their own: two that live and die together in one piece of memory.
at::Tensor part(const at::Tensor& x, int64_t at, int64_t n) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(x.storage()), x.key_set(), x.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(at);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return t;
}

bool integer(PyObject* o, int64_t& n) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  n = PyLong_AsLongLongAndOverflow(o, &overflow);
  return overflow == 0;
}

bool wants_gradient(const at::Tensor& x) { return at::GradMode::is_enabled() && x.requires_grad(); }

// Whether a derivative in forward mode is asked for: x has a tangent.
bool wants_tangent(const at::Tensor& x) { return x._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode(); }

PyObject* none() { Py_RETURN_NONE; }

// Without the interpreter's lock: a launch may wait for room in the stream's queue.
template <typename F> int called(F f) {
  pybind11::gil_scoped_release without_lock;
  return f();
}

PyObject* tensors(std::initializer_list<at::Tensor> ts) {
  PyObject* out = PyTuple_New((Py_ssize_t)ts.size());
  if (!out) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) PyTuple_SET_ITEM(out, i++, THPVariable_Wrap(t));
  return out;
}

// status(index, address): the device's status word
PyObject* status(PyObject*, PyObject* const* args, Py_ssize_t n) {
  int64_t index, address;
  if (n != 2 || !integer(args[0], index) || !integer(args[1], address) || index < 0) {
    PyErr_SetString(PyExc_TypeError, "status(index, address)");
    return nullptr;
  }
  if (index < kDevices) status_words[index] = reinterpret_cast<int32_t*>(address);
  Py_RETURN_NONE;
}

struct Buffer {   // of a ctypes array
  Py_buffer view;
  bool held;
  explicit Buffer(PyObject* o) : held(PyObject_GetBuffer(o, &view, PyBUF_SIMPLE) == 0) {}
  ~Buffer() {
    if (held) PyBuffer_Release(&view);
  }
};

// Turned copies of 1 or 2 tensors.  turns, axes: of each channel pair, as psa_rotate_axes takes them.
struct Rotation {
  const at::Tensor* pos;
  const uint64_t* turns;
  const uint8_t* axes;
  int64_t pairs;
  int half, inverse;

  bool fits(const at::Tensor& x) const {   // besides its rows
    const int dims = (int)pos->dim();
    return x.dim() == 4 && x.size(3) == 2 * pairs && x.size(1) <= INT32_MAX && x.size(2) == pos->size(dims - 1) &&
           (dims == 2 || pos->size(1) == x.size(0) || pos->size(1) == 1) && type_of(x) >= 0;
  }
  // Status of the call; -1: a result whose rows would not be words
  int run(const at::Tensor* const* xs, int n, at::Tensor* outs) const {
    int64_t src_strides[6], dst_strides[6];
    const void* src[2];
    void* dst[2];
    int32_t heads[2];
    const at::Tensor& x = *xs[0];
    c10::cuda::CUDAGuard guard(x.device());
    for (int i = 0; i < n; ++i) {
      outs[i] = rows_like(*xs[i]);
      if (!rows_of(*xs[i], src_strides + 3 * i) || !rows_of(outs[i], dst_strides + 3 * i)) return -1;
      src[i] = xs[i]->const_data_ptr();
      dst[i] = outs[i].data_ptr();
      heads[i] = (int32_t)xs[i]->size(1);
    }
    const int dims = (int)pos->dim();
    const int64_t pos_strides[3] = {pos->stride(0), dims == 3 && pos->size(1) > 1 ? pos->stride(1) : 0, pos->stride(dims - 1)};
    return psa_rotate_axes(src, src_strides, dst, dst_strides, heads, n, pos->const_data_ptr(), 8 * (int)pos->element_size(), pos_strides, turns, axes,
                           (int)pos->size(0), x.size(0), x.size(2), (int)(2 * pairs), half, inverse, type_of(x),
                           c10::cuda::getCurrentCUDAStream(x.get_device()).stream());
  }
};

// The same with a gradient, which is the rotation back through the same function: it can be differentiated again.  (As a function of the Python
// interpreter a step of a few tokens took 110 us of the host with its gradients, as this one 77.)
struct Rotate : torch::autograd::Function<Rotate> {
  using Context = torch::autograd::AutogradContext;
  static torch::autograd::variable_list forward(Context* ctx, const at::Tensor& positions, const std::string& turns, const std::string& axes, bool half,
                                                bool inverse, const at::Tensor& q, const std::optional<at::Tensor>& k) {
    ctx->saved_data["turns"] = turns;
    ctx->saved_data["axes"] = axes;
    ctx->saved_data["half"] = half;
    ctx->saved_data["inverse"] = inverse;
    ctx->save_for_backward({positions});
    ctx->set_materialize_grads(false);
    const Rotation rotation = {&positions, reinterpret_cast<const uint64_t*>(turns.data()), reinterpret_cast<const uint8_t*>(axes.data()),
                               (int64_t)axes.size(), half, inverse};
    // gradients come in any layout
    at::Tensor xs[2] = {q, k ? *k : at::Tensor()}, outs[2];
    const int n = 1 + k.has_value();
    const at::Tensor* at[2] = {xs, xs + 1};
    for (int i = 0; i < n; ++i) {
      int64_t unused[3];
      TORCH_CHECK(xs[i].is_cuda() && xs[i].get_device() == positions.get_device() && rotation.fits(xs[i]) && xs[i].scalar_type() == q.scalar_type() &&
                      xs[i].size(0) == q.size(0), "rotate_axes: a gradient of another shape, type or device");
      if (!rows_of(xs[i], unused)) xs[i] = xs[i].clone(at::MemoryFormat::Contiguous);
    }
    int rc = rotation.run(at, n, outs);
    if (rc == -1) {   // an order of dimensions that breaks rows apart
      for (int i = 0; i < n; ++i) xs[i] = xs[i].clone(at::MemoryFormat::Contiguous);
      rc = rotation.run(at, n, outs);
    }
    TORCH_CHECK(rc == 0, "psa_rotate_axes: ", psa_last_error_string(), " (status ", rc, ")");
    return k ? torch::autograd::variable_list{outs[0], outs[1]} : torch::autograd::variable_list{outs[0]};
  }
  static torch::autograd::variable_list backward(Context* ctx, torch::autograd::variable_list grads) {
    torch::autograd::variable_list back(7);
    const bool q = grads[0].defined() && ctx->needs_input_grad(1), k = grads.size() > 1 && grads[1].defined() && ctx->needs_input_grad(2);
    if (!q && !k) return back;
    const auto turned = apply(ctx->get_saved_variables()[0], ctx->saved_data["turns"].toStringRef(), ctx->saved_data["axes"].toStringRef(),
                              ctx->saved_data["half"].toBool(), !ctx->saved_data["inverse"].toBool(), q ? grads[0] : grads[1],
                              q && k ? std::optional<at::Tensor>(grads[1]) : std::nullopt);
    if (q) back[5] = turned[0];
    if (k) back[6] = turned[q ? 1 : 0];
    return back;
  }
};

// rotate(q, k or None, positions [axes, (B or 1,) S], turns, axis of pairs, half, inverse, axes) -> tuple
PyObject* rotate(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t axes;
  if (n != 8 || !integer(args[7], axes)) return none();
  const at::Tensor* q = plain(args[0]);
  if (!q) return none();
  const int index = q->get_device(), count = args[1] != Py_None ? 2 : 1;
  const at::Tensor* xs[2] = {q, count == 2 ? plain(args[1], index) : nullptr};
  const at::Tensor* pos = plain(args[2], index);
  if (!pos || (count == 2 && !xs[1]) || (pos->scalar_type() != at::kInt && pos->scalar_type() != at::kLong) || (pos->dim() != 2 && pos->dim() != 3) ||
      pos->size(0) != axes)
    return none();
  Buffer turns(args[3]), axis(args[4]);
  if (!turns.held || !axis.held || turns.view.len != 8 * axis.view.len) {
    PyErr_Clear();
    return none();
  }
  const Rotation rotation = {pos, static_cast<const uint64_t*>(turns.view.buf), static_cast<const uint8_t*>(axis.view.buf), (int64_t)axis.view.len,
                             args[5] == Py_True, args[6] == Py_True};
  bool gradient = false;
  for (int i = 0; i < count; ++i) {
    int64_t unused[3];
    if (!rotation.fits(*xs[i]) || !rows_of(*xs[i], unused) || xs[i]->scalar_type() != q->scalar_type() || xs[i]->size(0) != q->size(0) || wants_tangent(*xs[i]))
      return none();
    gradient = gradient || wants_gradient(*xs[i]);
  }
  at::Tensor outs[2];
  if (gradient) {
    const std::string turns_of(static_cast<const char*>(turns.view.buf), (size_t)turns.view.len), axis_of(static_cast<const char*>(axis.view.buf), (size_t)axis.view.len);
    pybind11::gil_scoped_release without_lock;
    const auto turned = Rotate::apply(*pos, turns_of, axis_of, (bool)rotation.half, (bool)rotation.inverse, *q, count == 2 ? std::optional<at::Tensor>(*xs[1]) : std::nullopt);
    for (int i = 0; i < count; ++i) outs[i] = turned[i];
  } else {
    const int rc = called([&] { return rotation.run(xs, count, outs); });
    if (rc == -1) return none();
    if (rc) return PyLong_FromLong(rc);
  }
  return count == 2 ? tensors({outs[0], outs[1]}) : tensors({outs[0]});
  END_HANDLE_TH_ERRORS
}

// plan_pages(table, lengths, counts, pool, free, page_size, tokens, out or None) -> (table, lengths, free, slots)
PyObject* plan_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) return none();
  const at::Tensor* table = plain(args[0]);
  if (!table) return none();
  const int index = table->get_device();
  if (!status_words[index]) return none();
  table = ints(args[0], index, 2);
  const at::Tensor *lengths = ints(args[1], index, 1), *counts = ints(args[2], index, 1), *pool = ints(args[3], index, 1), *free = ints(args[4], index, 1);
  int64_t page, tokens;
  if (!table || !lengths || !counts || !pool || !free || !integer(args[5], page) || !integer(args[6], tokens)) return none();
  const int64_t requests = table->size(0), width = table->size(1);
  if (requests < 1 || width < 1 || pool->size(0) < 1 || lengths->size(0) != requests || counts->size(0) != requests || free->size(0) != 1 || page < 16 ||
      page % 16 || page > INT32_MAX || tokens < 1)
    return none();
  at::Tensor out[3];
  if (args[7] != Py_None) {
    if (!PyTuple_CheckExact(args[7]) || PyTuple_GET_SIZE(args[7]) != 3) return none();
    for (int i = 0; i < 3; ++i) {
      const at::Tensor* t = ints(PyTuple_GET_ITEM(args[7], i), index, i ? 1 : 2);
      if (!t || t->sizes() != (i == 0 ? table : i == 1 ? lengths : free)->sizes()) return none();
      out[i] = *t;
    }
  }
  c10::cuda::CUDAGuard guard(table->device());
  if (args[7] == Py_None) {
    out[0] = made(table->sizes(), at::kInt, table->device());
    const at::Tensor counts_of = made({requests + 1}, at::kInt, table->device());
    out[1] = part(counts_of, 0, requests), out[2] = part(counts_of, requests, 1);
  }
  const at::Tensor slots = made({requests, tokens}, at::kInt, table->device());
  const size_t bytes = args[7] == Py_None && requests <= 1024 ? 0 : psa_plan_pages_scratch_bytes(requests);
  const at::Tensor scratch = bytes ? made({(int64_t)bytes}, at::kByte, table->device()) : at::Tensor();
  void* stream = c10::cuda::getCurrentCUDAStream(index).stream();
  const int rc = called([&] {
    return psa_plan_pages(table->const_data_ptr<int32_t>(), lengths->const_data_ptr<int32_t>(), counts->const_data_ptr<int32_t>(),
                          pool->const_data_ptr<int32_t>(), free->const_data_ptr<int32_t>(), out[0].data_ptr<int32_t>(), out[1].data_ptr<int32_t>(),
                          out[2].data_ptr<int32_t>(), slots.data_ptr<int32_t>(), bytes ? scratch.data_ptr() : nullptr, bytes, requests, width, pool->size(0), (int)page,
                          tokens, status_words[index], stream);
  });
  if (rc) return PyLong_FromLong(rc);
  return tensors({out[0], out[1], out[2], slots});
  END_HANDLE_TH_ERRORS
}

// The cache's tensor: uint8 [pages, heads, page / 16, slice], as head_dim and group want it.
const at::Tensor* cache_of(PyObject* o, int64_t dim, int64_t group) {
  const at::Tensor* t = plain(o);
  if (!t || t->scalar_type() != at::kByte || t->dim() != 4 || !t->is_contiguous() || t->numel() == 0 || dim > INT32_MAX || dim < 1 || group < 1 ||
      group > INT32_MAX || t->size(1) > INT32_MAX || t->size(2) > INT32_MAX / 16)
    return nullptr;
  const size_t slice = psa_kv4_slice_bytes((int)dim, (int)group);
  return slice && (int64_t)slice == t->size(3) ? t : nullptr;
}

// append(data, k, v, slots, group) -> 0
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t group, strides[6];
  if (n != 5 || !integer(args[4], group)) return none();
  const at::Tensor* k = plain(args[1]);
  if (!k || k->dim() != 4) return none();
  const int index = k->get_device();
  const at::Tensor *v = plain(args[2], index), *slots = ints(args[3], index, 2), *data = cache_of(args[0], k->size(3), group);
  const int type = type_of(*k);
  if (!v || !slots || !data || data->get_device() != index || type <= PSA_F32 || v->scalar_type() != k->scalar_type() || v->sizes() != k->sizes() ||
      !status_words[index] || !rows_of(*k, strides) || !rows_of(*v, strides + 3) || data->size(1) != k->size(1) || slots->size(0) != k->size(0) || slots->size(1) != k->size(2))
    return none();
  c10::cuda::CUDAGuard guard(k->device());
  void* stream = c10::cuda::getCurrentCUDAStream(index).stream();
  return PyLong_FromLong(called([&] {
    return psa_kv4_append(data->data_ptr(), k->const_data_ptr(), v->const_data_ptr(), strides, slots->const_data_ptr<int32_t>(), data->size(0),
                          (int)data->size(1), 16 * (int)data->size(2), k->size(0), k->size(2), (int)k->size(3), (int)group, type, status_words[index],
                          stream);
  }));
  END_HANDLE_TH_ERRORS
}

// read(data, slots, head_dim, group, code of the type) -> (keys, values)
PyObject* read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t dim, group, code;
  if (n != 5 || !integer(args[2], dim) || !integer(args[3], group) || !integer(args[4], code)) return none();
  const at::Tensor* data = cache_of(args[0], dim, group);
  if (!data) return none();
  const int index = data->get_device();
  const at::Tensor* slots = ints(args[1], index, 2);
  if (!status_words[index] || !slots || slots->numel() == 0 || (code != PSA_BF16 && code != PSA_F16)) return none();
  c10::cuda::CUDAGuard guard(data->device());
  const at::ScalarType type = code == PSA_BF16 ? at::kBFloat16 : at::kHalf;
  const int64_t batch = slots->size(0), heads = data->size(1), tokens = slots->size(1);
  const at::Tensor k = made({batch, heads, tokens, dim}, type, data->device()), v = made({batch, heads, tokens, dim}, type, data->device());
  const int64_t strides[6] = {heads * tokens * dim, tokens * dim, dim, heads * tokens * dim, tokens * dim, dim};
  void* stream = c10::cuda::getCurrentCUDAStream(index).stream();
  const int rc = called([&] {
    return psa_kv4_read(data->const_data_ptr(), k.data_ptr(), v.data_ptr(), strides, slots->const_data_ptr<int32_t>(), data->size(0), (int)heads,
                        16 * (int)data->size(2), batch, tokens, (int)dim, (int)group, (int)code, status_words[index], stream);
  });
  if (rc) return PyLong_FromLong(rc);
  return tensors({k, v});
  END_HANDLE_TH_ERRORS
}

// attend(q, data, table, lengths, group, counts or None, sm_scale or None, with lse) -> (out,) or (out, lse)
PyObject* attend(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t group, q_strides[3], out_strides[3];
  if (n != 8 || !integer(args[4], group)) return none();
  const at::Tensor* q = plain(args[0]);
  if (!q || !rows_of(*q, q_strides)) return none();
  const int index = q->get_device(), type = type_of(*q);
  const int64_t batch = q->size(0), heads = q->size(1), tokens = q->size(2), dim = q->size(3);
  const at::Tensor *data = cache_of(args[1], dim, group), *table = ints(args[2], index, 2), *lengths = ints(args[3], index, 1);
  const at::Tensor* counts = args[5] == Py_None ? nullptr : ints(args[5], index, 1);
  if (!status_words[index] || !data || data->get_device() != index || !table || !lengths || (!counts && args[5] != Py_None) || type <= PSA_F32) return none();
  if (table->size(0) != batch || table->size(1) < 1 || lengths->size(0) != batch || (counts && counts->size(0) != batch) || heads > INT32_MAX ||
      heads % data->size(1))
    return none();
  float scale = (float)(1. / std::sqrt((double)dim));
  if (args[6] != Py_None) {
    if (!PyFloat_CheckExact(args[6])) return none();
    scale = (float)PyFloat_AS_DOUBLE(args[6]);
  }
  const size_t bytes = psa_kv4_attention_scratch_bytes(batch, tokens, (int)heads, (int)data->size(1), (int)dim);
  if (!bytes) return none();
  c10::cuda::CUDAGuard guard(q->device());
  const at::Tensor out = rows_like(*q);
  if (!rows_of(out, out_strides)) return none();
  const at::Tensor scratch = made({(int64_t)bytes}, at::kByte, q->device());
  const bool with_lse = args[7] == Py_True;
  const at::Tensor lse = with_lse ? made({batch, heads, tokens}, at::kFloat, q->device()) : at::Tensor();
  void* stream = c10::cuda::getCurrentCUDAStream(index).stream();
  const int rc = called([&] {
    return psa_kv4_attention(q->const_data_ptr(), q_strides, data->const_data_ptr(), table->const_data_ptr<int32_t>(), lengths->const_data_ptr<int32_t>(),
                             counts ? counts->const_data_ptr<int32_t>() : nullptr, out.data_ptr(), out_strides, with_lse ? lse.data_ptr<float>() : nullptr,
                             scratch.data_ptr(), bytes, data->size(0), 16 * (int)data->size(2), table->size(1), batch, tokens, (int)heads,
                             (int)data->size(1), (int)dim, (int)group, scale, type, status_words[index], stream);
  });
  if (rc) return PyLong_FromLong(rc);
  return with_lse ? tensors({out, lse}) : tensors({out});
  END_HANDLE_TH_ERRORS
}

#define CALL(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {CALL(status), CALL(rotate), CALL(plan_pages), CALL(append), CALL(read), CALL(attend), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }
